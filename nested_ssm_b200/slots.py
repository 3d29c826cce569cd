"""Moves of slots: the states of sequences copied, forked, freed, compacted and reordered on the
device, in every buffer and layer that holds them.

``buffers`` is a :class:`~nested_ssm_b200.pool.TieredSlotPool` (all its buffers move together) or
a :class:`StateBuffers` of any slot-indexed tensors (the states of
:func:`~nested_ssm_b200.delta.gated_delta_state_update`, conv states, ...).  Slot lists are int32
tensors on the buffers' device; nothing is copied to the host.  A list is checked on the device before
any byte moves: moves out of range, into a slot named twice as a destination, or into a slot that
another move reads are dropped, and ``check_status()`` of the buffers raises for them.
"""
from __future__ import annotations

import torch

from . import _lib
from .pool import TieredSlotPool


def _layers_overlap(row, slot_stride, slots, outer_stride, layers):
    """Whether two slots of different layers share memory: the distance of a pair is least for the slots next to the
    layers' distance."""
    for n in range(1, layers):
        k = n * outer_stride // slot_stride if slots > 1 else 0
        if any(abs(n * outer_stride - m * slot_stride) < row for m in (k, k + 1) if m < slots):
            return True
    return False


def _describe(tensors, slot_dim):
    """One ``nssm_slot_buffer`` per tensor."""
    bufs = (_lib.NssmSlotBuffer * len(tensors))()
    for d, t in zip(bufs, tensors):
        es = t.element_size()
        row = 1
        for stride, size in sorted(zip(t.stride()[slot_dim + 1:], t.shape[slot_dim + 1:])):   # in any order of the axes
            if size != 1 and stride != row:
                raise ValueError(f"the values of a slot must be contiguous, got shape {tuple(t.shape)} strides {t.stride()}")
            row *= size
        if t.stride(slot_dim) < row and t.shape[slot_dim] > 1:
            raise ValueError("the slots of a buffer overlap")
        if slot_dim and _layers_overlap(row, t.stride(1), t.shape[1], t.stride(0), t.shape[0]):
            raise ValueError("the layers of a buffer overlap")
        d.base, d.row_bytes, d.slot_stride = t.data_ptr(), row * es, t.stride(slot_dim) * es
        d.outer, d.outer_stride = (t.shape[0], t.stride(0) * es) if slot_dim else (1, 0)
    return bufs


class StateBuffers:
    """Slot-indexed tensors that move together: each ``[S, ...]`` (``slot_dim=0``) or
    ``[layers, S, ...]`` (``slot_dim=1``), any dtype, the values of a slot contiguous in memory (their
    axes in any order: a channels-last conv state is one)."""

    def __init__(self, tensors, slot_dim: int = 0):
        tensors = [tensors] if isinstance(tensors, torch.Tensor) else list(tensors)
        if slot_dim not in (0, 1):
            raise ValueError(f"slot_dim must be 0 or 1, got {slot_dim}")
        if not 1 <= len(tensors) <= _lib.MAX_SLOT_BUFFERS:
            raise ValueError(f"1 to {_lib.MAX_SLOT_BUFFERS} tensors expected, got {len(tensors)}")
        for t in tensors:
            if t.dim() <= slot_dim or t.shape[slot_dim] != tensors[0].shape[slot_dim] or t.numel() == 0:
                raise ValueError(f"every tensor needs the same slots at dim {slot_dim}, got {tuple(t.shape)}")
        self.num_slots = tensors[0].shape[slot_dim]
        if self.num_slots > _lib.MAX_MOVE_SLOTS:
            raise ValueError(f"{self.num_slots} slots; at most {_lib.MAX_MOVE_SLOTS}")
        self.tensors, self.slot_dim = tensors, slot_dim
        self._bufs = _describe(tensors, slot_dim)
        _lib.device_index(*tensors)
        self.device = tensors[0].device
        self.status = torch.zeros(1, dtype=torch.int32, device=self.device)

    def check_status(self) -> None:
        """Raise if a move was dropped since the last call (synchronises)."""
        v = int(self.status.item())
        if v:
            self.status.zero_()
            what = [w for bit, w in ((1, f"a slot index outside [0, {self.num_slots})"),
                                     (_lib.NSSM_STATUS_CONFLICT, "a slot named twice or both read and written"))
                    if v & bit]
            raise IndexError(f"nested_ssm: {'; '.join(what) or 'error'} (status {v})")


def _target(buffers):
    """(descriptor array, slots, device, status) of a pool or StateBuffers."""
    if isinstance(buffers, StateBuffers):
        return buffers._bufs, buffers.num_slots, buffers.device, buffers.status
    if not isinstance(buffers, TieredSlotPool):
        raise TypeError(f"buffers must be a TieredSlotPool or StateBuffers, got {type(buffers).__name__}")
    if buffers._slot_bufs is None:
        buffers._slot_bufs = _describe([t for t in (buffers.hot, buffers.cold, buffers.scale, buffers.glog, buffers.t,
                                                    buffers.ring_x, buffers.ring_dt, buffers.ring_b)
                                        if t is not None], 1)
    return buffers._slot_bufs, buffers.S, buffers.device, buffers.status


def _list(t, name, n=None):
    t = _lib.int32_list(t, name)
    rows = t.numel()
    if n is not None and rows != n:
        raise ValueError(f"{name} has {rows} entries, expected {n}")
    if rows > _lib.MAX_SLOT_ROWS:
        raise ValueError(f"{name} has {rows} rows; at most {_lib.MAX_SLOT_ROWS} in one call")
    return t


def _workspace(n, device):
    return torch.empty(8 + 8 * max(n, 1), dtype=torch.uint8, device=device)


def _copy(buffers, src, dst, pad_slot_id):
    bufs, S, where, status = _target(buffers)
    n = dst.numel()
    dev = _lib.device_index(status, src, dst)
    ws = _workspace(n, where)
    _lib.call(_lib.load().nssm_slot_copy, dev, bufs, len(bufs), S, None if src is None else src.data_ptr(), dst.data_ptr(),
              n, int(pad_slot_id), ws.data_ptr(), ws.numel(), status.data_ptr())


def copy_slots(buffers, src: torch.Tensor, dst: torch.Tensor, pad_slot_id: int = -1) -> None:
    """Slot ``dst[i]`` becomes a copy of slot ``src[i]``; naming a source several times forks it.
    Pairs with ``pad_slot_id`` are skipped, a pair with ``src == dst`` does nothing."""
    src = _list(src, "src")
    _copy(buffers, src, _list(dst, "dst", src.numel()), pad_slot_id)


def clear_slots(buffers, slots: torch.Tensor, pad_slot_id: int = -1) -> None:
    """Free slots: every value of the named slots becomes zero, an empty state for the next
    sequence."""
    _copy(buffers, None, _list(slots, "slots"), pad_slot_id)


def compact_slots(buffers, slots: torch.Tensor, pad_slot_id: int = -1) -> torch.Tensor:
    """Move the m live slots of ``slots`` into slots 0 .. m-1 and return where each row's slot is
    now (int32, ``slots``' shape; padded rows stay padded).  Slots below m stay, the others take the
    free slots below m in row order: the fewest copies."""
    bufs, S, where, status = _target(buffers)
    s = _list(slots, "slots")
    n = s.numel()
    dev = _lib.device_index(status, s)
    ws = _workspace(n, where)
    new = torch.empty_like(s)
    _lib.call(_lib.load().nssm_slot_compact, dev, bufs, len(bufs), S, s.data_ptr(), n, int(pad_slot_id), new.data_ptr(),
              ws.data_ptr(), ws.numel(), status.data_ptr())
    return new


def reorder_slots(buffers, slots: torch.Tensor, parents: torch.Tensor, pad_slot_id: int = -1) -> torch.Tensor:
    """Let row r continue row ``parents[r]``: returns the rows' new slots (int32, ``slots``' shape).

    ``slots`` and ``parents`` ``[b, K]``: parents are beams of the same prompt
    (:func:`~nested_ssm_b200.beam.beam_select`); 1-D: parents are rows of the whole batch.  The first
    child of a row keeps its slot, every other child takes the slot of a row without children and
    gets a copy of the state there: the fewest copies.  A row whose parent is padded becomes padded.  A slot that
    two rows name is reported and never given to another row; a child for which no slot is left is reported and
    becomes padded."""
    shape = slots.shape
    if parents.shape != shape:
        raise ValueError(f"parents {tuple(parents.shape)} must have slots' shape {tuple(shape)}")
    bufs, S, where, status = _target(buffers)
    s, p = _list(slots, "slots"), _list(parents, "parents")
    n = s.numel()
    dev = _lib.device_index(status, s, p)
    ws = _workspace(n, where)
    new = torch.empty_like(s)
    _lib.call(_lib.load().nssm_slot_reorder, dev, bufs, len(bufs), S, s.data_ptr(), p.data_ptr(), n,
              max(shape[-1] if len(shape) > 1 else n, 1), int(pad_slot_id), new.data_ptr(), ws.data_ptr(), ws.numel(),
              status.data_ptr())
    return new
