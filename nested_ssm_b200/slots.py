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

import ctypes as C

import torch

from . import _lib
from .ops import _ptr, _require_cuda, _stream
from .pool import TieredSlotPool


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
        self.device = _require_cuda(*tensors)
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
    if t.is_floating_point() or t.dtype == torch.bool:
        raise ValueError(f"{name} must hold integers, got {t.dtype}")
    f = t.reshape(-1)
    if n is not None and f.numel() != n:
        raise ValueError(f"{name} has {f.numel()} entries, expected {n}")
    if f.numel() > _lib.MAX_SLOT_ROWS:
        raise ValueError(f"{name} has {f.numel()} rows; at most {_lib.MAX_SLOT_ROWS} in one call")
    if f.dtype != torch.int32 or not f.is_contiguous():
        f = f.to(torch.int32).contiguous()
    return f


def _workspace(n, dev):
    return torch.empty(8 + 8 * max(n, 1), dtype=torch.uint8, device=dev)


def copy_slots(buffers, src: torch.Tensor, dst: torch.Tensor, pad_slot_id: int = -1) -> None:
    """Slot ``dst[i]`` becomes a copy of slot ``src[i]``; naming a source several times forks it.
    Pairs with ``pad_slot_id`` are skipped, a pair with ``src == dst`` does nothing."""
    bufs, S, dev, status = _target(buffers)
    s = _list(src, "src")
    d = _list(dst, "dst", s.numel())
    _require_cuda(s, d, status)
    ws = _workspace(s.numel(), dev)
    lib = _lib.load()
    with torch.cuda.device(dev):
        _lib.check(lib.nssm_slot_copy(bufs, len(bufs), S, s.data_ptr(), d.data_ptr(), s.numel(), int(pad_slot_id),
                                      ws.data_ptr(), ws.numel(), status.data_ptr(), _stream(dev)))


def clear_slots(buffers, slots: torch.Tensor, pad_slot_id: int = -1) -> None:
    """Free slots: every value of the named slots becomes zero, an empty state for the next
    sequence."""
    bufs, S, dev, status = _target(buffers)
    d = _list(slots, "slots")
    _require_cuda(d, status)
    ws = _workspace(d.numel(), dev)
    lib = _lib.load()
    with torch.cuda.device(dev):
        _lib.check(lib.nssm_slot_copy(bufs, len(bufs), S, None, d.data_ptr(), d.numel(), int(pad_slot_id),
                                      ws.data_ptr(), ws.numel(), status.data_ptr(), _stream(dev)))


def compact_slots(buffers, slots: torch.Tensor, pad_slot_id: int = -1) -> torch.Tensor:
    """Move the m live slots of ``slots`` into slots 0 .. m-1 and return where each row's slot is
    now (int32, ``slots``' shape; padded rows stay padded).  Slots below m stay, the others take the
    free slots below m in row order: the fewest copies."""
    bufs, S, dev, status = _target(buffers)
    s = _list(slots, "slots")
    _require_cuda(s, status)
    ws = _workspace(s.numel(), dev)
    new = torch.empty_like(s)
    lib = _lib.load()
    with torch.cuda.device(dev):
        _lib.check(lib.nssm_slot_compact(bufs, len(bufs), S, s.data_ptr(), s.numel(), int(pad_slot_id), new.data_ptr(),
                                         ws.data_ptr(), ws.numel(), status.data_ptr(), _stream(dev)))
    return new.view(slots.shape)


def reorder_slots(buffers, slots: torch.Tensor, parents: torch.Tensor, pad_slot_id: int = -1) -> torch.Tensor:
    """Let row r continue row ``parents[r]``: returns the rows' new slots (int32, ``slots``' shape).

    ``slots`` and ``parents`` ``[b, K]``: parents are beams of the same prompt
    (:func:`~nested_ssm_b200.beam.beam_select`); 1-D: parents are rows of the whole batch.  The first
    child of a row keeps its slot, every other child takes the slot of a row without children and
    gets a copy of the state there: the fewest copies.  A row whose parent is padded becomes padded."""
    if parents.shape != slots.shape:
        raise ValueError(f"parents {tuple(parents.shape)} must have slots' shape {tuple(slots.shape)}")
    bufs, S, dev, status = _target(buffers)
    s, p = _list(slots, "slots"), _list(parents, "parents")
    _require_cuda(s, p, status)
    n = s.numel()
    group = slots.shape[-1] if slots.dim() > 1 else n
    ws = _workspace(n, dev)
    new = torch.empty_like(s)
    lib = _lib.load()
    with torch.cuda.device(dev):
        _lib.check(lib.nssm_slot_reorder(bufs, len(bufs), S, s.data_ptr(), p.data_ptr(), n, max(group, 1), int(pad_slot_id),
                                         new.data_ptr(), ws.data_ptr(), ws.numel(), status.data_ptr(), _stream(dev)))
    return new.view(slots.shape)
