"""The gated delta rule: a recurrent state rule beside the Mamba2 update, on states of the same
layout ``[slot, H, P, N]`` (fp32).  Per value head, with the log decay ``g`` and the write strength
``beta``:

    S <- exp(g) S;   u = beta (v - S k);   S <- S + u k^T;   y = scale S q

* :func:`gated_delta_state_update` -- one decode token per row with continuous-batching
  ``state_batch_indices``, beside :func:`~nested_ssm_b200.ops.selective_state_update`.
* :func:`gated_delta_chunk_scan` -- prompts (padded or packed), beside
  :func:`~nested_ssm_b200.ops.mamba_chunk_scan_combined`.

Inference only: tensors that require a gradient are refused.  All tensors must live on the same
CUDA device; work is enqueued on that device's current stream and never synchronised.
"""
from __future__ import annotations

import torch

from . import _lib
from .pool import nssm_dtype

_IO = (torch.bfloat16, torch.float32)
_pack_step = _lib.packer(_lib.NssmDeltaStepArgs)
_pack_scan = _lib.packer(_lib.NssmDeltaScanArgs)


def _no_grad(*ts):
    if torch.is_grad_enabled():
        for t in ts:
            if t is not None and t.requires_grad:
                raise RuntimeError("no backward pass: call under torch.no_grad() or detach the inputs")


def _check_status(status):
    if status.dtype != torch.int32 or status.numel() < 1:
        raise ValueError("status must be an int32 tensor")


def _indices(idx, n, name):
    if idx.dim() != 1:
        idx = idx.reshape(-1)
    if idx.shape[0] != n:
        raise ValueError(f"{name} has {idx.shape[0]} entries, expected {n}")
    return _lib.int32_list(idx, name)


def gated_delta_state_update(state: torch.Tensor, q, k, v, g, beta, scale: float | None = None,
                             state_batch_indices=None, pad_slot_id: int = -1, out=None, status=None):
    """One decode token of the gated delta rule on ``state [S, H, P, N]`` (fp32, updated in
    place; heads packed, slots at any stride that is a multiple of 4); returns ``out [b, H, P]``.

    ``q``, ``k`` ``[b, G, N]`` and ``v`` ``[b, H, P]`` bf16 or fp32 (head h uses group
    ``h // (H // G)``); ``g`` (log decay), ``beta`` ``[b, H]`` bf16 or fp32; ``scale`` defaults to
    ``N ** -0.5``.  Compiled for N 64 and 128, P a multiple of 16 up to 256.  Row b works on slot
    ``state_batch_indices[b]`` (row b without them); rows whose slot is ``pad_slot_id`` are skipped
    and their ``out`` rows untouched, as are rows whose slot is out of range (bit 0 of the int32
    ``status``) or was named by an earlier row (bit 3)."""
    if state.dim() != 4 or state.dtype != torch.float32:
        raise ValueError(f"state must be an fp32 [S, H, P, N] tensor, got {tuple(state.shape)} {state.dtype}")
    S, H, P, N = state.shape
    ss = state.stride()
    if ss[1:] != (P * N, N, 1) and not state[:1].flatten(0, 1).is_contiguous():   # (axes of one have any stride)
        raise ValueError("the heads of a slot must be contiguous in state")
    s0 = ss[0] if S > 1 else H * P * N
    qs = q.shape
    if len(qs) != 3 or k.shape != qs or qs[2] != N:
        raise ValueError(f"q and k must be [b, G, {N}], got {tuple(q.shape)} and {tuple(k.shape)}")
    b, G, _ = qs
    if v.shape != (b, H, P) or g.shape != (b, H) or beta.shape != (b, H):
        raise ValueError(f"v must be [{b}, {H}, {P}], g and beta [{b}, {H}], got {tuple(v.shape)}, {tuple(g.shape)}, "
                         f"{tuple(beta.shape)}")
    dt = q.dtype
    if dt not in _IO or k.dtype != dt or v.dtype != dt:
        raise ValueError("q, k and v must share a bf16 / fp32 dtype")
    _no_grad(state, q, k, v, g, beta)
    q0, q1, q2 = q.stride()
    k0, k1, k2 = k.stride()
    v0, v1, v2 = v.stride()
    if q2 != 1 or k2 != 1 or v2 != 1:
        q, k, v = q.contiguous(), k.contiguous(), v.contiguous()
        (q0, q1, _), (k0, k1, _), (v0, v1, _) = q.stride(), k.stride(), v.stride()
    idx = None if state_batch_indices is None else _indices(state_batch_indices, b, "state_batch_indices")
    if status is not None:
        _check_status(status)
    if out is None:
        out = torch.empty(b, H, P, dtype=dt, device=state.device)
    elif out.shape != (b, H, P) or out.stride(2) != 1 or out.dtype not in _IO:
        raise ValueError(f"out must be [{b}, {H}, {P}] bf16 / fp32 with unit inner stride")
    dev = _lib.device_index(state, q, k, v, g, beta, idx, out, status)
    o0, o1, _ = out.stride()
    g0, g1 = g.stride()
    b0, b1 = beta.stride()
    a = _pack_step(
        b, S, H, G, P, N, nssm_dtype(dt), nssm_dtype(g.dtype), nssm_dtype(beta.dtype), nssm_dtype(out.dtype),
        int(pad_slot_id), N ** -0.5 if scale is None else float(scale), state.data_ptr(), s0, q.data_ptr(), q0, q1,
        k.data_ptr(), k0, k1, v.data_ptr(), v0, v1, g.data_ptr(), g0, g1, beta.data_ptr(), b0, b1,
        0 if idx is None else idx.data_ptr(), out.data_ptr(), o0, o1, 0 if status is None else status.data_ptr())
    _lib.call(_lib.load().nssm_delta_step, dev, a)
    return out


def _rows(t: torch.Tensor):
    """(t, stride_b, stride_t) of ``[b, T, heads, dim]`` with packed (heads, dim), 16-byte aligned
    tokens and no broadcast axis: what the kernel loads; copied when it is not so."""
    d = t.shape[3]
    s0, s1, s2, s3 = t.stride()
    if s3 != 1 or s2 != d or s1 % 8 or s0 % 8 or t.data_ptr() % 16:
        t = t.contiguous()
        if t.data_ptr() % 16:     # a contiguous view that begins inside a 16-byte piece
            t = t.clone()
        s0, s1, _, _ = t.stride()
    return t, s0, s1


def gated_delta_chunk_scan(q, k, v, g, beta, scale: float | None = None, initial_states=None, cu_seqlens=None,
                           return_final_states: bool = False, *, out=None, final_states=None, status=None):
    """The gated delta rule over prompts: ``q``, ``k`` ``[b, T, G, N]`` and ``v`` ``[b, T, H, P]``
    bf16, ``g`` (log decay) and ``beta`` ``[b, T, H]`` bf16 or fp32; returns ``y [b, T, H, P]``
    (bf16) and with ``return_final_states`` also the fp32 states ``[n, H, P, N]`` after the last
    token of each sequence.  ``scale`` defaults to ``N ** -0.5``; N 64 or 128, P a multiple of 16 up
    to 256.

    ``cu_seqlens`` (int32 ``[n + 1]`` on the device, b == 1): sequence s has the tokens
    ``cu_seqlens[s]`` to ``cu_seqlens[s + 1]``; empty sequences keep their initial state, and
    the rows of ``out`` outside every sequence are left as they were.  Sequences whose bounds
    do not ascend inside ``[0, T]`` are skipped and set bit 3 of the int32 ``status``; they touch no
    other.  Sequences must not overlap.  Otherwise n == b.  ``initial_states [n, H, P, N]`` fp32
    (zeros without them); ``final_states`` may be the same tensor.  ``g`` may be ``-inf`` (the state
    is forgotten) and above 0 (it grows); any other value of a sequence that is not finite reaches
    every output of its 32-token block, those before it too, and the state.  What a head writes in a
    block, beta (v - S k), is held relative to the block's largest: with fewer than 22 bits below
    2^-17 of it, as nothing below 2^-40."""
    qs, vs = q.shape, v.shape
    if len(qs) != 4 or k.shape != qs or len(vs) != 4:
        raise ValueError("q / k [b, T, G, N], v [b, T, H, P], g / beta [b, T, H] expected")
    b, T, G, N = qs
    _, _, H, P = vs
    if vs[:2] != (b, T) or g.shape != (b, T, H) or beta.shape != (b, T, H):
        raise ValueError(f"shape mismatch: q {tuple(qs)} v {tuple(vs)} g {tuple(g.shape)} beta {tuple(beta.shape)}")
    if q.dtype != torch.bfloat16 or k.dtype != torch.bfloat16 or v.dtype != torch.bfloat16:
        raise ValueError("q, k and v must be bf16")
    _no_grad(q, k, v, g, beta, initial_states)
    n, cu = b, 0
    if cu_seqlens is not None:
        if b != 1 or cu_seqlens.dim() != 1 or cu_seqlens.shape[0] < 1:
            raise ValueError("cu_seqlens [n + 1] needs packed inputs with b == 1")
        n = cu_seqlens.shape[0] - 1
        cu_seqlens = _indices(cu_seqlens, n + 1, "cu_seqlens")
        cu = cu_seqlens.data_ptr()
    (q, q0, q1), (k, k0, k1), (v, v0, v1) = _rows(q), _rows(k), _rows(v)
    g0, g1, g2 = g.stride()
    b0, b1, b2 = beta.stride()
    if g2 != 1 or b2 != 1:
        g, beta = g.contiguous(), beta.contiguous()
        (g0, g1, _), (b0, b1, _) = g.stride(), beta.stride()
    def packed(t):     # the heads of a sequence are contiguous (axes of one have any stride)
        return t.stride()[1:] == (P * N, N, 1) or t[:1].flatten(0, 1).is_contiguous()

    init = init0 = fin = fin0 = 0
    if initial_states is not None:
        if initial_states.shape != (n, H, P, N):
            raise ValueError(f"initial_states must be [{n}, {H}, {P}, {N}], got {tuple(initial_states.shape)}")
        if (initial_states.dtype != torch.float32 or not packed(initial_states) or initial_states.stride(0) % 4
                or initial_states.data_ptr() % 16):
            initial_states = initial_states.float().contiguous()
        init, init0 = initial_states.data_ptr(), initial_states.stride(0)
    where = q.device
    if out is None:
        out = torch.empty(b, T, H, P, dtype=torch.bfloat16, device=where)
    elif out.shape != (b, T, H, P) or out.dtype != torch.bfloat16 or (
            out.stride()[2:] != (P, 1) and not out[:1, :1].flatten(0, 2).is_contiguous()):
        raise ValueError("out must be bf16 [b, T, H, P] with packed (H, P)")
    if final_states is not None:
        if final_states.shape != (n, H, P, N) or final_states.dtype != torch.float32 or not packed(final_states):
            raise ValueError(f"final_states must be fp32 [{n}, {H}, {P}, {N}] with contiguous rows")
    elif return_final_states:
        final_states = torch.empty(n, H, P, N, dtype=torch.float32, device=where)
    if final_states is not None:
        fin, fin0 = final_states.data_ptr(), final_states.stride(0)
    if status is not None:
        _check_status(status)
    dev = _lib.device_index(q, k, v, g, beta, cu_seqlens, initial_states, out, final_states, status)
    lib = _lib.load()
    nbytes = lib.nssm_delta_scan_workspace_bytes(n, T, H, G, N, 1 if cu else 0)
    ws = torch.empty(nbytes, dtype=torch.uint8, device=where) if nbytes else None
    o0, o1, _, _ = out.stride()
    a = _pack_scan(
        n, T, H, G, P, N, nssm_dtype(g.dtype), nssm_dtype(beta.dtype), N ** -0.5 if scale is None else float(scale), 0,
        q.data_ptr(), q0, q1, k.data_ptr(), k0, k1, v.data_ptr(), v0, v1, g.data_ptr(), g0, g1, beta.data_ptr(), b0, b1,
        cu, init, init0, out.data_ptr(), o0, o1, fin, fin0, 0 if ws is None else ws.data_ptr(), nbytes,
        0 if status is None else status.data_ptr())
    _lib.call(lib.nssm_delta_scan, dev, a)
    return (out, final_states) if return_final_states else out
