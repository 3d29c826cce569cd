"""Beam search's selection over beams and vocabulary.  The chosen continuations' states follow with
:func:`~nested_ssm_b200.slots.reorder_slots`."""
from __future__ import annotations

import torch

from . import _lib
from .delta import _no_grad
from .pool import nssm_dtype

_pack = _lib.packer(_lib.NssmBeamArgs)


def beam_select(logits: torch.Tensor, scores: torch.Tensor, num_out: int | None = None, finished=None,
                eos_token_id: int | None = None):
    """The ``num_out`` (default: as many as beams) best continuations of each prompt:
    ``total = scores + log_softmax(logits)`` over all beams and tokens.

    ``logits [b, K, V]`` bf16 or fp32 (unit inner stride, rows at any stride and alignment),
    ``scores [b, K]`` fp32, K up to 64, ``num_out`` up to 128.  Returns ``(scores [b, n] fp32,
    parents [b, n] int32, tokens [b, n] int32)`` in descending order, and with ``eos_token_id`` also
    ``finished [b, n]`` bool: the continuation ends its sequence.  ``finished [b, K]`` bool marks
    beams that ended before: such a beam's one continuation is ``eos_token_id`` at its own score.

    A logit that is not finite counts as masked (-inf).  Candidates of one beam rank by logit, then by
    the lower token; those of different beams by total (in 64 bits), then by the lower beam.  Masked
    candidates are returned, with a score of -inf, only when there are no others.  Totals are formed as
    (score + logit) - lse: a beam whose every logit is a finite mask of 1e16 and more loses its score beside
    them, so a beam without tokens is masked with -inf."""
    if logits.dim() != 3 or scores.shape != logits.shape[:2]:
        raise ValueError(f"logits [b, K, V] and scores [b, K] expected, got {tuple(logits.shape)} and {tuple(scores.shape)}")
    b, K, V = logits.shape
    n = K if num_out is None else int(num_out)
    if logits.dtype not in (torch.bfloat16, torch.float32) or scores.dtype != torch.float32:
        raise ValueError("logits must be bf16 or fp32, scores fp32")
    if finished is not None and (eos_token_id is None or finished.shape != (b, K) or finished.dtype != torch.bool):
        raise ValueError("finished must be a bool [b, K] tensor, with eos_token_id")
    if eos_token_id is not None and not 0 <= eos_token_id < V:
        raise ValueError(f"eos_token_id {eos_token_id} outside [0, {V})")
    if not 1 <= n <= min(_lib.MAX_BEAM_OUT, K * V):
        raise ValueError(f"num_out {n} outside [1, min({_lib.MAX_BEAM_OUT}, K * V)]")
    _no_grad(logits, scores)
    if logits.stride(2) != 1:
        logits = logits.contiguous()
    if not scores.is_contiguous():
        scores = scores.contiguous()
    if finished is not None and not finished.is_contiguous():
        finished = finished.contiguous()
    dev = _lib.device_index(logits, scores, finished)
    lib = _lib.load()
    where = logits.device
    out_s = torch.empty(b, n, dtype=torch.float32, device=where)
    out_p = torch.empty(b, n, dtype=torch.int32, device=where)
    out_t = torch.empty(b, n, dtype=torch.int32, device=where)
    out_f = torch.empty(b, n, dtype=torch.bool, device=where) if eos_token_id is not None else None
    dt = nssm_dtype(logits.dtype)
    nbytes = lib.nssm_beam_workspace_bytes(b, K, V, n, dt)
    ws = torch.empty(nbytes, dtype=torch.uint8, device=where)
    l0, l1, _ = logits.stride()
    a = _pack(b, K, V, n, dt, -1 if eos_token_id is None else int(eos_token_id), logits.data_ptr(), l0, l1,
              scores.data_ptr(), 0 if finished is None else finished.data_ptr(), out_s.data_ptr(), out_p.data_ptr(),
              out_t.data_ptr(), 0 if out_f is None else out_f.data_ptr(), ws.data_ptr(), nbytes)
    _lib.call(lib.nssm_beam_select, dev, a)
    return (out_s, out_p, out_t) if out_f is None else (out_s, out_p, out_t, out_f)
