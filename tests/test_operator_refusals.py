"""Argument checks of the gated delta rule, slot moves and beam selection: refused on the host, before
any device work, in Python and at the C entries."""
import ctypes as C

import pytest
import torch

from nested_ssm_b200 import _lib, beam_select, gated_delta_chunk_scan, gated_delta_state_update
from nested_ssm_b200 import StateBuffers, copy_slots


def _step(**kw):
    d = dict(state=torch.zeros(3, 4, 32, 64), q=torch.zeros(2, 2, 64), k=torch.zeros(2, 2, 64), v=torch.zeros(2, 4, 32),
             g=torch.zeros(2, 4), beta=torch.zeros(2, 4))
    d.update(kw)
    return gated_delta_state_update(**d)


@pytest.mark.parametrize("kw,err", [
    (dict(state=torch.zeros(3, 4, 32, 64).bfloat16()), ValueError),
    (dict(state=torch.zeros(3, 4, 64, 32).transpose(2, 3)), ValueError),
    (dict(q=torch.zeros(2, 2, 32)), ValueError),
    (dict(k=torch.zeros(2, 1, 64)), ValueError),
    (dict(v=torch.zeros(2, 3, 32)), ValueError),
    (dict(g=torch.zeros(2, 4, 1)), ValueError),
    (dict(v=torch.zeros(2, 4, 32).bfloat16()), ValueError),
    (dict(q=torch.zeros(2, 2, 64).half(), k=torch.zeros(2, 2, 64).half(), v=torch.zeros(2, 4, 32).half()), ValueError),
    (dict(out=torch.zeros(2, 4, 31)), ValueError),
    (dict(state_batch_indices=torch.zeros(3, dtype=torch.int32)), ValueError),
    (dict(status=torch.zeros(1)), ValueError),
    (dict(v=torch.zeros(2, 4, 32, requires_grad=True)), RuntimeError),
    (dict(), RuntimeError),                                     # CPU tensors
])
def test_step(kw, err):
    with pytest.raises(err):
        _step(**kw)


def _scan(**kw):
    z = lambda *s: torch.zeros(*s, dtype=torch.bfloat16)  # noqa: E731
    d = dict(q=z(1, 5, 2, 64), k=z(1, 5, 2, 64), v=z(1, 5, 4, 32), g=torch.zeros(1, 5, 4), beta=torch.zeros(1, 5, 4))
    d.update(kw)
    return gated_delta_chunk_scan(**d)


@pytest.mark.parametrize("kw,err", [
    (dict(q=torch.zeros(1, 5, 2, 64)), ValueError),
    (dict(k=torch.zeros(1, 5, 1, 64).bfloat16()), ValueError),
    (dict(v=torch.zeros(1, 4, 4, 32).bfloat16()), ValueError),
    (dict(beta=torch.zeros(1, 5, 2)), ValueError),
    (dict(initial_states=torch.zeros(2, 4, 32, 64)), ValueError),
    (dict(out=torch.zeros(1, 5, 4, 32)), ValueError),
    (dict(final_states=torch.zeros(1, 4, 32, 64).bfloat16()), ValueError),
    (dict(cu_seqlens=torch.zeros(2, 2, dtype=torch.int32)), ValueError),
    (dict(g=torch.zeros(1, 5, 4, requires_grad=True)), RuntimeError),
    (dict(), RuntimeError),
])
def test_scan(kw, err):
    with pytest.raises(err):
        _scan(**kw)


def test_scan_packed_needs_one_row():
    z = lambda *s: torch.zeros(*s, dtype=torch.bfloat16)  # noqa: E731
    with pytest.raises(ValueError, match="b == 1"):
        gated_delta_chunk_scan(z(2, 5, 2, 64), z(2, 5, 2, 64), z(2, 5, 4, 32), torch.zeros(2, 5, 4), torch.zeros(2, 5, 4),
                               cu_seqlens=torch.zeros(3, dtype=torch.int32))


@pytest.mark.parametrize("kw,err", [
    (dict(logits=torch.zeros(2, 3)), ValueError),
    (dict(scores=torch.zeros(2, 4)), ValueError),
    (dict(scores=torch.zeros(2, 3).double()), ValueError),
    (dict(logits=torch.zeros(2, 3, 10).half()), ValueError),
    (dict(num_out=0), ValueError),
    (dict(num_out=31), ValueError),
    (dict(logits=torch.zeros(2, 3, 100), num_out=129), ValueError),
    (dict(finished=torch.zeros(2, 3, dtype=torch.bool)), ValueError),           # without eos_token_id
    (dict(finished=torch.zeros(2, 3), eos_token_id=1), ValueError),
    (dict(eos_token_id=10), ValueError),
    (dict(logits=torch.zeros(2, 3, 10, requires_grad=True)), RuntimeError),
    (dict(), RuntimeError),
])
def test_beam(kw, err):
    d = dict(logits=torch.zeros(2, 3, 10), scores=torch.zeros(2, 3))
    d.update(kw)
    with pytest.raises(err):
        beam_select(**d)


@pytest.mark.parametrize("tensors,dim,err", [
    ([], 0, ValueError),
    ([torch.zeros(4, 3)] * 25, 0, ValueError),
    ([torch.zeros(4, 3), torch.zeros(5, 3)], 0, ValueError),
    ([torch.zeros(4, 3)], 2, ValueError),
    ([torch.zeros(4)], 1, ValueError),
    ([torch.zeros(4, 6)[:, ::2]], 0, ValueError),                # gaps inside a slot
    ([torch.zeros(1, 3).expand(4, 3)], 0, ValueError),           # slots that share memory
    ([torch.zeros(1 << 18, 1)], 0, ValueError),
    ([torch.zeros(4, 3)], 0, RuntimeError),                      # CPU tensors
])
def test_state_buffers(tensors, dim, err):
    with pytest.raises(err):
        StateBuffers(tensors, slot_dim=dim)


def test_moves_refuse_other_targets():
    with pytest.raises(TypeError):
        copy_slots(torch.zeros(4, 3), torch.zeros(1, dtype=torch.int32), torch.zeros(1, dtype=torch.int32))


# ---------------------------------------------------------------- C entries (pointers are never read)
def _err(rc, code=_lib.NSSM_ERR_INVALID):
    assert rc == code, _lib.load().nssm_last_error()


def test_null_arguments():
    lib = _lib.load()
    _err(lib.nssm_delta_step(None, None))
    _err(lib.nssm_delta_scan(None, None))
    _err(lib.nssm_beam_select(None, None))
    _err(lib.nssm_slot_copy(None, 1, 4, 16, 16, 1, -1, 16, 64, None, None))
    _err(lib.nssm_slot_reorder(None, 1, 4, None, 16, 1, 1, -1, 16, 16, 64, None, None))
    _err(lib.nssm_slot_compact(None, 1, 4, 16, 1, -1, None, 16, 64, None, None))


def _fill(a, **kw):
    for n, t in a._fields_:
        if t is C.c_void_p:
            setattr(a, n, 1 << 20)
    for n, v in kw.items():
        setattr(a, n, v)
    return a


DELTA = dict(batch=2, nheads=4, ngroups=2, headdim=32, dstate=64, scale=1.0)


@pytest.mark.parametrize("kw,code", [
    (dict(dstate=96), _lib.NSSM_ERR_UNSUPPORTED), (dict(headdim=24), _lib.NSSM_ERR_UNSUPPORTED),
    (dict(headdim=272), _lib.NSSM_ERR_UNSUPPORTED), (dict(ngroups=3), 1), (dict(nheads=0), 1), (dict(batch=-1), 1),
    (dict(batch=9), 1), (dict(io_dtype=2), 1), (dict(state_stride_s=8190), 1), (dict(state_stride_s=4096), 1),
    (dict(state=(1 << 20) + 4), 1), (dict(q=None), 1),
])
def test_delta_step_entry(kw, code):
    a = _fill(_lib.NssmDeltaStepArgs(), **{**DELTA, "num_slots": 8, "state_stride_s": 8192, "state_batch_indices": None, **kw})
    _err(_lib.load().nssm_delta_step(C.byref(a), None), code)


@pytest.mark.parametrize("kw,code", [
    (dict(dstate=256), _lib.NSSM_ERR_UNSUPPORTED), (dict(headdim=0), _lib.NSSM_ERR_UNSUPPORTED), (dict(seqlen=-1), 1),
    (dict(q_stride_t=132), 1), (dict(v=(1 << 20) + 2), 1), (dict(k=None), 1), (dict(final_stride_b=4), 1),
    (dict(g_dtype=2), 1), (dict(initial_states=(1 << 20) + 8), 1),
])
def test_delta_scan_entry(kw, code):
    a = _fill(_lib.NssmDeltaScanArgs(), **{**DELTA, "seqlen": 10, "q_stride_b": 1280, "q_stride_t": 128, "k_stride_b": 1280,
                                           "k_stride_t": 128, "v_stride_b": 1280, "v_stride_t": 128, "y_stride_b": 1280,
                                           "y_stride_t": 128, "final_stride_b": 8192, "init_stride_b": 8192,
                                           "workspace_bytes": 1 << 30, **kw})
    _err(_lib.load().nssm_delta_scan(C.byref(a), None), code)


@pytest.mark.parametrize("kw", [
    dict(beams=65), dict(beams=0), dict(vocab=0), dict(vocab=(1 << 26) + 1), dict(nout=129), dict(nout=0), dict(logits_dtype=2),
    dict(eos_token=1000), dict(eos_token=-1), dict(batch=30000, beams=4), dict(workspace_bytes=64), dict(scores=None),
])
def test_beam_entry(kw):
    a = _fill(_lib.NssmBeamArgs(), **{"batch": 2, "beams": 4, "vocab": 1000, "nout": 4, "eos_token": 1,
                                      "workspace_bytes": 1 << 30, **kw})
    _err(_lib.load().nssm_beam_select(C.byref(a), None))


def _buf(**kw):
    b = (_lib.NssmSlotBuffer * 1)()
    for n, v in {"base": 1 << 20, "outer": 2, "outer_stride": 4096, "slot_stride": 64, "row_bytes": 64, **kw}.items():
        setattr(b[0], n, v)
    return b


@pytest.mark.parametrize("buf,args", [
    (dict(base=None), {}), (dict(row_bytes=0), {}), (dict(slot_stride=32), {}), (dict(outer_stride=32), {}), (dict(outer=0), {}),
    (dict(row_bytes=1 << 50, slot_stride=1 << 50, outer_stride=1 << 60), {}), ({}, dict(nbuf=0)), ({}, dict(nbuf=25)),
    ({}, dict(S=0)), ({}, dict(S=131073)), ({}, dict(rows=4097)), ({}, dict(rows=-1)), ({}, dict(ws=16)), ({}, dict(group=3)),
])
def test_slot_entries(buf, args):
    lib = _lib.load()
    d = {"nbuf": 1, "S": 64, "rows": 8, "ws": 72, "group": 4, **args}
    b, p = _buf(**buf), 1 << 21
    _err(lib.nssm_slot_reorder(b, d["nbuf"], d["S"], p, p, d["rows"], d["group"], -1, p + 4096, p, d["ws"], None, None))
    if not args.get("group"):
        _err(lib.nssm_slot_copy(b, d["nbuf"], d["S"], p, p, d["rows"], -1, p, d["ws"], None, None))
        _err(lib.nssm_slot_compact(b, d["nbuf"], d["S"], p, d["rows"], -1, p, p, d["ws"], None, None))
    assert lib.nssm_slot_workspace_bytes(8) == 72 and lib.nssm_slot_workspace_bytes(0) == 0


def test_delta_scan_refuses_too_many_blocks():
    a = _fill(_lib.NssmDeltaScanArgs(), **{**DELTA, "batch": 65535, "seqlen": 1 << 20, "q_stride_t": 128, "k_stride_t": 128,
                                           "v_stride_t": 128, "y_stride_t": 128, "q_stride_b": 128, "k_stride_b": 128,
                                           "v_stride_b": 128, "y_stride_b": 128, "final_stride_b": 8192, "init_stride_b": 8192,
                                           "workspace_bytes": 1 << 62, "cu_seqlens": None})
    _err(_lib.load().nssm_delta_scan(C.byref(a), None))
    assert "too large" in _lib.load().nssm_last_error().decode()


def test_indices_that_int32_cannot_hold_stay_out_of_range():
    t = torch.tensor([3, -1, 1 << 32, (1 << 32) + 3, -(1 << 40), (1 << 31) - 1])
    assert _lib.int32_list(t, "t").tolist() == [3, -1, (1 << 31) - 1, (1 << 31) - 1, -(1 << 31), (1 << 31) - 1]
    same = torch.tensor([5, 6], dtype=torch.int32)
    assert _lib.int32_list(same, "t") is same
    assert _lib.int32_list(torch.tensor([200, 7], dtype=torch.uint8), "t").tolist() == [200, 7]
    for bad in (torch.zeros(2), torch.zeros(2, dtype=torch.bool)):
        with pytest.raises(ValueError, match="integers"):
            _lib.int32_list(bad, "t")


@pytest.mark.parametrize("idx", [torch.zeros(2), torch.zeros(2, dtype=torch.bool)])
def test_slots_and_bounds_are_integers(idx):
    with pytest.raises(ValueError, match="integers"):
        _step(state_batch_indices=idx)
    with pytest.raises(ValueError, match="integers"):
        _scan(cu_seqlens=idx)


def _strided(shape, strides):
    return torch.as_strided(torch.zeros(4096), shape, strides)


@pytest.mark.parametrize("t,fine", [
    (torch.zeros(3, 4, 5), True),
    (torch.zeros(4, 3, 5).transpose(0, 1), True),                 # layers inside a slot's row
    (torch.zeros(6, 8, 5)[::2, ::2], True),
    (torch.zeros(1, 4, 5).expand(3, 4, 5), False),                # one layer under three names
    (torch.zeros(1, 4, 5), True),
    (torch.zeros(3, 1, 5), True),
    (_strided((3, 4, 5), (5, 5, 1)), False),                      # layer 1 begins at slot 1 of layer 0
    (_strided((3, 1, 5), (4, 5, 1)), False),
    (_strided((2, 4, 5), (17, 10, 1)), False),                    # 17 is 3 before slot 2
    (_strided((2, 4, 5), (15, 10, 1)), True),                     # between the slots
    (_strided((2, 4, 5), (35, 10, 1)), True),                     # behind them
    (_strided((2, 4, 5), (34, 10, 1)), False),
])
def test_state_buffers_of_layers_that_share_memory(t, fine):
    with pytest.raises(RuntimeError if fine else ValueError, match="CUDA" if fine else "overlap"):
        StateBuffers([t], slot_dim=1)


def test_layers_overlap_equals_a_count_of_addresses():
    from nested_ssm_b200.slots import _layers_overlap
    for row in (1, 3):
        for s in range(row, 9):
            for o in range(0, 30):
                for S in (1, 2, 4):
                    for L in (1, 2, 3):
                        at = [i * o + j * s + e for i in range(L) for j in range(S) for e in range(row)]
                        assert _layers_overlap(row, s, S, o, L) == (len(set(at)) < len(at)), (row, s, o, S, L)


@pytest.mark.parametrize("kw", [dict(out_stride_b=0, out_stride_h=32), dict(out_stride_b=128, out_stride_h=0),
                                dict(out_stride_b=16, out_stride_h=128)])
def test_delta_step_refuses_rows_of_out_that_share_memory(kw):
    a = _fill(_lib.NssmDeltaStepArgs(), **{**DELTA, "num_slots": 8, "state_stride_s": 8192, **kw})
    _err(_lib.load().nssm_delta_step(C.byref(a), None))
    assert b"share memory" in _lib.load().nssm_last_error()


@pytest.mark.parametrize("kw", [dict(y_stride_t=0), dict(y_stride_t=64), dict(y_stride_b=0)])
def test_delta_scan_refuses_tokens_of_y_that_share_memory(kw):
    a = _fill(_lib.NssmDeltaScanArgs(), **{**DELTA, "seqlen": 10, "q_stride_b": 1280, "q_stride_t": 128, "k_stride_b": 1280,
                                           "k_stride_t": 128, "v_stride_b": 1280, "v_stride_t": 128, "y_stride_b": 1280,
                                           "y_stride_t": 128, "final_stride_b": 8192, "init_stride_b": 8192,
                                           "cu_seqlens": None, "workspace_bytes": 1 << 30, **kw})
    _err(_lib.load().nssm_delta_scan(C.byref(a), None))
    assert b"share memory" in _lib.load().nssm_last_error()
