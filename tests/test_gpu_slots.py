"""Slot moves (nssm_slot_copy, nssm_slot_reorder, nssm_slot_compact) against list simulations: copies are
exact, every byte outside the written slots stays, and conflicting moves are dropped."""
import pytest
import torch

import oracle.delta as OD
from tests import _helpers as Hh

pytestmark = pytest.mark.gpu


def _tensors(S, L, seed=0, odd=False):
    """State-like buffers of several types; `odd`: rows whose bytes allow no wide access."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    t = [r(L, S, 4, 48, 64), r(L, S, 40, 3).bfloat16(), (100 * r(L, S, 5)).int()]
    if odd:
        t += [(100 * r(L, S, 7)).to(torch.uint8), r(L, S, 3).bfloat16(), r(L, 2 * S, 12)[:, ::2],
              r(L, S, 3, 16).bfloat16().transpose(2, 3)]
    return t


def _apply(tensors, moves, slot_dim=1):
    want = [t.clone() for t in tensors]
    for w, t in zip(want, tensors):
        for s, d in moves:
            w.select(slot_dim, d).copy_(0 if s is None else t.select(slot_dim, s))
    return want


def _same(tensors, want):
    for t, w in zip(tensors, want):
        assert torch.equal(t, w)


def _i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("odd", [False, True])
@pytest.mark.parametrize("pairs", [
    [(0, 5)],
    [(3, 1), (3, 2), (3, 7), (9, 0)],                 # a fork
    [(4, 4), (-1, 2), (6, -1), (8, 3)],               # onto itself, padded
    [],
])
def test_copy(pairs, odd):
    from nested_ssm_b200 import StateBuffers, copy_slots
    t = _tensors(10, 2, odd=odd)
    bufs = StateBuffers(t, slot_dim=1)
    want = _apply(t, [(s, d) for s, d in pairs if s >= 0 and d >= 0])
    copy_slots(bufs, _i32([s for s, _ in pairs]), _i32([d for _, d in pairs]))
    _same(t, want)
    bufs.check_status()


@pytest.mark.parametrize("pairs,kept,status", [
    ([(0, 1), (1, 0)], [], 8),                        # a swap: each would read what the other writes
    ([(0, 1), (1, 2), (4, 5)], [(1, 2), (4, 5)], 8),  # a chain: the move into a slot that is read is dropped
    ([(0, 3), (1, 3), (2, 4)], [(2, 4)], 8),          # two moves into one slot
    ([(10, 1), (2, 77), (3, 4), (-7, 5)], [(3, 4)], 1),
])
def test_copy_conflicts_are_dropped(pairs, kept, status):
    from nested_ssm_b200 import StateBuffers, copy_slots
    t = _tensors(10, 1)
    bufs = StateBuffers(t, slot_dim=1)
    want = _apply(t, kept)
    copy_slots(bufs, _i32([s for s, _ in pairs]), _i32([d for _, d in pairs]))
    _same(t, want)
    assert int(bufs.status) == status
    with pytest.raises(IndexError):
        bufs.check_status()
    bufs.check_status()       # once only


def test_copy_single_layer_large_rows_and_many_slots():
    """slot_dim 0; a row of several work items with a ragged end; as many slots as a call takes."""
    from nested_ssm_b200 import StateBuffers, copy_slots
    g = torch.Generator(device="cuda").manual_seed(2)
    t = [torch.randn(6, 50003, generator=g, device="cuda")]
    want = _apply(t, [(1, 4), (2, 0)], 0)
    copy_slots(StateBuffers(t), _i32([1, 2]), _i32([4, 0]))
    _same(t, want)
    S = 131072
    big = torch.arange(S * 4, dtype=torch.int32, device="cuda").view(S, 4)
    src = torch.arange(0, 4096, device="cuda")
    dst = torch.randperm(S - 4096, generator=g, device="cuda")[:4096] + 4096
    ref = big.clone()
    ref[dst] = big[src]
    bufs = StateBuffers([big])
    copy_slots(bufs, src, dst)
    assert torch.equal(big, ref)
    bufs.check_status()


def test_copy_offsets_beyond_32_bits():
    from nested_ssm_b200 import StateBuffers, copy_slots
    t = torch.zeros(3, 9, 1 << 27, dtype=torch.uint8, device="cuda")
    t[2, 8] = 7
    copy_slots(StateBuffers(t, slot_dim=1), _i32([8]), _i32([1]))
    assert int(t[2, 1].min()) == 7 and int(t[0, 1].max()) == 0 and int(t[2].long().sum()) == 2 * 7 * (1 << 27)


@pytest.mark.parametrize("slots,status", [([2, 5], 0), ([3, -1, 3, 0], 0), ([11, 1], 1), ([], 0)])
def test_clear(slots, status):
    from nested_ssm_b200 import StateBuffers, clear_slots
    t = _tensors(10, 2, odd=True)
    bufs = StateBuffers(t, slot_dim=1)
    want = _apply(t, [(None, s) for s in slots if 0 <= s < 10])
    clear_slots(bufs, _i32(slots))
    _same(t, want)
    assert int(bufs.status) == status


@pytest.mark.parametrize("S,n,pads,seed", [(10, 10, 0, 0), (10, 1, 0, 1), (64, 20, 3, 2), (300, 140, 40, 3), (5000, 4096, 7, 4),
                                           (9, 4, 4, 5)])
def test_compact(S, n, pads, seed):
    from nested_ssm_b200 import StateBuffers, compact_slots
    g = torch.Generator().manual_seed(seed)
    slots = torch.randperm(S, generator=g)[:n].tolist()
    for i in torch.randperm(n, generator=g)[:pads].tolist():
        slots[i] = -1
    t = [torch.randn(2, S, 33, device="cuda"), torch.randn(2, S, 8, device="cuda").bfloat16()]
    bufs = StateBuffers(t, slot_dim=1)
    new, moves = OD.compact_plan(slots, -1)
    want = _apply(t, moves)
    got = compact_slots(bufs, _i32(slots))
    assert got.tolist() == new
    _same(t, want)
    bufs.check_status()
    live = [s for s in new if s >= 0]
    assert sorted(live) == list(range(len(live)))


def test_compact_reports_bad_and_repeated_slots():
    from nested_ssm_b200 import StateBuffers, compact_slots
    t = [torch.randn(1, 12, 8, device="cuda")]
    bufs = StateBuffers(t, slot_dim=1)
    got = compact_slots(bufs, _i32([9, 40, 0]))
    assert got.tolist() == [1, -1, 0] and int(bufs.status) == 1
    bufs.status.zero_()
    compact_slots(bufs, _i32([9, 9, 0]))
    assert int(bufs.status) == 8


@pytest.mark.parametrize("b,K,S,seed,pads", [(1, 1, 3, 0, 0), (1, 4, 4, 1, 0), (5, 3, 40, 2, 1), (64, 8, 600, 3, 0),
                                             (128, 32, 4100, 4, 3), (7, 5, 35, 5, 0)])
def test_reorder(b, K, S, seed, pads):
    """Random parents of each prompt's beams; `pads` prompts are padded."""
    from nested_ssm_b200 import StateBuffers, reorder_slots
    g = torch.Generator().manual_seed(seed)
    slots = torch.randperm(S, generator=g)[:b * K].view(b, K)
    parents = torch.randint(0, K, (b, K), generator=g)
    slots[:pads] = -1
    t = [torch.randn(2, S, 33, device="cuda"), torch.randn(2, S, 8, device="cuda").bfloat16()]
    bufs = StateBuffers(t, slot_dim=1)
    new, moves = OD.reorder_plan(slots.reshape(-1).tolist(), parents.reshape(-1).tolist(), K, -1)
    want = _apply(t, moves)
    got = reorder_slots(bufs, slots.cuda(), parents.cuda())
    assert got.dtype == torch.int32 and got.shape == (b, K) and got.reshape(-1).tolist() == new
    _same(t, want)
    bufs.check_status()
    # every row's slot holds what its parent's slot held
    old = [w.clone() for w in want]
    for r in range(pads * K, b * K):
        p = slots.reshape(-1)[r // K * K + int(parents.reshape(-1)[r])]
        assert int(new[r]) >= 0 and (new[r] == int(p) or (int(p), new[r]) in moves)
    _same(t, old)


def test_reorder_flat_rows_padding_and_bad_parents():
    from nested_ssm_b200 import StateBuffers, reorder_slots
    t = [torch.arange(20 * 4, dtype=torch.float32, device="cuda").view(1, 20, 4)]
    bufs = StateBuffers(t, slot_dim=1)
    old = t[0].clone()
    # rows of the whole batch; row 1 is padded, row 0 continues it and becomes padded; its slot is free
    got = reorder_slots(bufs, _i32([4, -1, 6, 8]), _i32([1, 2, 2, 3]))
    assert got.tolist() == [-1, 6, 4, 8]
    assert torch.equal(t[0][0, 4], old[0, 6]) and torch.equal(t[0][0, 6], old[0, 6])
    bufs.check_status()
    # more children than slots: a padded row is to be continued
    got = reorder_slots(bufs, _i32([4, -1]), _i32([0, 0]))
    assert got.tolist() == [4, -1] and int(bufs.status) == 8
    bufs.status.zero_()
    got = reorder_slots(bufs, _i32([4, 5]), _i32([2, -1]))
    assert got.tolist() == [-1, -1] and int(bufs.status) == 1


@pytest.mark.parametrize("cold", ["fp8", "bf16"])
def test_pool_slots_follow_their_sequences(cold):
    """Beams on a tiered pool: forked from one prefilled slot, decoded, reordered, compacted; every
    beam's output equals that of a pool on which the rows' states were moved by indexing."""
    from nested_ssm_b200 import compact_slots, copy_slots, prefill_split, reorder_slots, clear_slots
    case = Hh.make_case(b=4, S=12, H=16, G=2, pb=32, c=4, cold=cold, steps=7, seed=3)
    a, ref = Hh.gpu_pool(case), Hh.gpu_pool(case)
    prm = {k: v.cuda() for k, v in case["prm"].items()}
    st = case["state0"][:1].cuda()
    prefill_split(a, 0, st, _i32([7]))
    copy_slots(a, _i32([7, 7, 7]), _i32([2, 11, 5]))
    slots = _i32([7, 2, 11, 5])
    prefill_split(ref, 0, st.expand(4, -1, -1, -1).contiguous(), _i32([0, 1, 2, 3]))
    rows = _i32([0, 1, 2, 3])
    names = [n for n in ("hot", "cold", "scale", "glog", "t", "ring_x", "ring_dt", "ring_b") if getattr(ref, n) is not None]
    parents = [[0, 1, 2, 3], [1, 1, 0, 3], [2, 2, 2, 2], [0, 1, 3, 3], [3, 0, 1, 2], [0, 0, 1, 1], [1, 0, 0, 0]]
    for step, par in enumerate(parents):
        ya = _decode(a, case, prm, step, slots)
        yr = _decode(ref, case, prm, step, rows)
        assert torch.equal(ya, yr), step
        slots = reorder_slots(a, slots, _i32(par))
        for n in names:     # the reference moves every row's state
            buf = getattr(ref, n)
            raw = buf.view(torch.uint8) if n == "cold" and cold == "fp8" else buf
            raw[:, :4] = raw[:, torch.tensor(par, device="cuda")].clone()
        if step == 3:
            slots = compact_slots(a, slots)
            assert sorted(slots.tolist()) == [0, 1, 2, 3]
            free = [s for s in range(12) if s not in slots.tolist()]
            clear_slots(a, _i32(free))
            assert float(a.hot[:, free].abs().max()) == 0 and int(a.t[:, free].max()) == 0
    a.check_status()


def _decode(pool, case, prm, step, slots):
    from nested_ssm_b200 import tiered_state_update
    out = torch.zeros(4, case["H"], case["P"], device="cuda")
    return tiered_state_update(pool, 0, case["xs"][step].cuda(), case["dts"][step].cuda(), prm["A"], case["Bs"][step].cuda(),
                               case["Cs"][step].cuda(), prm["D"], prm["dt_bias"], True, slots, -1, out, prm["R"], 1e-3)


def test_two_replayed_graphs_and_another_stream():
    """Captured moves read their lists at the replay; two graphs share nothing."""
    from nested_ssm_b200 import StateBuffers, compact_slots, reorder_slots
    t = [torch.randn(2, 40, 33, device="cuda")]
    bufs = StateBuffers(t, slot_dim=1)
    slots, parents, live = _i32([[1, 2, 3], [7, 8, 9]]), _i32([[0, 1, 2], [0, 1, 2]]), _i32([30, 1, 39])
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        reorder_slots(bufs, slots, parents)
    torch.cuda.current_stream().wait_stream(s)
    g1, g2 = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(g1):
        o1 = reorder_slots(bufs, slots, parents)
    with torch.cuda.graph(g2):
        o2 = compact_slots(bufs, live)
    parents.copy_(_i32([[1, 1, 1], [2, 0, 0]]))
    live.copy_(_i32([5, 36, 0]))
    before = t[0].clone()
    g1.replay()
    new, moves = OD.reorder_plan([1, 2, 3, 7, 8, 9], [1, 1, 1, 2, 0, 0], 3, -1)
    want = _apply([before], moves)
    _same(t, want)
    assert o1.reshape(-1).tolist() == new
    g2.replay()
    new, moves = OD.compact_plan([5, 36, 0], -1)
    _same(t, _apply(want, moves))
    assert o2.tolist() == new


def test_nothing_to_do():
    """Empty lists and batches in every call."""
    from nested_ssm_b200 import (StateBuffers, beam_select, clear_slots, compact_slots, copy_slots, gated_delta_chunk_scan,
                                 reorder_slots)
    t = [torch.randn(2, 5, 33, device="cuda")]
    bufs = StateBuffers(t, slot_dim=1)
    want = t[0].clone()
    none = _i32([])
    copy_slots(bufs, none, none)
    clear_slots(bufs, none)
    assert compact_slots(bufs, none).shape == (0,)
    assert reorder_slots(bufs, none.view(0, 4), none.view(0, 4)).shape == (0, 4)
    assert compact_slots(bufs, _i32([-1, -1])).tolist() == [-1, -1]
    assert reorder_slots(bufs, _i32([[-1, -1]]), _i32([[0, 1]])).tolist() == [[-1, -1]]
    assert torch.equal(t[0], want)
    bufs.check_status()
    s, p, k = beam_select(torch.zeros(0, 3, 7, device="cuda"), torch.zeros(0, 3, device="cuda"), 2)
    assert s.shape == p.shape == k.shape == (0, 2)
    z = lambda *sh: torch.zeros(*sh, device="cuda", dtype=torch.bfloat16)  # noqa: E731
    y, S = gated_delta_chunk_scan(z(0, 9, 2, 64), z(0, 9, 2, 64), z(0, 9, 4, 32), z(0, 9, 4), z(0, 9, 4), return_final_states=True)
    assert y.shape == (0, 9, 4, 32) and S.shape == (0, 4, 32, 64)
    y, S = gated_delta_chunk_scan(z(1, 0, 2, 64), z(1, 0, 2, 64), z(1, 0, 4, 32), z(1, 0, 4), z(1, 0, 4),
                                  cu_seqlens=_i32([0, 0, 0]), return_final_states=True)
    assert y.shape == (1, 0, 4, 32) and S.shape == (2, 4, 32, 64) and float(S.abs().max()) == 0


def test_two_calls_at_once_on_two_streams():
    """Calls on two streams share no workspace: moves of other slots, and prompts, side by side."""
    from nested_ssm_b200 import StateBuffers, copy_slots, gated_delta_chunk_scan, beam_select
    t = [torch.randn(3, 64, 4, 64, 64, device="cuda")]
    bufs = StateBuffers(t, slot_dim=1)
    want = t[0].clone()
    want[:, 16:32], want[:, 48:64] = want[:, 0:16].clone(), want[:, 32:48].clone()
    g = torch.Generator(device="cuda").manual_seed(0)
    r = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    x = [(r(2, 150, 2, 64) / 8).bfloat16(), (r(2, 150, 2, 64) / 8).bfloat16(), r(2, 150, 4, 48).bfloat16(), -r(2, 150, 4).abs(),
         torch.sigmoid(r(2, 150, 4))]
    logits, scores = r(4, 4, 20000), r(4, 4)
    ref = gated_delta_chunk_scan(*x), beam_select(logits, scores)
    lists = [(_i32(range(0, 16)), _i32(range(16, 32))), (_i32(range(32, 48)), _i32(range(48, 64)))]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = []
    for _ in range(5):
        for st, (a, b) in zip(streams, lists):
            with torch.cuda.stream(st):
                copy_slots(bufs, a, b)
                got.append((gated_delta_chunk_scan(*x), beam_select(logits, scores)))
    torch.cuda.synchronize()
    assert torch.equal(t[0], want)
    for y, sel in got:
        assert torch.equal(y, ref[0]) and all(torch.equal(m, n) for m, n in zip(sel, ref[1]))
    bufs.check_status()


@pytest.mark.parametrize("slots,parents,new,moves", [
    ([4, 4, 6], [0, 2, 2], [4, 6, -1], []),                       # row 0 lives on in the slot that row 1 also names
    ([4, 6, 4], [1, 1, 2], [6, -1, 4], []),
    ([4, 4, 4], [0, 0, 0], [4, -1, -1], []),                      # rows that still share one slot
    ([4, 4, 6, 9], [0, 2, 2, 2], [4, 6, 9, -1], [(6, 9)]),        # the free slot that one row alone names is given
    ([4, 4, 6, 9], [2, 2, 3, 3], [6, -1, 9, -1], []),             # nobody continues 4, but two rows name it
])
def test_reorder_gives_no_slot_that_another_row_names(slots, parents, new, moves):
    """A slot named twice is reported and never counts as free: nobody's state is written over."""
    from nested_ssm_b200 import StateBuffers, reorder_slots
    t = [torch.arange(2 * 12 * 4, dtype=torch.float32, device="cuda").view(2, 12, 4)]
    bufs = StateBuffers(t, slot_dim=1)
    want = _apply(t, moves)
    got = reorder_slots(bufs, _i32(slots), _i32(parents))
    assert got.tolist() == new
    _same(t, want)
    assert int(bufs.status) == 8


def test_reorder_reports_a_slot_named_twice_without_moves():
    from nested_ssm_b200 import StateBuffers, reorder_slots
    t = [torch.arange(12 * 4, dtype=torch.float32, device="cuda").view(12, 4)]
    bufs = StateBuffers(t)
    want = [t[0].clone()]
    assert reorder_slots(bufs, _i32([[4, 7], [7, -1]]), _i32([[0, 1], [0, 1]])).tolist() == [[4, 7], [7, -1]]
    _same(t, want)
    assert int(bufs.status) == 8


def test_slots_beyond_32_bits_are_reported():
    from nested_ssm_b200 import StateBuffers, copy_slots
    t = [torch.randn(8, 5, device="cuda")]
    bufs = StateBuffers(t)
    want = _apply(t, [(2, 6)], 0)
    copy_slots(bufs, torch.tensor([2, 1 << 32, 3], device="cuda"), torch.tensor([6, 4, (1 << 32) + 5], device="cuda"))
    _same(t, want)
    assert int(bufs.status) == 1
