"""Beam selection (nssm_beam_select) against a full sort in fp64, and a beam search over the operators
together.  Tokens and parents are equal (ties included); a score is one fp32 rounding of a sum whose
log-sum-exp has V fp32 terms: off by 2^-24 |score| and at most (2 + log2 V) 2^-22 of 1 + |lse|."""
import math

import pytest
import torch

import oracle.delta as OD

pytestmark = pytest.mark.gpu


def _check(got, logits, scores, n, finished=None, eos=None):
    s, p, t = got[:3]
    ws, wp, wt = OD.beam_select(logits, scores, n, finished, eos)
    assert p.dtype == torch.int32 and t.dtype == torch.int32 and s.dtype == torch.float32
    assert torch.equal(p.cpu().long(), wp) and torch.equal(t.cpu().long(), wt)
    fine = torch.isfinite(ws)
    assert torch.equal(torch.isfinite(s.cpu()), fine)
    top = float(torch.nan_to_num(logits.float(), neginf=0.0, posinf=0.0).abs().max())
    bound = 2.0 ** -23 * ws.abs() + (2 + math.log2(logits.shape[-1] + 1)) * 2.0 ** -22 * (1 + top)
    assert bool(((s.cpu().double() - ws).abs() <= bound)[fine].all())
    if eos is not None:
        f = (wt == eos) | (finished.cpu().gather(1, wp) if finished is not None else False)
        assert got[3].dtype == torch.bool and torch.equal(got[3].cpu(), f)


def _case(b, K, V, dtype, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (3 * torch.randn(b, K, V, generator=g, device="cuda")).to(dtype), -10 * torch.rand(b, K, generator=g, device="cuda")


@pytest.mark.parametrize("b,K,V,n,dtype", [
    (1, 1, 1, 1, torch.float32),
    (1, 1, 7, 7, torch.bfloat16),
    (2, 3, 5, 15, torch.float32),         # every candidate
    (3, 4, 100, 8, torch.bfloat16),
    (2, 5, 8191, 10, torch.bfloat16),     # odd rows: every alignment of a row's start
    (2, 4, 8192, 4, torch.bfloat16),
    (2, 4, 8193, 8, torch.float32),
    (1, 64, 333, 128, torch.float32),
    (2, 32, 20000, 64, torch.bfloat16),
    (5, 2, 50257, 4, torch.float32),
    (1, 2, 300001, 128, torch.bfloat16),
])
def test_select(b, K, V, n, dtype):
    from nested_ssm_b200 import beam_select
    x, s = _case(b, K, V, dtype, seed=V)
    _check(beam_select(x, s, n), x, s, n)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_ties_go_to_the_lower_beam_and_token(dtype):
    from nested_ssm_b200 import beam_select
    x = torch.zeros(2, 3, 9000, dtype=dtype, device="cuda")      # every candidate of a prompt ties
    x[1, :, ::2] = -0.0
    s = torch.zeros(2, 3, device="cuda")
    got = beam_select(x, s, 6)
    _check(got, x, s, 6)
    assert got[1][0].tolist() == [0] * 6 and got[2][0].tolist() == list(range(6))
    g = torch.Generator(device="cuda").manual_seed(0)
    x = torch.randint(-3, 4, (3, 4, 9001), generator=g, device="cuda").to(dtype)   # many ties at the cut
    s = torch.tensor([[0.0, 0.0, -1.0, 0.0]] * 3, device="cuda")
    _check(beam_select(x, s, 8), x, s, 8)


@pytest.mark.parametrize("order", ["ascending", "descending"])
def test_sorted_logits(order):
    """The worst orders for a threshold: every thread's values, and every list's, in order."""
    from nested_ssm_b200 import beam_select
    x = torch.linspace(-20, 20, 40000, device="cuda")
    x = (x if order == "ascending" else x.flip(0)).expand(2, 3, -1).contiguous()
    s = torch.tensor([[0.0, -1e-4, -2.5], [-3.0, -0.5, -0.5]], device="cuda")
    _check(beam_select(x, s, 128), x, s, 128)


def test_masked_infinite_and_dead():
    from nested_ssm_b200 import beam_select
    x, s = _case(6, 3, 5000, torch.float32, seed=1)
    inf, nan = float("inf"), float("nan")
    x[0, :, 10:] = -inf                    # ten tokens left
    x[1, 0] = -inf                         # a beam without tokens
    x[2] = -inf                            # a prompt without tokens
    x[3, 1, ::3] = nan
    x[3, 2, ::5] = inf                     # not finite: masked
    x[4, 1] = torch.finfo(torch.float32).min
    s[4, 0] = -inf                         # dead beams
    s[5] = -inf
    got = beam_select(x, s, 12)
    _check(got, x, s, 12)
    assert bool((got[0][2] == -inf).all()) and got[2][2].tolist() == list(range(12))


def test_first_step_of_a_search():
    """One live beam per prompt (the others start at -inf): all continuations come from it."""
    from nested_ssm_b200 import beam_select
    x, s = _case(4, 4, 1000, torch.bfloat16, seed=2)
    s[:] = torch.tensor([0.0] + [float("-inf")] * 3, device="cuda")
    got = beam_select(x, s)
    _check(got, x, s, 4)
    assert int(got[1].max()) == 0


@pytest.mark.parametrize("dtype,V", [(torch.float32, 700), (torch.bfloat16, 20001)])
def test_finished_beams(dtype, V):
    from nested_ssm_b200 import beam_select
    x, s = _case(4, 5, V, dtype, seed=3)
    fin = torch.zeros(4, 5, dtype=torch.bool, device="cuda")
    fin[0, 2] = fin[1, :4] = fin[2] = True
    x[:, :, V - 1] += 12.0                 # some beams end here
    x[1, 0] = float("nan")                 # a finished beam's logits are not looked at
    for n in (3, 5, 9):
        _check(beam_select(x, s, n, fin, V - 1), x, s, n, fin, V - 1)
    _check(beam_select(x, s, 5, None, 0), x, s, 5, None, 0)


def test_strided_logits():
    """The last token's logits of a [b*K, T, V] forward pass, and rows at odd offsets."""
    from nested_ssm_b200 import beam_select
    g = torch.Generator(device="cuda").manual_seed(4)
    full = torch.randn(6, 3, 4099, generator=g, device="cuda").bfloat16()
    x = full[:, -1].view(2, 3, 4099)
    s = torch.randn(2, 3, generator=g, device="cuda")
    _check(beam_select(x, s, 6), x, s, 6)
    y = full[:, 0, 1:].view(2, 3, 4098)
    _check(beam_select(y, s.t().contiguous().t(), 6), y, s, 6)


def test_offsets_beyond_32_bits():
    from nested_ssm_b200 import beam_select
    V = 1 << 16
    x = torch.zeros(2, 1, V, device="cuda", dtype=torch.bfloat16)
    big = torch.zeros((1 << 31) // V + 2, V, dtype=torch.bfloat16, device="cuda")
    x = torch.as_strided(big, (2, 1, V), ((1 << 31) // V * V, V, 1))
    g = torch.Generator(device="cuda").manual_seed(5)
    x[1, 0] = torch.randn(V, generator=g, device="cuda").bfloat16()
    s = torch.zeros(2, 1, device="cuda")
    _check(beam_select(x, s, 2), x, s, 2)


def test_replayed_graphs_and_another_stream():
    from nested_ssm_b200 import beam_select
    x, s = _case(3, 4, 30000, torch.float32, seed=6)
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        a = beam_select(x, s, 5)
    torch.cuda.current_stream().wait_stream(st)
    _check(a, x, s, 5)
    graphs, outs = [], []
    for n in (4, 8):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(beam_select(x, s, n))
        graphs.append(g)
    x2, s2 = _case(3, 4, 30000, torch.float32, seed=7)
    x.copy_(x2)
    s.copy_(s2)
    for g in graphs + graphs:
        g.replay()
    for o, n in zip(outs, (4, 8)):
        _check(o, x, s, n)


def test_beam_search_over_a_recurrent_layer():
    """Together, as a search uses them: a packed prefill into slots, forked to the beams, then per token
    the recurrent update, the selection and the reorder.  Against the same search in fp64 that keeps
    every beam's state by indexing."""
    from nested_ssm_b200 import (StateBuffers, beam_select, copy_slots, gated_delta_chunk_scan, gated_delta_state_update,
                                 reorder_slots)
    g = torch.Generator(device="cuda").manual_seed(8)
    b, K, H, G, P, N, V, steps = 3, 4, 2, 1, 32, 64, 50, 9
    r = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    emb = {n: r(V, *s) for n, s in (("q", (G, N)), ("k", (G, N)), ("v", (H, P)))}
    emb = {n: (t / t.norm(dim=-1, keepdim=True) if n != "v" else t).bfloat16() for n, t in emb.items()}
    emb["g"], emb["beta"] = -0.3 * torch.rand(V, H, generator=g, device="cuda"), torch.sigmoid(r(V, H))
    head = r(H * P, V).double()
    x = lambda tok: [emb[n][tok] for n in ("q", "k", "v", "g", "beta")]  # noqa: E731
    lens = [5, 1, 70]
    prompt = torch.randint(0, V, (1, sum(lens)), generator=g, device="cuda")
    cu = torch.tensor([0] + lens, device="cuda").cumsum(0).to(torch.int32)
    y, S = gated_delta_chunk_scan(*x(prompt), cu_seqlens=cu, return_final_states=True)
    last = y[0, cu[1:].long() - 1]
    state = torch.zeros(20, H, P, N, device="cuda")
    perm = torch.randperm(20, generator=g, device="cuda").to(torch.int32)
    slots = perm[:b * K].view(b, K).contiguous()
    state[slots[:, 0].long()] = S
    bufs = StateBuffers([state])
    copy_slots(bufs, slots[:, :1].expand(b, K - 1).reshape(-1), slots[:, 1:].reshape(-1))
    scores = torch.full((b, K), float("-inf"), device="cuda")
    scores[:, 0] = 0.0
    fin = torch.zeros(b, K, dtype=torch.bool, device="cuda")
    logits = (last.double().reshape(b, 1, -1) @ head).float().expand(b, K, V)
    ref = S.double()[:, None].expand(b, K, H, P, N).clone()
    for step in range(steps):
        scores, parents, tokens, fin = beam_select(logits, scores, K, fin, 0)
        slots = reorder_slots(bufs, slots, parents)
        ref = ref.gather(1, parents.long()[..., None, None, None].expand(b, K, H, P, N))
        y = gated_delta_state_update(state, *x(tokens.reshape(-1).long()), state_batch_indices=slots.reshape(-1))
        q, k, v, gg, beta = (t.double() for t in x(tokens.long()))
        ref, yr = OD.gated_delta_token(ref, q.expand(b, K, H, N), k.expand(b, K, H, N), v, gg, beta, N ** -0.5)
        assert float((y.double().view(b, K, H, P) - yr).norm() / yr.norm()) <= 2.5e-3, step
        assert float((state[slots.long()].double() - ref).norm() / ref.norm()) <= 1e-5, step
        logits = (yr.reshape(b, K, -1) @ head).float()
    bufs.check_status()


@pytest.mark.parametrize("n", [3, 16, 128])
@pytest.mark.parametrize("order", ["random", "ascending", "descending", "few values"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_long_parts(n, order, dtype):
    """So many rows that one CTA walks a whole row in many steps, the bound rising on the way: against the
    sort for one prompt; every prompt has the same logits and scores."""
    from nested_ssm_b200 import beam_select
    b, K, V = 56, 16, 70001
    g = torch.Generator(device="cuda").manual_seed(n)
    x = {"random": lambda: 3 * torch.randn(K, V, generator=g, device="cuda"),
         "ascending": lambda: torch.linspace(-20, 20, V, device="cuda").expand(K, V),
         "descending": lambda: torch.linspace(20, -20, V, device="cuda").expand(K, V),
         "few values": lambda: torch.randint(-2, 3, (K, V), generator=g, device="cuda").float()}[order]()
    x = x.to(dtype)
    s = -torch.rand(b, K, generator=g, device="cuda")
    s[1:] = s[:1]
    got = beam_select(x.expand(b, K, V), s, n)
    _check([t[:1] for t in got], x[None], s[:1], n)
    for t in got:
        assert torch.equal(t, t[:1].expand_as(t))


def _best(logits, scores, n):
    """(totals fp64, parents, tokens) by a sort of (score + x) - lse in 64 bits, as the totals are defined: total
    descending, then beam, then logit descending, then token."""
    x = logits.double().cpu()
    top = x.amax(-1, keepdim=True)
    total = (scores.double().cpu()[..., None] + x) - ((x - top).exp().sum(-1, keepdim=True).log() + top)
    b, K, V = x.shape
    got = []
    for i in range(b):
        rank = torch.sort(x[i], dim=-1, descending=True, stable=True).indices[:, :n]
        kept = [(-float(total[i, k, t]), k, r, t) for k in range(K) for r, t in enumerate(rank[k].tolist())]
        got.append(sorted(kept)[:n])
    pick = lambda j, dt: torch.tensor([[c[j] for c in row] for row in got], dtype=dt)  # noqa: E731
    return -pick(0, torch.float64), pick(1, torch.long), pick(3, torch.long)


def _size(logits, parents):
    """The largest magnitude of each continued beam's logits that count in its sum (the largest is one)."""
    return logits.double().amax(-1).abs().cpu().gather(1, parents)


def _check_best(got, logits, scores, n):
    """A total is one fp32 rounding (2^-24 of it) of a sum whose log-sum-exp, with d = max - x, has terms off by
    3 2^-24 d in the exponent (the mean of d under the softmax is at most ln V), by 2^-22 of themselves and of
    their rescaling, and by 2^-24 for each of the at most 32 + V / 512 additions in turn.  Only the three 64-bit
    roundings behind a total grow with the logits."""
    ws, wp, wt = _best(logits, scores, n)
    V = logits.shape[-1]
    assert torch.equal(got[1].cpu().long(), wp) and torch.equal(got[2].cpu().long(), wt)
    bound = 2.0 ** -24 * (ws.abs() + 3 * math.log(V) + 8 + 32 + V / 512) + 3 * 2.0 ** -53 * _size(logits, wp)
    err = (got[0].cpu().double() - ws).abs()
    assert bool((err <= bound).all()), float((err / bound).max())


@pytest.mark.parametrize("value", [-1e4, -1e9, -1e10, -1e12, -1e18, -1e20, -1e30, -3e38])
@pytest.mark.parametrize("where", ["most", "tail", "head"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_finite_masks(value, where, dtype):
    """Banned tokens at a large negative number: a thread, or all of a part, sees nothing else at first or at
    all, and adds nothing to the sum."""
    from nested_ssm_b200 import beam_select
    V = 20001
    x, s = _case(2, 3, V, dtype, seed=11)
    keep = torch.zeros(V, dtype=torch.bool, device="cuda")
    keep[{"most": slice(5, None, 997), "tail": slice(0, 1200), "head": slice(V - 37, None)}[where]] = True
    x.masked_fill_(~keep, value)
    _check_best(beam_select(x, s, 8), x, s, 8)


@pytest.mark.parametrize("offset", [1e3, -1e3, 1e5, -1e5, 1e6, -1e6, 1e8, -1e8, -1e9, 1e20, -1e30])
@pytest.mark.parametrize("dtype,V", [(torch.float32, 5000), (torch.bfloat16, 30000)])
def test_logits_far_from_zero(offset, dtype, V):
    """The same selection at any offset, as far as the type holds the differences."""
    from nested_ssm_b200 import beam_select
    x, s = _case(3, 4, V, dtype, seed=12)
    x = (x.double() + offset).to(dtype)
    _check_best(beam_select(x, s, 6), x, s, 6)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_beams_of_one_large_value(dtype):
    """A beam whose every token has the same large value has finite totals, whatever the value."""
    from nested_ssm_b200 import beam_select
    x, s = _case(3, 3, 9000, dtype, seed=13)
    x[0, 1], x[1, 0], x[2] = -1e30, 3e38, torch.finfo(dtype).min
    _check_best(beam_select(x, s, 7), x, s, 7)
