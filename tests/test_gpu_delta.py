"""The gated delta rule (nssm_delta_step, nssm_delta_scan) against its definition in fp64.

Error bounds.  A rounding to a type of relative step eps is off by eps / 2 at most (fp32 2^-24,
bf16 2^-8).

* One decode token: every value is a dot product of N fp32 terms and a few more operations, so it
  is off by at most (N + 16) 2^-24 of the sum of its terms' magnitudes (`_step_bounds`), plus the
  rounding of the output.
* A prompt: the state's own roundings are 2^-24 each, and no product is formed from operands
  held to fewer than 17 bits, 2^-18 of each; a state remembers a handful of chunks, whose
  errors add up, so the norm of the difference is below 8 2^-18 = 3.1e-5 of the state's at worst and
  2^-18 sqrt(8) = 1.1e-5 for errors of random sign: 1e-5 is asked for.  An output may be formed
  from operands rounded to bf16 (2^-8 at most, 2^-9 / sqrt(3) = 1.1e-3 in the mean square): its own
  rounding (1.7e-3) and three such operands give 2.5e-3 of the norm; no value is off by more
  than its own half step and 3 2^-8 of the root mean square of its row times 4.
"""
import pytest
import torch

import oracle.delta as OD

pytestmark = pytest.mark.gpu
STATE_TOL, Y_TOL = 1e-5, 2.5e-3


def _unit(t):
    return t / t.norm(dim=-1, keepdim=True)


def _inputs(b, T, H, G, P, N, seed, dtype=torch.bfloat16, gdt=torch.float32, decay=0.3):
    g = torch.Generator(device="cuda").manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    return dict(q=_unit(r(b, T, G, N)).to(dtype), k=_unit(r(b, T, G, N)).to(dtype), v=r(b, T, H, P).to(dtype),
                g=(-decay * torch.nn.functional.softplus(r(b, T, H))).to(gdt), beta=torch.sigmoid(r(b, T, H)).to(gdt),
                s0=0.5 * r(b, H, P, N))


def _rel(got, want):
    n = float(want.double().norm())
    return float((got.double() - want.double()).norm()) / n if n else float(got.double().norm())


def _check_y(got, want, what=""):
    assert torch.isfinite(got).all(), what
    if not got.numel():
        return
    assert _rel(got, want) <= Y_TOL, f"{what}: {_rel(got, want):.2e}"
    rms = want.square().mean(-1, keepdim=True).sqrt()
    bound = 2.0 ** -8 * want.abs() + 12 * 2.0 ** -8 * rms + 1e-6
    err = (got.double() - want).abs()
    assert bool((err <= bound).all()), f"{what}: {float((err / bound).max()):.2f} of the bound"


def _check_state(got, want, what=""):
    assert torch.isfinite(got).all(), what
    assert _rel(got, want) <= STATE_TOL, f"{what}: {_rel(got, want):.2e}"


# ---------------------------------------------------------------- decode
def _step_case(b, S, H, G, P, N, dtype, seed, gdt=torch.float32):
    d = _inputs(b, 1, H, G, P, N, seed, dtype, gdt)
    x = {n: d[n][:, 0] for n in ("q", "k", "v", "g", "beta")}
    gen = torch.Generator(device="cuda").manual_seed(seed + 1)
    state = torch.randn(S, H, P, N, generator=gen, device="cuda")
    slots = torch.randperm(S, generator=gen, device="cuda")[:b].to(torch.int32)
    return x, state, slots


def _step_ref(x, state, slots, scale, out, rows):
    """(state', out') in fp64 with the listed rows taken, and the bounds of both."""
    S, y = state.double(), out.double()
    N = state.shape[-1]
    bS, by = torch.zeros_like(S), torch.zeros_like(y)
    rep = state.shape[1] // x["q"].shape[1]
    half = torch.finfo(out.dtype).eps / 2
    for r in rows:
        q, k = (x[n][r].double().repeat_interleave(rep, 0) for n in ("q", "k"))
        v, g, beta = (x[n][r].double() for n in ("v", "g", "beta"))
        old = torch.exp(g)[:, None, None] * S[slots[r]]
        new, yr = OD.gated_delta_token(S[slots[r]], q, k, v, g, beta, scale)
        e = (N + 16) * 2.0 ** -24
        u = beta.abs()[:, None] * (v.abs() + (old.abs() * k.abs()[:, None]).sum(-1))     # >= |u|
        bS[slots[r]] = e * (old.abs() + u[..., None] * k.abs()[:, None])
        by[r] = half * yr.abs() + 2 * e * scale * ((old.abs() * q.abs()[:, None]).sum(-1) + u * (k.abs() * q.abs()).sum(-1)[:, None])
        S[slots[r]], y[r] = new, yr
    return S, y, bS, by


def _check_step(state, out, ref):
    S, y, bS, by = ref
    assert bool(((state.double() - S).abs() <= bS).all())    # untouched slots: exactly
    assert bool(((out.double() - y).abs() <= by).all())


@pytest.mark.parametrize("b,S,H,G,P,N,dtype,gdt", [
    (1, 1, 1, 1, 16, 64, torch.bfloat16, torch.float32),
    (3, 7, 4, 2, 64, 128, torch.bfloat16, torch.bfloat16),
    (5, 5, 6, 2, 80, 128, torch.float32, torch.float32),
    (2, 9, 4, 4, 48, 64, torch.float32, torch.bfloat16),
    (4, 6, 8, 1, 112, 128, torch.bfloat16, torch.float32),
    (2, 3, 2, 1, 256, 128, torch.float32, torch.float32),
    (70, 300, 2, 1, 128, 64, torch.bfloat16, torch.float32),
])
def test_step(b, S, H, G, P, N, dtype, gdt):
    from nested_ssm_b200 import gated_delta_state_update
    x, state, slots = _step_case(b, S, H, G, P, N, dtype, seed=b + P, gdt=gdt)
    out = torch.full((b, H, P), 7.0, dtype=dtype, device="cuda")
    ref = _step_ref(x, state, slots.long(), N ** -0.5, out, range(b))
    got = gated_delta_state_update(state, x["q"], x["k"], x["v"], x["g"], x["beta"], state_batch_indices=slots, out=out)
    assert got is out
    _check_step(state, out, ref)


def test_step_padded_out_of_range_and_repeated_rows():
    from nested_ssm_b200 import gated_delta_state_update
    x, state, slots = _step_case(8, 12, 4, 2, 64, 128, torch.bfloat16, seed=3)
    slots[1] = -1           # padded
    slots[4] = 12           # out of range
    slots[6] = slots[2]     # named by an earlier row
    slots[7] = -5
    out = torch.full((8, 4, 64), 7.0, device="cuda", dtype=torch.bfloat16)
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    ref = _step_ref(x, state, slots.long(), 0.25, out, [0, 2, 3, 5])
    gated_delta_state_update(state, x["q"], x["k"], x["v"], x["g"], x["beta"], 0.25, slots, out=out, status=status)
    _check_step(state, out, ref)
    assert int(status) == 1 | 8


def test_step_pad_id_zero_and_index_column():
    """vLLM's null block 0 as the pad id, and indices of shape [b, 1]."""
    from nested_ssm_b200 import gated_delta_state_update
    x, state, slots = _step_case(4, 9, 2, 2, 32, 64, torch.float32, seed=5)
    slots = torch.tensor([3, 0, 8, 5], dtype=torch.int64, device="cuda")[:, None]
    out = torch.zeros(4, 2, 32, device="cuda")
    ref = _step_ref(x, state, slots[:, 0], 64 ** -0.5, out, [0, 2, 3])
    gated_delta_state_update(state, x["q"], x["k"], x["v"], x["g"], x["beta"], None, slots, pad_slot_id=0, out=out)
    _check_step(state, out, ref)


def test_step_strided_and_unaligned_inputs():
    """q, k, v, g, beta as slices of one projection (odd offsets), a state of spaced slots."""
    from nested_ssm_b200 import gated_delta_state_update
    b, S, H, G, P, N = 3, 5, 4, 2, 48, 128
    x, state, slots = _step_case(b, S, H, G, P, N, torch.bfloat16, seed=8)
    w = 2 * G * N + H * P + 2 * H + 3
    proj = torch.zeros(b, w, dtype=torch.bfloat16, device="cuda")
    at, v = 1, {}
    for n in ("q", "k", "v", "g", "beta"):
        size = x[n][0].numel()
        proj[:, at:at + size] = x[n].reshape(b, -1).to(torch.bfloat16)
        v[n] = proj[:, at:at + size].view(b, *x[n].shape[1:])
        at += size
    wide = torch.randn(S, 2, H, P, N, device="cuda")
    wide[:, 1] = state
    other = wide[:, 0].clone()
    out = torch.zeros(b, 2 * H, P, device="cuda")[:, ::2]
    ref = _step_ref(v, state, slots.long(), N ** -0.5, out, range(b))
    gated_delta_state_update(wide[:, 1], v["q"], v["k"], v["v"], v["g"], v["beta"], None, slots, out=out)
    _check_step(wide[:, 1], out, ref)
    assert torch.equal(wide[:, 0], other)


def test_step_empty_batch():
    from nested_ssm_b200 import gated_delta_state_update
    x, state, _ = _step_case(2, 2, 2, 1, 32, 64, torch.bfloat16, seed=9)
    before = state.clone()
    out = gated_delta_state_update(state, *(x[n][:0] for n in ("q", "k", "v", "g", "beta")))
    assert out.shape == (0, 2, 32) and torch.equal(state, before)


def test_step_state_offsets_beyond_32_bits():
    from nested_ssm_b200 import gated_delta_state_update
    H, P, N = 32, 128, 128
    S = (1 << 31) // (H * P * N) + 3
    state = torch.zeros(S, H, P, N, device="cuda")
    x, small, _ = _step_case(2, 2, H, 16, P, N, torch.bfloat16, seed=10)
    slots = torch.tensor([S - 1, 0], dtype=torch.int32, device="cuda")
    state[S - 1], state[0] = small[0], small[1]
    out = torch.zeros(2, H, P, device="cuda", dtype=torch.bfloat16)
    ref = _step_ref(x, small, torch.arange(2), N ** -0.5, out, range(2))
    gated_delta_state_update(state, x["q"], x["k"], x["v"], x["g"], x["beta"], None, slots, out=out)
    _check_step(torch.stack([state[S - 1], state[0]]), out, ref)
    assert float(state[1:S - 1].abs().max()) == 0.0


# ---------------------------------------------------------------- prompts
@pytest.mark.parametrize("b,T,H,G,P,N,init", [
    (1, 1, 1, 1, 16, 64, False),
    (2, 2, 2, 1, 32, 128, True),
    (1, 15, 4, 2, 80, 128, True),
    (3, 16, 2, 2, 64, 64, False),
    (1, 17, 2, 1, 112, 64, True),
    (2, 63, 4, 1, 48, 128, False),
    (1, 64, 4, 2, 128, 128, True),
    (1, 65, 2, 2, 96, 64, True),
    (2, 127, 3, 3, 16, 128, True),
    (1, 128, 2, 1, 256, 128, False),
    (1, 129, 2, 1, 144, 64, True),
    (2, 300, 4, 2, 80, 128, True),
    (1, 1000, 2, 1, 64, 128, False),
    (1, 777, 8, 8, 128, 64, True),
])
def test_scan(b, T, H, G, P, N, init):
    from nested_ssm_b200 import gated_delta_chunk_scan
    d = _inputs(b, T, H, G, P, N, seed=T + P)
    s0 = d["s0"] if init else None
    y, S = gated_delta_chunk_scan(d["q"], d["k"], d["v"], d["g"], d["beta"], initial_states=s0, return_final_states=True)
    yr, Sr = OD.gated_delta_scan(d["q"], d["k"], d["v"], d["g"], d["beta"], S0=s0)
    _check_y(y, yr)
    _check_state(S, Sr)


@pytest.mark.parametrize("lens,H,G,P,N,init", [
    ([5], 2, 1, 16, 64, True),
    ([0, 1, 0, 64, 65, 0], 4, 2, 80, 128, True),
    ([130, 1, 63, 200], 2, 2, 64, 128, False),
    ([3] * 40, 2, 1, 48, 64, True),
])
def test_scan_packed(lens, H, G, P, N, init):
    """Ragged sequences in one row, with empty ones, and rows behind the last that hold NaN: they are
    neither read nor written."""
    from nested_ssm_b200 import gated_delta_chunk_scan
    total = sum(lens) + 7
    d = _inputs(1, total, H, G, P, N, seed=len(lens))
    for n in ("q", "k", "v", "g", "beta"):
        d[n][:, sum(lens):] = float("nan")
    cu = torch.tensor([0] + lens, device="cuda").cumsum(0).to(torch.int32)
    g = torch.Generator(device="cuda").manual_seed(1)
    s0 = torch.randn(len(lens), H, P, N, generator=g, device="cuda") if init else None
    out = torch.full((1, total, H, P), 3.0, dtype=torch.bfloat16, device="cuda")
    y, S = gated_delta_chunk_scan(d["q"], d["k"], d["v"], d["g"], d["beta"], initial_states=s0, cu_seqlens=cu,
                                  return_final_states=True, out=out)
    assert S.shape == (len(lens), H, P, N)
    at = 0
    for i, n in enumerate(lens):
        x = [d[m][:, at:at + n] for m in ("q", "k", "v", "g", "beta")]
        yr, Sr = OD.gated_delta_scan(*x, S0=None if s0 is None else s0[i:i + 1])
        _check_y(y[:, at:at + n], yr, f"sequence {i}")
        if n == 0:
            assert torch.equal(S[i], s0[i] if init else torch.zeros_like(S[i]))
        else:
            _check_state(S[i], Sr[0], f"sequence {i}")
        at += n
    assert bool((y[:, at:] == 3.0).all())


def test_scan_bad_bounds_are_skipped():
    from nested_ssm_b200 import gated_delta_chunk_scan
    d = _inputs(1, 100, 2, 1, 32, 64, seed=4)
    cu = torch.tensor([0, 70, 40, 100, 170], dtype=torch.int32, device="cuda")   # 1 descends, 3 leaves the rows
    out = torch.full((1, 100, 2, 32), 3.0, dtype=torch.bfloat16, device="cuda")
    fin = torch.full((4, 2, 32, 64), 5.0, device="cuda")
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    # sequences 0 and 2 overlap: run each against a list in which the other is bad
    gated_delta_chunk_scan(d["q"], d["k"], d["v"], d["g"], d["beta"], cu_seqlens=cu, out=out, final_states=fin,
                           status=status)
    assert int(status) == 8
    assert bool((fin[1] == 5.0).all()) and bool((fin[3] == 5.0).all())
    for s, (a, e) in ((0, (0, 70)), (2, (40, 100))):
        _, Sr = OD.gated_delta_scan(*(d[m][:, a:e] for m in ("q", "k", "v", "g", "beta")))
        _check_state(fin[s], Sr[0])


@pytest.mark.parametrize("T", [0, 1, 70])
def test_scan_states_in_place_and_without_tokens(T):
    """final_states may be initial_states; without tokens the state stays."""
    from nested_ssm_b200 import gated_delta_chunk_scan
    d = _inputs(2, T, 4, 2, 48, 128, seed=6)
    s = d["s0"].clone()
    y, S = gated_delta_chunk_scan(d["q"], d["k"], d["v"], d["g"], d["beta"], initial_states=s, return_final_states=True,
                                  final_states=s)
    assert S is s and y.shape == (2, T, 4, 48)
    if T == 0:
        assert torch.equal(s, d["s0"])
        _, z = gated_delta_chunk_scan(d["q"], d["k"], d["v"], d["g"], d["beta"], return_final_states=True)
        assert float(z.abs().max()) == 0.0
    else:
        _, Sr = OD.gated_delta_scan(d["q"], d["k"], d["v"], d["g"], d["beta"], S0=d["s0"])
        _check_state(s, Sr)


@pytest.mark.parametrize("gdt", [torch.float32, torch.bfloat16])
def test_scan_strided_inputs_and_outputs(gdt):
    """q / k / v as slices of one conv output, g / beta of one projection, y into a wider row."""
    from nested_ssm_b200 import gated_delta_chunk_scan
    b, T, H, G, P, N = 2, 150, 4, 2, 80, 128
    d = _inputs(b, T, H, G, P, N, seed=12, gdt=gdt)
    conv = torch.cat([d[n].reshape(b, T, -1) for n in ("q", "k", "v")], -1)
    q, k, v = conv.split([G * N, G * N, H * P], -1)
    proj = torch.cat([d["g"], d["beta"]], -1)
    wide = torch.zeros(b, T, 2 * H * P, dtype=torch.bfloat16, device="cuda")
    out = wide[..., H * P:].view(b, T, H, P)
    y, S = gated_delta_chunk_scan(q.view(b, T, G, N), k.view(b, T, G, N), v.view(b, T, H, P), proj[..., :H], proj[..., H:],
                                  scale=0.3, initial_states=d["s0"], return_final_states=True, out=out)
    assert y.data_ptr() == out.data_ptr() and float(wide[..., :H * P].abs().max()) == 0.0
    yr, Sr = OD.gated_delta_scan(d["q"], d["k"], d["v"], d["g"], d["beta"], 0.3, d["s0"])
    _check_y(y, yr)
    _check_state(S, Sr)


def test_scan_takes_unaligned_heads_and_broadcast_batches():
    """Inputs the kernel cannot load as they lie (transposed heads, odd offsets, an expanded batch)
    are laid out by the call."""
    from nested_ssm_b200 import gated_delta_chunk_scan
    b, T, H, G, P, N = 2, 33, 4, 2, 16, 64
    d = _inputs(b, T, H, G, P, N, seed=13)
    q = d["q"].transpose(1, 2).contiguous().transpose(1, 2)
    flat = torch.zeros(d["v"].numel() + 1, dtype=torch.bfloat16, device="cuda")
    flat[1:] = d["v"].reshape(-1)
    v = flat[1:].view(b, T, H, P)
    k = d["k"][:1].expand(b, T, G, N)
    beta = d["beta"][:, :, :1].expand(b, T, H)
    y = gated_delta_chunk_scan(q, k, v, d["g"], beta)
    yr, _ = OD.gated_delta_scan(q, k, v, d["g"], beta)
    _check_y(y, yr)


def test_scan_forgets_at_minus_infinity_and_keeps_small_decays_beside_large_ones():
    """g = -inf forgets the state; a large decay early in a chunk does not blur the small ones behind
    it."""
    from nested_ssm_b200 import gated_delta_chunk_scan
    d = _inputs(1, 200, 2, 1, 32, 64, seed=14)
    d["g"] = -0.01 * torch.rand(1, 200, 2, device="cuda")
    d["g"][:, 3] = -3000.0
    d["g"][:, 70, 0] = float("-inf")
    d["g"][:, 128] = -50.0
    d["s0"] *= 100
    y, S = gated_delta_chunk_scan(d["q"], d["k"], d["v"], d["g"], d["beta"], initial_states=d["s0"], return_final_states=True)
    yr, Sr = OD.gated_delta_scan(d["q"], d["k"], d["v"], d["g"], d["beta"], S0=d["s0"])
    _check_y(y[:, 3:], yr[:, 3:])
    _check_state(S, Sr)


def test_scan_collinear_keys():
    """The same key at every token with beta near 1: the system of a chunk is as far from the identity
    as it gets, and u stays small only by cancellation."""
    from nested_ssm_b200 import gated_delta_chunk_scan
    d = _inputs(1, 160, 2, 1, 32, 64, seed=15)
    d["k"] = d["k"][:, :1].expand_as(d["k"]).contiguous()
    d["beta"] = torch.full_like(d["beta"], 0.97)
    d["g"] = torch.zeros_like(d["g"])
    y, S = gated_delta_chunk_scan(d["q"], d["k"], d["v"], d["g"], d["beta"], initial_states=d["s0"], return_final_states=True)
    yr, Sr = OD.gated_delta_scan(d["q"], d["k"], d["v"], d["g"], d["beta"], S0=d["s0"])
    _check_y(y, yr)
    _check_state(S, Sr)


def test_scan_without_writes_keeps_the_state_exactly():
    from nested_ssm_b200 import gated_delta_chunk_scan
    d = _inputs(1, 100, 2, 1, 48, 128, seed=16)
    _, S = gated_delta_chunk_scan(d["q"], d["k"], d["v"], torch.zeros_like(d["g"]), torch.zeros_like(d["beta"]),
                                  initial_states=d["s0"], return_final_states=True)
    assert torch.equal(S, d["s0"])


def test_scan_is_deterministic_and_sequences_are_independent():
    from nested_ssm_b200 import gated_delta_chunk_scan
    d = _inputs(3, 190, 4, 2, 64, 128, seed=17)
    x = [d[n] for n in ("q", "k", "v", "g", "beta")]
    a = gated_delta_chunk_scan(*x, initial_states=d["s0"], return_final_states=True)
    b = gated_delta_chunk_scan(*x, initial_states=d["s0"], return_final_states=True)
    one = gated_delta_chunk_scan(*(t[1:2] for t in x), initial_states=d["s0"][1:2], return_final_states=True)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    assert torch.equal(a[0][1:2], one[0]) and torch.equal(a[1][1:2], one[1])


def test_prefill_then_decode_equals_the_longer_prompt():
    """A packed prefill whose states go to slots, then decode tokens on the slots."""
    from nested_ssm_b200 import gated_delta_chunk_scan, gated_delta_state_update
    b, T, extra, H, G, P, N = 3, 70, 4, 4, 2, 80, 128
    d = _inputs(b, T + extra, H, G, P, N, seed=18)
    x = [d[n] for n in ("q", "k", "v", "g", "beta")]
    yr, Sr = OD.gated_delta_scan(*x)
    pack = [t[:, :T].reshape(1, b * T, *t.shape[2:]) for t in x]
    cu = torch.arange(0, b * T + 1, T, dtype=torch.int32, device="cuda")
    _, S = gated_delta_chunk_scan(*pack, cu_seqlens=cu, return_final_states=True)
    state = torch.zeros(8, H, P, N, device="cuda")
    slots = torch.tensor([5, 0, 7], dtype=torch.int32, device="cuda")
    state[slots.long()] = S
    for t in range(T, T + extra):
        y = gated_delta_state_update(state, *(z[:, t] for z in x), state_batch_indices=slots)
        _check_y(y, yr[:, t])
    _check_state(state[slots.long()], Sr)


def test_on_another_stream_and_in_a_replayed_graph():
    from nested_ssm_b200 import gated_delta_chunk_scan, gated_delta_state_update
    d = _inputs(2, 90, 4, 2, 64, 128, seed=19)
    names = ("q", "k", "v", "g", "beta")
    x = [d[n] for n in names]
    want = gated_delta_chunk_scan(*x, initial_states=d["s0"], return_final_states=True)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = gated_delta_chunk_scan(*x, initial_states=d["s0"], return_final_states=True)
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    graphs, outs = [], []
    for _ in range(2):      # two graphs, replayed in turn
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            y, S = gated_delta_chunk_scan(*x, initial_states=d["s0"], return_final_states=True)
            z = gated_delta_state_update(S, *(t[:, 0] for t in x))
        graphs.append(g)
        outs.append((y, S, z))
    e = _inputs(2, 90, 4, 2, 64, 128, seed=20)
    for n in names:
        d[n].copy_(e[n])
    d["s0"].copy_(e["s0"])
    y, S = gated_delta_chunk_scan(*x, initial_states=d["s0"], return_final_states=True)
    z = gated_delta_state_update(S, *(t[:, 0] for t in x))
    for g in graphs + graphs:
        g.replay()
    for o in outs:
        assert torch.equal(o[0], y) and torch.equal(o[1], S) and torch.equal(o[2], z)


def test_axes_of_one_may_have_any_stride():
    """One head, one sequence: the strides of such axes say nothing."""
    from nested_ssm_b200 import gated_delta_chunk_scan, gated_delta_state_update
    P, N, T = 32, 64, 40
    d = _inputs(1, T, 1, 1, P, N, seed=21)
    yr, Sr = OD.gated_delta_scan(d["q"], d["k"], d["v"], d["g"], d["beta"], S0=d["s0"])
    odd = lambda t, *s: torch.as_strided(t, t.shape, s)  # noqa: E731
    out = odd(torch.zeros(1, T, 1, P, device="cuda", dtype=torch.bfloat16), 8, P, 5, 1)
    fin = odd(torch.zeros(1, 1, P, N, device="cuda"), 4, 12, N, 1)
    y, S = gated_delta_chunk_scan(odd(d["q"], 8, N, 3, 1), d["k"], d["v"], d["g"], d["beta"],
                                  initial_states=odd(d["s0"], 8, 4, N, 1), return_final_states=True, out=out,
                                  final_states=fin)
    _check_y(y, yr)
    _check_state(S, Sr)
    state = odd(d["s0"].clone(), 0, 7, N, 1)
    x = [d[n][:, 0] for n in ("q", "k", "v", "g", "beta")]
    z = gated_delta_state_update(state, *x)
    _check_y(z, yr[:, 0])


def test_wide_ranges_of_values():
    """Keys of very different lengths from token to token (beta holds their step in range), values up to
    1e4 and down to 1e-4, a state of rows that differ by 1e4: the scales of the split operands."""
    from nested_ssm_b200 import gated_delta_chunk_scan
    b, T, H, G, P, N = 1, 150, 2, 1, 32, 128
    d = _inputs(b, T, H, G, P, N, seed=22)
    g = torch.Generator(device="cuda").manual_seed(23)
    length = 10.0 ** (2 * torch.rand(b, T, 1, 1, generator=g, device="cuda") - 1)
    d["k"] = (d["k"].float() * length).bfloat16()
    d["beta"] = d["beta"] / d["k"].float().square().sum(-1).expand(b, T, H)
    d["q"] = (d["q"].float() * 10.0 ** (6 * torch.rand(b, T, 1, 1, generator=g, device="cuda") - 3)).bfloat16()
    d["v"] = (d["v"].float() * 10.0 ** (8 * torch.rand(b, T, 1, 1, generator=g, device="cuda") - 4)).bfloat16()
    d["s0"] *= 10.0 ** (4 * torch.rand(b, H, P, 1, generator=g, device="cuda"))
    y, S = gated_delta_chunk_scan(d["q"], d["k"], d["v"], d["g"], d["beta"], initial_states=d["s0"], return_final_states=True)
    yr, Sr = OD.gated_delta_scan(d["q"], d["k"], d["v"], d["g"], d["beta"], S0=d["s0"])
    _check_state(S, Sr)
    assert _rel(y, yr) <= Y_TOL


def test_a_value_that_is_not_finite_stays_in_its_sequence_and_block():
    from nested_ssm_b200 import gated_delta_chunk_scan
    d = _inputs(2, 130, 2, 1, 32, 64, seed=24)
    yr, Sr = OD.gated_delta_scan(d["q"], d["k"], d["v"], d["g"], d["beta"])
    d["v"][0, 70, 1, 3] = float("nan")
    y, S = gated_delta_chunk_scan(d["q"], d["k"], d["v"], d["g"], d["beta"], return_final_states=True)
    _check_y(y[1], yr[1])
    _check_state(S[1], Sr[1])
    _check_y(y[0, :64], yr[0, :64])                      # blocks of 32 tokens before it
    assert bool(torch.isnan(y[0, 70:, 1, 3]).all())
    _check_y(y[0, :, 0], yr[0, :, 0])                    # the other head


@pytest.mark.parametrize("b,T,H,G,P,N,packed", [
    (24, 70, 8, 2, 80, 128, False),
    (80, 100, 8, 2, 16, 64, False),       # four heads in a CTA
    (40, 200, 16, 4, 128, 128, True),
    (50, 33, 12, 4, 48, 64, True),
])
def test_scan_of_more_work_than_sms(b, T, H, G, P, N, packed):
    """Enough sequences and heads that CTAs share SMs: the other form of the walk."""
    from nested_ssm_b200 import gated_delta_chunk_scan
    d = _inputs(b, T, H, G, P, N, seed=b + T)
    x = [d[n] for n in ("q", "k", "v", "g", "beta")]
    yr, Sr = OD.gated_delta_scan(*x, S0=d["s0"])
    cu = None
    if packed:
        x = [t.reshape(1, b * T, *t.shape[2:]) for t in x]
        cu = torch.arange(0, b * T + 1, T, dtype=torch.int32, device="cuda")
    y, S = gated_delta_chunk_scan(*x, initial_states=d["s0"], cu_seqlens=cu, return_final_states=True)
    _check_y(y.view(b, T, H, P), yr)
    _check_state(S, Sr)
    one = gated_delta_chunk_scan(*(d[n][:1] for n in ("q", "k", "v", "g", "beta")), initial_states=d["s0"][:1],
                                 return_final_states=True)
    assert torch.equal(one[0], y.view(b, T, H, P)[:1]) and torch.equal(one[1], S[:1])    # and the same values


@pytest.mark.parametrize("b,T", [(1, 100), (80, 40)])
def test_a_copy_that_never_completes_times_out(b, T):
    """The injected stuck copy (the first CTA announces 16 bytes more than arrive): its waits run out, the
    call returns with bit 1 set, other sequences are as ever and the next call is right."""
    from nested_ssm_b200 import _lib, gated_delta_chunk_scan
    lib = _lib.load()
    H, G, P, N = 8, 2, 64, 128
    d = _inputs(b, T, H, G, P, N, seed=25)
    x = [d[n] for n in ("q", "k", "v", "g", "beta")]
    want = gated_delta_chunk_scan(*x, return_final_states=True)
    torch.cuda.synchronize()
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    polls, stuck = lib.nssm_set_wait_polls(4096), lib.nssm_test_inject_stuck_copy(1)
    try:
        got = gated_delta_chunk_scan(*x, return_final_states=True, status=status)
        torch.cuda.synchronize()
    finally:
        lib.nssm_test_inject_stuck_copy(stuck)
        lib.nssm_set_wait_polls(polls)
    assert int(status) == 2
    assert torch.equal(got[0][1:], want[0][1:]) and torch.equal(got[1][1:], want[1][1:])
    again = gated_delta_chunk_scan(*x, return_final_states=True, status=status.zero_())
    assert torch.equal(again[0], want[0]) and torch.equal(again[1], want[1]) and int(status) == 0


def _both_walks():
    """A call with fewer CTAs than SMs and one with more."""
    return pytest.mark.parametrize("b,H", [(1, 2), (80, 8)])


@_both_walks()
@pytest.mark.parametrize("N,init", [(64, True), (128, False), (128, True)])
def test_an_output_is_the_formula_rounded_once(b, H, N, init):
    """y is formed in fp32 and rounded once: it equals the rounded formula but where that lies next to a border
    between two values.  With every term off by 2^-20 (pieces of 22 bits, fp32 sums) and terms that add up to
    sqrt(N) of the output, an output is off by 2^-16.5 before its rounding; a share of that over a step (2^-7 at
    most) of the values falls on the other side, so the norm of the difference is below sqrt(2^-16.5 2^-7) = 2.9e-4."""
    from nested_ssm_b200 import gated_delta_chunk_scan
    d = _inputs(b, 100, H, 1, 48, N, seed=30)
    x = [d[n] for n in ("q", "k", "v", "g", "beta")]
    s0 = d["s0"] if init else None
    y = gated_delta_chunk_scan(*x, initial_states=s0)
    yr, _ = OD.gated_delta_scan(*x, S0=s0)
    assert _rel(y, yr.bfloat16()) <= 3e-4


@pytest.mark.parametrize("repeat", [1, 40])
def test_scan_bad_bounds_touch_no_other_sequence(repeat):
    """Sequences whose bounds descend lie between others that end and begin anywhere, 40 times over the tokens of
    the first ones too: those with good bounds of their own tokens are as ever."""
    from nested_ssm_b200 import gated_delta_chunk_scan
    step = 100
    d = _inputs(1, step * repeat, 2, 1, 32, 64, seed=31)
    x = [d[n] for n in ("q", "k", "v", "g", "beta")]
    cu, good = [], []
    for r in reversed(range(repeat)):         # the last tokens first: every second sequence descends
        good += [(len(cu), step * r + 50, step * r + 100), (len(cu) + 2, step * r, step * r + 30)]
        cu += [step * r + 50, step * r + 100, step * r, step * r + 30]
    # (30 of one group to 50 of the one before it descends too)
    n = len(cu) - 1
    out = torch.full((1, step * repeat, 2, 32), 3.0, dtype=torch.bfloat16, device="cuda")
    fin = torch.full((n, 2, 32, 64), 5.0, device="cuda")
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    gated_delta_chunk_scan(*x, cu_seqlens=torch.tensor(cu, dtype=torch.int32, device="cuda"), out=out, final_states=fin,
                           status=status)
    assert int(status) == 8
    names = {s for s, _, _ in good}
    for s, a, e in good:
        yr, Sr = OD.gated_delta_scan(*(t[:, a:e] for t in x))
        _check_y(out[:, a:e], yr, f"sequence {s}")
        _check_state(fin[s], Sr[0], f"sequence {s}")
    bad = [s for s in range(n) if s not in names]
    assert all(cu[s + 1] < cu[s] for s in bad) and bool((fin[bad] == 5.0).all())
    for r in range(repeat):
        assert bool((out[:, step * r + 30:step * r + 50] == 3.0).all())


def test_scan_overlapping_sequences_without_room_are_skipped():
    """More blocks than the tokens can have: the sequences that still fit are run, the others reported."""
    from nested_ssm_b200 import gated_delta_chunk_scan
    d = _inputs(1, 100, 2, 1, 32, 64, seed=32)
    x = [d[n] for n in ("q", "k", "v", "g", "beta")]
    cu = torch.tensor([0, 100] * 3, dtype=torch.int32, device="cuda")      # 3 x 4 blocks; 100 / 32 + 5 = 8 fit
    fin = torch.full((5, 2, 32, 64), 5.0, device="cuda")
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    y = gated_delta_chunk_scan(*x, cu_seqlens=cu, final_states=fin, status=status)
    yr, Sr = OD.gated_delta_scan(*x)
    _check_y(y, yr)
    _check_state(fin[0], Sr[0])
    _check_state(fin[2], Sr[0])
    assert int(status) == 8 and all(bool((fin[s] == 5.0).all()) for s in (1, 3, 4))


def test_scan_of_many_packed_sequences():
    """More sequences than a CTA ranks or has threads, empty ones among them."""
    from nested_ssm_b200 import gated_delta_chunk_scan
    lens = [(7 * i) % 37 if i % 5 else 0 for i in range(700)]
    d = _inputs(1, sum(lens) + 5, 2, 1, 16, 64, seed=33)
    x = [d[n] for n in ("q", "k", "v", "g", "beta")]
    at = [0]
    for n in lens:
        at.append(at[-1] + n)
    y, S = gated_delta_chunk_scan(*x, cu_seqlens=torch.tensor(at, dtype=torch.int32, device="cuda"), return_final_states=True)
    for s in list(range(0, 700, 41)) + [698, 699]:
        part = [t[:, at[s]:at[s + 1]] for t in x]
        if lens[s]:
            yr, Sr = OD.gated_delta_scan(*part)
            _check_y(y[:, at[s]:at[s + 1]], yr, f"sequence {s}")
            _check_state(S[s], Sr[0], f"sequence {s}")
        else:
            assert float(S[s].abs().max()) == 0.0


@_both_walks()
@pytest.mark.parametrize("size", [1.0, 1e3, 1e5, 1e9, 1e25])
@pytest.mark.parametrize("how", ["at once", "at the first token", "by degrees"])
def test_scan_forgets_a_large_state_without_writing(b, H, size, how):
    """A block of 32 tokens that writes nothing (beta 0) and forgets a large state: the outputs before it are the
    large state's, those behind it and the state start from zero."""
    from nested_ssm_b200 import gated_delta_chunk_scan
    d = _inputs(b, 130, H, 1, 32, 128, seed=26)
    d["s0"] *= size
    d["beta"][:, :64] = 0.0
    if how == "by degrees":
        d["g"][:, :32] = 0.0
        d["g"][:, 32:64] = -12.0          # e^-384: nothing of the largest state is left in fp32
    else:
        d["g"][:, :64] = 0.0
        d["g"][:, 32 if how == "at the first token" else 61] = float("-inf")
    d["v"][:, 64:70] = 0.0
    x = [d[n] for n in ("q", "k", "v", "g", "beta")]
    y, S = gated_delta_chunk_scan(*x, initial_states=d["s0"], return_final_states=True)
    yr, Sr = OD.gated_delta_scan(*x, S0=d["s0"])
    _check_y(y[:, :32], yr[:, :32], "before")
    if how == "at once":
        _check_y(y[:, 32:61], yr[:, 32:61], "in the block, before")
        assert float(y[:, 61:70].abs().max()) == 0.0
    _check_y(y[:, 70:], yr[:, 70:], "behind")
    _check_state(S, Sr)
    _, none = gated_delta_chunk_scan(*(t[:, :64] for t in x), initial_states=d["s0"], return_final_states=True)
    assert float(none.abs().max()) <= 1e-30


@_both_walks()
def test_scan_writes_then_forgets_in_one_block(b, H):
    """Large values written and forgotten within one block, a block without writes, then usual ones."""
    from nested_ssm_b200 import gated_delta_chunk_scan
    d = _inputs(b, 130, H, 1, 32, 64, seed=27)
    d["v"][:, :20] *= 1e5
    d["g"][:, 31] = float("-inf")
    d["beta"][:, 31:64] = 0.0
    x = [d[n] for n in ("q", "k", "v", "g", "beta")]
    y, S = gated_delta_chunk_scan(*x, return_final_states=True)
    yr, Sr = OD.gated_delta_scan(*x)
    _check_y(y[:, :31], yr[:, :31])
    assert float(y[:, 31:64].abs().max()) == 0.0
    _check_y(y[:, 64:], yr[:, 64:])
    _check_state(S, Sr)


@_both_walks()
@pytest.mark.parametrize("N", [64, 128])
@pytest.mark.parametrize("decay", [-5.0, -12.0, -20.0, -40.0])
def test_scan_reads_a_state_that_has_decayed_since_its_writes(b, H, N, decay):
    """Values of 1 written, then a decay of up to e^-40 in the same block: the next block reads the small state
    to the same relative precision, and erases along its keys (v = 0)."""
    from nested_ssm_b200 import gated_delta_chunk_scan
    d = _inputs(b, 96, H, 1, 48, N, seed=28)
    d["g"][:, 16] = decay
    d["beta"][:, 16:40] = 0.0
    d["v"][:, 16:] = 0.0
    x = [d[n] for n in ("q", "k", "v", "g", "beta")]
    y, S = gated_delta_chunk_scan(*x, return_final_states=True)
    yr, Sr = OD.gated_delta_scan(*x)
    _check_state(S, Sr)
    assert _rel(y[:, 32:64], yr[:, 32:64]) <= Y_TOL
    assert _rel(y[:, 64:], yr[:, 64:]) <= Y_TOL


@_both_walks()
@pytest.mark.parametrize("g,T", [(0.02, 200), (0.1, 100), (0.3, 40), (1.0, 33), (2.0, 40)])
def test_scan_takes_states_that_grow(b, H, g, T):
    """g above zero, with keys and queries that point the same way and use the whole of their type's range of a
    token (every element the same size): D (q.k) is far above the state's own scale."""
    from nested_ssm_b200 import gated_delta_chunk_scan
    d = _inputs(b, T, H, 1, 32, 128, seed=29)
    one = torch.where(d["k"][:, :1] < 0, -1.0, 1.0).expand_as(d["k"]) * (255 / 256) * 128 ** -0.5
    d["k"], d["q"] = one.bfloat16().contiguous(), one.bfloat16().contiguous()
    d["g"] = torch.full_like(d["g"], g)
    d["beta"] *= 0.1
    x = [d[n] for n in ("q", "k", "v", "g", "beta")]
    y, S = gated_delta_chunk_scan(*x, initial_states=d["s0"], return_final_states=True)
    yr, Sr = OD.gated_delta_scan(*x, S0=d["s0"])
    _check_state(S, Sr)
    assert bool(torch.isfinite(y).all()) and _rel(y, yr) <= Y_TOL
    for t in range(0, T, 16):             # and of every stretch of tokens by itself
        assert _rel(y[:, t:t + 16], yr[:, t:t + 16]) <= Y_TOL, t


def test_step_reports_slots_beyond_32_bits():
    from nested_ssm_b200 import gated_delta_state_update
    x, state, _ = _step_case(3, 9, 2, 2, 32, 64, torch.float32, seed=34)
    slots = torch.tensor([3, (1 << 32) + 5, -(1 << 32)], device="cuda")
    out = torch.zeros(3, 2, 32, device="cuda")
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    ref = _step_ref(x, state, slots, 64 ** -0.5, out, [0])
    gated_delta_state_update(state, x["q"], x["k"], x["v"], x["g"], x["beta"], None, slots, out=out, status=status)
    _check_step(state, out, ref)
    assert int(status) == 1


@_both_walks()
@pytest.mark.parametrize("size", [1e11, 1e18])
@pytest.mark.parametrize("decay", [-50.0, -100.0, -160.0])
def test_scan_erases_and_forgets_a_large_state_in_one_block(b, H, size, decay):
    """A block whose first u are those of a state far above the values (it erases along its keys) and decay to
    nothing within it, and whose last tokens write little or nothing."""
    from nested_ssm_b200 import gated_delta_chunk_scan
    d = _inputs(b, 100, H, 1, 32, 64, seed=35)
    d["s0"] *= size
    d["g"][:, 20] = decay
    d["beta"][:, 20:40] = 0.0
    x = [d[n] for n in ("q", "k", "v", "g", "beta")]
    y, S = gated_delta_chunk_scan(*x, initial_states=d["s0"], return_final_states=True)
    yr, Sr = OD.gated_delta_scan(*x, S0=d["s0"])
    _check_y(y[:, :20], yr[:, :20], "before")
    _check_y(y[:, 40:], yr[:, 40:], "behind")
    _check_state(S, Sr)
