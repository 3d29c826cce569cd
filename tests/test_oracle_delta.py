"""The 64-bit restatements behind the tests of the gated delta rule, slot moves and beam selection, checked
against other forms of the same definitions (CPU)."""
import torch

import oracle.delta as OD


def test_token_by_token_equals_the_chunked_form():
    """u of a chunk solves (I + A) u = r; the state after it and y follow (see the formulas in
    csrc/nssm_delta_chunk.cuh)."""
    g = torch.Generator().manual_seed(0)
    b, T, H, G, P, N = 2, 21, 4, 2, 5, 8
    r = lambda *s: torch.randn(*s, generator=g, dtype=torch.float64)  # noqa: E731
    q, k, v, S0 = r(b, T, G, N), r(b, T, G, N) / N ** 0.5, r(b, T, H, P), r(b, H, P, N)
    gg, beta = -torch.rand(b, T, H, generator=g, dtype=torch.float64), torch.sigmoid(r(b, T, H))
    y, S = OD.gated_delta_scan(q, k, v, gg, beta, 0.7, S0)
    qh, kh = (x.repeat_interleave(H // G, 2).transpose(1, 2) for x in (q, k))
    vh, gh, bh = v.transpose(1, 2), gg.transpose(1, 2), beta.transpose(1, 2)
    Gc = gh.cumsum(-1)
    D = torch.exp(Gc[..., :, None] - Gc[..., None, :]).tril()
    A = (bh[..., None] * D * (kh @ kh.transpose(-1, -2))).tril(-1)
    e = torch.exp(Gc)[..., None]
    u = torch.linalg.solve(torch.eye(T, dtype=torch.float64) + A, bh[..., None] * (vh - e * (kh @ S0.transpose(-1, -2))))
    y2 = 0.7 * (e * (qh @ S0.transpose(-1, -2)) + (D * (qh @ kh.transpose(-1, -2))) @ u)
    S2 = e[..., -1:, :] * S0 + (torch.exp(Gc[..., -1:] - Gc)[..., None] * u).transpose(-1, -2) @ kh
    torch.testing.assert_close(y, y2.transpose(1, 2), rtol=1e-10, atol=1e-10)
    torch.testing.assert_close(S, S2, rtol=1e-10, atol=1e-10)


def test_beam_select_equals_a_sort_of_everything():
    g = torch.Generator().manual_seed(1)
    x, s = torch.randn(3, 4, 30, generator=g), torch.randn(3, 4, generator=g)
    sc, p, t = OD.beam_select(x, s, 7)
    total = s.double()[..., None] + torch.log_softmax(x.double(), -1)
    want, at = total.reshape(3, -1).topk(7)
    torch.testing.assert_close(sc, want)
    assert torch.equal(p, at // 30) and torch.equal(t, at % 30)


def test_plans_move_as_little_as_possible_and_never_what_is_read():
    g = torch.Generator().manual_seed(2)
    for seed in range(20):
        slots = torch.randperm(40, generator=g)[:12].tolist()
        parents = torch.randint(0, 4, (12,), generator=g).tolist()
        new, moves = OD.reorder_plan(slots, parents, 4, -1)
        assert sorted(new) == sorted(slots) and not {s for s, _ in moves} & {d for _, d in moves}
        kids = sum(len({parents[r] for r in range(i, i + 4)}) for i in (0, 4, 8))
        assert len(moves) == 12 - kids
        new, moves = OD.compact_plan(slots, -1)
        assert sorted(new) == list(range(12)) and len(moves) == sum(s >= 12 for s in slots)
