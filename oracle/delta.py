"""64-bit restatements of the gated delta rule, the slot moves and the beam selection (test-only)."""
from __future__ import annotations

import torch


def gated_delta_token(S, q, k, v, g, beta, scale):
    """One token in fp64: S [.., P, N], q / k [.., N], v [.., P], g / beta [..]; (S', y)."""
    S = torch.exp(g)[..., None, None] * S
    u = beta[..., None] * (v - (S * k[..., None, :]).sum(-1))
    S = S + u[..., None] * k[..., None, :]
    return S, scale * (S * q[..., None, :]).sum(-1)


def gated_delta_scan(q, k, v, g, beta, scale=None, S0=None):
    """Token by token: q / k [b, T, G, N], v [b, T, H, P], g / beta [b, T, H] of any dtype and
    device; (y [b, T, H, P], S [b, H, P, N]) in fp64."""
    b, T, G, N = q.shape
    H, P = v.shape[2:]
    scale = N ** -0.5 if scale is None else scale
    q, k = (x.double().repeat_interleave(H // G, 2) for x in (q, k))
    v, g, beta = v.double(), g.double(), beta.double()
    S = torch.zeros(b, H, P, N, dtype=torch.float64, device=v.device) if S0 is None else S0.double().clone()
    y = torch.empty(b, T, H, P, dtype=torch.float64, device=v.device)
    for t in range(T):
        S, y[:, t] = gated_delta_token(S, q[:, t], k[:, t], v[:, t], g[:, t], beta[:, t], scale)
    return y, S


def reorder_plan(slots, parents, group, pad):
    """(new slots, [(src, dst)]) of lists: the first child keeps its parent's slot, the others take the
    slots of rows without children, in row order."""
    n = len(slots)
    parent = [r // group * group + parents[r] for r in range(n)]
    live = [slots[parent[r]] != pad for r in range(n)]
    free = [slots[r] for r in range(n) if slots[r] != pad and not any(live[c] and parent[c] == r for c in range(n))]
    seen, new, moves = set(), [], []
    for r in range(n):
        s = slots[parent[r]]
        if live[r] and parent[r] in seen:
            s = free.pop(0) if free else pad
            if s != pad:
                moves.append((slots[parent[r]], s))
        seen.add(parent[r])
        new.append(s if live[r] else pad)
    return new, moves


def compact_plan(slots, pad):
    """(new slots, [(src, dst)]): the m live slots into [0, m)."""
    m = sum(s != pad for s in slots)
    holes = [i for i in range(m) if i not in slots]
    new, moves = [], []
    for s in slots:
        if s != pad and s >= m:
            moves.append((s, holes[0]))
            s = holes.pop(0)
        new.append(s)
    return new, moves


def beam_select(logits, scores, n, finished=None, eos=None):
    """(scores fp64, parents, tokens) of the n best continuations per prompt, by a full sort: total
    descending, then beam, then logit descending, then token."""
    b, K, V = logits.shape
    x = logits.double().cpu()
    x = torch.where(torch.isfinite(x), x, torch.tensor(float("-inf"), dtype=torch.float64))
    out = [[], [], []]
    for i in range(b):
        cands = []
        for k in range(K):
            row = x[i, k]
            if finished is not None and bool(finished[i, k]):
                row = torch.full((V,), float("-inf"), dtype=torch.float64)
                row[eos] = 0.0
            total = (float(scores[i, k]) + row) - torch.logsumexp(row, 0)
            total = torch.where(torch.isnan(total), torch.tensor(float("-inf"), dtype=torch.float64), total)
            order = torch.sort(row, descending=True, stable=True).indices[:n]
            cands += [(-float(total[t]), k, r, int(t)) for r, t in enumerate(order.tolist())]
        cands.sort()
        out[0].append([-c[0] for c in cands[:n]])
        out[1].append([c[1] for c in cands[:n]])
        out[2].append([c[3] for c in cands[:n]])
    return torch.tensor(out[0], dtype=torch.float64), torch.tensor(out[1]), torch.tensor(out[2])
