"""Measured cases of the recurrent-state operators: the gated delta rule (chunked over prompts, recurrent
over decode tokens), the moves of slots that hold recurrent states (fork, compact, reorder), and beam
search's selection.

``run`` computes an operator either with the framework's kernels (``own``) or in its plain form,
elementary torch operations in fp32 (fp64 where the order of near values decides).  ``exact`` computes
the same outputs in fp64 from the definition.
"""
import math
import random

import torch

own = False

DEV = "cuda"
DT = {"bf16": torch.bfloat16, "fp32": torch.float32}
CHUNK = 64        # tokens per chunk of the plain chunked form
PAD = -1          # slot of a padded row


# ---------------------------------------------------------------- cases
def listed():
    return [
        # one short prompt (an odd length, small heads): what a request costs when latency counts
        _chunk("chunk_short", 1, 77, 8, 2, 64, 64),
        # a packed batch of ragged prompts with states carried in and out, as a server prefills
        _chunk("chunk_packed", 24, 700, 32, 16, 128, 128, ragged=7, init=True),
        # the prefill of two long prompts
        _chunk("chunk_long", 2, 8192, 32, 16, 128, 128),
        # a prompt batch in the head layout of the repository's decode benchmark (128 heads of 80, 8 groups)
        _chunk("chunk_wide", 8, 2048, 128, 8, 80, 128, init=True),
        # one sequence decoding: latency
        _step("step_one", 1, 4, 32, 16, 128, 128, "bf16"),
        # a small fp32 batch with padded rows
        _step("step_padded_fp32", 57, 64, 24, 8, 64, 64, "fp32", pads=5),
        # the decode benchmark's batch and head layout
        _step("step_batch", 448, 512, 128, 8, 80, 128, "bf16"),
        # beams of a few prompts reordered after each token
        _slots("reorder_small", "reorder", 4, 4, 24, 2, 16, 64, 128),
        # the same for a full batch of beams: three layers of state
        _slots("reorder_batch", "reorder", 64, 8, 640, 3, 16, 80, 128),
        # live slots gathered to the front of the pool after many sequences ended
        _slots("compact", "compact", 300, 1, 896, 2, 24, 64, 128),
        # beam selection for one prompt
        _beam("beam_one", 1, 4, 4, 32001, "fp32"),
        # beam selection for a batch over a large vocabulary, twice as many candidates as beams,
        # some beams finished
        _beam("beam_batch", 64, 8, 16, 131072, "bf16", eos=2),
    ]


def _chunk(name, b, T, H, G, P, N, ragged=0, init=False):
    return {"name": name, "op": "chunk", "b": b, "T": T, "H": H, "G": G, "P": P, "N": N, "ragged": ragged, "init": init}


def _step(name, b, S, H, G, P, N, dtype, pads=0):
    return {"name": name, "op": "step", "b": b, "S": S, "H": H, "G": G, "P": P, "N": N, "dtype": dtype, "pads": pads}


def _slots(name, kind, b, K, S, L, H, P, N):
    return {"name": name, "op": "slots", "kind": kind, "b": b, "K": K, "S": S, "L": L, "H": H, "P": P, "N": N}


def _beam(name, b, K, n, V, dtype, eos=-1):
    return {"name": name, "op": "beam", "b": b, "K": K, "n": n, "V": V, "dtype": dtype, "eos": eos}


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["chunk", "step", "slots", "beam"])
    G = rng.choice([1, 2, 4, 8])
    H = G * rng.choice([1, 2, 4])
    N = rng.choice([64, 128])
    P = 16 * rng.randint(1, 8)
    if op == "chunk":
        T = _log(rng, 1, 6000)
        b = max(1, min(_log(rng, 1, 24), 60000 // T, 400000 // (T * H)))
        c = _chunk("", b, T, H, G, P, N, ragged=rng.randint(1, 10 ** 6) if rng.random() < 0.5 else 0, init=rng.random() < 0.5)
    elif op == "step":
        b = _log(rng, 1, 400)
        c = _step("", b, b + rng.randint(0, 40), H, G, P, N, rng.choice(["bf16", "fp32"]), pads=rng.randint(0, b // 8))
    elif op == "slots":
        kind = rng.choice(["reorder", "compact", "fork"])
        K = rng.randint(2, 12) if kind != "compact" else 1
        b = max(1, _log(rng, 1, 500) // K)
        c = _slots("", kind, b, K, b * K + rng.randint(b, 60 + b), rng.randint(1, 3), H, P, N)
    else:
        K = rng.randint(1, 12)
        V = _log(rng, 50, 140000)
        n = rng.randint(1, min(2 * K, K * V))
        c = _beam("", max(1, min(_log(rng, 1, 64), 30000000 // (K * V))), K, n, V, rng.choice(["bf16", "fp32"]),
                  eos=rng.randint(0, V - 1) if rng.random() < 0.5 else -1)
    del c["name"]
    return c


def _lengths(c):
    """Prompt lengths of a chunk case: all T, or ragged around T with one prompt of one token."""
    if not c["ragged"]:
        return [c["T"]] * c["b"]
    r = random.Random(c["ragged"])
    return [1 if i == 1 else max(1, int(c["T"] * r.uniform(0.05, 1.0))) for i in range(c["b"])]


def _moved(c):
    """How many slots a slots case moves, as far as the case says (a reorder: an expectation)."""
    n = c["b"] * c["K"]
    if c["kind"] == "fork":
        return c["b"] * (c["K"] - 1)
    if c["kind"] == "compact":
        return n * (c["S"] - n) / c["S"]
    return n * (1 - 1 / c["K"]) ** c["K"]


def work(c):
    if c["op"] == "chunk":
        tok = sum(_lengths(c))
        io = tok * (2 * 2 * c["G"] * c["N"] + 2 * 2 * c["H"] * c["P"] + 8 * c["H"])
        st = c["b"] * c["H"] * c["P"] * c["N"] * 4
        return {"bytes": io + st * (2 if c["init"] else 1), "flops": 6 * tok * c["H"] * c["P"] * c["N"]}
    if c["op"] == "step":
        live = c["b"] - c["pads"]
        es = 2 if c["dtype"] == "bf16" else 4
        st = live * c["H"] * c["P"] * c["N"]
        return {"bytes": 8 * st + live * (es * (2 * c["G"] * c["N"] + 2 * c["H"] * c["P"]) + 8 * c["H"]), "flops": 6 * st}
    if c["op"] == "slots":
        row = c["L"] * (c["H"] * c["P"] * c["N"] * 4 + c["H"] * c["P"] * 3 * 2)
        return {"bytes": 2 * row * _moved(c) + 12 * c["b"] * c["K"], "flops": 0}
    es = 2 if c["dtype"] == "bf16" else 4
    return {"bytes": c["b"] * (c["K"] * c["V"] * es + c["K"] * 5 + c["n"] * 13), "flops": 3 * c["b"] * c["K"] * c["V"]}


# ---------------------------------------------------------------- inputs
def prepare(c, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)

    def randn(*shape):
        return torch.randn(*shape, generator=g, device=DEV)

    def rand(*shape):
        return torch.rand(*shape, generator=g, device=DEV)

    def unit(t):
        return t / t.norm(dim=-1, keepdim=True)

    def decay(*shape):   # log decay -A softplus(. + bias), A = e^U(0, log 16), as Mamba2 layers initialise it
        H = shape[-1]
        A = torch.exp(rand(H) * math.log(16.0))
        bias = torch.log(torch.expm1(0.001 + 0.099 * rand(H)))
        return -A * torch.nn.functional.softplus(randn(*shape) + bias)

    s = {"case": c}
    if c["op"] == "chunk":
        lens = _lengths(c)
        if c["ragged"]:
            rows = sum(lens) + 3    # three rows behind the last sequence
            b, T = 1, rows
            s["cu"] = torch.tensor([0] + torch.tensor(lens).cumsum(0).tolist(), dtype=torch.int32, device=DEV)
        else:
            b, T = c["b"], c["T"]
            s["cu"] = None
        s["maxlen"] = max(lens)
        H, G, P, N = c["H"], c["G"], c["P"], c["N"]
        s["q"] = unit(randn(b, T, G, N)).bfloat16()
        s["k"] = unit(randn(b, T, G, N)).bfloat16()
        s["v"] = randn(b, T, H, P).bfloat16()
        s["g"] = decay(b, T, H)
        s["beta"] = torch.sigmoid(randn(b, T, H))
        s["init"] = 0.3 * randn(c["b"], H, P, N) if c["init"] else None
        s["out"] = torch.zeros(b, T, H, P, dtype=torch.bfloat16, device=DEV)
    elif c["op"] == "step":
        b, H, G, P, N = c["b"], c["H"], c["G"], c["P"], c["N"]
        dt = DT[c["dtype"]]
        s["state"] = randn(c["S"], H, P, N)
        slots = torch.randperm(c["S"], generator=g, device=DEV)[:b].to(torch.int32)
        if c["pads"]:
            at = torch.randperm(b, generator=g, device=DEV)
            slots[at[:c["pads"]]] = PAD
            s["live"] = at[c["pads"]:].sort().values
        else:
            s["live"] = torch.arange(b, device=DEV)
        s["slots"] = slots
        s["q"], s["k"] = unit(randn(b, G, N)).to(dt), unit(randn(b, G, N)).to(dt)
        s["v"] = randn(b, H, P).to(dt)
        s["g"], s["beta"] = decay(b, H), torch.sigmoid(randn(b, H))
        s["out"] = torch.zeros(b, H, P, dtype=dt, device=DEV)
    elif c["op"] == "slots":
        n, S = c["b"] * c["K"], c["S"]
        s["bufs"] = [randn(c["L"], S, c["H"], c["P"], c["N"]), randn(c["L"], S, c["H"] * c["P"], 3).bfloat16()]
        perm = torch.randperm(S, generator=g, device=DEV).to(torch.int32)
        if c["kind"] == "fork":    # each prompt's slot copied to its other beams
            s["src"] = perm[:c["b"]].repeat_interleave(c["K"] - 1)
            s["dst"] = perm[c["b"]:c["b"] * c["K"]].contiguous()
        else:
            s["slots"] = perm[:n].reshape(c["b"], c["K"]).contiguous()
            s["parents"] = torch.randint(0, c["K"], (c["b"], c["K"]), generator=g, device=DEV, dtype=torch.int32)
        s["handle"] = {}
    else:
        b, K, V = c["b"], c["K"], c["V"]
        s["logits"] = (3.0 * randn(b, K, V)).to(DT[c["dtype"]])
        s["logits"].masked_fill_(rand(b, K, V) < 0.1, float("-inf"))     # a tenth of the vocabulary banned
        s["scores"] = -20.0 * rand(b, K)
        s["finished"] = (rand(b, K) < 0.2) if c["eos"] >= 0 else None
    return s


# ---------------------------------------------------------------- one pass
def run(s):
    op = s["case"]["op"]
    if own:
        return {"chunk": _own_chunk, "step": _own_step, "slots": _own_slots, "beam": _own_beam}[op](s)
    return {"chunk": _plain_chunk, "step": _plain_step, "slots": _plain_slots, "beam": _plain_beam}[op](s)


def _own_chunk(s):
    from nested_ssm_b200 import gated_delta_chunk_scan
    return gated_delta_chunk_scan(s["q"], s["k"], s["v"], s["g"], s["beta"], initial_states=s["init"],
                                  cu_seqlens=s["cu"], return_final_states=True, out=s["out"])


def _own_step(s):
    from nested_ssm_b200 import gated_delta_state_update
    y = gated_delta_state_update(s["state"], s["q"], s["k"], s["v"], s["g"], s["beta"],
                                 state_batch_indices=s["slots"], pad_slot_id=PAD, out=s["out"])
    return y, s["state"]


def _own_slots(s):
    from nested_ssm_b200 import StateBuffers, compact_slots, copy_slots, reorder_slots
    if "own" not in s["handle"]:      # a program builds the handle of its states once
        s["handle"]["own"] = StateBuffers(s["bufs"], slot_dim=1)
    h = s["handle"]["own"]
    kind = s["case"]["kind"]
    if kind == "fork":
        copy_slots(h, s["src"], s["dst"])
        return s["bufs"]
    if kind == "compact":
        return compact_slots(h, s["slots"].reshape(-1)), s["bufs"]
    return reorder_slots(h, s["slots"], s["parents"]), s["bufs"]


def _own_beam(s):
    from nested_ssm_b200 import beam_select
    c = s["case"]
    if c["eos"] < 0:
        return beam_select(s["logits"], s["scores"], num_out=c["n"])
    return beam_select(s["logits"], s["scores"], num_out=c["n"], finished=s["finished"], eos_token_id=c["eos"])


# ---------------------------------------------------------------- plain forms
def _padded(s, dtype):
    """q, k, v, g, beta of a chunk case as [b, H, T', .] with heads expanded; padded tokens have
    beta = g = k = 0, which leaves the state as it is.  T' is a multiple of CHUNK."""
    c = s["case"]
    Tp = -(-s["maxlen"] // CHUNK) * CHUNK
    t = torch.arange(Tp, device=DEV)
    if s["cu"] is None:
        start = torch.zeros(1, dtype=torch.long, device=DEV)
        length = torch.full((1,), c["T"], device=DEV)
        take = lambda x: x[:, t.clamp(max=c["T"] - 1)]  # noqa: E731
    else:
        start, length = s["cu"][:-1].long(), (s["cu"][1:] - s["cu"][:-1]).long()
        at = (start[:, None] + t).clamp(max=s["q"].shape[1] - 1)
        take = lambda x: x[0][at]  # noqa: E731
    valid = t < length[:, None]
    rep = c["H"] // c["G"]
    q, k, v, g, beta = (take(s[n]).to(dtype).transpose(1, 2) for n in ("q", "k", "v", "g", "beta"))
    m = valid[:, None]
    q, k = (x.repeat_interleave(rep, 1) * m[..., None] for x in (q, k))
    return q, k, v * m[..., None], g * m, beta * m, start, valid


def _unpadded(s, o, start, valid):
    """o [b, H, T', P] rounded into the out buffer's rows of each sequence."""
    c = s["case"]
    o = o.transpose(1, 2).to(torch.bfloat16)
    if s["cu"] is None:
        s["out"].copy_(o[:, :c["T"]])
        return s["out"]
    rows = s["out"].shape[1]
    t = torch.arange(valid.shape[1], device=DEV)
    at = torch.where(valid, start[:, None] + t, rows)         # padded tokens go to a row of their own
    buf = torch.cat([s["out"][0], s["out"].new_zeros(1, c["H"], c["P"])])
    buf[at.reshape(-1)] = o.reshape(-1, c["H"], c["P"])
    s["out"][0].copy_(buf[:rows])
    return s["out"]


def _plain_chunk(s):
    c = s["case"]
    q, k, v, g, beta, start, valid = _padded(s, torch.float32)
    b, H, Tp, P = v.shape
    N, C = c["N"], CHUNK
    q, k, v = (x.reshape(b, H, -1, C, x.shape[-1]) for x in (q, k, v))
    beta = beta.reshape(b, H, -1, C)
    G = g.double().reshape(b, H, -1, C).cumsum(-1)
    lower = torch.ones(C, C, dtype=torch.bool, device=DEV).tril()
    decay = torch.where(lower, torch.exp((G[..., :, None] - G[..., None, :]).float()), 0.0)
    A = (k @ k.transpose(-1, -2)) * decay * beta[..., None]
    A = torch.where(lower & ~lower.t(), A, 0.0)
    T = torch.zeros_like(A)
    for i in range(C):       # (I + A) T = I by forward substitution
        T[..., i, :] = -(A[..., i, None, :i] @ T[..., :i, :]).squeeze(-2)
        T[..., i, i] += 1.0
    M = torch.where(lower, (q @ k.transpose(-1, -2)) * decay, 0.0)
    eG, eT = torch.exp(G.float()), torch.exp((G[..., -1:] - G).float())
    u0, w = T @ (v * beta[..., None]), T @ (k * (beta * eG)[..., None])
    qe, ke = q * eG[..., None], k * eT[..., None]
    S = s["init"].float() if s["init"] is not None else torch.zeros(b, H, P, N, device=DEV)
    o = torch.empty_like(v)
    for i in range(v.shape[2]):     # the state from chunk to chunk
        u = u0[:, :, i] - w[:, :, i] @ S.transpose(-1, -2)
        o[:, :, i] = qe[:, :, i] @ S.transpose(-1, -2) + M[:, :, i] @ u
        S = eG[:, :, i, -1, None, None] * S + u.transpose(-1, -2) @ ke[:, :, i]
    o = o.reshape(b, H, Tp, P) * N ** -0.5
    return _unpadded(s, o, start, valid), S


def _plain_step(s):
    c = s["case"]
    rep = c["H"] // c["G"]
    live = s["live"]
    at = s["slots"][live].long()
    q, k = (s[n][live].float().repeat_interleave(rep, 1) for n in ("q", "k"))
    v, g, beta = (s[n][live].float() for n in ("v", "g", "beta"))
    S = s["state"][at] * torch.exp(g)[..., None, None]
    u = beta[..., None] * (v - (S @ k[..., None]).squeeze(-1))
    S = S + u[..., None] * k[..., None, :]
    s["state"][at] = S
    s["out"][live] = ((S @ q[..., None]).squeeze(-1) * c["N"] ** -0.5).to(s["out"].dtype)
    return s["out"], s["state"]


def _plain_slots(s):
    c = s["case"]
    if c["kind"] == "fork":
        src, dst = s["src"].long(), s["dst"].long()
        new = None
    elif c["kind"] == "compact":
        src = s["slots"].reshape(-1).long()
        n = src.numel()
        used = torch.zeros(c["S"], dtype=torch.bool, device=DEV)
        used[src] = True
        holes = torch.sort(used[:n].to(torch.int8), stable=True).indices      # free slots below n, ascending
        move = src >= n
        dst = torch.where(move, holes[(move.cumsum(0) - 1).clamp(min=0)], src)
        new = dst.to(torch.int32)
    else:
        K = c["K"]
        slots, parents = s["slots"].long(), s["parents"].long()
        same = parents[:, :, None] == parents[:, None, :]
        first = ~(same & torch.ones(K, K, dtype=torch.bool, device=DEV).tril(-1)).any(-1)
        children = (parents[:, :, None] == torch.arange(K, device=DEV)).any(1)
        free = torch.sort(children.to(torch.int8), dim=1, stable=True).indices  # beams without a child, ascending
        extra = ((~first).cumsum(1) - 1).clamp(min=0)
        src = slots.gather(1, parents)
        dst = torch.where(first, src, slots.gather(1, free.gather(1, extra)))
        new = dst.to(torch.int32)
        src, dst = src.reshape(-1), dst.reshape(-1)
    for buf in s["bufs"]:
        buf[:, dst] = buf[:, src]
    return s["bufs"] if new is None else (new, s["bufs"])


def _rank_key(x):
    """int64 keys whose descending order is x [.., V] (fp32) descending, then the index ascending."""
    V = x.shape[-1]
    bits = (x + 0.0).view(torch.int32).long()
    order = torch.where(bits < 0, -(bits & 0x7FFFFFFF), bits)
    return order * (1 << 31) + torch.arange(V - 1, -1, -1, device=x.device)


def _plain_beam(s):
    c = s["case"]
    b, K, V, n = c["b"], c["K"], c["V"], c["n"]
    x = s["logits"].float()
    x = torch.where(torch.isfinite(x), x, float("-inf"))
    score = s["scores"].double()
    if c["eos"] >= 0:
        only = torch.where(torch.arange(V, device=DEV) == c["eos"], 0.0, float("-inf"))
        x = torch.where(s["finished"][..., None], only, x)
    top = x.amax(-1, keepdim=True)
    top = torch.where(torch.isfinite(top), top, 0.0)
    lse = torch.log(torch.exp(x - top).sum(-1, dtype=torch.float64)) + top.squeeze(-1)
    best = _rank_key(x).topk(min(n, V), dim=-1).values
    token = V - 1 - (best & ((1 << 31) - 1))
    total = score[..., None] + x.gather(-1, token).double() - lse[..., None]
    total = torch.where(torch.isnan(total), float("-inf"), total)
    total, at = torch.sort(total.reshape(b, -1), dim=1, descending=True, stable=True)
    at = at[:, :n]
    parent = at // min(n, V)
    token = token.reshape(b, -1).gather(1, at)
    out = total[:, :n].float(), parent.to(torch.int32), token.to(torch.int32)
    if c["eos"] < 0:
        return out
    return out + ((token == c["eos"]) | s["finished"].gather(1, parent),)


# ---------------------------------------------------------------- 64 bits
def exact(c, seed):
    """The definitions in fp64: the delta rule token by token, the log softmax over the vocabulary.
    Moved slots are copies and have no such value."""
    if c["op"] == "slots":
        return None
    s = prepare(c, seed)
    if c["op"] == "chunk":
        q, k, v, g, beta, start, valid = _padded(s, torch.float64)
        S = s["init"].double() if s["init"] is not None else torch.zeros(c["b"], c["H"], c["P"], c["N"], dtype=torch.float64, device=DEV)
        o = torch.zeros_like(v)
        for t in range(s["maxlen"]):
            S, o[:, :, t] = _token(S, q[:, :, t], k[:, :, t], v[:, :, t], g[:, :, t], beta[:, :, t])
        if s["cu"] is None:
            return o.transpose(1, 2)[:, :c["T"]], S
        out = torch.zeros(s["out"].shape, dtype=torch.float64, device=DEV)
        for i, (at, length) in enumerate(zip(start.tolist(), _lengths(c))):
            out[0, at:at + length] = o[i].transpose(0, 1)[:length]
        return out, S
    if c["op"] == "step":
        state, out = s["state"].double(), torch.zeros(s["out"].shape, dtype=torch.float64, device=DEV)
        rep = c["H"] // c["G"]
        for row, slot in enumerate(s["slots"].tolist()):
            if slot == PAD:
                continue
            q, k = (s[n][row].double().repeat_interleave(rep, 0) for n in ("q", "k"))
            state[slot], out[row] = _token(state[slot], q, k, *(s[n][row].double() for n in ("v", "g", "beta")))
        return out, state
    scores = []
    for i in range(c["b"]):
        x = s["logits"][i].double()
        lp = x - x.logsumexp(-1, keepdim=True)
        if c["eos"] >= 0:
            lp[s["finished"][i]] = float("-inf")
            lp[s["finished"][i], c["eos"]] = 0.0
        total = torch.nan_to_num(s["scores"][i].double()[:, None] + lp, nan=float("-inf"), neginf=float("-inf"))
        scores.append(total.reshape(-1).topk(c["n"]).values)
    return (torch.stack(scores), None, None) + ((None,) if c["eos"] >= 0 else ())


def _token(S, q, k, v, g, beta):
    """One token of the gated delta rule on S [.., P, N] in fp64: the new state and the output."""
    S = torch.exp(g)[..., None, None] * S
    u = beta[..., None] * (v - torch.einsum("...pn,...n->...p", S, k))
    S = S + torch.einsum("...p,...n->...pn", u, k)
    return S, torch.einsum("...pn,...n->...p", S, q) * q.shape[-1] ** -0.5
