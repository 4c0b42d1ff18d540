"""Workloads of the operators around a softmax over index rows.

Three operators, each in its elementary form and, with ``own`` set, as a call
of the framework:

  logprobs           log probability of a given row per query under
                     softmax(scale * q . x) over all (allowed) rows, with the
                     log-sum-exp, the entropy and the top alternatives
  logprobs_backward  its gradient with respect to the queries and the rows
  adamw              an AdamW step over many tensors, states in f32 or 8 bits
"""
import math

import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
BLOCK = 256  # elements that share a scale in the 8-bit optimizer states


def listed():
    return [
        # one user's query against a small index: latency is everything
        {"name": "logprobs one query", "op": "logprobs", "dtype": "f32", "nq": 1, "n": 10_000,
         "dim": 128, "k": 10, "mask": "none", "pad": 0},
        # a few concurrent queries, rows of an encoder of 768 dimensions: one pass over the rows
        {"name": "logprobs few queries", "op": "logprobs", "dtype": "bf16", "nq": 8, "n": 100_003,
         "dim": 768, "k": 5, "mask": "none", "pad": 0},
        # a batch of filtered queries, each with a filter of its own, some filters empty
        {"name": "logprobs filtered", "op": "logprobs", "dtype": "f32", "nq": 1_000, "n": 10_000,
         "dim": 128, "k": 10, "mask": "each", "pad": 0},
        # scoring a training batch over a large table
        {"name": "logprobs batch", "op": "logprobs", "dtype": "bf16", "nq": 2_048, "n": 131_072,
         "dim": 768, "k": 20, "mask": "none", "pad": 0},
        # offline evaluation over an embedding-scale index, 96 dimensions
        {"name": "logprobs large", "op": "logprobs", "dtype": "f32", "nq": 4_096, "n": 262_144,
         "dim": 96, "k": 10, "mask": "one", "pad": 0},
        # a small fine-tuning batch over a small table
        {"name": "backward small", "op": "logprobs_backward", "dtype": "f32", "nq": 100,
         "n": 10_000, "dim": 128, "mask": "none", "pad": 0},
        # odd sizes, filters of their own, rows that are a part of wider ones
        {"name": "backward filtered", "op": "logprobs_backward", "dtype": "f32", "nq": 777,
         "n": 20_003, "dim": 96, "mask": "each", "pad": 5},
        # an ordinary batch in 16 bits, odd number of rows
        {"name": "backward batch", "op": "logprobs_backward", "dtype": "bf16", "nq": 1_000,
         "n": 50_001, "dim": 768, "mask": "none", "pad": 0},
        # a large batch over a large table
        {"name": "backward large", "op": "logprobs_backward", "dtype": "bf16", "nq": 4_096,
         "n": 131_072, "dim": 768, "mask": "none", "pad": 0},
        # a query-side adapter: a matrix and its bias
        {"name": "adamw adapter", "op": "adamw", "dtype": "f32", "state": 32, "tensors": 2,
         "total": 16_512},
        # an encoder's tensors, large and odd small ones, 8-bit states
        {"name": "adamw 8-bit", "op": "adamw", "dtype": "bf16", "state": 8, "tensors": 40,
         "total": 40_000_000},
        # the rows of a large table
        {"name": "adamw table", "op": "adamw", "dtype": "f32", "state": 32, "tensors": 1,
         "total": 131_072 * 768},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["logprobs", "logprobs", "logprobs_backward", "logprobs_backward", "adamw"])
    if op == "adamw":
        return {"op": op, "dtype": rng.choice(["f32", "bf16"]), "state": rng.choice([8, 32]),
                "tensors": _log(rng, 1, 60), "total": _log(rng, 20_000, 60_000_000)}
    while True:
        c = {"op": op, "dtype": rng.choice(["f32", "bf16", "f16"]), "nq": _log(rng, 1, 4_096),
             "n": _log(rng, 500, 262_144), "dim": _log(rng, 16, 1_024),
             "mask": rng.choice(["none", "none", "one", "each"]), "pad": rng.choice([0, 0, 8, 3])}
        # no dearer than the largest listed case, in products and in scores held at once
        if c["nq"] * c["n"] * c["dim"] > 2_048 * 131_072 * 768 // (3 if c["dtype"] == "f32" else 1):
            continue
        if c["nq"] * c["n"] > 500_000_000:
            continue
        if op == "logprobs":
            c["k"] = rng.choice([0, 1, 5, 10, 20, 50])
        return c


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
def _sizes(case):
    """Elements of each tensor: the first takes most, the others fall off, none a round number."""
    t, total = case["tensors"], case["total"]
    if t == 1:
        return [total]
    w = [1.0 / (i + 1) ** 1.5 for i in range(t)]
    s = [max(1, int(total * x / sum(w))) for x in w]
    return s[:-1] + [max(1, total - sum(s[:-1]))]


def _scores_inputs(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    nq, n, d = case["nq"], case["n"], case["dim"]
    dt = DTYPES[case["dtype"]]
    wide_x = torch.randn(n, d + case["pad"], device="cuda", generator=gen)
    targets = torch.randint(0, n, (nq,), device="cuda", generator=gen)
    wide_q = torch.randn(nq, d + case["pad"], device="cuda", generator=gen)
    # a query lies near its target row: its score stands 0 to 12 above the others'
    near = torch.rand(nq, 1, device="cuda", generator=gen) * (6.0 / math.sqrt(d))
    wide_q[:, :d] += near * wide_x[targets, :d]
    x = wide_x.to(dt)[:, :d]
    q = wide_q.to(dt)[:, :d]
    if nq > 4:
        # some queries have no given row
        targets[torch.rand(nq, device="cuda", generator=gen) < 0.05] = -1
    allowed = None
    if case["mask"] != "none":
        rows = nq if case["mask"] == "each" else 1
        words = (n + 31) // 32
        # one bit a row, 32 to a word: filters that keep an eighth to nearly all
        bits = [torch.randint(-2 ** 31, 2 ** 31, (rows, words), device="cuda", generator=gen,
                              dtype=torch.int64).to(torch.int32) for _ in range(3)]
        kind = torch.randint(0, 3, (rows, 1), device="cuda", generator=gen)
        allowed = torch.where(kind == 0, bits[0] & bits[1] & bits[2],
                              torch.where(kind == 1, bits[0], bits[0] | bits[1] | bits[2]))
        if rows > 8:
            allowed[torch.rand(rows, device="cuda", generator=gen) < 0.02] = 0
        allowed = allowed.contiguous()
    return {"q": q, "x": x, "targets": targets, "allowed": allowed, "scale": 2.0 / math.sqrt(d),
            "gen": gen}


def prepare(case, seed):
    if case["op"] == "adamw":
        gen = torch.Generator(device="cuda").manual_seed(seed)
        dt = DTYPES[case["dtype"]]
        sizes = _sizes(case)
        starts, at = [], 0
        for s in sizes:  # every tensor starts at a multiple of a block, as an allocator would align it
            starts.append(at)
            at += (s + BLOCK - 1) // BLOCK * BLOCK
        real = torch.zeros(at, dtype=torch.bool, device="cuda")
        for s, b in zip(sizes, starts):
            real[b:b + s] = True
        row = torch.exp2(torch.randn(at // BLOCK, 1, device="cuda", generator=gen) * 2)
        flat = lambda: torch.randn(at, device="cuda", generator=gen)  # noqa: E731
        p = (flat() * 0.05 * real).to(dt)
        spread = (flat().view(-1, BLOCK) * row).view(-1) * 1e-3 * real
        g = spread.to(dt)
        m = spread * 0.3 + (flat().view(-1, BLOCK) * row).view(-1) * 2e-4 * real
        v = (spread * spread + 1e-8 * row.repeat_interleave(BLOCK, 0).view(-1) ** 2) * real
        state = {"op": "adamw", "bits": case["state"], "sizes": sizes, "starts": starts, "p": p,
                 "g": g, "lr": 1e-3, "betas": (0.9, 0.999), "eps": 1e-8, "weight_decay": 0.01,
                 "step": 10, "seed": seed & 0xFFFFFFFF}
        if case["state"] == 8:
            state["ordinal"] = torch.repeat_interleave(
                torch.arange(len(sizes), device="cuda"),
                torch.tensor([(s + BLOCK - 1) // BLOCK for s in sizes], device="cuda"))
            state["first"] = torch.tensor(starts, device="cuda")
            # states that an earlier step left: codes to the nearest, at least 1 for v > 0
            sm = m.view(-1, BLOCK).abs().amax(1)
            sv = v.view(-1, BLOCK).amax(1)
            cm = (127 * (m.view(-1, BLOCK).abs() / sm.clamp_min(1e-30)[:, None]).sqrt()).round()
            state["m"] = (cm * torch.sign(m).view(-1, BLOCK)).to(torch.int8).view(-1)
            cv = (255 * (v.view(-1, BLOCK) / sv.clamp_min(1e-30)[:, None]).sqrt().sqrt()).round()
            cv = torch.where((v.view(-1, BLOCK) > 0) & (cv < 1), torch.ones_like(cv), cv)
            state["v"] = cv.to(torch.uint8).view(-1)
            state["m_scale"], state["v_scale"] = sm, sv
        else:
            state["m"], state["v"] = m, v
        # the program's own lists of tensors: views of one allocation, as it keeps them
        parts = lambda x: [x[b:b + s] for s, b in zip(sizes, starts)]  # noqa: E731
        state["views"] = {k: parts(state[k]) for k in ("p", "g", "m", "v")}
        if case["state"] == 8:
            for k in ("m_scale", "v_scale"):
                state["views"][k] = [state[k][b // BLOCK:(b + s + BLOCK - 1) // BLOCK]
                                     for s, b in zip(sizes, starts)]
        return state
    state = _scores_inputs(case, seed)
    gen = state.pop("gen")
    state["op"], state["k"] = case["op"], case.get("k", 0)
    if case["op"] == "logprobs_backward":
        nq = case["nq"]
        out = _logprobs(dict(state, k=0))
        state["lse"], state["entropy"] = out["lse"], out["entropy"]
        # a weighted mean of -logprob, an entropy bonus and a pull of the normaliser to zero
        state["d_logprob"] = -torch.rand(nq, device="cuda", generator=gen) / nq
        state["d_entropy"] = -0.05 * torch.rand(nq, device="cuda", generator=gen) / nq
        state["d_lse"] = 2e-4 * torch.nan_to_num(state["lse"], neginf=0.0) / nq
    return state


# ---------------------------------------------------------------------------
# the plain forms
# ---------------------------------------------------------------------------
def _bits(allowed, n):
    """[rows, words] of 32 bits -> [rows, n] truth values."""
    j = torch.arange(32, device=allowed.device, dtype=torch.int32)
    return ((allowed[:, :, None] >> j) & 1).bool().reshape(allowed.shape[0], -1)[:, :n]


def _scores(st):
    s = (st["q"].float() @ st["x"].float().T) * st["scale"]
    if st["allowed"] is not None:
        s = s.masked_fill(~_bits(st["allowed"], s.shape[1]), -math.inf)
    return s


def _logprobs(st):
    s = _scores(st)
    nq, n = s.shape
    m = s.amax(1, keepdim=True)
    some = m[:, 0] > -math.inf
    z = s - m.masked_fill(~some[:, None], 0.0)
    e = z.exp()
    total = e.sum(1)
    lse = torch.where(some, m[:, 0] + total.log(), m[:, 0])
    # sum p (s - m) = sum e (s - m) / sum e, with 0 for what has no part
    mean = (e * z.masked_fill(z == -math.inf, 0.0)).sum(1) / total
    entropy = torch.where(some, total.log() - mean, torch.zeros_like(mean))
    given = st["targets"] >= 0
    at = s.gather(1, st["targets"].clamp_min(0)[:, None])[:, 0]
    logprob = torch.where(given, torch.where(some, at - lse, at), torch.zeros_like(at))
    out = {"logprob": logprob, "lse": lse, "entropy": entropy}
    k = st["k"]
    if k:
        # which rows stand at the border is decided in 64 bits, over more candidates than asked for
        c = min(n, k + 16)
        ids = s.topk(c, 1).indices.sort(1).values
        exact = (st["x"][ids].double() * st["q"].double()[:, None]).sum(2) * st["scale"]
        exact = exact.masked_fill(s.gather(1, ids) == -math.inf, -math.inf)
        exact, order = torch.sort(exact, dim=1, descending=True, stable=True)
        ids = ids.gather(1, order)
        ids = ids.masked_fill(exact == -math.inf, -1)
        top = torch.where(ids < 0, exact, exact - lse.double()[:, None])
        if c < k:
            ids = torch.cat([ids, ids.new_full((nq, k - c), -1)], 1)
            top = torch.cat([top, top.new_full((nq, k - c), -math.inf)], 1)
        out["top_ids"], out["top_logprobs"] = ids[:, :k], top[:, :k].float()
    return out


def _backward(st):
    s = _scores(st)
    some = st["lse"] > -math.inf
    lp = s - torch.where(some, st["lse"], torch.zeros_like(st["lse"]))[:, None]
    p = lp.exp()
    lp = lp.masked_fill(lp == -math.inf, 0.0)
    given = (st["targets"] >= 0) & some
    t = st["targets"].clamp_min(0)[:, None]
    given &= s.gather(1, t)[:, 0] > -math.inf
    g = torch.where(given, st["d_logprob"], torch.zeros_like(st["d_logprob"]))
    grad = p * ((st["d_lse"] - g)[:, None] - st["d_entropy"][:, None] *
                (lp + st["entropy"][:, None]))
    grad.scatter_add_(1, t, g[:, None])
    grad *= st["scale"]
    dt = st["q"].dtype
    return {"d_queries": (grad @ st["x"].float()).to(dt),
            "d_rows": (grad.T @ st["q"].float()).to(dt)}


def _mix(h):
    """A 32-bit finaliser (two multiply-xorshift rounds) on int64 lanes."""
    h = ((h ^ (h >> 16)) * 0x7FEB352D) & 0xFFFFFFFF
    h = ((h ^ (h >> 15)) * 0x846CA68B) & 0xFFFFFFFF
    return h ^ (h >> 16)


def _up(y, low, high, u):
    """Whether y, between the values low and high of two neighbouring codes, goes to the upper one."""
    return u < (y - low) / (high - low)


def _values(m, m_scale, v, v_scale):
    """What 8-bit states stand for."""
    c = m.view(-1, BLOCK).float()
    r = v.view(-1, BLOCK).float()
    r = r * r
    return ((c * c.abs()) * (m_scale * (1 / 127 ** 2))[:, None]).view(-1), \
        ((r * r) * (v_scale * (1 / 255 ** 4))[:, None]).view(-1)


def _adamw(st):
    b1, b2 = st["betas"]
    g = st["g"].float()
    if st["bits"] == 8:
        m, v = _values(st["m"], st["m_scale"], st["v"], st["v_scale"])
    else:
        m, v = st["m"], st["v"]
    m = m * b1 + g * (1 - b1)
    v = v * b2 + (g * g) * (1 - b2)
    root = 1 / math.sqrt(1 - b2 ** st["step"])
    upd = m / (v.sqrt() * root + st["eps"])
    p = st["p"].float() * (1 - st["lr"] * st["weight_decay"]) - upd * (
        st["lr"] / (1 - b1 ** st["step"]))
    st["p"].copy_(p)
    if st["bits"] == 32:
        st["m"].copy_(m)
        st["v"].copy_(v)
        return {"p": st["p"], "m": st["m"], "v": st["v"]}
    m, v = m.view(-1, BLOCK), v.view(-1, BLOCK)
    sm, sv = m.abs().amax(1), v.amax(1)
    index = torch.arange(m.numel(), device=m.device).view(-1, BLOCK) - \
        st["first"][st["ordinal"]][:, None]
    h = _mix((index & 0xFFFFFFFF) ^ _mix((st["ordinal"][:, None] + (st["step"] << 16) +
                                          st["seed"]) & 0xFFFFFFFF) ^
             ((index >> 32) * 0x9E3779B1 & 0xFFFFFFFF))
    um = (h >> 8).float() * 2.0 ** -24
    uv = (_mix(h ^ 0x5BD1E995) >> 8).float() * 2.0 ** -24
    least = 2.0 ** -90  # a block whose largest value is below this is held as zeros
    zero = torch.zeros_like(sm)
    y = m.abs() * torch.where(sm > least, torch.full_like(sm, 127 ** 2) / sm, zero)[:, None]
    c = y.sqrt().floor()
    c = (c + _up(y, c * c, (c + 1) * (c + 1), um).float()).clamp_max(127)
    st["m"].copy_((c * torch.sign(m)).to(torch.int8).view(-1))
    y = v * torch.where(sv > least, torch.full_like(sv, 255 ** 4) / sv, zero)[:, None]
    c = y.sqrt().sqrt().floor()
    c2, d2 = c * c, (c + 1) * (c + 1)
    c = (c + _up(y, c2 * c2, d2 * d2, uv).float()).clamp_max(255)
    c = torch.where((y > 0) & (c < 1), torch.ones_like(c), c)
    st["v"].copy_(c.to(torch.uint8).view(-1))
    st["m_scale"].copy_(torch.where(sm < least, zero, sm))
    st["v_scale"].copy_(torch.where(sv < least, zero, sv))
    m, v = _values(st["m"], st["m_scale"], st["v"], st["v_scale"])
    return {"p": st["p"], "m": m, "v": v}


def _framework():
    import os
    import sys
    at = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "forge-db_b200")
    if at not in sys.path:
        sys.path.insert(0, at)
    import forgegpu
    return forgegpu


def run(state):
    if own:
        fg = _framework()
        if state["op"] == "logprobs":
            r = fg.logprobs(state["q"], state["x"], state["targets"], scale=state["scale"],
                            allowed=state["allowed"], k=state["k"])
            out = {"logprob": r.logprob, "lse": r.lse, "entropy": r.entropy}
            if state["k"]:
                out["top_ids"], out["top_logprobs"] = r.top_ids, r.top_logprobs
            return out
        if state["op"] == "logprobs_backward":
            dq, dx = fg.logprobs_backward(
                state["q"], state["x"], state["targets"], state["lse"], state["entropy"],
                d_logprob=state["d_logprob"], d_lse=state["d_lse"], d_entropy=state["d_entropy"],
                scale=state["scale"], allowed=state["allowed"])
            return {"d_queries": dq, "d_rows": dx}
        v = state["views"]
        fg.adamw_step(v["p"], v["g"], v["m"], v["v"], m_scales=v.get("m_scale"),
                      v_scales=v.get("v_scale"), lr=state["lr"], betas=state["betas"],
                      eps=state["eps"], weight_decay=state["weight_decay"], step=state["step"],
                      seed=state["seed"])
        if state["bits"] == 32:
            return {"p": state["p"], "m": state["m"], "v": state["v"]}
        m, v = fg.adamw_state_values(state["m"], state["m_scale"], state["v"], state["v_scale"])
        return {"p": state["p"], "m": m, "v": v}
    if state["op"] == "logprobs":
        return _logprobs(state)
    if state["op"] == "logprobs_backward":
        return _backward(state)
    return _adamw(state)


def work(case):
    if case["op"] == "adamw":
        es = 4 if case["dtype"] == "f32" else 2
        n = case["total"]
        if case["state"] == 32:
            return {"bytes": n * (3 * es + 16), "flops": 12 * n}
        # codes and scales in and out, and the values the codes stand for written out
        return {"bytes": n * (3 * es + 4 + 8) + n // BLOCK * 16, "flops": 40 * n}
    nq, n, d = case["nq"], case["n"], case["dim"]
    es = 4 if case["dtype"] == "f32" else 2
    mask = {"none": 0, "one": 1, "each": nq}[case["mask"]] * ((n + 31) // 32) * 4
    if case["op"] == "logprobs":
        return {"bytes": (nq + n) * d * es + mask + nq * (20 + 12 * case["k"]),
                "flops": 2 * nq * n * d}
    return {"bytes": 2 * (nq + n) * d * es + mask + nq * 28, "flops": 6 * nq * n * d}


# ---------------------------------------------------------------------------
# the definitions in 64 bits
# ---------------------------------------------------------------------------
def _exact_rows(q, x, allowed, scale):
    """Scores of a few queries in 64 bits, disallowed rows at -inf."""
    s = torch.einsum("id,jd->ij", q.double(), x.double()) * scale
    if allowed is not None:
        j = torch.arange(x.shape[0], device=x.device)
        keep = (allowed.long()[:, j // 32] >> (j % 32)) & 1
        s = torch.where(keep == 1, s, torch.full_like(s, -math.inf))
    return s


def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] == "adamw":
        b1, b2 = st["betas"]
        t = st["step"]
        g, p = st["g"].double(), st["p"].double()
        if case["state"] == 8:
            c, r = st["m"].double(), st["v"].double()
            m = torch.sign(c) * (c / 127) ** 2 * st["m_scale"].double().repeat_interleave(BLOCK)
            v = (r / 255) ** 4 * st["v_scale"].double().repeat_interleave(BLOCK)
        else:
            m, v = st["m"].double(), st["v"].double()
        m.mul_(b1).add_(g, alpha=1 - b1)
        v.mul_(b2).addcmul_(g, g, value=1 - b2)
        hat = (m / (1 - b1 ** t)) / ((v / (1 - b2 ** t)).sqrt() + st["eps"])
        p = p - st["lr"] * st["weight_decay"] * p - st["lr"] * hat
        if case["state"] == 8:  # which code a value goes to is a draw: no value of its own
            return {"p": p, "m": None, "v": None}
        return {"p": p, "m": m, "v": v}
    q, x, nq = st["q"], st["x"], case["nq"]
    step = max(1, min(nq, 100_000_000 // case["n"]))
    parts = []
    dx = torch.zeros(x.shape, dtype=torch.float64, device="cuda")
    for i in range(0, nq, step):
        sl = slice(i, min(nq, i + step))
        al = st["allowed"]
        s = _exact_rows(q[sl], x, al[sl] if al is not None and al.shape[0] > 1 else al,
                        st["scale"])
        t = st["targets"][sl]
        if case["op"] == "logprobs":
            lse = torch.logsumexp(s, 1)
            lp = s - lse[:, None]
            ent = torch.special.entr(lp.exp()).nan_to_num(0.0).sum(1)
            at = lp[torch.arange(len(t), device="cuda"), t.clamp_min(0)]
            at = torch.where(torch.isnan(at), torch.full_like(at, -math.inf), at)
            part = [torch.where(t < 0, torch.zeros_like(at), at), lse, ent]
            if case["k"]:
                k = min(case["k"], case["n"])
                val, ids = torch.sort(s, dim=1, descending=True, stable=True) if case["n"] < 4096 \
                    else torch.topk(s, k, 1)
                val, ids = val[:, :k], ids[:, :k]
                ids = torch.where(val == -math.inf, torch.full_like(ids, -1), ids)
                val = torch.where(val == -math.inf, val, val - lse[:, None])
                part += [torch.nn.functional.pad(ids, (0, case["k"] - k), value=-1),
                         torch.nn.functional.pad(val, (0, case["k"] - k), value=-math.inf)]
            parts.append(part)
            continue
        # the loss's own definition, differentiated: sum of upstream times output,
        # around the normaliser and the entropy that the forward pass left
        lse, ent = st["lse"][sl].double(), st["entropy"][sl].double()
        lp = s - lse.masked_fill(lse == -math.inf, 0.0)[:, None]
        p = torch.exp(lp)
        lp = torch.where(p > 0, lp, torch.zeros_like(s))
        hit = torch.zeros_like(p)
        ok = (t >= 0) & (lse > -math.inf)
        ok &= s.gather(1, t.clamp_min(0)[:, None])[:, 0] > -math.inf
        hit[torch.arange(len(t), device="cuda")[ok], t[ok]] = 1.0
        up = st["d_logprob"][sl].double() * ok
        grad = up[:, None] * (hit - p) + st["d_lse"][sl].double()[:, None] * p \
            - st["d_entropy"][sl].double()[:, None] * p * (lp + ent[:, None])
        grad *= st["scale"]
        parts.append(grad @ x.double())
        dx += grad.T @ q[sl].double()
    if case["op"] == "logprobs_backward":
        return {"d_queries": torch.cat(parts), "d_rows": dx}
    names = ["logprob", "lse", "entropy", "top_ids", "top_logprobs"]
    return {k: torch.cat(v) for k, v in zip(names, zip(*parts))}
