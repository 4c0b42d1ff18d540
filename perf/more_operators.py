"""Workloads of distillation over index rows and of beam search over them.

Four operators, each in its elementary form and, with ``own`` set, as a call
of the framework:

  distill            loss of a teacher's best rows under softmax(scale * q . x)
                     over all (allowed) rows: its k ids and logits per query,
                     as a distribution over those rows, or with one more
                     outcome for all rows that the teacher does not name
  distill_backward   its gradient with respect to the queries and the rows
  beam_select        the best continuations over beams and columns
  beam_reorder       states that follow the beams they were taken from
"""
import math

import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def listed():
    return [
        # one interaction's candidates, re-scored by a teacher: latency is everything
        {"name": "distill one query", "op": "distill", "dtype": "f32", "nq": 1, "n": 10_000,
         "dim": 128, "k": 16, "rest": False, "mask": "none", "pad": 0},
        # an ordinary training batch, a teacher that gives log probabilities of its best 64
        {"name": "distill batch", "op": "distill", "dtype": "bf16", "nq": 1_000, "n": 50_001,
         "dim": 768, "k": 64, "rest": True, "mask": "none", "pad": 0},
        # odd sizes, a filter for each query (known false negatives taken out), some empty,
        # rows that are a part of wider ones
        {"name": "distill filtered", "op": "distill", "dtype": "f32", "nq": 777, "n": 20_003,
         "dim": 96, "k": 10, "rest": True, "mask": "each", "pad": 5},
        # a large batch over a large table
        {"name": "distill large", "op": "distill", "dtype": "bf16", "nq": 2_048, "n": 131_072,
         "dim": 768, "k": 32, "rest": False, "mask": "none", "pad": 0},
        # a small fine-tuning batch over a small table
        {"name": "distill backward small", "op": "distill_backward", "dtype": "f32", "nq": 100,
         "n": 10_000, "dim": 128, "k": 16, "rest": True, "mask": "none", "pad": 0},
        # filters, odd sizes, 16 bits of a small range
        {"name": "distill backward filtered", "op": "distill_backward", "dtype": "f16",
         "nq": 601, "n": 30_011, "dim": 200, "k": 7, "rest": False, "mask": "each", "pad": 0},
        # the large batch's
        {"name": "distill backward large", "op": "distill_backward", "dtype": "bf16",
         "nq": 2_048, "n": 131_072, "dim": 768, "k": 32, "rest": True, "mask": "none", "pad": 0},
        # one user's chains over a small index, scores of every row
        {"name": "select one user", "op": "beam_select", "form": "logits", "dtype": "f32",
         "groups": 1, "beams": 4, "n": 10_000, "width": 4, "mask": "none", "ended": False},
        # chains over a large index: each beam's best rows as a search left them
        {"name": "select from lists", "op": "beam_select", "form": "lists", "dtype": "f32",
         "groups": 64, "beams": 8, "n": 20, "width": 8, "mask": "none", "ended": True},
        # a serving batch over an output layer of many rows
        {"name": "select batch", "op": "beam_select", "form": "logits", "dtype": "bf16",
         "groups": 64, "beams": 8, "n": 131_072, "width": 8, "mask": "none", "ended": True},
        # what a chain carries in a retriever: its ids and its query vector
        {"name": "reorder chains", "op": "beam_reorder", "dtype": "f32", "groups": 8, "beams": 4,
         "width": 4, "tensors": 2, "heads": 1, "used": 1, "room": 1, "dim": 128},
        # what it carries in a decoder: caches of every layer, of which a part is in use
        {"name": "reorder caches", "op": "beam_reorder", "dtype": "bf16", "groups": 16,
         "beams": 8, "width": 8, "tensors": 16, "heads": 8, "used": 391, "room": 512, "dim": 64},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["distill", "distill", "distill_backward", "distill_backward", "beam_select",
                     "beam_select", "beam_reorder"])
    while True:
        if op == "beam_reorder":
            beams = rng.choice([1, 2, 3, 4, 5, 8, 12, 16, 32])
            c = {"op": op, "dtype": rng.choice(["f32", "bf16", "f16"]), "groups": _log(rng, 1, 64),
                 "beams": beams, "width": rng.choice([beams, 2 * beams]),
                 "tensors": _log(rng, 1, 40), "heads": rng.choice([1, 2, 3, 4, 8]),
                 "used": _log(rng, 1, 1_000), "dim": _log(rng, 1, 256)}
            c["room"] = c["used"] if c["heads"] == 1 else c["used"] + _log(rng, 1, 300)
            if _state_bytes(c) > 430_000_000:
                continue
            return c
        if op == "beam_select":
            beams = rng.choice([1, 2, 3, 4, 5, 6, 8, 10, 16, 32])
            c = {"op": op, "form": rng.choice(["logits", "logits", "lists"]),
                 "dtype": rng.choice(["f32", "bf16", "f16"]), "groups": _log(rng, 1, 256),
                 "beams": beams, "width": rng.choice([beams, beams, 2 * beams]),
                 "mask": rng.choice(["none", "none", "one", "each"]),
                 "ended": rng.choice([False, True])}
            if c["form"] == "lists":
                c["dtype"], c["mask"], c["n"] = "f32", "none", rng.randint(1, 64)
                return c
            c["n"] = _log(rng, 200, 262_144)
            if c["groups"] * beams * c["n"] > 64 * 8 * 131_072 // (2 if c["dtype"] == "f32" else 1):
                continue
            return c
        c = {"op": op, "dtype": rng.choice(["f32", "bf16", "f16"]), "nq": _log(rng, 1, 4_096),
             "n": _log(rng, 500, 262_144), "dim": _log(rng, 16, 1_024), "k": _log(rng, 1, 128),
             "rest": rng.choice([False, True]),
             "mask": rng.choice(["none", "none", "one", "each"]), "pad": rng.choice([0, 0, 8, 3])}
        # no dearer than the largest listed case, in products and in scores held at once
        if c["nq"] * c["n"] * c["dim"] > 2_048 * 131_072 * 768 // (3 if c["dtype"] == "f32" else 1):
            continue
        if c["nq"] * c["n"] > 300_000_000 or c["nq"] * c["k"] * c["dim"] > 100_000_000:
            continue
        return c


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
def _state_bytes(c):
    """Bytes of all rows that a reordering writes."""
    es = 4 if c["dtype"] == "f32" else 2
    rows = c["groups"] * c["width"]
    return rows * (c["tensors"] * c["heads"] * c["used"] * c["dim"] * es + 16 * 8)


def _filters(gen, rows, n):
    """One bit a column, 32 to a word: filters that keep an eighth to nearly all, a few none."""
    words = (n + 31) // 32
    bits = [torch.randint(-2 ** 31, 2 ** 31, (rows, words), device="cuda", generator=gen,
                          dtype=torch.int64).to(torch.int32) for _ in range(3)]
    kind = torch.randint(0, 3, (rows, 1), device="cuda", generator=gen)
    allowed = torch.where(kind == 0, bits[0] & bits[1] & bits[2],
                          torch.where(kind == 1, bits[0], bits[0] | bits[1] | bits[2]))
    if rows > 8:
        allowed[torch.rand(rows, device="cuda", generator=gen) < 0.02] = 0
    return allowed.contiguous()


def _distill_inputs(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    nq, n, d, k = case["nq"], case["n"], case["dim"], case["k"]
    dt = DTYPES[case["dtype"]]
    rand = lambda *s: torch.rand(*s, device="cuda", generator=gen)  # noqa: E731
    wide_x = torch.randn(n, d + case["pad"], device="cuda", generator=gen)
    wide_q = torch.randn(nq, d + case["pad"], device="cuda", generator=gen)
    ids = torch.randint(0, n, (nq, k), device="cuda", generator=gen)
    # a query lies near the teacher's first rows, some queries far nearer than others
    near = rand(nq, 1) * (6.0 / math.sqrt(d))
    for j in range(min(k, 3)):
        wide_q[:, :d] += near / (j + 1) * wide_x[ids[:, j], :d]
    x = wide_x.to(dt)[:, :d]
    q = wide_q.to(dt)[:, :d]
    # the teacher's logits, best first; as log probabilities they leave 1 to 50 % to other rows
    z = torch.sort(torch.randn(nq, k, device="cuda", generator=gen) * 3, 1, descending=True).values
    if case["rest"]:
        z = z - torch.logsumexp(z, 1, keepdim=True) + torch.log(1 - 0.5 ** (1 + 6 * rand(nq, 1)))
    # lists that are not full, and some that are empty
    full = torch.where(rand(nq, 1) < 0.9, torch.full((nq, 1), k, device="cuda"),
                       torch.randint(0, k + 1, (nq, 1), device="cuda", generator=gen))
    late = torch.arange(k, device="cuda") >= full
    ids = ids.masked_fill(late, -1)
    z = z.masked_fill(late, -math.inf)
    allowed = None
    if case["mask"] != "none":
        allowed = _filters(gen, nq if case["mask"] == "each" else 1, n)
    return {"op": case["op"], "q": q, "x": x, "ids": ids, "z": z, "rest": case["rest"],
            "allowed": allowed, "scale": 2.0 / math.sqrt(d),
            "teacher_scale": 1.0 if case["rest"] else 0.5, "gen": gen}


def _beam_inputs(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    g, b, n = case["groups"], case["beams"], case["n"]
    rand = lambda *s: torch.rand(*s, device="cuda", generator=gen)  # noqa: E731
    st = {"op": "beam_select", "width": case["width"], "scale": 1.0, "ids": None, "allowed": None,
          "ended": None, "end_id": 1}
    # summed log probabilities, best first, as the step before left them
    st["beam_scores"] = -torch.cumsum(rand(g, b) * 0.7, 1) - 3.0 * rand(g, 1)
    if case["form"] == "lists":
        # each beam's best rows with their log probabilities, some lists short
        st["normalise"] = False
        st["scores"] = -0.5 - torch.cumsum(rand(g, b, n) * 0.6, 2)
        ids = torch.randint(0, 1_000_000, (g, b, n), device="cuda", generator=gen)
        ids[:, :, n // 2:] = ids[:, :, n // 2:].masked_fill(rand(g, b, 1) < 0.1, -1)
        st["ids"] = ids
    else:
        st["normalise"] = True
        st["scale"] = 0.8
        logits = torch.randn(g, b, n, device="cuda", generator=gen)
        logits *= 1.0 + 2.0 * rand(g, b, 1)
        # a few columns stand out, in some rows by a lot
        peaks = torch.randint(0, n, (g, b, 6), device="cuda", generator=gen)
        logits.scatter_add_(2, peaks, 12.0 * rand(g, b, 6) * rand(g, b, 1))
        st["scores"] = logits.to(DTYPES[case["dtype"]])
        if case["mask"] != "none":
            rows = g * b if case["mask"] == "each" else 1
            st["allowed"] = _filters(gen, rows, n).view(rows, -1)
    if case["ended"]:
        ended = torch.zeros(g, b, dtype=torch.bool, device="cuda")
        ended[:, :(b + 7) // 8] = True
        order = torch.argsort(rand(g, b), 1)
        st["ended"] = ended.gather(1, order)
    return st


def _state_inputs(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    g, b, w = case["groups"], case["beams"], case["width"]
    dt = DTYPES[case["dtype"]]
    # about five eighths of the beams survive, the others' places are taken by copies of these
    kept = max(1, 5 * b // 8)
    first = torch.argsort(torch.rand(g, b, device="cuda", generator=gen), 1)[:, :kept]
    more = first.gather(1, torch.randint(0, kept, (g, w), device="cuda", generator=gen))
    parents = torch.cat([first, more[:, kept:]], 1)[:, :w]
    parents = parents.gather(1, torch.argsort(torch.rand(g, w, device="cuda", generator=gen), 1))
    shape = (case["heads"], case["room"], case["dim"])
    states, outs = [], []
    for _ in range(case["tensors"]):
        states.append(torch.randn(g, b, *shape, device="cuda", generator=gen).to(dt))
        outs.append(torch.empty(g, w, *shape, device="cuda", dtype=dt))
    # the chains' ids so far
    states.append(torch.randint(0, 1_000_000, (g, b, 16), device="cuda", generator=gen))
    outs.append(torch.empty(g, w, 16, device="cuda", dtype=torch.int64))
    # only the positions in use move
    used = case["used"]
    part = lambda t: t[:, :, :, :used] if t.dim() == 5 else t  # noqa: E731
    return {"op": "beam_reorder", "states": [part(t) for t in states],
            "outs": [part(t) for t in outs], "parents": parents}


def prepare(case, seed):
    if case["op"] == "beam_select":
        return _beam_inputs(case, seed)
    if case["op"] == "beam_reorder":
        return _state_inputs(case, seed)
    st = _distill_inputs(case, seed)
    gen = st.pop("gen")
    if case["op"] == "distill_backward":
        nq = case["nq"]
        out = _distill(st)
        st["lse"], st["logprobs"], st["rest_logprob"] = \
            out["lse"], out["logprobs"], out.get("rest")
        # a weighted mean of the losses; training in f16 scales its loss
        st["d_loss"] = torch.rand(nq, device="cuda", generator=gen) / nq * (
            1024.0 if case["dtype"] == "f16" else 1.0)
    return st


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


def _entries(st):
    """Which entries of the teacher's lists take part: rows of the index that the query may
    see, with some weight, each id once."""
    ids, n = st["ids"], st["x"].shape[0]
    ok = (ids >= 0) & (ids < n) & (st["z"] != -math.inf)
    at = ids.clamp(0, n - 1)
    if st["allowed"] is not None:
        al = st["allowed"].expand(ids.shape[0], -1)
        ok &= ((al.gather(1, at // 32) >> (at % 32).int()) & 1).bool()
    k = ids.shape[1]
    earlier = torch.ones(k, k, dtype=torch.bool, device=ids.device).tril(-1)
    again = ((ids[:, :, None] == ids[:, None, :]) & ok[:, None, :] & earlier).any(2)
    return ok & ~again, at


def _lse(s, dim=1):
    m = s.amax(dim, keepdim=True)
    m0 = m.masked_fill(m == -math.inf, 0.0)
    return ((s - m0).exp().sum(dim, keepdim=True).log() + m0).squeeze(dim)


def _teacher(st, ok, others):
    """(P, R) in 64 bits: the teacher's probabilities of its rows and of all others."""
    z = st["z"].double() * st["teacher_scale"]
    z = z.masked_fill(~ok, -math.inf)
    total = _lse(z)
    if not st["rest"]:
        return (z - total.masked_fill(total == -math.inf, 0.0)[:, None]).exp(), \
            torch.zeros_like(total)
    # (more than 1 in all, or no other row to see: as a distribution over its rows)
    whole = (total > 0) | ~others
    p = (z - total.masked_fill(~whole | (total == -math.inf), 0.0)[:, None]).exp()
    r = torch.where(whole, torch.zeros_like(total), 1 - p.sum(1))
    return p, r


def _distill(st):
    s = _scores(st)
    nq, n = s.shape
    ok, at = _entries(st)
    # the named rows' scores in 64 bits, as 1 - p of a sure student loses all else
    t = (st["x"][at].double() * st["q"].double()[:, None]).sum(2) * st["scale"]
    t = t.masked_fill(~ok, -math.inf)
    if st["rest"]:
        s = torch.cat([s, s.new_zeros(nq, 1)], 1)
        s.scatter_(1, torch.where(ok, at, n), -math.inf)
        s[:, n] = -math.inf
        other = _lse(s).double()
        both = torch.stack([other, _lse(t)], 1)
        lse = _lse(both)
        others = other > -math.inf
    else:
        lse = _lse(s).double()
        others = None
    some = lse > -math.inf
    lp = torch.where(ok, t - lse.masked_fill(~some, 0.0)[:, None], torch.zeros_like(t))
    p, r = _teacher(st, ok, others)
    logp = p.masked_fill(p == 0, 1.0).log()
    loss = (p * (logp - lp)).sum(1)
    out = {"lse": lse.float(), "logprobs": lp.float()}
    if st["rest"]:
        rest = torch.where(others, other - lse.masked_fill(~some, 0.0), other)
        named = ok.any(1)
        loss += torch.where((r > 0) & named, r * (r.clamp_min(1e-300).log() - rest),
                            torch.zeros_like(r))
        out["rest"] = rest.float()
    out["loss"] = loss.float()
    return out


def _distill_backward(st):
    s = _scores(st)
    nq, n = s.shape
    ok, at = _entries(st)
    some = (st["lse"] > -math.inf) & ok.any(1)
    u = torch.where(some, st["d_loss"], torch.zeros_like(st["d_loss"])).double() * st["scale"]
    ref = st["lse"].double().masked_fill(~some, 0.0)
    share = torch.ones_like(ref)
    others = None
    if st["rest"]:
        others = st["rest_logprob"] > -math.inf
        rest = st["rest_logprob"].double()
        share = rest.exp()
        ref = ref + rest.masked_fill(~others, 0.0)
    p, r = _teacher(st, ok, others)
    # of a row that the teacher does not name: exp(s - lse_rest) (r - R)
    grad = torch.cat([(s - ref.float()[:, None]).exp_(), s.new_zeros(nq, 1)], 1)
    grad *= (u * (share - r)).float()[:, None]
    named = u[:, None] * (st["logprobs"].double().exp() - p)
    grad.scatter_(1, torch.where(ok, at, n), torch.where(ok, named, torch.zeros_like(p)).float())
    grad[~some] = 0.0
    grad = grad[:, :n]
    dt = st["q"].dtype
    return {"d_queries": (grad @ st["x"].float()).to(dt),
            "d_rows": (grad.T @ st["q"].float()).to(dt)}


def _beam_select(st):
    x, w = st["scores"], st["width"]
    g, b, n = x.shape
    # borders between beams are decided in 64 bits
    s = x.double() * st["scale"]
    if st["ids"] is not None:
        s = s.masked_fill(st["ids"] < 0, -math.inf)
    if st["allowed"] is not None:
        keep = _bits(st["allowed"], n)
        s = s.masked_fill(~(keep.view(g, b, n) if keep.shape[0] > 1 else keep.view(1, 1, n)),
                          -math.inf)
    if st["normalise"]:
        lse = _lse(s, 2)
        s = s - lse.masked_fill(lse == -math.inf, 0.0)[:, :, None]
    s = s + st["beam_scores"].double()[:, :, None]
    ids = st["ids"]
    if st["ended"] is not None:
        # a chain that has ended goes on as it is: one candidate, in its first column
        s = s.masked_fill(st["ended"][:, :, None], -math.inf)
        s[:, :, 0] = torch.where(st["ended"], st["beam_scores"].double(), s[:, :, 0])
    s = s.view(g, b * n)
    # more candidates than asked for: equal ones at the border go by beam, then column
    c = min(b * n, w + 64)
    at = s.topk(c, 1).indices.sort(1).values
    val, order = torch.sort(s.gather(1, at), dim=1, descending=True, stable=True)
    at, val = at.gather(1, order)[:, :w], val[:, :w]
    if c < w:
        at = torch.cat([at, at.new_zeros(g, w - c)], 1)
        val = torch.cat([val, val.new_full((g, w - c), -math.inf)], 1)
    none = val == -math.inf
    parent, col = at // n, at % n
    out = col if ids is None else ids.view(g, -1).gather(1, at)
    done = torch.zeros_like(none)
    if st["ended"] is not None:
        done = st["ended"].gather(1, parent)
        out = torch.where(done, torch.full_like(out, st["end_id"]), out)
    done = (done | (out == st["end_id"])) & ~none
    return {"scores": val.float(), "parents": parent.masked_fill(none, -1),
            "ids": out.masked_fill(none, -1), "ended": done}


def _beam_reorder(st):
    g = torch.arange(st["parents"].shape[0], device="cuda")[:, None]
    for src, dst in zip(st["states"], st["outs"]):
        dst.copy_(src[g, st["parents"]])
    return list(st["outs"])


def _framework():
    import os
    import sys
    at = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "forge-db_b200")
    if at not in sys.path:
        sys.path.insert(0, at)
    import forgegpu
    return forgegpu


def run(state):
    op = state["op"]
    if own:
        fg = _framework()
        if op == "distill":
            r = fg.distill(state["q"], state["x"], state["ids"], state["z"], scale=state["scale"],
                           teacher_scale=state["teacher_scale"], rest=state["rest"],
                           allowed=state["allowed"])
            out = {"loss": r.loss, "lse": r.lse, "logprobs": r.logprobs}
            if state["rest"]:
                out["rest"] = r.rest
            return out
        if op == "distill_backward":
            dq, dx = fg.distill_backward(
                state["q"], state["x"], state["ids"], state["z"], state["lse"],
                state["logprobs"], state["rest_logprob"], d_loss=state["d_loss"],
                scale=state["scale"], teacher_scale=state["teacher_scale"],
                allowed=state["allowed"])
            return {"d_queries": dq, "d_rows": dx}
        if op == "beam_select":
            r = fg.beam_select(state["scores"], state["beam_scores"], width=state["width"],
                               ids=state["ids"], scale=state["scale"],
                               normalise=state["normalise"], allowed=state["allowed"],
                               ended=state["ended"], end_id=state["end_id"])
            return {"scores": r.scores, "parents": r.parents, "ids": r.ids, "ended": r.ended}
        return fg.beam_reorder(state["states"], state["parents"], out=state["outs"])
    if op == "distill":
        return _distill(state)
    if op == "distill_backward":
        return _distill_backward(state)
    if op == "beam_select":
        return _beam_select(state)
    return _beam_reorder(state)


def work(case):
    op = case["op"]
    if op == "beam_reorder":
        # of the rows, those that survive are read
        out = _state_bytes(case)
        return {"bytes": out + out // case["width"] * max(1, 5 * case["beams"] // 8), "flops": 0}
    es = 4 if case["dtype"] == "f32" else 2
    if op == "beam_select":
        g, b, n = case["groups"], case["beams"], case["n"]
        rows = g * (b - (b + 7) // 8 if case["ended"] else b)
        mask = {"none": 0, "one": 1, "each": rows}[case["mask"]] * ((n + 31) // 32) * 4
        each = es + (8 if case["form"] == "lists" else 0)
        return {"bytes": rows * n * each + mask + g * b * 5 + g * case["width"] * 21,
                "flops": 4 * rows * n}
    nq, n, d, k = case["nq"], case["n"], case["dim"], case["k"]
    mask = {"none": 0, "one": 1, "each": nq}[case["mask"]] * ((n + 31) // 32) * 4
    if op == "distill":
        return {"bytes": (nq + n) * d * es + mask + nq * (k * 16 + 12), "flops": 2 * nq * n * d}
    return {"bytes": 2 * (nq + n) * d * es + mask + nq * (k * 16 + 12), "flops": 6 * nq * n * d}


# ---------------------------------------------------------------------------
# the definitions in 64 bits
# ---------------------------------------------------------------------------
def _visible(allowed, rows, n):
    """[rows, n] truth values of what each row may see."""
    if allowed is None:
        return torch.ones(rows, n, dtype=torch.bool, device="cuda")
    j = torch.arange(n, device="cuda")
    return ((allowed.long()[:, j // 32] >> (j % 32)) & 1 == 1).expand(rows, n)


def _named(ids, z, seen):
    """Teacher's entries as weights of rows: [nq, n] logits (-inf: not named) and, for each
    entry, whether it is the one that stands for its row."""
    nq, n = seen.shape
    table = torch.full((nq, n), -math.inf, dtype=torch.float64, device="cuda")
    used = torch.zeros(ids.shape, dtype=torch.bool, device="cuda")
    row = torch.arange(nq, device="cuda")
    for j in range(ids.shape[1]):
        t = ids[:, j].clamp(0, n - 1)
        free = (ids[:, j] >= 0) & (ids[:, j] < n) & seen[row, t] & (table[row, t] == -math.inf)
        free &= z[:, j] > -math.inf
        table[row[free], t[free]] = z[free, j].double()
        used[:, j] = free
    return table, used


def _exact_distill(case, st):
    q, x, nq, n = st["q"], st["x"], case["nq"], case["n"]
    step = max(1, min(nq, 60_000_000 // n))
    back = case["op"] == "distill_backward"
    parts = {}
    dx = torch.zeros(x.shape, dtype=torch.float64, device="cuda") if back else None
    xd = x.double()
    for i in range(0, nq, step):
        sl = slice(i, min(nq, i + step))
        m = min(nq, i + step) - i
        al = st["allowed"]
        seen = _visible(al[sl] if al is not None and al.shape[0] > 1 else al, m, n)
        s = torch.einsum("id,jd->ij", q[sl].double(), xd) * st["scale"]
        s = torch.where(seen, s, torch.full_like(s, -math.inf))
        table, used = _named(st["ids"][sl], st["z"][sl], seen)
        known = table > -math.inf
        names = known.any(1)
        other = seen & ~known
        if case["rest"]:
            p = torch.exp(table)
            mass = p.sum(1)
            norm = (mass > 1) | ~other.any(1)
        else:
            p = torch.exp(table * st["teacher_scale"] -
                          (table * st["teacher_scale"]).amax(1, keepdim=True))
            p = torch.where(known, p, torch.zeros_like(p))
            mass = p.sum(1)
            norm = torch.ones_like(names)
        p = torch.where((norm & names)[:, None], p / mass[:, None], p)
        left = torch.where(norm, torch.zeros_like(mass), 1 - mass)
        at = st["ids"][sl].clamp(0, n - 1)
        if back:
            # around what the forward pass left
            lse = st["lse"][sl].double()
            live = names & (lse > -math.inf)
            u = torch.where(live, st["d_loss"][sl].double(), torch.zeros_like(lse))
            lpn = torch.full((m, n), -math.inf, dtype=torch.float64, device="cuda")
            pos = used.nonzero()
            lpn[pos[:, 0], at[used]] = st["logprobs"][sl].double()[used]
            grad = torch.exp(lpn) - p
            lr = st["rest_logprob"][sl].double() if case["rest"] else torch.zeros_like(lse)
            rest = torch.exp(s - lse[:, None] - lr[:, None]) * (torch.exp(lr) - left)[:, None]
            grad = torch.where(other, rest, grad) * u[:, None] * st["scale"]
            grad = torch.where(live[:, None], grad, torch.zeros_like(grad))
            parts.setdefault("d_queries", []).append(grad @ xd)
            dx += grad.T @ q[sl].double()
            continue
        lse = torch.logsumexp(s, 1)
        logp = torch.log_softmax(s, 1)
        # (0 log 0 = 0; a row that is not named has no part in the sum)
        each = torch.where(p > 0, p * (torch.log(p) - logp), torch.zeros_like(p))
        loss = each.sum(1)
        lp = torch.where(used, logp.gather(1, at), torch.zeros_like(at, dtype=torch.float64))
        if case["rest"]:
            rest = torch.logsumexp(torch.where(other, s, torch.full_like(s, -math.inf)), 1)
            rest = torch.where(rest == -math.inf, rest, rest - lse)
            loss += torch.where(names & (left > 0), left * (torch.log(left.clamp_min(1e-300)) - rest),
                                torch.zeros_like(left))
            parts.setdefault("rest", []).append(rest)
        parts.setdefault("loss", []).append(loss)
        parts.setdefault("lse", []).append(lse)
        parts.setdefault("logprobs", []).append(lp)
    out = {k: torch.cat(v) for k, v in parts.items()}
    if back:
        out["d_rows"] = dx
    return out


def _exact_select(st):
    x, w = st["scores"], st["width"]
    g, b, n = x.shape
    seen = _visible(st["allowed"], g * b, n).reshape(g, b, n)
    out = {"scores": [], "parents": [], "ids": [], "ended": []}
    for i in range(g):  # a group at a time
        keep = seen[i]
        if st["ids"] is not None:
            keep = keep & (st["ids"][i] >= 0)
        s = torch.where(keep, x[i].double() * st["scale"],
                        torch.full((), -math.inf, dtype=torch.float64, device="cuda"))
        if st["normalise"]:
            s = torch.where(keep.any(1, keepdim=True), torch.log_softmax(s, 1), s)
        s = s + st["beam_scores"][i].double()[:, None]
        names = torch.arange(n, device="cuda").expand(b, n) if st["ids"] is None else st["ids"][i]
        if st["ended"] is not None:
            done = st["ended"][i]
            own_place = torch.full_like(s, -math.inf)
            own_place[:, 0] = st["beam_scores"][i].double()
            s = torch.where(done[:, None], own_place, s)
            names = torch.where(done[:, None], torch.full_like(names, st["end_id"]), names)
        flat, names = s.reshape(-1), names.reshape(-1)
        # whatever reaches the last place's score, in order, equal ones as they stand
        m = min(w, flat.numel())
        least = torch.topk(flat, m).values[-1]
        at = (flat >= least).nonzero()[:, 0]
        at = at[torch.argsort(flat[at], descending=True, stable=True)][:m]
        val, name = flat[at], names[at]
        parent = torch.div(at, n, rounding_mode="floor")
        gone = val == -math.inf
        fill = lambda t, v: torch.nn.functional.pad(t, (0, w - m), value=v)  # noqa: E731
        done = (name == st["end_id"])
        if st["ended"] is not None:
            done |= st["ended"][i][parent]
        out["scores"].append(fill(val, -math.inf))
        out["parents"].append(fill(torch.where(gone, torch.full_like(parent, -1), parent), -1))
        out["ids"].append(fill(torch.where(gone, torch.full_like(name, -1), name), -1))
        out["ended"].append(fill((done & ~gone).to(torch.int64), 0).bool())
    return {k: torch.stack(v) for k, v in out.items()}


def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] == "beam_select":
        return _exact_select(st)
    if case["op"] == "beam_reorder":
        # a copy: every value is what its parent's is
        out = []
        for src in st["states"]:
            rows = src.reshape(src.shape[0] * src.shape[1], -1)
            b = src.shape[1]
            at = (st["parents"] + b * torch.arange(src.shape[0], device="cuda")[:, None]).view(-1)
            out.append(rows[at].view(*st["parents"].shape, *src.shape[2:]))
        return out
    return _exact_distill(case, st)
