"""Plain 64-bit forms of the distillation loss, its gradient and a beam search's
step, with bounds of what the kernels may be off by (numpy, on the CPU)."""
import numpy as np

import softmax_oracle as so

H32 = so.H32


def entries(ids, z, keep):
    """Which entries take part: of a visible row, not -inf, the first with its id."""
    nq, n = keep.shape
    used = np.zeros(ids.shape, bool)
    for i in range(nq):
        have = set()
        for e, t in enumerate(ids[i]):
            if 0 <= t < n and keep[i, t] and z[i, e] != -np.inf and int(t) not in have:
                used[i, e] = True
                have.add(int(t))
    return used


def teacher(ids, z, tscale, rest, keep, used):
    """P [nq, n] over rows, R [nq]."""
    nq, n = keep.shape
    P, R = np.zeros((nq, n)), np.zeros(nq)
    for i in range(nq):
        t, w = ids[i][used[i]], z[i][used[i]].astype(np.float64) * tscale
        others = keep[i].sum() > len(t)
        if len(t) == 0:
            R[i] = 1.0 if rest and others else 0.0
            continue
        with np.errstate(all="ignore"):
            m = w.max()
            total = m + np.log(np.exp(w - m).sum())
            if rest and others and not total > 0:
                P[i, t], R[i] = np.exp(w), -np.expm1(total)
            else:
                P[i, t] = np.exp(w - total)
    return P, R


def forward(q, x, ids, z, scale, tscale, rest, allowed):
    nq, n = q.shape[0], x.shape[0]
    keep = so.bits(allowed, nq, n)
    f = so.forward(q, x, None, scale, allowed, 0)
    used = entries(ids, z, keep)
    P, R = teacher(ids, z, tscale, rest, keep, used)
    named = np.zeros((nq, n), bool)
    lp = np.zeros(ids.shape)
    for i in range(nq):
        named[i, ids[i][used[i]]] = True
        lp[i][used[i]] = f["lp"][i, ids[i][used[i]]]
    with np.errstate(all="ignore"):
        loss = np.where(P > 0, P * (np.log(P) - np.where(P > 0, f["lp"], 0.0)), 0.0).sum(1)
        other = np.where(keep & ~named, f["s"], -np.inf)
        m = other.max(1)
        some = np.isfinite(m)
        m = np.where(some, m, 0.0)
        lse_o = np.where(some, m + np.log(np.exp(other - m[:, None]).sum(1)), -np.inf)
        lr = np.where(some, lse_o - np.where(some, f["lse"], 0.0), -np.inf)
        if rest:
            loss += np.where((R > 0) & used.any(1), R * (np.log(R) - lr), 0.0)
    return dict(loss=loss, lse=f["lse"], logprobs=lp, rest=lr, P=P, R=R, used=used, named=named,
                keep=keep, s=f["s"], f=f)


def forward_bounds(o, es):
    """lse: as the log-softmax's (es the scores' bound).  An entry's score is a sum in
    64 bits of f32 sums over a lane's columns, four vectors at most: chains of 4 fused
    products a vector of 16 bits (2 of f32), the first product of which is exact (of f32
    rounded), and one addition, (d / 64 + 4 + 1) 2^-24 of the products' sizes or less for
    lanes that share d columns 256 a step, and 17 * 2^-24 at most: less than es, which
    counts (d / 16 + 1) 2^-22 of them (f32: 15 * 2^-22).  Its log probability is off by
    that and as the lse is; log r is the difference of two such sums, the loss
    lse - R lse_rest and the mean of the named scores; each rounded once."""
    e = so.forward_bounds(o["f"], es)[0]
    named = np.where(o["keep"], es, 0.0).max(1)
    fin = lambda v: np.where(np.isfinite(v), np.abs(v), 0.0)  # noqa: E731
    return dict(lse=e, logprobs=(e + named)[:, None] + H32 * fin(o["logprobs"]),
                rest=2 * e + H32 * fin(o["rest"]), loss=2 * e + named + H32 * fin(o["loss"]))


def backward(q, x, o, ids, lse, logprobs, rest, d_loss, scale):
    """(dq, dx, size of G's terms) around what the forward pass left."""
    keep, used, named = o["keep"], o["used"], o["named"]
    nq, n = keep.shape
    live = used.any(1) & (lse > -np.inf)
    u = np.where(live, d_loss, 0.0) * scale
    lr = np.zeros(nq) if rest is None else np.where(rest > -np.inf, rest, 0.0)
    r = np.ones(nq) if rest is None else np.exp(rest)
    with np.errstate(all="ignore"):
        e = np.exp(np.where(keep, o["s"], -np.inf) - np.where(live, lse + lr, 0.0)[:, None])
    c = u * (r - o["R"])
    G = np.where(named, 0.0, e * c[:, None])
    size = np.where(named, 0.0, e * np.abs(c)[:, None])
    for i in range(nq):
        t = ids[i][used[i]]
        p = np.exp(logprobs[i][used[i]])
        G[i, t] = u[i] * (p - o["P"][i, t])
        size[i, t] = np.abs(u[i]) * (p + o["P"][i, t])
    G, size = np.where(live[:, None], G, 0.0), np.where(live[:, None], size, 0.0)
    x0 = np.where(keep.any(0)[:, None], x, 0.0)
    q0 = np.where(keep.any(1)[:, None], q, 0.0)
    return G @ x0, G.T @ q0, size


def gradient_bounds(q, x, o, es, size, dtype, dq, dx, lse, rest, u):
    """As the log-softmax's.  Besides: the reference lse + log r is rounded to f32,
    and G is stored with scale * |d_loss| at 2^13 or above, however small it is
    itself (2^-33 of that, see softmax_oracle)."""
    ref = np.where(np.isfinite(lse), lse, 0.0)
    if rest is not None:
        ref = ref + np.where(np.isfinite(rest), rest, 0.0)
    es = es + (H32 * np.abs(ref) + 2.0 ** -23)[:, None]
    bq, bx = so.gradient_bounds(q, x, es, size, o["keep"], dtype, dq, dx)
    floor = np.abs(u).max() * 2.0 ** -33
    x0 = np.where(o["keep"].any(0)[:, None], np.abs(x), 0.0)
    q0 = np.where(o["keep"].any(1)[:, None], np.abs(q), 0.0)
    return bq + floor * x0.shape[0] * x0.max(), bx + floor * q0.shape[0] * q0.max()


# ---------------------------------------------------------------------------
# a beam search's step
# ---------------------------------------------------------------------------
def select(x, beam_scores, width, *, ids=None, scale=1.0, normalise=True, allowed=None, ended=None,
           end_id=-1):
    """x [groups, beams, n] float64.  (scores float64, parents, ids, ended)"""
    g, b, n = x.shape
    keep = so.bits(allowed, g * b, n).reshape(g, b, n)
    if ids is not None:
        keep = keep & (ids >= 0)
    out = (np.full((g, width), -np.inf), np.full((g, width), -1), np.full((g, width), -1),
           np.zeros((g, width), bool))
    scale = np.float64(np.float32(scale))
    for i in range(g):
        rows, bad = [], False
        for j in range(b):
            s = np.float64(beam_scores[i, j])
            bad |= not s < np.inf
            if s == -np.inf:
                continue
            if ended is not None and ended[i, j]:
                rows.append((np.array([s]), j, np.array([0]), True))
                continue
            cols = np.nonzero(keep[i, j] & ~(x[i, j] == -np.inf))[0]
            v = x[i, j, cols] * scale
            bad |= not (v < np.inf).all()
            if len(cols) and normalise and not bad:
                m = v.max()
                v = v - (m + np.log(np.exp(v - m).sum()))
            rows.append((s + v, j, cols, False))
        if bad:
            out[0][i] = np.nan
            continue
        if not rows:
            continue
        v = np.concatenate([r[0] for r in rows])
        p = np.concatenate([np.full(len(r[0]), r[1]) for r in rows])
        c = np.concatenate([r[2] for r in rows])
        d = np.concatenate([np.full(len(r[0]), r[3]) for r in rows])
        if len(v) > width:  # (all that equal the width-th stay)
            near = v >= np.partition(v, len(v) - width)[len(v) - width]
            v, p, c, d = v[near], p[near], c[near], d[near]
        order = np.lexsort((c, p, -v))[:width]
        m = len(order)
        name = c[order] if ids is None else ids[i, p[order], c[order]]
        name = np.where(d[order], end_id, name)
        out[0][i, :m], out[1][i, :m], out[2][i, :m] = v[order], p[order], name
        out[3][i, :m] = d[order] | (name == end_id)
    return out
