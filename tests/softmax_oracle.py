"""Plain 64-bit forms of the softmax-over-rows operators and of AdamW, with
bounds of what the kernels may be off by (numpy, on the CPU)."""
import numpy as np

H32 = 2.0 ** -24   # half a step of f32, relative
HALF = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}


def products(q, x):
    """q @ x.T with every product summed in the same order, so that equal rows
    have equal scores (a library's product sums in blocks that depend on the
    row's place)."""
    out = np.zeros((q.shape[0], x.shape[0]))
    for c in range(q.shape[1]):
        out += q[:, c, None] * x[None, :, c]
    return out


def bits(allowed, nq, n):
    """int32 words [rows, words] (or None) -> truth values [nq, n]."""
    if allowed is None:
        return np.ones((nq, n), bool)
    a = np.atleast_2d(allowed).view(np.uint32)
    j = np.arange(n)
    keep = (a[:, j // 32] >> (j % 32).astype(np.uint32)) & 1
    return np.broadcast_to(keep.astype(bool), (nq, n))


def words(keep):
    """Truth values [rows, n] -> int32 words [rows, (n + 31) // 32]."""
    rows, n = keep.shape
    w = np.zeros((rows, (n + 31) // 32 * 32), np.uint64)
    w[:, :n] = keep
    w = (w.reshape(rows, -1, 32) << np.arange(32, dtype=np.uint64)).sum(2)
    return w.astype(np.uint32).view(np.int32)


def score_bound(q, x, scale, dtype):
    """What a score may be off by.  Each sum of products is cut once per
    16-wide step of the tensor core, by up to 2^-23 of the terms' sizes, and as
    much again for the alignment of the 16 terms; f32 operands are held in 22
    bits (2^-22 each, and 2^-22 for the product of the rests, left out), in
    sums of 12 such steps joined by f32 additions (the small kernel's f32
    sums of at most dim / 32 + 8 terms lie below that)."""
    d = q.shape[1]
    size = np.abs(np.nan_to_num(q, posinf=0, neginf=0)) @ \
        np.abs(np.nan_to_num(x, posinf=0, neginf=0)).T * scale
    if dtype == "f32":
        u = 3 * 2.0 ** -22 + 12 * 2.0 ** -22 + (d / 32 + 8) * 2.0 ** -24
    else:
        u = (d / 16 + 1) * 2.0 ** -22
    return size * u + 2.0 ** -23  # (the factor scale * log2 e, rounded once)


def forward(q, x, targets, scale, allowed, k):
    """q, x float64.  Outputs and the scores (disallowed at -inf)."""
    nq, n = q.shape[0], x.shape[0]
    keep = bits(allowed, nq, n)
    with np.errstate(all="ignore"):
        s = np.where(keep, products(q, np.where(keep.any(0)[:, None], x, 0.0)) * scale, -np.inf)
        m = s.max(1)
        some = keep.any(1)
        z = s - np.where(some, m, 0.0)[:, None]
        e = np.where(keep, np.exp(z), 0.0)
        lse = np.where(some, m + np.log(e.sum(1)), -np.inf)
        lp = np.where(keep, s - np.where(some, lse, 0.0)[:, None], -np.inf)
        p = np.where(keep, np.exp(lp), 0.0)
        ent = -(p * np.where(p > 0, lp, 0.0)).sum(1)
    t = np.full(nq, -1) if targets is None else targets
    given = (t >= 0) & (t < n)
    at = lp[np.arange(nq), np.where(given, t, 0)]
    at = np.where(keep[np.arange(nq), np.where(given, t, 0)], at, -np.inf)
    logprob = np.where(given, at, 0.0)
    ids = np.full((nq, k), -1)
    top = np.full((nq, k), -np.inf)
    for i in range(nq):
        order = np.lexsort((np.arange(n), -s[i]))
        order = order[keep[i][order]][:k]
        ids[i, :len(order)] = order
        top[i, :len(order)] = lp[i, order]
    return dict(logprob=logprob, lse=lse, entropy=ent, top_ids=ids, top_logprobs=top, s=s, p=p,
                lp=lp, keep=keep)


def forward_bounds(f, es, entropy_terms=True):
    """(lse, logprob, entropy) bounds from a score bound es [nq, n]: lse moves
    by at most the largest shift of a score that counts; 2^-20 covers ex2 (2
    units in the last place) and the f32 sums of the exponentials (up to a few
    hundred partial sums of 32 each, relative to a sum of positive terms).
    The entropy's derivative along the shifts is -sum p (lp + H) ds."""
    p, lp = f["p"], np.where(f["p"] > 0, f["lp"], 0.0)
    e = np.where(f["keep"], es, 0.0).max(1) + 2.0 ** -20
    h = np.nan_to_num(f["entropy"])
    ent = (p * np.abs(lp + h[:, None])).sum(1) * e + (1 + np.abs(h)) * 2.0 ** -19
    fin = lambda v: np.where(np.isfinite(v), np.abs(v), 0.0)  # noqa: E731
    return e + 2 * H32 * fin(f["lse"]), e + 2 * H32 * fin(f["logprob"]), ent


def backward(q, x, targets, lse, entropy, d_logprob, d_lse, d_entropy, scale, allowed):
    """(dq, dx, G, size of G's terms) from the definition, 64 bits."""
    nq, n = q.shape[0], x.shape[0]
    keep = bits(allowed, nq, n)
    with np.errstate(all="ignore"):
        s = np.where(keep, products(q, np.where(keep.any(0)[:, None], x, 0.0)) * scale, -np.inf)
        lp = np.where(keep & np.isfinite(lse)[:, None], s - np.where(np.isfinite(lse), lse, 0.0)
                      [:, None], -np.inf)
        p = np.exp(lp)
    lp = np.where(p > 0, lp, 0.0)
    t = np.full(nq, -1) if targets is None else targets
    ok = (t >= 0) & (t < n) & np.isfinite(lse)
    ok &= keep[np.arange(nq), np.where(ok, t, 0)]
    g = np.where(ok, d_logprob, 0.0)
    h = np.where(np.isfinite(lse), d_entropy, 0.0)
    ent = np.where(np.isfinite(lse), entropy, 0.0)
    G = p * ((d_lse - g)[:, None] - h[:, None] * (lp + ent[:, None]))
    size = p * ((np.abs(d_lse) + np.abs(g))[:, None] + np.abs(h)[:, None] *
                (np.abs(lp) + np.abs(ent)[:, None] + 1))
    i = np.arange(nq)[ok]
    G[i, t[ok]] += g[ok]
    size[i, t[ok]] += np.abs(g[ok])
    x0 = np.where(keep.any(0)[:, None], x, 0.0)
    q0 = np.where(keep.any(1)[:, None], q, 0.0)
    return G @ x0 * scale, G.T @ q0 * scale, G * scale, size * scale


def gradient_bounds(q, x, es, size, keep, dtype, dq, dx):
    """Elementwise: the scores' error moves p by that much of itself (and
    2^-19 for ex2 and the exponent's roundings), G is held in 11 bits (f32: 22),
    a product's sum of K terms is cut K / 16 times by up to 2^-22 of its terms
    (f32: sums of 12 steps, joined in f32), and the result is rounded once: by
    half a step of its value, or, in f16 below 2^-14, where the steps are
    2^-24 whatever the value, by 2^-25."""
    x0 = np.where(keep.any(0)[:, None], np.abs(x), 0.0)
    q0 = np.where(keep.any(1)[:, None], np.abs(q), 0.0)
    held = 3 * 2.0 ** -22 if dtype == "f32" else 2.0 ** -11

    def cut(k):
        return (12 + k / 64) * 2.0 ** -22 if dtype == "f32" else (k / 16 + 1) * 2.0 ** -22

    e = size * (np.where(keep, es, 0.0) + 2.0 ** -19 + held)
    # G is stored as fp16 with its largest value at 2^13 or above, so down to
    # 2^-25 absolutely (half of fp16's least step): 2^-38 of the largest; rows
    # and queries down to 2^-4 of the largest scale enlarge that by up to 2^4
    # each, and one of the two factors comes back with the small row itself:
    # 2^-33 with the factor 2 between a row's scale and its largest element.
    top = size.max() if size.size else 0.0
    sub = 2.0 ** -25 if dtype == "f16" else 0.0
    floor = top * 2.0 ** -33
    bq = e @ x0 + size @ x0 * cut(x.shape[0]) + HALF[dtype] * np.abs(dq) + floor * x0.shape[0] * x0.max() + sub
    bx = e.T @ q0 + size.T @ q0 * cut(q.shape[0]) + HALF[dtype] * np.abs(dx) + \
        floor * q0.shape[0] * q0.max() + sub
    return bq, bx


# ---------------------------------------------------------------------------
# AdamW, every operation in f32 in the documented order
# ---------------------------------------------------------------------------
f4 = np.float32


def mix(h):
    h = np.asarray(h, np.uint64)
    m = np.uint64(0xFFFFFFFF)
    h = ((h ^ (h >> np.uint64(16))) * np.uint64(0x7FEB352D)) & m
    h = ((h ^ (h >> np.uint64(15))) * np.uint64(0x846CA68B)) & m
    return h ^ (h >> np.uint64(16))


def values8(m, ms, v, vs):
    n = m.size
    b = np.arange(n) // 256
    c = m.astype(f4)
    r = v.astype(f4)
    r2 = r * r
    return (c * np.abs(c)) * (ms * f4(1 / 127 ** 2))[b], (r2 * r2) * (vs * f4(1 / 255 ** 4))[b]


def adamw(p, g, m, v, *, lr, step, betas, eps, wd, grad_scale=1.0):
    """f32 arrays -> (p before its last rounding, m, v)."""
    b1, b2 = betas
    g = g * f4(grad_scale)
    m = m * f4(b1) + g * f4(1 - b1)
    v = v * f4(b2) + (g * g) * f4(1 - b2)
    with np.errstate(all="ignore"):
        den = np.sqrt(v) * f4(1 / np.sqrt(1 - b2 ** step)) + f4(eps)
        p = p * f4(1 - lr * wd) - (m / den) * f4(lr / (1 - b1 ** step))
    return p, m, v


def codes8(m, v, *, seed, step, ordinal):
    """f32 moments -> codes and scales."""
    n = m.size
    nb = (n + 255) // 256
    pad = nb * 256 - n
    M = np.pad(m, (0, pad)).reshape(nb, 256)
    V = np.pad(v, (0, pad)).reshape(nb, 256)
    sm, sv = np.abs(M).max(1), V.max(1)
    least = f4(2.0 ** -90)
    i = np.arange(nb * 256, dtype=np.uint64).reshape(nb, 256)
    salt = mix((seed + (step << 16) + ordinal) & 0xFFFFFFFF)
    h = mix(i ^ salt)
    um = (h >> np.uint64(8)).astype(f4) * f4(2.0 ** -24)
    uv = (mix(h ^ np.uint64(0x5BD1E995)) >> np.uint64(8)).astype(f4) * f4(2.0 ** -24)
    with np.errstate(all="ignore"):
        y = np.abs(M) * np.where(sm > least, f4(127 ** 2) / sm, f4(0))[:, None]
        c = np.floor(np.sqrt(y))
        lo, hi = c * c, (c + f4(1)) * (c + f4(1))
        c = np.minimum(c + (um < (y - lo) / (hi - lo)), f4(127))
        cm = (c * np.sign(M)).astype(np.int8)
        y = V * np.where(sv > least, f4(255 ** 4) / sv, f4(0))[:, None]
        c = np.floor(np.sqrt(np.sqrt(y)))
        lo, hi = c * c, (c + f4(1)) * (c + f4(1))
        lo, hi = lo * lo, hi * hi
        c = np.minimum(c + (uv < (y - lo) / (hi - lo)), f4(255))
        c = np.where((y > 0) & (c < 1), f4(1), c)
        cv = c.astype(np.uint8)
    z = f4(0)
    return (cm.reshape(-1)[:n], np.where(sm < least, z, sm), cv.reshape(-1)[:n],
            np.where(sv < least, z, sv))
