"""Log probabilities and their gradient at sizes of several passes over the
units, beside extreme values, and called at once: against 64-bit forms on the
GPU (too large for the oracle on the CPU), with its bounds."""
import numpy as np
import pytest

import softmax_oracle as so

pytestmark = pytest.mark.gpu

HALF = so.HALF


def _type(dtype):
    import torch
    return {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}[dtype]


def _score_off(q, x, scale, dtype):
    """softmax_oracle.score_bound on GPU tensors (f64)."""
    d = q.shape[1]
    u = 3 * 2.0 ** -22 + 12 * 2.0 ** -22 + (d / 32 + 8) * 2.0 ** -24 if dtype == "f32" else \
        (d / 16 + 1) * 2.0 ** -22
    return (q.abs() @ x.abs().T) * (scale * u) + 2.0 ** -23


def _held(dtype):
    return 3 * 2.0 ** -22 if dtype == "f32" else 2.0 ** -11


def _cut(dtype, k):
    return (12 + k / 64) * 2.0 ** -22 if dtype == "f32" else (k / 16 + 1) * 2.0 ** -22


def _lse(q, x, scale, step=128):
    """lse of every query in f32, from 64-bit scores."""
    import torch
    return torch.cat([torch.logsumexp(q[i:i + step] @ x.T * scale, 1)
                      for i in range(0, q.shape[0], step)]).float()


def _least_time(f, runs=8):
    """The least time of a call on the device, of several."""
    import torch
    best = float("inf")
    for _ in range(runs):
        ev = [torch.cuda.Event(enable_timing=True) for _ in range(2)]
        ev[0].record()
        f()
        ev[1].record()
        torch.cuda.synchronize()
        best = min(best, ev[0].elapsed_time(ev[1]))
    return best


@pytest.mark.parametrize("dtype,nq,n,dim", [
    ("bf16", 520, 50000, 64),    # one pass over the units
    ("bf16", 1000, 131072, 32),  # two
    ("f16", 2008, 131072, 32),   # four
    ("bf16", 2008, 200000, 16),  # two chunks of rows
    ("f16", 16, 70000, 24), ("bf16", 24, 300000, 8), ("f32", 1000, 131072, 32),
])
def test_the_last_query_keeps_its_given_row(dtype, nq, n, dim):
    """Numbers of queries that leave part of a warp's 32 rows without one: the
    first query's given row lies among the first columns, the last one's among
    the last, so the units that hold the latter begin after those that hold the
    former are done.  d_queries of the last query, d_rows of its given row and
    of row 0, and the same bits from workspaces that held other things."""
    import forgegpu as fg
    import torch
    gen = torch.Generator(device="cuda").manual_seed(nq + n)
    q = torch.randn(nq, dim, device="cuda", generator=gen).to(_type(dtype))
    x = torch.randn(n, dim, device="cuda", generator=gen).to(_type(dtype))
    t = torch.randint(0, n, (nq,), device="cuda", generator=gen)
    t[0], t[-1] = 77, n - 5
    t[t == 0] = 1
    scale = float(np.float32(1.0 / np.sqrt(dim)))
    Q, X = q.double(), x.double()
    lse = _lse(Q, X, scale)
    up = -torch.rand(nq, device="cuda", generator=gen) - 0.5
    probe = fg.logprobs_backward(q, x, t, lse, d_logprob=up, scale=scale)
    for fill in (0, 255):
        ws = torch.full((6 << 30,), fill, dtype=torch.uint8, device="cuda")
        again = fg.logprobs_backward(q, x, t, lse, d_logprob=up, scale=scale, workspace=ws)
        assert torch.equal(again[0], probe[0]) and torch.equal(again[1], probe[1])
        del ws
    g = up.double()
    L = lse.double()

    # d_queries of the last query
    s = X @ Q[-1] * scale
    p = torch.exp(s - L[-1])
    G = -p * g[-1]
    G[t[-1]] += g[-1]
    size = p * g[-1].abs()
    size[t[-1]] += g[-1].abs()
    top = (g.abs() * 2 * scale).max()
    floor = top * 2.0 ** -33
    es = _score_off(Q[-1:], X, scale, dtype)[0] + 2.0 ** -19 + _held(dtype)
    want = (G @ X) * scale
    b = ((size * (es + _cut(dtype, n))) @ X.abs()) * scale + HALF[dtype] * want.abs() + \
        floor * n * X.abs().max() + (2.0 ** -25 if dtype == "f16" else 0.0)
    off = (probe[0][-1].double() - want).abs()
    assert (off <= b).all(), (off / b).max()

    # d_rows of its given row, of the first query's and of row 0
    for j in (int(t[-1]), 77, 0):
        s = Q @ X[j] * scale
        p = torch.exp(s - L)
        hit = (t == j).double() * g
        G, size = hit - p * g, p * g.abs() + hit.abs()
        es = _score_off(Q, X[j:j + 1], scale, dtype)[:, 0] + 2.0 ** -19 + _held(dtype)
        want = (G @ Q) * scale
        b = ((size * (es + _cut(dtype, nq))) @ Q.abs()) * scale + HALF[dtype] * want.abs() + \
            floor * nq * Q.abs().max() + (2.0 ** -25 if dtype == "f16" else 0.0)
        off = (probe[1][j].double() - want).abs()
        assert (off <= b).all(), (j, (off / b).max())


@pytest.mark.parametrize("dtype,nq,dims", [("f32", 8, (2048, 1400)), ("bf16", 2, (2048, 64)),
                                           ("f32", 2, (16384, 9000))])
@pytest.mark.parametrize("backward", [False, True])
def test_host_threads_at_once(dtype, nq, dims, backward):
    """The same kernels, launched by four threads with two amounts of shared
    memory: the limit that one of them needs is not taken away by another
    between its setting and the launch."""
    import ctypes as C
    import threading

    import forgegpu as fg
    import torch
    if backward:
        dims = tuple(max(8, d // 2) for d in dims)
    L, ctx, n, reps = fg.lib(), fg.default_context().h, 64, 8000
    gen = torch.Generator(device="cuda").manual_seed(1)
    code = {"f32": 0, "bf16": 2}[dtype]
    keep, calls, want = [], [], []
    for i in range(4):
        d = dims[i % 2]
        s = torch.cuda.Stream()
        q = torch.randn(nq, d, device="cuda", generator=gen).to(_type(dtype))
        x = torch.randn(n, d, device="cuda", generator=gen).to(_type(dtype))
        t = torch.arange(nq, device="cuda")
        up = torch.rand(nq, device="cuda", generator=gen)
        ws = torch.empty(64 << 20, dtype=torch.uint8, device="cuda")
        r = fg.logprobs(q, x, t, scale=0.02)
        if backward:
            out = [torch.empty_like(q), torch.empty_like(x)]
            a = fg.LogprobGradArgs(
                dtype=code, queries=q.data_ptr(), nq=nq, ld_queries=d, rows=x.data_ptr(), n=n,
                ld_rows=d, dim=d, scale=0.02, targets=t.data_ptr(), lse=r.lse.data_ptr(),
                d_logprob=up.data_ptr(), d_queries=out[0].data_ptr(), ld_d_queries=d,
                d_rows=out[1].data_ptr(), ld_d_rows=d, workspace=ws.data_ptr(),
                workspace_bytes=ws.numel(), stream=s.cuda_stream)
            want.append(fg.logprobs_backward(q, x, t, r.lse, d_logprob=up, scale=0.02))
        else:
            out = [torch.empty(nq, device="cuda") for _ in range(2)]
            a = fg.LogprobArgs(
                dtype=code, queries=q.data_ptr(), nq=nq, ld_queries=d, rows=x.data_ptr(), n=n,
                ld_rows=d, dim=d, scale=0.02, targets=t.data_ptr(), logprob=out[0].data_ptr(),
                lse=out[1].data_ptr(), workspace=ws.data_ptr(), workspace_bytes=ws.numel(),
                stream=s.cuda_stream)
            want.append(r[:2])
        keep.append((q, x, t, up, ws, r, s, out))
        calls.append(a)
    torch.cuda.synchronize()
    f = L.fdb_logprobs_backward if backward else L.fdb_logprobs
    failed = []

    def run(a):
        for _ in range(reps):
            if f(ctx, C.byref(a)):
                failed.append(L.fdb_last_error())
                return

    threads = [threading.Thread(target=run, args=(a,)) for a in calls]
    for th in threads:
        th.start()
    for th in threads:
        th.join()
    torch.cuda.synchronize()
    assert not failed, failed
    for w, k in zip(want, keep):
        assert all(torch.equal(a, b) for a, b in zip(w, k[-1]))


def _gradient(q, x, t, scale, keep, lse, ent, up):
    """softmax_oracle.backward and the size of its terms on GPU tensors (f64)."""
    import torch
    s = q @ x.T * scale
    if keep is not None:
        s = s.masked_fill(~keep, -float("inf"))
    some = lse > -float("inf")
    lp = s - torch.where(some, lse, 0.0)[:, None]
    p = torch.where(some[:, None], lp.exp(), 0.0)
    lp = torch.where(p > 0, lp, 0.0)
    i = torch.arange(len(t), device="cuda")
    ok = (t >= 0) & some
    ok &= s[i, t.clamp_min(0)] > -float("inf")
    dlp, dl, dh = up
    g = torch.where(ok, dlp, 0.0)
    e = torch.where(some, ent, 0.0)
    G = p * ((dl - g)[:, None] - dh[:, None] * (lp + e[:, None]))
    size = p * ((dl.abs() + g.abs())[:, None] + dh.abs()[:, None] * (lp.abs() + e.abs()[:, None] + 1))
    G[i[ok], t[ok]] += g[ok]
    size[i[ok], t[ok]] += g[ok].abs()
    return G * scale, size * scale


@pytest.mark.parametrize("dtype,nq,n,dim,mask", [
    ("f32", 64, 20000, 64, False), ("f32", 300, 3001, 33, True), ("f32", 17, 500, 200, False),
    ("bf16", 64, 20000, 64, False), ("bf16", 130, 1500, 129, True),
])
@pytest.mark.parametrize("which", ["d_logprob", "d_lse", "all"])
def test_upstream_gradients_of_many_sizes(dtype, nq, n, dim, mask, which):
    """Upstream gradients from 1e-8 to 1 of the largest: each query's d_queries
    within the bound that its own upstream gradient gives.  G is held down to
    2^-25 with its bound at 2^13 or above, rows down to 2^-4 of the largest
    scale enlarge that: 2^-33 of the query's own largest for each row."""
    import forgegpu as fg
    import torch
    gen = torch.Generator(device="cuda").manual_seed(nq)
    q = torch.randn(nq, dim, device="cuda", generator=gen).to(_type(dtype))
    x = torch.randn(n, dim, device="cuda", generator=gen).to(_type(dtype))
    t = torch.randint(-1, n, (nq,), device="cuda", generator=gen)
    keep = words = None
    if mask:
        keep = torch.rand(nq, n, device="cuda", generator=gen) < 0.4
        keep[3] = False
        words = torch.from_numpy(so.words(keep.cpu().numpy())).cuda()
    scale = float(np.float32(1.5 / np.sqrt(dim)))
    r = fg.logprobs(q, x, t, scale=scale, allowed=words)
    w = 10.0 ** -(torch.arange(nq, device="cuda") % 9).float()
    up = torch.randn(3, nq, device="cuda", generator=gen) * w
    if which != "all":
        up[[i for i, k in enumerate(("d_logprob", "d_lse", "d_entropy")) if k != which]] = 0.0
    dq, dx = fg.logprobs_backward(q, x, t, r.lse, r.entropy, d_logprob=up[0], d_lse=up[1],
                                  d_entropy=up[2], scale=scale, allowed=words)
    Q, X = q.double(), x.double()
    G, size = _gradient(Q, X, t, scale, keep, r.lse.double(), r.entropy.double(), up.double())
    e = size * (_score_off(Q, X, scale, dtype) + 2.0 ** -19 + _held(dtype))
    own = size.amax(1)
    want = G @ X
    b = e @ X.abs() + size @ X.abs() * _cut(dtype, n) + HALF[dtype] * want.abs() + \
        own[:, None] * 2.0 ** -33 * n * X.abs().max()
    off = (dq.double() - want).abs()
    assert (off <= b + 1e-35).all(), (off / (b + 1e-35)).max()
    want = G.T @ Q
    b = e.T @ Q.abs() + size.T @ Q.abs() * _cut(dtype, nq) + HALF[dtype] * want.abs() + \
        own.max() * 2.0 ** -33 * nq * Q.abs().max()
    off = (dx.double() - want).abs()
    assert (off <= b + 1e-35).all(), (off / (b + 1e-35)).max()
    # what another query's upstream gradient is does not change a bit
    up2 = up.clone()
    up2[:, 0] *= 2.0 ** 20
    dq2, _ = fg.logprobs_backward(q, x, t, r.lse, r.entropy, d_logprob=up2[0], d_lse=up2[1],
                                  d_entropy=up2[2], scale=scale, allowed=words)
    assert torch.equal(dq[1:], dq2[1:])


@pytest.mark.parametrize("dtype,shift", [("f32", 100), ("f32", -100), ("bf16", 90), ("bf16", -90)])
def test_gradients_of_very_large_and_small_operands(dtype, shift):
    """Rows of size 2^shift and queries of 2^-shift: the scores are those of
    both at 1, the gradients are scaled by the powers of two."""
    import forgegpu as fg
    import torch
    gen = torch.Generator(device="cuda").manual_seed(3)
    q = torch.randn(40, 48, device="cuda", generator=gen).to(_type(dtype))
    x = torch.randn(700, 48, device="cuda", generator=gen).to(_type(dtype))
    t = torch.randint(-1, 700, (40,), device="cuda", generator=gen)
    r = fg.logprobs(q, x, t, scale=0.2)
    up = torch.randn(40, device="cuda", generator=gen)
    dq, dx = fg.logprobs_backward(q, x, t, r.lse, d_logprob=up, scale=0.2)
    two = 2.0 ** shift
    eq, ex = fg.logprobs_backward(q / two, x * two, t, r.lse, d_logprob=up, scale=0.2)
    assert torch.equal(eq, dq * two) and torch.equal(ex, dx / two)


@pytest.mark.parametrize("dtype,nq,dim", [("f32", 1, 768), ("f32", 300, 96), ("bf16", 300, 128),
                                          ("f16", 2, 256)])
@pytest.mark.parametrize("bad", [float("inf"), 6e4])
@pytest.mark.parametrize("targets", [False, True])
@pytest.mark.parametrize("filters", ["one", "each"])
def test_a_row_that_is_not_seen_takes_no_part(dtype, nq, dim, bad, targets, filters):
    """A masked row, the first one or the given one, that holds an infinity or
    something large: the same bits, and no more work, than beside zeros (the
    alternatives of every query would be looked for in all rows if it counted
    for the size of the scores' errors: some hundred times the work)."""
    import forgegpu as fg
    import torch
    n = 200000
    gen = torch.Generator(device="cuda").manual_seed(5)
    q = torch.randn(nq, dim, device="cuda", generator=gen).to(_type(dtype))
    x = torch.randn(n, dim, device="cuda", generator=gen).to(_type(dtype))
    keep = torch.ones(1, n, dtype=torch.bool)
    keep[0, :2] = False
    words = torch.from_numpy(so.words(keep.numpy())).cuda()
    if filters == "each":
        words = words.repeat(nq, 1)
    t = torch.ones(nq, dtype=torch.int64, device="cuda") if targets else None
    out, times = [], []
    for value in (0.0, bad):
        x[:2] = value
        out.append(fg.logprobs(q, x, t, scale=0.1, allowed=words, k=10))
        times.append(_least_time(lambda: fg.logprobs(q, x, t, scale=0.1, allowed=words, k=10)))
    assert all(torch.equal(a, b) for a, b in zip(*out))
    assert times[1] < 3 * times[0], times


@pytest.mark.parametrize("nq,seed", [(1, 0), (1, 1), (1, 2), (1, 3), (8, 0), (16, 0), (40, 0),
                                     (300, 0)])
@pytest.mark.parametrize("dim", [64, 256])
def test_a_large_row_nearly_at_right_angles(nq, seed, dim):
    """Each query sees one row a million times the others', whose true score is
    just above their best; its 32-bit score may be far below all of them."""
    import forgegpu as fg
    import torch
    rng = np.random.default_rng(100 * nq + seed)
    n = 20000
    q = rng.standard_normal((nq, dim)).astype(np.float32)
    q[:, 0] = np.abs(q[:, 0]) + 1
    x = (rng.standard_normal((n + nq, dim)) / np.sqrt(dim)).astype(np.float32)
    q64 = q.astype(np.float64)
    best = (q64 @ x[:n].astype(np.float64).T).max(1)
    for i in range(nq):
        g = (1e6 * rng.standard_normal(dim)).astype(np.float32)
        g[0] = 0
        c = 1 + np.argmax(np.abs(q[i, 1:]))  # two corrections: most of it, then the rest
        g[c] -= np.float32((q64[i] @ g.astype(np.float64)) / q64[i, c])
        g[0] = np.float32((best[i] + 0.01 - q64[i] @ g.astype(np.float64)) / q64[i, 0])
        x[n + i] = g
    keep = np.ones((nq, n + nq), bool)
    keep[:, n:] = np.eye(nq, dtype=bool)
    s = np.where(keep, q64 @ x.astype(np.float64).T, -np.inf)
    s[np.arange(nq), n + np.arange(nq)] = [q64[i] @ x[n + i].astype(np.float64) for i in range(nq)]
    assert (np.abs(s[np.arange(nq), n + np.arange(nq)] - best - 0.01) < 1e-3).all()
    want = np.argsort(-s, 1)[:, :5]
    Q, X = torch.from_numpy(q).cuda(), torch.from_numpy(x).cuda()
    A = torch.from_numpy(so.words(keep)).cuda()
    r = fg.logprobs(Q, X, scale=1.0, allowed=A, k=5)
    assert np.array_equal(r.top_ids.cpu().numpy(), want)


@pytest.mark.parametrize("dtype,nq", [("f32", 2), ("f32", 7), ("bf16", 3), ("f32", 40)])
def test_a_product_out_of_range_that_is_masked(dtype, nq):
    """A large row that the last query may not see, and whose product with it is
    beyond f32: the others' gradients are those beside a query of zeros."""
    import forgegpu as fg
    import torch
    gen = torch.Generator(device="cuda").manual_seed(nq)
    q = torch.randn(nq, 40, device="cuda", generator=gen).to(_type(dtype))
    x = torch.randn(90, 40, device="cuda", generator=gen).to(_type(dtype))
    q[-1] *= 1e15
    x[50] *= 1e25
    scale = 1e-25
    keep = torch.ones(nq, 90, dtype=torch.bool)
    keep[-1, 50] = False
    words = torch.from_numpy(so.words(keep.numpy())).cuda()
    t = torch.full((nq,), 50, device="cuda")
    t[-1] = 3
    up = torch.rand(nq, device="cuda", generator=gen)
    got = []
    for last in (q[-1].clone(), torch.zeros_like(q[-1])):
        q[-1] = last
        r = fg.logprobs(q, x, t, scale=scale, allowed=words)
        dq, dx = fg.logprobs_backward(q, x, t, r.lse, d_logprob=up, scale=scale, allowed=words)
        got.append((r.lse[:-1], dq[:-1], dx[50]))
    assert got[0][1].float().abs().max() > 1e-3
    assert all(torch.isfinite(a.float()).all() for a in got[0])
    if nq <= 8:
        assert all(torch.equal(a, b) for a, b in zip(*got))
    else:  # (d_rows' scale is that of the largest query: its terms are 1e-15 of it)
        assert all(torch.equal(a, b) for a, b in zip(got[0][:2], got[1][:2]))


@pytest.mark.parametrize("dtype,size", [("f16", 200.0), ("bf16", 600.0)])
@pytest.mark.parametrize("nq,n,dim", [(20, 300, 16384), (140, 900, 5000), (33, 700, 2049)])
def test_long_rows_of_one_sign(dtype, size, nq, n, dim):
    """Scores of hundreds that are sums of thousands of terms of one sign: the
    tensor core's additions cut them all the same way, by up to 2^-22 of a sum
    for each of its 16-wide steps, at most 17 in a block of 256; the blocks are
    joined in f32.  The gradient's scores are those that the forward pass
    summed."""
    import forgegpu as fg
    import torch
    gen = torch.Generator(device="cuda").manual_seed(dim)
    q = (torch.rand(nq, dim, device="cuda", generator=gen) + 0.5).to(_type(dtype))
    x = (torch.rand(n, dim, device="cuda", generator=gen) + 0.5).to(_type(dtype))
    scale = float(np.float32(size / dim))
    Q, X = q.double(), x.double()
    lse = torch.logsumexp(Q @ X.T * scale, 1).float()
    up = torch.ones(nq, device="cuda")
    dq, dx = fg.logprobs_backward(q, x, None, lse, d_lse=up, scale=scale)
    P = torch.exp(Q @ X.T * scale - lse.double()[:, None])
    es = (Q @ X.T * scale) * (17 * 2.0 ** -22 + (dim / 256 + 2) * 2.0 ** -24)
    es = es + 2 * size * 2.0 ** -24  # (the score's factor, and t - lse, rounded to f32)
    e = P * (es + 2.0 ** -19 + _held(dtype)) * scale
    for got, want, b in ((dq, P @ X * scale, e @ X), (dx, P.T @ Q * scale, e.T @ Q)):
        k = n if got is dq else nq
        b = b * (1 + _cut(dtype, k)) + want * _cut(dtype, k) + HALF[dtype] * want + 2.0 ** -25
        off = (got.double() - want).abs()
        assert (off <= b).all(), (off / b).max()


@pytest.mark.parametrize("dtype,nq", [("f32", 4), ("f32", 300), ("bf16", 2), ("bf16", 300)])
def test_an_infinity_costs_its_queries_only(dtype, nq):
    """One query sees a row with an infinity: the others' bits stay, and they are
    not looked for in all rows (some hundred times the work)."""
    import forgegpu as fg
    import torch
    n = 200000
    gen = torch.Generator(device="cuda").manual_seed(6)
    q = torch.randn(nq, 96, device="cuda", generator=gen).to(_type(dtype))
    x = torch.randn(n, 96, device="cuda", generator=gen).to(_type(dtype))
    keep = torch.ones(nq, n, dtype=torch.bool)
    keep[1:, 70000] = False
    words = torch.from_numpy(so.words(keep.numpy())).cuda()
    out, times = [], []
    for value in (0.0, float("inf")):
        x[70000] = value
        out.append(fg.logprobs(q, x, scale=0.1, allowed=words, k=10))
        times.append(_least_time(lambda: fg.logprobs(q, x, scale=0.1, allowed=words, k=10)))
    assert torch.isnan(out[1].lse[0]) and (out[1].top_ids[0] == -1).all()
    assert all(torch.equal(a[1:], b[1:]) for a, b in zip(*out))
    assert times[1] < 3 * times[0], times


@pytest.mark.parametrize("nq", [5, 40])
@pytest.mark.parametrize("shift", [-90, -60, 60, 115])
def test_upstream_gradients_far_from_one(nq, shift):
    """Upstream gradients times a power of two: the gradients times it, bit for
    bit, up to the ends of f32's range."""
    import forgegpu as fg
    import torch
    gen = torch.Generator(device="cuda").manual_seed(8)
    q = torch.randn(nq, 64, device="cuda", generator=gen)
    x = torch.randn(800, 64, device="cuda", generator=gen)
    t = torch.randint(0, 800, (nq,), device="cuda", generator=gen)
    r = fg.logprobs(q, x, t, scale=0.2)
    up = torch.rand(nq, device="cuda", generator=gen) + 0.1
    dq, dx = fg.logprobs_backward(q, x, t, r.lse, d_logprob=up, scale=0.2)
    two = 2.0 ** shift
    eq, ex = fg.logprobs_backward(q, x, t, r.lse, d_logprob=up * two, scale=0.2)
    assert torch.equal(eq, dq * two) and torch.equal(ex, dx * two)
