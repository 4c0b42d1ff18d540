"""Log probabilities under a softmax over rows and their gradient, against the
64-bit definitions, elementwise within the bounds of softmax_oracle."""
import numpy as np
import pytest

import softmax_oracle as so

pytestmark = pytest.mark.gpu


def _types():
    import torch
    return {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def make(dtype, nq, n, dim, mask, pad=0, shift=0, seed=0, near=2.0):
    """Operands on the GPU (rows `pad` wider than dim, the first element `shift`
    past an aligned address) and the same values in 64 bits."""
    import torch
    rng = np.random.default_rng(seed)
    dt = _types()[dtype]

    def put(a):
        r, d = a.shape
        buf = torch.full((shift + r * (d + pad),), float("nan"), dtype=dt, device="cuda")
        view = buf[shift:].view(r, d + pad)[:, :d]
        view.copy_(torch.from_numpy(a).to(dt))
        return view

    x = rng.standard_normal((n, dim))
    t = rng.integers(-1, n, nq)
    q = rng.standard_normal((nq, dim)) + near * rng.random((nq, 1)) * x[np.maximum(t, 0)] / \
        np.sqrt(dim)
    Q, X = put(q), put(x)
    al = None
    if mask != "none":
        rows = nq if mask == "each" else 1
        keep = rng.random((rows, n)) < rng.choice([0.02, 0.5, 0.97], (rows, 1))
        if rows > 2:
            keep[rows // 2] = False
        if mask == "one":
            keep[0, 0] = True
        al = so.words(keep)
    T = torch.from_numpy(t).cuda()
    A = None if al is None else torch.from_numpy(al).cuda()
    return Q, X, T, A, Q.double().cpu().numpy(), X.double().cpu().numpy(), t, al


def check_forward(r, f, es, k, scores_exact=True):
    ble, bl, bh = so.forward_bounds(f, es)
    for name, bound in (("lse", ble), ("logprob", bl), ("entropy", bh)):
        got, want = getattr(r, name).double().cpu().numpy(), f[name]
        inf = ~np.isfinite(want)
        assert np.array_equal(got[inf], want[inf]), name
        off = np.abs(got[~inf] - want[~inf])
        assert (off <= bound[~inf]).all(), (name, (off / bound[~inf]).max())
    if k:
        assert np.array_equal(r.top_ids.cpu().numpy(), f["top_ids"])
        got, want = r.top_logprobs.double().cpu().numpy(), f["top_logprobs"]
        inf = ~np.isfinite(want)
        assert np.array_equal(got[inf], want[inf])
        off = np.where(inf, 0, np.abs(got - np.where(inf, 0, want)))
        off = np.where(inf, 0, off)
        assert (off <= ble[:, None] + 2 * so.H32 * np.where(inf, 0, np.abs(want))).all()


SHAPES = [
    # dtype, nq, n, dim, mask, pad, shift, k
    ("f32", 1, 1, 1, "none", 0, 0, 1), ("f32", 1, 31, 8, "none", 0, 0, 5),
    ("f32", 2, 33, 33, "one", 1, 1, 5), ("f32", 3, 1000, 64, "each", 0, 0, 10),
    ("f32", 8, 2049, 130, "each", 3, 0, 64), ("f32", 9, 700, 65, "none", 0, 1, 0),
    ("f32", 16, 5003, 100, "one", 4, 0, 7), ("f32", 17, 255, 96, "none", 0, 0, 5),
    ("f32", 17, 7, 33, "none", 0, 0, 10), ("f32", 128, 257, 64, "each", 1, 1, 3),
    ("f32", 129, 1000, 520, "none", 0, 0, 20), ("f32", 300, 4001, 200, "each", 2, 0, 10),
    ("f32", 40, 3000, 1030, "one", 0, 0, 1),
    ("bf16", 1, 1, 1, "none", 0, 0, 2), ("bf16", 1, 5003, 96, "one", 0, 0, 10),
    ("bf16", 2, 256, 64, "none", 0, 0, 0), ("bf16", 33, 511, 65, "each", 0, 0, 5),
    ("bf16", 128, 300, 72, "none", 8, 8, 5), ("bf16", 129, 1027, 200, "each", 3, 1, 64),
    ("bf16", 260, 5000, 768, "none", 0, 0, 20), ("bf16", 50, 2000, 1100, "none", 0, 0, 10),
    ("f16", 1, 100, 7, "none", 0, 0, 5), ("f16", 20, 32, 128, "one", 0, 0, 32),
    ("f16", 140, 3001, 129, "each", 0, 0, 11), ("f16", 65, 999, 256, "none", 8, 0, 0),
]


@pytest.mark.parametrize("dtype,nq,n,dim,mask,pad,shift,k", SHAPES)
def test_forward(dtype, nq, n, dim, mask, pad, shift, k):
    import forgegpu as fg
    Q, X, T, A, q, x, t, al = make(dtype, nq, n, dim, mask, pad, shift, seed=nq * 7 + n)
    scale = 2.0 / np.sqrt(dim)
    r = fg.logprobs(Q, X, T, scale=scale, allowed=A, k=k)
    f = so.forward(q, x, t, np.float64(np.float32(scale)), al, k)
    check_forward(r, f, so.score_bound(q, x, scale, dtype), k)


@pytest.mark.parametrize("dtype,nq,n,dim,mask,pad,shift", [
    ("f32", 1, 1, 1, "none", 0, 0), ("f32", 2, 33, 40, "one", 1, 1), ("f32", 5, 300, 8, "each", 0, 0),
    ("f32", 128, 256, 64, "none", 0, 0), ("f32", 129, 513, 65, "each", 0, 0),
    ("f32", 300, 1001, 200, "each", 3, 1), ("f32", 700, 90, 77, "none", 0, 0),
    ("f32", 40, 2000, 520, "one", 0, 0),
    ("bf16", 1, 31, 7, "none", 0, 0), ("bf16", 130, 257, 64, "each", 0, 0),
    ("bf16", 300, 1001, 200, "one", 3, 1), ("bf16", 64, 3000, 768, "none", 0, 0),
    ("bf16", 1000, 128, 300, "none", 8, 8),
    ("f16", 2, 64, 64, "none", 0, 0), ("f16", 150, 700, 129, "each", 1, 0),
])
def test_backward(dtype, nq, n, dim, mask, pad, shift):
    import forgegpu as fg
    import torch
    Q, X, T, A, q, x, t, al = make(dtype, nq, n, dim, mask, pad, shift, seed=nq + n)
    scale = np.float64(np.float32(2.0 / np.sqrt(dim)))
    f = so.forward(q, x, t, scale, al, 0)
    rng = np.random.default_rng(3)
    lse, ent = f["lse"].astype(np.float32), f["entropy"].astype(np.float32)
    up = rng.standard_normal((3, nq)).astype(np.float32) / nq
    dev = [torch.from_numpy(a).cuda() for a in (lse, ent, *up)]
    got = fg.logprobs_backward(Q, X, T, dev[0], dev[1], d_logprob=dev[2], d_lse=dev[3],
                               d_entropy=dev[4], scale=float(scale), allowed=A)
    args = [a.astype(np.float64) for a in (lse, ent, *up)]
    dq, dx, _, size = so.backward(q, x, t, *args, scale, al)
    es = so.score_bound(q, x, scale, dtype)
    bq, bx = so.gradient_bounds(q, x, es, size, f["keep"], dtype, dq, dx)
    for name, g, w, b in (("d_queries", got[0], dq, bq), ("d_rows", got[1], dx, bx)):
        assert g.dtype == Q.dtype and g.shape == w.shape
        off = np.abs(g.double().cpu().numpy() - w)
        assert (off <= b + 1e-30).all(), (name, (off / (b + 1e-30)).max())


def test_backward_parts_and_no_upstream():
    """A gradient that is not asked for is left out, a missing upstream is 0,
    and no upstream at all gives zeros."""
    import forgegpu as fg
    import torch
    Q, X, T, A, q, x, t, al = make("f32", 50, 300, 32, "none")
    r = fg.logprobs(Q, X, T, scale=0.3)
    g = torch.randn(50, device="cuda")
    a = fg.logprobs_backward(Q, X, T, r.lse, d_logprob=g, scale=0.3)
    b = fg.logprobs_backward(Q, X, T, r.lse, r.entropy, d_logprob=g, d_lse=torch.zeros_like(g),
                             d_entropy=torch.zeros_like(g), scale=0.3)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    c = fg.logprobs_backward(Q, X, T, r.lse, d_logprob=g, scale=0.3, need_rows=False)
    d = fg.logprobs_backward(Q, X, T, r.lse, d_logprob=g, scale=0.3, need_queries=False)
    assert c[1] is None and d[0] is None
    assert torch.equal(a[0], c[0]) and torch.equal(a[1], d[1])
    z = fg.logprobs_backward(Q, X, T, r.lse, scale=0.3)
    assert not z[0].any() and not z[1].any()


def test_backward_without_queries_zeroes_the_rows_gradient():
    import forgegpu as fg
    import torch
    x = torch.randn(10, 4, device="cuda")
    dq, dx = fg.logprobs_backward(x[:0], x, None, x.new_empty(0))
    assert dq.shape == (0, 4) and not dx.any()
    r = fg.logprobs(x[:0], x, k=3)
    assert r.lse.shape == (0,) and r.top_ids.shape == (0, 3)


@pytest.mark.parametrize("dtype,nq", [("f32", 3), ("f32", 40), ("bf16", 40)])
def test_equal_scores_go_to_the_lower_row(dtype, nq):
    """Rows repeated all over: among equal scores the lowest numbers win."""
    import forgegpu as fg
    import torch
    rng = np.random.default_rng(5)
    base = rng.standard_normal((7, 24))
    x = base[rng.integers(0, 7, 3000)]
    q = rng.standard_normal((nq, 24))
    dt = _types()[dtype]
    Q, X = torch.from_numpy(q).to(dt).cuda(), torch.from_numpy(x).to(dt).cuda()
    r = fg.logprobs(Q, X, k=64)
    f = so.forward(Q.double().cpu().numpy(), X.double().cpu().numpy(), None, 1.0, None, 64)
    assert np.array_equal(r.top_ids.cpu().numpy(), f["top_ids"])


@pytest.mark.parametrize("dtype,nq", [("f32", 2), ("f32", 130), ("bf16", 130)])
def test_alternatives_that_lie_side_by_side(dtype, nq):
    """Rows sorted by score: the best 40 share two groups of 32."""
    import forgegpu as fg
    import torch
    rng = np.random.default_rng(6)
    x = rng.standard_normal((2000, 16))
    q0 = rng.standard_normal(16)
    x = x[np.argsort(-(x @ q0))]
    q = q0 + 1e-3 * rng.standard_normal((nq, 16))
    dt = _types()[dtype]
    Q, X = torch.from_numpy(q).to(dt).cuda(), torch.from_numpy(x).to(dt).cuda()
    r = fg.logprobs(Q, X, k=40)
    f = so.forward(Q.double().cpu().numpy(), X.double().cpu().numpy(), None, 1.0, None, 40)
    assert np.array_equal(r.top_ids.cpu().numpy(), f["top_ids"])


BADS = [float("nan"), float("inf"), -float("inf"), 3e38]


@pytest.mark.parametrize("dtype,nq", [("f32", 4), ("f32", 140), ("bf16", 140)])
@pytest.mark.parametrize("bad", BADS)
def test_masked_rows_may_hold_anything(dtype, nq, bad):
    """Rows that no query may see, and a row that one may not, hold NaN,
    infinities or the type's largest values: the others' results are those of
    rows of zeros there."""
    import forgegpu as fg
    import torch
    Q, X, T, _, q, x, t, _ = make(dtype, nq, 500, 40, "none", seed=2)
    keep = np.random.default_rng(1).random((nq, 500)) < 0.6
    keep[:, [0, 77, 499]] = False
    keep[1:, 33] = False
    keep[0, 33] = bad == 3e38 and False
    keep[2] = False
    A = torch.from_numpy(so.words(keep)).cuda()
    up = torch.rand(3, nq, device="cuda")

    def go(X, Q):
        r = fg.logprobs(Q, X, T, scale=0.3, allowed=A, k=5)
        return list(r) + list(fg.logprobs_backward(Q, X, T, r.lse, r.entropy, d_logprob=up[0],
                                                   d_lse=up[1], d_entropy=up[2], scale=0.3,
                                                   allowed=A))

    X0, X1, Q0, Q1 = X.clone(), X.clone(), Q.clone(), Q.clone()
    X0[[0, 33, 77, 499]] = 0
    X1[[0, 33, 77, 499]] = bad
    Q0[2] = 0
    Q1[2] = bad  # a query that sees nothing
    for a, b in zip(go(X0, Q0), go(X1, Q1)):
        assert not torch.isnan(b).any()
        assert torch.equal(a, b)


@pytest.mark.parametrize("dtype,nq", [("f32", 4), ("f32", 140), ("bf16", 140), ("f16", 20)])
@pytest.mark.parametrize("bad", BADS)
def test_one_filter_hides_what_its_rows_hold(dtype, nq, bad):
    """The same with one filter for all queries."""
    import forgegpu as fg
    import torch
    Q, X, T, _, *_ = make(dtype, nq, 700, 40, "none", seed=2)
    keep = np.random.default_rng(1).random((1, 700)) < 0.6
    keep[0, [0, 77, 350, 699]] = False
    A = torch.from_numpy(so.words(keep)).cuda()
    up = torch.rand(3, nq, device="cuda")

    def go(X):
        r = fg.logprobs(Q, X, T, scale=0.3, allowed=A, k=5)
        return list(r) + list(fg.logprobs_backward(Q, X, T, r.lse, r.entropy, d_logprob=up[0],
                                                   d_lse=up[1], d_entropy=up[2], scale=0.3,
                                                   allowed=A))

    X0, X1 = X.clone(), X.clone()
    X0[[0, 77, 350, 699]] = 0
    X1[[0, 77, 350, 699]] = bad
    for a, b in zip(go(X0), go(X1)):
        assert not torch.isnan(b).any()
        assert torch.equal(a, b)


@pytest.mark.parametrize("dtype,nq", [("f32", 3), ("f32", 40), ("bf16", 40)])
def test_scores_that_lie_close_together(dtype, nq):
    """A common part of 100 under differences of 1e-3 and less: more rows than
    the picked groups hold are within the marks' reach of each other, and the
    order is still that of 64-bit scores."""
    import forgegpu as fg
    import torch
    rng = np.random.default_rng(7)
    x = np.concatenate([np.full((4000, 1), 10.0), 2.0 ** -7 * rng.integers(0, 64, (4000, 7))], 1)
    q = np.concatenate([np.full((nq, 1), 10.0), 2.0 ** -9 * rng.integers(1, 64, (nq, 7))], 1)
    dt = _types()[dtype]
    Q, X = torch.from_numpy(q).to(dt).cuda(), torch.from_numpy(x).to(dt).cuda()
    r = fg.logprobs(Q, X, k=30)
    f = so.forward(Q.double().cpu().numpy(), X.double().cpu().numpy(), None, 1.0, None, 30)
    assert np.array_equal(r.top_ids.cpu().numpy(), f["top_ids"])


@pytest.mark.parametrize("nq", [3, 40, 140])
@pytest.mark.parametrize("shift", [14, 17])
def test_scores_that_are_small_beside_their_rows(nq, shift):
    """Rows almost at right angles to their queries: what the 32-bit scores are
    off by is of the size of their differences, the order is that of the 64-bit
    ones."""
    import forgegpu as fg
    import torch
    rng = np.random.default_rng(shift)
    n, d = 3000, 64
    q = np.concatenate([np.ones((nq, 1)), rng.standard_normal((nq, d - 1))], 1).astype(np.float32)
    x = rng.standard_normal((n, d - 1)).astype(np.float32)
    q[:, 33:] = q[:, 1:32]  # the second half of a row takes the first one's part away
    q[:, 32] = 1
    x = np.concatenate([np.zeros((n, 1)), x[:, :31], np.zeros((n, 1)), -x[:, :31]], 1)
    x[:, 0] = rng.standard_normal(n)
    x[:, 32] = -x[:, 0] + 2.0 ** -shift * rng.standard_normal(n)
    Q, X = torch.from_numpy(q).cuda(), torch.from_numpy(x.astype(np.float32)).cuda()
    r = fg.logprobs(Q, X, k=10)
    # all but two products of a score take each other away, so it is the exact
    # sum of those two, a multiple of 2^-24 or so: rows may share one
    X = X.double().cpu().numpy()
    s = X[:, 0] + X[:, 32]
    best = np.sort(s)[::-1][:10]
    assert (s[r.top_ids.cpu().numpy()] == best).all()


@pytest.mark.parametrize("dtype,nq", [("f32", 4), ("f32", 140), ("bf16", 140), ("f16", 20)])
@pytest.mark.parametrize("bad", BADS[:3])
def test_what_is_not_finite_reaches_its_queries_only(dtype, nq, bad):
    import forgegpu as fg
    import torch
    Q, X, T, _, q, x, t, _ = make(dtype, nq, 300, 40, "none", seed=4)
    keep = np.ones((nq, 300), bool)
    keep[1:, 50] = False  # query 0 alone sees row 50
    A = torch.from_numpy(so.words(keep)).cuda()
    clean = fg.logprobs(Q, X, T, scale=0.3, allowed=A, k=5)
    X = X.clone()
    X[50, 3] = bad
    Q = Q.clone()
    Q[2, 1] = bad
    r = fg.logprobs(Q, X, T, scale=0.3, allowed=A, k=5)
    for i in (0, 2):
        assert torch.isnan(r.lse[i]) and torch.isnan(r.entropy[i]) and torch.isnan(r.logprob[i])
        assert (r.top_ids[i] == -1).all() and torch.isnan(r.top_logprobs[i]).all()
    rest = [i for i in range(nq) if i not in (0, 2)]
    for a, b in zip(clean, r):
        assert torch.equal(a[rest], b[rest])
    up = torch.rand(nq, device="cuda")
    dq, _ = fg.logprobs_backward(Q, X, T, r.lse, d_lse=up, scale=0.3, allowed=A)
    assert torch.isnan(dq[[0, 2]].float()).all() and not torch.isnan(dq[rest].float()).any()


def test_rows_of_very_different_sizes():
    """Rows and queries whose sizes spread over 2^60, rows of zeros among them:
    scores, and the gradient of every row, hold their own precision."""
    import forgegpu as fg
    import torch
    rng = np.random.default_rng(8)
    nq, n, d = 40, 600, 48
    q = rng.standard_normal((nq, d)) * 2.0 ** rng.integers(-6, 3, (nq, 1))
    x = rng.standard_normal((n, d)) * 2.0 ** rng.integers(-30, 2, (n, 1))
    x[5] = x[300] = 0
    q[7] = 0
    Q, X = torch.from_numpy(q).float().cuda(), torch.from_numpy(x).float().cuda()
    q, x = Q.double().cpu().numpy(), X.double().cpu().numpy()
    t = rng.integers(0, n, nq)
    T = torch.from_numpy(t).cuda()
    r = fg.logprobs(Q, X, T, scale=0.25, k=5)
    f = so.forward(q, x, t, 0.25, None, 5)
    es = so.score_bound(q, x, 0.25, "f32")
    check_forward(r, f, es, 5)
    g = rng.standard_normal(nq).astype(np.float32)
    lse = f["lse"].astype(np.float32)
    z = np.zeros(nq)
    got = fg.logprobs_backward(Q, X, T, torch.from_numpy(lse).cuda(),
                               d_logprob=torch.from_numpy(g).cuda(), scale=0.25)
    dq, dx, _, size = so.backward(q, x, t, lse.astype(np.float64), z, g.astype(np.float64), z, z,
                                  0.25, None)
    bq, bx = so.gradient_bounds(q, x, es, size, f["keep"], "f32", dq, dx)
    assert (np.abs(got[0].double().cpu().numpy() - dq) <= bq).all()
    assert (np.abs(got[1].double().cpu().numpy() - dx) <= bx).all()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_gradient_against_differences(dtype):
    """The kernels' gradient along random directions against differences of
    the 64-bit loss (error of the difference below 1e-7, see the CPU test of
    the same): within the sum of the elementwise bounds along the direction."""
    import forgegpu as fg
    import torch
    Q, X, T, A, q, x, t, al = make(dtype, 20, 150, 24, "each", seed=12)
    scale = 0.25
    rng = np.random.default_rng(2)
    up = rng.standard_normal((3, 20))
    up32 = torch.from_numpy(up).float().cuda()
    up = up32.double().cpu().numpy()
    r = fg.logprobs(Q, X, T, scale=scale, allowed=A)
    dq, dx = fg.logprobs_backward(Q, X, T, r.lse, r.entropy, d_logprob=up32[0], d_lse=up32[1],
                                  d_entropy=up32[2], scale=scale, allowed=A)

    def loss(q, x):
        f = so.forward(q, x, t, scale, al, 0)
        return sum((u * np.where(np.isfinite(f[k]), f[k], 0.0)).sum()
                   for u, k in zip(up, ("logprob", "lse", "entropy")))

    f = so.forward(q, x, t, scale, al, 0)
    es = so.score_bound(q, x, scale, dtype)
    es = es + so.forward_bounds(f, es)[0][:, None]  # (lse is the kernel's own here)
    wq, wx, _, size = so.backward(q, x, t, f["lse"], f["entropy"], *up, scale, al)
    bh = so.forward_bounds(f, es)[2]
    bq, bx = so.gradient_bounds(q, x, es + bh[:, None], size, f["keep"], dtype, wq, wx)
    dq, dx = dq.double().cpu().numpy(), dx.double().cpu().numpy()
    for _ in range(5):
        a, b, h = rng.standard_normal(q.shape), rng.standard_normal(x.shape), 1e-5
        diff = (loss(q + h * a, x + h * b) - loss(q - h * a, x - h * b)) / (2 * h)
        got = (dq * a).sum() + (dx * b).sum()
        assert abs(diff - got) <= (bq * np.abs(a)).sum() + (bx * np.abs(b)).sum() + 1e-6


def test_same_call_same_bits():
    import forgegpu as fg
    import torch
    Q, X, T, A, *_ = make("bf16", 300, 9000, 200, "each", seed=3)
    up = torch.rand(300, device="cuda")

    def go():
        r = fg.logprobs(Q, X, T, scale=0.2, allowed=A, k=10)
        return list(r) + list(fg.logprobs_backward(Q, X, T, r.lse, d_logprob=up, scale=0.2,
                                                   allowed=A))
    a, b = go(), go()
    assert all(torch.equal(u, v) for u, v in zip(a, b))


def test_on_another_stream_and_in_graphs():
    """The calls run on the current stream; captured calls replay with what
    their inputs hold then, each graph with its own workspace."""
    import forgegpu as fg
    import torch
    Q, X, T, A, *_ = make("f32", 100, 3000, 64, "each", seed=9)
    Q2, X2, T2, _, *_ = make("bf16", 200, 5000, 96, "none", seed=10)
    up, up2 = torch.rand(100, device="cuda"), torch.rand(200, device="cuda")

    def one():
        r = fg.logprobs(Q, X, T, scale=0.2, allowed=A, k=7)
        return list(r) + list(fg.logprobs_backward(Q, X, T, r.lse, d_logprob=up, scale=0.2,
                                                   allowed=A))

    def two():
        r = fg.logprobs(Q2, X2, T2, scale=0.2, k=3)
        return list(r) + list(fg.logprobs_backward(Q2, X2, T2, r.lse, d_lse=up2, scale=0.2))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        Q.mul_(1.0)
        a1 = one()
    torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for f in (one, two):
        f()
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = f()
        graphs.append((g, out))
    want1, want2 = one(), two()
    assert all(torch.equal(u, v) for u, v in zip(a1, want1))
    for _ in range(2):
        for g, _ in graphs:
            g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(u, v) for u, v in zip(graphs[0][1], want1))
        assert all(torch.equal(u, v) for u, v in zip(graphs[1][1], want2))
    # both at once on two streams
    other = torch.cuda.Stream()
    with torch.cuda.stream(side):
        graphs[0][0].replay()
    with torch.cuda.stream(other):
        graphs[1][0].replay()
    torch.cuda.synchronize()
    assert all(torch.equal(u, v) for u, v in zip(graphs[0][1], want1))
    assert all(torch.equal(u, v) for u, v in zip(graphs[1][1], want2))
    # new inputs in the captured buffers
    X.copy_(X.flip(0).clone())
    Q2.copy_(Q2.flip(0).clone())
    graphs[0][0].replay()
    graphs[1][0].replay()
    torch.cuda.synchronize()
    assert all(torch.equal(u, v) for u, v in zip(graphs[0][1], one()))
    assert all(torch.equal(u, v) for u, v in zip(graphs[1][1], two()))


def test_offsets_beyond_32_bits():
    """2.2e9 elements of rows: the rows past 2^32 bytes and past 2^31 elements
    score, and get their gradient, like copies of them in a small table."""
    import forgegpu as fg
    import torch
    n, d = 2_150_000, 1024
    g = torch.Generator(device="cuda").manual_seed(0)
    X = torch.empty(n, d, dtype=torch.bfloat16, device="cuda")
    for i in range(0, n, 50_000):
        X[i:i + 50_000] = torch.randn(min(50_000, n - i), d, generator=g, device="cuda")
    pick = torch.tensor([0, 1_048_576, 2_097_151, 2_097_152, 2_149_999], device="cuda")
    Q = (X[pick].float() * 1.5).to(torch.bfloat16)
    keep = torch.zeros((n + 31) // 32, dtype=torch.int32, device="cuda")
    near = (pick[:, None] + torch.arange(-40, 41, device="cuda")).flatten()
    near = near[(near >= 0) & (near < n)].unique()
    bits = np.zeros((1, n), bool)
    bits[0, near.cpu().numpy()] = True
    keep.copy_(torch.from_numpy(so.words(bits)[0]))
    full = fg.logprobs(Q, X, pick, scale=0.02, k=3)
    assert torch.equal(full.top_ids[:, 0], pick)
    some = fg.logprobs(Q, X, pick, scale=0.02, allowed=keep, k=3)
    small = X[near].contiguous()
    where = torch.searchsorted(near, pick)
    want = fg.logprobs(Q, small, where, scale=0.02, k=3)
    # (the same scores in groups of other sizes: each lse is within 2^-19)
    for a, b in ((some.lse, want.lse), (some.logprob, want.logprob), (some.entropy, want.entropy)):
        assert (a - b).abs().max() <= 2.0 ** -17
    assert torch.equal(some.top_ids, near[want.top_ids])
    up = torch.ones(5, device="cuda")
    dq, dx = fg.logprobs_backward(Q, X, pick, some.lse, d_logprob=up, scale=0.02, allowed=keep)
    wq, wx = fg.logprobs_backward(Q, small, where, some.lse, d_logprob=up, scale=0.02)
    # two roundings to bf16 of sums that differ far below them
    assert ((dq - wq).abs().float() <= 2.0 ** -7 * wq.abs().float() + 1e-6).all()
    assert ((dx[near] - wx).abs().float() <= 2.0 ** -7 * wx.abs().float() + 1e-6).all()
    assert not dx[1000:1_048_000].any()


def test_a_wait_that_runs_out(ctx):
    """The timeout path: NaN outputs and a Timeout from the status call; the
    next call is clean."""
    import forgegpu as fg
    import torch
    Q, X, T, A, *_ = make("f32", 64, 2000, 64, "none")
    want = fg.logprobs(Q, X, T, k=2)
    up = torch.rand(64, device="cuda")
    grads = fg.logprobs_backward(Q, X, T, want.lse, d_logprob=up)
    ws = torch.empty(256 << 20, dtype=torch.uint8, device="cuda")
    ctx.set_wait_limit(0.02)
    try:
        ctx.test_stall_scans(1)
        r = fg.logprobs(Q, X, T, k=2, workspace=ws)
        with pytest.raises(fg.ForgeGpuError) as e:
            fg.logprobs_status(ws)
        assert e.value.kind == "Timeout"
        assert torch.isnan(r.lse).all() and torch.isnan(r.logprob).all() and (r.top_ids == -1).all()
        ctx.test_stall_scans(1)
        g = fg.logprobs_backward(Q, X, T, want.lse, d_logprob=up, workspace=ws)
        with pytest.raises(fg.ForgeGpuError) as e:
            fg.logprobs_status(ws)
        assert e.value.kind == "Timeout"
        assert torch.isnan(g[0]).all() and torch.isnan(g[1]).all()
    finally:
        ctx.set_wait_limit(2.0)
    r = fg.logprobs(Q, X, T, k=2, workspace=ws)
    fg.logprobs_status(ws)
    assert all(torch.equal(a, b) for a, b in zip(r, want))
    g = fg.logprobs_backward(Q, X, T, want.lse, d_logprob=up, workspace=ws)
    fg.logprobs_status(ws)
    assert torch.equal(g[0], grads[0]) and torch.equal(g[1], grads[1])


def test_binding_refusals():
    import forgegpu as fg
    import torch
    Q, X, T, A, *_ = make("f32", 4, 100, 8, "each")
    with pytest.raises(fg.ForgeGpuError):
        fg.logprobs(Q, X.half())
    with pytest.raises(fg.ForgeGpuError):
        fg.logprobs(Q, X[:, :7])
    with pytest.raises(fg.ForgeGpuError):
        fg.logprobs(Q, X.t())
    with pytest.raises(fg.ForgeGpuError):
        fg.logprobs(Q, X, T[:3])
    with pytest.raises(fg.ForgeGpuError):
        fg.logprobs(Q, X, T.int())
    with pytest.raises(fg.ForgeGpuError):
        fg.logprobs(Q, X, allowed=A[:3])
    with pytest.raises(fg.ForgeGpuError):
        fg.logprobs(Q, X, allowed=A[:, :3])
    with pytest.raises(fg.ForgeGpuError):
        fg.logprobs(Q, X, k=65)
    with pytest.raises(fg.ForgeGpuError):
        fg.logprobs(Q, X, scale=0.0)
    with pytest.raises(fg.ForgeGpuError):
        fg.logprobs(Q, X[:0])
    with pytest.raises(fg.ForgeGpuError):
        fg.logprobs(Q, X, workspace=torch.empty(256, dtype=torch.uint8, device="cuda"))
    with pytest.raises(fg.ForgeGpuError):
        fg.logprobs_backward(Q, X, T, torch.zeros(4, device="cuda"),
                             d_entropy=torch.zeros(4, device="cuda"))


# ---- the index --------------------------------------------------------------
@pytest.mark.parametrize("nq,n,dim,k", [(1, 1, 3, 1), (3, 500, 128, 10), (70, 3001, 96, 10)])
def test_index_log_probs(nq, n, dim, k):
    import forgegpu as fg
    rng = np.random.default_rng(n)
    x = rng.standard_normal((n, dim)).astype(np.float32)
    q = rng.standard_normal((nq, dim)).astype(np.float32)
    ids = rng.permutation(10 * n)[:n].astype(np.uint64) + 7
    ix = fg.BruteForceIndex(fg.DistanceMetric.DotProduct).add(x, ids)
    t = rng.integers(0, n, nq)
    want_ids = ids[t].copy()
    want_ids[0] = 1  # an id that the index does not hold
    t[0] = -1
    temp = np.float32(3.0)
    r = ix.log_probs(q, want_ids, temperature=3.0, k=k)
    scale = np.float64(np.float32(1.0) / temp)
    q64, x64 = q.astype(np.float64), x.astype(np.float64)
    f = so.forward(q64, x64, t, scale, None, k)
    es = so.score_bound(q64, x64, scale, "f32")
    ble, bl, bh = so.forward_bounds(f, es)
    assert (np.abs(r.lse - f["lse"]) <= ble).all()
    assert (np.abs(r.logprob - f["logprob"]) <= bl).all() and r.logprob[0] == 0
    assert (np.abs(r.entropy - f["entropy"]) <= bh).all()
    want = np.where(f["top_ids"] < 0, np.uint64(2 ** 64 - 1), ids[np.maximum(f["top_ids"], 0)])
    assert np.array_equal(r.top_ids, want)
    # the best of the softmax are the best of the search, and their log
    # probabilities fall by the difference of the distances / temperature
    sid, sd, cnt = ix.batch_search_arrays(q, k)
    assert np.array_equal(sid, r.top_ids)


def test_index_follows_its_changes_and_refuses():
    import forgegpu as fg
    rng = np.random.default_rng(0)
    x = rng.standard_normal((50, 8)).astype(np.float32)
    q = rng.standard_normal((2, 8)).astype(np.float32)
    ix = fg.BruteForceIndex(fg.DistanceMetric.DotProduct)
    with pytest.raises(fg.ForgeGpuError) as e:
        ix.log_probs(q)
    assert e.value.kind == "EmptyVectorSet"
    ix.add(x[:30])
    a = ix.log_probs(q, k=3)
    ix.add(x[30:], np.array([5] + list(range(31, 50)), np.uint64))  # id 5 twice: its first row counts
    b = ix.log_probs(q, [5, 49], k=3)
    assert (b.lse > a.lse).all()
    s = q.astype(np.float64) @ x.T.astype(np.float64)
    lse = np.log(np.exp(s).sum(1))
    want = np.array([s[0, 5] - lse[0], s[1, 49] - lse[1]])
    assert np.abs(b.logprob - want).max() < 1e-5
    assert ix.remove(49)
    c = ix.log_probs(q, [49, 48])
    assert c.logprob[0] == 0 and c.logprob[1] < 0 and (c.lse < b.lse).all()
    assert c.top_ids.shape == (2, 0)
    for kw in (dict(temperature=0.0), dict(temperature=float("nan")), dict(k=65)):
        with pytest.raises(fg.ForgeGpuError):
            ix.log_probs(q, **kw)
    with pytest.raises(fg.ForgeGpuError):
        ix.log_probs(q[:, :5])
    with pytest.raises(fg.ForgeGpuError):
        ix.log_probs(q, [1])
    ix.shard(0, 2)
    with pytest.raises(fg.ForgeGpuError) as e:
        ix.log_probs(q)
    assert e.value.kind == "NotSupported"
    eu = fg.BruteForceIndex(fg.DistanceMetric.Euclidean).add(x)
    with pytest.raises(fg.ForgeGpuError) as e:
        eu.log_probs(q)
    assert e.value.kind == "NotSupported"


@pytest.mark.parametrize("dtype,nq,n,dim,mask,pad,shift,k", [
    # f32 rows of one block of K, tiles of 256 columns: both sides of its last dimension
    ("f32", 300, 4099, 128, "each", 0, 0, 10), ("f32", 257, 2050, 113, "one", 3, 1, 64),
    ("f32", 130, 2305, 129, "one", 0, 0, 5), ("f32", 520, 1, 16, "none", 0, 0, 3),
    ("f32", 18, 767, 64, "none", 0, 0, 0),
    # 16-bit rows whose alignment has them copied: to 4 queries, and more
    ("bf16", 4, 3001, 75, "each", 0, 0, 10), ("f16", 3, 800, 129, "one", 0, 1, 64),
    ("bf16", 5, 1500, 131, "each", 0, 0, 5), ("f16", 4, 40, 2049, "none", 0, 0, 3),
    # the largest dimension
    ("f32", 2, 70, 16384, "none", 0, 0, 4), ("f32", 33, 400, 16384, "each", 0, 0, 4),
    ("bf16", 5, 300, 16384, "one", 0, 0, 64), ("f16", 20, 90, 16383, "none", 1, 0, 2),
])
def test_forward_at_its_limits(dtype, nq, n, dim, mask, pad, shift, k):
    test_forward(dtype, nq, n, dim, mask, pad, shift, k)


@pytest.mark.parametrize("dtype,nq,n,dim,mask,pad,shift", [
    ("f32", 1, 4000, 128, "none", 0, 0), ("f32", 9, 50, 16384, "each", 0, 0),
    ("bf16", 9, 50, 16384, "none", 0, 0), ("f16", 3, 40, 16383, "one", 0, 1),
    ("f32", 600, 1, 32, "each", 0, 0), ("bf16", 70, 2, 1, "each", 0, 0),
    ("bf16", 1500, 700, 64, "each", 0, 0),
    # few queries: several steps a block, the largest dimension, one past either
    ("f32", 1, 16000, 100, "one", 0, 0), ("f32", 3, 9001, 61, "each", 1, 1),
    ("f32", 8, 500, 1024, "each", 0, 0), ("f32", 8, 30, 1025, "none", 0, 0),
    ("f32", 9, 700, 33, "each", 0, 0), ("bf16", 2, 12001, 200, "each", 3, 1),
    ("bf16", 6, 300, 1023, "one", 0, 0), ("f16", 8, 5000, 5, "each", 0, 0),
    ("f16", 4, 17, 96, "none", 0, 0),
])
def test_backward_at_its_limits(dtype, nq, n, dim, mask, pad, shift):
    test_backward(dtype, nq, n, dim, mask, pad, shift)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_one_target_for_all_queries(dtype):
    """Every query's given row is the same: its gradient is the sum of all of
    theirs, in a fixed order."""
    import forgegpu as fg
    import torch
    nq, n = 400, 900
    Q, X, _, _, q, x, _, _ = make(dtype, nq, n, 72, "none", seed=12)
    t = np.full(nq, 77)
    T = torch.from_numpy(t).cuda()
    f = so.forward(q, x, t, 0.25, None, 0)
    lse = f["lse"].astype(np.float32)
    up = torch.full((nq,), -1.0 / nq, device="cuda")
    run = lambda: fg.logprobs_backward(Q, X, T, torch.from_numpy(lse).cuda(), d_logprob=up,
                                       scale=0.25)
    got, again = run(), run()
    u = up.double().cpu().numpy()
    z = np.zeros(nq)
    dq, dx, _, size = so.backward(q, x, t, lse.astype(np.float64), z, u, z, z, 0.25, None)
    es = so.score_bound(q, x, 0.25, dtype)
    bounds = so.gradient_bounds(q, x, es, size, f["keep"], dtype, dq, dx)
    for g, h, w, b in zip(got, again, (dq, dx), bounds):
        assert torch.equal(g, h)
        assert (np.abs(g.double().cpu().numpy() - w) <= b + 1e-30).all()


@pytest.mark.parametrize("dtype,nq", [("f32", 3), ("f32", 40), ("bf16", 2), ("bf16", 300)])
@pytest.mark.parametrize("rows", [1, "nq"])
def test_a_filter_that_leaves_nothing(dtype, nq, rows):
    """No query sees a row: lse -inf, entropy 0, no alternatives, a given row
    -inf, gradients of zero."""
    import forgegpu as fg
    import torch
    Q, X, T, *_ = make(dtype, nq, 700, 24, "none", seed=13)
    A = torch.zeros((nq if rows == "nq" else 1, 22), dtype=torch.int32, device="cuda")
    r = fg.logprobs(Q, X, T, scale=0.5, allowed=A, k=4)
    assert (r.lse == -float("inf")).all() and (r.entropy == 0).all()
    assert torch.equal(r.logprob, torch.where(T >= 0, -float("inf"), 0.0))
    assert (r.top_ids == -1).all() and (r.top_logprobs == -float("inf")).all()
    up = torch.ones(nq, device="cuda")
    for g in fg.logprobs_backward(Q, X, T, r.lse, r.entropy, d_logprob=up, d_lse=up,
                                  d_entropy=up, scale=0.5, allowed=A):
        assert (g == 0).all()


def test_status_of_a_call_without_work():
    import forgegpu as fg
    import torch
    Q, X, T, *_ = make("bf16", 4, 50, 16, "none", seed=14)
    for call in (lambda ws: fg.logprobs(Q[:0], X, T[:0], k=2, workspace=ws),
                 lambda ws: fg.logprobs_backward(Q[:0], X, T[:0], torch.zeros(0, device="cuda"),
                                                 workspace=ws),
                 lambda ws: fg.logprobs_backward(Q, X, T, torch.zeros(4, device="cuda"),
                                                 need_queries=False, need_rows=False,
                                                 workspace=ws)):
        ws = torch.full((1 << 20,), 255, dtype=torch.uint8, device="cuda")
        call(ws)
        fg.logprobs_status(ws)


@pytest.mark.parametrize("dtype,nq", [("f32", 3), ("f32", 40), ("bf16", 2), ("bf16", 300)])
def test_gradients_into_parts_of_wider_buffers(dtype, nq):
    """Rows ld_d_* elements apart: what lies between and behind them stays."""
    import ctypes as C
    import forgegpu as fg
    import torch
    n, d, gap = 333, 41, 3
    Q, X, T, A, *_ = make(dtype, nq, n, d, "each", seed=15)
    r = fg.logprobs(Q, X, T, scale=0.3, allowed=A)
    up = torch.rand(nq, device="cuda")
    want = fg.logprobs_backward(Q, X, T, r.lse, d_logprob=up, scale=0.3, allowed=A)
    dq = torch.full((nq + 2, d + gap), 7.0, dtype=Q.dtype, device="cuda")
    dx = torch.full((n + 2, d + gap), 7.0, dtype=Q.dtype, device="cuda")
    ws = torch.empty(256 << 20, dtype=torch.uint8, device="cuda")
    a = fg.LogprobGradArgs(
        dtype={"f32": 0, "bf16": 2}[dtype], queries=Q.data_ptr(), nq=nq, ld_queries=d,
        rows=X.data_ptr(), n=n, ld_rows=d, dim=d, scale=0.3, targets=T.data_ptr(),
        allowed=A.data_ptr(), ld_allowed=A.stride(0), lse=r.lse.data_ptr(),
        d_logprob=up.data_ptr(), d_queries=dq.data_ptr(), ld_d_queries=d + gap,
        d_rows=dx.data_ptr(), ld_d_rows=d + gap, workspace=ws.data_ptr(),
        workspace_bytes=ws.numel(), stream=torch.cuda.current_stream().cuda_stream)
    assert fg.lib().fdb_logprobs_backward(fg.default_context().h, C.byref(a)) == 0
    for got, w in ((dq, want[0]), (dx, want[1])):
        assert torch.equal(got[:-2, :d], w)
        assert (got[:-2, d:] == 7).all() and (got[-2:] == 7).all()


def test_two_eager_calls_at_once():
    """Calls on two streams, each with a workspace of its own, over the same
    inputs: the same bits as one after the other."""
    import forgegpu as fg
    import torch
    Q, X, T, A, *_ = make("f32", 300, 20000, 96, "one", seed=16)
    up = torch.rand(300, device="cuda")

    def both(q, t, u):
        r = fg.logprobs(q, X, t, scale=0.2, allowed=A, k=9)
        return list(r) + list(fg.logprobs_backward(q, X, t, r.lse, d_logprob=u, scale=0.2,
                                                   allowed=A))

    parts = [(Q, T, up), (Q[:5], T[:5], up[:5])]
    want = [both(*p) for p in parts]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in parts]
    got = [[], []]
    for _ in range(4):
        for i, (s, p) in enumerate(zip(streams, parts)):
            with torch.cuda.stream(s):
                got[i].append(both(*p))
    torch.cuda.synchronize()
    for w, runs in zip(want, got):
        for g in runs:
            assert all(torch.equal(a, b) for a, b in zip(w, g))


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_a_few_queries_captured(dtype):
    """The passes for a few queries, with more shared memory than a kernel has
    by default, captured before their first eager call of that size."""
    import forgegpu as fg
    import torch
    Q, X, T, *_ = make(dtype, 5, 900, 1001, "none", seed=17)
    up = torch.rand(5, device="cuda")

    def run():
        r = fg.logprobs(Q, X, T, scale=0.05, k=3)
        return list(r) + list(fg.logprobs_backward(Q, X, T, r.lse, d_logprob=up, scale=0.05))

    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = run()
    X.copy_(X.flip(0).clone())
    g.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(out, run()))


@pytest.mark.parametrize("dtype,nq", [("f32", 1), ("f32", 7), ("bf16", 4), ("f16", 8)])
@pytest.mark.parametrize("bad", BADS)
def test_gradients_of_a_few_queries_beside_what_is_not_finite(dtype, nq, bad):
    """What a masked row, or a query that sees nothing, holds changes no bit; a
    row that one query may see makes that query's gradient NaN, and the others'
    stay."""
    import forgegpu as fg
    import torch
    Q, X, T, _, q, x, t, _ = make(dtype, nq, 700, 45, "none", seed=18)
    keep = np.random.default_rng(2).random((nq, 700)) < 0.6
    keep[:, 123] = False
    keep[:, 400] = False
    keep[0, 400] = True  # the first query alone
    if nq > 2:
        keep[2] = False
    A = torch.from_numpy(so.words(keep)).cuda()
    r = fg.logprobs(Q, X, T, scale=0.3, allowed=A)
    up = torch.rand(nq, device="cuda")
    go = lambda Q, X: fg.logprobs_backward(Q, X, T, r.lse, d_logprob=up, d_lse=up, scale=0.3,
                                           allowed=A)
    want = go(Q, X)
    X1, Q1 = X.clone(), Q.clone()
    X1[123, 4] = bad
    if nq > 2:
        Q1[2, 7] = bad
    for a, b in zip(want, go(Q1, X1)):
        assert torch.equal(a, b)
    if np.isfinite(bad):
        return
    X1[400, 9] = bad
    dq, dx = go(Q1, X1)
    assert torch.isnan(dq[0].float()).all() and torch.equal(dq[1:], want[0][1:])
    other = torch.arange(700, device="cuda") != 400
    assert torch.equal(dx[other], want[1][other]) and torch.isnan(dx[400].float()).all()
