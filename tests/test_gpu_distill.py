"""The loss of a teacher's best rows and its gradient, against the 64-bit
definitions, elementwise within the bounds of distill_oracle."""
import numpy as np
import pytest

import distill_oracle as do
import softmax_oracle as so
from test_gpu_softmax_rows import make

pytestmark = pytest.mark.gpu


def lists(nq, n, k, rest, seed=0, tail=0.3):
    """A teacher's lists: ids among them twice, outside of the rows, missing, and
    logits unsorted; with rest, log probabilities that leave `tail`."""
    rng = np.random.default_rng(seed + 100)
    ids = rng.integers(0, n, (nq, k))
    z = rng.standard_normal((nq, k)) * 2
    gone = rng.random((nq, k)) < 0.1
    ids[gone & (rng.random((nq, k)) < 0.5)] = -1
    ids[rng.random((nq, k)) < 0.03] = n
    if rest:
        z = z - np.log(np.exp(z).sum(1, keepdims=True)) + np.log(1 - tail)
    z = np.where(gone & (ids >= 0), -np.inf, z).astype(np.float32)
    if nq > 2:
        ids[nq // 3] = -1  # a list with nothing in it
    return ids, z


def cuda(*a):
    import torch
    return [torch.from_numpy(np.ascontiguousarray(v)).cuda() for v in a]


def check(got, want, bound, name):
    got = got.double().cpu().numpy()
    inf = ~np.isfinite(want)
    assert np.array_equal(got[inf], want[inf]), name
    off = np.abs(got[~inf] - want[~inf])
    assert (off <= bound[~inf]).all(), (name, (off / bound[~inf]).max())


def check_forward(r, o, es, rest):
    b = do.forward_bounds(o, es)
    for name in ("lse", "logprobs", "loss") + (("rest",) if rest else ()):
        check(getattr(r, name), o[name], b[name], name)


SHAPES = [
    # dtype, nq, n, dim, k, rest, mask, pad, shift
    ("f32", 1, 1, 1, 1, False, "none", 0, 0), ("f32", 1, 1, 1, 1, True, "none", 0, 0),
    ("f32", 1, 31, 8, 5, True, "none", 0, 0), ("f32", 3, 700, 64, 16, False, "each", 0, 0),
    ("f32", 8, 2049, 130, 33, True, "each", 3, 0), ("f32", 9, 700, 65, 256, True, "one", 0, 1),
    ("f32", 17, 255, 96, 7, False, "none", 0, 0), ("f32", 128, 257, 64, 20, True, "each", 1, 1),
    ("f32", 300, 4001, 200, 10, True, "none", 2, 0), ("f32", 33, 400, 2100, 4, False, "one", 0, 0),
    ("bf16", 1, 5003, 96, 10, True, "one", 0, 0), ("bf16", 2, 256, 64, 1, False, "none", 0, 0),
    ("bf16", 33, 511, 65, 12, True, "each", 0, 0), ("bf16", 129, 1027, 200, 64, False, "each", 3, 1),
    ("bf16", 260, 5000, 768, 32, True, "none", 0, 0), ("bf16", 50, 2000, 1100, 9, False, "none", 0, 0),
    ("bf16", 400, 900, 72, 256, True, "each", 8, 8),
    ("f16", 1, 100, 7, 3, False, "none", 0, 0), ("f16", 140, 3001, 129, 11, True, "each", 0, 0),
    ("f16", 65, 999, 256, 40, True, "none", 8, 0),
]


@pytest.mark.parametrize("dtype,nq,n,dim,k,rest,mask,pad,shift", SHAPES)
def test_loss(dtype, nq, n, dim, k, rest, mask, pad, shift):
    import forgegpu as fg
    Q, X, _, A, q, x, _, al = make(dtype, nq, n, dim, mask, pad, shift, seed=nq * 3 + n)
    ids, z = lists(nq, n, k, rest, seed=n)
    I, Z = cuda(ids, z)
    scale = np.float64(np.float32(2.0 / np.sqrt(dim)))
    ts = 1.0 if rest else 0.75
    r = fg.distill(Q, X, I, Z, scale=float(scale), teacher_scale=ts, rest=rest, allowed=A)
    o = do.forward(q, x, ids, z, scale, ts, rest, al)
    check_forward(r, o, so.score_bound(q, x, scale, dtype), rest)
    assert rest or r.rest is None


@pytest.mark.parametrize("dtype,nq,n,dim,k,rest,mask,pad,shift", SHAPES + [
    ("f32", 700, 90, 77, 5, True, "none", 0, 0), ("bf16", 1000, 128, 300, 30, False, "none", 8, 8),
    ("f32", 5, 9001, 61, 16, True, "each", 1, 1), ("bf16", 6, 300, 1023, 8, True, "one", 0, 0),
    ("f32", 2, 16000, 100, 100, False, "one", 0, 0), ("f16", 8, 5000, 5, 256, True, "each", 0, 0),
    ("f32", 8, 500, 1024, 30, False, "each", 0, 0), ("bf16", 1, 4000, 768, 64, True, "none", 0, 0),
])
def test_gradient(dtype, nq, n, dim, k, rest, mask, pad, shift):
    import forgegpu as fg
    Q, X, _, A, q, x, _, al = make(dtype, nq, n, dim, mask, pad, shift, seed=nq + n)
    ids, z = lists(nq, n, k, rest, seed=n + 1)
    scale = np.float64(np.float32(2.0 / np.sqrt(dim)))
    ts = 1.0 if rest else 1.5
    o = do.forward(q, x, ids, z, scale, ts, rest, al)
    rng = np.random.default_rng(3)
    lse, lp, rl = (o[v].astype(np.float32) for v in ("lse", "logprobs", "rest"))
    up = (rng.standard_normal(nq) * (64.0 if dtype == "f16" else 1.0) / nq).astype(np.float32)
    I, Z, L, P, R, U = cuda(ids, z, lse, lp, rl, up)
    got = fg.distill_backward(Q, X, I, Z, L, P, R if rest else None, d_loss=U, scale=float(scale),
                              teacher_scale=ts, allowed=A)
    r64 = rl.astype(np.float64) if rest else None
    dq, dx, size = do.backward(q, x, o, ids, lse.astype(np.float64), lp.astype(np.float64), r64,
                               up.astype(np.float64), scale)
    es = so.score_bound(q, x, scale, dtype)
    bq, bx = do.gradient_bounds(q, x, o, es, size, dtype, dq, dx, lse, r64, up * scale)
    for name, g, w, b in (("d_queries", got[0], dq, bq), ("d_rows", got[1], dx, bx)):
        assert g.dtype == Q.dtype and g.shape == w.shape
        off = np.abs(g.double().cpu().numpy() - w)
        assert (off <= b + 1e-30).all(), (name, (off / (b + 1e-30)).max())


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("rest", [False, True])
def test_gradient_against_differences(dtype, rest):
    """Along random directions against differences of the 64-bit loss (with h = 1e-5
    off by h^2 times third derivatives of size 1 and 2^-52 / h: 1e-6 is allowed)."""
    import forgegpu as fg
    Q, X, _, A, q, x, _, al = make(dtype, 20, 150, 24, "each", seed=12)
    ids, z = lists(20, 150, 8, rest, seed=5)
    I, Z = cuda(ids, z)
    up = np.random.default_rng(2).standard_normal(20).astype(np.float32)
    U, = cuda(up)
    scale = 0.25
    r = fg.distill(Q, X, I, Z, scale=scale, rest=rest, allowed=A)
    dq, dx = fg.distill_backward(Q, X, I, Z, r.lse, r.logprobs, r.rest, d_loss=U, scale=scale,
                                 allowed=A)
    up = up.astype(np.float64)

    def loss(q, x):
        return (up * do.forward(q, x, ids, z, scale, 1.0, rest, al)["loss"]).sum()

    o = do.forward(q, x, ids, z, scale, 1.0, rest, al)
    es = so.score_bound(q, x, scale, dtype)
    es = es + 2 * do.forward_bounds(o, es)["rest"][:, None]  # (lse, rest are the kernel's own)
    r64 = o["rest"] if rest else None
    wq, wx, size = do.backward(q, x, o, ids, o["lse"], o["logprobs"], r64, up, scale)
    bq, bx = do.gradient_bounds(q, x, o, es, size, dtype, wq, wx, o["lse"], r64, up * scale)
    dq, dx = dq.double().cpu().numpy(), dx.double().cpu().numpy()
    rng = np.random.default_rng(4)
    for _ in range(5):
        a, b, h = rng.standard_normal(q.shape), rng.standard_normal(x.shape), 1e-5
        diff = (loss(q + h * a, x + h * b) - loss(q - h * a, x - h * b)) / (2 * h)
        got = (dq * a).sum() + (dx * b).sum()
        assert abs(diff - got) <= (bq * np.abs(a)).sum() + (bx * np.abs(b)).sum() + 1e-6


@pytest.mark.parametrize("dtype,nq", [("f32", 3), ("f32", 40), ("bf16", 2), ("bf16", 40)])
def test_a_sure_student(dtype, nq):
    """The student leaves 1e-7 to 1e-3 to the rows that the teacher does not name:
    log r still holds its own precision (1 - sum p would have none)."""
    import forgegpu as fg
    rng = np.random.default_rng(1)
    n, d = 900, 32
    x = rng.standard_normal((n, d))
    t = rng.integers(0, n, nq)
    q = x[t] * rng.uniform(0.8, 1.2, (nq, 1))
    import torch
    dt = {"f32": torch.float32, "bf16": torch.bfloat16}[dtype]
    Q, X = torch.from_numpy(q).to(dt).cuda(), torch.from_numpy(x).to(dt).cuda()
    q, x = Q.double().cpu().numpy(), X.double().cpu().numpy()
    ids = np.stack([t, rng.integers(0, n, nq), rng.integers(0, n, nq)], 1)
    z = np.log(np.array([[0.7, 0.1, 0.05]], np.float32)).repeat(nq, 0)
    I, Z = cuda(ids, z)
    r = fg.distill(Q, X, I, Z, scale=1.0, rest=True)
    o = do.forward(q, x, ids, z, 1.0, 1.0, True, None)
    assert np.median(o["rest"]) < np.log(1e-3)
    check_forward(r, o, so.score_bound(q, x, 1.0, dtype), True)


@pytest.mark.parametrize("dtype,nq", [("f32", 4), ("bf16", 40)])
def test_all_rows_named(dtype, nq):
    """The lists hold every row that a query sees: there is no rest, whatever the
    teacher's probabilities leave, and the teacher's sum is made 1."""
    import forgegpu as fg
    Q, X, _, A, q, x, _, al = make(dtype, nq, 12, 16, "each", seed=3)
    ids = np.tile(np.arange(12), (nq, 1))
    z = np.log(np.full((nq, 12), 0.05, np.float32)) + \
        np.random.default_rng(0).random((nq, 12)).astype(np.float32)
    I, Z = cuda(ids, z)
    r = fg.distill(Q, X, I, Z, scale=0.5, rest=True, allowed=A)
    o = do.forward(q, x, ids, z, 0.5, 1.0, True, al)
    check_forward(r, o, so.score_bound(q, x, 0.5, dtype), True)
    assert (r.rest == -float("inf")).all()
    U = cuda(np.ones(nq, np.float32))[0]
    got = fg.distill_backward(Q, X, I, Z, r.lse, r.logprobs, r.rest, d_loss=U, scale=0.5, allowed=A)
    lse, lp, rl = (getattr(r, v).double().cpu().numpy() for v in ("lse", "logprobs", "rest"))
    dq, dx, size = do.backward(q, x, o, ids, lse, lp, rl, np.ones(nq), 0.5)
    bq, bx = do.gradient_bounds(q, x, o, so.score_bound(q, x, 0.5, dtype), size, dtype, dq, dx, lse,
                                rl, np.full(nq, 0.5))
    assert (np.abs(got[0].double().cpu().numpy() - dq) <= bq).all()
    assert (np.abs(got[1].double().cpu().numpy() - dx) <= bx).all()


def test_probabilities_above_one_are_made_one():
    import forgegpu as fg
    Q, X, _, _, q, x, _, _ = make("f32", 5, 300, 16, "none", seed=3)
    ids = np.arange(20).reshape(5, 4)
    z = np.log(np.array([[0.9, 0.4, 0.3, 0.2]], np.float32)).repeat(5, 0)
    I, Z = cuda(ids, z)
    r = fg.distill(Q, X, I, Z, scale=0.5, rest=True)
    o = do.forward(q, x, ids, z, 0.5, 1.0, True, None)
    assert (o["R"] == 0).all() and np.abs(o["P"].sum(1) - 1).max() < 1e-12
    check_forward(r, o, so.score_bound(q, x, 0.5, "f32"), True)
    assert (r.loss > 0).all()


@pytest.mark.parametrize("dtype,nq", [("f32", 4), ("f32", 40), ("bf16", 40)])
@pytest.mark.parametrize("rest", [False, True])
def test_a_student_that_agrees(dtype, nq, rest):
    """The teacher's logits are the student's own log probabilities: the loss is
    what rounding leaves of 0, the gradients are within their bounds of 0."""
    import forgegpu as fg
    Q, X, _, _, q, x, _, _ = make(dtype, nq, 200, 16, "none", seed=8)
    ids = np.stack([np.random.default_rng(i).permutation(200)[:40] for i in range(nq)])
    s = so.forward(q, x, None, 0.5, None, 0)["lp"]
    z = np.take_along_axis(s, ids, 1).astype(np.float32)
    I, Z = cuda(ids, z)
    if not rest:  # all mass on the listed rows: list them all
        ids = np.tile(np.arange(200), (nq, 1))
        I, Z = cuda(ids, s.astype(np.float32))
        z = s.astype(np.float32)
    r = fg.distill(Q, X, I, Z, scale=0.5, rest=rest)
    o = do.forward(q, x, ids, z, 0.5, 1.0, rest, None)
    check_forward(r, o, so.score_bound(q, x, 0.5, dtype), rest)


@pytest.mark.parametrize("dtype,nq", [("f32", 4), ("f32", 140), ("bf16", 140)])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf"), 3e38])
def test_masked_rows_may_hold_anything(dtype, nq, bad):
    """Rows that a query may not see, named or not, and a query that sees nothing:
    results are those of zeros there."""
    import forgegpu as fg
    import torch
    Q, X, _, _, *_ = make(dtype, nq, 500, 40, "none", seed=2)
    keep = np.random.default_rng(1).random((nq, 500)) < 0.6
    keep[:, [0, 33, 77, 499]] = False
    keep[2] = False
    ids, z = lists(nq, 500, 12, True, seed=1)
    ids[:, 3], ids[:, 7] = 33, 77
    A, I, Z = cuda(so.words(keep), ids, z)
    U = torch.rand(nq, device="cuda")

    def go(X, Q, rest):
        r = fg.distill(Q, X, I, Z, scale=0.3, allowed=A, rest=rest)
        out = [r.loss, r.lse, r.logprobs] + ([r.rest] if rest else [])
        return out + list(fg.distill_backward(Q, X, I, Z, r.lse, r.logprobs, r.rest, d_loss=U,
                                              scale=0.3, allowed=A))

    X0, X1, Q0, Q1 = X.clone(), X.clone(), Q.clone(), Q.clone()
    X0[[0, 33, 77, 499]] = 0
    X1[[0, 33, 77, 499]] = bad
    Q0[2] = 0
    Q1[2] = bad
    for rest in (False, True):
        for a, b in zip(go(X0, Q0, rest), go(X1, Q1, rest)):
            assert not torch.isnan(b).any()
            assert torch.equal(a, b)


@pytest.mark.parametrize("dtype,nq", [("f32", 4), ("f32", 140), ("bf16", 140), ("f16", 20)])
@pytest.mark.parametrize("rest", [False, True])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
def test_what_is_not_finite_reaches_its_queries_only(dtype, nq, rest, bad):
    """A row with it that one query sees (named by it or not), a query with it, a
    logit that is NaN or +inf."""
    import forgegpu as fg
    import torch
    Q, X, _, _, *_ = make(dtype, nq, 300, 40, "none", seed=4)
    keep = np.ones((nq, 300), bool)
    keep[1:, 50] = False
    ids = np.random.default_rng(3).integers(100, 300, (nq, 6))
    z = np.log(np.full((nq, 6), 0.1, np.float32))
    A, I, Z = cuda(so.words(keep), ids, z)
    kw = dict(scale=0.3, allowed=A, rest=rest)
    clean = fg.distill(Q, X, I, Z, **kw)
    X = X.clone()
    X[50, 3] = bad
    Q = Q.clone()
    Q[2, 1] = bad
    for named in (False, True):
        if named:
            I = I.clone()
            I[0, 5] = 50
        r = fg.distill(Q, X, I, Z, **kw)
        for i in (0, 2):
            assert torch.isnan(r.loss[i]) and torch.isnan(r.lse[i])
            assert torch.isnan(r.logprobs[i]).all() and (not rest or torch.isnan(r.rest[i]))
        others = [i for i in range(nq) if i not in (0, 2)]
        for a, b in zip(clean, r):
            assert a is None or torch.equal(a[others], b[others])
        U = torch.rand(nq, device="cuda")
        dq, _ = fg.distill_backward(Q, X, I, Z, r.lse, r.logprobs, r.rest, d_loss=U, scale=0.3,
                                    allowed=A)
        assert torch.isnan(dq[[0, 2]].float()).all() and not torch.isnan(dq[others].float()).any()
    if bad == -float("inf"):
        return
    Q, X, _, _, *_ = make(dtype, nq, 300, 40, "none", seed=4)
    Z = Z.clone()
    Z[1, 2] = bad
    r = fg.distill(Q, X, I, Z, **kw)
    assert torch.isnan(r.loss[1]) and not torch.isnan(r.loss[3:]).any()
    assert not torch.isnan(r.lse).any()
    dq, _ = fg.distill_backward(Q, X, I, Z, r.lse, r.logprobs, r.rest,
                                d_loss=torch.rand(nq, device="cuda"), scale=0.3, allowed=A)
    assert torch.isnan(dq[1].float()).all() and not torch.isnan(dq[3:].float()).any()


@pytest.mark.parametrize("dtype,nq", [("f32", 3), ("f32", 40), ("bf16", 2), ("bf16", 300)])
def test_a_filter_that_leaves_nothing(dtype, nq):
    import forgegpu as fg
    import torch
    Q, X, *_ = make(dtype, nq, 700, 24, "none", seed=13)
    ids, z = lists(nq, 700, 5, True)
    I, Z = cuda(ids, z)
    for rows in (1, nq):
        A = torch.zeros((rows, 22), dtype=torch.int32, device="cuda")
        for rest in (False, True):
            r = fg.distill(Q, X, I, Z, scale=0.5, allowed=A, rest=rest)
            assert (r.loss == 0).all() and (r.lse == -float("inf")).all()
            assert (r.logprobs == 0).all() and (not rest or (r.rest == -float("inf")).all())
            up = torch.ones(nq, device="cuda")
            for g in fg.distill_backward(Q, X, I, Z, r.lse, r.logprobs, r.rest, d_loss=up,
                                         scale=0.5, allowed=A):
                assert (g == 0).all()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_one_row_named_by_all(dtype):
    """Every teacher's list holds the same row: its gradient is the sum of all of
    theirs, in a fixed order."""
    import forgegpu as fg
    import torch
    nq, n = 400, 900
    Q, X, _, _, q, x, _, _ = make(dtype, nq, n, 72, "none", seed=12)
    ids, z = lists(nq, n, 6, True, seed=9)
    ids[:, 0] = 77
    z[:, 0] = -0.5
    o = do.forward(q, x, ids, z, 0.25, 1.0, True, None)
    lse, lp, rl = (o[v].astype(np.float32) for v in ("lse", "logprobs", "rest"))
    up = np.full(nq, 1.0 / nq, np.float32)
    I, Z, L, P, R, U = cuda(ids, z, lse, lp, rl, up)
    run = lambda: fg.distill_backward(Q, X, I, Z, L, P, R, d_loss=U, scale=0.25)  # noqa: E731
    got, again = run(), run()
    r64 = rl.astype(np.float64)
    dq, dx, size = do.backward(q, x, o, ids, lse.astype(np.float64), lp.astype(np.float64), r64,
                               up.astype(np.float64), 0.25)
    es = so.score_bound(q, x, 0.25, dtype)
    bounds = do.gradient_bounds(q, x, o, es, size, dtype, dq, dx, lse, r64, up * 0.25)
    for g, h, w, b in zip(got, again, (dq, dx), bounds):
        assert torch.equal(g, h)
        assert (np.abs(g.double().cpu().numpy() - w) <= b + 1e-30).all()


def test_lists_that_are_parts_of_wider_ones():
    import forgegpu as fg
    import torch
    Q, X, *_ = make("f32", 30, 400, 16, "none", seed=1)
    ids, z = lists(30, 400, 9, False)
    I, Z = cuda(ids, z)
    wide_i = torch.full((30, 14), 3, dtype=torch.int64, device="cuda")
    wide_z = torch.full((30, 11), 9.0, device="cuda")
    wide_i[:, 2:11] = I
    wide_z[:, 1:10] = Z
    a = fg.distill(Q, X, I, Z, scale=0.3)
    b = fg.distill(Q, X, wide_i[:, 2:11], wide_z[:, 1:10], scale=0.3)
    assert all(torch.equal(u, v) for u, v in zip(a[:3], b[:3]))
    U = torch.rand(30, device="cuda")
    g = fg.distill_backward(Q, X, I, Z, a.lse, a.logprobs, d_loss=U, scale=0.3)
    h = fg.distill_backward(Q, X, wide_i[:, 2:11], wide_z[:, 1:10], a.lse, a.logprobs, d_loss=U,
                            scale=0.3)
    assert all(torch.equal(u, v) for u, v in zip(g, h))
    c = fg.distill_backward(Q, X, I, Z, a.lse, a.logprobs, d_loss=U, scale=0.3, need_rows=False)
    d = fg.distill_backward(Q, X, I, Z, a.lse, a.logprobs, d_loss=U, scale=0.3, need_queries=False)
    assert c[1] is None and d[0] is None
    assert torch.equal(g[0], c[0]) and torch.equal(g[1], d[1])


def test_without_queries():
    import forgegpu as fg
    import torch
    x = torch.randn(10, 4, device="cuda")
    i, z = torch.zeros((0, 3), dtype=torch.int64, device="cuda"), torch.zeros((0, 3), device="cuda")
    r = fg.distill(x[:0], x, i, z, rest=True)
    assert r.loss.shape == (0,) and r.logprobs.shape == (0, 3) and r.rest.shape == (0,)
    dq, dx = fg.distill_backward(x[:0], x, i, z, r.lse, r.logprobs, r.rest, d_loss=r.loss)
    assert dq.shape == (0, 4) and not dx.any()


def test_passes_of_a_large_call():
    """More queries than the filters of one pass hold: each query's results are
    those of a call of its own (other sums: 2^-17 of the lse, as a log-softmax in
    other groups)."""
    import forgegpu as fg
    import torch
    g = torch.Generator(device="cuda").manual_seed(0)
    nq, n, d, k = 1100, 2_500_000, 8, 6
    X = torch.randn(n, d, device="cuda", generator=g).bfloat16()
    Q = torch.randn(nq, d, device="cuda", generator=g).bfloat16()
    I = torch.randint(0, n, (nq, k), device="cuda", generator=g)
    Z = torch.full((nq, k), -2.0, device="cuda")
    r = fg.distill(Q, X, I, Z, scale=0.5, rest=True)
    for at in ([0, 1], [831, 832], [856, 857], [1023, 1024], [nq - 2, nq - 1]):
        s = fg.distill(Q[at], X, I[at], Z[at], scale=0.5, rest=True)
        for a, b in zip(r, s):
            assert (a[at] - b).abs().max() <= 2.0 ** -17


def test_offsets_beyond_32_bits():
    """2.2e9 elements of rows: rows past 2^32 bytes and 2^31 elements are named, score and
    get their gradient like copies of them in a small table."""
    import forgegpu as fg
    import torch
    n, d = 2_150_000, 1024
    g = torch.Generator(device="cuda").manual_seed(0)
    X = torch.empty(n, d, dtype=torch.bfloat16, device="cuda")
    for i in range(0, n, 50_000):
        X[i:i + 50_000] = torch.randn(min(50_000, n - i), d, generator=g, device="cuda")
    pick = torch.tensor([0, 1_048_576, 2_097_151, 2_097_152, 2_149_999], device="cuda")
    near = (pick[:, None] + torch.arange(-40, 41, device="cuda")).flatten()
    near = near[(near >= 0) & (near < n)].unique()
    bits = np.zeros((1, n), bool)
    bits[0, near.cpu().numpy()] = True
    keep, = cuda(so.words(bits)[0])
    small = X[near].contiguous()
    I = torch.stack([pick, pick.roll(1), pick.roll(2)], 1).repeat(4, 1)
    where = torch.searchsorted(near, I)
    Q = (X[pick].float() * 1.2).bfloat16().repeat(4, 1)
    Z = torch.log(torch.tensor([[0.5, 0.2, 0.1]], device="cuda")).repeat(20, 1)
    up = torch.full((20,), 0.05, device="cuda")
    for nq in (5, 20):
        a = fg.distill(Q[:nq], X, I[:nq], Z[:nq], scale=0.02, rest=True, allowed=keep)
        b = fg.distill(Q[:nq], small, where[:nq], Z[:nq], scale=0.02, rest=True)
        for u, v in zip(a, b):  # (the same scores in other groups: each lse within 2^-19)
            assert (u - v).abs().max() <= 2.0 ** -17
        ga = fg.distill_backward(Q[:nq], X, I[:nq], Z[:nq], a.lse, a.logprobs, a.rest,
                                 d_loss=up[:nq], scale=0.02, allowed=keep)
        gb = fg.distill_backward(Q[:nq], small, where[:nq], Z[:nq], a.lse, a.logprobs, a.rest,
                                 d_loss=up[:nq], scale=0.02)
        # two roundings to bf16 of sums that differ far below them
        assert ((ga[0] - gb[0]).abs().float() <= 2.0 ** -7 * gb[0].abs().float() + 1e-6).all()
        assert ((ga[1][near] - gb[1]).abs().float() <= 2.0 ** -7 * gb[1].abs().float() + 1e-6).all()
        assert not ga[1][1000:1_048_000].any()


def test_same_call_same_bits_in_graphs_and_on_streams():
    import forgegpu as fg
    import torch
    Q, X, _, A, *_ = make("bf16", 300, 9000, 200, "each", seed=3)
    Q2, X2, _, _, *_ = make("f32", 5, 4000, 96, "none", seed=10)
    I, Z = cuda(*lists(300, 9000, 20, True))
    I2, Z2 = cuda(*lists(5, 4000, 9, False))
    U, U2 = torch.rand(300, device="cuda"), torch.rand(5, device="cuda")

    def one():
        r = fg.distill(Q, X, I, Z, scale=0.2, allowed=A, rest=True)
        return list(r) + list(fg.distill_backward(Q, X, I, Z, r.lse, r.logprobs, r.rest, d_loss=U,
                                                  scale=0.2, allowed=A))

    def two():
        r = fg.distill(Q2, X2, I2, Z2, scale=0.2)
        return list(r[:3]) + list(fg.distill_backward(Q2, X2, I2, Z2, r.lse, r.logprobs,
                                                      d_loss=U2, scale=0.2))

    same = lambda a, b: all(torch.equal(u, v) for u, v in zip(a, b))  # noqa: E731
    graphs = []
    for f in (one, two):
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = f()
        graphs.append((g, out))
    want = [one(), two()]
    assert same(one(), want[0]) and same(two(), want[1])
    side = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    for _ in range(2):
        for s, (g, _) in zip(side, graphs):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        for w, (_, out) in zip(want, graphs):
            assert same(out, w)
    got = [[], []]
    for _ in range(3):  # eager calls at once, each with a workspace of its own
        for i, (s, f) in enumerate(zip(side, (one, two))):
            with torch.cuda.stream(s):
                got[i].append(f())
    torch.cuda.synchronize()
    for w, runs in zip(want, got):
        assert all(same(r, w) for r in runs)
    X.copy_(X.flip(0).clone())
    Z2.copy_(Z2.flip(1).clone())
    for g, _ in graphs:
        g.replay()
    torch.cuda.synchronize()
    assert same(graphs[0][1], one()) and same(graphs[1][1], two())


@pytest.mark.parametrize("dtype,nq,n,dim,mask,rest", [
    ("f32", 1, 10000, 128, "none", False), ("f32", 8, 20000, 64, "each", True),
    ("f32", 300, 9000, 130, "each", True), ("bf16", 40, 5000, 96, "each", True),
    ("bf16", 200, 3000, 65, "none", False), ("f16", 700, 400, 256, "one", True)])
def test_inputs_written_just_before(dtype, nq, n, dim, mask, rest):
    """Kernels of a call overlap, a call and what wrote its inputs do not: calls behind
    writes to their inputs leave what they leave when all is waited for, eager and
    captured with the writes."""
    import forgegpu as fg
    import torch
    sets = []
    for i in range(4):
        Q, X, _, A, *_ = make(dtype, nq, n, dim, mask, seed=50 + i)
        sets.append([Q, X, *cuda(*lists(nq, n, 12, rest, seed=i)), torch.rand(nq, device="cuda")] +
                    ([] if A is None else [A]))
    now = [v.clone() for v in sets[0]]

    def call():
        q, x, ids, z, u = now[:5]
        A = now[5] if len(now) > 5 else None
        r = fg.distill(q, x, ids, z, scale=0.1, rest=rest, allowed=A)
        g = fg.distill_backward(q, x, ids, z, r.lse, r.logprobs, r.rest, d_loss=u, scale=0.1,
                                allowed=A)
        return [v for v in (*r, *g) if v is not None]

    def write(i):
        for v, w in zip(now, sets[i]):
            v.copy_(w)

    want = []
    for i in range(4):
        write(i)
        torch.cuda.synchronize()
        want.append(call())
        torch.cuda.synchronize()

    def run():
        got = []
        for i in (1, 3, 0, 2, 3, 1):
            write(i)
            got.append((i, call()))
        return got

    def check_all(got):
        torch.cuda.synchronize()
        for i, out in got:
            assert all(torch.equal(a, b) for a, b in zip(out, want[i])), i

    check_all(run())
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = run()
    for _ in range(3):
        g.replay()
        check_all(got)


def test_a_wait_that_runs_out(ctx):
    import forgegpu as fg
    import torch
    Q, X, *_ = make("f32", 64, 2000, 64, "none")
    I, Z = cuda(*lists(64, 2000, 7, True))
    want = fg.distill(Q, X, I, Z, rest=True)
    U = torch.rand(64, device="cuda")
    call = lambda r, ws: fg.distill_backward(Q, X, I, Z, r.lse, r.logprobs, r.rest,  # noqa: E731
                                             d_loss=U, workspace=ws)
    grads = call(want, None)
    ws = torch.empty(256 << 20, dtype=torch.uint8, device="cuda")
    ctx.set_wait_limit(0.02)
    try:
        ctx.test_stall_scans(1)
        r = fg.distill(Q, X, I, Z, rest=True, workspace=ws)
        with pytest.raises(fg.ForgeGpuError) as e:
            fg.logprobs_status(ws)
        assert e.value.kind == "Timeout"
        assert all(torch.isnan(v).all() for v in r)
        ctx.test_stall_scans(1)
        g = call(want, ws)
        with pytest.raises(fg.ForgeGpuError) as e:
            fg.logprobs_status(ws)
        assert e.value.kind == "Timeout"
        assert torch.isnan(g[0]).all() and torch.isnan(g[1]).all()
    finally:
        ctx.set_wait_limit(2.0)
    r = fg.distill(Q, X, I, Z, rest=True, workspace=ws)
    fg.logprobs_status(ws)
    assert all(torch.equal(a, b) for a, b in zip(r, want))
    g = call(want, ws)
    fg.logprobs_status(ws)
    assert all(torch.equal(a, b) for a, b in zip(g, grads))


def test_binding_refusals():
    import forgegpu as fg
    import torch
    Q, X, *_ = make("f32", 4, 100, 8, "none")
    I, Z = cuda(*lists(4, 100, 3, False))
    for bad in (lambda: fg.distill(Q, X, I.int(), Z), lambda: fg.distill(Q, X, I, Z.double()),
                lambda: fg.distill(Q, X, I[:3], Z), lambda: fg.distill(Q, X, I, Z[:, :2]),
                lambda: fg.distill(Q, X, I.t(), Z.t()), lambda: fg.distill(Q, X, I[0], Z[0]),
                lambda: fg.distill(Q, X, I, Z, scale=0.0),
                lambda: fg.distill(Q, X, I, Z, teacher_scale=0.0),
                lambda: fg.distill(Q, X, I, Z, teacher_scale=0.5, rest=True),
                lambda: fg.distill(Q, X, I[:, :0], Z[:, :0]), lambda: fg.distill(Q, X[:, :7], I, Z),
                lambda: fg.distill(Q, X, I.repeat(1, 100), Z.repeat(1, 100)),
                lambda: fg.distill(Q, X, I, Z, workspace=torch.empty(256, dtype=torch.uint8,
                                                                     device="cuda"))):
        with pytest.raises(fg.ForgeGpuError):
            bad()
    r = fg.distill(Q, X, I, Z)
    U = torch.ones(4, device="cuda")
    for bad in (lambda: fg.distill_backward(Q, X, I, Z, r.lse[:3], r.logprobs, d_loss=U),
                lambda: fg.distill_backward(Q, X, I, Z, r.lse, r.logprobs[:, :2], d_loss=U),
                lambda: fg.distill_backward(Q, X, I, Z, r.lse, r.logprobs, U[:2], d_loss=U),
                lambda: fg.distill_backward(Q, X, I, Z, r.lse, r.logprobs, d_loss=None)):
        with pytest.raises(fg.ForgeGpuError):
            bad()
