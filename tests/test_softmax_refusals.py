"""What the softmax-over-rows and AdamW calls refuse, without a GPU: every
check of arguments comes before any device work."""
import ctypes as C

import numpy as np
import pytest

import softmax_oracle as so


@pytest.fixture()
def call():
    """The library and a zeroed stand-in for a context: no refused call gets
    far enough to use more of it than its multiprocessor count."""
    import forgegpu as fg
    return fg, fg.lib(), C.cast(C.create_string_buffer(1 << 16), C.c_void_p)


BASE = dict(dtype=0, queries=256, nq=4, ld_queries=8, rows=512, n=100, ld_rows=8, dim=8, scale=1.0)


def _bytes(fg, L, ctx, **kw):
    a = fg.LogprobArgs(**{**BASE, **kw})
    n = C.c_size_t()
    rc = L.fdb_logprobs_workspace(ctx, C.byref(a), C.byref(n))
    return rc, n.value


@pytest.mark.parametrize("change,code,text", [
    (dict(dtype=3), -1, b"dtype"), (dict(dtype=-1), -1, b"dtype"),
    (dict(n=0), -10, b"no rows"), (dict(n=1 << 31), -1, b"too many"),
    (dict(nq=1 << 31), -1, b"too many"), (dict(dim=0), -1, b"dim"),
    (dict(dim=16385, ld_queries=16385, ld_rows=16385), -1, b"dim"),
    (dict(scale=0.0), -1, b"scale"), (dict(scale=-1.0), -1, b"scale"),
    (dict(scale=float("nan")), -1, b"scale"), (dict(scale=float("inf")), -1, b"scale"),
    (dict(ld_queries=7), -2, b"ld"), (dict(ld_rows=7), -2, b"ld"),
    (dict(allowed=64, ld_allowed=3), -2, b"ld_allowed"),
    (dict(k=65), -1, b"FDB_MAX_ALTERNATIVES"),
])
def test_forward_refuses(call, change, code, text):
    fg, L, ctx = call
    assert _bytes(fg, L, ctx, **change)[0] == code
    assert text in L.fdb_last_error()
    a = fg.LogprobArgs(**{**BASE, **change})
    assert L.fdb_logprobs(ctx, C.byref(a)) == code


@pytest.mark.parametrize("change,text", [
    (dict(queries=None), b"NULL"), (dict(rows=None), b"NULL"),
    (dict(queries=258), b"queries is not aligned"), (dict(rows=514), b"rows is not aligned"),
    (dict(targets=260), b"targets"), (dict(allowed=258), b"allowed"),
    (dict(workspace=None), b"workspace"), (dict(workspace=1024 + 128), b"workspace"),
    (dict(workspace_bytes=255), b"workspace"), (dict(lse=258), b"output"),
    (dict(k=2), b"top_ids"), (dict(k=2, top_ids=264), b"top_logprobs"),
])
def test_forward_refuses_buffers(call, change, text):
    fg, L, ctx = call
    rc, need = _bytes(fg, L, ctx, **{k: v for k, v in change.items() if k == "k"})
    assert rc == 0 and need > 0
    kw = {**BASE, "workspace": 1024, "workspace_bytes": need, **change}
    a = fg.LogprobArgs(**kw)
    assert L.fdb_logprobs(ctx, C.byref(a)) == -1
    assert text in L.fdb_last_error(), L.fdb_last_error()


def test_no_queries_is_no_work(call):
    fg, L, ctx = call
    a = fg.LogprobArgs(**{**BASE, "nq": 0, "queries": None, "rows": None})
    assert L.fdb_logprobs(ctx, C.byref(a)) == 0
    assert _bytes(fg, L, ctx, nq=0) == (0, 0)


@pytest.mark.parametrize("change,code,text", [
    (dict(n=0), -10, b"no rows"), (dict(scale=0.0), -1, b"scale"),
    (dict(d_queries=256, ld_d_queries=7), -2, b"d_queries"),
    (dict(d_rows=256, ld_d_rows=7), -2, b"d_rows"),
    (dict(d_rows=258, ld_d_rows=8), -1, b"d_rows"),
])
def test_backward_refuses(call, change, code, text):
    fg, L, ctx = call
    a = fg.LogprobGradArgs(**{**BASE, **change})
    assert L.fdb_logprobs_backward(ctx, C.byref(a)) == code
    assert text in L.fdb_last_error()


def test_workspace_sizes_follow_the_work(call):
    fg, L, ctx = call
    small, large = (_bytes(fg, L, ctx, nq=64, n=n, k=4)[1] for n in (1000, 100000))
    assert 0 < small < large
    # a 16-bit operand that a tensor map can describe is not copied
    assert _bytes(fg, L, ctx, dtype=2, nq=64, n=100000)[1] < 8 << 20
    plain = _bytes(fg, L, ctx, dtype=2, nq=64, n=100000)[1]
    copied = _bytes(fg, L, ctx, dtype=2, nq=64, n=100000, ld_rows=9)[1]
    assert copied >= plain + 100000 * 8 * 2


OPTS = dict(param_dtype=0, grad_dtype=0, state_bits=32, lr=1e-3, beta1=0.9, beta2=0.999, eps=1e-8,
            weight_decay=0.01, grad_scale=1.0, step=1)


@pytest.mark.parametrize("change,text", [
    (dict(param_dtype=5), b"dtype"), (dict(grad_dtype=-1), b"dtype"),
    (dict(state_bits=16), b"state_bits"), (dict(beta1=1.0), b"beta"), (dict(beta2=-0.1), b"beta"),
    (dict(eps=0.0), b"eps"), (dict(eps=1e-60), b"eps"), (dict(step=0), b"step"),
    (dict(lr=float("nan")), b"finite"), (dict(grad_scale=float("inf")), b"finite"),
])
def test_adamw_refuses_options(call, change, text):
    fg, L, ctx = call
    t = (fg.AdamwTensor * 1)(fg.AdamwTensor(4096, 8192, 12288, 16384, None, None, 10))
    o = fg.AdamwOpts(**{**OPTS, **change})
    assert L.fdb_adamw_step(ctx, C.byref(t), 1, C.byref(o)) == -1
    assert text in L.fdb_last_error()


def test_adamw_refuses_tensors(call):
    fg, L, ctx = call
    T = fg.AdamwTensor

    def rc(*ts, **o):
        arr = (T * len(ts))(*ts)
        return L.fdb_adamw_step(ctx, C.byref(arr), len(ts), C.byref(fg.AdamwOpts(**{**OPTS, **o})))

    ok = T(4096, 8192, 12288, 16384, None, None, 10)
    for bad in (T(None, 8192, 12288, 16384, None, None, 10),
                T(4096, 8192, None, 16384, None, None, 10),
                T(4098, 8192, 12288, 16384, None, None, 10),
                T(4096, 8193, 12288, 16384, None, None, 10),
                T(4096, 8192, 12289, 16384, None, None, 10)):
        assert rc(bad) == -1
    assert rc(ok, ok) == -1 and b"overlap" in L.fdb_last_error()
    assert rc(ok, T(4096 + 36, 8192, 12288, 16384, None, None, 4)) == -1
    assert b"overlap" in L.fdb_last_error()
    assert rc(ok, state_bits=8) == -1 and b"NULL" in L.fdb_last_error()
    # nothing to do is not an error, and needs no device
    assert L.fdb_adamw_state_values(ctx, None, None, None, None, 1, None, None, None) == -1


def test_python_binding_refuses_cpu_tensors():
    import forgegpu as fg
    import torch
    q, x = torch.zeros(2, 4), torch.zeros(5, 4)
    with pytest.raises(fg.ForgeGpuError):
        fg.logprobs(q, x)
    with pytest.raises(fg.ForgeGpuError):
        fg.logprobs_backward(q, x, None, torch.zeros(2))
    with pytest.raises(fg.ForgeGpuError):
        fg.adamw_step([q], [q], [q], [q], lr=1e-3)
    with pytest.raises(fg.ForgeGpuError):
        fg.adamw_step([q], [q], [q], [], lr=1e-3)
    with pytest.raises(fg.ForgeGpuError):
        fg.adamw_state_values(q, q, q, q)


# ---- the oracles themselves -------------------------------------------------
def test_oracle_gradient_against_differences():
    """The formula of the gradient against central differences of the outputs:
    an error of order h^2 = 1e-10, times third derivatives of order 1e2."""
    rng = np.random.default_rng(0)
    nq, n, d, scale = 5, 40, 6, 0.7
    q, x = rng.standard_normal((nq, d)), rng.standard_normal((n, d))
    t = np.array([3, 7, -1, 39, 0])
    keep = rng.random((nq, n)) < 0.7
    keep[4, 0] = False
    keep[1] = False
    al = so.words(keep)
    up = rng.standard_normal((3, nq))

    def loss(q, x):
        f = so.forward(q, x, t, scale, al, 0)
        parts = [np.where(np.isfinite(f[k]), f[k], 0.0) for k in ("logprob", "lse", "entropy")]
        return sum((u * v).sum() for u, v in zip(up, parts))

    f = so.forward(q, x, t, scale, al, 0)
    dq, dx, _, _ = so.backward(q, x, t, f["lse"], f["entropy"], up[0], up[1], up[2], scale, al)
    for _ in range(6):
        a, b, h = rng.standard_normal((nq, d)), rng.standard_normal((n, d)), 1e-5
        diff = (loss(q + h * a, x + h * b) - loss(q - h * a, x - h * b)) / (2 * h)
        assert abs(diff - ((dq * a).sum() + (dx * b).sum())) < 1e-7


def test_oracle_codes_keep_the_mean():
    """A value between two codes goes up with the probability that keeps its
    mean: over 4096 steps the mean is within 5 standard deviations."""
    rng = np.random.default_rng(1)
    m = rng.standard_normal(256).astype(np.float32)
    v = (rng.random(256) ** 3).astype(np.float32) + np.float32(1e-3)
    acc = np.zeros((2, 256))
    sq = np.zeros((2, 256))
    reps = 4096
    for step in range(reps):
        cm, sm, cv, sv = so.codes8(m, v, seed=9, step=step, ordinal=0)
        got = np.stack(so.values8(cm, sm, cv, sv)).astype(np.float64)
        acc += got
        sq += got ** 2
    mean = acc / reps
    sd = np.sqrt(np.maximum(sq / reps - mean ** 2, 0) / reps)
    assert (np.abs(mean - np.stack([m, v])) <= 5 * sd + 1e-6 * np.abs(mean)).all()
