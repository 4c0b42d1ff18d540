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
