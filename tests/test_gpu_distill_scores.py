"""Distillation where the last bits of scores count: the loss of a student that agrees is
not below 0, and the named rows' scores hold what a sum of large terms leaves."""
import numpy as np
import pytest

import distill_oracle as do
import softmax_oracle as so
from test_gpu_distill import cuda
from test_gpu_softmax_rows import make

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype,nq", [("f32", 1), ("f32", 8), ("f32", 300), ("bf16", 4), ("bf16", 300),
                                      ("f16", 60)])
@pytest.mark.parametrize("rest", [False, True])
def test_a_loss_is_not_below_zero(dtype, nq, rest):
    """A teacher that says what the student does, to the rounding of its logits: a
    divergence of 0 but for roundings, which may not leave it below 0.  A loss with a NaN
    in it stays NaN."""
    import forgegpu as fg
    for seed in range(4):
        Q, X, _, _, q, x, _, _ = make(dtype, nq, 200, 16, "none", seed=seed)
        s = so.forward(q, x, None, 0.5, None, 0)["lp"]
        ids = np.stack([np.random.default_rng(i).permutation(200)[:40 if rest else 200]
                        for i in range(nq)])
        z = np.take_along_axis(s, ids, 1).astype(np.float32)
        I, Z = cuda(ids, z)
        r = fg.distill(Q, X, I, Z, scale=0.5, rest=rest)
        o = do.forward(q, x, ids, z, 0.5, 1.0, rest, None)
        off = np.abs(r.loss.double().cpu().numpy() - o["loss"])
        assert (off <= do.forward_bounds(o, so.score_bound(q, x, 0.5, dtype))["loss"]).all()
        assert (r.loss >= 0).all(), r.loss.min()
        r = fg.distill(Q, X, I, r.logprobs, scale=0.5, rest=rest)  # (of the kernel's own)
        assert (r.loss >= 0).all(), r.loss.min()
        Z[0, 3] = float("nan")
        r = fg.distill(Q, X, I, Z, scale=0.5, rest=rest)
        assert r.loss[0].isnan() and (r.loss[1:] >= 0).all()


CANCEL = [
    # dtype, nq, n, half of dim, pad, shift
    ("f32", 3, 300, 32, 0, 0), ("f32", 40, 300, 200, 0, 0), ("f32", 40, 300, 333, 2, 0),
    ("f32", 9, 300, 50, 1, 1), ("bf16", 3, 300, 64, 0, 0), ("bf16", 40, 500, 384, 0, 0),
    ("bf16", 20, 300, 90, 4, 4), ("bf16", 20, 300, 130, 2, 0), ("bf16", 5, 300, 77, 1, 1),
    ("f16", 400, 300, 128, 0, 0), ("f16", 700, 300, 20, 0, 0), ("f16", 12, 300, 101, 1, 0),
    ("f32", 2, 40, 8192, 0, 0), ("f32", 30, 40, 8192, 0, 0), ("bf16", 30, 40, 8192, 0, 0),
]


@pytest.mark.parametrize("dtype,nq,n,half,pad,shift", CANCEL)
@pytest.mark.parametrize("rest", [False, True])
def test_named_scores_are_sums_in_64_bits(dtype, nq, n, half, pad, shift, rest):
    """Rows [a + e, f - a], queries [b, b]: scores are what large terms leave of one another,
    so that sums in f32 are off by 2^-24 of the terms, some 1e-4.  Two entries of a list
    share their lse, whatever that is off by: their log probabilities differ by their
    scores.  Products of f32 are exact in 64 bits (of 16-bit types in 32), dim of them are
    added: (dim + 4) 2^-52 of their sizes covers that, the product with the scale and the
    difference to the lse; and each log probability is rounded once."""
    import forgegpu as fg
    import torch
    rng = np.random.default_rng(half + nq)
    d = 2 * half
    dt = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}[dtype]

    def put(v):
        buf = torch.zeros(shift + v.shape[0] * (d + pad), dtype=dt, device="cuda")
        t = buf[shift:].view(v.shape[0], d + pad)[:, :d]
        t.copy_(torch.from_numpy(v))
        return t

    a, b = rng.standard_normal((1, half)) * 100.0, rng.standard_normal((nq, half))
    e, f = rng.standard_normal((2, n, half)) * (0.1 if dtype == "f32" else 1.0)
    order = rng.permutation(d)  # (so that no order of adding up cancels by itself)
    Q = put(np.concatenate([b, b], 1)[:, order])
    X = put(np.concatenate([a + e, f - a], 1)[:, order])
    q, x = Q.double().cpu().numpy(), X.double().cpu().numpy()
    ids = np.stack([rng.permutation(n)[:17] for _ in range(nq)])
    z = np.log(rng.dirichlet(np.ones(18), nq)[:, :17]).astype(np.float32)
    I, Z = cuda(ids, z)
    scale = 0.5
    r = fg.distill(Q, X, I, Z, scale=scale, rest=rest)
    lp = r.logprobs.double().cpu().numpy()
    s = np.einsum("qd,qkd->qk", q, x[ids]) * scale
    size = np.einsum("qd,qkd->qk", np.abs(q), np.abs(x[ids])) * scale
    off = np.abs((lp - lp[:, :1]) - (s - s[:, :1]))
    bound = do.H32 * (np.abs(lp) + np.abs(lp[:, :1])) + (d + 4) * 2.0 ** -52 * (size + size[:, :1])
    assert (off <= bound).all(), (off / bound).max()
    if rest:
        return
    # (a target's log probability under the same sums over all rows: of the same bits)
    p = fg.logprobs(Q, X, I[:, 3].contiguous(), scale=scale)
    off = (p.logprob - r.logprobs[:, 3]).double().abs().cpu().numpy()
    lse = (p.lse - r.lse).double().abs().cpu().numpy()
    far = np.abs(lp[:, 3]) + 2 * np.abs(r.lse.double().cpu().numpy())
    assert (off <= lse + 2 * do.H32 * far).all()


@pytest.mark.parametrize("dtype,nq,n,d", [("f16", 20, 262144, 1024), ("f16", 300, 100003, 512),
                                          ("bf16", 20, 262144, 1024), ("f32", 20, 262144, 256)])
def test_what_sums_lose_is_added_where_the_mass_lies(dtype, nq, n, d):
    """One row scores 10, all others 0, by sums of integers that lose nothing.  What a tensor
    core's sum of terms of one sign loses, 5.2e-8 a step of 16 columns (bf16 2.3e-8), is half
    added to every score, so that each is off by at most that share of itself here, and the
    lse by that share of their mean under the softmax, 0.8 or 1.8, however large the largest
    is.  Exponentials and f32 sums have 2^-20 and the output its rounding, as everywhere."""
    import forgegpu as fg
    import torch
    dt = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}[dtype]
    Q = torch.ones(nq, d, dtype=dt, device="cuda")
    X = torch.ones(n, d, dtype=dt, device="cuda")
    X[:, 1::2] = -1
    X[n // 3] = 1
    scale = float(np.float32(10 / d))
    I = torch.full((nq, 1), 5, dtype=torch.int64, device="cuda")
    r = fg.distill(Q, X, I, torch.zeros(nq, 1, device="cuda"), scale=scale)
    top = scale * d
    want = np.log(np.exp(top) + (n - 1))
    mean = top * np.exp(top - want)
    share = (2.3e-8 if dtype == "bf16" else 5.2e-8) / 2 * (d / 16)
    off = (r.lse.double() - want).abs().max().item()
    assert off <= share * mean + 2.0 ** -20 + do.H32 * want, off
