"""Distillation where the last bits of scores count: the loss of a student that agrees is
not below 0."""
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
