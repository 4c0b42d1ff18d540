"""Distillation and beam search from several threads at once, and under inference mode."""
import threading

import numpy as np
import pytest

from test_gpu_beam import turned
from test_gpu_distill import cuda, lists
from test_gpu_softmax_rows import make

pytestmark = pytest.mark.gpu


def test_two_threads():
    """Each thread on a stream of its own, the calls' sizes and kernels alike or not: what
    each call gives is what it gives alone."""
    import forgegpu as fg
    import torch
    work = []
    for i, (dtype, nq, n, dim) in enumerate([("bf16", 120, 5000, 96), ("f32", 5, 9000, 200),
                                             ("f32", 300, 4000, 64), ("bf16", 120, 5000, 96)]):
        Q, X, *_ = make(dtype, nq, n, dim, "none", seed=i)
        I, Z = cuda(*lists(nq, n, 12, True, seed=i))
        U = torch.rand(nq, device="cuda")
        S = torch.randn(3, 4 + i, 3000 + 500 * i, device="cuda")
        B = torch.zeros(3, 4 + i, device="cuda")

        def go(Q=Q, X=X, I=I, Z=Z, U=U, S=S, B=B):
            r = fg.distill(Q, X, I, Z, scale=0.2, rest=True)
            g = fg.distill_backward(Q, X, I, Z, r.lse, r.logprobs, r.rest, d_loss=U, scale=0.2)
            s = fg.beam_select(S, B)
            t, = fg.beam_reorder([S], s.parents)
            fg.beam_reorder([t], s.parents, out=[t])
            return [*r, *g, *s, t]
        work.append(go)
    want = [go() for go in work]
    torch.cuda.synchronize()
    got, errors = [[] for _ in work], []

    def run(i):
        try:
            stream = torch.cuda.Stream()
            with torch.cuda.stream(stream):
                for _ in range(15):
                    got[i].append(work[i]())
            stream.synchronize()
        except Exception as e:  # noqa: BLE001
            errors.append(e)

    threads = [threading.Thread(target=run, args=(i,)) for i in range(len(work))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors, errors
    torch.cuda.synchronize()
    for i, runs in enumerate(got):
        assert len(runs) == 15
        for r in runs:
            assert all(torch.equal(a, b) for a, b in zip(r, want[i])), i


def test_under_inference_mode():
    """Tensors made there and before, reordered in place and into others, inside and after."""
    import forgegpu as fg
    import torch
    gen = torch.Generator(device="cuda").manual_seed(0)
    parents = torch.tensor([[1, 1, 0, 3], [2, 0, 0, 1]], device="cuda")
    before = torch.randn(2, 4, 50, device="cuda", generator=gen)
    with torch.inference_mode():
        inside = torch.randn(2, 4, 50, device="cuda", generator=gen)
        for t in (before, inside):
            want = turned(t, parents)
            new, = fg.beam_reorder([t], parents)
            out = torch.zeros_like(t)
            fg.beam_reorder([t], parents, out=[out])
            version = None if t.is_inference() else t._version
            fg.beam_reorder([t], parents, out=[t])
            assert version is None or t._version > version
            assert all(torch.equal(v, want) for v in (new, out, t))
        S = torch.randn(2, 4, 9000, device="cuda", generator=gen)
        s = fg.beam_select(S, torch.zeros(2, 4, device="cuda"))
        Q, X = torch.randn(20, 32, device="cuda", generator=gen), torch.randn(700, 32, device="cuda",
                                                                           generator=gen)
        I, Z = cuda(*lists(20, 700, 6, False))
        r = fg.distill(Q, X, I, Z)
    want = turned(inside, parents)
    fg.beam_reorder([inside], parents, out=[inside])
    assert torch.equal(inside, want)
    for a, b in zip(s, fg.beam_select(S, torch.zeros(2, 4, device="cuda"))):
        assert torch.equal(a, b)
    for a, b in zip(r[:3], fg.distill(Q, X, I, Z)[:3]):
        assert torch.equal(a, b)
    assert np.isfinite(r.loss.cpu().numpy()).all()
