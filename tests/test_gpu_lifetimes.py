"""Contexts and indexes may be freed in any order, as a garbage collector does
with objects that refer to one another."""
import gc

import numpy as np
import pytest

pytestmark = pytest.mark.gpu


def _bf(fg, ctx, x):
    return fg.BruteForceIndex(fg.DistanceMetric.DotProduct, ctx).add(x)


def test_an_index_outlives_its_context():
    import forgegpu as fg
    rng = np.random.default_rng(0)
    x = rng.standard_normal((3000, 32)).astype(np.float32)
    q = rng.standard_normal((5, 32)).astype(np.float32)
    ctx = fg.Context(0)
    bf = _bf(fg, ctx, x)
    iv = fg.IVFPQIndex.build(x, 8, 8, ctx=ctx, seed=1)
    want = bf.batch_search_arrays(q, 3), iv.batch_search_arrays(q, 3)
    ctx.close()
    got = bf.batch_search_arrays(q, 3), iv.batch_search_arrays(q, 3)
    for a, b in zip(want, got):
        assert np.array_equal(a[0], b[0]) and np.array_equal(a[1], b[1])
    p = bf.log_probs(q, k=3)
    assert np.array_equal(p.top_ids, want[0][0])
    iv.close()
    assert np.array_equal(bf.log_probs(q, k=3).top_ids, p.top_ids)
    bf.close()
    other = _bf(fg, fg.Context(0), x)
    assert np.array_equal(other.batch_search_arrays(q, 3)[0], want[0][0])


def test_a_cycle_of_a_context_and_its_indexes_is_collected():
    """Cycles with the context in front of and behind its indexes; the next
    call finds no error that freeing them left."""
    import forgegpu as fg
    rng = np.random.default_rng(0)
    x = rng.standard_normal((500, 16)).astype(np.float32)
    keep = _bf(fg, fg.default_context(), x)
    for first in (True, False):
        for _ in range(4):
            ctx = fg.Context(0)
            parts = [_bf(fg, ctx, x) for _ in range(2)]
            cycle = [ctx, *parts] if first else [*parts, ctx]
            cycle.append(cycle)
            for p in parts:
                p.cycle = cycle
            ctx.cycle = cycle
            del ctx, parts, cycle, p
            gc.collect()
            assert keep.batch_search_arrays(x[:3], 1)[0].shape == (3, 1)


def test_a_failed_call_does_not_fail_the_next():
    """An allocation that cannot be had is reported once: the next call's
    launches do not find its error."""
    import ctypes as C

    import forgegpu as fg
    import torch
    rng = np.random.default_rng(0)
    x = rng.standard_normal((500, 16)).astype(np.float32)
    ix = _bf(fg, fg.default_context(), x)
    q = torch.randn(3, 16, device="cuda")
    want = ix.batch_search_arrays(x[:3], 2), fg.logprobs(q, q)
    out = C.c_void_p()
    for again in (lambda: ix.batch_search_arrays(x[:3], 2)[0], lambda: fg.logprobs(q, q).lse):
        assert fg.lib().fdb_host_alloc(1 << 60, C.byref(out)) != 0
        assert b"cudaHostAlloc" in fg.lib().fdb_last_error()
        got = again()
    assert np.array_equal(ix.batch_search_arrays(x[:3], 2)[0], want[0][0])
    assert torch.equal(got, want[1].lse)


_CAPTURED = r"""
import sys
sys.path.insert(0, %r)
import torch
import forgegpu as fg
q = torch.randn(20, 64, device="cuda")
x = torch.randn(3000, 64, device="cuda")
t = torch.arange(20, device="cuda")
up = torch.rand(20, device="cuda")
p, m, v = [x.clone()], [torch.zeros_like(x)], [torch.zeros_like(x)]

def step():
    r = fg.logprobs(q, x, t, scale=0.2, k=4)
    d = fg.logprobs_backward(q, x, t, r.lse, d_logprob=up, scale=0.2)
    fg.adamw_step(p, [d[1]], m, v, lr=1e-2)
    return list(r) + list(d)

torch.cuda.synchronize()
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):  # the first call of the process: its context is made here
    out = step()
g.replay()
torch.cuda.synchronize()
got = [a.clone() for a in out]
assert all(torch.equal(a, b) for a, b in zip(got, step()))
print("SAME")
"""


def test_the_first_call_of_a_process_is_captured():
    import os
    import subprocess
    import sys
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    r = subprocess.run([sys.executable, "-c", _CAPTURED % os.path.join(root, "forge-db_b200")],
                       capture_output=True, text=True, timeout=180)
    assert r.returncode == 0 and "SAME" in r.stdout, r.stderr[-3000:]
