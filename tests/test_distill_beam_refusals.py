"""What the distillation and beam-search calls refuse, without a GPU: every check of
arguments comes before any device work."""
import ctypes as C

import numpy as np
import pytest

import distill_oracle as do
import softmax_oracle as so


@pytest.fixture()
def call():
    import forgegpu as fg
    return fg, fg.lib(), C.cast(C.create_string_buffer(1 << 16), C.c_void_p)


BASE = dict(dtype=0, queries=256, nq=4, ld_queries=8, rows=512, n=100, ld_rows=8, dim=8, scale=1.0,
            teacher_ids=1024, teacher_logits=2048, k=3, ld_ids=3, ld_logits=3, teacher_scale=1.0)
GRAD = dict(lse=256, logprobs=512, rest_logprob=768, d_loss=1024, d_queries=4096, ld_d_queries=8,
            d_rows=8192, ld_d_rows=8)
BEAM = dict(dtype=0, scores=256, groups=2, beams=3, n=1000, ld_group=3000, ld_beam=1000, scale=1.0,
            normalise=1, beam_scores=512, width=3, out_scores=1024, out_parents=2048, out_ids=4096)


@pytest.mark.parametrize("change,code,text", [
    (dict(dtype=3), -1, b"dtype"), (dict(n=0), -10, b"no rows"), (dict(n=1 << 31), -1, b"too many"),
    (dict(nq=1 << 31), -1, b"too many"), (dict(dim=0), -1, b"dim"),
    (dict(scale=0.0), -1, b"scale"), (dict(scale=float("nan")), -1, b"scale"),
    (dict(ld_queries=7), -2, b"ld"), (dict(ld_rows=7), -2, b"ld"),
    (dict(allowed=64, ld_allowed=3), -2, b"ld_allowed"), (dict(k=0), -1, b"FDB_MAX_TEACHER"),
    (dict(k=257, ld_ids=257, ld_logits=257), -1, b"FDB_MAX_TEACHER"),
    (dict(ld_ids=2), -2, b"ld is below k"), (dict(ld_logits=2), -2, b"ld is below k"),
    (dict(teacher_scale=0.0), -1, b"teacher_scale"),
    (dict(teacher_scale=float("nan")), -1, b"teacher_scale"),
    (dict(teacher_scale=0.5, rest=1), -1, b"teacher_scale of 1"),
])
def test_both_refuse(call, change, code, text):
    fg, L, ctx = call
    n = C.c_size_t()
    for args, size, run in ((fg.DistillArgs(**{**BASE, **change}), L.fdb_distill_workspace,
                             L.fdb_distill),
                            (fg.DistillGradArgs(**{**BASE, **GRAD, **change}),
                             L.fdb_distill_backward_workspace, L.fdb_distill_backward)):
        assert size(ctx, C.byref(args), C.byref(n)) == code
        assert text in L.fdb_last_error()
        assert run(ctx, C.byref(args)) == code
        assert text in L.fdb_last_error()


@pytest.mark.parametrize("grad", [False, True])
@pytest.mark.parametrize("rest", [0, 1])
@pytest.mark.parametrize("change,text", [
    (dict(queries=None), b"NULL"), (dict(rows=None), b"NULL"), (dict(teacher_ids=None), b"teacher"),
    (dict(teacher_logits=None), b"teacher"), (dict(queries=258), b"queries is not aligned"),
    (dict(rows=514), b"rows is not aligned"), (dict(teacher_ids=1028), b"teacher_ids"),
    (dict(teacher_logits=2050), b"teacher_logits"), (dict(allowed=258), b"allowed"),
    (dict(workspace=None), b"workspace"), (dict(workspace=1024 + 128), b"workspace"),
    (dict(workspace_bytes=255), b"workspace"), (dict(lse=258), b"put"),
    (dict(logprobs=258), b"put"),
])
def test_buffers(call, grad, rest, change, text):
    fg, L, ctx = call
    kind, size, run = (fg.DistillGradArgs, L.fdb_distill_backward_workspace,
                       L.fdb_distill_backward) if grad else (
        fg.DistillArgs, L.fdb_distill_workspace, L.fdb_distill)
    base = {**BASE, **(GRAD if grad else {}), "rest": rest}
    n = C.c_size_t()
    assert size(ctx, C.byref(kind(**base)), C.byref(n)) == 0 and n.value > 0
    a = kind(**{**base, "workspace": 1024, "workspace_bytes": n.value, **change})
    assert run(ctx, C.byref(a)) == -1
    assert text in L.fdb_last_error()


@pytest.mark.parametrize("change,code,text", [
    (dict(lse=None), -1, b"NULL"), (dict(logprobs=None), -1, b"NULL"),
    (dict(d_loss=None), -1, b"NULL"), (dict(rest=1, rest_logprob=None), -1, b"NULL"),
    (dict(ld_d_queries=7), -2, b"d_queries rows overlap"),
    (dict(ld_d_rows=7), -2, b"d_rows rows overlap"), (dict(d_rows=8194), -1, b"d_rows"),
    (dict(d_loss=1026), -1, b"input"),
])
def test_gradient_buffers(call, change, code, text):
    fg, L, ctx = call
    a = fg.DistillGradArgs(**{**BASE, **GRAD, "workspace": 1024, "workspace_bytes": 1 << 40,
                              **change})
    assert L.fdb_distill_backward(ctx, C.byref(a)) == code
    assert text in L.fdb_last_error()


@pytest.mark.parametrize("change,code,text", [
    (dict(dtype=5), -1, b"dtype"), (dict(n=0), -10, b"no columns"), (dict(n=1 << 31), -1, b"columns"),
    (dict(beams=0), -1, b"FDB_MAX_BEAMS"), (dict(beams=129), -1, b"FDB_MAX_BEAMS"),
    (dict(width=0), -1, b"FDB_MAX_BEAMS"), (dict(width=129), -1, b"FDB_MAX_BEAMS"),
    (dict(groups=1 << 22), -1, b"groups"), (dict(scale=0.0), -1, b"scale"),
    (dict(scale=float("inf")), -1, b"scale"), (dict(ld_beam=999), -2, b"ld_beam"),
    (dict(ids=64, ld_ids=999), -2, b"ld_ids"), (dict(allowed=64, ld_allowed=31), -2, b"ld_allowed"),
])
def test_select_refuses(call, change, code, text):
    fg, L, ctx = call
    n = C.c_size_t()
    a = fg.BeamArgs(**{**BEAM, **change})
    assert L.fdb_beam_select_workspace(ctx, C.byref(a), C.byref(n)) == code
    assert text in L.fdb_last_error()
    assert L.fdb_beam_select(ctx, C.byref(a)) == code


@pytest.mark.parametrize("change,text", [
    (dict(scores=None), b"NULL"), (dict(beam_scores=None), b"NULL"), (dict(out_scores=None), b"NULL"),
    (dict(out_parents=None), b"NULL"), (dict(out_ids=None), b"NULL"), (dict(scores=258), b"scores"),
    (dict(ids=260, ld_ids=1000), b"ids"), (dict(beam_scores=514), b"beam_scores"),
    (dict(out_parents=2052), b"out_parents"), (dict(out_ids=4100), b"out_ids"),
    (dict(workspace=None), b"workspace"), (dict(workspace=1024 + 128), b"workspace"),
    (dict(workspace_bytes=1), b"workspace"), (dict(out_scores=512), b"an output is an input"),
    (dict(ended=600, out_ended=600), b"an output is an input"),
    (dict(ids=4096, ld_ids=1000), b"an output is an input"), (dict(out_ids=2048), b"another output"),
])
def test_select_buffers(call, change, text):
    fg, L, ctx = call
    a = fg.BeamArgs(**{**BEAM, "workspace": 1024, "workspace_bytes": 1 << 40, **change})
    assert L.fdb_beam_select(ctx, C.byref(a)) == -1
    assert text in L.fdb_last_error()


def test_reorder_refuses(call):
    fg, L, ctx = call

    def run(state, **kw):
        opts = fg.ReorderOpts(**{**dict(parents=64, groups=2, beams=3, width=3), **kw})
        table = (C.c_uint64 * 8)(*state)
        return L.fdb_beam_reorder(ctx, C.addressof(table), 1, C.byref(opts))

    good = (256, 4096, 64, 64, 1, 0, 0, 64)
    for kw in (dict(beams=0), dict(beams=129), dict(width=0), dict(width=129), dict(groups=1 << 22),
               dict(parents=None), dict(parents=68)):
        assert run(good, **kw) == -1
    assert run((0,) + good[1:]) == -1 and run(good[:1] + (0,) + good[2:]) == -1
    assert run((256, 4096, 64, 64, 2, 16, 16, 64)) == -2          # runs that overlap
    assert run((256, 4096, 64, 0, 1, 0, 0, 64)) == -2             # rows on top of each other
    assert run((256, 4096, 64, 48, 1, 0, 0, 64)) == -2
    assert run((256, 4096, 64, 80, 2, 100, 100, 64)) == -2        # runs between the rows
    assert run((256, 256, 64, 64, 1, 0, 0, 64), width=2) == -1    # in place, another width
    assert run((256, 256, 64, 128, 1, 0, 0, 64)) == -1            # in place, other strides


def test_reorder_refuses_states_that_meet(call):
    fg, L, ctx = call
    opts = fg.ReorderOpts(parents=64, groups=2, beams=3, width=3)

    def run(*pairs):
        flat = [v for s, d in pairs for v in (s, d, 64, 64, 1, 0, 0, 64)]
        table = (C.c_uint64 * len(flat))(*flat)
        return L.fdb_beam_reorder(ctx, C.addressof(table), len(pairs), C.byref(opts))

    assert run((4096, 8192), (12288, 8192)) == -1                 # one place for two
    assert run((4096, 4096), (4096, 4096)) == -1
    assert run((4096, 8192), (8192, 4096)) == -1                  # each other's places
    assert run((4096, 4096), (4096, 8192)) == -1                  # turned and read
    assert b"written" in L.fdb_last_error()


def test_oracle_gradient_against_differences():
    """The 64-bit gradient of the 64-bit loss: central differences with h = 1e-5 are off by
    h^2 times third derivatives of size 1, and by 2^-52 / h."""
    rng = np.random.default_rng(0)
    nq, n, d, k = 6, 30, 8, 5
    q, x, u = rng.standard_normal((nq, d)), rng.standard_normal((n, d)), rng.standard_normal(nq)
    al = so.words(rng.random((nq, n)) < 0.7)
    ids = rng.integers(-1, n, (nq, k))
    z = np.log(rng.dirichlet(np.ones(k + 1), nq)[:, :k]).astype(np.float32)
    for rest in (False, True):
        o = do.forward(q, x, ids, z, 0.5, 1.0, rest, al)
        assert (o["loss"] >= -1e-9).all()
        dq, dx, _ = do.backward(q, x, o, ids, o["lse"], o["logprobs"], o["rest"] if rest else None,
                                u, 0.5)
        loss = lambda q, x: (u * do.forward(q, x, ids, z, 0.5, 1.0, rest, al)["loss"]).sum()  # noqa
        for _ in range(3):
            a, b, h = rng.standard_normal(q.shape), rng.standard_normal(x.shape), 1e-5
            diff = (loss(q + h * a, x + h * b) - loss(q - h * a, x - h * b)) / (2 * h)
            assert abs(diff - ((dq * a).sum() + (dx * b).sum())) < 1e-6
