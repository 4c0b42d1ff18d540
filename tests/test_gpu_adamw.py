"""The AdamW step against the same operations in f32 on the CPU, bit for bit,
and a training step made of the three operators."""
import numpy as np
import pytest

import softmax_oracle as so

pytestmark = pytest.mark.gpu

OPT = dict(lr=1e-2, step=3, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.02)
ORC = dict(lr=1e-2, step=3, betas=(0.9, 0.999), eps=1e-8, wd=0.02)


def _dt(name):
    import torch
    return {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}[name]


def _put(a, dtype, shift=0):
    """A tensor of these values whose first element lies `shift` past an aligned address."""
    import torch
    buf = torch.empty(a.size + shift, dtype=dtype, device="cuda")
    buf[shift:].copy_(torch.from_numpy(np.ascontiguousarray(a)))
    return buf[shift:]


def _round(p, name):
    """Rounds f32 values to the parameters' type and back."""
    import torch
    return torch.from_numpy(p).to(_dt(name)).float().numpy()


def _inputs(sizes, pname, gname, seed=0):
    rng = np.random.default_rng(seed)
    ps = [_round(rng.standard_normal(n).astype(np.float32), pname) for n in sizes]
    gs = [_round((rng.standard_normal(n) * 10.0 ** rng.integers(-4, 1)).astype(np.float32), gname)
          for n in sizes]
    ms = [(0.5 * g + 0.1 * rng.standard_normal(g.size).astype(np.float32) * np.abs(g).max()
           ).astype(np.float32) for g in gs]
    vs = [(g * g * np.float32(0.7) + np.float32(1e-12)).astype(np.float32) for g in gs]
    return ps, gs, ms, vs


SIZES = [1, 2, 255, 256, 257, 8191, 8192, 8193, 30000]


@pytest.mark.parametrize("pname,gname,shift", [("f32", "f32", 0), ("f32", "f32", 1),
                                               ("bf16", "bf16", 0), ("bf16", "f32", 3),
                                               ("f16", "f16", 0), ("f32", "bf16", 0)])
def test_step_32(pname, gname, shift):
    import forgegpu as fg
    import torch
    ps, gs, ms, vs = _inputs(SIZES, pname, gname)
    P, G = [_put(p, _dt(pname), shift) for p in ps], [_put(g, _dt(gname), shift) for g in gs]
    M, V = [_put(m, torch.float32, shift) for m in ms], [_put(v, torch.float32) for v in vs]
    fg.adamw_step(P, G, M, V, **OPT)
    for i in range(len(SIZES)):
        p, m, v = so.adamw(ps[i], gs[i], ms[i], vs[i], **ORC)
        assert np.array_equal(M[i].cpu().numpy(), m) and np.array_equal(V[i].cpu().numpy(), v)
        assert np.array_equal(P[i].float().cpu().numpy(), _round(p, pname)), SIZES[i]


@pytest.mark.parametrize("pname,gname,shift", [("f32", "f32", 0), ("bf16", "bf16", 0),
                                               ("bf16", "f32", 1), ("f16", "f16", 0)])
def test_step_8(pname, gname, shift):
    import forgegpu as fg
    import torch
    ps, gs, ms, vs = _inputs(SIZES, pname, gname, seed=1)
    codes = [so.codes8(m, v, seed=1, step=1, ordinal=i) for i, (m, v) in enumerate(zip(ms, vs))]
    P, G = [_put(p, _dt(pname), shift) for p in ps], [_put(g, _dt(gname), shift) for g in gs]
    M, V = [_put(c[0], torch.int8, shift) for c in codes], [_put(c[2], torch.uint8) for c in codes]
    MS = [_put(c[1], torch.float32) for c in codes]
    VS = [_put(c[3], torch.float32, shift) for c in codes]
    fg.adamw_step(P, G, M, V, m_scales=MS, v_scales=VS, seed=77, **OPT)
    for i in range(len(SIZES)):
        m0, v0 = so.values8(*codes[i])
        p, m, v = so.adamw(ps[i], gs[i], m0, v0, **ORC)
        cm, sm, cv, sv = so.codes8(m, v, seed=77, step=3, ordinal=i)
        assert np.array_equal(M[i].cpu().numpy(), cm) and np.array_equal(MS[i].cpu().numpy(), sm)
        assert np.array_equal(V[i].cpu().numpy(), cv) and np.array_equal(VS[i].cpu().numpy(), sv)
        assert np.array_equal(P[i].float().cpu().numpy(), _round(p, pname))
        vm, vv = fg.adamw_state_values(M[i], MS[i], V[i], VS[i])
        wm, wv = so.values8(cm, sm, cv, sv)
        assert np.array_equal(vm.cpu().numpy(), wm) and np.array_equal(vv.cpu().numpy(), wv)


@pytest.mark.parametrize("bits", [32, 8])
def test_many_tensors_and_empty_ones(bits):
    import forgegpu as fg
    import torch
    rng = np.random.default_rng(4)
    sizes = [int(s) for s in rng.integers(0, 600, 250)]
    ps, gs, ms, vs = _inputs([max(s, 1) for s in sizes], "f32", "f32")
    ps, gs, ms, vs = ([a[:s] for a, s in zip(x, sizes)] for x in (ps, gs, ms, vs))
    P, G = [_put(p, torch.float32) for p in ps], [_put(g, torch.float32) for g in gs]
    if bits == 32:
        M, V = [_put(m, torch.float32) for m in ms], [_put(v, torch.float32) for v in vs]
        fg.adamw_step(P, G, M, V, **OPT)
    else:  # from the initial state: zeros
        M = [torch.zeros(s, dtype=torch.int8, device="cuda") for s in sizes]
        V = [torch.zeros(s, dtype=torch.uint8, device="cuda") for s in sizes]
        MS, VS = ([torch.zeros((s + 255) // 256, device="cuda") for s in sizes] for _ in range(2))
        fg.adamw_step(P, G, M, V, m_scales=MS, v_scales=VS, **OPT)
    for i, s in enumerate(sizes):
        if not s:
            continue
        z = np.zeros(s, np.float32)
        p, m, v = so.adamw(ps[i], gs[i], ms[i] if bits == 32 else z, vs[i] if bits == 32 else z,
                           **ORC)
        assert np.array_equal(P[i].cpu().numpy(), p)
        if bits == 8:
            cm, sm, cv, sv = so.codes8(m, v, seed=0, step=3, ordinal=i)
            assert np.array_equal(M[i].cpu().numpy(), cm) and np.array_equal(V[i].cpu().numpy(), cv)


def test_values_from_the_device_and_a_replayed_graph():
    """lr, step and the gradient's scale read when the kernels run."""
    import forgegpu as fg
    import torch
    ps, gs, ms, vs = _inputs([1000], "f32", "f32")
    P, G = [_put(ps[0], torch.float32)], [_put(gs[0], torch.float32)]
    M, V = [_put(ms[0], torch.float32)], [_put(vs[0], torch.float32)]
    lr = torch.tensor([1e-2], device="cuda")
    step = torch.tensor([3], dtype=torch.int64, device="cuda")
    gscale = torch.tensor([0.5], device="cuda")
    kw = dict(lr=0.0, betas=OPT["betas"], eps=1e-8, weight_decay=0.02, d_lr=lr, d_step=step,
              d_grad_scale=gscale)
    g = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(g):
        fg.adamw_step(P, G, M, V, **kw)
    p, m, v = ps[0], ms[0], vs[0]
    for t, rate, gs_ in ((3, 1e-2, 0.5), (4, 5e-3, 2.0)):
        lr.fill_(rate)
        step.fill_(t)
        gscale.fill_(gs_)
        g.replay()
        p, m, v = so.adamw(p, gs[0], m, v, lr=float(np.float32(rate)), step=t, betas=OPT["betas"],
                           eps=1e-8, wd=0.02, grad_scale=gs_)
        assert np.array_equal(M[0].cpu().numpy(), m) and np.array_equal(V[0].cpu().numpy(), v)
        # the step's constants are powers and roots in 64 bits, rounded to f32
        # once: the same but where two 64-bit results straddle a rounding (one
        # f32 step of the update, itself about lr)
        assert np.abs(P[0].cpu().numpy() - p).max() <= 2.0 ** -22 * np.abs(p).max()
        p = P[0].cpu().numpy()


def test_not_finite_gradients():
    import forgegpu as fg
    import torch
    n = 600
    for bits in (32, 8):
        P = [torch.ones(n, device="cuda")]
        G = [torch.full((n,), 0.1, device="cuda")]
        G[0][300] = float("nan")
        if bits == 32:
            M, V = [torch.zeros(n, device="cuda")], [torch.zeros(n, device="cuda")]
            fg.adamw_step(P, G, M, V, **OPT)
            m, v = M[0], V[0]
            hit = torch.zeros(n, dtype=torch.bool, device="cuda")
        else:
            M = [torch.zeros(n, dtype=torch.int8, device="cuda")]
            V = [torch.zeros(n, dtype=torch.uint8, device="cuda")]
            MS, VS = [torch.zeros(3, device="cuda")], [torch.zeros(3, device="cuda")]
            fg.adamw_step(P, G, M, V, m_scales=MS, v_scales=VS, **OPT)
            m, v = fg.adamw_state_values(M[0], MS[0], V[0], VS[0])
            hit = torch.zeros(n, dtype=torch.bool, device="cuda")
            hit[256:512] = True
        hit[300] = True
        assert torch.equal(torch.isnan(m), hit) and torch.equal(torch.isnan(v), hit)
        bad = torch.isnan(P[0])
        assert bad[300] and bad.sum() == 1


def test_binding_refusals():
    import forgegpu as fg
    import torch
    z = lambda n=10, **k: torch.zeros(n, device="cuda", **k)  # noqa: E731
    p, g, m, v = z(), z(), z(), z()
    for bad in (([p], [g], [m], [z(9)]), ([p], [z(10, dtype=torch.int32)], [m], [v]),
                ([p], [g], [m.half()], [v]), ([z(20)[::2]], [g], [m], [v])):
        with pytest.raises(fg.ForgeGpuError):
            fg.adamw_step(*bad, lr=1e-3)
    with pytest.raises(fg.ForgeGpuError):
        fg.adamw_step([p, p], [g, g], [m, z()], [v, z()], lr=1e-3)  # the same param twice
    with pytest.raises(fg.ForgeGpuError):
        fg.adamw_step([p], [g], [m], [v], lr=1e-3, step=0)
    with pytest.raises(fg.ForgeGpuError):
        fg.adamw_step([p], [g], [z(10, dtype=torch.int8)], [z(10, dtype=torch.uint8)], lr=1e-3,
                      m_scales=[z(2)], v_scales=[z(1)])
    fg.adamw_step([], [], [], [], lr=1e-3)


@pytest.mark.parametrize("bits", [32, 8])
def test_training_steps_of_an_index(bits):
    """As the operators are used together: queries and rows trained by the mean
    log probability of given rows, then the rows searched.  Three steps against
    the same in 64 bits.  AdamW's update is lr * m / (sqrt(v) + eps), about lr
    whatever the gradient's size, so a parameter whose gradient is within
    rounding of zero may move either way by lr a step: the parameters are held
    to 2 % of lr in the root mean square and to 2 lr a step each; with 8-bit
    moments a code is off by up to 1 in c <= 127 squared (1.6 % of the largest,
    more of small ones), which after its first step gives 20 % of lr."""
    import forgegpu as fg
    import torch
    rng = np.random.default_rng(3)
    nq, n, d, lr = 60, 400, 32, 1e-2
    q = rng.standard_normal((nq, d)).astype(np.float32)
    x = rng.standard_normal((n, d)).astype(np.float32)
    t = rng.integers(0, n, nq)
    Q, X, T = (torch.from_numpy(a).cuda() for a in (q, x, t))
    shape = [Q, X]
    if bits == 32:
        M, V = [torch.zeros_like(a) for a in shape], [torch.zeros_like(a) for a in shape]
        kw = {}
    else:
        M = [torch.zeros(a.shape, dtype=torch.int8, device="cuda") for a in shape]
        V = [torch.zeros(a.shape, dtype=torch.uint8, device="cuda") for a in shape]
        kw = {k: [torch.zeros((a.numel() + 255) // 256, device="cuda") for a in shape]
              for k in ("m_scales", "v_scales")}
    scale = 0.25
    up = torch.full((nq,), -1.0 / nq, device="cuda")
    w = {"q": q.astype(np.float64), "x": x.astype(np.float64)}
    m64 = {k: np.zeros_like(a) for k, a in w.items()}
    v64 = {k: np.zeros_like(a) for k, a in w.items()}
    z = np.zeros(nq)
    for step in (1, 2, 3):
        r = fg.logprobs(Q, X, T, scale=scale)
        dq, dx = fg.logprobs_backward(Q, X, T, r.lse, d_logprob=up, scale=scale)
        fg.adamw_step([Q, X], [dq, dx], M, V, lr=lr, step=step, weight_decay=0.01, **kw)
        f = so.forward(w["q"], w["x"], t, scale, None, 0)
        gq, gx, _, _ = so.backward(w["q"], w["x"], t, f["lse"], z, z - 1.0 / nq, z, z, scale, None)
        for k, g in (("q", gq), ("x", gx)):
            m64[k] = 0.9 * m64[k] + 0.1 * g
            v64[k] = 0.999 * v64[k] + 0.001 * g * g
            hat = (m64[k] / (1 - 0.9 ** step)) / (np.sqrt(v64[k] / (1 - 0.999 ** step)) + 1e-8)
            w[k] = w[k] * (1 - lr * 0.01) - lr * hat
    rms = 0.02 if bits == 32 else 0.2
    for got, want in ((Q, w["q"]), (X, w["x"])):
        off = np.abs(got.cpu().numpy() - want)
        assert np.sqrt((off ** 2).mean()) <= rms * lr and off.max() <= 6 * lr
    ix = fg.BruteForceIndex(fg.DistanceMetric.DotProduct).add(X.cpu().numpy())
    a = ix.log_probs(Q.cpu().numpy(), t.astype(np.uint64), temperature=1 / scale, k=10)
    b = fg.logprobs(Q, X, T, scale=scale, k=10)
    assert np.array_equal(a.top_ids.astype(np.int64), b.top_ids.cpu().numpy())
    assert np.array_equal(a.logprob, b.logprob.cpu().numpy())
    ids, _, _ = ix.batch_search_arrays(Q.cpu().numpy(), 10)
    assert np.array_equal(ids.astype(np.int64), b.top_ids.cpu().numpy())
