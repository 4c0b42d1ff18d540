"""AdamW steps with moments near the ends of their ranges and calls that share
tensors."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu


def _steps(g, eps, steps=4, pad=None):
    """Parameters and 8-bit state after a few steps from zeros."""
    import forgegpu as fg
    import torch
    n = g.shape[1]
    p = torch.linspace(-1, 1, n, device="cuda")
    m = torch.zeros(n, dtype=torch.int8, device="cuda")
    v = torch.zeros(n, dtype=torch.uint8, device="cuda")
    ms, vs = (torch.zeros((n + 255) // 256, device="cuda") for _ in range(2))
    for t in range(steps):
        fg.adamw_step([p], [g[t]], [m], [v], m_scales=[ms], v_scales=[vs], lr=1e-2, step=t + 1,
                      eps=eps, weight_decay=0.0, seed=5)
    return p, m, v, ms, vs, fg.adamw_state_values(m, ms, v, vs)


@pytest.mark.parametrize("shift", [24, 31, 33, 36])
def test_small_gradients_keep_their_8_bit_moments(shift):
    """AdamW does not change when gradients and eps are scaled alike: by powers
    of two every operation, code and parameter stays the same, as long as v
    (1e-8 to 1e-11 before the scaling) is in its range."""
    import torch
    rng = np.random.default_rng(0)
    g = rng.uniform(2e-4, 3e-3, (4, 3000)) * rng.choice([-1, 1], (4, 3000))
    g = torch.from_numpy(g).float().cuda()
    two = 2.0 ** -shift
    p, m, v, ms, vs, (vm, vv) = _steps(g, 2.0 ** -20)
    q, n, w, ns, ws, (wm, wv) = _steps(g * two, 2.0 ** -20 * two)
    assert (v > 0).all()
    assert torch.equal(p, q) and torch.equal(m, n) and torch.equal(v, w)
    assert torch.equal(ms * two, ns) and torch.equal(vs * two * two, ws)
    assert torch.equal(vm * two, wm) and torch.equal(vv * two * two, wv)


def test_a_block_without_v_has_no_m():
    """Gradients of 1e-17: v is below what 8 bits hold, m would be kept; both
    are zeros.  Where v is 0 because no gradient ever came, so is m."""
    import torch
    g = torch.full((4, 600), 1e-17, device="cuda")
    g[:, 256:512] = 1e-3
    g[:, 512:] = 0.0
    p, m, v, ms, vs, (vm, vv) = _steps(g, 1e-30)
    assert ms[0] == 0 and vs[0] == 0 and not m[:256].any() and not v[:256].any()
    assert (vm[256:512] > 0).all() and (vv[256:512] > 0).all()
    assert not vm[512:].any() and not vv[512:].any()
    assert torch.isfinite(p).all()
    # each step is then one from zeros: at most lr (1 - b1) / sqrt(1 - b2)
    assert (p - torch.linspace(-1, 1, 600, device="cuda")).abs()[:256].max() <= 4 * 1e-2 * 3.2


@pytest.mark.parametrize("bits", [32, 8])
def test_a_step_is_an_in_place_change_to_autograd(bits):
    """A graph that saved a parameter before the step refuses its backward
    pass; results of logprobs have no history."""
    import forgegpu as fg
    import torch
    w = torch.nn.Parameter(torch.randn(300, device="cuda"))
    g = torch.randn(300, device="cuda")
    if bits == 32:
        m, v = [torch.zeros(300, device="cuda")], [torch.zeros(300, device="cuda")]
        kw = {}
    else:
        m = [torch.zeros(300, dtype=torch.int8, device="cuda")]
        v = [torch.zeros(300, dtype=torch.uint8, device="cuda")]
        kw = {k: [torch.zeros(2, device="cuda")] for k in ("m_scales", "v_scales")}
    loss = (w * w).sum()
    before = w._version
    fg.adamw_step([w], [g], m, v, lr=1e-2, **kw)
    assert w._version > before
    with pytest.raises(RuntimeError):
        loss.backward()
    (w * w).sum().backward()
    assert torch.equal(w.grad, 2 * w.detach())
    q = torch.randn(3, 4, device="cuda", requires_grad=True)
    x = torch.nn.Parameter(torch.randn(9, 4, device="cuda"))
    r = fg.logprobs(q, x, k=1)
    assert not any(t.requires_grad for t in r)
    fg.adamw_step([w.detach()], [g], m, v, lr=1e-2, **kw)
    with torch.inference_mode():
        z = torch.zeros(5, device="cuda")
        s = [torch.zeros(5, device="cuda") for _ in range(3)]
        fg.adamw_step([z], s[:1], s[1:2], s[2:], lr=1e-2)
