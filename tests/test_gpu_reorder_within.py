"""Reordering of states that lie within one another's gaps, and refusals on the GPU."""
import pytest

from test_gpu_beam import turned

pytestmark = pytest.mark.gpu


def test_keys_and_values_of_one_tensor():
    """In place, and into another such tensor, in one call; what is not in use stays."""
    import forgegpu as fg
    import torch
    g, b, heads, room, dim, used = 3, 4, 2, 20, 8, 13
    gen = torch.Generator(device="cuda").manual_seed(0)
    parents = torch.randint(0, b, (g, b), device="cuda", generator=gen)
    for shape, at in (((g, b, 2, heads, room, dim), lambda t, i: t[:, :, i, :, :used]),
                      ((g, b, heads, 2, room, dim), lambda t, i: t[:, :, :, i, :used])):
        t = torch.randn(shape, device="cuda", generator=gen)
        o, want = torch.full_like(t, 7), torch.full_like(t, 7)
        for i in range(2):
            at(want, i).copy_(turned(at(t, i), parents))
        fg.beam_reorder([at(t, 0), at(t, 1)], parents, out=[at(o, 0), at(o, 1)])
        assert torch.equal(o, want)
        want = t.clone()
        for i in range(2):
            at(want, i).copy_(turned(at(t, i), parents))
        fg.beam_reorder([at(t, 0), at(t, 1)], parents, out=[at(t, 0), at(t, 1)])
        assert torch.equal(t, want)


def test_layers_of_one_tensor():
    import forgegpu as fg
    import torch
    gen = torch.Generator(device="cuda").manual_seed(1)
    t = torch.randn(2, 5, 48, 6, 10, device="cuda", generator=gen)
    parents = torch.randint(-1, 6, (2, 5), device="cuda", generator=gen)
    want = turned(t, parents, t)
    layers = [t[:, :, i] for i in range(48)]
    fg.beam_reorder(layers, parents, out=layers)
    assert torch.equal(t, want)


def test_one_half_into_the_other():
    """Positions 0 to 7 of every head into 8 to 15, and heads outside of the rows."""
    import forgegpu as fg
    import torch
    gen = torch.Generator(device="cuda").manual_seed(2)
    parents = torch.tensor([[1, 2, 0], [0, 0, 1]], device="cuda")
    t = torch.randn(2, 3, 4, 16, device="cuda", generator=gen)
    want = t.clone()
    want[..., 8:] = turned(t[..., :8], parents)
    fg.beam_reorder([t[..., :8]], parents, out=[t[..., 8:]])
    assert torch.equal(t, want)
    t = torch.randn(4, 2, 3, 16, device="cuda", generator=gen)
    want = t.clone()
    view = lambda v: v.permute(1, 2, 0, 3)  # noqa: E731
    view(want)[..., 8:] = turned(view(t)[..., :8], parents)
    fg.beam_reorder([view(t)[..., :8]], parents, out=[view(t)[..., 8:]])
    assert torch.equal(t, want)


def test_refused_before_anything_moves():
    import forgegpu as fg
    import torch
    t = torch.randn(2, 3, 4, 16, device="cuda")
    parents = torch.tensor([[1, 2, 0], [0, 0, 1]], device="cuda")
    flat = torch.randn(400, device="cuda")
    a, b = flat[:96].view(2, 3, 16), flat[95:191].view(2, 3, 16)
    hist = torch.zeros(18, dtype=torch.int64, device="cuda")
    inside = hist[:6].view(2, 3)
    for states, p, out in (([t[..., :8]], parents, [t[..., 1:9]]), ([a], parents, [b]),
                           ([a, flat[200:296].view(2, 3, 16)], parents, [flat[300:396].view(2, 3, 16), b]),
                           ([hist.view(2, 3, 3)], inside, [hist.view(2, 3, 3)])):
        before = [s.clone() for s in (t, flat, hist)]
        with pytest.raises(fg.ForgeGpuError, match="written"):
            fg.beam_reorder(states, p, out=out)
        assert all(torch.equal(u, v) for u, v in zip(before, (t, flat, hist)))
