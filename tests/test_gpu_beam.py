"""A beam search's step and the reordering of states, against the 64-bit
definitions: ids, chains and ends have to be equal."""
import numpy as np
import pytest

import distill_oracle as do
import softmax_oracle as so

pytestmark = pytest.mark.gpu


def _types():
    import torch
    return {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def put(a, dtype, pad=0, shift=0):
    """[groups, beams, n] on the GPU, chains `pad` wider, the first element `shift` past
    an aligned address, and the values it holds in 64 bits."""
    import torch
    g, b, n = a.shape
    buf = torch.full((shift + g * b * (n + pad),), float("nan"), dtype=_types()[dtype],
                     device="cuda")
    v = buf[shift:].view(g, b, n + pad)[:, :, :n]
    v.copy_(torch.from_numpy(np.array(a)).to(v.dtype))
    return v, v.double().cpu().numpy()


def check(r, want, n=2 ** 17):
    """Scores.  A chain's normaliser is a sum of n f32 exponentials 2^t relative to a
    reference at most 8 below the largest: each is within 2^-22 of itself, as are up to
    three factors (a raised reference, the thread's and its block's), ten additions are off
    by 2^-24, and the exponent by the roundings of its product and of scale * log2 e: ln 2 *
    2 * 2^-24 |t|, of which the sum sees the mean under the softmax, at most log2 n (the
    entropy) + 8.  Their sum, and half a step of f32 for the score itself."""
    s, p, i, e = want
    assert np.array_equal(r.parents.cpu().numpy(), p)
    assert np.array_equal(r.ids.cpu().numpy(), i)
    assert np.array_equal(r.ended.cpu().numpy(), e)
    got = r.scores.double().cpu().numpy()
    fin = np.isfinite(s)
    assert np.array_equal(got[~fin], s[~fin], equal_nan=True)
    off = np.abs(got[fin] - s[fin])
    lse = 2.0 ** -20 + 10 * 2.0 ** -24 + 1.4 * 2.0 ** -24 * (np.log2(n) + 8)
    assert (off <= so.H32 * np.abs(s[fin]) * (1 + 2.0 ** -10) + lse).all(), off.max()


def problem(g, b, n, mask, ended, ids, seed):
    rng = np.random.default_rng(seed)
    x = rng.standard_normal((g, b, n)) * rng.uniform(0.5, 4, (g, b, 1))
    bs = -np.cumsum(rng.random((g, b)), 1).astype(np.float32)
    al = None
    if mask != "none":
        rows = g * b if mask == "each" else 1
        keep = rng.random((rows, n)) < rng.choice([0.02, 0.5, 0.97], (rows, 1))
        if rows > 2:
            keep[rows // 2] = False
        al = so.words(keep)
    en = (rng.random((g, b)) < 0.25) if ended else None
    names = rng.integers(-n // 4 - 1, 1000, (g, b, n)) if ids else None
    return x, bs, al, en, names


SHAPES = [
    # dtype, groups, beams, n, width, mask, ended, ids, pad, shift
    ("f32", 1, 1, 1, 1, "none", False, False, 0, 0), ("f32", 1, 1, 3, 8, "none", False, False, 0, 0),
    ("f32", 1, 4, 1000, 4, "none", False, False, 0, 0), ("f32", 3, 5, 333, 10, "each", True, False, 1, 1),
    ("f32", 2, 128, 70, 128, "none", True, True, 0, 0), ("f32", 5, 8, 20, 8, "none", True, True, 0, 0),
    ("f32", 1, 2, 50001, 64, "one", False, False, 3, 2), ("f32", 2, 3, 9000, 128, "none", True, False, 0, 0),
    ("bf16", 1, 1, 7, 2, "none", False, False, 0, 0), ("bf16", 4, 8, 5003, 8, "none", True, False, 0, 0),
    ("bf16", 2, 16, 2049, 32, "each", False, False, 5, 3), ("bf16", 70, 4, 300, 4, "one", True, False, 0, 1),
    ("bf16", 2, 6, 40000, 100, "none", False, False, 0, 7), ("bf16", 1, 1, 131072, 16, "none", False, False, 0, 0),
    ("f16", 3, 7, 1111, 14, "each", True, True, 1, 0), ("f16", 300, 2, 64, 4, "none", False, False, 0, 0),
    ("f16", 2, 10, 20000, 10, "none", False, False, 0, 0), ("f32", 40, 32, 500, 32, "none", True, False, 0, 0),
]


@pytest.mark.parametrize("normalise", [True, False])
@pytest.mark.parametrize("dtype,g,b,n,w,mask,ended,ids,pad,shift", SHAPES)
def test_select(dtype, g, b, n, w, mask, ended, ids, pad, shift, normalise):
    import forgegpu as fg
    import torch
    x, bs, al, en, names = problem(g, b, n, mask, ended, ids, g * 7 + n)
    X, x = put(x, dtype, pad, shift)
    cu = lambda a: None if a is None else torch.from_numpy(a).cuda()  # noqa: E731
    end = int(names[0, 0].max()) if ids else 3
    r = fg.beam_select(X, cu(bs), width=w, ids=cu(names), scale=0.7, normalise=normalise,
                       allowed=cu(al), ended=cu(en), end_id=end)
    assert r.scores.shape == r.parents.shape == r.ids.shape == r.ended.shape == (g, w)
    check(r, do.select(x, bs, w, ids=names, scale=0.7, normalise=normalise, allowed=al, ended=en,
                       end_id=end))


@pytest.mark.parametrize("normalise", [True, False])
@pytest.mark.parametrize("dtype,b,n,w", [("f32", 32, 131072, 2), ("f32", 16, 140000, 3),
                                         ("bf16", 1, 4900000, 1), ("bf16", 1, 2500000, 3),
                                         ("f16", 64, 80000, 1), ("f32", 128, 270001, 10)])
def test_more_lists_than_threads(dtype, b, n, w, normalise):
    """One search's chains in so many parts that a block of 256 threads joins more lists
    than that, of few columns each."""
    import forgegpu as fg
    import torch
    x, bs, _, _, _ = problem(1, b, n, "none", False, False, b + n)
    X, x = put(x, dtype, 0, 0)
    r = fg.beam_select(X, torch.from_numpy(bs).cuda(), width=w, normalise=normalise)
    check(r, do.select(x, bs, w, normalise=normalise), n)


def test_more_lists_than_a_round():
    """128 chains of nine parts: 1152 lists.  Without normalisers and with equal scores of
    the chains the best are the largest columns, in order."""
    import forgegpu as fg
    import torch
    b, n, w = 128, 1060000, 40
    gen = torch.Generator(device="cuda").manual_seed(5)
    x = torch.randn((1, b, n), device="cuda", generator=gen)
    r = fg.beam_select(x, torch.zeros((1, b), device="cuda"), width=w, normalise=False)
    flat = x.view(-1)
    at = (flat >= flat.topk(w).values[-1]).nonzero().view(-1)
    at = at[flat[at].sort(descending=True, stable=True).indices][:w]
    assert torch.equal(r.scores[0], flat[at])
    assert torch.equal(r.parents[0], at // n) and torch.equal(r.ids[0], at % n)


@pytest.mark.parametrize("dtype,g,b,n,w", [("f32", 2, 4, 10000, 4), ("bf16", 3, 8, 30000, 8),
                                           ("f16", 1, 16, 5000, 16), ("f32", 1, 64, 3000, 64)])
@pytest.mark.parametrize("kind", ["same", "rising", "falling", "steps", "few values"])
def test_equal_and_sorted_scores(dtype, g, b, n, w, kind):
    """Equal scores go by chain, then column, however many there are; columns in
    order of their scores, either way."""
    import forgegpu as fg
    import torch
    j = np.arange(n)
    rng = np.random.default_rng(0)
    row = {"same": j * 0.0, "rising": j / n * 8, "falling": -j / n * 8, "steps": (j // 100) % 7 * 1.0,
           "few values": rng.integers(0, 3, n) * 0.5}[kind]
    X, x = put(np.broadcast_to(row, (g, b, n)), dtype)
    bs = np.zeros((g, b), np.float32)
    if kind == "steps":
        bs[:] = np.arange(b) % 3
    r = fg.beam_select(X, torch.from_numpy(bs).cuda(), width=w)
    check(r, do.select(x, bs, w))


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("n", [50, 9000])
@pytest.mark.parametrize("normalise", [True, False])
def test_zeros_of_either_sign_are_equal(dtype, n, normalise):
    import forgegpu as fg
    import torch
    x = np.full((1, 3, n), -1.0)
    x[0, :, 3::5] = -0.0
    x[0, :, 4::5] = 0.0
    X, x = put(x, dtype)
    bs = np.array([[0.0, -0.0, -0.5]], np.float32)
    r = fg.beam_select(X, torch.from_numpy(bs).cuda(), width=12, normalise=normalise)
    check(r, do.select(x, bs, 12, normalise=normalise))


@pytest.mark.parametrize("dtype,g,b,n,w", [("f32", 3, 4, 5000, 8), ("bf16", 2, 8, 3000, 16)])
def test_chains_whose_normalisers_nearly_agree(dtype, g, b, n, w):
    """The chains' best columns are the same, their normalisers differ by 1e-6 to 1e-10:
    the order is that of 64-bit scores."""
    import forgegpu as fg
    import torch
    rng = np.random.default_rng(4)
    x = np.repeat(rng.standard_normal((g, 1, n)) * 2, b, 1)
    x[:, :, :4] = 12.0 + np.arange(4)
    for c in range(b):  # a column far below the others, a little higher in each chain
        x[:, c, n - 1] = -2.0 - c * 0.5
    X, x = put(x, dtype)
    bs = np.zeros((g, b), np.float32)
    want = do.select(x, bs, w)
    gaps = -np.diff(want[0][:, :4])
    assert (gaps > 1e-12).all() and gaps.min() < 1e-5  # (what 64 bits hold apart, 32 do not)
    check(fg.beam_select(X, torch.from_numpy(bs).cuda(), width=w), want)


@pytest.mark.parametrize("dtype,g,b,n,w", [("f32", 2, 4, 5003, 9), ("bf16", 1, 8, 30001, 16),
                                           ("f16", 3, 5, 2049, 20)])
def test_equal_chains_of_any_alignment(dtype, g, b, n, w):
    """The chains hold the same columns and start at different places of 16 bytes: their
    columns are equal and go by chain."""
    import forgegpu as fg
    import torch
    x = np.repeat(np.random.default_rng(6).standard_normal((g, 1, n)) * 3, b, 1)
    X, x = put(x, dtype)
    bs = np.zeros((g, b), np.float32)
    r = fg.beam_select(X, torch.from_numpy(bs).cuda(), width=w)
    check(r, do.select(x, bs, w))


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("n", [40, 9000])
def test_masks_by_value(dtype, n):
    """-inf takes no part; a type's lowest value is a score like others, alone in its
    row too; a row of -inf has no candidates, nor has a chain with a score of -inf."""
    import forgegpu as fg
    import torch
    rng = np.random.default_rng(1)
    low = torch.finfo(_types()[dtype]).min
    x = rng.standard_normal((2, 6, n))
    x[0, 0, rng.random(n) < 0.9] = -np.inf
    x[0, 1] = -np.inf
    x[0, 2, rng.random(n) < 0.9] = low
    x[1, 0] = low
    x[1, 1] = low
    x[1, 1, 5] = 1.0
    x[1, 2:] = -np.inf
    X, x = put(x, dtype)
    X[0, 3] = float("nan")  # (of a chain that is not there)
    bs = np.array([[0, -1, -2, -np.inf, -3, -4], [-8, 0, -1, -2, -np.inf, -np.inf]], np.float32)
    for normalise in (True, False):
        r = fg.beam_select(X, torch.from_numpy(bs).cuda(), width=10, normalise=normalise)
        x[0, 3] = 0
        check(r, do.select(x, bs, 10, normalise=normalise))
    none = fg.beam_select(X, torch.full((2, 6), -float("inf"), device="cuda"), width=3)
    assert (none.parents == -1).all() and (none.ids == -1).all() and not none.ended.any()
    assert (none.scores == -float("inf")).all()


@pytest.mark.parametrize("n", [40, 9000])
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
@pytest.mark.parametrize("normalise", [True, False])
def test_what_is_not_finite(n, bad, normalise):
    """A NaN or +inf in a search makes that one NaN; masked, in a chain that has ended
    or without an id it does nothing."""
    import forgegpu as fg
    import torch
    rng = np.random.default_rng(2)
    g, b = 5, 3
    X, x = put(rng.standard_normal((g, b, n)), "f32")
    bs = torch.zeros(g, b, device="cuda") - torch.arange(b, device="cuda")
    keep = np.ones((g * b, n), bool)
    ids = np.tile(np.arange(n), (g, b, 1))
    ended = np.zeros((g, b), bool)
    clean = fg.beam_select(X, bs, normalise=normalise)
    X[0, 1, 7] = bad                       # counts
    X[2, 0, n - 1] = bad                   # masked
    keep[2 * b, n - 1] = False
    ids[3, 2, 9] = -1                      # without an id
    X[3, 2, 9] = bad
    ended[4, 2] = True                     # in a chain that has ended
    X[4, 2] = bad
    cu = lambda a: torch.from_numpy(a).cuda()  # noqa: E731
    r = fg.beam_select(X, bs, normalise=normalise, allowed=cu(so.words(keep)), ids=cu(ids),
                       ended=cu(ended))
    assert torch.isnan(r.scores[0]).all() and (r.parents[0] == -1).all() and (r.ids[0] == -1).all()
    assert not r.ended[0].any() and not torch.isnan(r.scores[1:]).any()
    assert torch.equal(r.ids[1], clean.ids[1]) and torch.equal(r.scores[1], clean.scores[1])
    bs[1, 2] = bad
    r = fg.beam_select(X, bs, normalise=normalise, allowed=cu(so.words(keep)), ids=cu(ids),
                       ended=cu(ended))
    assert torch.isnan(r.scores[1]).all() and not torch.isnan(r.scores[2:]).any()


def test_ended_chains():
    """They keep their scores and are not read; a chosen end_id ends a chain."""
    import forgegpu as fg
    import torch
    X = torch.full((1, 3, 50), -5.0, device="cuda")
    X[0, 0, 7], X[0, 2, 9] = 4.0, 4.0
    X[0, 1] = float("nan")
    bs = torch.tensor([[-1.0, -1.5, -2.0]], device="cuda")
    ended = torch.tensor([[False, True, False]], device="cuda")
    r = fg.beam_select(X, bs, width=3, ended=ended, end_id=9)
    assert r.parents.tolist() == [[0, 1, 2]] and r.ids.tolist() == [[7, 9, 9]]
    assert r.ended.tolist() == [[False, True, True]] and r.scores[0, 1] == -1.5


@pytest.mark.parametrize("dtype", ["f32", "f16"])
@pytest.mark.parametrize("scale", [3e37, 1e20, 1e-6])
def test_scales_at_the_ends_of_f32(dtype, scale):
    """scale * x out of f32's range either way: scores are those of 64 bits."""
    import forgegpu as fg
    import torch
    rng = np.random.default_rng(5)
    X, x = put(rng.standard_normal((2, 3, 40000)) * 100, dtype)
    bs = -np.arange(6, dtype=np.float32).reshape(2, 3)
    r = fg.beam_select(X, torch.from_numpy(bs).cuda(), width=6, scale=scale)
    s, p, i, e = do.select(x, bs, 6, scale=scale)
    assert np.array_equal(r.ids.cpu().numpy(), i) and np.array_equal(r.parents.cpu().numpy(), p)
    with np.errstate(over="ignore", invalid="ignore"):
        s = np.where(np.abs(s) > 3.4e38, np.sign(s) * np.inf, s)
    got = r.scores.double().cpu().numpy()
    assert np.array_equal(np.isinf(got), np.isinf(s))
    fin = np.isfinite(s)
    assert (np.abs(got[fin] - s[fin]) <= 2.0 ** -23 * np.abs(s[fin]) + 2.0 ** -17).all()


def test_without_searches():
    import forgegpu as fg
    import torch
    x = torch.zeros((0, 3, 5000), device="cuda")
    r = fg.beam_select(x, x[:, :, 0].contiguous(), width=4)
    assert r.ids.shape == (0, 4)
    o, = fg.beam_reorder([x], r.parents[:, :3].contiguous())
    assert o.shape == (0, 3, 5000)


def test_large_offsets():
    """Chains more than 2^31 elements apart."""
    import forgegpu as fg
    import torch
    step = 1_200_000_000
    buf = torch.zeros(2 * step + 5000, dtype=torch.bfloat16, device="cuda")
    X = buf.as_strided((1, 3, 5000), (0, step, 1))
    rng = np.random.default_rng(3)
    x = rng.standard_normal((1, 3, 5000))
    X.copy_(torch.from_numpy(x).to(buf.dtype))
    bs = np.zeros((1, 3), np.float32)
    r = fg.beam_select(X, torch.from_numpy(bs).cuda(), width=20)
    check(r, do.select(X.double().cpu().numpy(), bs, 20))


# ---------------------------------------------------------------------------
def turned(t, parents, out=None):
    """Plain form: out[g, w] = t[g, parents[g, w]] where there is such a parent."""
    import torch
    g, w = parents.shape
    res = torch.zeros((g, w) + t.shape[2:], dtype=t.dtype, device=t.device) if out is None \
        else out.clone()
    for i in range(g):
        for j in range(w):
            p = int(parents[i, j])
            if 0 <= p < t.shape[1]:
                res[i, j] = t[i, p]
    return res


@pytest.mark.parametrize("g,b,w,shape", [
    (1, 1, 1, ()), (3, 4, 4, (5,)), (2, 5, 3, (2, 7, 3)), (2, 3, 6, (1000, 33)), (4, 8, 8, (3, 64, 16)),
    (2, 128, 128, (40,)), (7, 2, 1, (1,)), (1, 16, 16, (70001,)), (2, 4, 4, (0, 3)),
])
def test_reorder(g, b, w, shape):
    import forgegpu as fg
    import torch
    gen = torch.Generator(device="cuda").manual_seed(g * 10 + b)
    states = [torch.randint(0, 120, (g, b) + shape, device="cuda", generator=gen).to(dt)
              for dt in (torch.float32, torch.bfloat16, torch.int64, torch.uint8)]
    parents = torch.randint(-1, b + 1, (g, w), device="cuda", generator=gen)
    for s, o in zip(states, fg.beam_reorder(states, parents)):
        assert o.shape == (g, w) + shape and torch.equal(o, turned(s, parents))
    outs = [torch.full((g, w) + shape, 9, device="cuda").to(s.dtype) for s in states]
    want = [turned(s, parents, o) for s, o in zip(states, outs)]
    got = fg.beam_reorder(states, parents, out=outs)
    assert all(a is o and torch.equal(a, v) for a, o, v in zip(got, outs, want))
    if w == b:
        want = [turned(s, parents, s) for s in states]
        fg.beam_reorder(states, parents, out=states)
        assert all(torch.equal(a, v) for a, v in zip(states, want))


@pytest.mark.parametrize("dtype,heads,room,used,dim,off", [
    ("bf16", 3, 20, 13, 5, 0), ("f32", 4, 64, 40, 16, 0), ("f16", 1, 9, 8, 3, 1),
    ("bf16", 8, 300, 257, 64, 0), ("bf16", 5, 50, 1, 8, 0),
])
@pytest.mark.parametrize("inplace", [False, True])
def test_the_used_part_of_a_cache_moves(dtype, heads, room, used, dim, off, inplace):
    """What lies behind the positions in use, and in front of the first, is left as it
    was, of chains with and without a parent."""
    import forgegpu as fg
    import torch
    g, b = 3, 4
    gen = torch.Generator(device="cuda").manual_seed(room)
    buf = torch.randn(off + g * b * heads * room * dim, device="cuda", generator=gen)
    full = buf.to(_types()[dtype])[off:].view(g, b, heads, room, dim)
    out = full if inplace else torch.randn(full.shape, device="cuda", generator=gen).to(full.dtype)
    parents = torch.tensor([[1, 1, 0, 2], [3, 2, 1, 0], [0, -1, 4, 1]], device="cuda")
    first = 0 if used == 1 else 1
    part = lambda t: t[:, :, :, first:used]  # noqa: E731
    want = out.clone()
    part(want).copy_(turned(part(full), parents, part(out)))
    fg.beam_reorder([part(full)], parents, out=[part(out)])
    assert torch.equal(out, want)


def test_states_with_their_heads_outside():
    """[heads][groups * beams][positions] seen as [groups, beams, heads, positions]: rows lie
    between each other's heads."""
    import forgegpu as fg
    import torch
    t = torch.randn(5, 6, 40, device="cuda")
    view = lambda a: a.view(5, 2, 3, 40).permute(1, 2, 0, 3)  # noqa: E731
    o = torch.empty_like(t)
    parents = torch.tensor([[2, 2, 0], [1, 0, 2]], device="cuda")
    want = turned(view(t), parents)
    fg.beam_reorder([view(t)], parents, out=[view(o)])
    assert torch.equal(view(o), want)
    before = t.clone()
    fg.beam_reorder([view(t)[:, :, :, :7]], parents, out=[view(t)[:, :, :, :7]])
    assert torch.equal(view(t)[:, :, :, :7], want[:, :, :, :7])
    assert torch.equal(t[:, :, 7:], before[:, :, 7:])
    with pytest.raises(fg.ForgeGpuError):
        fg.beam_reorder([view(t)], parents, out=[o[0, 0].expand(2, 3, 5, 40)])


def test_reorder_many_states_on_a_stream_and_captured():
    import forgegpu as fg
    import torch
    gen = torch.Generator(device="cuda").manual_seed(1)
    states = [torch.randn(2, 4, 1 + 37 * i, device="cuda", generator=gen) for i in range(230)]
    parents = torch.randint(0, 4, (2, 4), device="cuda", generator=gen)
    want = [turned(s, parents) for s in states]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = fg.beam_reorder(states, parents)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = fg.beam_reorder(states, parents)
    parents.copy_(parents.flip(1).clone())
    g.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, turned(s, parents)) for a, s in zip(out, states))
    first = states[0].clone().requires_grad_()
    saved = (first * 2).sum()
    before = first._version
    with torch.no_grad():
        fg.beam_reorder([states[1]], parents, out=[torch.empty_like(states[1])])
        fg.beam_reorder([first], parents, out=[first])
    assert first._version > before and saved.requires_grad


def test_reorder_offsets_beyond_32_bits():
    import forgegpu as fg
    import torch
    n = 1_150_000_000  # rows of 2.3 GB
    t = torch.empty(1, 3, n, dtype=torch.bfloat16, device="cuda")
    for b in range(3):
        t[0, b] = b + 1
        t[0, b, -3:] = 10 * (b + 1)
    parents = torch.tensor([[2, 0, 0]], device="cuda")
    o, = fg.beam_reorder([t], parents)
    assert o[0, :, -1].tolist() == [30, 10, 10] and o[0, :, 0].tolist() == [3, 1, 1]
    assert (o[0, 0, :-3] == 3).all() and (o[0, 2, :-3] == 1).all()
    del o
    fg.beam_reorder([t], parents, out=[t])
    assert t[0, :, -1].tolist() == [30, 10, 10] and (t[0, 1, :-3] == 1).all()
    assert (t[0, 0, :-3] == 3).all()


def test_select_on_streams_and_in_graphs():
    import forgegpu as fg
    import torch
    X, _ = put(np.random.default_rng(0).standard_normal((4, 8, 20000)), "bf16")
    Y, _ = put(np.random.default_rng(1).standard_normal((2, 4, 300)), "f32")
    bx, by = torch.zeros(4, 8, device="cuda"), torch.zeros(2, 4, device="cuda")
    fs = [lambda: fg.beam_select(X, bx, width=16), lambda: fg.beam_select(Y, by)]
    same = lambda a, b: all(torch.equal(u, v) for u, v in zip(a, b))  # noqa: E731
    graphs = []
    for f in fs:
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = f()
        graphs.append((g, out))
    want = [f() for f in fs]
    side = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(3):
        for i, s in enumerate(side):
            with torch.cuda.stream(s):
                graphs[i][0].replay()
                got[i].append(fs[i]())
    torch.cuda.synchronize()
    for i in range(2):
        assert same(graphs[i][1], want[i]) and all(same(r, want[i]) for r in got[i])
    X.copy_(X.flip(1).clone())
    graphs[0][0].replay()
    torch.cuda.synchronize()
    assert same(graphs[0][1], fs[0]())


def test_binding_refusals():
    import forgegpu as fg
    import torch
    X = torch.randn(2, 3, 40, device="cuda")
    b = torch.zeros(2, 3, device="cuda")
    ids = torch.zeros((2, 3, 40), dtype=torch.int64, device="cuda")
    words = torch.zeros((6, 2), dtype=torch.int32, device="cuda")
    for bad in (lambda: fg.beam_select(X[0], b), lambda: fg.beam_select(X.double(), b),
                lambda: fg.beam_select(X.transpose(1, 2), b), lambda: fg.beam_select(X, b[:1]),
                lambda: fg.beam_select(X, b.double()), lambda: fg.beam_select(X, b, width=0),
                lambda: fg.beam_select(X, b, width=129), lambda: fg.beam_select(X, b, scale=0.0),
                lambda: fg.beam_select(X, b, ids=ids.int()), lambda: fg.beam_select(X, b, ids=ids[:1]),
                lambda: fg.beam_select(X, b, allowed=words[:2]),
                lambda: fg.beam_select(X, b, allowed=words[:, :1]),
                lambda: fg.beam_select(X, b, ended=b), lambda: fg.beam_select(X[:, :, :0], b),
                lambda: fg.beam_select(X.cpu(), b),
                lambda: fg.beam_select(X.repeat(1, 1, 50), b, workspace=torch.empty(0, dtype=torch.uint8,
                                                                   device="cuda"))):
        with pytest.raises(fg.ForgeGpuError):
            bad()
    p = torch.zeros((2, 3), dtype=torch.int64, device="cuda")
    for bad in (lambda: fg.beam_reorder([X], p.int()), lambda: fg.beam_reorder([X], p.cpu()),
                lambda: fg.beam_reorder([X], p[:1]), lambda: fg.beam_reorder([X], p, out=[]),
                lambda: fg.beam_reorder([X], p, out=[X.half()]),
                lambda: fg.beam_reorder([X], p[:, :2].contiguous(), out=[X]),
                lambda: fg.beam_reorder([X.transpose(0, 1)], p),
                lambda: fg.beam_reorder([X[:, :, ::2]], p, out=[torch.empty_like(X[:, :, 1:4:2])]),
                lambda: fg.beam_reorder([X, X[:, :2]], p)):
        with pytest.raises(fg.ForgeGpuError):
            bad()
    assert fg.beam_reorder([], p) == []


# ---------------------------------------------------------------------------
def test_chains_of_rows():
    """The operators together: chains of three rows, each step's queries the chain's
    state plus the row it took, decoded by logprobs, beam_select and beam_reorder,
    against every chain's score in 64 bits."""
    import forgegpu as fg
    import torch
    rng = np.random.default_rng(11)
    g, n, d, w = 3, 40, 16, 5
    x = rng.standard_normal((n, d))
    start = rng.standard_normal((g, d))
    X = torch.from_numpy(x).float().cuda()
    x = X.double().cpu().numpy()
    state = torch.from_numpy(start).float().cuda()[:, None].contiguous()
    start = state[:, 0].double().cpu().numpy()
    scores = torch.zeros(g, 1, device="cuda")
    chain = torch.empty((g, 1, 0), dtype=torch.int64, device="cuda")
    keep = (start[:, None], np.zeros((g, 1)), [[()] for _ in range(g)])
    for step in range(3):
        b = state.shape[1]
        r = fg.logprobs(state.view(g * b, d), X, scale=0.4, k=12)
        sel = fg.beam_select(r.top_logprobs.view(g, b, 12), scores, width=w,
                             ids=r.top_ids.view(g, b, 12), normalise=False)
        # (12 a chain are more than the width: the best of all rows are among them)
        full = torch.einsum("gbd,nd->gbn", state.double(), X.double()).float()
        dense = fg.beam_select(full, scores, width=w, scale=0.4)
        assert torch.equal(sel.ids, dense.ids) and torch.equal(sel.parents, dense.parents)
        state, chain = fg.beam_reorder([state, chain] if chain.shape[2] else [state],
                                       sel.parents) + ([] if chain.shape[2] else [chain.expand(g, w, 0)])
        state = state * 0.5 + X[sel.ids]
        chain = torch.cat([chain, sel.ids[:, :, None]], 2)
        scores = sel.scores
        # the same in 64 bits
        q, s, names = keep
        nq, ns, nn = [], [], []
        for i in range(g):
            lp = q[i] @ x.T * np.float64(np.float32(0.4))
            lp = lp - np.log(np.exp(lp).sum(1, keepdims=True)) + s[i][:, None]
            at = np.argsort(-lp.ravel(), kind="stable")[:w]
            p, c = at // n, at % n
            nq.append(q[i][p] * 0.5 + x[c])
            ns.append(lp.ravel()[at])
            nn.append([names[i][a] + (int(t),) for a, t in zip(p, c)])
        keep = (np.stack(nq), np.stack(ns), nn)
    want = np.array([[list(c) for c in row] for row in keep[2]])
    assert np.array_equal(chain.cpu().numpy(), want)
    assert np.abs(scores.double().cpu().numpy() - keep[1]).max() < 1e-4
    # and a step of training on what was decoded: the chains' first rows as a teacher's list
    z = torch.log_softmax(scores, 1)
    q = torch.from_numpy(start).float().cuda()
    loss = fg.distill(q, X, chain[:, :, 0].contiguous(), z, scale=0.4)
    dq, dx = fg.distill_backward(q, X, chain[:, :, 0].contiguous(), z, loss.lse, loss.logprobs,
                                 d_loss=torch.ones(g, device="cuda"), scale=0.4)
    m, v = [torch.zeros_like(q), torch.zeros_like(X)], [torch.zeros_like(q), torch.zeros_like(X)]
    before = X.clone()
    fg.adamw_step([q, X], [dq, dx], m, v, lr=1e-3)
    assert torch.isfinite(X).all() and not torch.equal(before, X)
