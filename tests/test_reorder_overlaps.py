"""States of one reordering may not share a byte that the call writes (no GPU: the check
comes before any device work, and the context names a device that is not there)."""
import ctypes as C

import numpy as np
import pytest

PARENTS = 1 << 20


def call(*states, groups=2, beams=3, width=3, parents=PARENTS):
    """(src, dst, src_stride, dst_stride, parts, src_part_stride, dst_part_stride, bytes)"""
    import forgegpu as fg
    L = fg.lib()
    raw = C.create_string_buffer(1 << 16)
    C.cast(raw, C.POINTER(C.c_int))[0] = 1 << 20  # (the context's device)
    flat = [v for t in states for v in t]
    table = (C.c_uint64 * len(flat))(*flat)
    opts = fg.ReorderOpts(parents=parents, groups=groups, beams=beams, width=width)
    rc = L.fdb_beam_reorder(C.cast(raw, C.c_void_p), C.addressof(table), len(states),
                            C.byref(opts))
    return rc, L.fdb_last_error()


def refused(*states, **kw):
    rc, text = call(*states, **kw)
    assert rc != 0  # (no device)
    if rc == -1:
        assert b"written" in text, text
    else:
        assert rc != -2, text
    return rc == -1


ROW = (64, 64, 1, 0, 0, 64)  # six rows of 64 bytes beside each other


@pytest.mark.parametrize("shift", [1, 16, 64, 383])
@pytest.mark.parametrize("back", [False, True])
def test_shifted_states(shift, back):
    a, b = 65536, 65536 + (-shift if back else shift)
    assert refused((a, b) + ROW)                                     # out in the state
    assert refused((4096, a) + ROW, (8192, b) + ROW)                 # two outs
    assert refused((4096, a) + ROW, (b, 8192) + ROW)                 # another's source
    assert refused((a, a) + ROW, (b, b) + ROW)                       # both in place
    assert refused((a, a) + ROW, (b, 8192) + ROW)
    assert not refused((a, 4096) + ROW, (b, 8192) + ROW)             # two that are read
    assert not refused((a, a - 384) + ROW, (8192, a + 384) + ROW)    # side by side


def test_parents_in_a_state():
    for at in (PARENTS, PARENTS + 47, PARENTS - 383):
        assert refused((4096, at) + ROW) and refused((at, at) + ROW)
        assert not refused((at, 4096) + ROW)
    assert not refused((4096, PARENTS + 48) + ROW, (8192, PARENTS - 384) + ROW)


def test_positions_of_one_cache():
    """[2][3][heads 4][room 16] of 2 bytes: positions 0 to 7 into 1 to 8, and into 8 to 15."""
    def part(src, dst, used):
        return (65536 + 2 * src, 65536 + 2 * dst, 128, 128, 4, 32, 32, 2 * used)
    assert refused(part(0, 1, 8)) and refused(part(1, 0, 8)) and refused(part(0, 7, 8))
    assert not refused(part(0, 8, 8)) and not refused(part(8, 0, 8))
    assert refused(part(0, 9, 8))  # (the last position of a head is the next one's first)
    assert refused(part(0, 0, 8), part(7, 7, 8)) and not refused(part(0, 0, 8), part(8, 8, 8))


def test_many_states_within_one_tensor():
    """[rows][layers][keys, values][64]: every layer's in place, beside one more that is not
    beside them."""
    rows, layers = 6, 80
    step = layers * 2 * 64
    states = [(1 << 24) + 64 * i for i in range(2 * layers)]
    kv = [(a, a, step, step, 1, 0, 0, 64) for a in states]
    assert not refused(*kv)
    assert refused(*kv, (4096, (1 << 24) + 5 * step + 100) + ROW)
    assert not refused(*kv, (4096, (1 << 24) + rows * step) + ROW)
    assert not refused(*kv, (4096, (1 << 24) - 384) + ROW)


def test_other_strides():
    # heads outside of the rows, a row of 48 bytes in a place of 64: the gaps are free
    a = (65536, 65536, 64, 64, 4, 64 * 6, 64 * 6, 48)
    assert not refused(a, (4096, 65536 + 48, 64 * 6, 64, 1, 0, 0, 16))
    assert refused(a, (4096, 65536 + 47, 64 * 6, 64, 1, 0, 0, 16))
    # rows that are nowhere near each other's, by the distance between them
    assert not refused((4096, 65536, 10, 1000, 1, 0, 0, 10), (4096, 65536 + 500, 10, 2000, 1, 0, 0, 10))
    assert refused((4096, 65536, 10, 1000, 1, 0, 0, 10), (4096, 65536 + 2995, 10, 2000, 1, 0, 0, 10))


def test_too_large():
    rc, text = call((1 << 40, 1 << 41, (1 << 40) - 1, 64, 1, 0, 0, 64), groups=(1 << 22) - 1, beams=128)
    assert rc == -1 and b"large" in text
    rc, text = call((1 << 40, 1 << 57) + ROW)
    assert rc == -1 and b"large" in text


def test_against_every_byte():
    """Random pairs of states: refused where a byte that one writes is another's."""
    rng = np.random.default_rng(0)

    def bytes_of(at, rows, stride, parts, step, size):
        r = np.arange(rows)[:, None, None] * stride + np.arange(parts)[None, :, None] * step
        return set((at + r + np.arange(size)).ravel().tolist())

    kinds = {True: 0, False: 0}
    for _ in range(4000):
        g, b = int(rng.integers(1, 4)), int(rng.integers(1, 4))
        w = b if rng.random() < 0.6 else int(rng.integers(1, 5))
        rows = max(g * w, g * b)
        states, read, written = [], [], []
        for _ in range(int(rng.integers(1, 4))):
            parts, size = int(rng.integers(1, 4)), int(rng.integers(1, 9))
            step = size + int(rng.integers(0, 12))
            inside = (parts - 1) * step + size
            stride = inside + int(rng.integers(0, 3)) * int(rng.integers(0, 30))
            if rng.random() < 0.3:  # rows within each other's runs
                stride = size + int(rng.integers(0, 4))
                step = (rows - 1) * stride + size + int(rng.integers(0, 9))
            dst = 5000 + int(rng.integers(0, 120))
            src, ss, sp = dst, stride, step
            if w != b or rng.random() < 0.5:
                src = 5000 + int(rng.integers(0, 120)) if rng.random() < 0.3 else 9000
                if src == dst:
                    src += 1
                if rng.random() < 0.3:
                    ss, sp = int(rng.integers(0, 40)), int(rng.integers(0, 40))
            states.append((src, dst, ss, stride, parts, sp, step, size))
            written.append(bytes_of(dst, g * w, stride, parts, step, size))
            read.append(bytes_of(src, g * b, ss, parts, sp, size) if src != dst else set())
        bad = any(written[i] & read[j] or (i < j and written[i] & written[j])
                  for i in range(len(states)) for j in range(len(states)))
        kinds[bad] += 1
        assert refused(*states, groups=g, beams=b, width=w) == bad, (states, g, b, w, bad)
    assert min(kinds.values()) > 1000
