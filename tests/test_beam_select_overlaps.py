"""Outputs of a beam step may not share a byte with what the call reads or writes elsewhere
(no GPU: the check comes before any device work, and the context names a device that is
not there)."""
import ctypes as C

import pytest

# two searches of three chains of 1000 columns in rows of 1016, four best of each
BASE = dict(dtype=0, groups=2, beams=3, n=1000, ld_group=3560, ld_beam=1016, scale=1.0,
            normalise=1, width=4, scores=1 << 20, beam_scores=1 << 16, ended=2 << 16, ids=1 << 22,
            ld_ids=1000, allowed=3 << 16, ld_allowed=32, out_scores=4 << 16, out_parents=5 << 16,
            out_ids=6 << 16, out_ended=7 << 16, workspace=1 << 24, workspace_bytes=1 << 40)
SIZES = dict(out_scores=2 * 4 * 4, out_parents=2 * 4 * 8, out_ids=2 * 4 * 8, out_ended=2 * 4,
             beam_scores=6 * 4, ended=6, allowed=6 * 128, ids=6 * 8000,
             scores=4 * (3560 + 2 * 1016 + 1000))
STEP = dict(out_scores=4, out_parents=8, out_ids=8, out_ended=1)


def refused(**change):
    import forgegpu as fg
    L = fg.lib()
    raw = C.create_string_buffer(1 << 16)
    C.cast(raw, C.POINTER(C.c_int))[0] = 1 << 20  # (the context's device)
    rc = L.fdb_beam_select(C.cast(raw, C.c_void_p), C.byref(fg.BeamArgs(**{**BASE, **change})))
    assert rc != 0  # (no device)
    if rc == -1:
        assert b"output" in L.fdb_last_error(), L.fdb_last_error()
    else:
        assert rc != -2
    return rc == -1


def test_apart():
    assert not refused()
    assert not refused(ids=None, allowed=None, ended=None, out_ended=None)
    assert not refused(ld_allowed=0, beams=1, ld_beam=0)
    # searches and chains that are read more than once
    assert not refused(ld_group=0) and not refused(allowed=BASE["scores"]) and not refused(ids=1 << 20)


@pytest.mark.parametrize("out", list(STEP))
@pytest.mark.parametrize("other", list(SIZES))
def test_shared_bytes(out, other):
    if out == other:
        return
    at, step = BASE[other], STEP[out]
    last = (SIZES[other] - 1) // step * step  # the other's last byte lies in it
    for shift in (0, step, last, step - SIZES[out]):
        # (in front of it: its last element is the other's first bytes)
        hit = -SIZES[out] < shift < SIZES[other]
        assert refused(**{out: at + shift}) == hit, shift
    assert not refused(**{out: at + (SIZES[other] + 7) // 8 * 8})
    assert not refused(**{out: at - SIZES[out]})


def test_gaps_of_the_scores():
    # columns 1000 to 1015 of a row are no chain's
    for out in STEP:
        assert not refused(**{out: BASE["scores"] + 4000})
        assert refused(**{out: BASE["scores"] + 3992})
        assert not refused(**{out: BASE["scores"] + 4 * 3048})
        assert refused(**{out: BASE["scores"] + 4 * 3560})


def test_the_workspace():
    for other in ("scores", "beam_scores", "out_scores", "out_parents", "out_ids", "ids", "allowed"):
        assert refused(workspace=BASE[other])
    assert not refused(workspace=(1 << 22) + (48000 + 255) // 256 * 256)
    # (a search without one does not look at it)
    small = dict(n=20, ld_beam=20, ld_group=60, ld_ids=20, ld_allowed=1)
    assert not refused(**small, workspace=BASE["scores"])
    assert not refused(**small, workspace=None)


def test_too_large():
    import forgegpu as fg
    L = fg.lib()
    raw = C.create_string_buffer(1 << 16)
    C.cast(raw, C.POINTER(C.c_int))[0] = 1 << 20
    for change in (dict(ld_group=(1 << 40) - 1, groups=(1 << 22) - 1), dict(ld_ids=1 << 60),
                   dict(ld_allowed=1 << 61)):
        a = fg.BeamArgs(**{**BASE, **change})
        assert L.fdb_beam_select(C.cast(raw, C.c_void_p), C.byref(a)) == -1
        assert b"large" in L.fdb_last_error()
