"""Tensors of one AdamW call may not share what the call writes (no GPU: the
check comes before any device work)."""
import ctypes as C

import pytest

OPTS = dict(param_dtype=0, grad_dtype=0, lr=1e-3, beta1=0.9, beta2=0.999, eps=1e-8,
            weight_decay=0.01, grad_scale=1.0, step=1)
A = dict(param=0x10000, grad=0x20000, m=0x30000, v=0x40000, m_scale=0x50000, v_scale=0x60000,
         n=300)
B = {k: v + 0x100000 for k, v in A.items() if k != "n"} | dict(n=257)


def _rc(bits, *tensors):
    import forgegpu as fg
    L = fg.lib()
    ctx = C.cast(C.create_string_buffer(1 << 16), C.c_void_p)
    arr = (fg.AdamwTensor * len(tensors))(*(fg.AdamwTensor(**t) for t in tensors))
    rc = L.fdb_adamw_step(ctx, C.byref(arr), len(tensors),
                          C.byref(fg.AdamwOpts(**OPTS, state_bits=bits)))
    return rc, L.fdb_last_error()


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("name", ["param", "m", "v", "m_scale", "v_scale"])
@pytest.mark.parametrize("other", ["param", "m", "v", "m_scale", "v_scale"])
def test_shared_states_are_refused(bits, name, other):
    if bits == 32 and "scale" in name + other:
        return
    size = dict(param=1200, m=300 * bits // 8, v=300 * bits // 8, m_scale=8, v_scale=8)[name]
    step = 1 if bits == 8 and other in "mv" else 4
    for at in (A[name], A[name] + size - step):  # the whole of it, its last element
        rc, msg = _rc(bits, A, {**B, other: at})
        assert rc == -1 and b"overlap" in msg, msg
    if name != other:  # within one tensor
        rc, msg = _rc(bits, {**A, other: A[name]})
        assert rc == -1 and b"overlap" in msg, msg
