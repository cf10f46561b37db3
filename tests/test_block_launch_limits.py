"""CPU-only: calls of the grouped-query block whose launches would pass 2^32
threads are refused with the documented code and before any GPU work."""
import ctypes as C

import pytest

import evk_amd as evk
from test_block_refusals import UNSUPPORTED, Mem, window

b = C.byref


@pytest.fixture(scope="module")
def L():
    if not evk.available():
        pytest.fail("libevkhip.so is not built: run `python -m evk_amd.build`")
    return evk.lib()


@pytest.mark.parametrize("t,d,f", [(1 << 30, 8, 1 << 16), (1 << 30, 24, 100_001), (1 << 29, 1000, 1 << 20)])
def test_gated_linear(L, t, d, f):
    m = Mem()
    assert L.evkhip_gated_linear(b(m(t, d)), b(m(2, d, f)), b(m(t, f)), None, 0, None) == UNSUPPORTED
    assert b"workgroups" in L.evkhip_last_error()


@pytest.mark.parametrize("t,d,f,which", [(1 << 30, 1 << 16, 8, "dx"), (8, 1 << 30, 1 << 16, "dw"), (3, 1 << 29, 100_001, "dw"), (1 << 30, 8, 1 << 20, "neither")])
def test_gated_linear_backward(L, t, d, f, which):
    m = Mem()
    need = L.evkhip_gated_linear_backward_workspace(t, d, f)
    dx, dw = m(t, d) if which == "dx" else None, m(2, d, f) if which == "dw" else None
    rc = L.evkhip_gated_linear_backward(b(m(t, d)), b(m(2, d, f)), b(m(2, t, f)), b(m(t, f)), dx and b(dx), dw and b(dw), 0, 0, 1 << 60, need, None)
    assert rc == UNSUPPORTED
    assert b"workgroups" in L.evkhip_last_error()


def test_window_attention(L):
    n = 16_500_000
    assert window(L, Mem(), q=(n, 65, 256), k=(n, 65, 256), dh=256, w=0, s=0) == UNSUPPORTED
    assert b"workgroups" in L.evkhip_last_error()
