"""CPU-only: the grouped-query block's entry points refuse what they do not
take, with the documented codes and before any GPU call, and name the workspace
that a call needs."""
import ctypes as C

import pytest
import torch

import evk_amd as evk

OK, INVALID, SHAPE, UNSUPPORTED = 0, -1, -2, -3


@pytest.fixture(scope="module")
def L():
    if not evk.available():
        pytest.fail("libevkhip.so is not built: run `python -m evk_amd.build`")
    return evk.lib()


class Mem:
    """Descriptors of tensors one behind another at made-up addresses."""

    def __init__(self):
        self.at = 1 << 20

    def __call__(self, *shape, at=None):
        n = 2
        for s in shape:
            n *= s
        p = self.at if at is None else at
        if at is None:
            self.at += (n + 4095) // 4096 * 4096 + 4096
        return evk.desc((p, tuple(shape)))


b = C.byref


def rope(L, m, qkv=(2, 5, 8 * 64), q=(2, 5, 4 * 64), k=(2, 9, 2 * 64), v=None, dh=64, eps=1e-4, base=1e4, p0=0, off=None, wq=None, wk=None, alias=None):
    t = dict(qkv=m(*qkv), q=m(*q), k=m(*k), v=m(*(v or k)))
    if alias:
        t[alias[0]].data = t[alias[1]].data + (alias[2] if len(alias) > 2 else 0)
    return L.evkhip_qkv_norm_rope(b(t["qkv"]), b(wq) if wq else None, b(wk) if wk else None, b(t["q"]), b(t["k"]), b(t["v"]), dh, eps, base, p0, off, None)


def test_qkv_norm_rope(L):
    m = Mem()
    assert rope(L, m, p0=5) == SHAPE  # rows 5 .. 9 of 9
    assert rope(L, m, p0=0xffffffff) == SHAPE
    assert rope(L, m, p0=1, off=4096) == INVALID  # both
    assert rope(L, m, off=4097) == INVALID
    assert rope(L, m, dh=0) == INVALID
    assert rope(L, m, dh=512) == UNSUPPORTED
    assert rope(L, m, dh=48) == SHAPE
    assert rope(L, m, qkv=(2, 5, 10 * 25), q=(2, 5, 4 * 25), k=(2, 9, 3 * 25), dh=25) == SHAPE  # 4 heads over 3
    assert rope(L, m, qkv=(2, 5, 8 * 25), q=(2, 5, 4 * 25), k=(2, 9, 2 * 25), dh=25) == SHAPE  # odd head size
    assert rope(L, m, qkv=(2, 5, 7 * 64)) == SHAPE
    assert rope(L, m, qkv=(2, 6, 8 * 64)) == SHAPE
    assert rope(L, m, k=(3, 9, 128)) == SHAPE
    assert rope(L, m, v=(2, 8, 128)) == SHAPE
    assert rope(L, m, wq=m(63)) == SHAPE
    assert rope(L, m, wk=m(64, 1)) == SHAPE
    for eps in (-1.0, float("nan"), float("inf")):
        assert rope(L, m, eps=eps) == INVALID
    for base in (0.0, -2.0, float("nan"), float("inf")):
        assert rope(L, m, base=base) == INVALID
    for alias in (("q", "qkv"), ("k", "qkv", 2), ("v", "k"), ("v", "q", 1022)):
        assert rope(L, m, alias=alias) == INVALID
        assert b"overlaps" in L.evkhip_last_error()
    assert rope(L, m, qkv=(0, 5, 512), q=(0, 5, 256), k=(0, 9, 128)) == OK  # nothing to do
    assert rope(L, m, qkv=(2, 0, 512), q=(2, 0, 256)) == OK
    assert L.evkhip_qkv_norm_rope(None, None, None, None, None, None, 64, 1e-4, 1e4, 0, None, None) == INVALID
    assert rope(L, m, qkv=(1 << 15, 1 << 16, 6), q=(1 << 15, 1 << 16, 2), k=(1 << 15, 1 << 16, 2), dh=2) == UNSUPPORTED


def test_qkv_norm_rope_backward(L):
    m = Mem()
    ws = L.evkhip_qkv_norm_rope_backward_workspace(10, 64)
    assert ws > 0 and L.evkhip_qkv_norm_rope_backward_workspace(0, 64) == 0

    def call(qkv=(2, 5, 512), dq=(2, 5, 256), dk=(2, 5, 128), dqkv=(2, 5, 512), wq=(64,), wk=(64,), dwq=(64,), dwk=(64,), dh=64, p0=0, work=1 << 40,
             have=None, alias=None):
        t = dict(qkv=m(*qkv), wq=wq and m(*wq), wk=wk and m(*wk), dq=m(*dq), dk=m(*dk), dv=m(*dk), dqkv=m(*dqkv), dwq=dwq and m(*dwq), dwk=dwk and m(*dwk))
        if alias:
            t[alias[0]].data = t[alias[1]].data
        return L.evkhip_qkv_norm_rope_backward(*[x and b(x) for x in t.values()], dh, 1e-4, 1e4, p0, 0, work, ws if have is None else have, None)

    assert call(have=ws - 1) == INVALID
    assert call(work=None) == INVALID
    assert call(work=(1 << 40) + 8) == INVALID  # 16-byte aligned
    assert call(wq=None) == INVALID  # the gradient of a weight that is not there
    assert call(dk=(2, 6, 128)) == SHAPE
    assert call(dqkv=(2, 5, 511)) == SHAPE
    assert call(dwq=(63,)) == SHAPE
    assert call(p0=1 << 30) == UNSUPPORTED
    for alias in (("dqkv", "qkv"), ("dwq", "wq"), ("dwk", "dwq"), ("dqkv", "dq")):
        assert call(alias=alias) == INVALID
    assert call(qkv=(0, 5, 512), dq=(0, 5, 256), dk=(0, 5, 128), dqkv=(0, 5, 512), wq=None, wk=None, dwq=None, dwk=None, work=None) == OK


def window(L, m, q=(2, 5, 256), k=(2, 9, 128), v=None, o=None, dh=64, w=4, s=1, p0=0, off=None, work=None, have=0, alias=None, lse=None):
    t = dict(q=m(*q), k=m(*k), v=m(*(v or k)), o=m(*(o or q)))
    if alias:
        t[alias[0]].data = t[alias[1]].data
    return L.evkhip_window_attention(*[b(x) for x in t.values()], dh, w, s, p0, off, lse, work, have, None)


def test_window_attention(L):
    m = Mem()
    assert window(L, m, p0=5) == SHAPE
    assert window(L, m, p0=1, off=4096) == INVALID
    assert window(L, m, off=4098) == INVALID
    assert window(L, m, dh=0) == INVALID
    assert window(L, m, q=(2, 5, 1024), k=(2, 9, 1024), dh=512) == UNSUPPORTED
    assert window(L, m, q=(2, 5, 192)) == SHAPE  # 3 heads over 2
    assert window(L, m, q=(2, 5, 250)) == SHAPE
    assert window(L, m, o=(2, 5, 255)) == SHAPE
    assert window(L, m, k=(1, 9, 128)) == SHAPE
    assert window(L, m, v=(2, 9, 64)) == SHAPE
    assert window(L, m, q=(2, 0, 256)) == OK
    assert window(L, m, q=(0, 5, 256), k=(0, 9, 128)) == OK
    assert window(L, m, q=(1 << 15, 1 << 16, 1), k=(1 << 15, 1 << 16, 1), dh=1) == UNSUPPORTED
    for alias in (("o", "q"), ("o", "k"), ("o", "v")):
        assert window(L, m, alias=alias) == INVALID
    # one sequence over a long cache is split: it needs a workspace
    big = dict(q=(1, 1, 256), k=(1, 50000, 128), w=0, p0=49999)
    need = L.evkhip_window_attention_workspace(1, 1, 50000, 4, 2, 64, 0, 1)
    assert need > 0
    assert window(L, m, **big) == INVALID and b"workspace" in L.evkhip_last_error()
    assert window(L, m, **big, work=1 << 41, have=need - 1) == INVALID
    assert window(L, m, **big, work=(1 << 41) + 4, have=need) == INVALID
    assert L.evkhip_window_attention_workspace(0, 1, 50000, 4, 2, 64, 0, 1) == 0
    assert L.evkhip_window_attention_workspace(1, 1, 50000, 4, 0, 64, 0, 1) == 0  # sizes that the call refuses


def test_window_attention_bwd(L):
    m = Mem()
    need = L.evkhip_window_attention_bwd_workspace(2, 5, 4, 2, 64, 4, 1)
    assert need >= 2 * 5 * 4 * 8

    def call(q=(2, 5, 256), k=(2, 5, 128), dq=None, dk=None, lse=1 << 42, dh=64, w=4, s=1, work=1 << 41, have=None, alias=None):
        t = dict(q=m(*q), k=m(*k), v=m(*k), o=m(*q), dO=m(*q), dQ=m(*(dq or q)), dK=m(*(dk or k)), dV=m(*k))
        if alias:
            t[alias[0]].data = t[alias[1]].data
        return L.evkhip_window_attention_bwd(*[b(x) for x in t.values()], lse, dh, w, s, work, need if have is None else have, None)

    assert call(k=(2, 9, 128)) == SHAPE  # rows of a cache
    assert call(lse=None) == INVALID
    assert call(have=need - 1) == INVALID
    assert call(work=None) == INVALID
    assert call(dq=(2, 5, 128)) == SHAPE
    assert call(dk=(2, 4, 128)) == SHAPE
    for alias in (("dQ", "q"), ("dK", "k"), ("dV", "dK"), ("dQ", "dO"), ("dV", "v")):
        assert call(alias=alias) == INVALID
    assert call(q=(0, 5, 256), k=(0, 5, 128), lse=None) == OK


def test_gated_linear(L):
    m = Mem()

    def call(x=(3, 64), w=(2, 64, 48), h=(3, 48), gu=None, act=0, alias=None):
        t = dict(x=m(*x), w=m(*w), h=m(*h), gu=gu and m(*gu))
        if alias:
            t[alias[0]].data = t[alias[1]].data
        return L.evkhip_gated_linear(*[v and b(v) for v in t.values()], act, None)

    assert call(w=(3, 64, 48)) == SHAPE
    assert call(w=(64, 96)) == SHAPE
    assert call(x=(3, 63)) == SHAPE
    assert call(h=(2, 48)) == SHAPE
    assert call(h=(3, 96)) == SHAPE
    assert call(gu=(2, 3, 47)) == SHAPE
    assert call(gu=(3, 2, 48)) == SHAPE
    assert call(act=3) == INVALID and call(act=-1) == INVALID
    assert call(x=(0, 64), h=(0, 48)) == OK
    for alias in (("h", "x"), ("h", "w")):
        assert call(alias=alias) == INVALID
    assert call(gu=(2, 3, 48), alias=("gu", "h")) == INVALID


def test_gated_linear_backward(L):
    m = Mem()
    need = L.evkhip_gated_linear_backward_workspace(3, 64, 48)
    assert need == 2 * 3 * 48 * 2

    def call(x=(3, 64), w=(2, 64, 48), gu=(2, 3, 48), dh=(3, 48), dx=(3, 64), dw=(2, 64, 48), act=1, work=1 << 41, have=need, alias=None):
        t = dict(x=m(*x), w=m(*w), gu=gu and m(*gu), dh=m(*dh), dx=dx and m(*dx), dw=dw and m(*dw))
        if alias:
            t[alias[0]].data = t[alias[1]].data
        return L.evkhip_gated_linear_backward(*[v and b(v) for v in t.values()], act, 0, work, have, None)

    assert call(gu=None) == INVALID
    assert call(dx=(3, 63)) == SHAPE
    assert call(dw=(2, 64, 47)) == SHAPE
    assert call(dh=(3, 47)) == SHAPE
    assert call(have=need - 1) == INVALID
    assert call(work=None) == INVALID
    assert call(act=7) == INVALID
    for alias in (("dx", "x"), ("dw", "w"), ("dx", "dh"), ("dw", "gu")):
        assert call(alias=alias) == INVALID
    # dx and dw at one address
    assert call(x=(3, 64), dx=(3, 64), alias=("dx", "dw")) == INVALID


def test_python_wrappers_refuse():
    """Types, devices and names are checked before the library is called."""
    f16 = torch.float16
    x, w, h = torch.zeros(3, 64, dtype=f16), torch.zeros(2, 64, 48, dtype=f16), torch.zeros(3, 48, dtype=f16)
    with pytest.raises(ValueError, match="GPU"):
        evk.gated_linear(x, w, h)
    with pytest.raises(ValueError, match="float16"):
        evk.gated_linear(x.float(), w, h)
    with pytest.raises(ValueError, match="float16"):
        evk.window_attention(x.float(), w, h, h, 64)
    with pytest.raises(ValueError, match="activation"):
        evk._activation("swish")
    with pytest.raises(ValueError, match="at least"):
        evk._at_least(0, window=-1)
    # another type, another device than the call's first tensor
    with pytest.raises(ValueError, match="float16"):
        evk._H(x.bfloat16(), -1)
    with pytest.raises(ValueError, match="float16"):
        evk._H(x, 0)
    assert evk._H(None, 0) is None
    # strides, lengths and types of the other tensors
    with pytest.raises(ValueError, match="contiguous"):
        evk._H(x.t(), -1)
    with pytest.raises(ValueError, match="5 contiguous"):
        evk._P(torch.zeros(4, dtype=torch.int32), -1, torch.int32, 5)
    with pytest.raises(ValueError, match="contiguous"):
        evk._P(torch.zeros(5, dtype=torch.int64), -1, torch.int32, 5)
    # a stream of the caller's own needs a workspace of its own
    with pytest.raises(ValueError, match="workspace"):
        evk._workspace(None, 64, 0, 12345)
    assert evk._workspace(None, 0, 0, 12345) == (None, None, 0)


def test_more_rows_than_a_launch_holds(L):
    """Sizes below the 2^30 rows of the checks whose launches would pass 2^32 threads."""
    m = Mem()
    n = 1 << 26
    assert rope(L, m, qkv=(n, 1, 6), q=(n, 1, 2), k=(n, 1, 2), dh=2) == UNSUPPORTED
    assert window(L, m, q=(n, 1, 8), k=(n, 1, 8), dh=8) == UNSUPPORTED  # single tokens
    assert window(L, m, q=(n, 1, 3), k=(n, 1, 3), dh=3) == UNSUPPORTED  # row by row
    need = L.evkhip_window_attention_bwd_workspace(n, 1, 1, 1, 8, 4, 1)
    t = [m(n, 1, 8) for _ in range(8)]
    assert L.evkhip_window_attention_bwd(*[b(x) for x in t], 1 << 50, 8, 4, 1, 1 << 51, need, None) == UNSUPPORTED
    assert b"workgroups" in L.evkhip_last_error()


def test_lse_alignment(L):
    m = Mem()
    q, k = m(2, 5, 256), m(2, 9, 128)
    args = [b(x) for x in (q, k, m(2, 9, 128), m(2, 5, 256))]
    assert L.evkhip_window_attention(*args, 64, 4, 1, 0, None, (1 << 42) + 2, None, 0, None) == INVALID
    assert b"lse" in L.evkhip_last_error()


@pytest.mark.parametrize("name,value", [("window", 1 << 32), ("sinks", -1), ("position_offset", (1 << 32) + 3)])
def test_python_sizes_are_not_cut_to_32_bits(name, value):
    with pytest.raises(ValueError, match=name):
        evk._at_least(0, **{name: value})
