"""CPU-only: the entry points of the operators of a group of continuations
refuse what they do not take, with the documented codes and before any GPU call,
and name the workspace that a call needs."""
import ctypes as C

import pytest
import torch

import evk_amd as evk
from test_block_refusals import INVALID, OK, SHAPE, UNSUPPORTED, Mem

b = C.byref


@pytest.fixture(scope="module")
def L():
    if not evk.available():
        pytest.fail("libevkhip.so is not built: run `python -m evk_amd.build`")
    return evk.lib()


def opt(m, shape):
    return None if shape is None else m(*shape)


def norm(L, m, x=(2, 5, 64), y=(2, 5, 64), wo=(64,), gate=None, wi=(64,), s=(2, 5, 64), h=(2, 5, 64), scale=1.0, post=1, eps=1e-4, alias=None, null=None):
    t = dict(x=m(*x), y=opt(m, y), wo=opt(m, wo), gate=opt(m, gate), wi=opt(m, wi), s=opt(m, s), h=m(*h))
    if alias:
        t[alias[0]].data = t[alias[1]].data + (alias[2] if len(alias) > 2 else 0)
    if null:
        t[null].data = None
    return L.evkhip_residual_norm(*[v and b(v) for v in t.values()], scale, post, eps, None)


def test_residual_norm(L):
    m = Mem()
    assert norm(L, m, y=(2, 5, 63)) == SHAPE
    assert norm(L, m, y=(10, 64)) == SHAPE
    assert norm(L, m, s=(2, 4, 64)) == SHAPE
    assert norm(L, m, h=(2, 5, 65)) == SHAPE
    assert norm(L, m, wo=(63,)) == SHAPE
    assert norm(L, m, wi=(1, 64)) == SHAPE
    assert norm(L, m, gate=(3, 64)) == SHAPE
    assert norm(L, m, gate=(2, 63)) == SHAPE
    assert norm(L, m, gate=(2, 5, 64)) == SHAPE
    assert norm(L, m, x=(64,), y=(64,), s=(64,), h=(64,), gate=(1, 64)) == SHAPE  # no sequences
    assert norm(L, m, s=None) == INVALID
    assert norm(L, m, y=None, wo=None) == INVALID  # s without y
    assert norm(L, m, y=None, s=None) == INVALID  # the weight of a norm that is not there
    assert norm(L, m, y=None, s=None, wo=None, gate=(64,)) == INVALID
    assert norm(L, m, y=None, s=None, wo=None, scale=0.5) == INVALID
    assert norm(L, m, post=0) == INVALID
    assert norm(L, m, null="x") == INVALID and norm(L, m, null="h") == INVALID and norm(L, m, null="wi") == INVALID
    for eps in (-1.0, float("nan"), float("inf")):
        assert norm(L, m, eps=eps) == INVALID
    for scale in (float("nan"), float("inf"), 65505.0, -70000.0, 2.0 ** -25):
        assert norm(L, m, scale=scale) == INVALID
    for alias in (("s", "x"), ("h", "y", 2), ("h", "s", 1278), ("s", "wi"), ("h", "wo")):
        assert norm(L, m, alias=alias) == INVALID, alias
        assert b"overlaps" in L.evkhip_last_error()
    wide = (1, 1, 16385)
    assert norm(L, m, x=wide, y=wide, s=wide, h=wide, wo=None, wi=None) == UNSUPPORTED
    many = ((1 << 30) + 1, 1)
    assert norm(L, m, x=many, y=many, s=many, h=many, wo=None, wi=None) == UNSUPPORTED
    past = (1 << 31, 1 << 31, 1 << 31, 64)  # 2^99 values
    assert L.evkhip_residual_norm(b(evk.desc((4096, past))), None, None, None, None, None, b(evk.desc((4096, past))), 1.0, 1, 1e-4, None) == UNSUPPORTED
    assert L.evkhip_residual_norm(None, None, None, None, None, None, None, 1.0, 1, 1e-4, None) == INVALID
    none = (2, 0, 64)
    assert norm(L, m, x=none, y=none, s=none, h=none, gate=(2, 64)) == OK
    none = (2, 5, 0)
    assert norm(L, m, x=none, y=none, s=none, h=none, wo=(0,), wi=(0,)) == OK


def test_residual_norm_backward(L):
    m = Mem()
    ws = L.evkhip_residual_norm_backward_workspace(10, 2, 64)
    assert ws > 0 and L.evkhip_residual_norm_backward_workspace(0, 1, 64) == 0 and L.evkhip_residual_norm_backward_workspace(10, 11, 64) == 0

    def call(x=(2, 5, 64), y=(2, 5, 64), wo=(64,), gate=(2, 64), wi=(64,), ds=(2, 5, 64), dh=(2, 5, 64), dx=(2, 5, 64), dy=(2, 5, 64), dwo=(64,),
             dgate=(2, 64), dwi=(64,), scale=1.0, post=1, work=1 << 40, have=None, alias=None):
        t = dict(x=m(*x), y=opt(m, y), wo=opt(m, wo), gate=opt(m, gate), wi=opt(m, wi), ds=opt(m, ds), dh=m(*dh), dx=m(*dx), dy=opt(m, dy),
                 dwo=opt(m, dwo), dgate=opt(m, dgate), dwi=opt(m, dwi))
        if alias:
            t[alias[0]].data = t[alias[1]].data
        return L.evkhip_residual_norm_backward(*[v and b(v) for v in t.values()], scale, post, 1e-4, 0, work, ws if have is None else have, None)

    assert call(have=ws - 1) == INVALID
    assert call(work=None) == INVALID
    assert call(work=(1 << 40) + 8) == INVALID
    assert call(dy=None) == INVALID
    assert call(y=None, wo=None, gate=None, dwo=None, dgate=None) == INVALID  # dy without y
    assert call(wo=None) == INVALID and call(gate=None) == INVALID and call(wi=None) == INVALID  # gradients of what is not there
    assert call(ds=(2, 5, 65)) == SHAPE and call(dh=(2, 4, 64)) == SHAPE and call(dx=(10, 64)) == SHAPE and call(dy=(2, 5, 8)) == SHAPE
    assert call(dwo=(63,)) == SHAPE and call(dgate=(64,)) == SHAPE and call(dwi=(65,)) == SHAPE
    for alias in (("dx", "x"), ("dy", "ds"), ("dx", "dy"), ("dwo", "wo"), ("dgate", "gate"), ("dwi", "dwo"), ("dx", "dh")):
        assert call(alias=alias) == INVALID, alias
        assert b"overlaps" in L.evkhip_last_error()
    none = dict(x=(2, 0, 64), y=(2, 0, 64), ds=None, dh=(2, 0, 64), dx=(2, 0, 64), dy=(2, 0, 64), dwo=None, dgate=None, dwi=None, work=None, have=0)
    assert call(**none) == OK
    # gates one a row, more than a launch holds
    n = 1 << 29
    need = L.evkhip_residual_norm_backward_workspace(n, n, 8)
    big = dict(x=(n, 8), y=(n, 8), ds=None, dh=(n, 8), dx=(n, 8), dy=(n, 8), wo=None, gate=(n, 8), wi=None, dwo=None, dgate=(n, 8), dwi=None)
    assert call(**big, work=1 << 60, have=need) == UNSUPPORTED
    assert b"workgroups" in L.evkhip_last_error()


def prefix(L, m, q=(2, 5, 256), pk=(7, 128), pv=None, k=(2, 9, 128), v=None, o=None, dh=64, p0=0, off=None, lse=None, work=1 << 41, have=1 << 40, alias=None):
    t = dict(q=m(*q), pk=m(*pk), pv=m(*(pv or pk)), k=m(*k), v=m(*(v or k)), o=m(*(o or q)))
    if alias:
        t[alias[0]].data = t[alias[1]].data
    return L.evkhip_prefix_attention(*[b(x) for x in t.values()], dh, p0, off, lse, work, have, None)


def test_prefix_attention(L):
    m = Mem()
    assert prefix(L, m, p0=5) == SHAPE
    assert prefix(L, m, p0=0xffffffff) == SHAPE
    assert prefix(L, m, p0=1, off=4096) == INVALID
    assert prefix(L, m, off=4098) == INVALID
    assert prefix(L, m, lse=4098) == INVALID
    assert prefix(L, m, dh=0) == INVALID
    assert prefix(L, m, q=(2, 5, 1024), pk=(7, 1024), k=(2, 9, 1024), dh=512) == UNSUPPORTED
    assert prefix(L, m, q=(2, 5, 192)) == SHAPE  # 3 heads over 2
    assert prefix(L, m, q=(2, 5, 250)) == SHAPE
    assert prefix(L, m, pk=(7, 64)) == SHAPE
    assert prefix(L, m, pk=(1, 7, 128)) == SHAPE
    assert prefix(L, m, pv=(8, 128)) == SHAPE
    assert prefix(L, m, o=(2, 5, 255)) == SHAPE
    assert prefix(L, m, k=(1, 9, 128)) == SHAPE
    assert prefix(L, m, v=(2, 9, 64)) == SHAPE
    assert prefix(L, m, pk=(1 << 30, 128)) == UNSUPPORTED
    assert prefix(L, m, q=(1, 1, 64), pk=(1 << 29, 64), k=(1, (1 << 29) + 1, 64)) == UNSUPPORTED
    assert prefix(L, m, q=(1 << 29, 1, 256), k=(1 << 29, 1, 128)) == UNSUPPORTED
    for alias in (("o", "q"), ("o", "pk"), ("o", "pv"), ("o", "k"), ("o", "v")):
        assert prefix(L, m, alias=alias) == INVALID, alias
        assert b"overlaps" in L.evkhip_last_error()
    assert prefix(L, m, q=(0, 5, 256), k=(0, 9, 128), work=None, have=0) == OK
    assert prefix(L, m, q=(2, 0, 256), work=None, have=0) == OK
    assert prefix(L, m, q=(2, 0, 256), pk=(0, 128), k=(2, 0, 128), work=None, have=0) == OK
    for sizes in ((0, 1, 1, 1, 1, 1, 64), (1, 1, 1, 1, 3, 2, 64), (1, 1, 1, 1, 1, 1, 0), (1, 1, 1, 1, 1, 1, 257), (1 << 31, 1 << 31, 1, 1, 1, 1, 64)):
        assert L.evkhip_prefix_attention_workspace(*sizes) == 0, sizes


def test_qkv_norm_rope_behind(L):
    m = Mem()
    t = [m(2, 5, 512), None, None, m(2, 5, 256), m(2, 9, 128), m(2, 9, 128)]
    call = lambda first, p0: L.evkhip_qkv_norm_rope_behind(*[x and b(x) for x in t], 64, 1e-4, 1e4, first, p0, None, None)  # noqa: E731
    assert call((1 << 30) + 1, 0) == UNSUPPORTED
    assert call(100, 5) == SHAPE


def scores(L, m, logits=(6, 100), tokens=(6,), lp=4096, ent=8192, ids=(6, 5), alt=1 << 16, stats=1 << 17, c=1.0, alias=None):
    t = dict(logits=m(*logits), tokens=m(*tokens), ids=opt(m, ids))
    if alias:
        t[alias[0]].data = t[alias[1]].data
    return L.evkhip_token_logprobs(b(t["logits"]), b(t["tokens"]), lp, ent, t["ids"] and b(t["ids"]), alt, stats, c, None)


def test_token_logprobs(L):
    m = Mem()
    assert scores(L, m, tokens=(5,)) == SHAPE
    assert scores(L, m, logits=(6, 0)) == SHAPE
    assert scores(L, m, logits=(6, 65537)) == UNSUPPORTED
    assert scores(L, m, ids=(5, 5)) == SHAPE
    assert scores(L, m, logits=(6, 4)) == SHAPE  # 5 of 4
    assert scores(L, m, ids=(6, 33)) == UNSUPPORTED
    assert scores(L, m, lp=None) == INVALID
    assert scores(L, m, ids=None) == INVALID and scores(L, m, alt=None) == INVALID
    for name in ("lp", "ent", "alt", "stats"):
        assert scores(L, m, **{name: 4098}) == INVALID
    for c in (0.0, -1.0, float("nan"), float("inf"), 70000.0, 2.0 ** -25):
        assert scores(L, m, c=c) == INVALID
    assert scores(L, m, alias=("ids", "logits")) == INVALID and scores(L, m, alias=("ids", "tokens")) == INVALID
    assert scores(L, m, ent=4096) == INVALID and scores(L, m, stats=4100) == INVALID
    assert L.evkhip_token_logprobs(None, None, None, None, None, None, None, 1.0, None) == INVALID
    assert scores(L, m, logits=(0, 100), tokens=(0,), lp=None, ent=None, ids=None, alt=None, stats=None) == OK
    past = (1 << 31, 1 << 31, 1 << 31, 64)
    assert scores(L, m, logits=past) == UNSUPPORTED
    many = 1 << 24  # workgroups of 256 threads
    assert scores(L, m, logits=(many, 32000), tokens=(many,), lp=1 << 50, ent=1 << 51, ids=None, alt=None, stats=1 << 52) == UNSUPPORTED


def test_token_logprobs_backward(L):
    m = Mem()

    def call(logits=(6, 100), tokens=(6,), stats=4096, ent=8192, dlp=1 << 16, dent=1 << 17, d=(6, 100), c=1.0, alias=None):
        t = dict(logits=m(*logits), tokens=m(*tokens), d=m(*d))
        if alias:
            t[alias[0]].data = t[alias[1]].data
        return L.evkhip_token_logprobs_backward(b(t["logits"]), b(t["tokens"]), stats, ent, dlp, dent, b(t["d"]), c, None)

    assert call(d=(6, 99)) == SHAPE and call(tokens=(7,)) == SHAPE
    assert call(stats=None) == INVALID and call(dlp=None, dent=None) == INVALID and call(ent=None) == INVALID
    for name in ("stats", "ent", "dlp", "dent"):
        assert call(**{name: 4098}) == INVALID
    assert call(alias=("d", "logits")) == INVALID and call(alias=("d", "tokens")) == INVALID
    assert call(c=0.0) == INVALID
    assert call(logits=(0, 100), tokens=(0,), d=(0, 100), stats=None, ent=None, dlp=None, dent=None) == OK


def test_python_checks():
    """The wrappers name a wrong type or device themselves."""
    x = torch.zeros(2, 3, 64)
    with pytest.raises(ValueError, match="float16"):
        evk.residual_norm(x, x, x, x)
    h = x.half()
    for call in (lambda: evk.residual_norm(h, h, h, h), lambda: evk.token_logprobs(h, x, x), lambda: evk.prefix_attention(h, h, h, h, h, h, 64),
                 lambda: evk.residual_norm_backward(h, h, h, h, h, h), lambda: evk.token_logprobs_backward(h, x, x, x, h)):
        with pytest.raises((ValueError, RuntimeError)):
            call()


@pytest.mark.parametrize("rank", [0, 9, 1 << 31])
def test_alternatives_of_a_rank_that_is_none(L, rank):
    """The descriptor's sizes are not read before its rank has been checked, with or without a place for their log p."""
    m = Mem()
    for alt in (None, 1 << 16):
        ids = m(6, 5)
        ids.rank = rank
        logits, tokens = m(6, 100), m(6)
        assert L.evkhip_token_logprobs(b(logits), b(tokens), 4096, None, b(ids), alt, None, 1.0, None) == SHAPE
        assert b"rank" in L.evkhip_last_error()
