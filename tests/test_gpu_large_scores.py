"""GPU: attention over a window and behind a shared prefix at scores whose exponents
pass what 32 bits hold beside small differences.

The inputs make every score a whole number below 2^24 (or equal scores of any
size): 32 bits hold them exactly in any order of the sum, and the softmax in 64
bits from the same numbers is what the operators have to give.  H, T and E as in
test_gpu_block.py."""
import math

import pytest
import torch

import evk_amd as evk
from test_gpu_block import E, F16, F64, H, T, Rng, close, empty

pytestmark = pytest.mark.gpu


def softmax_want(s, v, scale):
    """o (rows, dh), lse (rows) in 64 bits from whole-number scores s (rows, n) and v (n, dh), and their tolerances."""
    lse = torch.logsumexp(s * scale, 1)
    p = torch.exp(s * scale - lse[:, None])
    o = p @ v
    # a weight: its rounding to fp16 (H); the exponent below 2^12 is one product and one sum (E 2^12 each), past that a
    # difference is formed first; parts' references meet by such differences as well
    rel = 2 * H + 4 * E * 2.0 ** 12
    o_t = rel * (p @ v.abs()) + s.shape[1] * (T + E) * v.abs().amax(0, keepdim=True) + T
    # |m| / sqrt(dh) and the logarithm, a product and a sum in 32 bits; l is off as the weights are
    return o, lse, o_t, 4 * E * lse.abs() + rel + (s.shape[1] + 16) * E


def inputs(r, dh, heads, n, size, sign, span):
    """Queries (n, heads, dh) and keys of whole numbers: `dh - 1` products that add up to about sign * size, the same for
    every key, and one of -span .. span that differs; keys come as a function of their number."""
    big = 2.0 ** round(math.log2(max(size / (dh - 1), 1.0)) / 2)
    q = torch.full((n, heads, dh), big, dtype=F64, device=r.dev)
    q[..., -1] = 1.0

    def keys(*shape):
        k = torch.full((*shape, dh), sign * big, dtype=F64, device=r.dev)
        k[..., -1] = torch.randint(-span, span + 1, shape, device=r.dev, generator=r.g).to(F64)
        return k

    assert (dh - 1) * big * big + span < 2 ** 24
    return q, keys


SIZES = [2.0 ** 8, 2.0 ** 14, 2.0 ** 17, 2.0 ** 20, 2.0 ** 23]
# heads, key heads, head size, queries: single tokens, some, prompts; a head size that goes row by row
WINDOW = [(8, 2, 64, 1, 6000), (4, 1, 128, 3, 700), (2, 1, 256, 1, 3000), (8, 2, 128, 700, 700), (4, 2, 40, 900, 900), (2, 1, 256, 600, 600), (2, 1, 36, 3, 300)]


@pytest.mark.parametrize("sign", [1.0, -1.0])
@pytest.mark.parametrize("size", SIZES)
@pytest.mark.parametrize("h,kv,dh,n,rows", WINDOW)
def test_window_attention(dev, h, kv, dh, n, rows, size, sign):
    r = Rng(dev, 11 + dh)
    span = int(3 * dh ** 0.5)
    q, keys = inputs(r, dh, h, n, size, sign, span)
    k, v = keys(rows, kv), r(rows, kv, dh).to(F64)
    o, lse = empty(dev, 1, n, h * dh), torch.zeros(1, h, n, device=dev)
    evk.window_attention(q.to(F16).view(1, n, -1), k.to(F16).view(1, rows, -1), v.to(F16).view(1, rows, -1), o, dh, position_offset=rows - n, lse=lse)
    check(o[0], lse[0], q, [k] * n, [v] * n, [rows - n + t + 1 for t in range(n)], kv, f"window {size} {sign}")


def check(o, lse, q, ks, vs, seen, kv, what):
    """Every query's output against the softmax over the first seen[t] rows of its ks[t] and vs[t] (one list for runs of queries)."""
    n, h, dh = q.shape
    o = o.view(n, h, dh)
    step = max(1, n // 20)  # of a prompt some, among them the first and the last
    for t in sorted({*range(0, n, step), n - 1}):
        for c in range(kv):
            at = slice(c * (h // kv), (c + 1) * (h // kv))
            k, v = ks[t][:seen[t], c], vs[t][:seen[t], c]
            want = softmax_want(q[t, at] @ k.t(), v, dh ** -0.5)
            close(o[t, at], want[0], want[2], f"o {what} query {t}")
            close(lse[at, t], want[1], want[3], f"lse {what} query {t}", norm=None)


# sequences, queries, heads, key heads, head size, prefix, own rows: steps in one workgroup and in parts, the prefix shared (64 and
# 128 rows a tile), prompts with a list in one part and in several, row by row
PREFIX = [(3, 1, 8, 2, 64, 300, 50), (1, 1, 8, 2, 128, 9000, 40), (6, 1, 8, 2, 64, 20000, 70), (64, 1, 32, 8, 128, 2000, 300), (3, 5, 2, 1, 256, 6000, 90),
          (3, 150, 8, 2, 64, 333, 200), (2, 300, 4, 1, 128, 2000, 320), (2, 300, 2, 1, 256, 300, 300), (2, 2, 2, 1, 36, 100, 30)]


@pytest.mark.parametrize("sign", [1.0, -1.0])
@pytest.mark.parametrize("size", SIZES)
@pytest.mark.parametrize("b,n,h,kv,dh,p,rows", PREFIX)
def test_prefix_attention(dev, b, n, h, kv, dh, p, rows, size, sign):
    r = Rng(dev, 31 + dh)
    span = int(3 * dh ** 0.5)
    q, keys = inputs(r, dh, h, n, size, sign, span)
    pk, k, pv, v = keys(p, kv), keys(b, rows, kv), r(p, kv, dh), r(b, rows, kv, dh)
    off = [(7 * s) % (rows - n + 1) for s in range(b)]
    half = lambda t: t.to(F16).reshape(*t.shape[:-2], -1).contiguous()  # noqa: E731
    o, lse = empty(dev, b, n, h * dh), torch.zeros(b, h, n, device=dev)
    evk.prefix_attention(half(q)[None].expand(b, -1, -1).contiguous(), half(pk), half(pv), half(k), half(v), o, dh,
                         offsets=torch.tensor(off, dtype=torch.int32, device=dev), lse=lse)
    for s in sorted({0, b // 2, b - 1}):
        kk, vv = torch.cat([pk, k[s]]), torch.cat([pv, v[s]]).to(F64)
        check(o[s], lse[s], q, [kk] * n, [vv] * n, [p + off[s] + t + 1 for t in range(n)], kv, f"prefix {size} {sign}")


def equal_scores(dev, c, dh, heads, *shape):
    return torch.full((*shape, heads * dh), c, dtype=F16, device=dev)


@pytest.mark.parametrize("sign", [1.0, -1.0])
@pytest.mark.parametrize("c", [1000.0, 5000.0, 6000.0, 8000.0, 16000.0, 60000.0])
@pytest.mark.parametrize("b,n,h,kv,dh,p,rows", PREFIX)
def test_prefix_attention_equal_scores(dev, b, n, h, kv, dh, p, rows, c, sign):
    """Equal scores up to 10^12: the mean of the values.  The sum of n values in 32 bits, one rounding."""
    r = Rng(dev, 51 + dh)
    pv, v = r(p, kv * dh), r(b, rows, kv * dh)
    o, lse = empty(dev, b, n, h * dh), torch.zeros(b, h, n, device=dev)
    evk.prefix_attention(equal_scores(dev, c, dh, h, b, n), equal_scores(dev, sign * c, dh, kv, p), pv, equal_scores(dev, sign * c, dh, kv, b, rows), v, o, dh,
                         rows - n, lse=lse)
    for s in sorted({0, b - 1}):
        for t in sorted({0, n - 1}):
            vv = torch.cat([pv, v[s, :rows - n + t + 1]]).to(F64).view(-1, kv, dh)
            mean_check(o[s, t].view(kv, h // kv, dh), lse[s, :, t], vv, sign * c * c * dh ** 0.5)


@pytest.mark.parametrize("sign", [1.0, -1.0])
@pytest.mark.parametrize("c", [1000.0, 5000.0, 8000.0, 16000.0, 60000.0])
@pytest.mark.parametrize("h,kv,dh,n,rows", WINDOW)
def test_window_attention_equal_scores(dev, h, kv, dh, n, rows, c, sign):
    r = Rng(dev, 61 + dh)
    v = r(1, rows, kv * dh)
    o, lse = empty(dev, 1, n, h * dh), torch.zeros(1, h, n, device=dev)
    evk.window_attention(equal_scores(dev, c, dh, h, 1, n), equal_scores(dev, sign * c, dh, kv, 1, rows), v, o, dh, position_offset=rows - n, lse=lse)
    for t in sorted({0, n // 2, n - 1}):
        mean_check(o[0, t].view(kv, h // kv, dh), lse[0, :, t], v[0, :rows - n + t + 1].to(F64).view(-1, kv, dh), sign * c * c * dh ** 0.5)


def mean_check(o, lse, v, score):
    """o (kv, group, dh): the mean over v (rows, kv, dh); lse (heads): the score and log of the rows.  A score is dh products'
    sum, the same for every key, off by (dh + 4) E of itself."""
    rows, _, dh = v.shape
    want, size = v.mean(0)[:, None].expand_as(o), v.abs().mean(0)[:, None].expand_as(o)
    close(o, want, H * want.abs() + T + (rows + 64) * E * size, "o")
    w = torch.full_like(lse, score + math.log(rows), dtype=F64)
    close(lse, w, (dh + 8) * E * abs(score) + (rows + 64) * E + 4 * E * w.abs(), "lse", norm=None)


@pytest.mark.parametrize("dh,n,p", [(64, 1, 100), (128, 9, 4000), (64, 300, 200), (256, 2, 3000)])
@pytest.mark.parametrize("size", [2.0 ** 8, 2.0 ** 20, 2.0 ** 23])
def test_values_that_are_not_finite_at_large_scores(dev, dh, n, p, size):
    """A row of V with one infinity, which not every query of a tile sees: its other values come with the weight that the sum
    holds for it."""
    r = Rng(dev, 71 + dh)
    b, h, kv, rows = 3, 2, 1, n + 5
    q, keys = inputs(r, dh, h, n, size, 1.0, int(3 * dh ** 0.5))
    pk, k, pv, v = keys(p, kv), keys(b, rows, kv), r(p, kv, dh), r(b, rows, kv, dh)
    j = n // 2
    v[:, j, 0, 3] = math.inf
    k[:, j, 0, -1] = int(3 * dh ** 0.5)  # not a small weight
    half = lambda t: t.to(F16).reshape(*t.shape[:-2], -1).contiguous()  # noqa: E731
    o = empty(dev, b, n, h * dh)
    evk.prefix_attention(half(q)[None].expand(b, -1, -1).contiguous(), half(pk), half(pv), half(k), half(v), o, dh)
    for s in (0, b - 1):
        for t in sorted({0, max(j - 1, 0), j, n - 1}):
            kk, vv = torch.cat([pk, k[s, :t + 1]])[:, 0], torch.cat([pv, v[s, :t + 1]]).to(F64)[:, 0]
            want = softmax_want(q[t] @ kk.t(), vv.nan_to_num(posinf=0.0), dh ** -0.5)
            got = o[s, t].view(h, dh).to(F64)
            clear = torch.ones(dh, dtype=torch.bool, device=dev)
            if t >= j:
                assert (got[:, 3] == math.inf).all()
                clear[3] = False
            close(got[:, clear], want[0][:, clear], want[2][:, clear], f"o of query {t}")
