"""GPU: the operators of a grouped-query block (qkv_norm_rope, window_attention,
gated_linear, forward and backward) against plain 64-bit formulas.

Tolerances are worst cases of the roundings that the operators make, element by
element: H = 2^-11 is half a step of fp16 relative to a value, T = 2^-25 half a
step of its subnormals, E = 2^-24 half a step of 32 bits.  Sums of n products in
32 bits are off by at most n E times the sum of the products' magnitudes.  The
norm of the whole difference is bounded as well: k independent roundings are off
by at most sqrt(k) H of the norm, so 2 H covers the two to four that each output
has behind it (a term left out of a sum of a thousand would show as 3e-2)."""
import math

import pytest
import torch

import evk_amd as evk

pytestmark = pytest.mark.gpu

H, T, E = 2.0 ** -11, 2.0 ** -25, 2.0 ** -24
F16, F32, F64 = torch.float16, torch.float32, torch.float64


class Rng:
    def __init__(self, dev, seed):
        self.dev, self.g = dev, torch.Generator(device=dev)
        self.g.manual_seed(seed)

    def __call__(self, *shape, std=1.0, mean=0.0, odd=False):
        """Normal fp16 values; `odd` puts them at an address that is no multiple of 4."""
        n = math.prod(shape)
        t = torch.empty(n + 8, dtype=F16, device=self.dev).normal_(mean, std, generator=self.g)
        return t[1:1 + n].view(shape) if odd else t[:n].view(shape)


def empty(dev, *shape, odd=False, fill=7.0):
    n = math.prod(shape)
    t = torch.full((n + 8,), fill, dtype=F16, device=dev)
    return t[1:1 + n].view(shape) if odd else t[:n].view(shape)


def close(got, want, tol, what, norm=2 * H):
    got, want = got.to(F64), want.to(F64)
    assert got.shape == want.shape, what
    assert torch.equal(torch.isnan(got), torch.isnan(want)), f"{what}: NaN in other places"
    ok = torch.isfinite(want)
    assert torch.equal(got[~ok & ~torch.isnan(want)], want[~ok & ~torch.isnan(want)]), f"{what}: infinities differ"
    d = torch.where(ok, got - want, torch.zeros_like(want)).abs()
    bad = (d > tol) & ok
    if bad.any():
        i = int((d - tol).masked_fill(~ok, -1).argmax())
        raise AssertionError(f"{what}: {int(bad.sum())} of {d.numel()} values off; at {i}: got {got.flatten()[i]:.6g}, "
                             f"want {want.flatten()[i]:.6g}, tolerance {tol.expand_as(d).flatten()[i]:.3g}")
    w = want[ok]
    if norm and w.numel() > 200:
        rel = float(d[ok].norm() / w.norm().clamp(min=1e-30))
        assert rel <= norm, f"{what}: relative norm of the difference {rel:.3g} > {norm:.3g}"


# ---------------------------------------------------------------------------
# qkv_norm_rope
# ---------------------------------------------------------------------------
def turn(x, pos, base, sign=1.0):
    """Pairs of the last dimension turned; x (B, N, heads, dh), pos (B, N)."""
    dh = x.shape[-1]
    ang = pos.to(F64)[..., None, None] * base ** (-torch.arange(0, dh, 2, device=x.device, dtype=F64) / dh)
    c, s = torch.cos(ang), sign * torch.sin(ang)
    a, b = x[..., 0::2], x[..., 1::2]
    return torch.stack([a * c - b * s, a * s + b * c], -1).flatten(-2)


def rope_want(qkv, wq, wk, h, kv, dh, pos, eps, base):
    """(q, k, v) heads in 64 bits and the largest error of q and k before the rounding."""
    b, n, _ = qkv.shape
    x = qkv.to(F64).view(b, n, h + 2 * kv, dh)
    w = torch.ones(h + kv, dh, dtype=F64, device=qkv.device)
    if wq is not None:
        w[:h] = wq.to(F64)
    if wk is not None:
        w[h:] = wk.to(F64)
    y = x[:, :, :h + kv]
    y = y / torch.sqrt(y.square().mean(-1, keepdim=True) + eps) * w
    size = y.abs()[..., 0::2] + y.abs()[..., 1::2]  # a turned pair's members are at most this
    return turn(y, pos, base), x[:, :, h + kv:], torch.repeat_interleave(size, 2, -1)


ROPE = [  # b, n, heads, kv, dh, rows, p0, weights, odd
    (1, 1, 1, 1, 2, 1, 0, True, False), (2, 3, 4, 2, 64, 3, 0, True, False), (3, 7, 12, 4, 64, 20, 9, False, False),
    (1, 130, 8, 1, 128, 140, 10, True, False), (2, 5, 3, 3, 80, 5, 0, True, True), (1, 33, 6, 2, 96, 64, 31, True, False),
    (2, 9, 2, 1, 256, 9, 0, True, False), (1, 4, 5, 5, 34, 4, 0, True, True), (2, 2, 2, 2, 250, 7, 5, False, True),
    (1, 2, 4, 2, 6, 2, 0, True, False), (4, 600, 16, 8, 128, 600, 0, True, False), (1, 2, 2, 1, 32, 100002, 100000, True, False),
]


@pytest.mark.parametrize("b,n,h,kv,dh,rows,p0,weights,odd", ROPE)
def test_qkv_norm_rope(dev, b, n, h, kv, dh, rows, p0, weights, odd):
    r = Rng(dev, 1000 + n + dh)
    qkv = r(b, n, (h + 2 * kv) * dh, odd=odd)
    wq, wk = (r(dh, std=0.2, mean=1.0, odd=odd), r(dh, std=0.2, mean=1.0)) if weights else (None, None)
    q, k, v = empty(dev, b, n, h * dh, odd=odd), empty(dev, b, rows, kv * dh, odd=odd), empty(dev, b, rows, kv * dh)
    evk.qkv_norm_rope(qkv, q, k, v, dh, wq, wk, 1e-4, 10000.0, p0)
    pos = (p0 + torch.arange(n, device=dev)).expand(b, n)
    y, vw, size = rope_want(qkv, wq, wk, h, kv, dh, pos, 1e-4, 10000.0)
    tol = H * y.abs() + 2.0 ** -20 * size + T  # the norm, the angle's 24 bits and the turn: a dozen roundings of 2^-24
    close(q.view(b, n, h, dh), y[:, :, :h], tol[:, :, :h], "q")
    close(k[:, p0:p0 + n].view(b, n, kv, dh), y[:, :, h:], tol[:, :, h:], "k")
    assert torch.equal(v[:, p0:p0 + n].view(b, n, kv, dh).to(F64), vw), "v"
    for t in (k, v):  # the other rows keep their values
        assert (t[:, :p0] == 7.0).all() and (t[:, p0 + n:] == 7.0).all()


def test_qkv_norm_rope_offsets(dev):
    """Sequences at positions of their own; an idle one (-5) and one past the cache write no rows."""
    b, n, h, kv, dh, rows = 6, 3, 4, 2, 64, 40
    r = Rng(dev, 5)
    qkv, wq, wk = r(b, n, (h + 2 * kv) * dh), r(dh, mean=1.0), r(dh, mean=1.0)
    off = torch.tensor([0, 37, -5, 38, 11, 2 ** 31 - 2], dtype=torch.int32, device=dev)
    q, k, v = empty(dev, b, n, h * dh), empty(dev, b, rows, kv * dh), empty(dev, b, rows, kv * dh)
    evk.qkv_norm_rope(qkv, q, k, v, dh, wq, wk, 1e-4, 500.0, 0, off)
    pos = off.long()[:, None] + torch.arange(n, device=dev)
    y, vw, size = rope_want(qkv, wq, wk, h, kv, dh, pos, 1e-4, 500.0)
    tol = H * y.abs() + 2.0 ** -20 * size + T
    close(q.view(b, n, h, dh)[:5], y[:5, :, :h], tol[:5, :, :h], "q")
    wk_, wv_ = torch.full((b, rows, kv, dh), 7.0, dtype=F64, device=dev), torch.full((b, rows, kv, dh), 7.0, dtype=F64, device=dev)
    wt = torch.zeros_like(wk_)
    for s in range(b):
        for t in range(n):
            p = int(pos[s, t])
            if 0 <= p < rows:
                wk_[s, p], wv_[s, p], wt[s, p] = y[s, t, h:], vw[s, t], tol[s, t, h:]
    close(k.view(b, rows, kv, dh), wk_, wt, "k")
    assert torch.equal(v.view(b, rows, kv, dh).to(F64), wv_)


@pytest.mark.parametrize("b,n,h,kv,dh,rows,p0,weights,odd", ROPE)
def test_qkv_norm_rope_backward(dev, b, n, h, kv, dh, rows, p0, weights, odd):
    r = Rng(dev, 2000 + n + dh)
    qkv = r(b, n, (h + 2 * kv) * dh, odd=odd)
    wq, wk = (r(dh, std=0.2, mean=1.0, odd=odd), r(dh, std=0.2, mean=1.0)) if weights else (None, None)
    dq, dk, dv = r(b, n, h * dh, odd=odd), r(b, n, kv * dh), r(b, n, kv * dh, odd=odd)
    g = torch.cat([dq.view(b, n, h, dh), dk.view(b, n, kv, dh)], 2).to(F64)
    pos = (p0 + torch.arange(n, device=dev)).expand(b, n)
    g = turn(g, pos, 10000.0, -1.0)
    x = qkv.to(F64).view(b, n, h + 2 * kv, dh)[:, :, :h + kv]
    rr = 1.0 / torch.sqrt(x.square().mean(-1, keepdim=True) + 1e-4)
    w = torch.ones(h + kv, dh, dtype=F64, device=dev)
    if weights:
        w[:h], w[h:] = wq.to(F64), wk.to(F64)
    gw = g * w
    dx = rr * (gw - x * rr.square() * (gw * x).mean(-1, keepdim=True))
    # the terms of dx, each a dozen 32-bit roundings off, the mean dh / 8 + 5 more
    size = rr * (gw.abs() + x.abs() * rr.square() * (gw * x).abs().mean(-1, keepdim=True))
    pair = torch.repeat_interleave(size[..., 0::2] + size[..., 1::2], 2, -1)
    rows_ = b * n
    for accumulate in (False, True):
        dqkv = empty(dev, b, n, (h + 2 * kv) * dh, odd=odd)
        dwq, dwk = (empty(dev, dh), empty(dev, dh, odd=odd)) if weights else (None, None)
        evk.qkv_norm_rope_backward(qkv, dq, dk, dv, dqkv, dh, wq, wk, dwq, dwk, 1e-4, 10000.0, p0, accumulate)
        got = dqkv.view(b, n, h + 2 * kv, dh)
        close(got[:, :, :h + kv], dx, H * dx.abs() + 2.0 ** -19 * pair + T, "dqkv")
        assert torch.equal(got[:, :, h + kv:].reshape(b, n, -1), dv), "dv"
        if weights:
            term = g * x * rr
            big = torch.repeat_interleave((g * rr * x.abs()).abs()[..., 0::2] + (g * rr * x.abs()).abs()[..., 1::2], 2, -1)
            for got_w, sl, what in ((dwq, slice(0, h), "dq_weight"), (dwk, slice(h, h + kv), "dk_weight")):
                want = term[:, :, sl].sum((0, 1, 2)) + (7.0 if accumulate else 0.0)
                mag = big[:, :, sl].sum((0, 1, 2)) + 7.0
                close(got_w, want, H * want.abs() + (2.0 ** -19 + rows_ * E) * mag + T, what, norm=None)


def test_qkv_norm_rope_backward_differences(dev):
    """dqkv and the weights' gradients against differences of the forward's formula in 64 bits."""
    b, n, h, kv, dh = 1, 3, 2, 1, 8
    r = Rng(dev, 77)
    qkv, wq, wk = r(b, n, (h + 2 * kv) * dh), r(dh, mean=1.0, std=0.3), r(dh, mean=1.0, std=0.3)
    dq, dk, dv = r(b, n, h * dh), r(b, n, kv * dh), r(b, n, kv * dh)
    dqkv, dwq, dwk = torch.empty_like(qkv), torch.empty_like(wq), torch.empty_like(wk)
    evk.qkv_norm_rope_backward(qkv, dq, dk, dv, dqkv, dh, wq, wk, dwq, dwk)
    pos = torch.arange(n, device=dev).expand(b, n)

    def loss(x, a, c):
        y, v, _ = rope_want(x, a, c, h, kv, dh, pos, 1e-4, 10000.0)
        g = torch.cat([dq.view(b, n, h, dh), dk.view(b, n, kv, dh)], 2).to(F64)
        return float((y * g).sum() + (v * dv.view(b, n, kv, dh).to(F64)).sum())

    step = 1e-5
    args = [qkv.to(F64), wq.to(F64), wk.to(F64)]
    for which, got in enumerate((dqkv, dwq, dwk)):
        flat = args[which].reshape(-1)
        for i in range(flat.numel()):
            old = float(flat[i])
            flat[i] = old + step
            up = loss(*args)
            flat[i] = old - step
            down = loss(*args)
            flat[i] = old
            want = (up - down) / (2 * step)  # off by step^2 and 1e-16 / step times values of a few units
            assert abs(float(got.flatten()[i]) - want) <= H * abs(want) + 1e-4, (which, i)


# ---------------------------------------------------------------------------
# window_attention
# ---------------------------------------------------------------------------
def seen(p, rows, window, sinks):
    """(queries, rows) truth values for queries at the positions p."""
    j = torch.arange(rows, device=p.device)[None]
    p = p[:, None]
    s = j <= p
    if window:
        s &= (j > p - window) | (j < sinks)
    return s


def window_want(q, k, v, h, kv, dh, p0, window, sinks, do=None):
    """o, lse and (with do) gradients in 64 bits with their tolerances; p0: a position for each sequence.

    Rows that a query does not see take no part in its sums, whatever they hold."""
    b, n, _ = q.shape
    rows, grp, scale = k.shape[1], h // kv, dh ** -0.5
    out = {x: [] for x in ("o", "o_t", "lse", "lse_t", "dq", "dq_t")}
    dk, dv, dk_t, dv_t = (torch.zeros(b, rows, kv, dh, dtype=F64, device=q.device) for _ in range(4))
    for s in range(b):
        m = seen(p0[s] + torch.arange(n, device=q.device), rows, window, sinks)
        any_ = m.any(1)
        for hd in range(h):
            at, to = slice(hd * dh, hd * dh + dh), slice(hd // grp * dh, hd // grp * dh + dh)
            Q, K, V = q[s, :, at].to(F64), k[s, :, to].to(F64), v[s, :, to].to(F64)
            # what is hidden from every query does not count at all; what some see and hold NaN is dealt with
            # row by row (few such rows in a test)
            wild = ~(torch.isfinite(K).all(1) & torch.isfinite(V).all(1))
            K0, V0 = K.masked_fill(wild[:, None], 0.0), V.masked_fill(wild[:, None], 0.0)
            bad = (m & wild[None]).any(1)  # queries that do see such a row
            sc = (Q @ K0.t() * scale).masked_fill(~m, -math.inf)
            lse = torch.logsumexp(sc, 1)
            p = torch.where(m, torch.exp(sc - torch.where(any_, lse, torch.zeros_like(lse))[:, None]), torch.zeros_like(sc))
            o = p @ V0
            es = (dh + 4) * E * (Q.abs() @ K0.abs().t()) * scale  # error of a score
            es = es.masked_fill(~m, 0.0).amax(1, keepdim=True)
            rel = 2 * H + 4 * es + 2.0 ** -20  # the rounding of p and of o; exp of scores so far off; exp2 and the sum
            n_seen = m.sum(1, keepdim=True)
            vmax = V0.abs().amax(0, keepdim=True)
            o_t = rel * (p @ V0.abs()) + n_seen * (T + E) * vmax + T
            o[bad], lse[bad] = math.nan, math.nan
            out["o"].append(o)
            out["o_t"].append(o_t)
            out["lse"].append(lse)
            out["lse_t"].append((2 * es[:, 0] + (n_seen[:, 0] + 16) * E + 2.0 ** -21 * lse.abs().clamp(min=1.0)))
            if do is None:
                continue
            G = do[s, :, at].to(F64)
            o0 = p @ V0
            delta = (G * o0).sum(1, keepdim=True)
            # o is read rounded to fp16 and comes with its own error
            edelta = (G.abs() * (o_t + H * o0.abs())).sum(1, keepdim=True) + dh * E * (G.abs() * o0.abs()).sum(1, keepdim=True)
            dp = G @ V0.t()
            edp = (dh + 4) * E * (G.abs() @ V0.abs().t())
            ds = p * (dp - delta)
            # dS passes through fp16 (H, T); P is off by its score's error
            eds = (H + 4 * es + 2.0 ** -20) * ds.abs() + p * (edelta + edp) + T * m
            ep = (H + 4 * es + 2.0 ** -20) * p + T * m
            sums = 1.0 + n * grp * E
            out["dq"].append(scale * (ds @ K0))
            out["dq_t"].append(scale * (eds @ K0.abs()) * sums + H * (ds @ K0).abs() * scale + rows * E * scale * (ds.abs() @ K0.abs()) + T)
            c = hd // grp
            dk[s, :, c] += scale * (ds.t() @ Q)
            dk_t[s, :, c] += scale * (eds.t() @ Q.abs()) * sums + scale * n * grp * E * (ds.abs().t() @ Q.abs())
            dv[s, :, c] += p.t() @ G
            dv_t[s, :, c] += (ep.t() @ G.abs()) * sums + n * grp * E * (p.t() @ G.abs())
    got = {}
    for x in ("o", "o_t", "dq", "dq_t"):
        if out[x]:
            got[x] = torch.stack(out[x]).view(b, h, n, dh).transpose(1, 2).reshape(b, n, h * dh)
    for x in ("lse", "lse_t"):
        got[x] = torch.stack(out[x]).view(b, h, n)
    if do is not None:
        got.update(dk=dk.flatten(2), dv=dv.flatten(2), dk_t=(dk_t + H * dk.abs() + T).flatten(2), dv_t=(dv_t + H * dv.abs() + T).flatten(2))
    return got



WINDOW = [  # b, n, heads, kv, dh, rows, p0, window, sinks, odd
    (1, 1, 1, 1, 64, 1, 0, 0, 0, False), (2, 17, 4, 2, 64, 17, 0, 5, 0, False), (1, 130, 6, 2, 64, 130, 0, 33, 4, False),
    (1, 200, 3, 1, 128, 200, 0, 64, 1, False), (2, 65, 8, 8, 32, 65, 0, 16, 16, False), (1, 333, 4, 1, 128, 333, 0, 0, 0, False),
    (1, 100, 2, 2, 256, 100, 0, 40, 3, False), (2, 70, 5, 1, 80, 70, 0, 20, 2, False), (1, 96, 4, 4, 96, 96, 0, 31, 100, False),
    (1, 50, 2, 1, 33, 50, 0, 9, 1, True), (1, 64, 2, 1, 64, 64, 0, 7, 2, True), (3, 40, 4, 2, 64, 200, 90, 25, 4, False),
    (2, 129, 4, 2, 128, 300, 171, 64, 130, False), (1, 77, 12, 4, 64, 80, 3, 1, 0, False), (1, 300, 8, 2, 40, 300, 0, 128, 70, False),
    (1, 600, 2, 1, 64, 600, 0, 300, 300, False), (1, 64, 16, 1, 16, 64, 0, 10, 0, False), (4, 3, 8, 2, 128, 1000, 900, 256, 4, False),
    (1, 1100, 1, 1, 64, 1100, 0, 1024, 8, False), (1, 20, 7, 7, 100, 20, 0, 6, 1, True),
]


@pytest.mark.parametrize("b,n,h,kv,dh,rows,p0,window,sinks,odd", WINDOW)
def test_window_attention(dev, b, n, h, kv, dh, rows, p0, window, sinks, odd):
    r = Rng(dev, 3000 + n + dh)
    q, k, v = r(b, n, h * dh, odd=odd), r(b, rows, kv * dh, odd=odd), r(b, rows, kv * dh, odd=odd)
    # rows past the last query hold what a cache may hold
    k[:, p0 + n:], v[:, p0 + n:] = math.nan, math.inf
    o = empty(dev, b, n, h * dh, odd=odd)
    lse = torch.full((b, h, n), 7.0, device=dev)
    evk.window_attention(q, k, v, o, dh, window, sinks, p0, lse=lse)
    w = window_want(q, k, v, h, kv, dh, [p0] * b, window, sinks)
    close(o, w["o"], w["o_t"], "o")
    close(lse, w["lse"], w["lse_t"], "lse", norm=None)
    o2 = torch.empty_like(o)
    evk.window_attention(q, k, v, o2, dh, window, sinks, p0)
    assert torch.equal(o, o2), "without lse, or a second time"


DECODE = [  # b, heads, kv, dh, rows, window, sinks
    (1, 1, 1, 64, 1, 0, 0), (1, 12, 4, 64, 1056, 512, 4), (9, 32, 8, 128, 3000, 1024, 4), (3, 8, 1, 64, 700, 0, 0),
    (2, 3, 3, 80, 90, 33, 40), (5, 16, 2, 256, 400, 100, 1), (4, 6, 2, 33, 300, 50, 2), (70, 2, 2, 32, 129, 64, 0),
    (2, 24, 1, 128, 5000, 4096, 16), (1, 4, 2, 96, 2000, 0, 8),
]


@pytest.mark.parametrize("b,h,kv,dh,rows,window,sinks", DECODE)
@pytest.mark.parametrize("n", [1, 2])
def test_window_attention_ragged(dev, b, h, kv, dh, rows, window, sinks, n):
    """Every sequence at its own position: the first row, the last one, idle (nothing seen) and past the cache."""
    r = Rng(dev, 4000 + rows + dh)
    q, k, v = r(b, n, h * dh), r(b, rows, kv * dh), r(b, rows, kv * dh)
    off = torch.randint(0, rows, (b,), device=dev, generator=r.g, dtype=torch.int32)
    off[0] = rows - 1
    if b > 1:
        off[1] = 0
    if b > 2:
        off[2] = -n
    if b > 3:
        off[3] = rows + 7  # sees the rows that are there
    for s in range(b):
        k[s, max(0, int(off[s]) + n):], v[s, max(0, int(off[s]) + n):] = math.nan, math.nan
    o, lse = empty(dev, b, n, h * dh), torch.full((b, h, n), 7.0, device=dev)
    evk.window_attention(q, k, v, o, dh, window, sinks, 0, off, lse)
    w = window_want(q, k, v, h, kv, dh, off.tolist(), window, sinks)
    close(o, w["o"], w["o_t"], "o")
    close(lse, w["lse"], w["lse_t"], "lse", norm=None)
    if b > 2:
        assert (o[2] == 0).all() and (lse[2] == -math.inf).all()


@pytest.mark.parametrize("dh,h,kv", [(64, 4, 2), (128, 4, 1), (32, 2, 2), (256, 2, 1), (80, 3, 1), (33, 2, 1)])
def test_window_attention_wild_rows(dev, dh, h, kv):
    """NaN and infinities in rows that some queries see: those queries' outputs are NaN, the others' untouched."""
    b, n, window, sinks = 1, 150, 20, 2
    r = Rng(dev, 6)
    q, k, v = r(b, n, h * dh), r(b, n, kv * dh), r(b, n, kv * dh)
    v[0, 40], k[0, 90] = math.inf, math.nan
    v[0, 41, 0] = math.nan
    k[0, n - 1] = math.inf
    o, lse = empty(dev, b, n, h * dh), torch.empty(b, h, n, device=dev)
    evk.window_attention(q, k, v, o, dh, window, sinks, lse=lse)
    p = torch.arange(n, device=dev)
    hit = torch.zeros(n, dtype=torch.bool, device=dev)
    for j in (40, 41, 90, n - 1):
        hit |= seen(p, n, window, sinks)[:, j]
    w = window_want(q, k, v, h, kv, dh, [0], window, sinks)
    assert torch.isfinite(o[:, ~hit]).all(), "rows that the queries do not see reach their outputs"
    close(o[:, ~hit], w["o"][:, ~hit], w["o_t"][:, ~hit], "o")
    # columns of v that hold what is not finite are not finite in the queries that see it
    assert not torch.isfinite(o[0, 40:60].float()).any()
    assert not torch.isfinite(o[0, 90:110].float()).any()


def test_window_attention_large_scores(dev):
    """Scores of some hundreds, rising and falling along the rows: the running maximum moves at every step."""
    b, n, h, kv, dh = 1, 400, 4, 2, 64
    for sign in (1.0, -1.0):
        r = Rng(dev, 8)
        q = (1.0 + 0.01 * r(b, n, h * dh).float()).to(F16)
        ramp = torch.arange(n, device=dev, dtype=F32)[None, :, None] * 0.1 * sign
        k = (ramp * (1.0 + 0.01 * r(b, n, kv * dh).float())).to(F16)
        v = r(b, n, kv * dh)
        o, lse = torch.empty_like(q), torch.empty(b, h, n, device=dev)
        evk.window_attention(q, k, v, o, dh, 128, 4, lse=lse)
        w = window_want(q, k, v, h, kv, dh, [0], 128, 4)
        close(o, w["o"], w["o_t"], "o")
        close(lse, w["lse"], w["lse_t"], "lse", norm=None)


def window_grads(q, k, v, do, dh, h, window, sinks):
    b, n, _ = q.shape
    o, lse = torch.empty_like(q), torch.empty(b, h, n, device=q.device)
    evk.window_attention(q, k, v, o, dh, window, sinks, lse=lse)
    dq, dk, dv = (empty(q.device, *t.shape, odd=t.data_ptr() % 4 != 0) for t in (q, k, v))
    evk.window_attention_bwd(q, k, v, o, do, dq, dk, dv, lse, dh, window, sinks)
    return dq, dk, dv


@pytest.mark.parametrize("b,n,h,kv,dh,rows,p0,window,sinks,odd", [w for w in WINDOW if w[5] == w[1]])
def test_window_attention_bwd(dev, b, n, h, kv, dh, rows, p0, window, sinks, odd):
    r = Rng(dev, 5000 + n + dh)
    q, k, v, do = r(b, n, h * dh, odd=odd), r(b, n, kv * dh, odd=odd), r(b, n, kv * dh, odd=odd), r(b, n, h * dh, odd=odd)
    got = window_grads(q, k, v, do, dh, h, window, sinks)
    w = window_want(q, k, v, h, kv, dh, [0] * b, window, sinks, do)
    for g, x in zip(got, ("dq", "dk", "dv")):
        # one row that sees itself alone has dS = 0 up to roundings: no norm to hold it against
        close(g, w[x], w[x + "_t"], x, norm=4 * H if n > 16 and window != 1 else None)
    for g, x in zip(window_grads(q, k, v, do, dh, h, window, sinks), got):
        assert torch.equal(g, x), "a second time"


@pytest.mark.parametrize("dh,h,kv", [(64, 4, 2), (128, 4, 1), (32, 2, 2), (256, 2, 1), (80, 3, 1), (33, 2, 1)])
def test_window_attention_bwd_wild_rows(dev, dh, h, kv):
    """A padded batch: the last 30 positions hold NaN and infinities.  Gradients that no padded query or row takes part
    in are those of the sequence without them."""
    b, n, pad, window, sinks = 1, 170, 30, 20, 0
    r = Rng(dev, 9)
    q, k, v, do = r(b, n, h * dh), r(b, n, kv * dh), r(b, n, kv * dh), r(b, n, h * dh)
    m = n - pad
    short = [t[:, :m].contiguous() for t in (q, k, v, do)]
    q[:, m:], k[:, m:], v[:, m:], do[:, m:] = math.nan, math.inf, math.nan, math.inf
    dq, dk, dv = window_grads(q, k, v, do, dh, h, window, sinks)
    w = window_want(*short[:3], h, kv, dh, [0], window, sinks, short[3])
    close(dq[:, :m], w["dq"], w["dq_t"], "dq")
    far = m - window + 1  # rows before this one are seen by no padded query
    for g, x in ((dk, "dk"), (dv, "dv")):
        close(g[:, :far], w[x][:, :far], w[x + "_t"][:, :far], x)


def test_window_attention_bwd_differences(dev):
    b, n, h, kv, dh, window, sinks = 1, 9, 2, 1, 8, 3, 1
    r = Rng(dev, 11)
    q, k, v, do = r(b, n, h * dh), r(b, n, kv * dh), r(b, n, kv * dh), r(b, n, h * dh)
    got = window_grads(q, k, v, do, dh, h, window, sinks)
    args = [t.to(F64) for t in (q, k, v)]

    def loss():
        total = 0.0
        m = seen(torch.arange(n, device=dev), n, window, sinks)
        for hd in range(h):
            at = slice(hd * dh, hd * dh + dh)
            sc = (args[0][0, :, at] @ args[1][0].t() * dh ** -0.5).masked_fill(~m, -math.inf)
            total += float((torch.softmax(sc, 1) @ args[2][0] * do[0, :, at].to(F64)).sum())
        return total

    step = 1e-5
    for x, g in zip(args, got):
        flat = x.view(-1)
        for i in range(0, flat.numel(), 5):
            old = float(flat[i])
            flat[i] = old + step
            up = loss()
            flat[i] = old - step
            down = loss()
            flat[i] = old
            # dS and P of at most 4 terms of a few units pass through fp16: 16 H covers them
            assert abs(float(g.flatten()[i]) - (up - down) / (2 * step)) <= 16 * H * 4, i


# ---------------------------------------------------------------------------
# gated_linear
# ---------------------------------------------------------------------------
def act64(g, act):
    if act == "relu":
        return g.clamp(min=0), (g > 0).to(F64)
    if act == "silu":
        s = torch.sigmoid(g)
        return g * s, s * (1 + g * (1 - s))
    a = math.sqrt(2 / math.pi)
    t = torch.tanh(a * (g + 0.044715 * g ** 3))
    return 0.5 * g * (1 + t), 0.5 * (1 + t) + 0.5 * g * (1 - t * t) * a * (1 + 3 * 0.044715 * g * g)


GATED = [  # t, d, f, odd
    (1, 64, 128, False), (1, 768, 2048, False), (2, 136, 520, False), (3, 1, 1, False), (5, 33, 77, True), (16, 512, 1000, False),
    (17, 64, 64, False), (16, 1100, 264, True), (40, 129, 200, False), (64, 256, 512, False), (100, 72, 1048, False),
    (130, 300, 301, False), (257, 512, 1024, False), (600, 768, 2048, False), (1000, 520, 776, False), (2100, 256, 1288, False),
    (33, 2048, 96, False), (31, 7, 2000, False), (4, 4096, 1376, False), (9, 4096, 2752, False),
]


@pytest.mark.parametrize("t,d,f,odd", GATED)
@pytest.mark.parametrize("act", ["silu", "gelu", "relu"])
def test_gated_linear(dev, t, d, f, odd, act):
    r = Rng(dev, 7000 + t + f)
    x, w = r(t, d, odd=odd), r(2, d, f, std=1.5 / math.sqrt(d), odd=odd)
    X, W = x.to(F64), w.to(F64)
    g, u = X @ W[0], X @ W[1]
    a, da = act64(g, act)
    eg, eu = (d + 2) * E * (X.abs() @ W[0].abs()), (d + 2) * E * (X.abs() @ W[1].abs())
    want = a * u
    # the products' 32-bit sums, exp2, reciprocal and tanh to 2^-20, one rounding; |act'| <= 1.13
    tol = H * want.abs() + 1.2 * (eg * u.abs() + a.abs() * eu + eg * eu) + 2.0 ** -20 * (g * u).abs() + T
    h, gu = empty(dev, t, f, odd=odd), empty(dev, 2, t, f, odd=odd)
    evk.gated_linear(x, w, h, gu, act)
    close(h, want, tol, "h")
    close(gu[0], g, H * g.abs() + eg + T, "gate")
    close(gu[1], u, H * u.abs() + eu + T, "up")
    h2 = torch.empty_like(h)
    evk.gated_linear(x, w, h2, activation=act)
    # with and without gate_up may take different splits of the sums
    close(h2, want, tol, "h alone")
    evk.gated_linear(x, w, h, activation=act)
    assert torch.equal(h, h2), "a second time"


@pytest.mark.parametrize("t,d,f,odd", GATED)
@pytest.mark.parametrize("act", ["silu", "gelu", "relu"])
def test_gated_linear_backward(dev, t, d, f, odd, act):
    r = Rng(dev, 8000 + t + f)
    x, w = r(t, d, odd=odd), r(2, d, f, std=1.5 / math.sqrt(d), odd=odd)
    gu, dh = r(2, t, f, odd=odd), r(t, f, odd=odd)
    X, W, G = x.to(F64), w.to(F64), dh.to(F64)
    a, da = act64(gu[0].to(F64), act)
    dgu = torch.stack([G * gu[1].to(F64) * da, G * a])
    # fp16 roundings of both, after the fast functions' 2^-20 of terms of the size of 1 + |g|
    edgu = H * dgu.abs() + T + 2.0 ** -19 * torch.stack([(G * gu[1].to(F64)).abs(), G.abs()]) * (1 + gu[0].to(F64).abs())
    dx = dgu[0] @ W[0].t() + dgu[1] @ W[1].t()
    mag = dgu[0].abs() @ W[0].abs().t() + dgu[1].abs() @ W[1].abs().t()
    dx_t = edgu[0] @ W[0].abs().t() + edgu[1] @ W[1].abs().t() + (2 * f + 2) * E * mag + H * dx.abs() + T
    dw = torch.stack([X.t() @ dgu[0], X.t() @ dgu[1]])
    dw_t = torch.stack([X.abs().t() @ (edgu[i] + (t + 2) * E * dgu[i].abs()) for i in range(2)])
    for accumulate in (False, True):
        gx, gw = empty(dev, t, d, odd=odd), empty(dev, 2, d, f, odd=odd)
        evk.gated_linear_backward(x, w, gu, dh, gx, gw, act, accumulate)
        want = dw + (7.0 if accumulate else 0.0)
        close(gx, dx, dx_t, "dx")
        close(gw, want, dw_t + H * want.abs() + T, "dw")
    only = torch.empty_like(gx)
    evk.gated_linear_backward(x, w, gu, dh, dx=only, activation=act)
    assert torch.equal(only, gx)
    gw2 = torch.empty_like(gw)
    evk.gated_linear_backward(x, w, gu, dh, dw=gw2, activation=act)
    close(gw2, dw, dw_t + H * dw.abs() + T, "dw alone")


def test_gated_linear_wild_values(dev):
    """An infinite gate: silu passes it on above and ends at 0 below; a NaN stays in its row."""
    t, d, f = 20, 64, 128
    r = Rng(dev, 13)
    x, w = r(t, d), r(2, d, f, std=0.1)
    clean = torch.empty(t, f, dtype=F16, device=dev)
    evk.gated_linear(x, w, clean)
    x[7, 3] = math.nan
    h = torch.empty_like(clean)
    evk.gated_linear(x, w, h)
    rows = torch.arange(t, device=dev) != 7
    assert torch.isnan(h[7]).all() and torch.equal(h[rows], clean[rows])


def test_gated_linear_higher_ranks_and_empty(dev):
    r = Rng(dev, 14)
    x, w = r(2, 3, 64), r(2, 64, 72, std=0.1)
    h, gu = torch.empty(2, 3, 72, dtype=F16, device=dev), torch.empty(2, 2, 3, 72, dtype=F16, device=dev)
    evk.gated_linear(x, w, h, gu)
    flat, fgu = torch.empty(6, 72, dtype=F16, device=dev), torch.empty(2, 6, 72, dtype=F16, device=dev)
    evk.gated_linear(x.view(6, 64), w, flat, fgu)
    assert torch.equal(h.view(6, 72), flat) and torch.equal(gu.view(2, 6, 72), fgu)
    none = torch.empty(0, 64, dtype=F16, device=dev)
    evk.gated_linear(none, w, torch.empty(0, 72, dtype=F16, device=dev))
    dw = torch.full_like(w, 3.0)
    evk.gated_linear_backward(none, w, torch.empty(2, 0, 72, dtype=F16, device=dev), torch.empty(0, 72, dtype=F16, device=dev), none.clone(), dw,
                              accumulate=True)
    assert (dw == 3.0).all()
    evk.gated_linear_backward(none, w, torch.empty(2, 0, 72, dtype=F16, device=dev), torch.empty(0, 72, dtype=F16, device=dev), none.clone(), dw)
    assert (dw == 0.0).all()
