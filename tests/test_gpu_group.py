"""GPU: the operators of a group of continuations of one prompt (residual_norm,
prefix_attention, token_logprobs, the first and last with their gradients)
against plain 64-bit formulas.

Tolerances are worst cases of the roundings that the operators make: H = 2^-11
is half a step of fp16 relative to a value, T = 2^-25 half a step of its
subnormals, E = 2^-24 half a step of 32 bits.  Sums of n products in 32 bits are
off by at most n E times the sum of the products' magnitudes; a row's sums here
are at most 64 additions deep (16 values a thread, 6 steps of a wave, 16 waves),
a column's rows / 64 + 400.  The norm of a whole difference is at most 2 H of
the norm (close())."""
import math

import pytest
import torch

import evk_amd as evk
from test_gpu_block import E, F16, F32, F64, H, T, Rng, close, empty, window_want

pytestmark = pytest.mark.gpu

ROW = 128 * E  # of a norm: 64 additions, the square root, the products


# ---------------------------------------------------------------------------
# residual_norm
# ---------------------------------------------------------------------------
class Norms:
    """Inputs of residual_norm and its results in 64 bits."""

    def __init__(self, dev, seed, b, n, d, post=True, gate=None, weights=True, y=True, scale=1.0, eps=1e-4, odd=False, std=3.0):
        r = Rng(dev, seed)
        self.b, self.n, self.d, self.post, self.scale, self.eps, self.dev, self.odd = b, n, d, post and y, scale, eps, dev, odd
        self.x, self.y = r(b, n, d, std=std, odd=odd), r(b, n, d, odd=odd) if y else None
        self.wo = r(d, std=0.2, mean=1.0, odd=odd) if weights and post and y else None
        self.wi = r(d, std=0.2, mean=1.0) if weights else None
        self.gate = None
        if gate and y:
            self.gate = r(d, std=0.5, odd=odd) if gate == "channel" else r(b, d, std=0.5)
        self.ds, self.dh = r(b, n, d), r(b, n, d, odd=odd)

    def kw(self):
        return dict(residual_scale=self.scale, post_norm=self.post, eps=self.eps)

    def forward(self):
        s = None if self.y is None else empty(self.dev, self.b, self.n, self.d, odd=self.odd)
        h = empty(self.dev, self.b, self.n, self.d, odd=self.odd)
        evk.residual_norm(self.x, self.y, s, h, self.wo, self.gate, self.wi, **self.kw())
        return s, h

    def backward(self, ds=True, old=None, **more):
        e = lambda t, fill=7.0: None if t is None else torch.full_like(t, fill)  # noqa: E731
        g = dict(dx=empty(self.dev, self.b, self.n, self.d, odd=self.odd), dy=e(self.y), dwo=e(self.wo), dgate=e(self.gate), dwi=e(self.wi))
        if old is not None:
            for k in ("dwo", "dgate", "dwi"):
                if g[k] is not None:
                    g[k].copy_(old[k])
        evk.residual_norm_backward(self.x, self.y, self.ds if ds else None, self.dh, g["dx"], g["dy"], self.wo, self.gate, self.wi, g["dwo"],
                                   g["dgate"], g["dwi"], accumulate=old is not None, **self.kw(), **more)
        return g

    def leaves(self):
        return {k: getattr(self, k).to(F64).requires_grad_(True) for k in ("x", "y", "wo", "gate", "wi") if getattr(self, k) is not None}

    def formula(self, t):
        x, y = t["x"], t.get("y")
        norm = lambda v: v / torch.sqrt(v.square().mean(-1, keepdim=True) + self.eps)  # noqa: E731
        st = x
        if y is not None:
            y = norm(y) if self.post else y
            y = y * t["wo"] if "wo" in t else y
            if "gate" in t:
                y = y * (t["gate"] if t["gate"].dim() == 1 else t["gate"][:, None])
            st = self.scale * x + y
        h = norm(st)
        return st, h * t["wi"] if "wi" in t else h

    def want(self, ds=True):
        """Results, and the sizes of what was added on the way to each, both in 64 bits."""
        t = self.leaves()
        st, h = self.formula(t)
        grads = torch.autograd.grad([st, h], list(t.values()), [self.ds.to(F64) if ds else torch.zeros_like(st), self.dh.to(F64)])
        st, h = st.detach(), h.detach()
        t = {k: v.detach() for k, v in t.items()}
        size = {}
        x, y = t["x"], t.get("y")
        rms = lambda v: 1 / torch.sqrt(v.square().mean(-1, keepdim=True) + self.eps)  # noqa: E731
        gate = t.get("gate", torch.ones(self.d, dtype=F64, device=self.dev))
        gate = gate if gate.dim() == 1 else gate[:, None]
        wo, wi = (t.get(k, torch.ones(self.d, dtype=F64, device=self.dev)) for k in ("wo", "wi"))
        q = rms(y) if self.post else 1.0
        size["s"] = x.abs() if y is None else (self.scale * x).abs() + (y * q * wo * gate).abs()
        r = rms(st)
        size["h"] = size["s"] * r * wi.abs()
        # S = ds + r (c - u mean(c u)); an error of s reaches u and r
        c, u = (self.dh.to(F64) * wi).abs(), size["s"] * r
        size["S"] = (self.ds.to(F64).abs() if ds else 0.0) + r * (c + u * (c * u).mean(-1, keepdim=True)) * 2
        size["dx"] = size["S"] * abs(self.scale if y is not None else 1.0)
        size["dwi"] = (self.dh.to(F64).abs() * u).sum((0, 1))
        if y is not None:
            m = (y * q).abs()
            e = size["S"] * (gate * wo).abs()
            size["dy"] = q * (e + m * (e * m).mean(-1, keepdim=True)) * 2 if self.post else e
            size["dgate"] = (size["S"] * m * wo.abs()).sum((0, 1) if gate.dim() == 1 else 1)
            size["dwo"] = (size["S"] * m * gate.abs()).sum((0, 1))
        return dict(s=st, h=h, **{"d" + k: v for k, v in zip(t, grads)}), size

    def check(self, got, want, size, rows=None):
        for k, v in got.items():
            if v is None:
                continue
            sums = 0.0 if k in ("s", "h", "dx", "dy") else (self.b * self.n / 64 + 400) * E
            tol = H * want[k].abs() + T + (2 * ROW + sums) * size[k]
            close(v, want[k], tol, k)


NORM = [  # b, n, d, post, gate, weights, y, scale, odd
    (1, 1, 1, True, None, True, True, 1.0, False), (1, 1, 2, True, "channel", True, True, 0.5, True), (2, 3, 7, True, "sequence", True, True, -1.5, False),
    (1, 5, 8, False, None, True, True, 1.0, False), (3, 4, 31, True, "sequence", False, True, 1.0, True), (2, 17, 64, True, None, True, True, 0.0, False),
    (1, 33, 100, False, "channel", True, True, 0.7, True), (2, 9, 511, True, "channel", True, True, 1.0, True), (1, 6, 512, True, None, True, False, 1.0, False),
    (1, 6, 513, True, None, True, True, 1.0, False), (4, 130, 768, True, "sequence", True, True, 1.0, False), (16, 1, 768, True, None, True, True, 1.0, False),
    (1, 1000, 1001, True, "channel", True, True, 1.0, True), (2, 40, 1024, False, None, False, True, 1.0, False), (1, 7, 1025, True, None, True, False, 1.0, True),
    (2, 21, 2048, True, "sequence", True, True, 1.0, False), (1, 300, 2050, True, "channel", True, True, 2.0, False), (2, 700, 4096, True, "channel", True, True, 1.0, False),
    (1, 5, 5000, False, "sequence", True, True, 1.0, False), (3, 11, 8192, True, None, True, True, 1.0, False), (1, 4, 8200, True, "channel", True, True, 1.0, False),
    (1, 9, 16383, True, "sequence", True, True, 1.0, True), (2, 3, 16384, True, "channel", True, True, 1.0, False), (70, 1, 300, True, "sequence", True, True, 1.0, False),
]


@pytest.mark.parametrize("b,n,d,post,gate,weights,y,scale,odd", NORM)
def test_residual_norm(dev, b, n, d, post, gate, weights, y, scale, odd):
    c = Norms(dev, 100 + n + d, b, n, d, post, gate, weights, y, scale, odd=odd)
    s, h = c.forward()
    want, size = c.want()
    c.check(dict(s=s, h=h), want, size)


@pytest.mark.parametrize("b,n,d,post,gate,weights,y,scale,odd", NORM)
def test_residual_norm_backward(dev, b, n, d, post, gate, weights, y, scale, odd):
    c = Norms(dev, 200 + n + d, b, n, d, post, gate, weights, y, scale, odd=odd)
    want, size = c.want()
    got = c.backward()
    c.check(got, want, size)
    again = c.backward()
    for k, v in got.items():  # no order that changes from call to call
        assert v is None or torch.equal(v, again[k]), k


@pytest.mark.parametrize("d", [40, 768, 4096])
def test_residual_norm_backward_without_ds_and_accumulating(dev, d):
    c = Norms(dev, 7 + d, 3, 50, d, gate="sequence")
    want, size = c.want(ds=False)
    c.check(c.backward(ds=False), want, size)
    want, size = c.want()
    old = {k: torch.full_like(getattr(c, k[1:]), 0.5) for k in ("dwo", "dgate", "dwi")}
    got = c.backward(old=old)
    for k in old:
        want[k] = want[k] + 0.5
    c.check(got, want, size)


@pytest.mark.parametrize("which", ["dwo", "dgate", "dwi"])
def test_residual_norm_backward_one_weight(dev, which):
    """One weight's gradient alone, and none: the others are not touched and need not be there."""
    c = Norms(dev, 31, 2, 70, 256, gate="sequence")
    want, size = c.want()
    g = dict(dx=torch.empty_like(c.x), dy=torch.empty_like(c.y))
    one = {which: torch.empty_like(getattr(c, which[1:]))}
    names = dict(dwo="dpost_weight", dgate="dgate", dwi="dpre_weight")
    evk.residual_norm_backward(c.x, c.y, c.ds, c.dh, g["dx"], g["dy"], c.wo, c.gate, c.wi, **{names[which]: one[which]}, **c.kw())
    c.check({**g, **one}, want, size)
    evk.residual_norm_backward(c.x, c.y, c.ds, c.dh, g["dx"], g["dy"], c.wo, c.gate, c.wi, **c.kw())
    c.check(g, want, size)


def test_residual_norm_gradient_against_differences(dev):
    """The gradient along random directions against central differences of the formula in 64 bits: the results' roundings
    add up in quadrature, six of their steps."""
    c = Norms(dev, 41, 2, 30, 96, gate="sequence", scale=0.5)
    g = c.backward()
    t = {k: v.detach() for k, v in c.leaves().items()}
    for k in t:
        r = torch.randn(t[k].shape, dtype=F64, device=dev, generator=torch.Generator(device=dev).manual_seed(3))
        loss = []
        for sign in (1, -1):
            st, h = c.formula({**t, k: t[k] + sign * 1e-5 * r})
            loss.append((st * c.ds.to(F64)).sum() + (h * c.dh.to(F64)).sum())
        want = (loss[0] - loss[1]) / 2e-5
        got = (g["d" + k].to(F64) * r).sum()
        assert abs(got - want) <= 6 * H * float((g["d" + k].to(F64) * r).norm()) + 1e-6 * abs(loss[0]), k


def test_residual_norm_rows_apart(dev):
    """What a row holds stays in that row: infinities, NaN, rows of zeros with and without eps."""
    c = Norms(dev, 51, 2, 40, 300, gate="channel")
    s0, h0 = c.forward()
    c.x[0, 3], c.y[1, 5], c.y[0, 7, 11], c.x[1, 2] = math.inf, math.nan, -math.inf, 0.0
    c.y[1, 2] = 0.0
    s, h = c.forward()
    same = torch.ones(2, 40, dtype=torch.bool, device=dev)
    for at in ((0, 3), (1, 5), (0, 7), (1, 2)):
        same[at] = False
    assert torch.equal(s[same], s0[same]) and torch.equal(h[same], h0[same])
    assert torch.isnan(h[1, 5]).all() and torch.isnan(h[0, 3]).all()
    assert (s[1, 2] == 0).all() and (h[1, 2] == 0).all()
    g = c.backward()
    assert torch.isfinite(g["dx"][same]).all() and torch.isfinite(g["dy"][same]).all()


def test_residual_norm_large_values(dev):
    """Values near fp16's largest: squares and the stream before its rounding stay inside 32 bits."""
    c = Norms(dev, 52, 1, 8, 1000, gate="channel", scale=2.0)
    c.x.copy_(c.x.sign() * 60000)
    c.y.copy_(c.y.sign() * 65504)
    c.gate.mul_(1000)
    s, h = c.forward()
    want, size = c.want()
    ok = want["s"].abs() < 65504
    assert torch.isinf(s[want["s"].abs() > 65536]).all()
    assert ((s.to(F64) - want["s"]).abs() <= H * want["s"].abs() + 2 * ROW * size["s"])[ok].all()
    c.check(dict(h=h), want, size)


def test_residual_norm_nothing(dev):
    for b, n, d in ((0, 3, 64), (2, 0, 64), (2, 3, 0)):
        c = Norms(dev, 1, b, n, d, gate="sequence")
        c.forward()
        g = c.backward()
        for k in ("dwo", "dgate", "dwi"):
            assert (g[k] == 0).all(), (b, n, d, k)
        g = c.backward(old={k: torch.full_like(getattr(c, k[1:]), 2.0) for k in ("dwo", "dgate", "dwi")})
        for k in ("dwo", "dgate", "dwi"):
            assert (g[k] == 2).all()


# ---------------------------------------------------------------------------
# token_logprobs
# ---------------------------------------------------------------------------
def u16(t):
    return t.long() & 0xFFFF


def ids16(t):
    return torch.where(t > 32767, t - 65536, t).to(torch.int16)


def scores_want(logits, tokens, c, top):
    """Results in 64 bits; rows without a distribution are NaN."""
    x = logits.to(F64)
    t, v = u16(tokens), logits.shape[-1]
    m = x.amax(-1, keepdim=True)
    z = (x - m) * c
    L = torch.log(torch.exp(z).sum(-1))
    lp = z.gather(-1, t.clamp(max=v - 1)[:, None])[:, 0] - L
    p = torch.exp(z - L[:, None])
    ent = L - torch.where(p > 0, p * z, torch.where(torch.isnan(p), p, 0.0)).sum(-1)
    w = dict(lp=torch.where(t < v, lp, 0.0), ent=ent, p=p, logp=z - L[:, None], L=L, z=z)
    # how far |t| of a likely logit reaches: exp's argument is off by 2 E of it, the sums are 64 + 16 deep
    w["rel"] = (100 + 3 * torch.nan_to_num(ent + L, nan=0.0)) * E
    if top:
        key = torch.where(torch.isnan(x), torch.full_like(x, math.inf), x)
        order = torch.sort(key, dim=-1, descending=True, stable=True)[1]
        if torch.isnan(x).any():  # NaN above +inf
            first = torch.isnan(x).gather(-1, order).to(torch.int64)
            order = order.gather(-1, torch.sort(first, dim=-1, descending=True, stable=True)[1])
        w["ids"] = order[:, :top]
        w["alt"] = w["logp"].gather(-1, w["ids"])
    return w


def scores_check(dev, logits, tokens, c, top):
    rows = logits.shape[0]
    f = lambda *s: torch.full(s, 7.0, device=dev)  # noqa: E731
    lp, ent, stats = f(rows), f(rows), f(rows, 2)
    ids, alt = (torch.full((rows, top), 123, dtype=torch.int16, device=dev), f(rows, top)) if top else (None, None)
    evk.token_logprobs(logits, tokens, lp, ent, ids, alt, stats, input_scale=c)
    w = scores_want(logits, tokens, c, top)
    tol = lambda v: w["rel"].view(-1, *[1] * (v.dim() - 1)) + 4 * E * torch.nan_to_num(v, neginf=0.0).abs()  # noqa: E731
    close(lp, w["lp"], tol(w["lp"]), "logprobs", norm=None)
    close(ent, w["ent"], tol(w["ent"]) * (1 + w["ent"].nan_to_num(0.0)), "entropy", norm=None)
    if top:
        assert torch.equal(u16(ids), w["ids"])
        close(alt, w["alt"], tol(w["alt"]), "top_logprobs", norm=None)
    only = f(rows)
    evk.token_logprobs(logits, tokens, only, input_scale=c)  # nothing else asked for
    assert torch.equal(torch.nan_to_num(only, nan=5.0), torch.nan_to_num(lp, nan=5.0))
    return lp, ent, stats, w


def some_tokens(rows, v, dev, seed, pad=True):
    t = torch.randint(0, v, (rows,), device=dev, generator=torch.Generator(device=dev).manual_seed(seed))
    if pad and v < 65535 and rows > 2:
        t[rows // 2], t[-1] = 65535, v
    return ids16(t)


SCORES = [(1, 1, 1, 1.0), (5, 2, 2, 1.0), (3, 7, 7, 0.5), (4, 8, 0, 1.0), (9, 63, 5, 1.0), (9, 65, 32, 1.3), (16, 144, 5, 1.0), (33, 144, 20, 2.0),
          (7, 500, 32, 1.0), (5, 1000, 1, 1.0), (3, 1024, 32, 1.0), (3, 1025, 32, 1.0), (6, 4001, 8, 0.7), (2, 8192, 20, 1.0), (2, 8193, 20, 1.0),
          (3, 30001, 5, 1.0), (64, 32000, 8, 1.0), (2, 32768, 32, 1.0), (2, 32769, 32, 1.0), (3, 50257, 10, 1.0), (2, 65535, 5, 1.0), (5, 65536, 32, 1.0)]


@pytest.mark.parametrize("rows,v,top,c", SCORES)
@pytest.mark.parametrize("odd", [False, True])
def test_token_logprobs(dev, rows, v, top, c, odd):
    r = Rng(dev, 300 + v)
    scores_check(dev, r(rows, v, std=3.0, odd=odd), some_tokens(rows, v, dev, v), c, top)


@pytest.mark.parametrize("v", [9, 144, 1024, 2000, 32000, 65536])
def test_token_logprobs_ties(dev, v):
    """Equal logits: the lowest ids, however many there are; zeros of both signs are equal."""
    r = Rng(dev, 310 + v)
    top = min(v, 32)
    x = torch.stack([r(v, std=0.2).float().round().half(), torch.full((v,), -3.0, dtype=F16, device=dev), r(v).sign() * 0.0,
                     (r(v) > 1.0).half(), torch.full((v,), 65504.0, dtype=F16, device=dev), torch.full((v,), -65504.0, dtype=F16, device=dev),
                     torch.arange(v, device=dev).mul(-1).clamp(min=-2000).half()])
    scores_check(dev, x.contiguous(), some_tokens(len(x), v, dev, 5), 1.0, top)


@pytest.mark.parametrize("v", [9, 144, 1025, 32000, 65536])
def test_token_logprobs_masks(dev, v):
    """-inf among the logits, all but one, all; +inf and NaN; the type's lowest value."""
    r = Rng(dev, 320 + v)
    x = r(9, v, std=2.0)
    x[0, : v // 2] = -math.inf
    x[1, 1:] = -math.inf
    x[2] = -math.inf
    x[3, v // 3] = math.inf
    x[4, v - 1] = math.nan
    x[5, 2:] = -65504.0
    x[6, :-3] = -math.inf
    x[7, 3], x[7, 4], x[7, 5] = math.nan, math.inf, math.nan
    lp, ent, stats, w = scores_check(dev, x, some_tokens(9, v, dev, 7, pad=False), 1.0, min(v, 9))
    assert torch.isnan(lp[[2, 3, 4, 7]]).all() and torch.isnan(ent[[2, 3, 4, 7]]).all()
    assert ent[1] == 0


def test_token_logprobs_large_logits(dev):
    """Logits of tens of thousands, scaled: differences keep their bits."""
    r = Rng(dev, 330)
    x = (r(6, 3000, std=0.001).float() + 60000).half()
    x[:, ::7] = 59968.0
    x[:, 5] = -60000.0
    for c in (1.0, 0.01, 0.0321, 3.7, 1000.0, 2.0 ** -20):
        scores_check(dev, x, some_tokens(6, 3000, dev, 9), c, 5)


def grad_check(dev, logits, tokens, c, dlp, dent, odd=False):
    rows, v = logits.shape
    lp, ent, stats = (torch.empty(rows, device=dev), torch.empty(rows, device=dev), torch.empty(rows, 2, device=dev))
    evk.token_logprobs(logits, tokens, lp, ent, stats=stats, input_scale=c)
    d = empty(dev, rows, v, odd=odd)
    evk.token_logprobs_backward(logits, tokens, stats, dlp, d, ent if dent is not None else None, dent, input_scale=c)
    w = scores_want(logits, tokens, c, 0)
    t = u16(tokens)
    wt = torch.where(t < v, dlp.to(F64) if dlp is not None else torch.zeros(rows, dtype=F64, device=dev), 0.0)[:, None]
    he = (dent.to(F64) if dent is not None else torch.zeros(rows, dtype=F64, device=dev))[:, None]
    p, logp, H_ = w["p"], w["logp"], w["ent"][:, None]
    hot = torch.zeros(rows, v, dtype=F64, device=dev).scatter_(1, t.clamp(max=v - 1)[:, None], 1.0)
    inner = torch.where(p > 0, logp, torch.where(torch.isnan(p), p, 0.0)) + H_
    want = c * (wt * (hot - p) - torch.where(he != 0, he * p * inner, 0.0))
    # p is off by the error of its exponent (3 E of the difference) and of L
    rel = (3 * w["z"].nan_to_num(0.0, neginf=0.0).abs() * E + w["rel"][:, None]) * 2
    mag = wt.abs() * (hot * 2.0 ** -20 + p * rel) + he.abs() * p * (rel * (inner.abs() + 1) + w["rel"][:, None] * (1 + H_) + 8 * E * (logp.nan_to_num(0.0, neginf=0.0).abs() + H_))
    idle = (wt[:, 0] == 0) & (he[:, 0] == 0)
    want[idle], mag[idle] = 0.0, 0.0
    close(d, want, H * want.abs() + T + c * mag.nan_to_num(0.0), "dlogits")
    return d, idle


@pytest.mark.parametrize("rows,v,top,c", SCORES)
@pytest.mark.parametrize("which", ["both", "logprobs", "entropy"])
def test_token_logprobs_backward(dev, rows, v, top, c, which):
    r = Rng(dev, 340 + v)
    logits, tokens = r(rows, v, std=3.0, odd=rows % 2 == 1), some_tokens(rows, v, dev, v)
    dlp, dent = r(rows, std=20.0).float(), r(rows, std=5.0).float()
    grad_check(dev, logits, tokens, c, dlp if which != "entropy" else None, dent if which != "logprobs" else None, odd=rows % 2 == 0)


def test_token_logprobs_backward_masks(dev):
    """No gradient to what cannot be sampled, zeros for rows that nothing is asked of, whatever they hold."""
    v, rows = 1000, 10
    r = Rng(dev, 350)
    x = r(rows, v, std=2.0)
    x[:, 100:300] = -math.inf
    tokens = some_tokens(rows, v, dev, 3, pad=False)
    tokens.copy_(torch.where((u16(tokens) >= 100) & (u16(tokens) < 300), 5, u16(tokens)).to(torch.int16))
    dlp, dent = r(rows).float() + 3.0, r(rows).float() + 3.0
    x[1], x[2, 7], x[3] = math.nan, math.inf, -math.inf
    dlp[1:5], dent[1:5] = 0.0, 0.0
    tokens[5], dent[5] = -1, 0.0  # no token: its dlogprob does not count
    d, idle = grad_check(dev, x, tokens, 1.0, dlp, dent)
    assert idle[1:6].all() and (d[1:6] == 0).all() and (d[6:, 100:300] == 0).all() and (d[0, 100:300] == 0).all()
    x[6, 3] = math.nan  # and a row without a distribution that something is asked of
    lp, ent, stats = torch.empty(rows, device=dev), torch.empty(rows, device=dev), torch.empty(rows, 2, device=dev)
    evk.token_logprobs(x, tokens, lp, ent, stats=stats)
    evk.token_logprobs_backward(x, tokens, stats, dlp, d, ent, dent)
    assert torch.isnan(d[6]).all() and torch.isfinite(d[[0, 1, 2, 3, 4, 5, 7, 8, 9]]).all()


def test_token_logprobs_gradient_against_differences(dev):
    """Along random directions, against central differences of the 64-bit formulas."""
    rows, v, c = 12, 300, 0.8
    r = Rng(dev, 360)
    x, tokens = r(rows, v, std=2.0), some_tokens(rows, v, dev, 2, pad=False)
    dlp, dent = r(rows, std=100.0).float(), r(rows, std=30.0).float()
    d, _ = grad_check(dev, x, tokens, c, dlp, dent)
    u = torch.randn(rows, v, dtype=F64, device=dev, generator=torch.Generator(device=dev).manual_seed(3))
    loss = []
    for sign in (1, -1):
        lp = torch.log_softmax((x.to(F64) + sign * 1e-5 * u) * c, -1)
        loss.append((lp.gather(1, u16(tokens)[:, None])[:, 0] * dlp).sum() - ((lp.exp() * lp).sum(1) * dent).sum())
    want, got = (loss[0] - loss[1]) / 2e-5, (d.to(F64) * u).sum()
    assert abs(got - want) <= 6 * H * float((d.to(F64) * u).norm()) + 1e-6 * abs(loss[0])


def test_token_logprobs_no_rows(dev):
    f = lambda *s: torch.zeros(*s, device=dev)  # noqa: E731
    x, t = torch.empty(0, 50, dtype=F16, device=dev), torch.empty(0, dtype=torch.int16, device=dev)
    evk.token_logprobs(x, t, f(0), f(0), torch.empty(0, 3, dtype=torch.int16, device=dev), f(0, 3), f(0, 2))
    evk.token_logprobs_backward(x, t, f(0, 2), f(0), torch.empty_like(x), f(0), f(0))


# ---------------------------------------------------------------------------
# prefix_attention
# ---------------------------------------------------------------------------
def prefix_want(q, pk, pv, k, v, h, kv, dh, first):
    """o and lse in 64 bits with their tolerances: attention over the rows of the prefix with each sequence's own behind
    them; `first` the own row of each sequence's first query."""
    got = {x: [] for x in ("o", "o_t", "lse", "lse_t")}
    n, p = q.shape[1], pk.shape[0]
    for s in range(q.shape[0]):
        end = max(0, min(first[s] + n, k.shape[1]))
        kk, vv = torch.cat([pk, k[s, :end]])[None], torch.cat([pv, v[s, :end]])[None]
        if kk.shape[1] == 0:
            z = torch.zeros(1, n, h * dh, dtype=F64, device=q.device)
            w = dict(o=z, o_t=z, lse=torch.full((1, h, n), -math.inf, dtype=F64, device=q.device), lse_t=torch.zeros(1, h, n, dtype=F64, device=q.device))
        else:
            # below its own rows a query sees the whole prefix: no position of window_want's, so those are done alone
            below = min(n, max(0, -first[s]))
            parts = []
            if below:
                parts.append(window_want(q[s:s + 1, :below].reshape(1, below, -1), pk[None], pv[None], h, kv, dh, [p - 1], 0, 0) if p and below == 1 else None)
                if parts[-1] is None:
                    one = [window_want(q[s:s + 1, i:i + 1], pk[None], pv[None], h, kv, dh, [p - 1], 0, 0) if p else
                           dict(o=torch.zeros(1, 1, h * dh, dtype=F64, device=q.device), o_t=torch.zeros(1, 1, h * dh, dtype=F64, device=q.device),
                                lse=torch.full((1, h, 1), -math.inf, dtype=F64, device=q.device), lse_t=torch.zeros(1, h, 1, dtype=F64, device=q.device))
                           for i in range(below)]
                    parts[-1] = {x: torch.cat([w[x] for w in one], 1 if x[0] == "o" else 2) for x in got}
            if below < n:
                parts.append(window_want(q[s:s + 1, below:], kk, vv, h, kv, dh, [p + max(0, first[s])], 0, 0))
            w = {x: torch.cat([u[x] for u in parts], 1 if x[0] == "o" else 2) for x in got}
        for x in got:
            got[x].append(w[x])
    return {x: torch.cat(y) for x, y in got.items()}


def prefix_check(dev, q, pk, pv, k, v, h, kv, dh, offsets=None, p0=0, odd=False):
    o = empty(dev, *q.shape, odd=odd)
    lse = torch.full((q.shape[0], h, q.shape[1]), 7.0, device=dev)
    off = None if offsets is None else torch.tensor(offsets, dtype=torch.int32, device=dev)
    evk.prefix_attention(q, pk, pv, k, v, o, dh, p0, off, lse)
    w = prefix_want(q, pk, pv, k, v, h, kv, dh, offsets or [p0] * q.shape[0])
    close(o, w["o"], w["o_t"], "o")
    close(lse, w["lse"], w["lse_t"], "lse", norm=None)
    o2 = torch.empty_like(o)
    evk.prefix_attention(q, pk, pv, k, v, o2, dh, p0, off)
    assert torch.equal(o.nan_to_num(7.0), o2.nan_to_num(7.0))
    return o


PREFIX = [  # b, n, heads, kv, dh, prefix, rows, odd
    (1, 1, 1, 1, 2, 1, 1, False), (2, 1, 4, 2, 64, 3, 5, False), (3, 1, 12, 4, 64, 100, 33, False), (1, 1, 8, 1, 128, 1, 200, False),
    (16, 1, 1, 1, 256, 64, 160, False), (5, 1, 6, 2, 80, 77, 40, True), (4, 1, 4, 2, 34, 129, 10, False), (2, 1, 32, 8, 128, 1000, 300, False),
    (64, 1, 8, 2, 64, 500, 64, False), (40, 1, 12, 4, 96, 257, 100, False), (3, 1, 5, 5, 32, 2049, 7, False), (2, 5, 12, 4, 64, 301, 60, False),
    (8, 3, 4, 1, 128, 63, 20, False), (2, 17, 8, 2, 40, 65, 64, False), (1, 64, 2, 1, 256, 31, 64, False), (3, 100, 4, 2, 64, 128, 100, False),
    (2, 130, 8, 8, 128, 200, 140, False), (1, 300, 16, 4, 64, 1, 300, False), (2, 33, 3, 1, 100, 50, 40, True), (1, 1, 7, 7, 48, 0, 20, False),
    (2, 20, 4, 2, 64, 0, 30, False), (200, 1, 2, 1, 64, 90, 12, False), (2, 1, 64, 1, 64, 700, 90, False), (300, 2, 4, 2, 32, 33, 8, False),
]


@pytest.mark.parametrize("b,n,h,kv,dh,p,rows,odd", PREFIX)
def test_prefix_attention(dev, b, n, h, kv, dh, p, rows, odd):
    r = Rng(dev, 400 + p + dh)
    q, pk, pv = r(b, n, h * dh, odd=odd), r(p, kv * dh), r(p, kv * dh, odd=odd)
    k, v = r(b, rows, kv * dh), r(b, rows, kv * dh, odd=odd)
    prefix_check(dev, q, pk, pv, k, v, h, kv, dh, odd=odd)
    prefix_check(dev, q, pk, pv, k, v, h, kv, dh, p0=rows - n, odd=odd)
    g = torch.Generator().manual_seed(p)
    off = torch.randint(0, rows - n + 1, (b,), generator=g).tolist()
    for s in range(b):  # rows past each sequence's end hold anything
        k[s, off[s] + n:], v[s, off[s] + n:] = math.nan, math.inf
    prefix_check(dev, q, pk, pv, k, v, h, kv, dh, off, odd=odd)


@pytest.mark.parametrize("dh,h,kv,n", [(64, 8, 2, 1), (64, 8, 2, 7), (128, 4, 1, 40), (256, 2, 1, 9), (40, 6, 3, 1), (36, 2, 1, 5), (64, 4, 2, 150)])
@pytest.mark.parametrize("p", [0, 1, 64, 200])
def test_prefix_attention_offsets(dev, dh, h, kv, n, p):
    """Sequences before their own rows, at their first and last, and past them."""
    rows = n + 30
    off = [0, -1, -n, -n + 1, -1000, 30, 31, rows, 5, -2 ** 31, 2 ** 31 - 1]
    b = len(off)
    r = Rng(dev, 500 + p + dh)
    q, pk, pv = r(b, n, h * dh), r(p, kv * dh), r(p, kv * dh)
    k, v = r(b, rows, kv * dh), r(b, rows, kv * dh)
    prefix_check(dev, q, pk, pv, k, v, h, kv, dh, off)


@pytest.mark.parametrize("dh,h,kv,n", [(64, 4, 2, 1), (64, 4, 2, 6), (128, 8, 2, 40), (256, 1, 1, 20), (36, 2, 1, 5), (64, 4, 2, 200)])
def test_prefix_attention_values_apart(dev, dh, h, kv, n):
    """Own rows that hold NaN or infinities reach the queries that see them and no other; the prefix reaches all."""
    b, p, rows = 3, 70, n + 20
    r = Rng(dev, 520 + dh)
    q, pk, pv = r(b, n, h * dh), r(p, kv * dh), r(p, kv * dh)
    k, v = r(b, rows, kv * dh), r(b, rows, kv * dh)
    off = [3, 0, 11]
    k[0, 3 + n // 2], v[1, n - 1, 3], v[2, 11 + n // 2] = math.nan, math.inf, math.nan
    o = empty(dev, b, n, h * dh)
    evk.prefix_attention(q, pk, pv, k, v, o, dh, offsets=torch.tensor(off, dtype=torch.int32, device=dev))
    clean_k, clean_v = k.nan_to_num(0.0, posinf=0.0), v.nan_to_num(0.0, posinf=0.0)
    w = prefix_want(q, pk, pv, clean_k, clean_v, h, kv, dh, off)
    t = torch.arange(n, device=dev)
    hit = torch.zeros(b, n, h, dh, dtype=torch.bool, device=dev)
    hit[0, t >= n // 2] = True
    hit[2, t >= n // 2] = True
    hit[1, n - 1, : h // kv, 3] = True
    hit = hit.view(b, n, h * dh)
    assert (~torch.isfinite(o[hit])).all() and torch.isfinite(o[~hit]).all()
    assert ((o.to(F64) - w["o"]).abs() <= w["o_t"])[~hit].all()
    pv[5, 2] = math.inf
    evk.prefix_attention(q, pk, pv, clean_k, clean_v, o, dh, offsets=torch.tensor(off, dtype=torch.int32, device=dev))
    reach = torch.zeros(b, n, h, dh, dtype=torch.bool, device=dev)
    reach[:, :, : h // kv, 2] = True
    assert torch.equal(~torch.isfinite(o), reach.view(b, n, h * dh))


@pytest.mark.parametrize("dh,n", [(64, 1), (128, 70), (36, 3)])
def test_prefix_attention_scores_without_a_softmax(dev, dh, n):
    """Scores that are all -inf, in the prefix alone and everywhere."""
    r = Rng(dev, 530)
    q, p, rows = torch.full((2, n, dh), 1.0, dtype=F16, device=dev), 40, n + 5
    pk, k = torch.full((p, dh), -math.inf, dtype=F16, device=dev), r(2, rows, dh)
    pv, v = r(p, dh), r(2, rows, dh)
    k[1] = -math.inf
    o, lse = empty(dev, 2, n, dh), torch.zeros(2, 1, n, device=dev)
    evk.prefix_attention(q, pk, pv, k, v, o, dh, lse=lse)
    w = prefix_want(q[:1], pk[:0], pv[:0], k[:1], v[:1], 1, 1, dh, [0])
    assert ((o[:1].to(F64) - w["o"]).abs() <= w["o_t"]).all()
    assert torch.isnan(o[1]).all() and (lse[1] == -math.inf).all()


@pytest.mark.parametrize("dh,h,kv,n,p", [(128, 8, 2, 1, 3000), (64, 4, 1, 5, 500), (256, 2, 2, 1, 1000), (64, 2, 1, 300, 700)])
def test_prefix_attention_large_scores(dev, dh, h, kv, n, p):
    """Scores of thousands, the largest anywhere in the list: one row takes all."""
    r = Rng(dev, 540 + dh)
    b, rows = 3, n + 40
    q, pk, pv = r(b, n, h * dh, std=30.0), r(p, kv * dh, std=30.0), r(p, kv * dh)
    k, v = r(b, rows, kv * dh, std=30.0), r(b, rows, kv * dh)
    prefix_check(dev, q, pk, pv, k, v, h, kv, dh, [0, 40, 17])


@pytest.mark.parametrize("b,n,h,kv,dh,p,rows", [(64, 1, 32, 8, 128, 2000, 300), (4, 400, 16, 4, 128, 1000, 400), (16, 1, 8, 1, 64, 9000, 100),
                                                (1, 1, 8, 2, 128, 40000, 10), (2, 1, 4, 2, 64, 20, 30000), (3, 600, 8, 2, 64, 333, 700), (2, 300, 4, 2, 256, 400, 300)])
def test_prefix_attention_many_rows(dev, b, n, h, kv, dh, p, rows):
    r = Rng(dev, 550 + p)
    q, pk, pv = r(b, n, h * dh), r(p, kv * dh), r(p, kv * dh)
    k, v = r(b, rows, kv * dh), r(b, rows, kv * dh)
    g = torch.Generator().manual_seed(p)
    prefix_check(dev, q, pk, pv, k, v, h, kv, dh, torch.randint(0, rows - n + 1, (b,), generator=g).tolist())


def test_prefix_attention_is_window_attention_over_both(dev):
    """The same rows in one cache a sequence: both operators sum in orders of their own, a rounding of P and of the result each."""
    b, n, h, kv, dh, p, rows = 3, 4, 8, 2, 64, 150, 50
    r = Rng(dev, 560)
    q, pk, pv, k, v = r(b, n, h * dh), r(p, kv * dh), r(p, kv * dh), r(b, rows, kv * dh), r(b, rows, kv * dh)
    o, o2 = torch.empty_like(q), torch.empty_like(q)
    evk.prefix_attention(q, pk, pv, k, v, o, dh, 20)
    evk.window_attention(q, torch.cat([pk.expand(b, -1, -1), k], 1), torch.cat([pv.expand(b, -1, -1), v], 1), o2, dh, position_offset=p + 20)
    assert float((o.double() - o2.double()).norm() / o2.double().norm()) <= 4 * H


def test_qkv_norm_rope_behind_a_prefix(dev):
    """Row p of the cache takes the token at position first + p: the rows of a longer cache, moved down."""
    b, n, h, kv, dh, rows, first = 2, 7, 4, 2, 64, 30, 100
    r = Rng(dev, 570)
    x, wq, wk = r(b, n, (h + 2 * kv) * dh), r(dh, mean=1.0), r(dh, mean=1.0)
    q, k, v = empty(dev, b, n, h * dh), empty(dev, b, rows, kv * dh), empty(dev, b, rows, kv * dh)
    q2, k2, v2 = empty(dev, b, n, h * dh), empty(dev, b, first + rows, kv * dh), empty(dev, b, first + rows, kv * dh)
    for off in (None, torch.tensor([5, 23], dtype=torch.int32, device=dev)):
        evk.qkv_norm_rope(x, q, k, v, dh, wq, wk, position_offset=0 if off is not None else 9, offsets=off, first_position=first)
        evk.qkv_norm_rope(x, q2, k2, v2, dh, wq, wk, position_offset=0 if off is not None else first + 9, offsets=None if off is None else off + first)
        assert torch.equal(q, q2) and torch.equal(k, k2[:, first:]) and torch.equal(v, v2[:, first:])
