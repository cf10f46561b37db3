"""Cases of the operators of a grouped-query transformer block: norms and
rotation of queries and keys with the cache rows in the same pass, attention
over a sliding window and the first tokens, and the gated linear unit of the
feed-forward block, each for prompts, for single tokens and, where training
uses it, with its backward pass.

  listed()            the named cases
  draw(rng)           one more case of the same ranges
  prepare(case, seed) inputs, outputs and caches on the GPU
  run(state)          one pass: torch operations in 32 bits, or with `own` the
                      calls of evk_amd
  exact(case, seed)   the same outputs in 64 bits
  work(case)          bytes and flops that the pass cannot do without

All tensors are fp16 unless said otherwise.  Heads are grouped: `heads` query
heads share `kv` key and value heads of `dh` values.  Query t of a sequence
that starts at position p0 stands at p = p0 + t and sees the cache rows j <= p
with j > p - window or j < sinks (window 0: every row up to p).
"""
import math

import torch

own = False

F16, F32, F64 = torch.float16, torch.float32, torch.float64
EPS, BASE = 1e-4, 10000.0


def listed():
    return [
        # one token of each of 16 sequences decoded together, rows into their caches: the smallest call
        dict(name="rope_decode", kind="rope", b=16, n=1, heads=12, kv=4, dh=64, rows=1056, ragged=True, weights=True),
        # the queries, keys and values of a long prompt
        dict(name="rope_prompt", kind="rope", b=1, n=8192, heads=32, kv=8, dh=128, rows=8192, ragged=False, weights=True),
        # a training batch, forward and backward, a length that is no multiple of anything
        dict(name="rope_train", kind="rope_train", b=4, n=1999, heads=12, kv=4, dh=64),
        # one token behind a short context: latency
        dict(name="window_decode_one", kind="window", b=1, n=1, heads=12, kv=4, dh=64, rows=1056, p0=1055, ragged=False, window=512, sinks=4),
        # one token of each of 64 sequences at positions of their own: bandwidth
        dict(name="window_decode_batch", kind="window", b=64, n=1, heads=32, kv=8, dh=128, rows=8192, p0=0, ragged=True, window=1024, sinks=4),
        # a long prompt
        dict(name="window_prompt", kind="window", b=1, n=8192, heads=16, kv=4, dh=128, rows=8192, p0=0, ragged=False, window=1024, sinks=4),
        # training, forward and backward, a ragged length
        dict(name="window_train", kind="window_train", b=2, n=1999, heads=8, kv=2, dh=128, window=512, sinks=4),
        # the shape of the reference's training program: one head of 256 over 160 positions
        dict(name="window_train_d256", kind="window_train", b=16, n=160, heads=1, kv=1, dh=256, window=64, sinks=2),
        # one token through a small layer: latency
        dict(name="gated_one", kind="gated", t=1, d=768, h=2048, act="silu"),
        # one token of each of 16 sequences through a large layer: bandwidth
        dict(name="gated_decode_batch", kind="gated", t=16, d=4096, h=11008, act="silu"),
        # a long prompt through the large layer: the largest product
        dict(name="gated_prompt", kind="gated", t=6001, d=4096, h=11008, act="silu"),
        # training, forward and backward
        dict(name="gated_train", kind="gated_train", t=2560, d=768, h=2048, act="gelu"),
    ]


def _log(rng, lo, hi, step=1):
    """A size from lo to hi, spread over its logarithm, a multiple of step."""
    v = math.exp(rng.uniform(math.log(lo), math.log(hi)))
    return max(lo, min(hi, int(round(v / step)) * step))


def _heads(rng):
    dh = rng.choice([32, 64, 64, 80, 96, 128, 128, 256])
    kv = rng.choice([1, 2, 4, 8]) if dh < 256 else rng.choice([1, 2])
    return dict(heads=kv * rng.choice([1, 2, 3, 4, 8]), kv=kv, dh=dh)


def draw(rng):
    kind = rng.choice(["rope", "rope_one", "rope_train", "window", "window_one", "window_one", "window_train", "gated", "gated_one", "gated_odd",
                       "gated_train"])
    if kind in ("rope", "rope_one", "rope_train"):
        while True:
            g = _heads(rng)
            b = _log(rng, 1, 64) if kind == "rope_one" else _log(rng, 1, 8)
            n = 1 if kind == "rope_one" else _log(rng, 2, 8192)
            rows = n + rng.randrange(0, 1500)
            width = (g["heads"] + 2 * g["kv"]) * g["dh"]
            if b * n * width <= (48 << 20) and b * rows * g["kv"] * g["dh"] <= (48 << 20):
                if kind == "rope_train":
                    return dict(kind=kind, b=b, n=n, **g)
                return dict(kind="rope", b=b, n=n, **g, rows=rows, ragged=kind == "rope_one", weights=rng.random() < 0.8)
    if kind in ("window", "window_one", "window_train"):
        while True:
            g = _heads(rng)
            window, sinks = rng.choice([0, 1, 1, 1]) * _log(rng, 16, 4096), rng.choice([0, 1, 4, 4, 16, 100])
            if kind == "window_one":
                b, rows = _log(rng, 1, 64), _log(rng, 33, 8192)
                if b * rows * g["kv"] * g["dh"] > (512 << 20):
                    continue
                p0 = 0 if rng.random() < 0.7 else rows - 1
                return dict(kind="window", b=b, n=1, **g, rows=rows, p0=p0, ragged=p0 == 0, window=window, sinks=sinks)
            b, n = _log(rng, 1, 16), _log(rng, 17, 4096)
            p0 = rng.choice([0, 0, rng.randrange(0, 2000)]) if kind == "window" else 0
            if b * g["heads"] * n * (n + p0) > 2.6e8:
                continue
            if kind == "window_train":
                return dict(kind=kind, b=b, n=n, **g, window=window, sinks=sinks)
            return dict(kind=kind, b=b, n=n, **g, rows=n + p0 + rng.randrange(0, 64), p0=p0, ragged=False, window=window, sinks=sinks)
    act = rng.choice(["silu", "silu", "gelu", "relu"])
    if kind == "gated_one":
        return dict(kind="gated", t=_log(rng, 1, 40), d=_log(rng, 128, 4096, 8), h=_log(rng, 256, 11008, 8), act=act)
    while True:
        odd = kind == "gated_odd"
        t = _log(rng, 2, 2000) if odd else _log(rng, 41, 6000)
        d, h = (_log(rng, 33, 1500), _log(rng, 33, 3000)) if odd else (_log(rng, 128, 4096, 8), _log(rng, 256, 11008, 8))
        if 4.0 * t * d * h <= (4e11 if kind == "gated" else 1e11):
            return dict(kind="gated_train" if kind == "gated_train" else "gated", t=t, d=d, h=h, act=act)


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
def _inputs(c, seed):
    """The inputs of a case, by name (those that exact() reads too)."""
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))

    def normal(*shape, std=1.0, mean=0.0):
        return torch.empty(*shape, dtype=F16, device="cuda").normal_(mean, std, generator=g)

    kind = c["kind"]
    if kind in ("gated", "gated_train"):
        t, d, h = c["t"], c["d"], c["h"]  # normalised rows against weights that keep their spread
        i = dict(x=normal(t, d), w=normal(2, d, h, std=1.0 / math.sqrt(d)))
        if kind == "gated_train":
            i["dh"] = normal(t, h)
        return i
    b, n, dq, dkv = c["b"], c["n"], c["heads"] * c["dh"], c["kv"] * c["dh"]
    if kind in ("rope", "rope_train"):
        i = dict(qkv=normal(b, n, dq + 2 * dkv), offsets=None, wq=None, wk=None)
        if kind == "rope_train" or c["weights"]:
            i.update(wq=normal(c["dh"], std=0.1, mean=1.0), wk=normal(c["dh"], std=0.1, mean=1.0))
        if kind == "rope_train":
            i.update(dq=normal(b, n, dq), dk=normal(b, n, dkv), dv=normal(b, n, dkv))
            return i
        i.update(k=normal(b, c["rows"], dkv), v=normal(b, c["rows"], dkv))
        if c["ragged"]:  # where each sequence has got to
            i["offsets"] = torch.randint(0, c["rows"] - n + 1, (b,), dtype=torch.int32, device="cuda", generator=g)
        return i
    rows = c.get("rows", n)
    i = dict(q=normal(b, n, dq), k=normal(b, rows, dkv), v=normal(b, rows, dkv), offsets=None)
    if kind == "window_train":
        i["do"] = normal(b, n, dq)
    elif c["ragged"]:
        i["offsets"] = torch.randint(0, rows - n + 1, (b,), dtype=torch.int32, device="cuda", generator=g)
    return i


def prepare(case, seed):
    c = case
    s = dict(_inputs(c, seed), case=c)
    kind = c["kind"]
    like = torch.empty_like
    if kind in ("gated", "gated_train"):
        s["y"] = torch.empty(c["t"], c["h"], dtype=F16, device="cuda")
        if kind == "gated_train":
            s.update(gu=torch.empty(2, c["t"], c["h"], dtype=F16, device="cuda"), dx=like(s["x"]), dw=like(s["w"]))
    elif kind == "rope":
        s["q"] = torch.empty(c["b"], c["n"], c["heads"] * c["dh"], dtype=F16, device="cuda")
    elif kind == "rope_train":
        s.update(q=like(s["dq"]), k=like(s["dk"]), v=like(s["dv"]), dqkv=like(s["qkv"]), dwq=like(s["wq"]), dwk=like(s["wk"]))
    else:
        s["o"] = like(s["q"])
        s["lse"] = None
        if kind == "window_train":
            s.update(lse=torch.empty(c["b"], c["heads"], c["n"], dtype=F32, device="cuda"), gq=like(s["q"]), gk=like(s["k"]), gv=like(s["v"]))
    return s


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------
def run(s):
    c = s["case"]
    return (_run_own if own else _PLAIN[c["kind"]])(s, c)


def _run_own(s, c):
    import evk_amd as evk
    kind = c["kind"]
    if kind == "rope":
        evk.qkv_norm_rope(s["qkv"], s["q"], s["k"], s["v"], c["dh"], s["wq"], s["wk"], EPS, BASE, 0, s["offsets"])
        return {k: s[k] for k in ("q", "k", "v")}
    if kind == "rope_train":
        evk.qkv_norm_rope(s["qkv"], s["q"], s["k"], s["v"], c["dh"], s["wq"], s["wk"], EPS, BASE)
        evk.qkv_norm_rope_backward(s["qkv"], s["dq"], s["dk"], s["dv"], s["dqkv"], c["dh"], s["wq"], s["wk"], s["dwq"], s["dwk"], EPS, BASE)
        return {k: s[k] for k in ("q", "k", "v", "dqkv", "dwq", "dwk")}
    if kind == "window":
        evk.window_attention(s["q"], s["k"], s["v"], s["o"], c["dh"], c["window"], c["sinks"], c["p0"], s["offsets"])
        return s["o"]
    if kind == "window_train":
        evk.window_attention(s["q"], s["k"], s["v"], s["o"], c["dh"], c["window"], c["sinks"], lse=s["lse"])
        evk.window_attention_bwd(s["q"], s["k"], s["v"], s["o"], s["do"], s["gq"], s["gk"], s["gv"], s["lse"], c["dh"], c["window"], c["sinks"])
        return {k: s[k] for k in ("o", "lse", "gq", "gk", "gv")}
    if kind == "gated":
        evk.gated_linear(s["x"], s["w"], s["y"], activation=c["act"])
        return s["y"]
    evk.gated_linear(s["x"], s["w"], s["y"], s["gu"], activation=c["act"])
    evk.gated_linear_backward(s["x"], s["w"], s["gu"], s["dh"], s["dx"], s["dw"], activation=c["act"])
    return {k: s[k] for k in ("y", "gu", "dx", "dw")}


# ---- the plain forms: 32 bits, rounded once at the end ----
def _angles(c, offsets):
    """cos and sin (B or 1, N, 1, dh / 2): the angles of far positions need 64 bits."""
    t = torch.arange(c["n"], device="cuda", dtype=F64)[None]
    pos = t if offsets is None else offsets.to(F64)[:, None] + t
    freq = BASE ** (torch.arange(c["dh"] // 2, device="cuda", dtype=F64) * (-2.0 / c["dh"]))
    ang = (pos[..., None] * freq)[:, :, None]
    return torch.cos(ang).to(F32), torch.sin(ang).to(F32)


def _rotate(x, cs, sn):
    """Pairs (2 i, 2 i + 1) of the last dimension turned by their angle."""
    a, b = x[..., 0::2], x[..., 1::2]
    return torch.stack([a * cs - b * sn, a * sn + b * cs], -1).flatten(-2)


def _norm_rope(s, c):
    """Rotated queries and keys and the values: (B, N, heads, dh) each, with the pieces the backward reads."""
    h, kv, dh = c["heads"], c["kv"], c["dh"]
    x = s["qkv"].to(F32).reshape(c["b"], c["n"], h + 2 * kv, dh)
    x, v = x[:, :, :h + kv], x[:, :, h + kv:]
    r = torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS)
    w = None
    y = x * r
    if s["wq"] is not None:
        w = torch.cat([s["wq"].to(F32).expand(h, dh), s["wk"].to(F32).expand(kv, dh)])
        y = y * w
    cs, sn = _angles(c, s["offsets"])
    y = _rotate(y, cs, sn)
    return y[:, :, :h], y[:, :, h:], v, x, r, w, cs, sn


def _plain_rope(s, c):
    b, n = c["b"], c["n"]
    q, k, v = _norm_rope(s, c)[:3]
    s["q"].copy_(q.reshape(b, n, -1))
    if s["offsets"] is None:
        s["k"][:, :n] = k.reshape(b, n, -1).to(F16)
        s["v"][:, :n] = v.reshape(b, n, -1).to(F16)
    else:
        at = (torch.arange(b, device="cuda")[:, None], s["offsets"].long()[:, None] + torch.arange(n, device="cuda"))
        s["k"][at] = k.reshape(b, n, -1).to(F16)
        s["v"][at] = v.reshape(b, n, -1).to(F16)
    return {k: s[k] for k in ("q", "k", "v")}


def _plain_rope_train(s, c):
    b, n, h, kv, dh = c["b"], c["n"], c["heads"], c["kv"], c["dh"]
    q, k, v, x, r, w, cs, sn = _norm_rope(s, c)
    g = torch.cat([s["dq"].reshape(b, n, h, dh), s["dk"].reshape(b, n, kv, dh)], 2).to(F32)
    g = _rotate(g, cs, -sn)
    dw = g * x * r
    g = g * w
    dx = r * (g - x * r.square() * (g * x).mean(-1, keepdim=True))
    dqkv = torch.cat([dx.reshape(b, n, -1), s["dv"].to(F32)], -1)
    out = dict(q=q.reshape(b, n, -1), k=k.reshape(b, n, -1), v=v.reshape(b, n, -1), dqkv=dqkv, dwq=dw[:, :, :h].sum((0, 1, 2)),
               dwk=dw[:, :, h:].sum((0, 1, 2)))
    return {k: t.to(F16) for k, t in out.items()}


def _visible(p, j, window, sinks):
    """Whether the query at position p sees row j."""
    seen = j <= p
    if window:
        seen &= (j > p - window) | (j < sinks)
    return seen


def _scores(s, c):
    """Masked scores (B, kv, group * N, rows) and the query, key and value rows behind them."""
    b, n, h, kv, dh = c["b"], c["n"], c["heads"], c["kv"], c["dh"]
    rows = s["k"].shape[1]
    q = s["q"].to(F32).reshape(b, n, kv, h // kv, dh).permute(0, 2, 3, 1, 4).reshape(b, kv, -1, dh)
    k, v = (s[t].to(F32).reshape(b, rows, kv, dh).transpose(1, 2).contiguous() for t in ("k", "v"))
    t, j = torch.arange(n, device="cuda"), torch.arange(rows, device="cuda")
    p0 = s["offsets"].long()[:, None] if s["offsets"] is not None else c.get("p0", 0)
    p = (p0 + t[None]).reshape(-1, 1, 1, n, 1)
    sc = torch.matmul(q, k.transpose(-1, -2).contiguous()) / math.sqrt(dh)
    sc = sc.reshape(b, kv, h // kv, n, rows).masked_fill(~_visible(p, j, c["window"], c["sinks"]), -math.inf)
    return sc.reshape(b, kv, -1, rows), q, k, v


def _attend(sc, v):
    m = sc.amax(-1, keepdim=True)
    e = torch.exp(sc - m)
    total = e.sum(-1, keepdim=True)
    p = e / total
    return p, torch.matmul(p, v), (m + torch.log(total))[..., 0]


def _rows_of(x, c):
    """(B, kv, group * N, dh) as (B, N, heads * dh)."""
    return x.reshape(c["b"], c["kv"], c["heads"] // c["kv"], c["n"], c["dh"]).permute(0, 3, 1, 2, 4).reshape(c["b"], c["n"], -1)


def _plain_one(s, c):
    """Single tokens: the rows of the window and the sinks gathered, every sequence at its own position."""
    b, h, kv, dh, rows = c["b"], c["heads"], c["kv"], c["dh"], c["rows"]
    window = min(c["window"], rows) if c["window"] else rows
    p = s["offsets"].long()[:, None] if s["offsets"] is not None else torch.full((b, 1), c["p0"], device="cuda")
    j = p - window + 1 + torch.arange(window, device="cuda")  # the window, and before it the sinks outside it
    first = torch.arange(min(c["sinks"], rows), device="cuda").expand(b, -1)
    ok = torch.cat([first < p - window + 1, j >= 0], 1)
    j = torch.cat([first, j.clamp(min=0)], 1)
    at = (torch.arange(b, device="cuda")[:, None], j)
    k, v = (s[t][at].to(F32).reshape(b, -1, kv, dh).transpose(1, 2) for t in ("k", "v"))
    q = s["q"].to(F32).reshape(b, kv, h // kv, dh)
    sc = torch.matmul(q, k.transpose(-1, -2).contiguous()) / math.sqrt(dh)
    o = _attend(sc.masked_fill(~ok[:, None, None], -math.inf), v.contiguous())[1]
    return o.reshape(b, 1, h * dh).to(F16)


def _plain_window(s, c):
    if c["n"] == 1:
        return _plain_one(s, c)
    sc, _, _, v = _scores(s, c)
    return _rows_of(_attend(sc, v)[1], c).to(F16)


def _plain_window_train(s, c):
    b, n, h, kv, dh = c["b"], c["n"], c["heads"], c["kv"], c["dh"]
    sc, q, k, v = _scores(s, c)
    p, o, lse = _attend(sc, v)
    do = s["do"].to(F32).reshape(b, n, kv, h // kv, dh).permute(0, 2, 3, 1, 4).reshape(b, kv, -1, dh)
    dp = torch.matmul(do, v.transpose(-1, -2).contiguous())
    ds = p * (dp - (do * o).sum(-1, keepdim=True)) / math.sqrt(dh)
    gq = torch.matmul(ds, k)
    gk = torch.matmul(ds.transpose(-1, -2).contiguous(), q)
    gv = torch.matmul(p.transpose(-1, -2).contiguous(), do)
    gk, gv = (t.transpose(1, 2).reshape(b, n, -1).to(F16) for t in (gk, gv))
    return dict(o=_rows_of(o, c).to(F16), lse=lse.reshape(b, h, n), gq=_rows_of(gq, c).to(F16), gk=gk, gv=gv)


def _activation(g, act):
    """act(g) and its derivative."""
    if act == "relu":
        on = (g > 0).to(g.dtype)
        return g * on, on
    if act == "silu":
        sg = 1.0 / (1.0 + torch.exp(-g))
        return g * sg, sg * (1.0 + g * (1.0 - sg))
    a = math.sqrt(2.0 / math.pi)
    th = torch.tanh(a * (g + 0.044715 * g * g * g))
    return 0.5 * g * (1.0 + th), 0.5 * (1.0 + th) + 0.5 * g * (1.0 - th * th) * a * (1.0 + 3.0 * 0.044715 * g * g)


def _plain_gated(s, c):
    x, w = s["x"].to(F32), s["w"].to(F32)
    return (_activation(torch.matmul(x, w[0]), c["act"])[0] * torch.matmul(x, w[1])).to(F16)


def _plain_gated_train(s, c):
    x, w, dh = s["x"].to(F32), s["w"].to(F32), s["dh"].to(F32)
    g, u = torch.matmul(x, w[0]), torch.matmul(x, w[1])
    a, da = _activation(g, c["act"])
    dg, du = dh * u * da, dh * a
    xt = x.t().contiguous()
    dx = torch.matmul(dg, w[0].t().contiguous()) + torch.matmul(du, w[1].t().contiguous())
    out = dict(y=a * u, gu=torch.stack([g, u]), dx=dx, dw=torch.stack([torch.matmul(xt, dg), torch.matmul(xt, du)]))
    return {k: t.to(F16) for k, t in out.items()}


_PLAIN = {"rope": _plain_rope, "rope_train": _plain_rope_train, "window": _plain_window, "window_train": _plain_window_train, "gated": _plain_gated,
          "gated_train": _plain_gated_train}


# ---------------------------------------------------------------------------
# 64 bits, from the definitions
# ---------------------------------------------------------------------------
def _exact_rope(c, i):
    b, n, h, kv, dh = c["b"], c["n"], c["heads"], c["kv"], c["dh"]
    train = c["kind"] == "rope_train"
    x = i["qkv"].to(F64).reshape(b, n, h + 2 * kv, dh).requires_grad_(train)
    one = torch.ones(dh, dtype=F64, device="cuda")
    wq, wk = (one if i[t] is None else i[t].to(F64).requires_grad_(train) for t in ("wq", "wk"))
    start = torch.zeros(b, dtype=torch.long, device="cuda") if i["offsets"] is None else i["offsets"].long()
    pos = start[:, None] + torch.arange(n, device="cuda")
    turn = pos[:, :, None, None].to(F64) / BASE ** (torch.arange(0, dh, 2, device="cuda", dtype=F64) / dh)
    unit = torch.polar(torch.ones_like(turn), turn)

    def head(t, w):
        t = t / (t.pow(2).sum(-1, keepdim=True) / dh + EPS).sqrt() * w
        return torch.view_as_real(torch.view_as_complex(t.reshape(*t.shape[:-1], dh // 2, 2)) * unit).reshape(b, n, -1)

    q, k, v = head(x[:, :, :h], wq), head(x[:, :, h:h + kv], wk), x[:, :, h + kv:].reshape(b, n, -1)
    if train:
        g = torch.autograd.grad([q, k, v], [x, wq, wk], [i[t].to(F64) for t in ("dq", "dk", "dv")])
        return dict(q=q.detach(), k=k.detach(), v=v.detach(), dqkv=g[0].reshape(b, n, -1), dwq=g[1], dwk=g[2])
    out = dict(q=q)
    for name, new in (("k", k), ("v", v)):
        out[name] = i[name].to(F64)
        for s in range(b):
            out[name][s, pos[s]] = new[s]
    return out


def _exact_window(c, i):
    b, n, h, kv, dh = c["b"], c["n"], c["heads"], c["kv"], c["dh"]
    train = c["kind"] == "window_train"
    rows, group = i["k"].shape[1], h // kv
    out = dict(o=torch.empty(b, n, h, dh, dtype=F64, device="cuda"))
    if train:
        out.update(lse=torch.empty(b, h, n, dtype=F64, device="cuda"), gq=torch.empty_like(out["o"]),
                   gk=torch.zeros(b, rows, kv, dh, dtype=F64, device="cuda"), gv=torch.zeros(b, rows, kv, dh, dtype=F64, device="cuda"))
    starts = i["offsets"].tolist() if i["offsets"] is not None else [c.get("p0", 0)] * b
    for s in range(b):
        p = starts[s] + torch.arange(n, device="cuda")[:, None]
        lo = max(0, starts[s] - c["window"] + 1) if c["window"] else 0
        hi = starts[s] + n
        j = torch.arange(hi, device="cuda")
        j = j[(j >= lo) | (j < c["sinks"])]
        hidden = j[None] > p
        if c["window"]:
            hidden |= (j[None] <= p - c["window"]) & (j[None] >= c["sinks"])
        for head in range(h):
            at = slice(head * dh, head * dh + dh)
            to = slice(head // group * dh, head // group * dh + dh)
            q, k, v = i["q"][s, :, at].to(F64), i["k"][s, j, to].to(F64), i["v"][s, j, to].to(F64)
            sc = (q @ k.t()) * dh ** -0.5
            sc[hidden] = -math.inf
            lse = torch.logsumexp(sc, 1)
            p_ = (sc - lse[:, None]).exp_()
            o = p_ @ v
            out["o"][s, :, head] = o
            if train:
                do = i["do"][s, :, at].to(F64)
                ds = p_ * (do @ v.t() - (do * o).sum(1, keepdim=True)) * dh ** -0.5
                out["lse"][s, head] = lse
                out["gq"][s, :, head] = ds @ k
                out["gk"][s, j, head // group] += ds.t() @ q
                out["gv"][s, j, head // group] += p_.t() @ do
    out = {k: t if k == "lse" else t.flatten(2) for k, t in out.items()}
    return out if train else out["o"]


def _exact_gated(c, i):
    act = {"silu": torch.nn.functional.silu, "relu": torch.relu,
           "gelu": lambda t: t * torch.sigmoid(2.0 * math.sqrt(2.0 / math.pi) * (t + 0.044715 * t ** 3))}[c["act"]]
    x, wg, wu = i["x"].to(F64), i["w"][0].to(F64), i["w"][1].to(F64)
    g, u = x @ wg, x @ wu
    if c["kind"] == "gated":
        return act(g) * u
    g.requires_grad_(True)
    u.requires_grad_(True)
    y = act(g) * u
    dg, du = torch.autograd.grad(y, [g, u], i["dh"].to(F64))
    return dict(y=y.detach(), gu=torch.stack([g, u]).detach(), dx=dg @ wg.t() + du @ wu.t(), dw=torch.stack([x.t() @ dg, x.t() @ du]))


def exact(case, seed):
    c = case
    i = _inputs(c, seed)
    if c["kind"] in ("gated", "gated_train"):
        return _exact_gated(c, i)
    return _exact_rope(c, i) if c["kind"] in ("rope", "rope_train") else _exact_window(c, i)


# ---------------------------------------------------------------------------
# work
# ---------------------------------------------------------------------------
def _seen(p, c):
    """Rows that a query at position p sees."""
    w = c["window"]
    return p + 1 if not w or p < w else w + min(c["sinks"], p + 1 - w)


def work(case):
    c = case
    kind = c["kind"]
    if kind in ("gated", "gated_train"):
        t, d, h = c["t"], c["d"], c["h"]
        if kind == "gated":
            return dict(bytes=2.0 * (t * d + 2 * d * h + t * h), flops=4.0 * t * d * h)
        return dict(bytes=2.0 * (2 * t * d + 4 * d * h + 4 * t * h), flops=12.0 * t * d * h)
    b, n, h, kv, dh = c["b"], c["n"], c["heads"], c["kv"], c["dh"]
    if kind in ("rope", "rope_train"):
        values = 1.0 * b * n * (h + 2 * kv) * dh
        if kind == "rope":  # products in, rotated rows and values out; about ten operations a value
            return dict(bytes=4.0 * values, flops=10.0 * values)
        return dict(bytes=8.0 * values, flops=30.0 * values)
    if kind == "window" and n == 1:  # positions that differ: half of the rows on average
        p = [c["p0"]] if not c["ragged"] else range(0, c["rows"], max(1, c["rows"] // 64))
        rows = sum(_seen(x, c) for x in p) / len(p)
        return dict(bytes=4.0 * b * dh * (h + rows * kv), flops=4.0 * b * h * dh * rows)
    p0 = c.get("p0", 0)
    pairs = 1.0 * sum(_seen(p0 + t, c) for t in range(n))
    rows = p0 + n if not c["window"] else min(p0 + n, n + c["window"] + c["sinks"])
    if kind == "window":
        return dict(bytes=4.0 * b * dh * (n * h + rows * kv), flops=4.0 * b * h * dh * pairs)
    return dict(bytes=b * (2.0 * dh * (4 * n * h + 4 * n * kv) + 4.0 * h * n), flops=14.0 * b * h * dh * pairs)
