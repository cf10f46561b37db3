"""Cases of the operators that a group of continuations of one prompt needs:
the norms after and before a block with its gate and residual scale, attention
of a batch over a prefix that its sequences share, and log-probabilities of
given tokens with entropy and alternatives; the first and the last with their
backward passes.

  listed()            the named cases
  draw(rng)           one more case of the same ranges
  prepare(case, seed) inputs, outputs and caches on the GPU
  run(state)          one pass: torch operations in 32 bits, or with `own` the
                      calls of evk_amd
  exact(case, seed)   the same outputs in 64 bits
  work(case)          bytes and flops that the pass cannot do without

All tensors are fp16 unless said otherwise.  Token ids are 16-bit values in
int16 tensors.
"""
import math

import torch

own = False

F16, F32, F64 = torch.float16, torch.float32, torch.float64
EPS = 1e-4
PAD = 65535  # an id past every vocabulary here: a place that holds no token


def listed():
    return [
        # one token of each of 16 sequences decoded together, a small model: the smallest call
        dict(name="norm_decode", kind="norm", b=16, n=1, d=768, post=True, gate="none", scale=1.0),
        # a long prompt of a large model, gates and a residual scale of its own
        dict(name="norm_prompt", kind="norm", b=1, n=8192, d=4096, post=True, gate="channel", scale=0.5),
        # training, forward and backward, a gate for each sequence, a length that is no multiple of anything
        dict(name="norm_train", kind="norm_train", b=4, n=1999, d=768, post=True, gate="sequence", scale=1.0),
        # training of a large model, forward and backward
        dict(name="norm_train_wide", kind="norm_train", b=2, n=2048, d=4096, post=True, gate="channel", scale=1.0),
        # one step of 16 sequences over the vocabulary of the reference's training program: latency
        dict(name="score_step", kind="score", t=16, v=144, top=5, c=1.0, banned=0),
        # one step of 64 sequences, alternatives shown, some ids never allowed
        dict(name="score_batch", kind="score", t=64, v=32000, top=8, c=0.7, banned=100),
        # the tokens of a batch of texts scored: bandwidth
        dict(name="score_prompt", kind="score", t=4001, v=32000, top=5, c=1.0, banned=0),
        # policy gradients: log-probabilities and entropies with their gradients, ends of the sequences padded
        dict(name="score_train", kind="score_train", t=2560, v=32000, c=1.0, banned=0, pad=200),
        # a token of each of 16 continuations behind a short prompt, the reference's heads: latency
        dict(name="prefix_decode_d256", kind="prefix", b=16, n=1, heads=1, kv=1, dh=256, prefix=64, rows=160, ragged=True),
        # a token of each of 64 continuations behind a long prompt: bandwidth
        dict(name="prefix_decode_batch", kind="prefix", b=64, n=1, heads=32, kv=8, dh=128, prefix=8192, rows=1024, ragged=True),
        # a few tokens of each sequence at once, a ragged prefix
        dict(name="prefix_few", kind="prefix", b=8, n=5, heads=12, kv=4, dh=64, prefix=3001, rows=300, ragged=True),
        # questions about one long text: prompts of their own behind it
        dict(name="prefix_prompt", kind="prefix", b=8, n=500, heads=16, kv=4, dh=128, prefix=4096, rows=512, ragged=False),
    ]


def _log(rng, lo, hi, step=1):
    """A size from lo to hi, spread over its logarithm, a multiple of step."""
    v = math.exp(rng.uniform(math.log(lo), math.log(hi)))
    return max(lo, min(hi, int(round(v / step)) * step))


def draw(rng):
    kind = rng.choice(["norm", "norm_one", "norm_train", "score", "score_one", "score_train", "prefix", "prefix_one", "prefix_one"])
    if kind in ("norm", "norm_one", "norm_train"):
        while True:
            b = _log(rng, 1, 64) if kind == "norm_one" else _log(rng, 1, 8)
            n = 1 if kind == "norm_one" else _log(rng, 2, 8192)
            d = _log(rng, 32, 8192, rng.choice([1, 8, 8, 64]))
            if b * n * d <= ((16 << 20) if kind == "norm_train" else (32 << 20)):
                return dict(kind="norm_train" if kind == "norm_train" else "norm", b=b, n=n, d=d, post=rng.random() < 0.7,
                            gate=rng.choice(["none", "channel", "sequence"]), scale=rng.choice([1.0, 1.0, 0.5, 1.5]))
    if kind in ("score", "score_one", "score_train"):
        while True:
            t = _log(rng, 1, 64) if kind == "score_one" else _log(rng, 2, 8192)
            v = _log(rng, 64, 65000, rng.choice([1, 8, 16]))
            if t * v > ((64 << 20) if kind == "score_train" else (96 << 20)):
                continue
            c = dict(t=t, v=v, c=rng.choice([1.0, 1.0, 0.7, 1.3]), banned=rng.choice([0, 0, rng.randrange(0, v // 2)]))
            if kind == "score_train":
                return dict(kind=kind, **c, pad=rng.choice([0, rng.randrange(0, t)]))
            return dict(kind="score", **c, top=rng.choice([0, 1, 5, 8, 20]))
    while True:
        dh = rng.choice([32, 64, 64, 80, 96, 128, 128, 256])
        kv = rng.choice([1, 2, 4, 8]) if dh < 256 else rng.choice([1, 2])
        heads = kv * rng.choice([1, 2, 3, 4, 8])
        b = _log(rng, 1, 64) if kind == "prefix_one" else _log(rng, 1, 16)
        n = 1 if kind == "prefix_one" else _log(rng, 2, 600)
        prefix, rows = _log(rng, 17, 16384), n + _log(rng, 1, 2000)
        if b * heads * n * (prefix + rows) > 2.0e8 or b * rows * kv * dh > (64 << 20):
            continue
        return dict(kind="prefix", b=b, n=n, heads=heads, kv=kv, dh=dh, prefix=prefix, rows=rows, ragged=rng.random() < 0.7)


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
    if kind in ("norm", "norm_train"):
        b, n, d = c["b"], c["n"], c["d"]
        i = dict(x=normal(b, n, d, std=4.0), y=normal(b, n, d), wi=normal(d, std=0.1, mean=1.0), wo=None, gate=None)
        if c["post"]:
            i["wo"] = normal(d, std=0.1, mean=1.0)
        if c["gate"] != "none":
            i["gate"] = normal(d, std=0.5) if c["gate"] == "channel" else normal(b, d, std=0.5)
        if kind == "norm_train":
            i.update(ds=normal(b, n, d), dh=normal(b, n, d))
        return i
    if kind in ("score", "score_train"):
        t, v = c["t"], c["v"]
        ids = torch.randint(c["banned"], v, (t,), device="cuda", generator=g)
        i = dict(logits=normal(t, v, std=2.5))
        i["logits"][torch.arange(t, device="cuda"), ids] += 8.0  # sampled tokens are likely ones
        i["logits"][:, :c["banned"]] = -math.inf
        if kind == "score_train":
            ids[t - c["pad"]:] = PAD
            i.update(dlp=normal(t).to(F32), dent=0.01 * normal(t).to(F32))
        i["tokens"] = torch.where(ids > 32767, ids - 65536, ids).to(torch.int16)
        return i
    b, n, dq, dkv = c["b"], c["n"], c["heads"] * c["dh"], c["kv"] * c["dh"]
    i = dict(q=normal(b, n, dq), pk=normal(c["prefix"], dkv), pv=normal(c["prefix"], dkv), k=normal(b, c["rows"], dkv),
             v=normal(b, c["rows"], dkv), offsets=None)
    if c["ragged"]:  # how far each continuation has got
        i["offsets"] = torch.randint(0, c["rows"] - n + 1, (b,), dtype=torch.int32, device="cuda", generator=g)
    return i


def prepare(case, seed):
    c = case
    s = dict(_inputs(c, seed), case=c)
    kind = c["kind"]
    like = torch.empty_like
    if kind in ("norm", "norm_train"):
        s.update(s=like(s["x"]), h=like(s["x"]))
        if kind == "norm_train":
            s.update(dx=like(s["x"]), dy=like(s["x"]), dwi=like(s["wi"]))
            s["dwo"] = None if s["wo"] is None else like(s["wo"])
            s["dgate"] = None if s["gate"] is None else like(s["gate"])
    elif kind in ("score", "score_train"):
        t = c["t"]
        s.update(lp=torch.empty(t, dtype=F32, device="cuda"), ent=torch.empty(t, dtype=F32, device="cuda"), ids=None, alt=None)
        if kind == "score_train":
            s.update(stats=torch.empty(t, 2, dtype=F32, device="cuda"), dlogits=like(s["logits"]))
        elif c["top"]:
            s.update(ids=torch.empty(t, c["top"], dtype=torch.int16, device="cuda"), alt=torch.empty(t, c["top"], dtype=F32, device="cuda"))
    else:
        s["o"] = like(s["q"])
    return s


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------
def run(s):
    c = s["case"]
    return (_run_own if own else _PLAIN[c["kind"]])(s, c)


def _pick(s, names):
    return {k: s[k] for k in names if s[k] is not None}


def _run_own(s, c):
    import evk_amd as evk
    kind = c["kind"]
    if kind in ("norm", "norm_train"):
        evk.residual_norm(s["x"], s["y"], s["s"], s["h"], s["wo"], s["gate"], s["wi"], residual_scale=c["scale"], post_norm=c["post"], eps=EPS)
        if kind == "norm":
            return _pick(s, ("s", "h"))
        evk.residual_norm_backward(s["x"], s["y"], s["ds"], s["dh"], s["dx"], s["dy"], s["wo"], s["gate"], s["wi"], s["dwo"], s["dgate"], s["dwi"],
                                   residual_scale=c["scale"], post_norm=c["post"], eps=EPS)
        return _pick(s, ("s", "h", "dx", "dy", "dwo", "dgate", "dwi"))
    if kind == "score":
        evk.token_logprobs(s["logits"], s["tokens"], s["lp"], s["ent"], s["ids"], s["alt"], input_scale=c["c"])
        return _pick(s, ("lp", "ent", "ids", "alt"))
    if kind == "score_train":
        evk.token_logprobs(s["logits"], s["tokens"], s["lp"], s["ent"], stats=s["stats"], input_scale=c["c"])
        evk.token_logprobs_backward(s["logits"], s["tokens"], s["stats"], s["dlp"], s["dlogits"], s["ent"], s["dent"], input_scale=c["c"])
        return _pick(s, ("lp", "ent", "dlogits"))
    evk.prefix_attention(s["q"], s["pk"], s["pv"], s["k"], s["v"], s["o"], c["dh"], offsets=s["offsets"])
    return s["o"]


# ---- the plain forms: 32 bits, rounded once at the end ----
def _norm_parts(s, c):
    x, y = s["x"].to(F32), s["y"].to(F32)
    q, wo, g = None, None, None
    yn = y
    if c["post"]:
        q = torch.rsqrt(y.square().mean(-1, keepdim=True) + EPS)
        wo, yn = s["wo"].to(F32), y * q
    out = yn if wo is None else yn * wo
    if s["gate"] is not None:
        g = s["gate"].to(F32)
        g = g if g.dim() == 1 else g[:, None]
        out = out * g
    st = c["scale"] * x + out
    r = torch.rsqrt(st.square().mean(-1, keepdim=True) + EPS)
    return yn, q, wo, g, st, r


def _plain_norm(s, c):
    _, _, _, _, st, r = _norm_parts(s, c)
    return dict(s=st.to(F16), h=(st * r * s["wi"].to(F32)).to(F16))


def _plain_norm_train(s, c):
    yn, q, wo, g, st, r = _norm_parts(s, c)
    wi, dh = s["wi"].to(F32), s["dh"].to(F32)
    u = st * r
    dn = dh * wi
    grad = s["ds"].to(F32) + r * (dn - u * (dn * u).mean(-1, keepdim=True))
    out = dict(s=st, h=u * wi, dx=c["scale"] * grad, dwi=(dh * u).sum((0, 1)))
    dy = grad if g is None else grad * g
    if g is not None:
        dg = grad * (yn if wo is None else yn * wo)
        out["dgate"] = dg.sum((0, 1) if s["gate"].dim() == 1 else 1)
    if wo is not None:
        out["dwo"] = (dy * yn).sum((0, 1))
        dy = dy * wo
        dy = q * (dy - yn * (dy * yn).mean(-1, keepdim=True))
    out["dy"] = dy
    return {k: t.to(F16) for k, t in out.items()}


def _ids(tokens):
    return tokens.long() & 0xFFFF


def _scores(s, c):
    """Logits below their row's largest, scaled; the logarithm of the sum of their exponentials; the tokens' places."""
    x = s["logits"].to(F32)
    z = (x - x.amax(-1, keepdim=True)) * c["c"]
    total = torch.log(torch.exp(z).sum(-1))
    t = _ids(s["tokens"])
    return z, total, t, t < c["v"]


def _plain_score(s, c):
    z, total, t, there = _scores(s, c)
    lp = z.gather(-1, t.clamp(max=c["v"] - 1)[:, None])[:, 0] - total
    p = torch.exp(z - total[:, None])
    out = dict(lp=torch.where(there, lp, 0.0), ent=total - torch.where(p > 0, p * z, 0.0).sum(-1))
    if c.get("top"):
        # order of the values, then of the ids: one whole number for each logit
        bits = s["logits"].view(torch.int16).long()
        rank = torch.where(bits < 0, -(bits & 0x7FFF), bits) * 65536 + (65535 - torch.arange(c["v"], device="cuda"))
        ids = 65535 - (rank.topk(c["top"], -1)[0] & 0xFFFF)
        out["alt"] = z.gather(-1, ids) - total[:, None]
        out["ids"] = torch.where(ids > 32767, ids - 65536, ids).to(torch.int16)
    return out


def _plain_score_train(s, c):
    out = _plain_score(s, c)
    z, total, t, there = _scores(s, c)
    logp = z - total[:, None]
    p = torch.exp(logp)
    dlp = torch.where(there, s["dlp"], 0.0)[:, None]
    grad = -dlp * p - torch.where(p > 0, s["dent"][:, None] * p * (logp + out["ent"][:, None]), 0.0)
    grad.scatter_add_(-1, t.clamp(max=c["v"] - 1)[:, None], dlp)
    out["dlogits"] = (c["c"] * grad).to(F16)
    return out


def _plain_prefix(s, c):
    b, n, h, kv, dh, rows, p = (c[x] for x in ("b", "n", "heads", "kv", "dh", "rows", "prefix"))
    gr = h // kv
    q = s["q"].to(F32).reshape(b, n, kv, gr, dh).permute(2, 0, 3, 1, 4).contiguous()  # kv, b, group, n, dh
    pk, pv = (s[t].to(F32).reshape(p, kv, dh).transpose(0, 1).contiguous() for t in ("pk", "pv"))
    k, v = (s[t].to(F32).reshape(b, rows, kv, dh).permute(2, 0, 1, 3).reshape(kv * b, rows, dh) for t in ("k", "v"))
    shared = torch.matmul(q.reshape(kv, -1, dh), pk.transpose(1, 2).contiguous()).reshape(kv, b, gr, n, p)
    alone = torch.matmul(q.reshape(kv * b, gr * n, dh), k.transpose(1, 2).contiguous()).reshape(kv, b, gr, n, rows)
    first = torch.zeros(b, dtype=torch.long, device="cuda") if s["offsets"] is None else s["offsets"].long()
    last = (first[:, None] + torch.arange(n, device="cuda"))[:, None, :, None]
    alone = alone.masked_fill(torch.arange(rows, device="cuda") > last, -math.inf)
    sc = torch.cat([shared, alone], -1) / math.sqrt(dh)
    e = torch.exp(sc - sc.amax(-1, keepdim=True))
    w = e / e.sum(-1, keepdim=True)
    o = torch.matmul(w[..., :p].reshape(kv, -1, p), pv).reshape(kv * b, gr * n, dh)
    o = o + torch.matmul(w[..., p:].reshape(kv * b, gr * n, rows), v)
    return o.reshape(kv, b, gr, n, dh).permute(1, 3, 0, 2, 4).reshape(b, n, h * dh).to(F16)


_PLAIN = {"norm": _plain_norm, "norm_train": _plain_norm_train, "score": _plain_score, "score_train": _plain_score_train,
          "prefix": _plain_prefix}


# ---------------------------------------------------------------------------
# 64 bits, from the definitions
# ---------------------------------------------------------------------------
def _rms(t):
    return t / (t.pow(2).sum(-1, keepdim=True) / t.shape[-1] + EPS).sqrt()


def _exact_norm(c, i):
    train = c["kind"] == "norm_train"
    leaves = {k: i[k].to(F64).requires_grad_(train) for k in ("x", "y", "wi", "wo", "gate") if i[k] is not None}
    x, y = leaves["x"], leaves["y"]
    if c["post"]:
        y = _rms(y) * leaves["wo"]
    if "gate" in leaves:
        g = leaves["gate"]
        y = torch.einsum("bnd,bd->bnd", y, g.expand(c["b"], c["d"]))
    st = x * c["scale"] + y
    h = _rms(st) * leaves["wi"]
    if not train:
        return dict(s=st, h=h)
    grads = torch.autograd.grad([st, h], list(leaves.values()), [i["ds"].to(F64), i["dh"].to(F64)])
    return dict(s=st.detach(), h=h.detach(), **{"d" + k: t for k, t in zip(leaves, grads)})


def _exact_score(c, i):
    x = i["logits"].to(F64)
    lp = torch.log_softmax(x * c["c"], -1)
    p = lp.exp()
    there = torch.tensor([k & 0xFFFF for k in i["tokens"].tolist()], device="cuda")
    ok = there < c["v"]
    at = torch.arange(c["t"], device="cuda")
    chosen = lp[at, torch.where(ok, there, 0)]
    plogp = torch.special.entr(p)
    ent = plogp.sum(-1)
    out = dict(lp=chosen.masked_fill(~ok, 0.0), ent=ent)
    if c["kind"] == "score_train":
        w = i["dlp"].to(F64) * ok
        d = plogp - p * ent[:, None]  # of the entropy: -p (log p + H)
        d = d * i["dent"].to(F64)[:, None] - p * w[:, None]
        d[at, torch.where(ok, there, 0)] += w
        out["dlogits"] = d * c["c"]
    elif c["top"]:
        ids = torch.sort(x, dim=-1, descending=True, stable=True)[1][:, :c["top"]]
        out["alt"] = lp.gather(-1, ids)
        out["ids"] = ((ids + 32768) % 65536 - 32768).to(torch.int16)
    return out


def _exact_prefix(c, i):
    b, n, h, kv, dh, p = (c[x] for x in ("b", "n", "heads", "kv", "dh", "prefix"))
    o = torch.empty(b, n, h, dh, dtype=F64, device="cuda")
    starts = i["offsets"].tolist() if i["offsets"] is not None else [0] * b
    for s in range(b):
        end = starts[s] + n
        k, v = (torch.cat([i["p" + t], i[t][s, :end]]).to(F64).view(p + end, kv, dh) for t in ("k", "v"))
        hidden = torch.arange(p + end, device="cuda")[None] > p + starts[s] + torch.arange(n, device="cuda")[:, None]
        for head in range(h):
            q = i["q"][s, :, head * dh:head * dh + dh].to(F64)
            sc = (q @ k[:, head // (h // kv)].t()) * dh ** -0.5
            o[s, :, head] = torch.softmax(sc.masked_fill_(hidden, -math.inf), -1) @ v[:, head // (h // kv)]
    return o.flatten(2)


def exact(case, seed):
    c = case
    i = _inputs(c, seed)
    if c["kind"] in ("norm", "norm_train"):
        return _exact_norm(c, i)
    return _exact_score(c, i) if c["kind"] in ("score", "score_train") else _exact_prefix(c, i)


# ---------------------------------------------------------------------------
# work
# ---------------------------------------------------------------------------
def work(case):
    c = case
    kind = c["kind"]
    if kind in ("norm", "norm_train"):
        values = 1.0 * c["b"] * c["n"] * c["d"]
        if kind == "norm":  # x and y in, s and h out
            return dict(bytes=8.0 * values, flops=10.0 * values)
        return dict(bytes=16.0 * values, flops=40.0 * values)  # x, y, ds, dh in, s, h, dx, dy out
    if kind in ("score", "score_train"):
        values = 1.0 * c["t"] * c["v"]
        return dict(bytes=2.0 * values, flops=6.0 * values) if kind == "score" else dict(bytes=4.0 * values, flops=16.0 * values)
    b, n, h, kv, dh, p, rows = (c[x] for x in ("b", "n", "heads", "kv", "dh", "prefix", "rows"))
    start = (rows - n) / 2 if c["ragged"] else 0  # of offsets that differ, on average
    seen = n * p + n * start + n * (n + 1) / 2  # rows that the queries of one head see
    return dict(bytes=4.0 * kv * dh * (p + b * (start + n)) + 4.0 * b * n * h * dh, flops=4.0 * b * h * dh * seen)
