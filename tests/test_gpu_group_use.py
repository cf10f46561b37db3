"""GPU: the operators of a group of continuations as programs use them: a group
decoded behind one prompt and scored, a policy-gradient step, streams, captured
graphs, calls at the same time, tensors past 4 GiB."""
import math

import pytest
import torch

import evk_amd as evk
from test_gpu_block import E, F16, F32, F64, H, T, Rng, close, empty
from test_gpu_block_use import rel
from test_gpu_group import ROW, ids16, prefix_want, scores_want, u16

pytestmark = pytest.mark.gpu


class Model:
    """Layers of a grouped-query block with norms before and after, an embedding and an output product."""

    def __init__(self, dev, r, layers=2, d=192, heads=6, kv=2, dh=32, f=256, vocab=301):
        self.dev, self.layers, self.d, self.heads, self.kv, self.dh, self.f, self.vocab = dev, layers, d, heads, kv, dh, f, vocab
        wide = (heads + 2 * kv) * dh
        one = lambda n: r(n, mean=1.0, std=0.1)  # noqa: E731
        self.w = dict(emb=r(vocab, d), first=one(d), out=r(d, vocab, std=2 * d ** -0.5))
        for i in range(layers):
            self.w.update({f"qkv{i}": r(d, wide, std=d ** -0.5), f"nq{i}": one(dh), f"nk{i}": one(dh), f"o{i}": r(heads * dh, d, std=(heads * dh) ** -0.5),
                           f"gu{i}": r(2, d, f, std=d ** -0.5), f"down{i}": r(f, d, std=f ** -0.5), f"pa{i}": one(d), f"pf{i}": one(d),
                           f"ra{i}": one(d), f"rf{i}": one(d), f"ga{i}": r(d, mean=0.7, std=0.1), f"gf{i}": r(d, mean=0.7, std=0.1)})

    def cache(self, b, rows):
        return [[torch.full((b, rows, self.kv * self.dh), math.nan, dtype=F16, device=self.dev) for _ in range(2)] for _ in range(self.layers)]

    def forward(self, ids, prefix=None, cache=None, offsets=None, first=0, keep=None):
        """Logits (B, N, vocab) of ids (B, N).  With a prefix (per layer k, v (P, kv dh)) the rows go to the cache at
        offsets[b]; without, whole sequences, whose keys and values are returned as a prefix."""
        w, dev, e = self.w, self.dev, lambda *s: torch.empty(*s, dtype=F16, device=self.dev)  # noqa: E731
        b, n = ids.shape
        x, h = e(b, n, self.d), e(b, n, self.d)
        evk.embed(w["emb"], ids16(ids), x)
        evk.residual_norm(x, None, None, h, pre_weight=w["first"])
        made, a = [], dict(x0=x, h0=h)
        for i in range(self.layers):
            qkv, q, att, y = e(b, n, w[f"qkv{i}"].shape[1]), e(b, n, self.heads * self.dh), e(b, n, self.heads * self.dh), e(b, n, self.d)
            evk.matmul(h, w[f"qkv{i}"], qkv)
            if prefix is None:
                k, v, lse = e(b, n, self.kv * self.dh), e(b, n, self.kv * self.dh), torch.empty(b, self.heads, n, device=dev)
                evk.qkv_norm_rope(qkv, q, k, v, self.dh, w[f"nq{i}"], w[f"nk{i}"])
                evk.window_attention(q, k, v, att, self.dh, lse=lse)
                a.update({f"k{i}": k, f"v{i}": v, f"lse{i}": lse})
                made.append((k[0], v[0]))
            else:
                k, v = cache[i]
                evk.qkv_norm_rope(qkv, q, k, v, self.dh, w[f"nq{i}"], w[f"nk{i}"], offsets=offsets, first_position=first)
                evk.prefix_attention(q, *prefix[i], k, v, att, self.dh, offsets=offsets)
            evk.matmul(att, w[f"o{i}"], y)
            s, ha = e(b, n, self.d), e(b, n, self.d)
            evk.residual_norm(x, y, s, ha, w[f"pa{i}"], w[f"ga{i}"], w[f"ra{i}"])
            u, gu, z = e(b, n, self.f), e(2, b, n, self.f), e(b, n, self.d)
            evk.gated_linear(ha, w[f"gu{i}"], u, gu)
            evk.matmul(u, w[f"down{i}"], z)
            x2, h2 = e(b, n, self.d), e(b, n, self.d)
            evk.residual_norm(s, z, x2, h2, w[f"pf{i}"], w[f"gf{i}"], w[f"rf{i}"], residual_scale=0.9)
            a.update({f"x{i}": x, f"h{i}": h, f"qkv{i}": qkv, f"q{i}": q, f"att{i}": att, f"y{i}": y, f"s{i}": s, f"ha{i}": ha, f"u{i}": u, f"gate_up{i}": gu,
                      f"z{i}": z})
            x, h = x2, h2
        logits = e(b, n, self.vocab)
        evk.matmul(h, w["out"], logits)
        a["h"] = h
        if keep is not None:
            keep.update(a)
        return logits, made

    def backward(self, ids, a, dlogits):
        """Gradients of every weight from that of the logits, by the operators."""
        w, like = self.w, torch.empty_like
        b, n = ids.shape
        flat = lambda t: t.view(b * n, -1)  # noqa: E731
        g = {k: like(v) for k, v in w.items()}
        dh, ds = like(a["h"]), None
        evk.matmul(flat(a["h"]), flat(dlogits), g["out"], transpose_a=True)
        evk.matmul(flat(dlogits), w["out"], flat(dh), transpose_b=True)
        for i in reversed(range(self.layers)):
            dstream, dz, du, dha = like(a[f"s{i}"]), like(a[f"z{i}"]), like(a[f"u{i}"]), like(a[f"ha{i}"])
            evk.residual_norm_backward(a[f"s{i}"], a[f"z{i}"], ds, dh, dstream, dz, w[f"pf{i}"], w[f"gf{i}"], w[f"rf{i}"], g[f"pf{i}"], g[f"gf{i}"],
                                       g[f"rf{i}"], residual_scale=0.9)
            evk.matmul(flat(a[f"u{i}"]), flat(dz), g[f"down{i}"], transpose_a=True)
            evk.matmul(flat(dz), w[f"down{i}"], flat(du), transpose_b=True)
            evk.gated_linear_backward(a[f"ha{i}"], w[f"gu{i}"], a[f"gate_up{i}"], du, dha, g[f"gu{i}"])
            dx, dy = like(dstream), like(dz)
            evk.residual_norm_backward(a[f"x{i}"], a[f"y{i}"], dstream, dha, dx, dy, w[f"pa{i}"], w[f"ga{i}"], w[f"ra{i}"], g[f"pa{i}"], g[f"ga{i}"],
                                       g[f"ra{i}"])
            datt, dq, dk, dv, dqkv = like(a[f"att{i}"]), like(a[f"q{i}"]), like(a[f"k{i}"]), like(a[f"v{i}"]), like(a[f"qkv{i}"])
            evk.matmul(flat(a[f"att{i}"]), flat(dy), g[f"o{i}"], transpose_a=True)
            evk.matmul(flat(dy), w[f"o{i}"], flat(datt), transpose_b=True)
            evk.window_attention_bwd(a[f"q{i}"], a[f"k{i}"], a[f"v{i}"], a[f"att{i}"], datt, dq, dk, dv, a[f"lse{i}"], self.dh)
            evk.qkv_norm_rope_backward(a[f"qkv{i}"], dq, dk, dv, dqkv, self.dh, w[f"nq{i}"], w[f"nk{i}"], g[f"nq{i}"], g[f"nk{i}"])
            evk.matmul(flat(a[f"h{i}"]), flat(dqkv), g[f"qkv{i}"], transpose_a=True)
            dh = like(dh)
            evk.matmul(flat(dqkv), w[f"qkv{i}"], flat(dh), transpose_b=True)
            ds = dx
        dx = like(ds)
        evk.residual_norm_backward(a["x0"], None, ds, dh, dx, None, pre_weight=w["first"], dpre_weight=g["first"])
        g["emb"].zero_()
        evk.embed_backward(dx, ids16(ids), g["emb"])
        return g

    def exact(self, ids, w):
        """Logits in 64 bits on weights that autograd follows."""
        b, n = ids.shape
        norm = lambda t: t / torch.sqrt(t.square().mean(-1, keepdim=True) + 1e-4)  # noqa: E731
        x = w["emb"][ids]
        h = norm(x) * w["first"]
        ang = torch.arange(n, device=self.dev, dtype=F64)[:, None, None] * 10000.0 ** (-torch.arange(0, self.dh, 2, device=self.dev, dtype=F64) / self.dh)
        c, s = torch.cos(ang), torch.sin(ang)

        def turned(t):
            p, q = t[..., 0::2], t[..., 1::2]
            return torch.stack([p * c - q * s, p * s + q * c], -1).flatten(-2)

        hidden = torch.ones(n, n, device=self.dev).triu(1).bool()
        for i in range(self.layers):
            t = (h.reshape(b * n, -1) @ w[f"qkv{i}"]).view(b, n, self.heads + 2 * self.kv, self.dh)
            q = turned(norm(t[:, :, :self.heads]) * w[f"nq{i}"])
            k = turned(norm(t[:, :, self.heads:self.heads + self.kv]) * w[f"nk{i}"]).repeat_interleave(self.heads // self.kv, 2)
            v = t[:, :, self.heads + self.kv:].repeat_interleave(self.heads // self.kv, 2)
            q, k, v = (u.permute(0, 2, 1, 3).contiguous() for u in (q, k, v))
            sc = (torch.matmul(q, k.transpose(2, 3).contiguous()) * self.dh ** -0.5).masked_fill(hidden, -math.inf)
            att = torch.matmul(torch.softmax(sc, -1), v).permute(0, 2, 1, 3).reshape(b * n, -1)
            st = x + w[f"ga{i}"] * norm((att @ w[f"o{i}"]).view(b, n, -1)) * w[f"pa{i}"]
            h = (norm(st) * w[f"ra{i}"]).reshape(b * n, -1)
            u = torch.nn.functional.silu(h @ w[f"gu{i}"][0]) * (h @ w[f"gu{i}"][1])
            x = 0.9 * st + w[f"gf{i}"] * norm((u @ w[f"down{i}"]).view(b, n, -1)) * w[f"pf{i}"]
            h = norm(x) * w[f"rf{i}"]
        return (h.reshape(b * n, -1) @ w["out"]).view(b, n, -1)


def test_group_behind_one_prompt(dev):
    """Continuations of one prompt, decoded behind its rows that lie in memory once (first a few tokens at once, then one by
    one, each sequence at its own length), give the logits and the scores of the whole sequences."""
    r = Rng(dev, 11)
    m = Model(dev, r)
    b, p, rows = 5, 77, 40
    g = torch.Generator(device=dev).manual_seed(4)
    prompt = torch.randint(0, m.vocab, (1, p), device=dev, generator=g)
    more = torch.randint(0, m.vocab, (b, 30), device=dev, generator=g)
    whole = torch.cat([m.forward(torch.cat([prompt, more[i:i + 1]], 1))[0][:, p:] for i in range(b)])
    _, prefix = m.forward(prompt)
    cache = m.cache(b, rows)
    # the same sums in another order and with other roundings of P, two layers of a dozen roundings: as for one block, twice
    n = 6
    first, _ = m.forward(more[:, :n].contiguous(), prefix, cache, torch.zeros(b, dtype=torch.int32, device=dev), p)
    assert rel(first, whole[:, :n].to(F64)) <= 16 * H
    at = torch.full((b,), n, dtype=torch.int32, device=dev)
    for step in range(8):
        ids = more.gather(1, at.long()[:, None])
        logits, _ = m.forward(ids, prefix, cache, at, p)
        want = torch.stack([whole[i, int(at[i])] for i in range(b)])[:, None]
        assert rel(logits, want.to(F64)) <= 16 * H, step
        nxt = more.gather(1, at.long()[:, None] + 1)
        lp, ent = torch.empty(b, device=dev), torch.empty(b, device=dev)
        top, alt = torch.empty(b, 3, dtype=torch.int16, device=dev), torch.empty(b, 3, device=dev)
        evk.token_logprobs(logits, ids16(nxt), lp, ent, top, alt)
        w = scores_want(logits.view(b, -1), ids16(nxt[:, 0]), 1.0, 3)
        assert torch.equal(u16(top), w["ids"]) and ((lp - w["lp"]).abs() <= 1e-4).all()
        at += 1 if step % 2 else torch.arange(b, device=dev) % 2  # some stay where they are and decode the same token again
    k = cache[0][0]
    assert torch.isnan(k[0, int(at[0]) + 1:]).all() and not torch.isnan(k[0, :int(at[0])]).any()


def test_policy_gradient_step(dev):
    """Log-probabilities and entropies of sampled tokens, and the gradients of every weight, against 64 bits.  Every
    gradient has at most about 60 roundings to fp16 behind it, each at most H of its tensor's norm: 8 H in quadrature,
    passed on with at most a few times their size by norms and softmaxes of two layers."""
    r = Rng(dev, 21)
    m = Model(dev, r)
    b, n = 3, 50
    g = torch.Generator(device=dev).manual_seed(5)
    ids = torch.randint(0, m.vocab, (b, n), device=dev, generator=g)
    nxt = torch.randint(0, m.vocab, (b, n), device=dev, generator=g)
    nxt[1, -7:] = 65535  # a sequence that ended before
    dlp = 0.25 * torch.randn(b, 1, device=dev, generator=g).expand(b, n).contiguous().view(-1)  # advantages
    dent = torch.full((b * n,), -0.01, device=dev)
    dent.view(b, n)[1, -7:] = 0.0
    keep = {}
    logits, _ = m.forward(ids, keep=keep)
    lp, ent, stats = torch.empty(b * n, device=dev), torch.empty(b * n, device=dev), torch.empty(b * n, 2, device=dev)
    evk.token_logprobs(logits, ids16(nxt), lp, ent, stats=stats)
    dlogits = torch.empty_like(logits)
    evk.token_logprobs_backward(logits, ids16(nxt), stats, dlp, dlogits, ent, dent)
    assert (dlogits[1, -7:] == 0).all()
    got = m.backward(ids, keep, dlogits)
    w64 = {k: t.to(F64).requires_grad_(True) for k, t in m.w.items()}
    logp = torch.log_softmax(m.exact(ids, w64), -1)
    there = nxt < m.vocab
    chosen = logp.gather(-1, nxt.clamp(max=m.vocab - 1)[..., None])[..., 0] * there
    loss = (chosen.view(-1) * dlp).sum() - ((logp.exp() * logp).sum(-1).view(-1) * dent).sum()
    want = torch.autograd.grad(loss, list(w64.values()))
    assert rel(lp.view(b, n), chosen.detach()) <= 16 * H
    for (k, t), x in zip(w64.items(), want):
        assert rel(got[k], x) <= 32 * H, (k, rel(got[k], x) / H)


def steps(dev):
    """Calls of every entry point on static tensors: (inputs, outputs, call)."""
    r = Rng(dev, 81)
    b, n, d = 3, 40, 768
    x, y, ds, dh = (r(b, n, d) for _ in range(4))
    wo, wi, gate = r(d, mean=1.0), r(d, mean=1.0), r(b, d)
    s, h, dx, dy = (empty(dev, b, n, d) for _ in range(4))
    dwo, dwi, dg = empty(dev, d), empty(dev, d), empty(dev, b, d)
    t, v = 70, 5000
    logits, tok = r(t, v, std=3.0), ids16(torch.arange(t, device=dev) * 13)
    f = lambda *z: torch.zeros(*z, device=dev)  # noqa: E731
    lp, ent, stats, alt = f(t), f(t), f(t, 2), f(t, 5)
    ids = torch.zeros(t, 5, dtype=torch.int16, device=dev)
    dlp, dent, dl = r(t).float(), r(t).float(), empty(dev, t, v)
    hh, kv, dq = 8, 2, 64
    sets, outs = [], []
    for (qb, qn, p, rows) in ((6, 1, 20000, 70), (4, 3, 400, 90), (2, 150, 300, 160), (1, 1, 9000, 40)):
        q, pk, pv, k, vv = r(qb, qn, hh * dq), r(p, kv * dq), r(p, kv * dq), r(qb, rows, kv * dq), r(qb, rows, kv * dq)
        off = torch.arange(qb, dtype=torch.int32, device=dev) + 3
        o, lse = empty(dev, qb, qn, hh * dq), f(qb, hh, qn)
        sets.append((q, pk, pv, k, vv, o, off, lse))
        outs += [o, lse]
    # prefix shared with a second launch, in one launch, by tiles, split
    assert [evk.prefix_attention_workspace(z[0], z[1], z[3], dq) > 0 for z in sets] == [True, False, True, True]

    def call():
        evk.residual_norm(x, y, s, h, wo, gate, wi, residual_scale=0.5)
        evk.residual_norm_backward(x, y, ds, dh, dx, dy, wo, gate, wi, dwo, dg, dwi, residual_scale=0.5)
        evk.token_logprobs(logits, tok, lp, ent, ids, alt, stats)
        evk.token_logprobs_backward(logits, tok, stats, dlp, dl, ent, dent)
        for q, pk, pv, k, vv, o, off, lse in sets:
            evk.prefix_attention(q, pk, pv, k, vv, o, dq, offsets=off, lse=lse)

    ins = [x, y, ds, dh, logits] + [z[0] for z in sets] + [z[1] for z in sets]
    return ins, [s, h, dx, dy, dwo, dwi, dg, lp, ent, stats, alt, ids, dl] + outs, call


def test_other_stream(dev):
    ins, outs, call = steps(dev)
    call()
    torch.cuda.synchronize()
    want = [t.clone() for t in outs]
    for t in outs:
        t.fill_(9)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        call()
    torch.cuda.current_stream().wait_stream(s)
    for t, w in zip(outs, want):
        assert torch.equal(t, w)


def test_streams_at_once(dev):
    """The same calls on two streams at the same time, on tensors and workspaces of their own."""
    sets = [steps(dev) for _ in range(2)]
    for _, _, call in sets:
        call()
    torch.cuda.synchronize()
    want = [[t.clone() for t in outs] for _, outs, _ in sets]
    streams = [torch.cuda.Stream() for _ in sets]
    for _ in range(5):
        for (_, outs, call), s in zip(sets, streams):
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                call()
    torch.cuda.synchronize()
    for (_, outs, _), w in zip(sets, want):
        for t, x in zip(outs, w):
            assert torch.equal(t, x)


def test_two_graphs(dev):
    """Two captured graphs, replayed in turn with eager calls, allocations and new inputs between the replays."""
    sets = [steps(dev) for _ in range(2)]
    graphs = []
    s = torch.cuda.Stream()
    for _, _, call in sets:
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            call()
        torch.cuda.current_stream().wait_stream(s)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            call()
        graphs.append(g)
    r = Rng(dev, 5)
    other = steps(dev)[2]
    for it in range(4):
        for (ins, outs, call), g in zip(sets, graphs):
            for t in ins:
                t.copy_(r(*t.shape, std=0.5 if it % 2 else 1.0))
            for t in outs:
                t.fill_(3)
            junk = torch.full((1 << 22,), math.nan, device=dev)  # what a released workspace would be taken by
            other()
            g.replay()
            torch.cuda.synchronize()
            got = [t.clone() for t in outs]
            call()
            torch.cuda.synchronize()
            for t, w in zip(got, outs):
                assert torch.equal(t, w)
            del junk


def test_explicit_workspace_and_stream(dev):
    r = Rng(dev, 91)
    q, pk, pv, k, v = r(1, 1, 256), r(9000, 128), r(9000, 128), r(1, 30, 128), r(1, 30, 128)
    o, o2 = torch.empty_like(q), torch.empty_like(q)
    evk.prefix_attention(q, pk, pv, k, v, o, 64, 29)
    need = evk.prefix_attention_workspace(q, pk, k, 64)
    assert need > 0
    s = torch.cuda.Stream()
    torch.cuda.synchronize()
    with pytest.raises(ValueError, match="workspace"):
        evk.prefix_attention(q, pk, pv, k, v, o2, 64, 29, stream=s.cuda_stream)
    with pytest.raises(evk.EvkError, match="workspace"):
        evk.prefix_attention(q, pk, pv, k, v, o2, 64, 29, workspace=torch.empty(need - 1, dtype=torch.uint8, device=dev))
    evk.prefix_attention(q, pk, pv, k, v, o2, 64, 29, workspace=torch.full((need,), 255, dtype=torch.uint8, device=dev), stream=s.cuda_stream)
    s.synchronize()
    assert torch.equal(o, o2)


def test_python_refusals(dev):
    r = Rng(dev, 92)
    x, w = r(2, 3, 64), r(64)
    with pytest.raises(ValueError, match="contiguous"):
        evk.residual_norm(x.transpose(0, 1), x, x, x)
    with pytest.raises(ValueError, match="float16"):
        evk.residual_norm(x, x.float(), empty(dev, 2, 3, 64), empty(dev, 2, 3, 64))
    with pytest.raises(evk.EvkError, match="overlaps"):
        evk.residual_norm(x, r(2, 3, 64), x, empty(dev, 2, 3, 64), w)
    with pytest.raises(ValueError, match="16-bit"):
        evk.token_logprobs(r(3, 50), torch.zeros(3, dtype=torch.int32, device=dev), torch.zeros(3, device=dev))
    with pytest.raises(ValueError, match="3 contiguous"):
        evk.token_logprobs(r(3, 50), torch.zeros(3, dtype=torch.int16, device=dev), torch.zeros(4, device=dev))
    with pytest.raises(ValueError, match="-1"):
        evk.prefix_attention(r(1, 1, 64), r(5, 64), r(5, 64), r(1, 4, 64), r(1, 4, 64), r(1, 1, 64), 64, -1)


# ---------------------------------------------------------------------------
# past 4 GiB
# ---------------------------------------------------------------------------
def test_residual_norm_past_4_gib(dev):
    """2.3e9 values: the last rows, and the columns' sums over all of them."""
    n, d = 140_001, 16384
    assert n * d > 2 ** 31
    r = Rng(dev, 95)
    one, oney, oneh = r(1, d), r(1, d), r(1, d)
    x, y, dh = (t.expand(n, d).contiguous() for t in (one, oney, oneh))
    wi = r(d, mean=1.0)
    s, h = torch.empty_like(x), torch.empty_like(x)
    evk.residual_norm(x, y, s, h, pre_weight=wi)
    assert torch.equal(s[-1], s[0]) and torch.equal(h[-1], h[0]) and bool((h[::9973] == h[0]).all())
    dx, dy, dwi = s, h, torch.empty_like(wi)
    evk.residual_norm_backward(x, y, None, dh, dx, dy, pre_weight=wi, dpre_weight=dwi)
    assert torch.equal(dx[-1], dx[0]) and torch.equal(dy[-1], dy[0])
    X, Y = one.to(F64), oney.to(F64)
    st = X + Y / torch.sqrt(Y.square().mean() + 1e-4)
    u = st / torch.sqrt(st.square().mean() + 1e-4)
    want = n * (oneh.to(F64) * u)[0]
    size = n * (oneh.to(F64).abs() * (X.abs() + Y.abs()) / st.square().mean().sqrt())[0]
    big = want.abs() > 65504 * (1 + H)
    assert torch.isinf(dwi[big]).all()
    ok = want.abs() < 65504
    # equal terms: a run of 547 of them, then 256 / 64 + 20 runs
    assert ((dwi.to(F64) - want).abs() <= H * want.abs() + T + (2 * ROW + 600 * E) * size)[ok].all()


def test_token_logprobs_past_4_gib(dev):
    t, v = 70_001, 32000
    assert t * v > 2 ** 31
    r = Rng(dev, 96)
    some = r(7, v, std=3.0)
    x = some.repeat(t // 7 + 1, 1)[:t].contiguous()
    tok = ids16(torch.arange(t, device=dev) % 7 * 4000)
    lp, ent, stats = torch.empty(t, device=dev), torch.empty(t, device=dev), torch.empty(t, 2, device=dev)
    ids, alt = torch.empty(t, 4, dtype=torch.int16, device=dev), torch.empty(t, 4, device=dev)
    evk.token_logprobs(x, tok, lp, ent, ids, alt, stats)
    w = scores_want(some, tok[:7], 1.0, 4)
    at = torch.arange(t, device=dev) % 7
    assert ((lp - w["lp"][at]).abs() <= 1e-4).all() and torch.equal(u16(ids), w["ids"][at])
    assert torch.equal(lp, lp[:7][at]) and torch.equal(ent, ent[:7][at])
    d = torch.empty_like(x)
    evk.token_logprobs_backward(x, tok, stats, torch.ones(t, device=dev), d)
    assert torch.equal(d[-7:], d[(t - 7) % 7:(t - 7) % 7 + 7])


@pytest.mark.parametrize("b,n,h", [(2, 1, 32), (2, 30, 32), (3, 2, 16)])
def test_prefix_attention_past_4_gib(dev, b, n, h):
    """Rows of the prefix and of the caches past 2^32 bytes; the queries' largest scores lie at their ends."""
    kv, dh, p, rows = 8, 128, 2_200_000, 900_000
    assert p * kv * dh * 2 > 2 ** 32 and (b - 1) * rows * kv * dh * 2 + rows * kv * dh * 2 > 2 ** 31
    r = Rng(dev, 97)
    q = r(b, n, h * dh)
    pk, pv = torch.full((p, kv * dh), -8.0, dtype=F16, device=dev), torch.zeros(p, kv * dh, dtype=F16, device=dev)
    k, v = torch.full((b, rows, kv * dh), -8.0, dtype=F16, device=dev), torch.zeros(b, rows, kv * dh, dtype=F16, device=dev)
    q.abs_()  # scores of the rows above are far below those of the ends
    tail = 40
    pk[-tail:], pv[-tail:] = r(tail, kv * dh), r(tail, kv * dh)
    k[:, -tail:], v[:, -tail:] = r(b, tail, kv * dh), r(b, tail, kv * dh)
    o, lse = torch.empty_like(q), torch.empty(b, h, n, device=dev)
    evk.prefix_attention(q, pk, pv, k, v, o, dh, rows - n, lse=lse)
    # exp(-8 sqrt(dh) mean|q| ...) of the rest: below e^-60 of the largest, 3e6 rows of it nothing
    w = prefix_want(q, pk[-tail:], pv[-tail:], k[:, -tail:].contiguous(), v[:, -tail:].contiguous(), h, kv, dh, [tail - n] * b)
    close(o, w["o"], w["o_t"], "o")
    close(lse, w["lse"], w["lse_t"], "lse", norm=None)
