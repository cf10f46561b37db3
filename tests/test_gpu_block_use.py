"""GPU: the grouped-query block's operators as programs use them: a block's
training step and its decoding against 64 bits, streams, captured graphs, calls
at the same time, caches past 2 GiB."""
import math

import pytest
import torch

import evk_amd as evk
import test_gpu_block as gb
from test_gpu_block import F16, F32, F64, H, Rng, close, empty, seen, window_want

pytestmark = pytest.mark.gpu


class Block:
    """One grouped-query block on evk_amd's operators: weights, and the activations of a forward pass."""

    def __init__(self, dev, r, d, heads, kv, dh, f, window, sinks, act):
        self.dev, self.d, self.heads, self.kv, self.dh, self.f = dev, d, heads, kv, dh, f
        self.window, self.sinks, self.act = window, sinks, act
        wide = (heads + 2 * kv) * dh
        self.w = dict(qkv=r(d, wide, std=d ** -0.5), q=r(dh, mean=1.0, std=0.1), k=r(dh, mean=1.0, std=0.1),
                      o=r(heads * dh, d, std=(heads * dh) ** -0.5), gu=r(2, d, f, std=d ** -0.5), down=r(f, d, std=f ** -0.5))

    def forward(self, x, kc=None, vc=None, p0=0, offsets=None):
        """x (B, N, d) -> (B, N, d); rows into the caches kc, vc (B, rows, kv dh), or into tensors of their own."""
        b, n, d = x.shape
        w, e = self.w, lambda *s: torch.empty(*s, dtype=F16, device=self.dev)  # noqa: E731
        a = dict(x=x, xn=e(b, n, d), qkv=e(b, n, w["qkv"].shape[1]), q=e(b, n, self.heads * self.dh), att=e(b, n, self.heads * self.dh),
                 lse=torch.empty(b, self.heads, n, device=self.dev), y=e(b, n, d), x1=e(b, n, d), x1n=e(b, n, d), gu=e(2, b, n, self.f),
                 h=e(b, n, self.f), z=e(b, n, d), out=e(b, n, d))
        a["k"], a["v"] = (e(b, n, self.kv * self.dh), e(b, n, self.kv * self.dh)) if kc is None else (kc, vc)
        evk.rms_norm(x, a["xn"])
        evk.matmul(a["xn"], w["qkv"], a["qkv"])
        evk.qkv_norm_rope(a["qkv"], a["q"], a["k"], a["v"], self.dh, w["q"], w["k"], 1e-4, 10000.0, p0, offsets)
        evk.window_attention(a["q"], a["k"], a["v"], a["att"], self.dh, self.window, self.sinks, p0, offsets, a["lse"])
        evk.matmul(a["att"], w["o"], a["y"])
        evk.add(x, a["y"], a["x1"])
        evk.rms_norm(a["x1"], a["x1n"])
        evk.gated_linear(a["x1n"], w["gu"], a["h"], a["gu"], self.act)
        evk.matmul(a["h"], w["down"], a["z"])
        evk.add(a["x1"], a["z"], a["out"])
        return a

    def backward(self, a, dout):
        """Gradients of x and of every weight."""
        w, like = self.w, torch.empty_like
        b, n, d = dout.shape
        flat = lambda t: t.view(b * n, -1)  # noqa: E731
        g = {k: like(v) for k, v in w.items()}
        dh, dx1n, datt, dxn, dqkv = like(a["h"]), like(a["x1n"]), like(a["att"]), like(a["xn"]), like(a["qkv"])
        dq, dk, dv = like(a["q"]), like(a["k"]), like(a["v"])
        evk.matmul(flat(a["h"]), flat(dout), g["down"], transpose_a=True)
        evk.matmul(flat(dout), w["down"], flat(dh), transpose_b=True)
        evk.gated_linear_backward(a["x1n"], w["gu"], a["gu"], dh, dx1n, g["gu"], self.act)
        dx1 = dout.clone()
        evk.rms_norm_backward(a["x1"], dx1n, dx1)  # adds to the residual's gradient
        evk.matmul(flat(a["att"]), flat(dx1), g["o"], transpose_a=True)
        evk.matmul(flat(dx1), w["o"], flat(datt), transpose_b=True)
        evk.window_attention_bwd(a["q"], a["k"], a["v"], a["att"], datt, dq, dk, dv, a["lse"], self.dh, self.window, self.sinks)
        evk.qkv_norm_rope_backward(a["qkv"], dq, dk, dv, dqkv, self.dh, w["q"], w["k"], g["q"], g["k"])
        evk.matmul(flat(a["xn"]), flat(dqkv), g["qkv"], transpose_a=True)
        evk.matmul(flat(dqkv), w["qkv"], flat(dxn), transpose_b=True)
        dx = dx1.clone()
        evk.rms_norm_backward(a["x"], dxn, dx)
        return dx, g

    def exact(self, x, w):
        """The block in 64 bits on tensors that autograd follows."""
        b, n, d = x.shape
        norm = lambda t: t / torch.sqrt(t.square().mean(-1, keepdim=True) + 1e-4)  # noqa: E731
        hq = self.heads * self.dh
        qkv = norm(x).reshape(b * n, d) @ w["qkv"]
        heads = qkv.view(b, n, self.heads + 2 * self.kv, self.dh)
        ang = torch.arange(n, device=self.dev, dtype=F64)[:, None, None] * 10000.0 ** (-torch.arange(0, self.dh, 2, device=self.dev, dtype=F64) / self.dh)
        c, s = torch.cos(ang), torch.sin(ang)

        def turned(t):
            p, q = t[..., 0::2], t[..., 1::2]
            return torch.stack([p * c - q * s, p * s + q * c], -1).flatten(-2)

        q = turned(norm(heads[:, :, :self.heads]) * w["q"])
        k = turned(norm(heads[:, :, self.heads:self.heads + self.kv]) * w["k"])
        v = heads[:, :, self.heads + self.kv:]
        m = seen(torch.arange(n, device=self.dev), n, self.window, self.sinks)
        att = []
        for i in range(b):
            for hd in range(self.heads):
                to = hd // (self.heads // self.kv)
                sc = (q[i, :, hd] @ k[i, :, to].t() * self.dh ** -0.5).masked_fill(~m, -math.inf)
                att.append(torch.softmax(sc, 1) @ v[i, :, to])
        att = torch.stack(att).view(b, self.heads, n, self.dh).transpose(1, 2).reshape(b * n, hq)
        x1 = x + (att @ w["o"]).view(b, n, d)
        xn = norm(x1).reshape(b * n, d)
        g, u = xn @ w["gu"][0], xn @ w["gu"][1]
        h = (torch.nn.functional.silu(g) if self.act == "silu" else g * torch.sigmoid(2 * math.sqrt(2 / math.pi) * (g + 0.044715 * g ** 3))) * u
        return x1 + (h @ w["down"]).view(b, n, d)


def rel(got, want):
    return float((got.to(F64) - want).norm() / want.norm())


@pytest.mark.parametrize("b,n,d,heads,kv,dh,f,window,sinks,act", [(2, 150, 256, 8, 2, 32, 384, 40, 4, "silu"), (1, 97, 200, 3, 1, 64, 136, 0, 0, "gelu"),
                                                                  (2, 260, 384, 6, 6, 64, 512, 64, 1, "silu")])
def test_block_training_step(dev, b, n, d, heads, kv, dh, f, window, sinks, act):
    """A block forward and backward.  Every gradient has at most about 30 roundings to fp16 behind it, each off by at most
    H of its tensor's norm; added in quadrature 5.5 H, and the softmax and the norms pass on at most three times as much."""
    r = Rng(dev, 60 + n)
    blk = Block(dev, r, d, heads, kv, dh, f, window, sinks, act)
    x, dout = r(b, n, d), r(b, n, d)
    a = blk.forward(x)
    dx, g = blk.backward(a, dout)
    x64 = x.to(F64).requires_grad_(True)
    w64 = {k: t.to(F64).requires_grad_(True) for k, t in blk.w.items()}
    out = blk.exact(x64, w64)
    want = torch.autograd.grad(out, [x64, *w64.values()], dout.to(F64))
    assert rel(a["out"], out.detach()) <= 16 * H
    assert rel(dx, want[0]) <= 16 * H
    for k, t in zip(w64, want[1:]):
        assert rel(g[k], t) <= 16 * H, k


def test_block_decodes_what_it_computes_at_once(dev):
    """A prompt in two chunks and then single tokens, each sequence at its own length, against the whole sequence."""
    b, n, rows = 3, 90, 120
    r = Rng(dev, 71)
    blk = Block(dev, r, 192, 6, 2, 32, 256, 24, 3, "silu")
    x = r(b, n, 192)
    whole = blk.forward(x)["out"]
    lengths = [50, 64, 80]
    kc, vc = (torch.full((b, rows, 2 * 32), math.nan, dtype=F16, device=dev) for _ in range(2))
    for i, m in enumerate(lengths):
        k1, v1 = kc[i:i + 1], vc[i:i + 1]
        first = blk.forward(x[i:i + 1, :31].contiguous(), k1, v1)["out"]
        second = blk.forward(x[i:i + 1, 31:m].contiguous(), k1, v1, p0=31)["out"]
        # the same sums in another order and with other roundings of P: sqrt(2 * 30) H at most of the norm
        assert rel(torch.cat([first, second], 1), whole[i:i + 1, :m].to(F64)) <= 8 * H
    for step in range(10):
        at = torch.tensor([m + step for m in lengths], dtype=torch.int32, device=dev)
        tok = torch.stack([x[i, int(at[i])] for i in range(b)])[:, None]
        out = blk.forward(tok.contiguous(), kc, vc, offsets=at)["out"]
        want = torch.stack([whole[i, int(at[i])] for i in range(b)])[:, None]
        assert rel(out, want.to(F64)) <= 8 * H, step
    assert torch.isnan(kc[0, 60:]).all() and not torch.isnan(kc[0, :60]).any()


def steps(dev):
    """Calls of every entry point on static tensors: [(name, inputs, outputs, call)]."""
    r = Rng(dev, 81)
    b, n, h, kv, dh, rows, f = 2, 130, 4, 2, 64, 2100, 256
    wide = (h + 2 * kv) * dh
    qkv, wq, wk = r(b, n, wide), r(dh, mean=1.0), r(dh, mean=1.0)
    q, k, v = empty(dev, b, n, h * dh), empty(dev, b, n, kv * dh), empty(dev, b, n, kv * dh)
    o, lse, do = empty(dev, b, n, h * dh), torch.zeros(b, h, n, device=dev), r(b, n, h * dh)
    dq, dk, dv = empty(dev, b, n, h * dh), empty(dev, b, n, kv * dh), empty(dev, b, n, kv * dh)
    dqkv, dwq, dwk = empty(dev, b, n, wide), empty(dev, dh), empty(dev, dh)
    kc, vc, q1, o1 = r(1, rows, kv * dh), r(1, rows, kv * dh), r(1, 1, h * dh), empty(dev, 1, 1, h * dh)
    off = torch.tensor([rows - 1], dtype=torch.int32, device=dev)
    x, w, hh, gu = r(70, 128), r(2, 128, f, std=0.1), empty(dev, 70, f), empty(dev, 2, 70, f)
    x1, h1 = r(3, 128), empty(dev, 3, f)
    dh_, dx, dw = r(70, f), empty(dev, 70, 128), empty(dev, 2, 128, f)

    def call():
        evk.qkv_norm_rope(qkv, q, k, v, dh, wq, wk)
        evk.window_attention(q, k, v, o, dh, 40, 3, lse=lse)
        evk.window_attention_bwd(q, k, v, o, do, dq, dk, dv, lse, dh, 40, 3)
        evk.qkv_norm_rope_backward(qkv, dq, dk, dv, dqkv, dh, wq, wk, dwq, dwk)
        evk.window_attention(q1, kc, vc, o1, dh, 0, 0, 0, off)  # split over workgroups
        evk.gated_linear(x, w, hh, gu)
        evk.gated_linear_backward(x, w, gu, dh_, dx, dw)
        evk.gated_linear(x1, w, h1)

    ins = [qkv, do, kc, vc, q1, x, w, dh_, x1]
    outs = [q, k, v, o, lse, dq, dk, dv, dqkv, dwq, dwk, o1, hh, gu, dx, dw, h1]
    assert evk.window_attention_workspace(q1, kc, dh) > 0
    return ins, outs, call


def test_other_stream(dev):
    ins, outs, call = steps(dev)
    call()
    torch.cuda.synchronize()
    want = [t.clone() for t in outs]
    for t in outs:
        t.fill_(9.0)
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
                t.fill_(3.0)
            junk = torch.full((1 << 20,), math.nan, device=dev)  # what a released workspace would be taken by
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
    q, kc, vc = r(1, 1, 256), r(1, 5000, 128), r(1, 5000, 128)
    o, o2 = torch.empty_like(q), torch.empty_like(q)
    evk.window_attention(q, kc, vc, o, 64, 0, 0, 4999)
    need = evk.window_attention_workspace(q, kc, 64)
    s = torch.cuda.Stream()
    torch.cuda.synchronize()
    with pytest.raises(ValueError, match="workspace"):
        evk.window_attention(q, kc, vc, o2, 64, 0, 0, 4999, stream=s.cuda_stream)
    with pytest.raises(evk.EvkError, match="workspace"):
        evk.window_attention(q, kc, vc, o2, 64, 0, 0, 4999, workspace=torch.empty(need - 1, dtype=torch.uint8, device=dev))
    evk.window_attention(q, kc, vc, o2, 64, 0, 0, 4999, workspace=torch.full((need,), 255, dtype=torch.uint8, device=dev), stream=s.cuda_stream)
    s.synchronize()
    assert torch.equal(o, o2)


@pytest.mark.parametrize("n,sinks", [(1, 4), (1, 0), (20, 70), (600, 70), (600, 64), (600, 0)])
def test_cache_past_2_gib(dev, n, sinks):
    """One sequence whose rows of K pass 2 GiB, queries at its end: the sinks and the window lie that far apart."""
    h, kv, dh, window, rows = 32, 8, 128, 200, 1_100_000
    tail = n + window
    assert rows * kv * dh * 2 > 2 ** 31
    r = Rng(dev, 95)
    q = r(1, n, h * dh)
    k, v = (torch.empty(1, rows, kv * dh, dtype=F16, device=dev) for _ in range(2))
    for t in (k, v):
        t[:, sinks:rows - tail] = math.nan  # seen by nobody
        t[:, :sinks], t[:, rows - tail:] = r(1, sinks, kv * dh), r(1, tail, kv * dh)
    o, lse = torch.empty_like(q), torch.empty(1, h, n, device=dev)
    evk.window_attention(q, k, v, o, dh, window, sinks, rows - n, lse=lse)
    # the rows that count, and positions moved down with them
    kk, vv = (torch.cat([t[:, :sinks], t[:, rows - tail:]], 1) for t in (k, v))
    w = window_want(q, kk, vv, h, kv, dh, [sinks + window], window, sinks)
    close(o, w["o"], w["o_t"], "o")
    close(lse, w["lse"], w["lse_t"], "lse", norm=None)


def test_rows_into_a_cache_past_4_gib(dev):
    """Cache rows whose elements lie past 2^32 bytes."""
    b, n, kv, dh, rows = 2, 3, 8, 128, 1_200_000
    r = Rng(dev, 96)
    qkv = r(b, n, 3 * kv * dh)
    q = empty(dev, b, n, kv * dh)
    k, v = (torch.zeros(b, rows, kv * dh, dtype=F16, device=dev) for _ in range(2))
    assert k.numel() * 2 > 2 ** 32
    off = torch.tensor([5, rows - n], dtype=torch.int32, device=dev)
    evk.qkv_norm_rope(qkv, q, k, v, dh, offsets=off)
    for s in range(b):
        at = int(off[s])
        assert torch.equal(v[s, at:at + n], qkv[s, :, 2 * kv * dh:])
        assert (k[s, at:at + n] != 0).any(1).all()
        assert int((k[s] != 0).any(1).sum()) == n and int((v[s] != 0).any(1).sum()) == n


@pytest.mark.parametrize("size", [2.0 ** -13, 2.0 ** -6, 4000.0])
@pytest.mark.parametrize("dh,h,kv,n,window", [(64, 4, 2, 300, 100), (128, 4, 1, 200, 0), (40, 2, 2, 150, 0), (256, 2, 1, 130, 50)])
def test_window_attention_bwd_gradient_sizes(dev, dh, h, kv, n, window, size):
    """Output gradients as small as those of a mean over a batch, and as large as loss scaling makes them: the scores'
    gradients pass fp16 on their way into the products, and must neither vanish nor overflow there."""
    g = torch.Generator(device=dev).manual_seed(dh)
    rnd = lambda std, heads: torch.empty(1, n, heads * dh, dtype=F16, device=dev).normal_(0, std, generator=g)
    q, k, v, do = rnd(0.25, h), rnd(0.25, kv), rnd(1.0, kv), rnd(size, h)
    o, lse = torch.empty_like(q), torch.empty(1, h, n, dtype=F32, device=dev)
    evk.window_attention(q, k, v, o, dh, window, 3, lse=lse)
    got = [torch.empty_like(t) for t in (q, k, v)]
    evk.window_attention_bwd(q, k, v, o, do, *got, lse, dh, window, 3)

    heads = lambda t, m: t.view(n, m, dh).transpose(0, 1).double()
    Q, K, V, G = heads(q, h), heads(k, kv).repeat_interleave(h // kv, 0), heads(v, kv).repeat_interleave(h // kv, 0), heads(do, h)
    i, j = torch.arange(n, device=dev)[:, None], torch.arange(n, device=dev)[None]
    see = (j <= i) & ((j > i - (window or n)) | (j < 3))
    P = torch.softmax((Q @ K.transpose(1, 2) / dh ** 0.5).masked_fill(~see, -torch.inf), -1)
    dP = G @ V.transpose(1, 2)
    # D from the rounded output, as the operator takes it
    dS = P * (dP - (G * heads(o, h)).sum(-1, keepdim=True)) / dh ** 0.5
    share = lambda t: t.view(kv, h // kv, n, dh).sum(1)
    want = [dS @ K, share(dS.transpose(1, 2) @ Q), share(P.transpose(1, 2) @ G)]
    for what, a, w in zip(("dQ", "dK", "dV"), got, want):
        a = heads(a, a.shape[2] // dh)
        assert torch.isfinite(a).all(), what
        # roundings of P or dS and of the result (each at most half a step of the norm), the result's subnormals, and P's
        # (products in fp16 of probabilities below 2^-14, off by 2^-25 each, at most the norm of G's columns)
        tol = 2 * 2.0 ** -11 * w.norm() + 2.0 ** -25 * w.numel() ** 0.5
        if what == "dV":
            tol = tol + 2.0 ** -25 * n ** 0.5 * (h // kv) * G.norm()
        assert (a - w).norm() <= tol, f"{what}: off by {float((a - w).norm() / w.norm()):.3g} of the norm, {float(tol / w.norm()):.3g} allowed"


WIDE = [  # b, n, heads, kv: workgroups of 64 rows (a few to every compute unit), and of 128 where there are more
    (2, 300, 16, 8), (1, 1100, 12, 4), (8, 300, 16, 16), (3, 701, 24, 8),
]


@pytest.mark.parametrize("dh", [32, 40, 64, 96, 128, 256])
@pytest.mark.parametrize("b,n,h,kv", WIDE)
def test_window_attention_many_rows(dev, b, n, h, kv, dh):
    """Grids of hundreds of workgroups, forward and backward, with rows that some query of a tile does not see at both
    ends of its list; a chunk of a longer sequence in the forward."""
    gb.test_window_attention(dev, b, n, h, kv, dh, n, 0, 100, 5, False)
    gb.test_window_attention(dev, b, n, h, kv, dh, n + 90, 77, 0, 0, False)
    gb.test_window_attention_bwd(dev, b, n, h, kv, dh, n, 0, 100, 5, False)


@pytest.mark.parametrize("dh,h,kv,n", [(128, 4, 2, 150), (64, 2, 2, 2000), (256, 1, 1, 70)])
def test_window_attention_bwd_large_values(dev, dh, h, kv, n):
    """Values near fp16's largest, and output gradients that point along them: the scores' gradients pass 65504 though no
    gradient that is asked for does."""
    r = Rng(dev, dh)
    q, k = r(1, n, h * dh, std=0.02), r(1, n, kv * dh, std=0.02)
    v = r(1, n, kv * dh, std=40000.0).clamp_(-60000, 60000)
    do = v.view(1, n, kv, 1, dh).expand(1, n, kv, h // kv, dh).float()
    do = (do / do.norm(dim=-1, keepdim=True)).reshape(1, n, h * dh).half()
    got = gb.window_grads(q, k, v, do, dh, h, 2, 0)
    w = window_want(q, k, v, h, kv, dh, [0], 2, 0, do)
    P = 0.5  # two rows of nearly equal scores
    assert float((do.view(n, h, dh).double() * v.view(n, kv, 1, dh).expand(n, kv, h // kv, dh).reshape(n, h, dh).double()).sum(-1).max()) * P * P > 65504
    for g, x in zip(got, ("dq", "dk", "dv")):
        close(g, w[x], w[x + "_t"], x, norm=None)


def test_window_attention_bwd_millions_of_positions(dev):
    """Enough key blocks that the number of their parts, summed, passes 32 bits; the sinks' blocks are joined from parts."""
    n, dh, window, sinks = 3_200_000, 8, 64, 200
    r = Rng(dev, 5)
    q, k, v, do = (r(1, n, dh) for _ in range(4))
    o, lse = torch.empty_like(q), torch.empty(1, 1, n, device=dev)
    evk.window_attention(q, k, v, o, dh, window, sinks, lse=lse)
    dq, dk, dv = (empty(dev, 1, n, dh) for _ in range(3))
    evk.window_attention_bwd(q, k, v, o, do, dq, dk, dv, lse, dh, window, sinks)
    Q, K, V, G, O = (t[0].double() for t in (q, k, v, do, o))  # noqa: E741
    D = (G * O).sum(1)
    for j in (0, 63, 64, 130, 199, 200, 255, 1_500_000, n - 65, n - 1):
        first, last = j, n if j < sinks else min(n, j + window)
        s = Q[first:last] @ K[j] * dh ** -0.5
        p = torch.exp(s - lse[0, 0, first:last].double())
        ds = p * (G[first:last] @ V[j] - D[first:last]) * dh ** -0.5
        for what, g, want, mag in (("dk", dk[0, j], ds @ Q[first:last], (ds.abs() @ Q[first:last].abs())),
                                   ("dv", dv[0, j], p @ G[first:last], (p.abs() @ G[first:last].abs()))):
            # P and dS rounded, their exponent's and the sums' errors in 32 bits (a part adds a few hundred thousand
            # rows, 32 by 32, in order: the error of a term is at most half a step of the sum so far), the result's
            terms = last - first
            tol = (H + 2.0 ** -18 + (terms / 32 + 100) * gb.E) * mag + H * want.abs() + gb.T * (1 + terms * 2.0 ** -10)
            assert ((g.double() - want).abs() <= tol).all(), (what, j, g, want, tol)


def test_empty_cache(dev):
    """No row in the cache: nothing is written, nothing is seen."""
    b, n, h, kv, dh = 2, 3, 4, 2, 64
    r = Rng(dev, 1)
    off = torch.zeros(b, dtype=torch.int32, device=dev)
    x, q = r(b, n, (h + 2 * kv) * dh), empty(dev, b, n, h * dh)
    k, v = torch.empty(b, 0, kv * dh, dtype=F16, device=dev), torch.empty(b, 0, kv * dh, dtype=F16, device=dev)
    evk.qkv_norm_rope(x, q, k, v, dh, offsets=off)
    o, lse = empty(dev, b, n, h * dh), torch.zeros(b, h, n, device=dev)
    evk.window_attention(q, k, v, o, dh, 4, 1, offsets=off, lse=lse)
    assert (o == 0).all() and (lse == -math.inf).all()
    assert torch.isfinite(q).all() and (q != 7.0).any()
