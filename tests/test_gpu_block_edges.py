"""GPU: the grouped-query block's operators at the ends of their ranges: positions
next to 2^31, scores that are all -inf, NaN and infinities beside finite rows, long
contexts, gradients of every size.  Tolerances as in test_gpu_block.py: H is half
a step of fp16, T of its subnormals, E of 32 bits."""
import math

import pytest
import torch

import evk_amd as evk
from test_gpu_block import E, F16, F64, H, T, Rng, act64, close, empty, rope_want, seen, window_want

pytestmark = pytest.mark.gpu


# ---------------------------------------------------------------------------
# positions up to 2^31 and past it (offsets[b] + t)
# ---------------------------------------------------------------------------
def test_qkv_norm_rope_far_positions(dev):
    """Queries behind a position of 2^31 turn by their own angle, not by that of 2^31 - 1."""
    b, n, h, kv, dh, rows = 3, 4, 2, 1, 64, 8
    r = Rng(dev, 21)
    qkv, wq, wk = r(b, n, (h + 2 * kv) * dh), r(dh, mean=1.0), r(dh, mean=1.0)
    off = torch.tensor([2 ** 31 - 2, 2 ** 31 - 1, -2], dtype=torch.int32, device=dev)
    q, k, v = empty(dev, b, n, h * dh), empty(dev, b, rows, kv * dh), empty(dev, b, rows, kv * dh)
    evk.qkv_norm_rope(qkv, q, k, v, dh, wq, wk, 1e-4, 500.0, 0, off)
    y, _, size = rope_want(qkv, wq, wk, h, kv, dh, off.long()[:, None] + torch.arange(n, device=dev), 1e-4, 500.0)
    # beside the dozen roundings of 2^-24: angles of 2^31 off by 2^-53 of themselves, 2^-22, six times here and twice in the
    # formula in 64 bits
    close(q.view(b, n, h, dh), y[:, :, :h], H * y[:, :, :h].abs() + (2.0 ** -20 + 8 * 2.0 ** -22) * size[:, :, :h] + T, "q")
    assert (k[:2] == 7.0).all() and (v[:2] == 7.0).all(), "rows that the cache does not have"


@pytest.mark.parametrize("dh,h,kv", [(64, 4, 2), (128, 4, 1), (256, 2, 1), (33, 2, 1)])
@pytest.mark.parametrize("n,rows", [(1, 40), (3, 700), (70, 90)])
@pytest.mark.parametrize("window,sinks", [(0, 0), (0, 3), (2 ** 31 - 5, 0), (2 ** 31 + 1, 2), (2 ** 32 - 1, 0), (50, 2)])
def test_window_attention_far_positions(dev, dh, h, kv, n, rows, window, sinks):
    """Positions next to 2^31 and past it: no window shows every row, a window as long as that cuts where it should."""
    b = 3
    r = Rng(dev, 22 + dh + n)
    q, k, v = r(b, n, h * dh), r(b, rows, kv * dh), r(b, rows, kv * dh)
    off = torch.tensor([2 ** 31 - 1, 2 ** 31 - 2 - n // 2, rows - n], dtype=torch.int32, device=dev)
    o, lse = empty(dev, b, n, h * dh), torch.full((b, h, n), 7.0, device=dev)
    evk.window_attention(q, k, v, o, dh, window, sinks, 0, off, lse)
    w = window_want(q, k, v, h, kv, dh, off.tolist(), window, sinks)
    none = torch.isinf(w["lse"])
    close(o, w["o"], w["o_t"], "o")
    close(lse, w["lse"], torch.where(none, torch.zeros_like(w["lse"]), w["lse_t"]), "lse", norm=None)


# ---------------------------------------------------------------------------
# scores of -inf
# ---------------------------------------------------------------------------
def plain_want(q, k, v, h, kv, dh, p0, window, sinks):
    """o and lse by the definition in 64 bits, whatever visible rows hold (hidden rows of v have to be finite)."""
    b, n, _ = q.shape
    o, lse = [], []
    for s in range(b):
        m = seen(p0 + torch.arange(n, device=q.device), k.shape[1], window, sinks)
        for hd in range(h):
            at, to = slice(hd * dh, hd * dh + dh), slice(hd // (h // kv) * dh, hd // (h // kv) * dh + dh)
            sc = torch.where(m, q[s, :, at].to(F64) @ k[s, :, to].to(F64).t() * dh ** -0.5, torch.full((), -math.inf, dtype=F64, device=q.device))
            o.append(torch.softmax(sc, 1) @ v[s, :, to].to(F64))
            lse.append(torch.logsumexp(sc, 1))
    return torch.stack(o).view(b, h, n, dh).transpose(1, 2).reshape(b, n, h * dh), torch.stack(lse).view(b, h, n)


HEADS = [(64, 4, 2), (128, 4, 1), (256, 2, 1), (80, 2, 2), (33, 2, 1)]


@pytest.mark.parametrize("dh,h,kv", HEADS)
@pytest.mark.parametrize("b,n,rows,p0,window", [(1, 1, 1, 0, 0), (2, 1, 30, 20, 1), (1, 20, 20, 0, 1), (1, 150, 150, 0, 70), (9, 300, 300, 0, 70),
                                               (1, 1, 20000, 19999, 0), (1, 2, 20000, 19990, 0)])
def test_window_attention_scores_of_minus_infinity(dev, dh, h, kv, b, n, rows, p0, window):
    """K that overflowed in its leading rows: a query that sees no other row has no softmax (NaN, log-sum-exp -inf), one
    that sees a finite score too has that of the finite ones."""
    r = Rng(dev, 30 + dh)
    q, k, v = r(b, n, h * dh), r(b, rows, kv * dh), r(b, rows, kv * dh)
    q.view(b, n, h, dh)[..., 0] = 1.0
    for lead in sorted({min(rows, 80), rows - 3, rows} - {0}):
        if lead <= 0:
            continue
        kk = k.clone()
        kk.view(b, rows, kv, dh)[:, :lead, :, 0] = -math.inf
        o, lse = empty(dev, b, n, h * dh), torch.full((b, h, n), 7.0, device=dev)
        evk.window_attention(q, kk, v, o, dh, window, 0, p0, lse=lse)
        ow, lw = plain_want(q, kk, v, h, kv, dh, p0, window, 0)
        # what remains is the softmax of the finite rows, with the roundings of any other
        t = window_want(q, k, v, h, kv, dh, [p0] * b, window, 0)
        few = 2 * (2 * H + 2.0 ** -16) * v.abs().max().to(F64)  # as o_t, whatever weights the finite rows have
        close(o, ow, t["o_t"] + few, f"o, {lead} rows", norm=None)
        close(lse, lw, t["lse_t"] + 2.0 ** -19, f"lse, {lead} rows", norm=None)
        sees = seen(p0 + torch.arange(n, device=dev), rows, window, 0)
        dead = ~sees[:, lead:].any(1)
        assert torch.isnan(o[:, dead]).all() and torch.isfinite(o[:, ~dead]).all()


@pytest.mark.parametrize("dh,h,kv", HEADS)
def test_window_attention_bwd_scores_of_minus_infinity(dev, dh, h, kv):
    """The gradients of a query without a softmax are NaN; rows that no such query sees keep theirs."""
    b, n, window = 1, 200, 20
    r = Rng(dev, 33 + dh)
    q, k, v, do = r(b, n, h * dh), r(b, n, kv * dh), r(b, n, kv * dh), r(b, n, h * dh)
    q.view(b, n, h, dh)[..., 0] = 1.0
    k.view(b, n, kv, dh)[:, :40, :, 0] = -math.inf
    o, lse = torch.empty_like(q), torch.empty(b, h, n, device=dev)
    evk.window_attention(q, k, v, o, dh, window, 0, lse=lse)
    dq, dk, dv = (torch.empty_like(t) for t in (q, k, v))
    evk.window_attention_bwd(q, k, v, o, do, dq, dk, dv, lse, dh, window, 0)
    assert torch.isnan(dq[:, :40]).all()
    far = 40 + window  # queries from here on see finite rows only
    assert torch.isnan(dk[:, :40]).any(-1).all() and torch.isnan(dv[:, :40]).any(-1).all()
    fin = k.clone()
    fin.view(b, n, kv, dh)[:, :40, :, 0] = -100.0
    w = window_want(q, fin, v, h, kv, dh, [0], window, 0, do)
    close(dq[:, far:], w["dq"][:, far:], w["dq_t"][:, far:], "dq")
    for g, x in ((dk, "dk"), (dv, "dv")):
        close(g[:, far:], w[x][:, far:], w[x + "_t"][:, far:], x)


# ---------------------------------------------------------------------------
# long contexts: probabilities of 2^-16 and less, and gradients of very different sizes
# ---------------------------------------------------------------------------
def bwd64(q, k, v, o, do, h, dh, window=0, chunk=4096):
    """Gradients of one sequence with one key head in 64 bits, a chunk of queries at a time; D from the forward's rounded
    o, as the operator takes it."""
    n = q.shape[1]
    K, V = k[0].to(F64), v[0].to(F64)
    dq, dk, dv = [], torch.zeros_like(K), torch.zeros_like(V)
    for t0 in range(0, n, chunk):
        t1 = min(n, t0 + chunk)
        j0 = max(0, t0 - window + 1) if window else 0
        p, j = torch.arange(t0, t1, device=q.device)[:, None], torch.arange(j0, t1, device=q.device)[None]
        m = (j <= p) & (j > p - window) if window else j <= p
        row = []
        for hd in range(h):
            Q, G, O = (x[0, t0:t1, hd * dh:hd * dh + dh].to(F64) for x in (q, do, o))  # noqa: E741
            P = torch.softmax((Q @ K[j0:t1].t() * dh ** -0.5).masked_fill(~m, -math.inf), 1)
            dS = P * (G @ V[j0:t1].t() - (G * O).sum(1, keepdim=True)) * dh ** -0.5
            row.append(dS @ K[j0:t1])
            dk[j0:t1] += dS.t() @ Q
            dv[j0:t1] += P.t() @ G
        dq.append(torch.cat(row, 1))
    return torch.cat(dq)[None], dk[None], dv[None]


def grads(q, k, v, do, dh, h, window):
    o, lse = torch.empty_like(q), torch.empty(1, h, q.shape[1], device=q.device)
    evk.window_attention(q, k, v, o, dh, window, 0, lse=lse)
    out = [torch.empty_like(t) for t in (q, k, v)]
    evk.window_attention_bwd(q, k, v, o, do, *out, lse, dh, window, 0)
    return o, out


@pytest.mark.parametrize("n,h,dh,size", [(65536, 1, 128, 1.0), (65536, 2, 64, 1.0), (131072, 1, 64, 4000.0), (65536, 1, 64, 2.0 ** -10), (40000, 1, 256, 1.0)])
def test_window_attention_bwd_long_context(dev, n, h, dh, size):
    """Nearly flat attention over all of a long context: P and dS of 1 / n keep the bits that fp16 has."""
    r = Rng(dev, 60)
    q, k, v, do = r(1, n, h * dh, std=0.3), r(1, n, dh), r(1, n, dh), r(1, n, h * dh, std=size)
    o, got = grads(q, k, v, do, dh, h, 0)
    want = bwd64(q, k, v, o, do, h, dh)
    for what, g, w in zip(("dq", "dk", "dv"), got, want):
        g = g.to(F64)
        for part in (slice(0, n // 8), slice(n // 8, n // 2), slice(n // 2, n - 2048), slice(n - 2048, n)):
            a, b = g[:, part], w[:, part]
            # 2 H for the roundings of P or dS, of O in D and of the result, and the result's own subnormals
            tol = 2 * H * b.norm() + T * b.numel() ** 0.5
            assert (a - b).norm() <= tol, f"{what} {part}: off by {float((a - b).norm() / b.norm() / H):.2f} H of the norm"


@pytest.mark.parametrize("dh,h,n,window", [(128, 2, 4096, 512), (64, 1, 6000, 0), (40, 3, 3000, 256), (256, 1, 2000, 300)])
def test_window_attention_bwd_gradients_of_two_sizes(dev, dh, h, n, window):
    """Short output gradients (2^-12 of the long ones) in the same parts of a key block's queries: the gradients that they
    alone make keep their bits."""
    r = Rng(dev, 65)
    q, k, v, do = r(1, n, h * dh, std=0.3), r(1, n, dh), r(1, n, dh), r(1, n, h * dh)
    short = torch.arange(n, device=dev) >= n // 2 + 37
    do[:, ~short] *= 256.0
    do[:, short] *= 2.0 ** -4
    o, got = grads(q, k, v, do, dh, h, window)
    want = bwd64(q, k, v, o, do, h, dh, window)
    for what, g, w in zip(("dq", "dk", "dv"), got, want):
        for part in (~short, short):  # keys from there on are seen by the short ones alone
            a, b = g[:, part].to(F64), w[:, part]
            tol = 2 * H * b.norm() + T * b.numel() ** 0.5
            assert (a - b).norm() <= tol, f"{what}: off by {float((a - b).norm() / b.norm() / H):.2f} H of the norm"


# ---------------------------------------------------------------------------
# NaN and infinities beside finite rows
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("dh,h,kv", HEADS)
@pytest.mark.parametrize("what", ["q", "k", "v", "do"])
@pytest.mark.parametrize("b,n,window,sinks", [(1, 300, 40, 3), (3, 700, 90, 0), (1, 333, 0, 0)])
@pytest.mark.parametrize("value", [math.inf, math.nan])
def test_window_attention_bwd_single_wild_rows(dev, dh, h, kv, what, b, n, window, sinks, value):
    """One row of q, k, v or dO that is not finite, in the middle: outputs and gradients that it takes no part in are those
    without it, the others say so."""
    at = n // 2 + 5
    r = Rng(dev, 40 + dh + n)
    t = dict(q=r(b, n, h * dh), k=r(b, n, kv * dh), v=r(b, n, kv * dh), do=r(b, n, h * dh))
    w = window_want(t["q"], t["k"], t["v"], h, kv, dh, [0] * b, window, sinks, t["do"])
    t[what][0, at] = value
    q, k, v, do = t["q"], t["k"], t["v"], t["do"]
    o, lse = torch.empty_like(q), torch.empty(b, h, n, device=dev)
    evk.window_attention(q, k, v, o, dh, window, sinks, lse=lse)
    dq, dk, dv = (torch.empty_like(x) for x in (q, k, v))
    evk.window_attention_bwd(q, k, v, o, do, dq, dk, dv, lse, dh, window, sinks)
    m = seen(torch.arange(n, device=dev), n, window, sinks)
    rows = torch.zeros(b, n, dtype=torch.bool, device=dev)  # queries whose gradient is touched
    rows[0] = m[:, at] if what in "kv" else torch.arange(n, device=dev) == at
    keys = torch.zeros(b, n, dtype=torch.bool, device=dev)  # keys that such a query sees
    keys[0] = (m & rows[0][:, None]).any(0)
    outs = rows if what != "do" else torch.zeros_like(rows)
    close(o[~outs], w["o"][~outs], w["o_t"][~outs], "o")
    if outs.any():
        assert not torch.isfinite(o[outs].float()).all(-1).any()
    close(dq[~rows], w["dq"][~rows], w["dq_t"][~rows], "dq", norm=4 * H)
    assert not torch.isfinite(dq[rows].float()).all(-1).any(), "dq"
    for g, x in ((dk, "dk"), (dv, "dv")):
        close(g[~keys], w[x][~keys], w[x + "_t"][~keys], x, norm=4 * H)
        if not (what in "kv" and x == "dv"):  # P of a row that overflowed may be 0 for the others
            assert not torch.isfinite(g[keys].float()).all(-1).any(), x


@pytest.mark.parametrize("dh,h,kv", HEADS)
@pytest.mark.parametrize("b,n,window,sinks", [(1, 40, 9, 0), (1, 300, 40, 3), (5, 700, 90, 0), (1, 333, 0, 0)])
@pytest.mark.parametrize("value", [math.inf, -math.inf, math.nan])
def test_window_attention_single_wild_values(dev, dh, h, kv, b, n, window, sinks, value):
    """One value of v, one of dO: the other columns of o and of dV are those without it, for queries and keys that take part
    in the row and for those that do not; its own column says so where the row is seen, and only there."""
    at, col, hd = n // 2 + 3, dh // 2 + 1, h - 1
    c = hd // (h // kv)
    r = Rng(dev, 90 + dh + n)
    q, k, v, do = r(b, n, h * dh), r(b, n, kv * dh), r(b, n, kv * dh), r(b, n, h * dh)
    w = window_want(q, k, v, h, kv, dh, [0] * b, window, sinks, do)
    m = seen(torch.arange(n, device=dev), n, window, sinks)
    v2 = v.clone()
    v2[0, at, c * dh + col] = value
    o, lse = torch.empty_like(q), torch.empty(b, h, n, device=dev)
    evk.window_attention(q, k, v2, o, dh, window, sinks, lse=lse)
    hit = torch.zeros(b, n, h, dh, dtype=torch.bool, device=dev)
    hit[0, m[:, at], c * (h // kv):(c + 1) * (h // kv), col] = True
    hit = hit.view(b, n, h * dh)
    close(o[~hit], w["o"][~hit], w["o_t"][~hit], "o")
    assert not torch.isfinite(o[hit].float()).any()
    close(lse, w["lse"], w["lse_t"], "lse", norm=None)
    do2 = do.clone()
    do2[0, at, hd * dh + col] = value
    evk.window_attention(q, k, v, o, dh, window, sinks, lse=lse)
    dq, dk, dv = (torch.empty_like(x) for x in (q, k, v))
    evk.window_attention_bwd(q, k, v, o, do2, dq, dk, dv, lse, dh, window, sinks)
    hit = torch.zeros(b, n, kv, dh, dtype=torch.bool, device=dev)
    hit[0, m[at], c, col] = True
    hit = hit.view(b, n, kv * dh)
    close(dv[~hit], w["dv"][~hit], w["dv_t"][~hit], "dv")
    assert not torch.isfinite(dv[hit].float()).any()
    rows = torch.zeros(b, n, h, dh, dtype=torch.bool, device=dev)
    rows[0, at, hd] = True
    rows = rows.view(b, n, h * dh)
    close(dq[~rows], w["dq"][~rows], w["dq_t"][~rows], "dq", norm=4 * H)
    assert not torch.isfinite(dq[rows].float()).any()
    keys = torch.zeros(b, n, kv, dh, dtype=torch.bool, device=dev)
    keys[0, m[at], c] = True
    keys = keys.view(b, n, kv * dh)
    close(dk[~keys], w["dk"][~keys], w["dk_t"][~keys], "dk", norm=4 * H)
    # dP - D is an infinity where v and o have other signs in that column, else infinity less infinity
    assert not torch.isfinite(dk[keys].float()).any()


@pytest.mark.parametrize("dh,h,kv", [(64, 4, 2), (128, 4, 1), (256, 2, 1), (40, 2, 2)])
@pytest.mark.parametrize("n,window", [(200, 0), (700, 60)])
def test_window_attention_bwd_wild_rows_beside_large_values(dev, dh, h, kv, n, window):
    """Values near fp16's largest with output gradients along them, whose scores' gradients pass fp16, and a row of k, a row
    of q and one of dO that are not finite."""
    r = Rng(dev, 80 + dh)
    q, k = r(1, n, h * dh, std=0.02), r(1, n, kv * dh, std=0.02)
    v = r(1, n, kv * dh, std=20000.0).clamp_(-60000, 60000)
    do = v.view(1, n, kv, 1, dh).expand(1, n, kv, h // kv, dh).float()
    do = (do / do.norm(dim=-1, keepdim=True)).reshape(1, n, h * dh).half()
    w = window_want(q, k, v, h, kv, dh, [0], window, 0, do)
    j, t, u = n - 40, n - 25, n - 10
    k[0, j, 1], q[0, t], do[0, u, :dh] = math.nan, math.nan, math.inf
    o, lse = torch.empty_like(q), torch.empty(1, h, n, device=dev)
    evk.window_attention(q, k, v, o, dh, window, 0, lse=lse)
    dq, dk, dv = (torch.empty_like(x) for x in (q, k, v))
    evk.window_attention_bwd(q, k, v, o, do, dq, dk, dv, lse, dh, window, 0)
    m = seen(torch.arange(n, device=dev), n, window, 0)
    rows = m[:, j].clone()
    rows[t] = rows[u] = True
    keys = (m & rows[:, None]).any(0)
    assert not (window and (rows.all() or keys.all()))
    close(dq[:, ~rows], w["dq"][:, ~rows], w["dq_t"][:, ~rows], "dq", norm=None)
    for g, x in ((dk, "dk"), (dv, "dv")):
        close(g[:, ~keys], w[x][:, ~keys], w[x + "_t"][:, ~keys], x, norm=None)


def passes_us(f, n=5):
    f()
    best = math.inf
    for _ in range(n):
        a, e = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        a.record()
        f()
        e.record()
        e.synchronize()
        best = min(best, a.elapsed_time(e) * 1e3)
    return best


@pytest.mark.parametrize("where", ["do", "k", "q", "do everywhere"])
@pytest.mark.parametrize("dh,h,kv,n,window", [(128, 8, 2, 4096, 512), (64, 4, 1, 8192, 0)])
def test_window_attention_bwd_overflow_costs_no_more(dev, dh, h, kv, n, window, where):
    """A gradient that overflowed (the step that loss scaling skips) must not send its rows and keys through scalar code:
    at most three passes where one serves, and as much again.  With an infinity in every row, the rows of the tiles that
    are not seen whole are added one by one, whose number does not grow with the pairs of a key."""
    r = Rng(dev, 50)
    t = dict(q=r(1, n, h * dh), k=r(1, n, kv * dh), v=r(1, n, kv * dh), do=r(1, n, h * dh))
    q, k, v, do = t.values()
    o, lse = torch.empty_like(q), torch.empty(1, h, n, device=dev)
    g = [torch.empty_like(x) for x in (q, k, v)]
    ws = torch.empty(1 << 28, dtype=torch.uint8, device=dev)

    def step():
        evk.window_attention(q, k, v, o, dh, window, 0, lse=lse, workspace=ws)
        evk.window_attention_bwd(q, k, v, o, do, *g, lse, dh, window, 0, workspace=ws)

    clean = passes_us(step)
    if where == "do everywhere":
        t["do"][0, :, 5] = torch.where(torch.arange(n, device=dev) % 3 == 0, math.inf, -math.inf).to(F16)
    else:
        t[where][0, n // 2 + 3, 5] = math.inf
    wild = passes_us(step, 2)
    assert not torch.isfinite(g[1].float()).all()
    assert wild <= (20 if where == "do everywhere" else 6) * clean + 50, f"{wild:.0f} us with an infinity, {clean:.0f} without"


# ---------------------------------------------------------------------------
# gated_linear: gradients of every size, an infinite gate
# ---------------------------------------------------------------------------
SIZES = [  # dh, up, x and w: std
    (2.0 ** -17, 1.0, 4.0, 4.0), (2.0 ** -13, 1.0, 2.0, 2.0), (4000.0, 30.0, 2.0 ** -10, 2.0 ** -10), (10000.0, 200.0, 2.0 ** -14, 2.0 ** -14),
]


@pytest.mark.parametrize("size,up,sx,sw", SIZES)
@pytest.mark.parametrize("t,d,f,odd", [(1, 64, 128, False), (3, 40, 56, False), (37, 520, 200, False), (600, 768, 1024, False), (1500, 96, 640, False),
                                       (50, 33, 77, True), (300, 100, 201, False), (5, 33, 77, True), (20, 64, 96, False),
                                       (2, 300, 128, False), (1, 24, 257, False)])
@pytest.mark.parametrize("act", ["silu", "gelu", "relu"])
def test_gated_linear_backward_gradient_sizes(dev, t, d, f, odd, act, size, up, sx, sw):
    """Gradients as small as a mean over a batch makes them and as large as loss scaling does: the products' gradients
    neither vanish nor overflow on their way into dx and dw."""
    r = Rng(dev, 9000 + t + f)
    x, w = r(t, d, odd=odd, std=sx), r(2, d, f, std=sw, odd=odd)
    gu, dh = torch.stack([r(t, f), r(t, f, std=up)]), r(t, f, std=size)
    if odd:
        gu, dh = empty(dev, 2, t, f, odd=True).copy_(gu), empty(dev, t, f, odd=True).copy_(dh)
    X, W, G = x.to(F64), w.to(F64), dh.to(F64)
    a, da = act64(gu[0].to(F64), act)
    dgu = torch.stack([G * gu[1].to(F64) * da, G * a])
    # rounded to fp16 with what bounds them, |dh u| and |dh g| (1.13 being the steepest slope), at 2^14 at least, so that
    # subnormals are off by 2^-39 of that; the functions to 2^-20
    most = max(float((G * gu[1].to(F64)).abs().max()) * 1.13, float((G * gu[0].to(F64)).abs().max()))
    edgu = H * dgu.abs() + 2.0 ** -39 * most + 2.0 ** -19 * torch.stack([(G * gu[1].to(F64)).abs(), G.abs()]) * (1 + gu[0].to(F64).abs())
    dx = dgu[0] @ W[0].t() + dgu[1] @ W[1].t()
    mag = dgu[0].abs() @ W[0].abs().t() + dgu[1].abs() @ W[1].abs().t()
    dx_t = edgu[0] @ W[0].abs().t() + edgu[1] @ W[1].abs().t() + (2 * f + 2) * E * mag + H * dx.abs() + T
    dw = torch.stack([X.t() @ dgu[0], X.t() @ dgu[1]])
    dw_t = torch.stack([X.abs().t() @ (edgu[i] + (t + 2) * E * dgu[i].abs()) for i in range(2)]) + H * dw.abs() + T
    assert dx.abs().max() < 60000 and dw.abs().max() < 60000
    gx, gw = empty(dev, t, d, odd=odd), empty(dev, 2, d, f, odd=odd)
    evk.gated_linear_backward(x, w, gu, dh, gx, gw, act)
    for g, want, tol, what in ((gx, dx, dx_t, "dx"), (gw, dw, dw_t, "dw")):
        close(g, want, tol, what, norm=None)
        # two roundings, and the result's own subnormals
        assert (g.to(F64) - want).norm() <= 2 * H * want.norm() + T * want.numel() ** 0.5, what
    more = gw.clone()
    evk.gated_linear_backward(x, w, gu, dh, None, more, act, True)
    close(more, 2 * dw, 2 * dw_t + H * (2 * dw).abs() + T, "dw added to", norm=None)


@pytest.mark.parametrize("t,f", [(1, 64), (40, 200)])
def test_gated_linear_backward_wild_values(dev, t, f):
    """A row of the gradient that overflowed stays in its own row of dx; the others keep their bits."""
    r = Rng(dev, 70)
    d = 64
    x, w, gu, dh = r(t + 1, d), r(2, d, f, std=0.1), r(2, t + 1, f), r(t + 1, f)
    clean, dx = torch.empty(t + 1, d, dtype=F16, device=dev), torch.empty(t + 1, d, dtype=F16, device=dev)
    evk.gated_linear_backward(x, w, gu, dh, clean)
    dh[t, 1] = math.inf
    gu[1, t, 3] = math.nan
    dw = torch.empty_like(w)
    evk.gated_linear_backward(x, w, gu, dh, dx, dw)
    assert not torch.isfinite(dx[t].float()).any()
    if t > 1:
        close(dx[:t], clean[:t].to(F64), 2 * H * clean[:t].abs().to(F64) + T, "dx")
    hit = torch.zeros(f, dtype=torch.bool, device=dev)
    hit[1] = hit[3] = True
    assert torch.isfinite(dw[:, :, ~hit]).all() and not torch.isfinite(dw[0][:, hit].float()).any()


@pytest.mark.parametrize("act", ["silu", "gelu", "relu"])
def test_gated_linear_infinite_gate(dev, act):
    """A gate past fp16, kept as an infinity: its slope is 1 above and 0 below; the second product's gradient is infinite
    above and 0 below."""
    t, d, f = 3, 64, 128
    r = Rng(dev, 71)
    x, w, dh = r(t, d), r(2, d, f, std=0.1), r(t, f)
    gu = r(2, t, f)
    gu[0, 0, 5], gu[0, 1, 6] = math.inf, -math.inf
    gu[1, 0, 5], gu[1, 1, 6] = 1.0, 1.0
    dw = torch.empty_like(w)
    evk.gated_linear_backward(x, w, gu, dh, dw=dw, activation=act)
    gc = gu.to(F64).clamp(-60000, 60000)
    a, da = act64(gc[0], act)
    X, G = x.to(F64), dh.to(F64)
    dgu = torch.stack([G * gc[1] * da, G * a])
    assert abs(float(da[0, 5]) - 1) < 1e-9 and abs(float(da[1, 6])) < 1e-9
    edgu = H * dgu.abs() + T + 2.0 ** -19 * torch.stack([(G * gc[1]).abs(), G.abs()]) * (1 + gc[0].abs().clamp(max=100.0))
    want = torch.stack([X.t() @ dgu[0], X.t() @ dgu[1]])
    tol = torch.stack([X.abs().t() @ (edgu[i] + (t + 2) * E * dgu[i].abs()) for i in range(2)]) + H * want.abs() + T
    close(dw[0], want[0], tol[0], "dw of the gate", norm=None)
    up = torch.ones(f, dtype=torch.bool, device=dev)
    up[5] = False
    close(dw[1][:, up], want[1][:, up], tol[1][:, up], "dw of the second product", norm=None)
    assert not torch.isfinite(dw[1][:, 5].float()).any()
    # forward: sums past fp16 but within 32 bits
    big = torch.full((t, d), 60000.0, dtype=F16, device=dev)
    one = torch.zeros(2, d, f, dtype=F16, device=dev)
    one[0, 0, 0], one[0, 0, 1], one[1, 0, :2] = 60000.0, -60000.0, 2.0 ** -18
    h, keep = torch.empty(t, f, dtype=F16, device=dev), torch.empty(2, t, f, dtype=F16, device=dev)
    evk.gated_linear(big, one, h, keep, act)
    assert torch.isinf(keep[0, :, :2]).all() and torch.isinf(h[:, 0]).all() and (h[:, 1] == 0).all()
