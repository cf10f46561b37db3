"""GPU: the group's operators at the ends of their ranges: prefixes long enough to be
read once for all sequences, behind sequences that have no rows, few or stale
ones; rows that hold nothing but equal logits, few allowed ids, long ids."""
import math

import pytest
import torch

import evk_amd as evk
from test_gpu_block import E, F16, F64, H, T, Rng, close, empty
from test_gpu_group import Norms, grad_check, ids16, prefix_check, prefix_want, scores_check, some_tokens

pytestmark = pytest.mark.gpu

SHARED = [  # heads, kv, dh, n, prefix: tiles of 64 rows and of 128, one launch and a join
    (8, 2, 64, 1, 5000), (8, 2, 64, 7, 5000), (4, 4, 128, 1, 4100), (16, 4, 128, 9, 9001), (2, 1, 256, 2, 6000), (6, 3, 40, 1, 8003), (4, 1, 96, 3, 7000),
    (2, 2, 32, 5, 9000), (64, 8, 128, 7, 2500),
]


@pytest.mark.parametrize("h,kv,dh,n,p", SHARED)
def test_prefix_shared_offsets(dev, h, kv, dh, n, p):
    """Sequences before their own rows, at their first and last, and past them."""
    rows = n + 30
    off = [0, -1, -n, -n + 1, -1000, 30, 31, rows, 5, -2 ** 31, 2 ** 31 - 1]
    r = Rng(dev, 600 + dh)
    q, pk, pv = r(len(off), n, h * dh), r(p, kv * dh), r(p, kv * dh)
    k, v = r(len(off), rows, kv * dh), r(len(off), rows, kv * dh)
    prefix_check(dev, q, pk, pv, k, v, h, kv, dh, off)


@pytest.mark.parametrize("h,kv,dh,n,p", SHARED)
def test_prefix_shared_values_apart(dev, h, kv, dh, n, p):
    """Stale rows of any content stay out; own rows that hold NaN or infinities reach the queries that see them and no
    other; values of the prefix that are not finite reach all, in their column."""
    b, rows = 6, n + 600
    r = Rng(dev, 610 + dh)
    q, pk, pv = r(b, n, h * dh), r(p, kv * dh), r(p, kv * dh)
    k, v = r(b, rows, kv * dh), r(b, rows, kv * dh)
    off = [3, 0, 11, 600, 555, 31]
    for s in range(b):
        k[s, off[s] + n:], v[s, off[s] + n:] = math.nan, math.inf
    clean = prefix_check(dev, q, pk, pv, k, v, h, kv, dh, off)
    k[0, 3 + n // 2], v[1, n - 1, 3], v[2, 11 + n // 2] = math.nan, math.inf, math.nan
    o = empty(dev, b, n, h * dh)
    evk.prefix_attention(q, pk, pv, k, v, o, dh, offsets=torch.tensor(off, dtype=torch.int32, device=dev))
    t = torch.arange(n, device=dev)
    hit = torch.zeros(b, n, h, dh, dtype=torch.bool, device=dev)
    hit[0, t >= n // 2] = True
    hit[2, t >= n // 2] = True
    hit[1, n - 1, : h // kv, 3] = True
    hit = hit.view(b, n, h * dh)
    assert (~torch.isfinite(o[hit])).all()
    assert torch.isfinite(o[~hit]).all()
    assert float((o[~hit].double() - clean[~hit].double()).norm() / clean[~hit].double().norm()) <= 4 * H
    pv[p - 1, 2] = math.inf
    evk.prefix_attention(q, pk, pv, torch.zeros_like(k), torch.zeros_like(v), o, dh, offsets=torch.tensor(off, dtype=torch.int32, device=dev))
    reach = torch.zeros(b, n, h, dh, dtype=torch.bool, device=dev)
    reach[:, :, : h // kv, 2] = True
    assert torch.equal(~torch.isfinite(o), reach.view(b, n, h * dh))


@pytest.mark.parametrize("h,kv,dh,n,p", SHARED)
def test_prefix_shared_large_scores(dev, h, kv, dh, n, p):
    """Scores of thousands, in the prefix or in the own rows: one row takes all; and of -inf everywhere."""
    b, rows = 4, n + 60
    r = Rng(dev, 620 + dh)
    q, pk, pv = r(b, n, h * dh, std=30.0), r(p, kv * dh, std=30.0), r(p, kv * dh)
    k, v = r(b, rows, kv * dh, std=30.0), r(b, rows, kv * dh)
    off = [0, 60, 17, -n]
    prefix_check(dev, q, pk, pv, k, v, h, kv, dh, off)
    q.fill_(1.0)
    pk.fill_(-math.inf)
    k[1] = -math.inf
    o, lse = empty(dev, b, n, h * dh), torch.zeros(b, h, n, device=dev)
    evk.prefix_attention(q, pk, pv, k, v, o, dh, offsets=torch.tensor(off, dtype=torch.int32, device=dev), lse=lse)
    w = prefix_want(q[:1], pk[:0], pv[:0], k[:1], v[:1], h, kv, dh, [0])
    assert ((o[:1].to(F64) - w["o"]).abs() <= w["o_t"]).all()
    for s in (1, 3):
        assert torch.isnan(o[s]).all() and (lse[s] == -math.inf).all()


@pytest.mark.parametrize("b,n,h,kv,dh,p,rows", [(64, 1, 8, 8, 64, 600, 20000), (3, 1, 4, 2, 64, 3000, 30000), (2, 1, 2, 2, 128, 70000, 5), (500, 1, 4, 1, 32, 600, 9),
                                                (70, 3, 16, 4, 64, 1500, 700), (9, 60, 4, 1, 64, 900, 80), (40, 40, 8, 2, 64, 1200, 64), (40, 70, 4, 2, 128, 1030, 75)])
def test_prefix_long_and_many(dev, b, n, h, kv, dh, p, rows):
    r = Rng(dev, 630 + p)
    q, pk, pv = r(b, n, h * dh), r(p, kv * dh), r(p, kv * dh)
    k, v = r(b, rows, kv * dh), r(b, rows, kv * dh)
    g = torch.Generator().manual_seed(p)
    prefix_check(dev, q, pk, pv, k, v, h, kv, dh, torch.randint(0, rows - n + 1, (b,), generator=g).tolist())


@pytest.mark.parametrize("b,n,h,kv,dh,p", [(4, 130, 8, 4, 64, 0), (1, 256, 1, 1, 128, 0), (1, 256, 1, 1, 128, 1), (2, 200, 6, 2, 80, 63), (2, 129, 4, 2, 256, 65), (1, 700, 2, 1, 32, 3000)])
def test_prefix_prompts(dev, b, n, h, kv, dh, p):
    """Tiles of one sequence's rows: no prefix, one row, ends inside a tile; the first queries before their own rows."""
    rows = n + 9
    r = Rng(dev, 640 + p + dh)
    q, pk, pv = r(b, n, h * dh), r(p, kv * dh), r(p, kv * dh)
    k, v = r(b, rows, kv * dh), r(b, rows, kv * dh)
    for off in ([0] * b, [9] * b, [-5] * b, [-n + 1] * b, [5] * b):
        prefix_check(dev, q, pk, pv, k, v, h, kv, dh, off)


@pytest.mark.parametrize("v", [40, 1000, 3000, 8000, 16000, 32000, 65536])
@pytest.mark.parametrize("allowed", [1, 3, 20, 33, 200])
def test_few_allowed_ids(dev, v, allowed):
    """Constrained decoding: all but a few ids at -inf; what is missing among the alternatives are the first of those."""
    if allowed > v:
        return
    r = Rng(dev, 650 + v)
    rows = 6
    x = torch.full((rows, v), -math.inf, dtype=F16, device=dev)
    g = torch.Generator(device=dev).manual_seed(v + allowed)
    for i in range(rows):
        at = torch.randperm(v, device=dev, generator=g)[:allowed]
        if i == 1:
            at = torch.arange(allowed, device=dev)  # the first ids
        if i == 2:
            at = v - 1 - torch.arange(allowed, device=dev)
        x[i, at] = r(allowed, std=3.0)
        if i == 3:
            x[i, at] = -65504.0
    scores_check(dev, x, some_tokens(rows, v, dev, 3, pad=False), 1.0, min(v, 32))


@pytest.mark.parametrize("v", [513, 1025, 2049, 4097, 8193, 16385, 32769])
@pytest.mark.parametrize("top", [1, 32])
def test_vocabularies_past_a_shape(dev, v, top):
    """One logit more than a workgroup's shape before holds, the best ones at the row's end; half as many ties."""
    r = Rng(dev, 660 + v)
    x = r(5, v, std=2.0)
    x[0, -1] = 40.0
    x[1, -3:] = 30.0
    x[2, v // 2:] = 5.0
    x[3, ::2] = 9.0
    scores_check(dev, x, some_tokens(5, v, dev, 3, pad=False), 1.0, top)


def test_candidates_past_their_list(dev):
    """More logits at the bound than the list of candidates holds, in few threads and in many."""
    r = Rng(dev, 670)
    for v in (1000, 4096, 32000):
        x = r(6, v, std=0.5)
        n = 1100 if v > 1100 else 1000
        x[0, :n] = 7.0
        x[1, torch.randperm(v, device=dev)[:n]] = 7.0
        x[2, :1024 if v > 1024 else 900] = 7.0
        x[3] = 0.0
        x[4, ::3] = 1.0
        scores_check(dev, x, some_tokens(6, v, dev, 4, pad=False), 1.0, 32)


@pytest.mark.parametrize("d", [8, 63, 64, 65, 127, 128, 129, 200, 255, 256, 257])
@pytest.mark.parametrize("b,n,gate", [(1, 1, "channel"), (5, 37, "sequence"), (1, 3001, None), (33, 1, "sequence")])
def test_residual_norm_narrow_rows(dev, d, b, n, gate):
    """Rows that share a wave, as many as fill it and not, of one gate and several."""
    c = Norms(dev, 700 + d + n, b, n, d, True, gate, scale=0.5, odd=d % 2 == 1)
    s, h = c.forward()
    want, size = c.want()
    c.check(dict(s=s, h=h), want, size)
    c.check(c.backward(), want, size)


@pytest.mark.parametrize("d", [24, 100, 250])
def test_residual_norm_narrow_rows_apart(dev, d):
    """A row that holds NaN or infinities leaves its neighbours in the wave alone."""
    c = Norms(dev, 720 + d, 1, 70, d, True, "channel")
    s0, h0 = c.forward()
    g0 = c.backward()
    c.x[0, 9], c.y[0, 34, d - 1], c.x[0, 69, 0] = math.nan, math.inf, -math.inf
    s, h = c.forward()
    g = c.backward()
    same = torch.ones(70, dtype=torch.bool, device=dev)
    same[[9, 34, 69]] = False
    for got, was in ((s, s0), (h, h0), (g["dx"], g0["dx"]), (g["dy"], g0["dy"])):
        assert torch.equal(got[0, same], was[0, same])
        assert not torch.isfinite(got[0, ~same]).all()


@pytest.mark.parametrize("v", [8, 120, 144, 256, 257, 512, 513, 1001, 1024, 1025, 2048, 2049])
@pytest.mark.parametrize("rows", [1, 15, 17, 2000])
def test_token_logprobs_backward_short_rows(dev, v, rows):
    """Rows that share a workgroup, as many as fill it and not; behind the last one nothing is written."""
    r = Rng(dev, 740 + v + rows)
    logits, tokens = r(rows, v, std=3.0, odd=v % 2 == 1), some_tokens(rows, v, dev, v)
    dlp, dent = r(rows, std=20.0).float(), r(rows, std=5.0).float()
    d, _ = grad_check(dev, logits, tokens, 0.7, dlp, dent, odd=v % 2 == 0)
    lp, ent, stats = torch.empty(rows, device=dev), torch.empty(rows, device=dev), torch.empty(rows, 2, device=dev)
    evk.token_logprobs(logits, tokens, lp, ent, stats=stats, input_scale=0.7)
    longer = torch.full((rows + 40, v), 9.0, dtype=F16, device=dev)
    evk.token_logprobs_backward(logits, tokens, stats, dlp, longer[:rows], ent, dent, input_scale=0.7)
    assert torch.equal(longer[:rows], d) and (longer[rows:] == 9.0).all()


@pytest.mark.parametrize("b,n,d,gate", [(1, 1, 8193, None), (2, 5, 9000, "sequence"), (1, 700, 12001, "channel"), (3, 130, 16384, "sequence")])
def test_residual_norm_widest_rows(dev, b, n, d, gate):
    """Rows whose sums over a run lie in LDS, runs of one row and of several."""
    c = Norms(dev, 760 + d, b, n, d, True, gate, scale=1.5, odd=d % 2 == 1)
    s, h = c.forward()
    want, size = c.want()
    c.check(dict(s=s, h=h), want, size)
    got = c.backward()
    c.check(got, want, size)
    again = c.backward()
    assert all(v is None or torch.equal(v, again[k]) for k, v in got.items())
    c = Norms(dev, 761 + d, b, n, d, y=False)  # and the norm alone
    want, size = c.want()
    c.check(c.backward(), want, size)


@pytest.mark.parametrize("b,n,h,kv,dh,p", [(1, 1, 8, 2, 64, 9000), (8, 3, 8, 2, 128, 9000), (16, 40, 4, 4, 64, 9000), (2, 300, 4, 2, 96, 9000), (3, 1, 2, 1, 256, 300)])
def test_prefix_a_row_that_draws_most(dev, b, n, h, kv, dh, p):
    """The first row's score is 2^18 above the others' and its values are zeros, so that the output is a sum of small
    weights.  A weight of 2^-18 of the largest, with 2^7 in front 2^-11, is off by half a step of its 11 bits, as is the
    result: 2^-12 each in quadrature of the uniform error, below 2^-11 of the norm together."""
    r = Rng(dev, 780 + dh)
    q, pk, pv = torch.zeros(b, n, h * dh, dtype=F16, device=dev), torch.zeros(p, kv * dh, dtype=F16, device=dev), r(p, kv * dh)
    rows = n + 9
    k, v = torch.zeros(b, rows, kv * dh, dtype=F16, device=dev), r(b, rows, kv * dh)
    q.view(b, n, h, dh)[..., 0] = 4.0
    q.view(b, n, h, dh)[..., 1:] = r(b, n, h, dh - 1, std=0.1)
    pk.view(p, kv, dh)[..., 1:] = r(p, kv, dh - 1)
    pk.view(p, kv, dh)[0] = 0.0
    pk.view(p, kv, dh)[0, :, 0] = 18.0 * math.log(2.0) * dh ** 0.5 / 4.0
    pv[0] = 0.0
    o, lse = empty(dev, b, n, h * dh), torch.empty(b, h, n, device=dev)
    evk.prefix_attention(q, pk, pv, k, v, o, dh, lse=lse)
    w = prefix_want(q, pk, pv, k, v, h, kv, dh, [0] * b)
    assert float((o.to(F64) - w["o"]).norm() / w["o"].norm()) <= 2.0 ** -11
    assert ((lse.to(F64) - w["lse"]).abs() <= w["lse_t"]).all()
