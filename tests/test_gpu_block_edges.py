"""GPU: the grouped-query block's operators at the ends of their ranges: positions
next to 2^31, scores that are all -inf, NaN and infinities beside finite rows, long
contexts, gradients of every size.  Tolerances as in test_gpu_block.py: H is half
a step of fp16, T of its subnormals, E of 32 bits."""
import pytest
import torch

import evk_amd as evk
from test_gpu_block import H, T, Rng, close, empty, rope_want, window_want

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
