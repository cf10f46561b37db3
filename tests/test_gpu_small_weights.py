"""GPU: window_attention where the first rows draw most of the weight, as sinks do."""
import math

import pytest
import torch

import evk_amd as evk
from test_gpu_block import F16, F64, Rng, close, empty, window_want

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("b,n,h,kv,dh,rows,window,sinks", [
    (1, 1, 8, 2, 64, 9000, 0, 0), (8, 3, 8, 2, 128, 9000, 8000, 1), (16, 1, 4, 1, 256, 4000, 2000, 4), (2, 300, 4, 2, 96, 6000, 5000, 2),
    (1, 2000, 8, 4, 64, 9000, 6000, 1), (3, 1, 2, 1, 32, 900, 0, 0), (1, 700, 2, 1, 128, 9000, 0, 0)])
def test_window_attention_a_sink_that_draws_most(dev, b, n, h, kv, dh, rows, window, sinks):
    """The first row's score is 2^18 above the others' and its values are zeros, so that the output is a sum of small
    weights.  A weight of 2^-18 of the largest, with 2^7 in front 2^-11, is off by half a step of its 11 bits, as is the
    result: 2^-12 each in quadrature of the uniform error, below 2^-11 of the norm together."""
    r = Rng(dev, 790 + dh)
    q, v = torch.zeros(b, n, h * dh, dtype=F16, device=dev), r(b, rows, kv * dh)
    k = torch.zeros(b, rows, kv * dh, dtype=F16, device=dev)
    q.view(b, n, h, dh)[..., 0] = 4.0
    q.view(b, n, h, dh)[..., 1:] = r(b, n, h, dh - 1, std=0.1)
    k.view(b, rows, kv, dh)[..., 1:] = r(b, rows, kv, dh - 1)
    k.view(b, rows, kv, dh)[:, 0] = 0.0
    k.view(b, rows, kv, dh)[:, 0, :, 0] = 18.0 * math.log(2.0) * dh ** 0.5 / 4.0
    v[:, 0] = 0.0
    o, lse = empty(dev, b, n, h * dh), torch.empty(b, h, n, device=dev)
    evk.window_attention(q, k, v, o, dh, window, sinks, rows - n, lse=lse)
    w = window_want(q, k, v, h, kv, dh, [rows - n] * b, window, sinks)
    assert float((o.to(F64) - w["o"]).norm() / w["o"].norm()) <= 2.0 ** -11
    close(lse, w["lse"], w["lse_t"], "lse", norm=None)
