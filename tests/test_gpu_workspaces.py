"""GPU: workspaces that the caller passes, on a stream of its own.

What a workspace holds before a call does not count.  Streams run apart: whoever
fills or allocates it on one stream has the other wait before the call."""
import pytest
import torch

import evk_amd as evk
from test_gpu_block import F16, Rng

pytestmark = pytest.mark.gpu


def empty(dev, *shape):
    return torch.empty(*shape, dtype=F16, device=dev)


def window(dev, r):
    q, k, v, o = r(1, 1, 256), r(1, 5000, 128), r(1, 5000, 128), empty(dev, 1, 1, 256)
    need = evk.window_attention_workspace(q, k, 64)
    return need, [o], lambda **kw: evk.window_attention(q, k, v, o, 64, 0, 0, 4999, **kw)


def window_bwd(dev, r):
    n, h, kv, dh = 700, 4, 2, 64
    q, k, v, do, o = r(1, n, h * dh), r(1, n, kv * dh), r(1, n, kv * dh), r(1, n, h * dh), empty(dev, 1, n, h * dh)
    lse, grads = torch.empty(1, h, n, device=dev), [empty(dev, 1, n, h * dh), empty(dev, 1, n, kv * dh), empty(dev, 1, n, kv * dh)]
    evk.window_attention(q, k, v, o, dh, 100, 4, lse=lse)
    need = evk.lib().evkhip_window_attention_bwd_workspace(1, n, h, kv, dh, 100, 4)
    return need, grads, lambda **kw: evk.window_attention_bwd(q, k, v, o, do, *grads, lse, dh, 100, 4, **kw)


def prefix(dev, r, b=1, n=1, p=9000, rows=30):
    q, pk, pv, k, v, o = r(b, n, 256), r(p, 128), r(p, 128), r(b, rows, 128), r(b, rows, 128), empty(dev, b, n, 256)
    need = evk.prefix_attention_workspace(q, pk, k, 64)
    return need, [o], lambda **kw: evk.prefix_attention(q, pk, pv, k, v, o, 64, rows - n, **kw)


def prefix_shared(dev, r):
    return prefix(dev, r, 6, 2, 20000, 70)


def prefix_prompts(dev, r):
    return prefix(dev, r, 2, 150, 300, 160)


def norm_bwd(dev, r):
    b, n, d = 3, 40, 768
    x, y, ds, dh, wo, wi, gate = r(b, n, d), r(b, n, d), r(b, n, d), r(b, n, d), r(d), r(d), r(b, d)
    outs = [empty(dev, b, n, d), empty(dev, b, n, d), empty(dev, d), empty(dev, b, d), empty(dev, d)]
    need = evk.lib().evkhip_residual_norm_backward_workspace(b * n, b, d)
    return need, outs, lambda **kw: evk.residual_norm_backward(x, y, ds, dh, outs[0], outs[1], wo, gate, wi, *outs[2:], **kw)


@pytest.mark.parametrize("op", [window, window_bwd, prefix, prefix_shared, prefix_prompts, norm_bwd])
def test_workspace_on_another_stream(dev, op):
    need, outs, call = op(dev, Rng(dev, 91))
    assert need > 0
    call()
    want = [t.clone() for t in outs]
    for t in outs:
        t.fill_(7)
    s = torch.cuda.Stream()
    with pytest.raises(ValueError, match="workspace"):  # torch's allocator would give one in the order of the current stream
        call(stream=s.cuda_stream)
    with pytest.raises(evk.EvkError, match="workspace"):
        call(workspace=torch.empty(need - 1, dtype=torch.uint8, device=dev))
    ws = torch.full((need,), 255, dtype=torch.uint8, device=dev)
    s.wait_stream(torch.cuda.current_stream())
    call(workspace=ws, stream=s.cuda_stream)
    torch.cuda.current_stream().wait_stream(s)
    for t, w in zip(outs, want):
        assert torch.equal(t, w)
