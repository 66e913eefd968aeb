"""Sliding-window attention on the CPU: the mask, the reference against a loop over queries, gradients, refusals."""
import math

import pytest
import torch

from pytorch_distributed_amd import ops

CASES = [(1, 1, 1, 8, 1, 0), (2, 7, 2, 4, 3, 0), (1, 9, 3, 8, 1, 2), (2, 12, 1, 4, 4, 5), (1, 6, 2, 8, 100, 3), (1, 8, 1, 4, 2, 100)]


@pytest.mark.parametrize("B,T,H,D,window,sinks", CASES)
def test_against_a_loop(B, T, H, D, window, sinks):
    g = torch.Generator().manual_seed(T)
    qkv = torch.randn(B, T, 3 * H * D, generator=g)
    out = ops.window_attention(qkv, H, window, sinks).view(B, T, H, D)
    q, k, v = qkv.double().view(B, T, 3, H, D).unbind(2)
    for b in range(B):
        for h in range(H):
            for t in range(T):
                seen = [s for s in range(t + 1) if t - s < window or s < sinks]
                w = torch.softmax(torch.stack([q[b, t, h] @ k[b, s, h] for s in seen]) / math.sqrt(D), 0)
                want = sum(a * v[b, s, h] for a, s in zip(w, seen))
                assert torch.allclose(out[b, t, h].double(), want, rtol=0, atol=1e-5)
    mask = ops.visible_mask(T, window, sinks)
    assert all(bool(mask[t, s]) == (s <= t and (t - s < window or s < sinks)) for t in range(T) for s in range(T))


def test_gradient_against_differences():
    g = torch.Generator().manual_seed(0)
    qkv = torch.randn(1, 6, 3 * 2 * 4, generator=g)
    dout = torch.randn(1, 6, 8, generator=g)
    leaf = qkv.clone().requires_grad_()
    ops.window_attention(leaf, 2, 2, 1).backward(dout)
    step = 1e-2
    for i in range(0, qkv.numel(), 5):
        e = torch.zeros(qkv.numel())
        e[i] = step
        e = e.view_as(qkv)
        diff = ((ops.window_attention(qkv + e, 2, 2, 1) - ops.window_attention(qkv - e, 2, 2, 1)).double() * dout).sum() / (2 * step)
        # third derivative of a softmax of O(1) scores times step^2, and fp32 rounding over the step
        assert abs(float(diff) - float(leaf.grad.view(-1)[i])) < 20 * step ** 2 + 64 * 2.0 ** -24 / step


def test_wide_window_is_causal_attention():
    qkv = torch.randn(2, 10, 3 * 2 * 8, generator=torch.Generator().manual_seed(1))
    want = ops.causal_attention(qkv, 2)
    for window, sinks in ((10, 0), (1000, 0), (1, 10)):
        assert torch.allclose(ops.window_attention(qkv, 2, window, sinks), want, rtol=0, atol=1e-6)


def test_empty():
    assert ops.window_attention(torch.zeros(0, 5, 24), 2, 2).shape == (0, 5, 8)


def test_refusals():
    qkv = torch.zeros(1, 4, 24)
    with pytest.raises(ValueError, match="window must be"):
        ops.window_attention(qkv, 2, 0)
    with pytest.raises(ValueError, match="sinks"):
        ops.window_attention(qkv, 2, 1, -1)
    with pytest.raises(ValueError, match="head size"):
        ops.window_attention(qkv, 5, 1)
    with pytest.raises(ValueError, match="head size"):
        ops.window_attention(qkv[0], 2, 1)
    with pytest.raises(ValueError, match="dropout_p"):
        ops.window_attention(qkv, 2, 1, dropout_p=1.0, training=True)
