"""Gradients of sliding-window attention where the forward's tests stop: keys that nobody sees, scores of several
hundred, dropout over several chunks of far queries."""
import math

import pytest
import torch

from pytorch_distributed_amd import _ext, ops
from tests import test_window_attention_gpu as win

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("T,window,sinks", [(600, 100, 10), (1500, 70, 0), (1500, 129, 40)])
def test_keys_that_are_not_seen_leave_gradients_alone(D, T, window, sinks):
    """Other keys and values at positions sinks .. c - 1 change nothing, to the bit, for the queries from c + window on
    (none of which sees them), nor for the keys from c + window on (whose queries are among these)."""
    c = T // 3
    qkv, dout = win.inputs(1, T, 2, D, seed=13)
    other = qkv.clone()
    other.view(1, T, 3, 2, D)[:, sinks:c, 1:] = 3.0
    a, ga = win.run(qkv, dout, 2, window, sinks)
    b, gb = win.run(other, dout, 2, window, sinks)
    far = c + window
    assert torch.equal(a[:, far:], b[:, far:]) and torch.equal(ga[:, far:], gb[:, far:])
    assert torch.equal(a[:, :sinks], b[:, :sinks])
    assert not torch.equal(a, b) and not torch.equal(ga[:, :c], gb[:, :c])
    # and gradients of later outputs alone never reach the keys that they do not see
    late = dout.clone()
    late[:, :far] = 0
    _, g = win.run(qkv, late, 2, window, sinks)
    dk, dv = g.view(1, T, 3, 2, D)[:, sinks:c, 1], g.view(1, T, 3, 2, D)[:, sinks:c, 2]
    assert not dk.any() and not dv.any() and not g.view(1, T, 3, 2, D)[:, :far, 0].any()


@pytest.mark.parametrize("D", [64, 128])
def test_large_scores(D):
    """Scores of several hundreds: both passes."""
    T, window, sinks = 400, 90, 3
    qkv, dout = win.inputs(1, T, 2, D, seed=1)
    v = qkv.view(1, T, 3, 2, D)
    v[:, :sinks, 1] *= 30.0
    v[:, 100:110, 1] *= 20.0
    out, g = win.run(qkv, dout, 2, window, sinks)
    want, tol, wg, tg = win.oracle(qkv, dout, 2, window, sinks)
    # A score is a sum of D products in fp32, in D / 16 instructions, and meets its row's constant there, which is no
    # larger than the largest score plus log T: it is good to (D / 16 + 2) 2^-24 * 2 size, size the largest
    # sum |q k| / sqrt(D). With size < 2^10 and D = 128 that is 10 * 2^-13 < 2^-9, and as much again for the row's
    # constant in the backward: a probability is off by less than 2^-8 of itself, half a step of bf16. The oracle's
    # tolerance counts such a half step on every probability and on every dS once already, so twice covers both.
    q, k = v[:, :, 0].double().cpu(), v[:, :, 1].double().cpu()
    assert torch.einsum("bthd,bshd->bhts", q.abs(), k.abs()).max() / math.sqrt(D) < 2.0 ** 10
    win.check(out, want, 2 * tol)
    win.check(g, wg, 2 * tg)


@pytest.mark.parametrize("B,T,H,D,window,sinks", [(1, 2600, 2, 64, 100, 5), (1, 2600, 1, 128, 65, 40), (2, 1100, 3, 128, 300, 4), (1, 4100, 1, 64, 65, 1)])
def test_dropout_over_many_tiles(B, T, H, D, window, sinks):
    p, seed = 0.1, 77
    threshold, keep_scale = ops.attention.dropout_quantised(p)
    qkv, dout = win.inputs(B, T, H, D, seed=T)
    out, g = win.run(qkv, dout, H, window, sinks, dropout_p=p, training=True, seed=seed)
    keep = _ext.require().attention_dropout_mask(B, H, T, p, seed, torch.device(DEV))
    want, tol, wg, tg = win.oracle(qkv, dout, H, window, sinks, keep=keep, keep_scale=keep_scale)
    win.check(out, want, tol)
    win.check(g, wg, tg)
    again, g2 = win.run(qkv, dout, H, window, sinks, dropout_p=p, training=True, seed=seed)
    assert torch.equal(out, again) and torch.equal(g, g2)


def test_most_heads_of_one_launch():
    """As many single-token sequences as one launch has workgroups for, where the result is V itself; one more is refused."""
    n = 2 ** 24
    qkv = torch.empty(n, 1, 192, device=DEV, dtype=torch.bfloat16)
    qkv.view(-1, 2 ** 20, 192).copy_(win.inputs(1, 2 ** 20, 1, 64)[0])
    with pytest.raises(RuntimeError, match="32-bit indices"):
        ops.window_attention(qkv, 1, 1)
    out = ops.window_attention(qkv[1:], 1, 1)
    assert torch.equal(out, qkv[1:, :, 128:])
