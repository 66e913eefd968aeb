"""8-bit layers and sliding-window attention on tensors whose offsets pass 32 bits."""
import pytest
import torch

from pytorch_distributed_amd import ops
from tests import test_fp8_gpu as fp8
from tests import test_window_attention_gpu as win

pytestmark = pytest.mark.gpu
DEV = "cuda"


def test_window_attention():
    """A batch of 2^31 values and more: its last sequence alone gives the same bits (a workgroup's sums do not depend on
    the batch where there are no sinks)."""
    B, T, H, D, window = 23, 8192, 32, 128, 200
    one = win.inputs(1, T, H, D, seed=3)
    qkv = torch.empty(B, T, 3 * H * D, device=DEV, dtype=torch.bfloat16)
    dout = torch.empty(B, T, H * D, device=DEV, dtype=torch.bfloat16)
    assert qkv.numel() > 2 ** 31
    qkv.copy_(one[0])
    dout.copy_(one[1])
    qkv[:-1, :, :64] += 1.0  # the other sequences are others
    want = win.run(*one, H, window, 0)
    out, g = win.run(qkv, dout, H, window, 0)
    assert torch.equal(out[-1:], want[0]) and torch.equal(g[-1:], want[1])
    assert torch.equal(out[0], out[B - 2]) and torch.equal(g[0], g[B - 2]) and not torch.equal(out[0], out[-1])


def test_layer():
    """A matrix of 2^32 values: the last tokens of the result and of the input gradient, the last features of the weight
    gradient."""
    m, n, k = 2 ** 20, 256, 4096
    part = fp8.rand(2 ** 12, k, seed=1, dtype=torch.bfloat16)
    x = part.repeat(m // 2 ** 12, 1)
    x[-300:] = fp8.rand(300, k, seed=2, dtype=torch.bfloat16)
    x.requires_grad_()
    w = fp8.rand(n, k, seed=3, dtype=torch.bfloat16, spread=0.0).requires_grad_()
    dy = fp8.rand(m, n, seed=4, dtype=torch.bfloat16)
    y = ops.fp8_linear(x, w)
    dx, dw = torch.autograd.grad(y, [x, w], dy)
    with torch.no_grad():
        last = x[-300:]
        by_tiles = ops.quantize_fp8(w, "tiles")
        fp8.check_product(ops.quantize_fp8(last), by_tiles[0], None, torch.bfloat16, y[-300:])
        fp8.check_product(ops.quantize_fp8(dy[-300:]), by_tiles[1], None, torch.bfloat16, dx[-300:])
        fp8.check_product(ops.quantize_fp8(dy, "columns"), ops.quantize_fp8(x[:, -9:], "columns"), None, torch.bfloat16, dw[:, -9:])
