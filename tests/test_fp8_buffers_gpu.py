"""The 8-bit layer's gradients into their owner's buffers, as under a reducer or a sharded unit, at sizes of several tiles."""
import pytest
import torch

from pytorch_distributed_amd import ops
from tests import test_fp8_gpu as fp8

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("m,n,k", [(260, 130, 140), (1003, 777, 515), (4096, 2560, 1280), (8200, 1203, 5127), (8192, 5120, 1280)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("accumulate", [False, True])
def test_gradients_into_buffers(m, n, k, dtype, accumulate):
    x, w, b, dy = fp8.layer_case(m, n, k, torch.bfloat16)
    plain = torch.autograd.grad(ops.fp8_linear(x, w, b), [x, w, b], dy)
    before = fp8.rand(n * k + n, 1, seed=8, dtype=dtype)[:, 0]
    flat = before.clone()
    w._pda_grad_sink, b._pda_grad_sink = (lambda: (flat[:n * k], accumulate)), (lambda: (flat[n * k:], accumulate))
    w._pda_grad_sink_dtype = b._pda_grad_sink_dtype = dtype
    y = ops.fp8_linear(x, w, b)
    y.backward(dy)
    assert w.grad is None and b.grad is None
    # x's gradient does not go through a buffer, but may share a launch with one that does
    want, bound = fp8.product_bounds(ops.quantize_fp8(dy), ops.quantize_fp8(w.detach(), "tiles")[1], None, torch.bfloat16)
    assert ((x.grad.double() - want).abs() <= bound).all()
    assert ((plain[0].double() - want).abs() <= bound).all()
    # the sum in the buffer's dtype: the product's own bound there, and the rounding of the sum
    half = 2.0 ** -8 if dtype == torch.bfloat16 else 2.0 ** -24
    old = before.double() * accumulate
    want, bound = fp8.product_bounds(ops.quantize_fp8(dy, "columns"), ops.quantize_fp8(x.detach(), "columns"), None, dtype)
    want, bound = want + old[:n * k].view(n, k), bound + half * (want.abs() + old[:n * k].view(n, k).abs())
    assert ((flat[:n * k].view(n, k).double() - want).abs() <= bound).all()
    want, size = dy.double().sum(0), dy.double().abs().sum(0)
    off = (flat[n * k:].double() - want - old[n * k:]).abs()
    assert (off <= half * (want.abs() + old[n * k:].abs()) * 1.01 + (m / 128 + 16) * 2.0 ** -24 * size).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_buffers_repeat_bit_for_bit(dtype):
    """Twice the same calls into zeroed buffers, and a captured pass replayed beside eager ones."""
    m, n, k = 2100, 1300, 1400
    x, w, b, dy = fp8.layer_case(m, n, k, torch.bfloat16)
    flat = torch.zeros(n * k + n, device=DEV, dtype=dtype)
    w._pda_grad_sink, b._pda_grad_sink = (lambda: (flat[:n * k], True)), (lambda: (flat[n * k:], True))
    w._pda_grad_sink_dtype = b._pda_grad_sink_dtype = dtype

    def twice():
        flat.zero_()
        for _ in range(2):
            (dx, *_) = torch.autograd.grad(ops.fp8_linear(x, w, b), [x, w, b], dy, allow_unused=True)
        return dx.clone(), flat.clone()

    want = twice()
    assert want[1].any()
    assert all(torch.equal(a, c) for a, c in zip(want, twice()))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = twice()
    for _ in range(3):
        graph.replay()
        assert all(torch.equal(a, c) for a, c in zip(got, want))
        assert all(torch.equal(a, c) for a, c in zip(want, twice()))
        torch.cuda.synchronize()


def test_evaluation_keeps_nothing():
    """Without grad mode a layer whose gradients have an owner makes no copy of its input, in values or in memory."""
    m, n, k = 4096, 256, 2048
    x, w, b, _ = fp8.layer_case(m, n, k, torch.bfloat16)
    x = x.detach()

    def peak():
        torch.cuda.synchronize()
        torch.cuda.reset_peak_memory_stats()
        before = torch.cuda.memory_allocated()
        with torch.no_grad():
            y = ops.fp8_linear(x, w, b)
        return y, torch.cuda.max_memory_allocated() - before

    want, plain = peak()
    w._pda_grad_sink = b._pda_grad_sink = lambda: None
    got, owned = peak()
    assert torch.equal(got, want) and not got.requires_grad
    assert owned <= plain  # (the copy alone is m * k bytes, 8 MiB)
