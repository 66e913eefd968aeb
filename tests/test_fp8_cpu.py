"""8-bit linear layer on the CPU: the references against the definition in 64 bits, the autograd rule, refusals."""
import math

import pytest
import torch

from pytorch_distributed_amd import ops
from pytorch_distributed_amd.ops.regen import GeluRegen


def definition(v, tile):
    """(values / scale, exponent) of every 1 x 128 or 128 x 128 block of v, element by element, in 64 bits."""
    rows, cols = v.shape
    step_r = 128 if tile else 1
    q, e = torch.zeros(rows, cols, dtype=torch.float64), {}
    for r in range(0, rows, step_r):
        for c in range(0, cols, 128):
            block = v[r:r + step_r, c:c + 128].double()
            finite = block[torch.isfinite(block)].abs()
            amax = float(finite.max()) if finite.numel() else 0.0
            k = -127
            while amax > 448.0 * 2.0 ** k:
                k += 1
            e[r // step_r, c // 128] = k
            y = block / 2.0 ** k
            exponent = torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6)))
            y = torch.round(y / torch.exp2(exponent - 3)) * torch.exp2(exponent - 3)  # ties to even
            q[r:r + step_r, c:c + 128] = torch.where(torch.isfinite(block), y, torch.full_like(y, math.nan))
    return q, e


def same(m, v, tile):
    q, e = definition(v, tile)
    got = m.q.to(torch.float64)
    assert m.rows == v.shape[0] and m.cols == v.shape[1] and m.tiles == tile
    assert torch.equal(got[:, :m.cols].nan_to_num(1e6), q.nan_to_num(1e6))
    assert not got[:, m.cols:].any()
    for (r, c), k in e.items():
        assert int(m.scale[r, c]) == k + 127, (r, c)


@pytest.mark.parametrize("rows,cols", [(1, 1), (3, 128), (130, 129), (257, 300)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_quantize_reference(rows, cols, dtype):
    g = torch.Generator().manual_seed(rows * 1000 + cols)
    v = (torch.randn(rows, cols, generator=g) * torch.exp2(8 * torch.randn(rows, 1, generator=g))).to(dtype)
    a, b = ops.quantize_fp8(v, "both")
    same(a, v, False)
    same(b, v.t(), False)
    same(ops.quantize_fp8(v, "rows"), v, False)
    same(ops.quantize_fp8(v, "columns"), v.t(), False)
    a, b = ops.quantize_fp8(v, "tiles")
    same(a, v, True)
    same(b, v.t(), True)


def test_quantize_special_values():
    v = torch.zeros(8, 128)
    v[1] = 448.0  # exactly representable at scale 1
    v[2, 5] = torch.nextafter(torch.tensor(448.0), torch.tensor(500.0))  # the next float needs the next scale
    v[3, :3] = torch.tensor([math.inf, -math.inf, math.nan])
    v[3, 3] = 7.0
    v[4] = math.nan  # nothing finite
    v[5, 0] = 3.0e38
    v[6, 0] = 1.0e-40  # subnormal
    v[7, 0], v[7, 1] = 1.0, 2.0 ** -20  # far below the block's largest: zero
    m = ops.quantize_fp8(v, "rows")
    same(m, v, False)
    assert int(m.scale[0, 0]) == 0 and int(m.scale[1, 0]) == 127 and int(m.scale[2, 0]) == 128
    assert int(m.scale[4, 0]) == 0 and int(m.scale[5, 0]) == 120 + 127 and int(m.scale[6, 0]) == 0


def test_matmul_reference():
    g = torch.Generator().manual_seed(0)
    x, w, bias = torch.randn(5, 200, generator=g), torch.randn(131, 200, generator=g), torch.randn(131, generator=g)
    a, b = ops.quantize_fp8(x), ops.quantize_fp8(w, "tiles")[0]
    want = a.dequantize().double() @ b.dequantize().double().t() + bias.double()
    y = ops.fp8_matmul(a, b, bias, torch.float32)
    assert torch.allclose(y.double(), want, rtol=0, atol=200 * 2.0 ** -24 * float(want.abs().max()) * 4)
    # half a step of e4m3 per operand: (1 + 2^-4)^2 - 1 of each term at most, plus what became subnormal
    bound = ((1 + 2.0 ** -4) ** 2 - 1) * (x.abs() @ w.abs().t()) + 2e-2
    assert ((want - bias - (x @ w.t())).abs() <= bound).all()


def test_linear_of_representable_values_is_exact():
    """Integers up to 15 are e4m3 numbers under every scale, so the layer is the exact bilinear map on them:
    its gradients are the formula's, and differences along integer steps are the gradients'."""
    g = torch.Generator().manual_seed(1)
    x = torch.randint(-7, 8, (2, 9, 140), generator=g).float().requires_grad_()
    w = torch.randint(-7, 8, (133, 140), generator=g).float().requires_grad_()
    b = torch.randint(-7, 8, (133,), generator=g).float().requires_grad_()
    dy = torch.randint(-7, 8, (2, 9, 133), generator=g).float()
    y = ops.fp8_linear(x, w, b)
    y.backward(dy)
    assert torch.equal(y, x @ w.t() + b)
    assert torch.equal(x.grad, dy @ w)
    assert torch.equal(w.grad, dy.reshape(-1, 133).t() @ x.reshape(-1, 140))
    assert torch.equal(b.grad, dy.sum((0, 1)))
    with torch.no_grad():
        for leaf, place in ((x, (1, 3, 7)), (w, (130, 2)), (b, (5,))):
            step = torch.zeros_like(leaf)
            step[place] = 3.0
            args = [t + step if t is leaf else t for t in (x, w, b)]
            diff = ((ops.fp8_linear(*args) - y) * dy).sum()
            assert diff == 3.0 * leaf.grad[place]


def test_linear_regen_and_partial_gradients():
    g = torch.Generator().manual_seed(2)
    u = torch.randn(6, 40, generator=g, requires_grad=True)
    w = torch.randn(24, 40, generator=g, requires_grad=True)
    kept = ops.fp8_linear(ops.gelu_new(u), w)
    rebuilt = ops.fp8_linear(ops.gelu_new(u), w, regen=GeluRegen(u))
    assert torch.equal(kept, rebuilt)
    dy = torch.randn(6, 24, generator=g)
    for a, b in zip(torch.autograd.grad(kept, [u, w], dy), torch.autograd.grad(rebuilt, [u, w], dy)):
        assert torch.equal(a, b)
    x = torch.randn(3, 40, generator=g)
    (only_w,) = torch.autograd.grad(ops.fp8_linear(x, w), [w], dy[:3])
    assert only_w.shape == w.shape
    xg = x.clone().requires_grad_()
    (only_x,) = torch.autograd.grad(ops.fp8_linear(xg, w.detach()), [xg], dy[:3])
    assert only_x.shape == x.shape


@pytest.mark.parametrize("tokens", [0, 1])
def test_linear_few_tokens(tokens):
    x = torch.randn(tokens, 16, requires_grad=True)
    w = torch.randn(8, 16, requires_grad=True)
    b = torch.zeros(8, requires_grad=True)
    y = ops.fp8_linear(x, w, b)
    y.sum().backward()
    assert y.shape == (tokens, 8) and x.grad.shape == x.shape and w.grad.shape == w.shape
    assert torch.equal(b.grad, torch.full((8,), float(tokens)))


@pytest.mark.parametrize("shape,out", [((2, 3, 0), 8), ((2, 3, 16), 0), ((2, 0, 16), 8), ((0, 3, 0), 4)])
def test_linear_without_elements(shape, out):
    x, w, b = torch.randn(shape, requires_grad=True), torch.randn(out, shape[-1], requires_grad=True), torch.ones(out, requires_grad=True)
    y = ops.fp8_linear(x, w, b)
    assert torch.equal(y, torch.ones(*shape[:-1], out))
    y.sum().backward()
    assert x.grad.shape == x.shape and not x.grad.any() and w.grad.shape == w.shape and not w.grad.any()
    assert torch.equal(b.grad, torch.full((out,), float(shape[0] * shape[1])))


def test_refusals():
    x = torch.randn(4, 16)
    w = torch.randn(8, 16)
    with pytest.raises(ValueError, match="blocks must be"):
        ops.quantize_fp8(x, "row")
    with pytest.raises(ValueError, match="matrix"):
        ops.quantize_fp8(x[0])
    with pytest.raises(NotImplementedError, match="dtype"):
        ops.quantize_fp8(x.half())
    a, b = ops.quantize_fp8(x), ops.quantize_fp8(w)
    with pytest.raises(ValueError, match="contraction"):
        ops.fp8_matmul(a, ops.quantize_fp8(torch.randn(8, 17)))
    with pytest.raises(NotImplementedError, match="out_dtype"):
        ops.fp8_matmul(a, b, out_dtype=torch.float16)
    with pytest.raises(ValueError, match="bias"):
        ops.fp8_matmul(a, b, bias=torch.zeros(7))
    with pytest.raises(ValueError, match="scale must be"):
        ops.Fp8Matrix(a.q, a.scale[:, :2], 16)
    with pytest.raises(ValueError, match="q must be"):
        ops.Fp8Matrix(a.q, a.scale, 200)
    with pytest.raises(ValueError, match="scale must be"):
        ops.Fp8Matrix(torch.zeros(200, 128).to(torch.float8_e4m3fn), torch.zeros(200, 4, dtype=torch.uint8), 16, tiles=True)
    with pytest.raises(ValueError, match="do not match"):
        ops.fp8_linear(x, torch.randn(8, 17))
    with pytest.raises(ValueError, match="weight"):
        ops.fp8_linear(x, w.bfloat16())
    with pytest.raises(ValueError, match="bias"):
        ops.fp8_linear(x, w, torch.zeros(9))
    with pytest.raises(NotImplementedError, match="dtype"):
        ops.fp8_linear(x.half(), w.half())
