"""What an 8-bit matrix stands for, exactly, on the GPU."""
import pytest
import torch

from pytorch_distributed_amd import _ext, ops

pytestmark = pytest.mark.gpu
DEV = "cuda"


def all_values(rows):
    """Every e4m3 number in each of `rows` rows of 256."""
    codes = torch.arange(256, dtype=torch.uint8, device=DEV)
    codes[(codes & 0x7F) == 0x7F] = 0  # (NaN)
    return codes.view(torch.float8_e4m3fn).expand(rows, 256).contiguous()


def test_dequantize_is_exact_at_every_scale():
    byte = torch.arange(248, dtype=torch.uint8, device=DEV)
    scale = torch.zeros(248, 4, dtype=torch.uint8, device=DEV)
    scale[:, :2] = byte[:, None]
    m = ops.Fp8Matrix(all_values(248), scale, 256)
    # in 64 bits, and from there to fp32: 2^128, a quotient of 256 at the largest scale, is its infinity
    want = m.q.double() * torch.tensor([2.0 ** (b - 127) for b in range(248)], dtype=torch.float64, device=DEV)[:, None]
    assert torch.equal(m.dequantize(), want.float())


@pytest.mark.parametrize("blocks", ["both", "tiles"])
def test_reference_on_the_gpu_agrees_with_the_kernel_at_ties(blocks, monkeypatch):
    """Values half way between two e4m3 numbers, and their neighbours, at many scales."""
    q = all_values(1).float()[0].sort().values.unique()
    ties = (q[1:] + q[:-1]) / 2
    up = torch.nextafter(ties, torch.full_like(ties, 1e9))
    row = torch.cat([ties, up, torch.full((1,), 448.0, device=DEV)])
    e = torch.arange(-100, 112, device=DEV)
    x = row[None, :] * torch.tensor([2.0 ** int(k) for k in e], dtype=torch.float64, device=DEV).float()[:, None]
    kernel = ops.quantize_fp8(x, blocks)
    monkeypatch.setenv("PDA_FORCE_REFERENCE", "1")
    assert not _ext.use_hip(x)
    for a, b in zip(kernel, ops.quantize_fp8(x, blocks)):
        blocks_in_row = -(-a.cols // 128)
        assert torch.equal(a.q.view(torch.uint8), b.q.view(torch.uint8)) and torch.equal(a.scale[:, :blocks_in_row], b.scale[:, :blocks_in_row])


@pytest.mark.parametrize("byte", [0, 1, 2, 3, 9, 60])
@pytest.mark.parametrize("left", [True, False])
def test_products_at_the_smallest_scales(byte, left):
    """One operand at the smallest scales, the other so large that the product is an ordinary number. To bf16 the scale
    is applied inside the instruction; to fp32 the operand is widened to bf16 first, whose smallest number is 2^-133:
    exact from byte 3 on, below that each element is off by half of it at the most."""
    g = torch.Generator(device=DEV).manual_seed(byte)
    m, n, k = 70, 100, 300
    small = torch.randint(-60, 61, (m, k), generator=g, device=DEV).float() * 2.0 ** -9  # subnormal and small e4m3 numbers
    q = torch.zeros(m, 384, device=DEV)
    q[:, :k] = small
    a = ops.Fp8Matrix(q.to(torch.float8_e4m3fn), torch.full((m, 4), byte, dtype=torch.uint8, device=DEV), k)
    b = ops.quantize_fp8(torch.randn(n, k, generator=g, device=DEV) * 2.0 ** 112)
    x, w = a.q.double()[:, :k] * 2.0 ** (byte - 127), b.dequantize().double()
    want, size = x @ w.t().contiguous(), x.abs() @ w.abs().t().contiguous()
    if not left:
        a, b, want, size = b, a, want.t(), size.t()
    y = ops.fp8_matmul(a, b, None, torch.bfloat16).double()
    assert ((y - want).abs() <= 2.0 ** -8 * want.abs() + 2.0 ** -12 * size).all()
    y = ops.fp8_matmul(a, b, None, torch.float32).double()
    rounded = 2.0 ** -134 * w.abs().sum(1) if byte < 3 else torch.zeros(n, dtype=torch.float64, device=DEV)
    rounded = rounded[None, :] if left else rounded[:, None]
    assert ((y - want).abs() <= 2.0 ** -24 * want.abs() + (k / 16 + 16) * 2.0 ** -23 * size + rounded * 1.01).all()
