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
