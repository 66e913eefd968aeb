"""How the 8-bit products of a call are planned (host code of the extension; no GPU needed)."""
import pytest

from pytorch_distributed_amd import _ext

SIZES = [(8192, 1280, 5120), (8192, 4096, 22016), (8192, 5120, 1280), (1000, 513, 257), (64, 1280, 1280), (30000, 1600, 6400)]


def plan(*products):
    return [tuple(p) for p in _ext.require().fp8_plan([list(p) for p in products])]


@pytest.mark.parametrize("m,k,n", SIZES)
@pytest.mark.parametrize("accumulate", [0, 1])
def test_an_fp32_weight_gradient_leaves_the_input_gradient_its_plan(m, k, n, accumulate):
    """The two take different kernels, so they are launched, and have to be planned, one by one."""
    dx, dw = (m, k, n, 0, 0), (n, k, m, 1, accumulate)
    assert plan(dx, dw) == plan(dx) + plan(dw)
    assert plan(dw, dx) == plan(dw) + plan(dx)
    assert plan(dw)[0][0] == 128


def test_large_products_to_bf16_take_a_large_tile():
    for m, k, n in SIZES[:3]:
        assert plan((m, k, n, 0, 0))[0][0] > 128 and plan((m, n, k, 0, 0))[0][0] > 128


@pytest.mark.parametrize("m,k,n", SIZES)
def test_products_of_one_kernel_share_a_tile(m, k, n):
    a, b = plan((m, k, n, 0, 0), (n, k, m, 0, 0))
    assert a[0] == b[0]


def test_accumulating_counts_the_fold():
    """An accumulating product goes through partial sums and a fold anyway, so cutting its contraction costs it less:
    it is never cut less often than the same product into fresh memory."""
    for m, n, k in ((1280, 5120, 8192), (512, 512, 4096), (1024, 1024, 8192), (2048, 2048, 2048), (1280, 1280, 8192)):
        for f32 in (0, 1):
            assert plan((m, n, k, f32, 1))[0][1] >= plan((m, n, k, f32, 0))[0][1]


def test_bounds():
    assert plan() == []
    with pytest.raises(RuntimeError, match="at most two"):
        plan((1, 1, 1, 0, 0), (1, 1, 1, 0, 0), (1, 1, 1, 0, 0))
    with pytest.raises(RuntimeError, match="between 1 and"):
        plan((0, 1, 1, 0, 0))
