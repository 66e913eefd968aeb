"""The 8-bit kernels against plain 64-bit computations."""
import math

import pytest
import torch

from pytorch_distributed_amd import _ext, ops

pytestmark = pytest.mark.gpu
DEV = "cuda"


def rand(*shape, seed=0, dtype=torch.float32, spread=2.0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    v = torch.randn(*shape, generator=g, device=DEV)
    return (v * torch.exp2(spread * torch.randn(shape[0], 1, generator=g, device=DEV))).to(dtype)


def same_matrix(a, b):
    assert a.cols == b.cols and a.tiles == b.tiles
    assert torch.equal(a.q.view(torch.uint8) & 0x7F == 0x7F, b.q.view(torch.uint8) & 0x7F == 0x7F)  # NaN of either sign
    assert torch.equal(a.q.float().nan_to_num(1e6), b.q.float().nan_to_num(1e6))
    blocks = -(-a.cols // 128)
    assert torch.equal(a.scale[:, :blocks], b.scale[:, :blocks])


def on_cpu(x, blocks):
    got = ops.quantize_fp8(x.cpu(), blocks)
    return [ops.Fp8Matrix(m.q.to(DEV), m.scale.to(DEV), m.cols, m.tiles) for m in (got if isinstance(got, tuple) else (got,))]


# --------------------------------------------------------------------------- quantisation
@pytest.mark.parametrize("rows,cols", [(1, 1), (1, 128), (7, 24), (128, 128), (129, 300), (257, 1000), (1000, 129)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("blocks", ["rows", "columns", "both", "tiles"])
def test_quantize(rows, cols, dtype, blocks):
    x = rand(rows, cols, seed=rows + cols, dtype=dtype, spread=10.0)
    got = ops.quantize_fp8(x, blocks)
    for a, b in zip(got if isinstance(got, tuple) else (got,), on_cpu(x, blocks)):
        same_matrix(a, b)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_quantize_strides_and_offsets(dtype):
    big = rand(200, 400, seed=3, dtype=dtype)
    for x in (big[3:190, 5:300], big[:, :256], big[::2], big.t(), big[10:11], big[:, 7:8], big[5:5]):
        for blocks in ("both", "tiles"):
            for a, b in zip(ops.quantize_fp8(x, blocks), on_cpu(x.contiguous(), blocks)):
                same_matrix(a, b)


@pytest.mark.parametrize("blocks", ["both", "tiles"])
def test_quantize_special_values(blocks):
    v = torch.zeros(140, 260)
    v[1] = 448.0
    v[2, 5] = torch.nextafter(torch.tensor(448.0), torch.tensor(500.0))
    v[3, :3] = torch.tensor([math.inf, -math.inf, math.nan])
    v[3, 3] = 7.0
    v[4] = math.nan
    v[5, 0] = 3.0e38
    v[6, 0] = 1.0e-40
    v[7, 0], v[7, 1] = 1.0, 2.0 ** -20
    v[130, 200] = -2.0 ** -130
    v = v.to(DEV)
    for a, b in zip(ops.quantize_fp8(v, blocks), on_cpu(v, blocks)):
        same_matrix(a, b)


# --------------------------------------------------------------------------- product
def product_bounds(a, b, bias, dtype):
    """64-bit product of the quantised operands and what each element may be off by: the result's rounding
    (half a step) and the sums'. An 8-bit matrix instruction keeps its 64 products to 2^-12 of the sum of their
    magnitudes; the widened form rounds in 24 bits at each of its K / 16 instructions, and for the slices.
    Below the smallest normal number, 2^-126 in either dtype, nothing is promised: a product of the two largest
    values over 2^-127 scales has no relative precision left there (2^-190 is not representable at all)."""
    x, w = a.dequantize().double(), b.dequantize().double()
    want = x @ w.t()
    size = x.abs() @ w.abs().t()
    if bias is not None:
        want, size = want + bias.double(), size + bias.double().abs()
    size = size + 2.0 ** -126 * 2.0 ** 12
    if dtype == torch.bfloat16:
        return want, 2.0 ** -8 * want.abs() + 2.0 ** -12 * size
    size = size + 2.0 ** -126 * 2.0 ** 23
    return want, 2.0 ** -24 * want.abs() + (a.cols / 16 + 16) * 2.0 ** -23 * size


def check_product(a, b, bias, dtype, y):
    want, bound = product_bounds(a, b, bias, dtype)
    assert y.shape == want.shape and y.dtype == dtype
    off = (y.double() - want).abs()
    assert (off <= bound).all(), float((off / bound.clamp(min=1e-300)).max())


SIZES = [(1, 1, 1), (1, 32, 64), (5, 33, 129), (16, 3840, 1280), (128, 128, 128), (129, 257, 513), (300, 701, 1100), (33, 65, 5000),
         (2048, 2049, 640), (4100, 4096, 260)]


@pytest.mark.parametrize("m,n,k", SIZES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("tiles", [False, True])
def test_product(m, n, k, dtype, tiles):
    x, w = rand(m, k, seed=1), rand(n, k, seed=2)
    bias = rand(n, 1, seed=3)[:, 0].to(dtype) if tiles else None
    a = ops.quantize_fp8(x)
    b = ops.quantize_fp8(w, "tiles")[0] if tiles else ops.quantize_fp8(w)
    y = ops.fp8_matmul(a, b, bias, dtype)
    check_product(a, b, bias, dtype, y)
    assert torch.equal(y, ops.fp8_matmul(a, b, bias, dtype))  # the same bits again
    if tiles and m * n < 10 ** 6:
        check_product(b, a, None, dtype, ops.fp8_matmul(b, a, None, dtype))  # tiles on the left


@pytest.mark.parametrize("m,n,k", [(8192, 5120, 1280), (8100, 5001, 1300), (16500, 2600, 1400), (2000, 2048, 65536), (2000, 2001, 65536),
                                   (8192, 1280, 5120), (16384, 1403, 1300), (2000, 1501, 65536),
                                   (16384, 5120, 100), (16384, 5127, 100)])
@pytest.mark.parametrize("bias", [None, torch.bfloat16, torch.float32])
def test_product_of_many_tiles(m, n, k, bias):
    """Sizes at which a workgroup goes through several tiles, and through slices of a long contraction."""
    a, b = ops.quantize_fp8(rand(m, k, seed=1)), ops.quantize_fp8(rand(n, k, seed=2))
    c = None if bias is None else rand(n, 1, seed=3)[:, 0].to(bias)
    y = ops.fp8_matmul(a, b, c, torch.bfloat16)
    check_product(a, b, c, torch.bfloat16, y)
    for _ in range(3):
        assert torch.equal(y, ops.fp8_matmul(a, b, c, torch.bfloat16))


def test_bias_at_any_alignment():
    a, b = ops.quantize_fp8(rand(8192, 1300, seed=1)), ops.quantize_fp8(rand(5001, 1300, seed=2))
    c = rand(5003, 1, seed=3)[:, 0].bfloat16()[1:5002]
    check_product(a, b, c, torch.bfloat16, ops.fp8_matmul(a, b, c, torch.bfloat16))


def test_product_of_non_finite_values():
    x, w = rand(200, 300, seed=1), rand(140, 300, seed=2)
    x[3, 200], x[150, 7], w[9, 299] = math.inf, math.nan, -math.inf
    for dtype in (torch.bfloat16, torch.float32):
        y = ops.fp8_matmul(ops.quantize_fp8(x), ops.quantize_fp8(w), None, dtype)
        bad = torch.zeros(200, 140, dtype=torch.bool, device=DEV)
        bad[3], bad[150], bad[:, 9] = True, True, True
        assert torch.equal(torch.isnan(y), bad)


def test_product_scales_far_apart():
    """Scales near both ends of their range, and blocks of zeros."""
    x, w = rand(130, 512, seed=1, spread=0.0), rand(131, 512, seed=2, spread=0.0)
    x[:, 128:256] = 0
    x[0], x[1], w[0], w[1] = x[0] * 2.0 ** 100, x[1] * 2.0 ** -90, w[0] * 2.0 ** -100, w[1] * 2.0 ** 20
    a, b = ops.quantize_fp8(x), ops.quantize_fp8(w)
    for dtype in (torch.bfloat16, torch.float32):
        check_product(a, b, None, dtype, ops.fp8_matmul(a, b, None, dtype))


# --------------------------------------------------------------------------- layer
def layer_case(m, n, k, dtype, bias=True):
    x = rand(m, k, seed=4, dtype=dtype).requires_grad_()
    w = rand(n, k, seed=5, dtype=dtype, spread=0.0).requires_grad_()
    b = rand(n, 1, seed=6, dtype=dtype)[:, 0].clone().requires_grad_() if bias else None
    return x, w, b, rand(m, n, seed=7, dtype=dtype)


def check_layer(x, w, b, dy, y, dx, dw, db):
    dtype = x.dtype
    with torch.no_grad():
        check_product(ops.quantize_fp8(x), ops.quantize_fp8(w, "tiles")[0], b, dtype, y)
        check_product(ops.quantize_fp8(dy), ops.quantize_fp8(w, "tiles")[1], None, dtype, dx)
        check_product(ops.quantize_fp8(dy, "columns"), ops.quantize_fp8(x, "columns"), None, dtype, dw)
        if b is not None:
            want, size = dy.double().sum(0), dy.double().abs().sum(0)
            step = 2.0 ** -8 if dtype == torch.bfloat16 else 2.0 ** -24
            assert ((db.double() - want).abs() <= step * want.abs() + (dy.shape[0] / 128 + 16) * 2.0 ** -24 * size).all()


@pytest.mark.parametrize("m,n,k", [(1, 1, 1), (7, 40, 24), (200, 300, 129), (1000, 513, 257), (3000, 512, 1000), (4096, 2560, 1280), (8200, 1203, 5127)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_layer(m, n, k, dtype):
    x, w, b, dy = layer_case(m, n, k, dtype)
    y = ops.fp8_linear(x, w, b)
    check_layer(x, w, b, dy, y, *torch.autograd.grad(y, [x, w, b], dy))


def test_layer_integers_are_exact():
    g = torch.Generator(device=DEV).manual_seed(1)
    draw = lambda *s: torch.randint(-7, 8, s, generator=g, device=DEV).float()  # noqa: E731
    x, w, b, dy = draw(3, 70, 140).requires_grad_(), draw(133, 140).requires_grad_(), draw(133).requires_grad_(), draw(3, 70, 133)
    y = ops.fp8_linear(x, w, b)
    y.backward(dy)
    assert torch.equal(y.double(), x.double() @ w.double().t() + b.double())
    assert torch.equal(x.grad.double(), dy.double() @ w.double())
    assert torch.equal(w.grad.double(), dy.double().view(-1, 133).t() @ x.double().view(-1, 140))
    assert torch.equal(b.grad.double(), dy.double().sum((0, 1)))
    step = torch.zeros_like(x)
    step[1, 5, 130] = 2.0
    with torch.no_grad():
        assert ((ops.fp8_linear(x + step, w, b) - y).double() * dy.double()).sum() == 2.0 * x.grad[1, 5, 130].double()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_layer_accumulates_into_grad(dtype):
    x, w, b, dy = layer_case(300, 130, 140, dtype)
    want = torch.autograd.grad(ops.fp8_linear(x, w, b), [w, b], dy)
    for _ in range(2):
        ops.fp8_linear(x, w, b).backward(dy)
    before = w.grad.clone()
    again = torch.autograd.grad(ops.fp8_linear(x, w, b), [w, b], dy)  # asked for: returned, .grad left alone
    assert torch.equal(again[0], want[0]) and torch.equal(again[1], want[1]) and torch.equal(w.grad, before)
    step = 2.0 ** -8 if dtype == torch.bfloat16 else 2.0 ** -23
    for g, p in zip(want, (w, b)):  # twice the same sum: one more rounding
        assert ((p.grad.double() - 2 * g.double()).abs() <= 2 * step * 2 * g.double().abs().clamp(min=float(g.abs().max()) * 1e-3)).all()


def test_layer_gradient_sink():
    x, w, b, dy = layer_case(260, 130, 140, torch.bfloat16)
    plain = torch.autograd.grad(ops.fp8_linear(x, w, b), [w, b], dy)
    flat = torch.full((130 * 140 + 130,), 2.0, device=DEV)  # fp32 buffer of a reducer
    w._pda_grad_sink, b._pda_grad_sink = (lambda: (flat[:130 * 140], True)), (lambda: (flat[130 * 140:], False))
    w._pda_grad_sink_dtype = b._pda_grad_sink_dtype = torch.float32
    ops.fp8_linear(x, w, b).backward(dy)
    assert w.grad is None and b.grad is None
    gw, gb = flat[:130 * 140].view(130, 140) - 2.0, flat[130 * 140:]
    a, c = ops.quantize_fp8(dy, "columns"), ops.quantize_fp8(x.detach(), "columns")
    want = a.dequantize().double() @ c.dequantize().double().t()
    size = a.dequantize().double().abs() @ c.dequantize().double().abs().t() + 4.0
    assert ((gw.double() - want).abs() <= 40 * 2.0 ** -23 * size).all()
    assert ((gb.double() - plain[1].double()).abs() <= 2.0 ** -8 * gb.double().abs() + 1e-4).all()


def test_layer_empty_and_strided():
    w, b = rand(24, 40, seed=1).requires_grad_(), torch.ones(24, device=DEV, requires_grad=True)
    x = torch.zeros(0, 40, device=DEV, requires_grad=True)
    y = ops.fp8_linear(x, w, b)
    y.sum().backward()
    assert y.shape == (0, 24) and not w.grad.any() and not b.grad.any() and x.grad.shape == (0, 40)
    wide = rand(50, 200, seed=2)
    view, same = wide[:, 3:43], wide[:, 3:43].contiguous()
    dy = rand(24, 50, seed=3).t()  # a gradient that is not contiguous
    for p in (view.detach().requires_grad_(),):
        q = same.requires_grad_()
        a = torch.autograd.grad(ops.fp8_linear(p, w, b), [p, w, b], dy)
        c = torch.autograd.grad(ops.fp8_linear(q, w, b), [q, w, b], dy.contiguous())
        assert all(torch.equal(i, j) for i, j in zip(a, c))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("shape,out", [((2, 3, 0), 8), ((2, 3, 16), 0), ((2, 0, 16), 8), ((0, 3, 0), 4)])
def test_layer_without_elements(shape, out, dtype):
    make = lambda *s: torch.ones(s, device=DEV, dtype=dtype).requires_grad_()  # noqa: E731
    x, w, b = make(*shape), make(out, shape[-1]), make(out)
    y = ops.fp8_linear(x, w, b)
    assert y.shape == (*shape[:-1], out) and (y == (1.0 + shape[-1])).all()
    y.sum().backward()
    assert x.grad.shape == x.shape and (x.grad == out).all() and w.grad.shape == w.shape and (w.grad == shape[0] * shape[1]).all()
    assert (b.grad == shape[0] * shape[1]).all()


@pytest.mark.parametrize("m,n,k", [(0, 5, 200), (7, 0, 200), (7, 5, 0), (0, 0, 0)])
def test_product_without_elements(m, n, k):
    a, b = ops.quantize_fp8(torch.ones(m, k, device=DEV)), ops.quantize_fp8(torch.ones(n, k, device=DEV))
    c = torch.arange(n, device=DEV, dtype=torch.float32)
    for dtype in (torch.bfloat16, torch.float32):
        y = ops.fp8_matmul(a, b, c, dtype)
        assert y.dtype == dtype and torch.equal(y.float(), (c + k).expand(m, n))


def test_no_second_derivative():
    x, w, b, dy = layer_case(20, 30, 40, torch.bfloat16)
    y = ops.fp8_linear(x, w, b)
    with pytest.raises(RuntimeError, match="second derivative"):
        torch.autograd.grad(y, [x], dy, create_graph=True)


def test_two_graphs_in_turn():
    """Two captured layers, replayed in turn and beside each other's eager form: neither uses the other's workspace."""
    made = []
    for m, n, k in ((700, 256, 384), (130, 1000, 2600)):
        x, w, b, dy = layer_case(m, n, k, torch.bfloat16)
        want = [t.clone() for t in torch.autograd.grad(ops.fp8_linear(x, w, b), [x, w, b], dy)]
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = torch.autograd.grad(ops.fp8_linear(x, w, b), [x, w, b], dy)
        made.append((graph, got, want, (x, w, b, dy)))
    for _ in range(3):
        for graph, *_ in made:
            graph.replay()
        for _, got, want, (x, w, b, dy) in made:
            assert all(torch.equal(i, j) for i, j in zip(got, want))
            assert all(torch.equal(i, j) for i, j in zip(torch.autograd.grad(ops.fp8_linear(x, w, b), [x, w, b], dy), want))


def test_side_stream_and_graph():
    x, w, b, dy = layer_case(512, 256, 384, torch.bfloat16)
    want = [t.clone() for t in (lambda y: (y.detach(), *torch.autograd.grad(y, [x, w, b], dy)))(ops.fp8_linear(x, w, b))]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        y = ops.fp8_linear(x, w, b)
        got = [y.detach(), *torch.autograd.grad(y, [x, w, b], dy)]
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(i, j) for i, j in zip(got, want))
    del y, got
    graph = torch.cuda.CUDAGraph()
    xs, dys = x.detach().clone().requires_grad_(), dy.clone()
    with torch.cuda.graph(graph):
        y = ops.fp8_linear(xs, w, b)
        got = [y.detach(), *torch.autograd.grad(y, [xs, w, b], dys)]
    for k in range(3):  # new values between the replays, eager work beside them
        with torch.no_grad():
            xs.copy_(x * (k + 1))
            dys.copy_(dy * (k + 2))
        graph.replay()
        xk = (x.detach() * (k + 1)).requires_grad_()
        yk = ops.fp8_linear(xk, w, b)
        wantk = [yk.detach(), *torch.autograd.grad(yk, [xk, w, b], dy * (k + 2))]
        assert all(torch.equal(i, j) for i, j in zip(got, wantk)), k
        torch.cuda.synchronize()


def test_native_checks():
    """What the Python layer would refuse is refused by the extension too."""
    ext = _ext.require()
    a, b = ops.quantize_fp8(rand(8, 300)), ops.quantize_fp8(rand(8, 300))
    with pytest.raises(RuntimeError, match="padded to 128"):
        ext.fp8_matmul(a.q, a.scale, False, b.q, b.scale, False, 400, None, False)
    with pytest.raises(RuntimeError, match="scales"):
        ext.fp8_matmul(a.q, a.scale[:, :2].contiguous(), False, b.q, b.scale, False, 300, None, False)
    with pytest.raises(RuntimeError, match="bias"):
        ext.fp8_matmul(a.q, a.scale, False, b.q, b.scale, False, 300, torch.zeros(7, device=DEV), False)
    with pytest.raises(RuntimeError, match="float8"):
        ext.fp8_matmul(a.q.view(torch.uint8), a.scale, False, b.q, b.scale, False, 300, None, False)
    with pytest.raises(RuntimeError, match="contiguous"):
        ext.fp8_quantize(rand(8, 300).t(), True, False, False)
