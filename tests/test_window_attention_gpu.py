"""The sliding-window attention kernels against plain 64-bit computations."""
import math

import pytest
import torch

from pytorch_distributed_amd import _ext, ops

pytestmark = pytest.mark.gpu
DEV = "cuda"
HALF = 2.0 ** -8  # half a step of bf16, relative


def inputs(B, T, H, D, seed=0, size=1.0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    qkv = (size * torch.randn(B, T, 3 * H * D, generator=g, device=DEV)).to(torch.bfloat16)
    return qkv, torch.randn(B, T, H * D, generator=g, device=DEV).to(torch.bfloat16)


def oracle(qkv, dout, H, window, sinks, scale=None, keep=None, keep_scale=1.0):
    """(out, dqkv) in 64 bits and how far each element of a kernel's may be off.

    Rounded to bf16 are: P as the operand of P V and of P^T dO, O, dS as the operand of dS K and dS^T Q, and the
    gradients. So, with p = softmax probabilities, |d out| <= HALF (sum p |v| + |out|); the row constant
    delta = dO . O inherits that error; |d dS| <= p |d delta| + HALF |dS|. fp32 scores, exponentials and sums add
    2^-12 of the same magnitudes at the most (scores of some tens, each good to 2^-20)."""
    B, T, width = qkv.shape
    D = width // (3 * H)
    scale = 1.0 / math.sqrt(D) if scale is None else scale
    q, k, v = (t.transpose(1, 2).contiguous() for t in qkv.detach().double().view(B, T, 3, H, D).unbind(2))
    do = dout.double().view(B, T, H, D).transpose(1, 2).contiguous()
    i = torch.arange(T, device=qkv.device)
    age = i[:, None] - i[None, :]
    seen = (age >= 0) & ((age < window) | (i[None, :] < sinks))
    s = (q @ k.transpose(2, 3).contiguous() * scale).masked_fill(~seen, -math.inf)
    p = torch.softmax(s, -1)
    m = torch.ones_like(p) if keep is None else keep.double() * keep_scale
    pm = p * m
    small = 2.0 ** -12
    out = pm @ v
    spread = pm @ v.abs()
    out_tol = HALF * (spread + out.abs()) * 1.01 + small * spread
    delta = (do * out).sum(-1, keepdim=True)
    delta_tol = (do.abs() * out_tol).sum(-1, keepdim=True)
    dp = (do @ v.transpose(2, 3).contiguous()) * m
    ds = p * (dp - delta)
    size = p * (do.abs() @ v.abs().transpose(2, 3).contiguous() * m + (do.abs() * spread).sum(-1, keepdim=True))
    ds_tol = p * delta_tol + HALF * ds.abs() * 1.01 + small * size
    dst, dstt = ds.transpose(2, 3).contiguous(), ds_tol.transpose(2, 3).contiguous()
    dq, dk, dv = ds @ k * scale, dst @ q * scale, pm.transpose(2, 3).contiguous() @ do
    pt = pm.transpose(2, 3).contiguous() @ do.abs()
    tol = [ds_tol @ k.abs() * scale + HALF * dq.abs(), dstt @ q.abs() * scale + HALF * dk.abs(), (HALF * 1.01 + small) * pt + HALF * dv.abs()]
    join = lambda ts: torch.stack([t.transpose(1, 2) for t in ts], 2).reshape(B, T, width)  # noqa: E731
    flat = lambda t: t.transpose(1, 2).reshape(B, T, H * D)  # noqa: E731
    return flat(out), flat(out_tol), join([dq, dk, dv]), join(tol)


def check(got, want, tol):
    off = (got.double() - want).abs()
    assert torch.isfinite(got).all()
    assert (off <= tol + 1e-30).all(), float((off / (tol + 1e-30)).max())


def run(qkv, dout, H, window, sinks, **kw):
    leaf = qkv.detach().clone().requires_grad_()
    out = ops.window_attention(leaf, H, window, sinks, **kw)
    (g,) = torch.autograd.grad(out, leaf, dout)
    return out.detach(), g


CASES = [(1, 1, 1, 64, 1, 0), (1, 2, 1, 128, 1, 1), (2, 5, 2, 128, 3, 1), (1, 64, 1, 64, 64, 0), (1, 65, 2, 64, 1, 0), (2, 128, 2, 64, 32, 0),
         (2, 200, 2, 128, 1, 5), (3, 333, 5, 64, 100, 5), (1, 700, 2, 128, 64, 70), (1, 1000, 2, 64, 37, 130), (1, 1000, 1, 128, 500, 200),
         (1, 1024, 1, 64, 2000, 3), (1, 2000, 1, 128, 129, 64), (1, 513, 3, 64, 128, 513), (1, 4100, 1, 64, 65, 1), (1, 4096, 2, 128, 1024, 4)]


@pytest.mark.parametrize("B,T,H,D,window,sinks", CASES)
def test_forward_and_backward(B, T, H, D, window, sinks):
    qkv, dout = inputs(B, T, H, D, seed=T)
    out, g = run(qkv, dout, H, window, sinks)
    want, tol, wg, tg = oracle(qkv, dout, H, window, sinks)
    check(out, want, tol)
    check(g, wg, tg)
    again, g2 = run(qkv, dout, H, window, sinks)
    assert torch.equal(out, again) and torch.equal(g, g2)  # the same bits again


def test_large_scores():
    """Scores of several hundreds: the running maximum has to move with the tiles, also towards the sinks."""
    qkv, dout = inputs(1, 400, 2, 64, seed=1)
    v = qkv.view(1, 400, 3, 2, 64)
    v[:, :3, 1] *= 30.0
    v[:, 100:110, 1] *= 20.0
    out, _ = run(qkv, dout, 2, 90, 3)
    want, tol, _, _ = oracle(qkv, dout, 2, 90, 3)
    check(out, want, tol + 2.0 ** -8 * want.abs())  # scores of 2^9 are good to 2^-12 in the exponent


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("slope", [-0.2, -0.05, -0.01, 0.01, 0.2])
def test_scores_that_grow_from_tile_to_tile(D, slope):
    """Scores rise or fall steadily with the key's age, a little or a lot per tile, and reach some 120."""
    T, window, sinks = 600, 500, 70
    qkv, dout = inputs(1, T, 1, D, seed=21, size=0.05)
    v = qkv.view(1, T, 3, D)
    v[:, :, 0, 0], v[:, :, 1, 0] = 1.0, slope * math.sqrt(D) * torch.arange(T, device=DEV)
    v[:, :, 2] *= 20.0
    out, g = run(qkv, dout, 1, window, sinks)
    want, tol, wg, tg = oracle(qkv, dout, 1, window, sinks)
    check(out, want, tol)
    check(g, wg, tg)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("window,sinks", [(50, 3), (150, 40)])
def test_dropout(D, window, sinks):
    B, T, H, p, seed = 2, 300, 2, 0.25, 1234
    qkv, dout = inputs(B, T, H, D, seed=5)
    out, g = run(qkv, dout, H, window, sinks, dropout_p=p, training=True, seed=seed)
    keep = _ext.require().attention_dropout_mask(B, H, T, p, seed, torch.device(DEV))
    want, tol, wg, tg = oracle(qkv, dout, H, window, sinks, keep=keep, keep_scale=4.0 / 3.0)
    check(out, want, tol)
    check(g, wg, tg)
    plain, _ = run(qkv, dout, H, window, sinks, dropout_p=p, training=False)
    want, tol, _, _ = oracle(qkv, dout, H, window, sinks)
    check(plain, want, tol)
    torch.manual_seed(3)
    a, _ = run(qkv, dout, H, window, sinks, dropout_p=p, training=True)
    torch.manual_seed(3)
    b, _ = run(qkv, dout, H, window, sinks, dropout_p=p, training=True)
    assert torch.equal(a, b)


def test_wide_window_matches_causal_attention():
    qkv, dout = inputs(2, 300, 2, 64, seed=9)
    want, tol, _, _ = oracle(qkv, dout, 2, 300, 0)
    check(ops.causal_attention(qkv, 2), want, tol)
    check(ops.window_attention(qkv, 2, 300), want, tol)


def test_scale_strides_and_fp32():
    qkv, dout = inputs(2, 150, 2, 64, seed=11)
    out, g = run(qkv, dout, 2, 40, 2, scale=0.05)
    want, tol, wg, tg = oracle(qkv, dout, 2, 40, 2, scale=0.05)
    check(out, want, tol)
    check(g, wg, tg)
    wide = torch.zeros(2, 150, 2 * 3 * 128 + 8, device=DEV, dtype=torch.bfloat16)
    view = wide[:, :, 1:1 + 384]  # rows apart and off 16 bytes
    view.copy_(qkv)
    late = torch.zeros(dout.numel() + 1, device=DEV, dtype=torch.bfloat16)[1:].view_as(dout)  # contiguous, 2-byte aligned
    late.copy_(dout)
    out, g = run(qkv, dout, 2, 40, 2)
    leaf = view.detach().requires_grad_()
    o2 = ops.window_attention(leaf, 2, 40, 2)
    (g2,) = torch.autograd.grad(o2, leaf, late)
    assert torch.equal(out, o2) and torch.equal(g, g2)
    o32, g32 = run(qkv.float(), dout.float(), 2, 40, 2)
    assert o32.dtype == torch.float32 and torch.equal(o32, out.float()) and torch.equal(g32, g.float())


def test_keys_outside_the_window_do_not_matter():
    """Other values in keys that a query does not see leave its result and gradients as they were, to the bit."""
    qkv, dout = inputs(1, 600, 1, 64, seed=13)
    other = qkv.clone()
    other.view(1, 600, 3, 64)[:, 10:200] = 3.0  # seen by no query from 300 on (window 100, 10 sinks)
    a, _ = run(qkv, dout, 1, 100, 10)
    b, _ = run(other, dout, 1, 100, 10)
    assert torch.equal(a[:, 300:], b[:, 300:]) and torch.equal(a[:, :10], b[:, :10])


def test_side_stream_and_graph():
    H, window, sinks = 2, 100, 4
    qkv, dout = inputs(2, 700, H, 64, seed=17)
    want = run(qkv, dout, H, window, sinks)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = run(qkv, dout, H, window, sinks)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    leaf, do = qkv.detach().clone().requires_grad_(), dout.clone()
    with torch.cuda.graph(graph):
        out = ops.window_attention(leaf, H, window, sinks)
        (g,) = torch.autograd.grad(out, leaf, do)
    for k in range(3):
        with torch.no_grad():
            leaf.copy_(qkv * (1 + 0.25 * k))
            do.copy_(dout * (k + 1))
        graph.replay()
        eager = run(qkv * (1 + 0.25 * k), dout * (k + 1), H, window, sinks)
        assert torch.equal(out, eager[0]) and torch.equal(g, eager[1]), k
        torch.cuda.synchronize()


def test_no_second_derivative():
    qkv, dout = inputs(1, 70, 1, 64)
    leaf = qkv.requires_grad_()
    with pytest.raises(RuntimeError, match="second derivative"):
        torch.autograd.grad(ops.window_attention(leaf, 1, 20), leaf, dout, create_graph=True)


def test_two_graphs_in_turn():
    made = []
    for T, H, D, window, sinks in ((900, 2, 64, 100, 4), (500, 3, 128, 64, 70)):
        qkv, dout = inputs(1, T, H, D, seed=T)
        want = run(qkv, dout, H, window, sinks)
        leaf = qkv.detach().clone().requires_grad_()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = ops.window_attention(leaf, H, window, sinks)
            (g,) = torch.autograd.grad(out, leaf, dout)
        made.append((graph, (out, g), want, (qkv, dout, H, window, sinks)))
    for _ in range(3):
        for graph, *_ in made:
            graph.replay()
        for _, got, want, args in made:
            assert all(torch.equal(a, b) for a, b in zip(got, want))
            assert all(torch.equal(a, b) for a, b in zip(run(*args), want))


def test_empty_batch_and_refusals():
    assert ops.window_attention(torch.zeros(0, 8, 192, device=DEV, dtype=torch.bfloat16), 1, 4).shape == (0, 8, 64)
    with pytest.raises(NotImplementedError, match="head size"):
        ops.window_attention(torch.zeros(1, 8, 96, device=DEV, dtype=torch.bfloat16), 1, 4)
    with pytest.raises(NotImplementedError, match="dtype"):
        ops.window_attention(torch.zeros(1, 8, 192, device=DEV, dtype=torch.float16), 1, 4)
    with pytest.raises(ValueError, match="positive scale"):
        ops.window_attention(torch.zeros(1, 8, 192, device=DEV, dtype=torch.bfloat16), 1, 4, scale=-1.0)
    ext = _ext.require()
    good = torch.zeros(1, 8, 192, device=DEV, dtype=torch.bfloat16)
    with pytest.raises(RuntimeError, match="window must be"):
        ext.window_attention_forward(good, 1, 0, 0, 0.125, 0.0, 0)
    with pytest.raises(RuntimeError, match="sinks must"):
        ext.window_attention_forward(good, 1, 1, -1, 0.125, 0.0, 0)
    with pytest.raises(RuntimeError, match="head_dim"):
        ext.window_attention_forward(torch.zeros(1, 8, 96, device=DEV, dtype=torch.bfloat16), 1, 1, 0, 0.125, 0.0, 0)
