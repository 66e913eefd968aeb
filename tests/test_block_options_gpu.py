"""8-bit linear layers and sliding-window attention together, as the models run them: every call of a training step
against the 64-bit definition on the call's own operands, recomputation, fp32 gradient buffers, a captured step."""
import pytest
import torch

from pytorch_distributed_amd import ops
from pytorch_distributed_amd.models import LlamaForCausalLM, MyGPT2LMHeadModel, get_config
from tests import test_fp8_gpu as fp8
from tests import test_window_attention_gpu as win

pytestmark = pytest.mark.gpu
DEV = "cuda"
OPTIONS = dict(linear_precision="fp8", sliding_window=50, attention_sinks=3)


def build(name, policy="none", dtype=torch.bfloat16, **options):
    torch.manual_seed(0)
    cfg = get_config(name, **{**OPTIONS, **options}).without_dropout()
    cls = LlamaForCausalLM if name.startswith("llama") else MyGPT2LMHeadModel
    return cls(cfg, activation_checkpoint=policy).to(device=DEV, dtype=dtype)


def batch(n=2, T=128, vocab=512, seed=1):
    ids = torch.randint(0, vocab, (n, T + 1), generator=torch.Generator().manual_seed(seed)).to(DEV)
    return ids[:, :-1].contiguous(), ids[:, 1:].contiguous()


def step(model, x, y):
    for p in model.parameters():
        p.grad = None
    loss = model(x, y)
    loss.backward()
    return loss.detach(), {n: p.grad.clone() for n, p in model.named_parameters()}


@pytest.mark.parametrize("name", ["gpt2-tiny", "llama-tiny"])
@pytest.mark.parametrize("T", [128, 77])
def test_every_call_of_a_step(name, T, monkeypatch):
    linears, windows = [], []
    real_linear, real_window = ops.fp8_linear, ops.window_attention

    def linear(x, weight, bias=None, regen=None):
        xr = x.detach().clone().requires_grad_()  # the call's own leaf, so that its input gradient can be read
        y = real_linear(xr, weight, bias, regen)
        linears.append((xr, weight, bias, y))
        return _Join.apply(x, [y, xr])

    def window(qkv, H, w, s, **kw):
        leaf = qkv.detach().clone().requires_grad_()
        out = real_window(leaf, H, w, s, **kw)
        windows.append((leaf, H, w, s, out))
        return _Join.apply(qkv, [out, leaf])

    monkeypatch.setattr(ops, "fp8_linear", linear)
    monkeypatch.setattr(ops, "window_attention", window)
    model = build(name)
    x, y = batch(T=T)
    model(x, y).backward()
    assert len(linears) == 8 and len(windows) == 2
    for xr, w, b, out in linears:
        dy = out.dy.reshape(-1, out.shape[-1])
        x2 = xr.detach().reshape(-1, xr.shape[-1])
        leaves = [x2.requires_grad_(), w] + ([b] if b is not None else [])
        y2 = real_linear(x2, w, b)
        g = torch.autograd.grad(y2, leaves, dy)
        assert torch.equal(y2, out.reshape(-1, out.shape[-1])) and torch.equal(g[0], xr.grad.reshape(g[0].shape))
        fp8.check_layer(x2, w, b, dy, y2, g[0], g[1], g[2] if b is not None else None)
    for leaf, H, w, s, out in windows:
        want, tol, wg, tg = win.oracle(leaf, out.dy, H, w, s)
        win.check(out, want, tol)
        win.check(leaf.grad, wg, tg)


class _Join(torch.autograd.Function):
    """Passes a recorded call's result on as a function of `x`; in backward runs that call's own graph."""

    @staticmethod
    def forward(ctx, x, call):
        ctx.out, ctx.leaf = call
        return ctx.out.detach().clone()

    @staticmethod
    def backward(ctx, dy):
        ctx.out.dy = dy.detach().clone()
        with torch.enable_grad():
            torch.autograd.backward(ctx.out, dy)
        return ctx.leaf.grad, None


@pytest.mark.parametrize("name", ["gpt2-tiny", "llama-tiny"])
def test_recomputation_policies_agree(name):
    x, y = batch()
    want = step(build(name, "none"), x, y)
    for policy in ("selective", "full"):
        got = step(build(name, policy), x, y)
        assert torch.equal(want[0], got[0])
        for n in want[1]:
            assert torch.equal(want[1][n], got[1][n]), (policy, n)


def test_fp32_gradient_buffers_and_windows():
    """Two micro-batches into fp32 buffers (gradient sinks): the sum of the two bf16 gradients up to their own
    rounding, also inside an accumulation window."""
    from pytorch_distributed_amd.parallel import GradAccumulator

    x, y = batch(4)
    model = build("gpt2-tiny")
    parts = [step(model, x[i:i + 2], y[i:i + 2])[1] for i in (0, 2)]
    for p in model.parameters():
        p.grad = None
    acc = GradAccumulator(model, grad_accum_dtype="fp32")
    for i in range(2):
        with ops.accumulation_window(i, 2):
            ctx = acc.no_sync() if i == 0 else torch.enable_grad()
            with ctx:
                acc(x[2 * i:2 * i + 2], y[2 * i:2 * i + 2]).backward()
    for n, p in model.named_parameters():
        a, b = (g[n].double() for g in parts)
        # each part and the sum are rounded to bf16; products into a buffer take the 24-bit form of the sums
        # (2^-12 of the products' magnitudes apart, which the gradients' largest entries bound here)
        bound = 2.0 ** -8 * (a.abs() + b.abs() + (a + b).abs()) + 2.0 ** -7 * max(a.abs().max(), b.abs().max())
        assert ((p.grad.double() - a - b).abs() <= bound).all(), n


def test_fp32_storage():
    model = build("gpt2-tiny", dtype=torch.float32)
    x, y = batch()
    loss, g = step(model, x, y)
    assert loss.dtype == torch.float32 and all(t.dtype == torch.float32 and torch.isfinite(t).all() for t in g.values())


def test_captured_training_step():
    from pytorch_distributed_amd.optim import FusedAdamW
    from pytorch_distributed_amd.utils.graphs import GraphedTrainStep

    def losses(graphed):
        model = build("llama-tiny")
        opt = FusedAdamW(model.parameters(), lr=1e-3, capturable=True)
        run = GraphedTrainStep(model, opt, 2, 64, warmup_steps=2) if graphed else None
        out = []
        for k in range(6):
            x, y = batch(2, 64, seed=k)
            if graphed:
                out.append(run(x, y).clone())
            else:
                loss = model(x, y)
                loss.backward()
                opt.step(zero_grad=True)
                out.append(loss.detach().float())
            torch.cuda.synchronize()
        return torch.stack([t.reshape(()) for t in out]), model

    eager, m0 = losses(False)
    replayed, m1 = losses(True)
    assert torch.equal(eager, replayed)
    for (n, a), (_, b) in zip(m0.named_parameters(), m1.named_parameters()):
        assert torch.equal(a, b), n


def test_training_step_runs_with_dropout():
    torch.manual_seed(0)
    model = MyGPT2LMHeadModel(get_config("gpt2-tiny", **OPTIONS)).to(device=DEV, dtype=torch.bfloat16).train()
    x, y = batch()
    loss, g = step(model, x, y)
    assert torch.isfinite(loss) and all(torch.isfinite(t).all() for t in g.values())
