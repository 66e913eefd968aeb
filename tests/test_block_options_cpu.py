"""8-bit linear layers and sliding-window attention inside the models, on the CPU reference paths."""
import copy
import dataclasses
import types

import pytest
import torch

from pytorch_distributed_amd import ops
from pytorch_distributed_amd.models import LlamaForCausalLM, MyGPT2LMHeadModel, get_config, normalize_gpt2_config
from pytorch_distributed_amd.utils import cli
from pytorch_distributed_amd.utils.flops import model_flops_per_token
from tests.dist_utils import run_distributed


def build(name, policy="none", seed=0, **options):
    torch.manual_seed(seed)
    cfg = get_config(name, **options).without_dropout()
    cls = LlamaForCausalLM if name.startswith("llama") else MyGPT2LMHeadModel
    return cls(cfg, activation_checkpoint=policy)


def batch(n=2, T=40, vocab=512, seed=1):
    ids = torch.randint(0, vocab, (n, T + 1), generator=torch.Generator().manual_seed(seed))
    return ids[:, :-1].contiguous(), ids[:, 1:].contiguous()


def grads(model, x, y):
    model.zero_grad()
    loss = model(x, y)
    loss.backward()
    return loss.detach(), {n: p.grad.clone() for n, p in model.named_parameters()}


@pytest.mark.parametrize("name", ["gpt2-tiny", "llama-tiny"])
def test_a_window_of_the_whole_context_changes_nothing(name):
    x, y = batch()
    plain, wide = build(name), build(name, sliding_window=64, attention_sinks=2)
    (l0, g0), (l1, g1) = grads(plain, x, y), grads(wide, x, y)
    assert torch.allclose(l0, l1, rtol=1e-5)
    for n in g0:
        assert torch.allclose(g0[n], g1[n], rtol=1e-3, atol=1e-6), n
    narrow, _ = grads(build(name, sliding_window=4), x, y)
    assert not torch.allclose(narrow, l0, rtol=1e-6)


@pytest.mark.parametrize("name", ["gpt2-tiny", "llama-tiny"])
def test_options_reach_every_layer(name, monkeypatch):
    calls = {"fp8": 0, "window": []}
    fp8, window = ops.fp8_linear, ops.window_attention
    monkeypatch.setattr(ops, "fp8_linear", lambda *a, **k: calls.__setitem__("fp8", calls["fp8"] + 1) or fp8(*a, **k))
    monkeypatch.setattr(ops, "window_attention", lambda *a, **k: calls["window"].append(a[2:4]) or window(*a, **k))
    model = build(name, linear_precision="fp8", sliding_window=7, attention_sinks=3)
    x, y = batch()
    grads(model, x, y)
    assert calls["fp8"] == 4 * model.config.n_layer if hasattr(model, "config") else calls["fp8"] == 8
    assert calls["window"] == [(7, 3)] * 2


@pytest.mark.parametrize("name", ["gpt2-tiny", "llama-tiny"])
def test_recomputation_policies_agree(name):
    options = dict(linear_precision="fp8", sliding_window=9, attention_sinks=2)
    x, y = batch()
    want = grads(build(name, "none", **options), x, y)
    for policy in ("selective", "full"):
        got = grads(build(name, policy, **options), x, y)
        assert torch.equal(want[0], got[0])
        for n in want[1]:
            assert torch.equal(want[1][n], got[1][n]), (policy, n)


def _ddp_fp8(rank, world):
    from pytorch_distributed_amd.parallel import DDP

    options = dict(linear_precision="fp8", sliding_window=9, attention_sinks=2)
    model = build("gpt2-tiny", **options)
    x, y = batch(4)
    # a rank's gradient is its own half's; the ranks' mean is what one process gets from the two halves
    halves = [grads(copy.deepcopy(model), x[2 * r:2 * r + 2], y[2 * r:2 * r + 2])[1] for r in range(world)]
    ddp = DDP(model)
    ddp(x[2 * rank:2 * rank + 2], y[2 * rank:2 * rank + 2]).backward()
    for n, p in model.named_parameters():
        mean = sum(h[n] for h in halves) / world
        assert torch.allclose(p.grad, mean, rtol=1e-5, atol=1e-7), n


def test_ddp():
    run_distributed(_ddp_fp8, 2)


def _fsdp_fp8(rank, world):
    from pytorch_distributed_amd.parallel import ShardingStrategy, fsdp_wrap_gpt

    options = dict(linear_precision="fp8", sliding_window=9, attention_sinks=2)
    model = build("gpt2-tiny", **options)
    x, y = batch(4)
    alone = [float(copy.deepcopy(model)(x[2 * r:2 * r + 2], y[2 * r:2 * r + 2])) for r in range(world)]
    wrapped = fsdp_wrap_gpt(model, ShardingStrategy.FULL_SHARD)
    loss = wrapped(x[2 * rank:2 * rank + 2], y[2 * rank:2 * rank + 2])
    assert abs(float(loss) - alone[rank]) < 1e-5
    loss.backward()
    assert all(torch.isfinite(p.grad).all() for p in wrapped.parameters() if p.grad is not None)


def test_fsdp():
    run_distributed(_fsdp_fp8, 2)


def test_refusals_and_plumbing():
    with pytest.raises(ValueError, match="linear_precision"):
        build("gpt2-tiny", linear_precision="int4")
    with pytest.raises(ValueError, match="sliding_window"):
        build("llama-tiny", sliding_window=0)
    with pytest.raises(ValueError, match="needs a sliding_window"):
        build("gpt2-tiny", attention_sinks=2)
    with pytest.raises(ValueError, match="negative"):
        build("gpt2-tiny", sliding_window=3, attention_sinks=-1)
    cfg = get_config("gpt2-tiny", linear_precision="fp8", sliding_window=5)
    assert dataclasses.asdict(cfg)["sliding_window"] == 5 and normalize_gpt2_config(cfg) is cfg
    ap = cli.add_common_args(__import__("argparse").ArgumentParser())
    args = ap.parse_args(["--model", "llama-tiny", "--linear-precision", "fp8", "--sliding-window", "16", "--attention-sinks", "2"])
    model, cfg = cli.build_model(args, "cpu", torch.float32)
    assert model.transformer.h[0].attn.sliding_window == 16 and model.transformer.h[0].attn.linear is ops.fp8_linear
    plain, _ = cli.build_model(ap.parse_args(["--model", "llama-tiny"]), "cpu", torch.float32)
    # 12 L d per token and visible key
    assert model_flops_per_token(plain, 128) - model_flops_per_token(model, 128) == 12.0 * 2 * 256 * (128 - 18)


def test_build_refuses_spilling_kernels():
    """The build's check of kernels that must not spill, on the compiler's own wording."""
    from pytorch_distributed_amd._build import spilling_kernels
    report = """a.hip:3:1: remark: Function Name: first [-Rpass-analysis=kernel-resource-usage]
a.hip:3:1: remark:     ScratchSize [bytes/lane]: 0 [-Rpass-analysis=kernel-resource-usage]
a.hip:9:1: remark: Function Name: second [-Rpass-analysis=kernel-resource-usage]
a.hip:9:1: remark:     ScratchSize [bytes/lane]: 52 [-Rpass-analysis=kernel-resource-usage]
"""
    assert spilling_kernels(report) == ["second"] and spilling_kernels("") == []


def test_a_configuration_without_the_options_has_their_defaults():
    """Any object with the fields that the models read is a configuration; the options are optional."""
    fields = {k: v for k, v in dataclasses.asdict(get_config("llama-tiny")).items()
              if k not in ("linear_precision", "sliding_window", "attention_sinks")}
    cfg = types.SimpleNamespace(**fields, head_dim=get_config("llama-tiny").head_dim)
    torch.manual_seed(0)
    model = LlamaForCausalLM(cfg, activation_checkpoint="none")
    x, y = batch()
    assert torch.equal(model(x, y), build("llama-tiny")(x, y))
    assert model_flops_per_token(model, 64) == model_flops_per_token(build("llama-tiny"), 64)
    cfg.sliding_window = 16
    assert model_flops_per_token(model, 64) == model_flops_per_token(build("llama-tiny", sliding_window=16), 64)
