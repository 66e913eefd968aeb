"""8-bit linear layers and sliding-window attention under the multi-rank runtimes with the GPU kernels: ranks sharing one
card against a single process on the whole batch."""
import pytest
import torch

from tests import test_shared_gpu_rehearsal_gpu as rehearsal
from tests.dist_utils import run_distributed

pytestmark = pytest.mark.gpu
OPTIONS = dict(linear_precision="fp8", sliding_window=100, attention_sinks=4)


def _model(seed, n_layer=2):
    from pytorch_distributed_amd.models import MyGPT2LMHeadModel, get_config

    torch.manual_seed(seed)
    cfg = get_config("gpt2", n_layer=n_layer, **OPTIONS).without_dropout()
    return MyGPT2LMHeadModel(cfg).to(device="cuda", dtype=torch.bfloat16), cfg


def _train(rank, world, kind, accum):
    rehearsal._model = _model  # (in the rank's own process)
    rehearsal._train(rank, world, kind, accum)


@pytest.mark.parametrize("kind,world,accum", [("ddp", 2, 2), ("ddp_fp32", 2, 2), ("FULL_SHARD", 2, 2), ("SHARD_GRAD_OP", 2, 1),
                                              ("FULL_SHARD_units2", 2, 2)])
def test_multi_rank_training_matches_single_process(kind, world, accum, monkeypatch):
    monkeypatch.setenv("PDA_SHARED_GPU", "1")
    run_distributed(_train, world=world, args=(kind, accum), timeout=110.0, backend="rccl")
