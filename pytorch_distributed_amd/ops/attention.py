"""Causal self-attention over a packed QKV activation.

``causal_attention(qkv, num_heads)`` takes the ``[B, T, 3*H*D]`` output of the
fused QKV projection and returns ``[B, T, H*D]``. On the GPU this is one
flash-style forward kernel and two backward kernels (``csrc/kernels/
attention_*.hip``) that read Q, K and V in place with strides; the
``[B, H, T, T]`` score tensor the reference materialises
(assignments/assignment1/model/my_gpt2.py:60-77) never exists, and no causal
mask buffer is needed.

Attention-probability dropout (``attn_pdrop > 0`` in training mode, the setting of
every Hugging Face GPT-2 config) runs inside the same kernels: the keep mask is a
counter-based Philox function of (seed, batch, head, query, key), regenerated by the
backward kernels instead of being stored. The seed of each call is drawn from PyTorch's
CPU generator, so ``torch.manual_seed`` makes runs repeatable and activation
recomputation (which restores the RNG state) reproduces the same mask. The drop
probability is quantised to a multiple of 1/256.

fp32 activations on the GPU (``--dtype fp32``, the reference's storage precision) use the same
kernels: Q, K and V are rounded to bf16 for the MFMA products, accumulation and the softmax are
fp32, the result is widened back. Any other GPU input (head sizes other than 64 / 128, fp16) is an
error — there is no eager fallback on the GPU.

``attention_reference`` is the reference's eager op sequence in fp32 and is the
oracle of the kernel tests (``PDA_FORCE_REFERENCE=1`` routes every op to its oracle); with
``keep_mask`` it applies a given dropout mask.
"""
from __future__ import annotations

import math

import torch
import torch.nn.functional as F

from .. import _ext


def visible_mask(T: int, window: int | None = None, sinks: int = 0, device=None) -> torch.Tensor:
    """``[T, T]`` bool: may query t (row) see key s (column)? Causal, and with a ``window`` only where
    ``t - s < window`` or ``s < sinks``."""
    mask = torch.ones(T, T, dtype=torch.bool, device=device).tril()
    if window is not None:
        near = torch.ones(T, T, dtype=torch.bool, device=device).triu(1 - min(window, T))
        near[:, :sinks] = True
        mask &= near
    return mask


def attention_reference(qkv: torch.Tensor, num_heads: int, scale: float | None = None,
                        dropout_p: float = 0.0, training: bool = False, keep_mask=None,
                        keep_scale: float | None = None, window: int | None = None, sinks: int = 0) -> torch.Tensor:
    B, T, three_hd = qkv.shape
    D = three_hd // (3 * num_heads)
    scale = 1.0 / math.sqrt(D) if scale is None else scale
    q, k, v = qkv.float().view(B, T, 3, num_heads, D).permute(2, 0, 3, 1, 4)  # each [B, H, T, D]
    scores = torch.matmul(q, k.transpose(-2, -1)) * scale
    mask = visible_mask(T, window, sinks, qkv.device)
    scores = scores.masked_fill(~mask, float("-inf"))
    probs = torch.softmax(scores, dim=-1)
    if keep_mask is not None:  # explicit mask [B, H, T, T] (the kernels' mask in the parity tests)
        probs = probs * keep_mask.to(probs.dtype) * (keep_scale if keep_scale is not None else 1.0 / (1.0 - dropout_p))
    elif dropout_p > 0.0 and training:
        probs = F.dropout(probs, p=dropout_p, training=True)
    out = torch.matmul(probs, v)  # [B, H, T, D]
    return out.transpose(1, 2).reshape(B, T, num_heads * D).to(qkv.dtype)


def attention_sdpa(qkv: torch.Tensor, num_heads: int, scale: float | None = None) -> torch.Tensor:
    """Memory-light CPU path (no T x T tensor in autograd) for the multi-process gloo tests."""
    B, T, three_hd = qkv.shape
    D = three_hd // (3 * num_heads)
    q, k, v = qkv.view(B, T, 3, num_heads, D).permute(2, 0, 3, 1, 4)
    out = F.scaled_dot_product_attention(q, k, v, is_causal=True, scale=scale)
    return out.transpose(1, 2).reshape(B, T, num_heads * D)


class _CausalAttentionFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, qkv, num_heads, scale, dropout_p, seed):
        ext = _ext.require()
        qkv = qkv.contiguous()
        out, lse = ext.attention_forward(qkv, num_heads, scale, dropout_p, seed)
        ctx.save_for_backward(qkv, out, lse)
        ctx.num_heads, ctx.scale, ctx.dropout_p, ctx.seed = num_heads, scale, dropout_p, seed
        return out

    @staticmethod
    def backward(ctx, dout):
        qkv, out, lse = ctx.saved_tensors
        dqkv = _ext.require().attention_backward(qkv, out, dout.contiguous(), lse, ctx.num_heads, ctx.scale,
                                                 ctx.dropout_p, ctx.seed)
        return dqkv, None, None, None, None


def dropout_quantised(dropout_p: float):
    """(threshold/256, keep_scale) the kernels actually use for a requested drop probability."""
    thr = min(255, max(0, int(dropout_p * 256.0 + 0.5)))
    return thr / 256.0, 256.0 / (256 - thr)


def _draw_seed() -> int:
    # CPU generator: no device synchronisation, follows torch.manual_seed and checkpoint's RNG restore
    return int(torch.randint(0, 2 ** 62, (1,), dtype=torch.int64).item())


def causal_attention(qkv: torch.Tensor, num_heads: int, scale: float | None = None,
                     dropout_p: float = 0.0, training: bool = False, seed: int | None = None) -> torch.Tensor:
    D = qkv.shape[-1] // (3 * num_heads)
    scale = 1.0 / math.sqrt(D) if scale is None else float(scale)
    want_dropout = dropout_p > 0.0 and training
    if _ext.use_hip(qkv):
        if D not in (64, 128) or qkv.dtype not in (torch.bfloat16, torch.float32):
            raise NotImplementedError(f"causal_attention on the GPU: head size {D} / dtype {qkv.dtype} has no kernel "
                                      "(head sizes 64 and 128; bf16, or fp32 computed through bf16 MFMA inputs)")
        if qkv.dtype == torch.float32:  # fp32 storage: bf16 MFMA inputs, fp32 accumulation, widened result
            return causal_attention(qkv.to(torch.bfloat16), num_heads, scale, dropout_p, training, seed).to(torch.float32)
        if not want_dropout:
            return _CausalAttentionFn.apply(qkv, num_heads, scale, 0.0, 0)
        return _CausalAttentionFn.apply(qkv, num_heads, scale, float(dropout_p),
                                        _draw_seed() if seed is None else int(seed))
    if want_dropout or qkv.is_cuda:  # CPU with dropout, or the forced-reference oracle mode on a GPU
        return attention_reference(qkv, num_heads, scale, dropout_p, training)
    return attention_sdpa(qkv, num_heads, scale)


def window_attention(qkv: torch.Tensor, num_heads: int, window: int, sinks: int = 0, scale: float | None = None,
                     dropout_p: float = 0.0, training: bool = False, seed: int | None = None) -> torch.Tensor:
    """:func:`causal_attention` inside a sliding window: query t sees the ``window`` keys ``t - window + 1 .. t``
    (itself included, so ``window >= 1``) and the first ``sinks`` keys of the sequence, which stay visible however
    far behind they are. Time and memory grow with ``T * window``; a window of T or more is causal attention.

    Layout, dtypes, head sizes, scale and dropout as for :func:`causal_attention` (the same dropout mask for the
    same seed); on the GPU ``csrc/kernels/attention_window.hip``. A NaN or infinity in a key or value reaches
    the queries that see it, and may reach others whose tile of 64 keys holds it (as in a plain product of
    probabilities and values, where a masked probability of zero times an infinity is NaN)."""
    if qkv.dim() != 3 or num_heads < 1 or qkv.shape[-1] % (3 * num_heads) != 0:
        raise ValueError(f"window_attention: qkv {tuple(qkv.shape)} is not [B, T, 3 * {num_heads} * head size]")
    window, sinks = int(window), int(sinks)
    if window < 1 or sinks < 0:
        raise ValueError(f"window_attention: window must be at least 1 and sinks at least 0, got {window} and {sinks}")
    B, T, width = qkv.shape
    D = width // (3 * num_heads)
    window, sinks = min(window, max(T, 1)), min(sinks, T)
    scale = 1.0 / math.sqrt(D) if scale is None else float(scale)
    p = float(dropout_p) if training else 0.0
    if not 0.0 <= p < 1.0:
        raise ValueError(f"window_attention: dropout_p must be in [0, 1), got {p}")
    if not _ext.use_hip(qkv):
        return attention_reference(qkv, num_heads, scale, p, training, window=window, sinks=sinks)
    if D not in (64, 128) or qkv.dtype not in (torch.bfloat16, torch.float32):
        raise NotImplementedError(f"window_attention on the GPU: head size {D} / dtype {qkv.dtype} has no kernel "
                                  "(head sizes 64 and 128; bf16, or fp32 computed through bf16 MFMA inputs)")
    if not 1e-20 <= scale <= 1e20:
        raise ValueError(f"window_attention: the kernels take a positive scale between 1e-20 and 1e20, got {scale}")
    if B * T == 0:
        return qkv[..., : width // 3] * 0
    if qkv.dtype == torch.float32:  # fp32 storage: bf16 MFMA inputs, fp32 accumulation, widened result
        return window_attention(qkv.to(torch.bfloat16), num_heads, window, sinks, scale, p, training, seed).to(torch.float32)
    if p > 0.0:
        seed = _draw_seed() if seed is None else int(seed)
    return _ext.require().window_attention(qkv, num_heads, window, sinks, scale, p, seed if p > 0.0 else 0)
