"""Linear layers on 8-bit floating point operands with a scale for each block of 128 values.

``fp8_linear(x, weight, bias)`` is :func:`ops.linear` with the three products of a training step —
``y = x W^T``, ``dx = dy W``, ``dW = dy^T x`` — on e4m3 operands at twice the matrix rate of bf16:

* activations and output gradients are quantised in blocks of 1 x 128 along the contraction of the
  product they enter (along the features for ``y`` and ``dx``, along the tokens for ``dW``; both layouts
  come out of one pass over the tensor), weights in tiles of 128 x 128, which serve both contractions;
* a block's scale is a power of two, the smallest one under which its largest magnitude fits e4m3's
  largest value (448), so scaling is exact and the matrix instruction applies it from its exponent byte;
* products accumulate in fp32 and are rounded once, to the tensors' dtype; the bias and its gradient
  never leave full precision;
* what the backward keeps of ``x`` is its 8-bit transposed copy, half the bytes of a bf16 activation
  (or nothing but a recipe, with ``regen`` as in :func:`ops.linear`). The weight is quantised anew in
  every pass (a few microseconds next to a product of hundreds), so a sharded weight can be freed in
  between.

The pieces are public: ``quantize_fp8`` (layouts in its docstring) and ``fp8_matmul``, for a program that
quantises a weight once and multiplies by it many times.

Numbers: an element is off by at most half a step of e4m3, 2^-4 of its own size as long as it is within
2^-13 of its block's largest, so a product of random operands is off by some 4 % of its own size. Values
far below their block's largest become subnormal or zero. An infinity or NaN of the input is a NaN of the
quantised matrix in its place alone and takes no part in the scale: it shows up in the products that read
it. Gradients are those of the product of the quantised operands with respect to these operands (the
rounding's own derivative is taken as one).

GPU tensors run ``csrc/kernels/fp8_{quant,gemm}.hip`` (bf16 or fp32 tensors; other dtypes are an error).
CPU tensors and ``PDA_FORCE_REFERENCE=1`` run the PyTorch references below, the oracles of the kernel tests.
"""
from __future__ import annotations

import math
from typing import Optional, Tuple, Union

import torch
import torch.nn.functional as F

from .. import _ext

BLOCK = 128
_DTYPES = (torch.bfloat16, torch.float32)


def _exp2(e: torch.Tensor) -> torch.Tensor:
    """2^e in fp32 for whole numbers from -127 to 127, exact on every device (``torch.ldexp`` and ``exp2`` are off by
    the last bit at some exponents on the GPU): the number's own bits."""
    return torch.where(e >= -126, (e + 127) << 23, 1 << 22).to(torch.int32).view(torch.float32)


class Fp8Matrix:
    """A quantised matrix of ``rows`` x ``cols`` values.

    ``q``: float8_e4m3fn ``[rows, ceil(cols / 128) * 128]``, zeros behind column ``cols``. ``scale``:
    uint8 ``[rows, S]`` — or ``[ceil(rows / 128), S]`` with ``tiles`` — the byte ``b`` of a block, at most 254,
    standing for ``2^(b - 127)``; S is the number of blocks in a row rounded up to 4 (the padding is not read)."""

    __slots__ = ("q", "scale", "cols", "tiles")

    def __init__(self, q: torch.Tensor, scale: torch.Tensor, cols: int, tiles: bool = False):
        self.q, self.scale, self.cols, self.tiles = q, scale, int(cols), bool(tiles)
        blocks = -(-self.cols // BLOCK)
        if q.dim() != 2 or q.dtype != torch.float8_e4m3fn or q.shape[1] != blocks * BLOCK:
            raise ValueError(f"Fp8Matrix: q must be float8_e4m3fn [rows, {blocks * BLOCK}] for {self.cols} columns, "
                             f"got {q.dtype} {tuple(q.shape)}")
        rows = -(-q.shape[0] // BLOCK) if self.tiles else q.shape[0]
        want = (rows, -(-blocks // 4) * 4)
        if scale.dtype != torch.uint8 or tuple(scale.shape) != want:
            raise ValueError(f"Fp8Matrix: scale must be uint8 {want}, got {scale.dtype} {tuple(scale.shape)}")
        if q.device != scale.device:
            raise ValueError(f"Fp8Matrix: q is on {q.device}, scale on {scale.device}")

    @property
    def rows(self) -> int:
        return self.q.shape[0]

    def dequantize(self) -> torch.Tensor:
        """The values it stands for, fp32 ``[rows, cols]``."""
        blocks = self.q.shape[1] // BLOCK
        e = self.scale[:, :blocks].to(torch.int32) - 127
        if self.tiles:
            e = e.repeat_interleave(BLOCK, 0)[: self.rows]
        v = self.q.to(torch.float32).view(self.rows, blocks, BLOCK)
        return (v * _exp2(e).unsqueeze(2)).view(self.rows, blocks * BLOCK)[:, : self.cols]


# --------------------------------------------------------------------------- references
def _exponent_reference(amax: torch.Tensor) -> torch.Tensor:
    m, k = torch.frexp(amax)  # amax = m 2^k with 0.5 <= m < 1; 448 = 0.875 * 2^9
    return torch.where(amax > 0, torch.where(m <= 0.875, k - 9, k - 8), -127).clamp(min=-127)


def _quantize_reference(v: torch.Tensor, rows_per_block: int) -> Tuple[torch.Tensor, torch.Tensor]:
    rows, cols = v.shape
    blocks = -(-cols // BLOCK)
    v = F.pad(v.float(), (0, blocks * BLOCK - cols, 0, -rows % rows_per_block))
    v = v.view(v.shape[0] // rows_per_block, rows_per_block, blocks, BLOCK)
    a = v.abs()
    a = torch.where(torch.isfinite(a), a, torch.zeros_like(a))
    e = _exponent_reference(a.amax((1, 3)) if v.numel() else a.new_zeros(v.shape[0], blocks))
    q = v * _exp2(-e)[:, None, :, None]
    q = torch.where(torch.isfinite(v), q, torch.full_like(q, float("nan"))).to(torch.float8_e4m3fn)
    scale = F.pad((e + 127).to(torch.uint8), (0, -blocks % 4))
    return q.view(q.shape[0] * rows_per_block, blocks * BLOCK)[:rows], scale


def quantize_fp8_reference(x: torch.Tensor, blocks: str = "rows"):
    rows, cols = x.shape
    if blocks == "tiles":
        return (Fp8Matrix(*_quantize_reference(x, BLOCK), cols, True), Fp8Matrix(*_quantize_reference(x.t(), BLOCK), rows, True))
    by_rows = Fp8Matrix(*_quantize_reference(x, 1), cols) if blocks != "columns" else None
    by_cols = Fp8Matrix(*_quantize_reference(x.t(), 1), rows) if blocks != "rows" else None
    return (by_rows, by_cols) if blocks == "both" else by_cols if by_rows is None else by_rows


def fp8_matmul_reference(a: Fp8Matrix, b: Fp8Matrix, bias=None, out_dtype=torch.bfloat16) -> torch.Tensor:
    y = a.dequantize() @ b.dequantize().t()
    return (y if bias is None else y + bias.float()).to(out_dtype)


# --------------------------------------------------------------------------- pieces
def _check_source(x: torch.Tensor, what: str) -> torch.Tensor:
    if x.dtype not in _DTYPES:
        raise NotImplementedError(f"{what}: dtype {x.dtype} has no kernel (bf16 or fp32)")
    x = x.detach()
    if x.dim() == 2 and (x.shape[1] <= 1 or x.stride(1) == 1) and (x.shape[0] <= 1 or x.stride(0) >= x.shape[1]):
        return x
    return x.contiguous()


def quantize_fp8(x: torch.Tensor, blocks: str = "rows") -> Union[Fp8Matrix, Tuple[Fp8Matrix, Fp8Matrix]]:
    """Quantises a bf16 / fp32 matrix ``x [R, C]`` (any row pitch) in blocks of 128 values.

    ``"rows"``: blocks along a row, a matrix ``[R, C]`` for products that contract over C. ``"columns"``:
    blocks along a column, laid out transposed, ``[C, R]``, for products that contract over R. ``"both"``: the
    two of them, from one read of ``x``. ``"tiles"``: one scale for each 128 x 128 tile, as ``[R, C]`` and as
    ``[C, R]`` (a weight, for the forward product and its input gradient). Not differentiable."""
    if blocks not in ("rows", "columns", "both", "tiles"):
        raise ValueError(f"quantize_fp8: blocks must be 'rows', 'columns', 'both' or 'tiles', got {blocks!r}")
    if x.dim() != 2:
        raise ValueError(f"quantize_fp8: a matrix is needed, got {x.dim()} dimensions")
    x = _check_source(x, "quantize_fp8")
    if not _ext.use_hip(x):
        with torch.no_grad():
            return quantize_fp8_reference(x, blocks)
    rows, cols = x.shape
    got = _ext.require().fp8_quantize(x, blocks != "columns", blocks != "rows", blocks == "tiles")
    if blocks == "rows":
        return Fp8Matrix(got[0], got[1], cols)
    if blocks == "columns":
        return Fp8Matrix(got[0], got[1], rows)
    tiles = blocks == "tiles"
    return Fp8Matrix(got[0], got[1], cols, tiles), Fp8Matrix(got[2], got[3], rows, tiles)


def fp8_matmul(a: Fp8Matrix, b: Fp8Matrix, bias: Optional[torch.Tensor] = None,
               out_dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """``a @ b.T + bias`` for ``a [M, K]`` and ``b [N, K]``, accumulated in fp32, as bf16 or fp32 ``[M, N]``.
    An fp32 result takes what its operands hold in blocks of scale bytes 0 to 2 (magnitudes below 2^-116) to multiples
    of 2^-133 first. ``bias``: bf16 or fp32 ``[N]``. Not differentiable (``fp8_linear`` is)."""
    if a.cols != b.cols:
        raise ValueError(f"fp8_matmul: contraction lengths differ, {a.cols} and {b.cols}")
    if out_dtype not in _DTYPES:
        raise NotImplementedError(f"fp8_matmul: out_dtype {out_dtype} (bf16 or fp32)")
    if a.q.device != b.q.device or (bias is not None and bias.device != a.q.device):
        raise ValueError("fp8_matmul: operands on different devices")
    if bias is not None:
        if bias.dtype not in _DTYPES or tuple(bias.shape) != (b.rows,):
            raise ValueError(f"fp8_matmul: bias must be bf16 or fp32 [{b.rows}], got {bias.dtype} {tuple(bias.shape)}")
        bias = bias.detach().contiguous()
    if not _ext.use_hip(a.q):
        return fp8_matmul_reference(a, b, bias, out_dtype)
    return _ext.require().fp8_matmul(a.q, a.scale, a.tiles, b.q, b.scale, b.tiles, a.cols, bias, out_dtype == torch.float32)


# --------------------------------------------------------------------------- the layer
def _rows(x: torch.Tensor) -> torch.Tensor:
    return x.reshape(math.prod(x.shape[:-1]), x.shape[-1])


def _reference_backward(dy2, weight, x2, need_x, need_w, need_b):
    dx = dw = db = None
    if need_x:
        dx = fp8_matmul_reference(quantize_fp8_reference(dy2), quantize_fp8_reference(weight, "tiles")[1], None, dy2.dtype)
    if need_w:
        dw = fp8_matmul_reference(quantize_fp8_reference(dy2, "columns"), quantize_fp8_reference(x2, "columns"), None, dy2.dtype)
    if need_b:
        db = dy2.float().sum(0).to(dy2.dtype)
    return dx, dw, db


class _Fp8LinearFn(torch.autograd.Function):
    """The layer where a Python object takes part: a gradient goes straight into its owner's buffer (gradient
    sink, see ops.linear), or ``x`` is rebuilt from a recipe; and the reference path. (Otherwise the extension's
    own node runs: the same computation with two thirds of the host time.)"""

    @staticmethod
    def forward(ctx, x, weight, bias, regen):
        ctx.hip = _ext.use_hip(x)
        ctx.regen = None if regen is None else regen.recipe()
        ctx.x_shape = x.shape
        ctx.has_bias = bias is not None
        ctx.sinks = (getattr(weight, "_pda_grad_sink", None), getattr(bias, "_pda_grad_sink", None))
        keep = ctx.needs_input_grad[1] and regen is None
        if ctx.hip:
            y, *kept = _ext.require().fp8_linear_forward(x, weight, bias, keep)
        else:
            x2 = _rows(x)
            y = fp8_matmul_reference(quantize_fp8_reference(x2), quantize_fp8_reference(weight, "tiles")[0], bias, x.dtype)
            y = y.view(*x.shape[:-1], weight.shape[0])
            kept = [x2] if keep else []
        if regen is not None:
            ctx.regen_none = tuple(t is None for t in regen.tensors)
            kept = [t for t in regen.tensors if t is not None] if ctx.needs_input_grad[1] else []
        ctx.save_for_backward(weight, *kept)
        return y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        weight, *kept = ctx.saved_tensors
        need_x, need_w = ctx.needs_input_grad[0], ctx.needs_input_grad[1]
        need_b = ctx.has_bias and ctx.needs_input_grad[2]
        x = None
        if need_w and ctx.regen is not None:
            it = iter(kept)
            x = ctx.regen.rebuild(*[None if missing else next(it) for missing in ctx.regen_none])
        if not ctx.hip:
            if need_w:
                x = kept[0] if x is None else _rows(x)
            dx, dw, db = _reference_backward(_rows(dy), weight, x, need_x, need_w, need_b)
            return (None if dx is None else dx.view(ctx.x_shape)), dw, db, None
        w_sink, b_sink = ctx.sinks
        w_target = w_sink() if need_w and w_sink is not None else None
        b_target = b_sink() if need_b and b_sink is not None else None
        w_out, w_acc = w_target if w_target is not None else (None, False)
        b_out, b_acc = b_target if b_target is not None else (None, False)
        xq, xs = kept if need_w and x is None else (None, None)
        dx, dw, db = _ext.require().fp8_linear_backward(dy, weight, x, xq, xs, need_x, need_w, need_b, w_out, bool(w_acc),
                                                        b_out, bool(b_acc))
        # A gradient written into its target is reported to autograd as None (the accumulator node still
        # runs and fires the owner's hook).
        return (dx, dw if need_w and w_target is None else None, db if need_b and b_target is None else None, None)


def fp8_linear(x: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor] = None, regen=None) -> torch.Tensor:
    """``x @ weight.T + bias`` with 8-bit operands in the product and in both products of its backward.

    ``x [..., in]``, ``weight [out, in]`` and ``bias [out]`` share one dtype, bf16 or fp32, which is the
    result's too. Every size is allowed, zero tokens included. ``regen`` as in :func:`ops.linear`."""
    if x.dim() < 1 or weight.dim() != 2 or x.shape[-1] != weight.shape[1]:
        raise ValueError(f"fp8_linear: x {tuple(x.shape)} and weight {tuple(weight.shape)} do not match")
    if x.dtype not in _DTYPES:
        raise NotImplementedError(f"fp8_linear: dtype {x.dtype} has no kernel (bf16 or fp32)")
    if weight.dtype != x.dtype or weight.device != x.device:
        raise ValueError(f"fp8_linear: x is {x.dtype} on {x.device}, weight {weight.dtype} on {weight.device}")
    if bias is not None and (bias.dtype != x.dtype or bias.device != x.device or tuple(bias.shape) != (weight.shape[0],)):
        raise ValueError(f"fp8_linear: bias must be {x.dtype} [{weight.shape[0]}] on {x.device}, "
                         f"got {bias.dtype} {tuple(bias.shape)} on {bias.device}")
    # (without grad mode nobody asks for gradients, whoever owns them, and nothing is kept of x)
    if _ext.use_hip(x) and (not torch.is_grad_enabled() or (regen is None and getattr(weight, "_pda_grad_sink", None) is None
                                                            and getattr(bias, "_pda_grad_sink", None) is None)):
        return _ext.require().fp8_linear(x, weight, bias)
    return _Fp8LinearFn.apply(x, weight, bias, regen)
