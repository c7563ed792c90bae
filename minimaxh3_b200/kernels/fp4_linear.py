"""4-bit linear layers beside the FP8 ones: microscaled e2m1 weights and activations.

The same place, policy and LoRA contract as ``fp8_linear`` (the reference's
``kernels/fp8_linear.py``, which stops at 8 bits): ``FP4Linear`` replaces an
``nn.Linear``, keeps the mutable ``adapters`` list of ``(A, B, scale)`` and runs
an activation rounding plus one tcgen05 GEMM that applies the scales, the bias
and every adapter's delta and writes bf16 once.  Weights take 0.5625 bytes each.

A 4-bit matrix is three tensors ``(values, blocks, scale)``: see ``quantize_fp4``.
The functions are registered as operators ``torch.ops.mh3.*`` of the same names with fake
implementations for ``torch.compile``.  Inference only: asking for a gradient raises, as with ``FP8Linear``.
"""
from __future__ import annotations

import torch
import torch.nn as nn

from .. import ops as _ops
from .fp8_linear import convert_linears

_LIB = torch.library.Library("mh3", "FRAGMENT")
_LIB.define("fp4_linear(Tensor x2d, Tensor w4, Tensor w_blocks, Tensor w_scale, Tensor? bias, Tensor[] lora_a, "
            "Tensor[] lora_b, float[] lora_scale) -> Tensor")
_LIB.define("quantize_fp4(Tensor x2d) -> (Tensor, Tensor, Tensor)")
_LIB.define("dequantize_fp4(Tensor values, Tensor blocks, Tensor scale, ScalarType dtype) -> Tensor")
_LIB.define("fp4_matmul(Tensor[] a, Tensor[] b, Tensor? bias) -> Tensor")


def _fp4_linear_cuda(x2d, w4, w_blocks, w_scale, bias, lora_a, lora_b, lora_scale):
    return _ops.fp4_linear(x2d, w4, w_blocks, w_scale, bias, list(zip(lora_a, lora_b, lora_scale)))


def _fp4_matmul_cuda(a, b, bias):
    return _ops.fp4_gemm(a, b, bias=bias)


_LIB.impl("fp4_linear", _fp4_linear_cuda, "CUDA")
_LIB.impl("quantize_fp4", _ops.quantize_fp4, "CUDA")
_LIB.impl("dequantize_fp4", _ops.dequantize_fp4, "CUDA")
_LIB.impl("fp4_matmul", _fp4_matmul_cuda, "CUDA")


@torch.library.register_fake("mh3::fp4_linear", lib=_LIB)
def _(x2d, w4, w_blocks, w_scale, bias, lora_a, lora_b, lora_scale):
    return x2d.new_empty((x2d.shape[0], w4.shape[0]), dtype=torch.bfloat16)


@torch.library.register_fake("mh3::quantize_fp4", lib=_LIB)
def _(x2d):
    M, K = x2d.shape
    return (x2d.new_empty((M, K // 2), dtype=torch.uint8),
            x2d.new_empty((-(-M // 128), -(-K // 64), 32, 4, 4), dtype=torch.float8_e4m3fn),
            x2d.new_empty((M, 1), dtype=torch.float32))


@torch.library.register_fake("mh3::dequantize_fp4", lib=_LIB)
def _(values, blocks, scale, dtype):
    return values.new_empty((values.shape[0], 2 * values.shape[1]), dtype=dtype)


@torch.library.register_fake("mh3::fp4_matmul", lib=_LIB)
def _(a, b, bias):
    return a[0].new_empty((a[0].shape[0], b[0].shape[0]), dtype=torch.bfloat16)


class _NoGradient(torch.autograd.Function):
    """Passes a result on, tied to the inputs that ask for a gradient, so that asking for it raises."""

    @staticmethod
    def forward(ctx, out, *inputs):
        ctx.mark_dirty(out)  # out itself, no view of it: callers may add to it in place
        return out

    @staticmethod
    def backward(ctx, grad):
        raise RuntimeError("fp4_linear has no gradient, nor have the other 4-bit operators: they are for inference")


def quantize_fp4(x2d: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """x2d [M, K] (bf16, f16 or f32, K a multiple of 32) rounded to 4 bits: ``(values, blocks, scale)``.

    values uint8 [M, K/2]: element 2j in the low half of byte j, 2j+1 in the high
    half, e2m1 codes (0, 0.5, 1, 1.5, 2, 3, 4, 6 and a sign).  blocks
    float8_e4m3fn [ceil(M/128), ceil(K/64), 32, 4, 4]: the scale of elements
    16b..16b+15 of row m at [m // 128, b // 4, m % 32, m % 128 // 32, b % 4].
    scale float32 [M, 1]: a power of two that puts the row's largest block scale
    at the upper end of e4m3.  Entries of blocks past M and K are 0.  The value is
    code * block * scale; all roundings are to nearest even.  A row that holds an infinity or NaN gets scale NaN.
    """
    if _ops.forward_ad._current_level >= 0:
        _ops.refuse_forward_mode("quantize_fp4", x2d)
    return (_ops.quantize_fp4 if _ops.plain(x2d) else torch.ops.mh3.quantize_fp4)(x2d)


def _asking(*ts):
    """Those of ts (None where one is left out) that ask for a gradient."""
    return [t for t in ts if t is not None and t.requires_grad] if torch.is_grad_enabled() else []


def dequantize_fp4(values: torch.Tensor, blocks: torch.Tensor, scale: torch.Tensor,
                   dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """The [M, K] numbers that a 4-bit matrix stands for, exact in bfloat16 and float32 (infinite where a
    magnitude within a twentieth of the type's end was rounded up past it)."""
    if _ops.forward_ad._current_level >= 0:
        _ops.refuse_forward_mode("dequantize_fp4", scale)
    plain = _ops.plain(values, blocks, scale)
    out = (_ops.dequantize_fp4 if plain else torch.ops.mh3.dequantize_fp4)(values, blocks, scale, dtype)
    asks = _asking(blocks, scale)
    return _NoGradient.apply(out, *asks) if asks else out


def fp4_matmul(a, b, bias: torch.Tensor | None = None) -> torch.Tensor:
    """bf16 ``a b^T + bias`` of two 4-bit matrices ``(values, blocks, scale)``, a [M, K], b [N, K], N a multiple of 8."""
    a, b = tuple(a), tuple(b)
    if _ops.forward_ad._current_level >= 0:
        _ops.refuse_forward_mode("fp4_matmul", a[2], b[2], bias)
    out = (_fp4_matmul_cuda if _ops.plain(*a, *b, bias) else torch.ops.mh3.fp4_matmul)(a, b, bias)
    asks = _asking(*a[1:], *b[1:], bias)
    return _NoGradient.apply(out, *asks) if asks else out


def fp4_linear(x: torch.Tensor, w4: torch.Tensor, w_blocks: torch.Tensor, w_scale: torch.Tensor,
               bias: torch.Tensor | None = None, adapters=()) -> torch.Tensor:
    """bf16 ``x W^T + bias + sum_i scale_i (x A_i^T) B_i^T`` with W [N, K] in 4 bits and x [..., K] rounded to 4 bits.

    (w4, w_blocks, w_scale) is ``quantize_fp4(W)``; adapters are
    ``(A [r, K], B [N, r], scale)`` and see the unrounded x.  One or two rows run as one
    launch, up to 16 on a kernel that streams W once, more at the tensor cores' 4-bit rate.
    """
    N, K = _ops.check_fp4(w4, w_blocks, w_scale, "fp4_linear weight")
    if not isinstance(x, torch.Tensor) or x.dim() < 1 or x.shape[-1] != K or not x.is_floating_point():
        raise ValueError(f"fp4_linear: x must be a float tensor [..., {K}]")
    if N % 8 or N == 0:
        raise ValueError("fp4_linear: the number of output features must be a positive multiple of 8")
    if not x.is_cuda or x.device != w4.device:
        raise ValueError("fp4_linear: x and the weight must be on one CUDA device")
    x2d = x if x.dim() == 2 else x.reshape(-1, K)
    low_rank = [t for a, b, _ in adapters for t in (a, b)] if adapters else ()
    if _ops.forward_ad._current_level >= 0:
        _ops.refuse_forward_mode("fp4_linear", x, w_scale, bias, *low_rank)
    asks = _asking(x, w_blocks, w_scale, bias, *low_rank)
    if not asks and _ops.plain(x, w4, w_blocks, w_scale, bias, *low_rank):
        out = _ops.fp4_linear(x2d, w4, w_blocks, w_scale, bias, adapters, checked=True)
    else:
        out = torch.ops.mh3.fp4_linear(x2d, w4, w_blocks, w_scale, bias, [a for a, _, _ in adapters], [b for _, b, _ in adapters],
                                       [float(s) for _, _, s in adapters])
        if asks:
            out = _NoGradient.apply(out, *asks)
    return out if x.dim() == 2 else out.reshape(*x.shape[:-1], N)


class FP4Linear(nn.Module):
    """e2m1 weights with e4m3 block scales; fused scaled GEMM forward (the 4-bit ``FP8Linear``)."""

    def __init__(self, in_features: int, out_features: int) -> None:
        super().__init__()
        self.in_features = in_features
        self.out_features = out_features
        self.adapters: list[tuple[torch.Tensor, torch.Tensor, float]] = []

    @classmethod
    @torch.no_grad()
    def from_linear(cls, linear: nn.Linear) -> "FP4Linear":
        """Round ``linear``'s weight once and free it (buffers ``w4``, ``w_blocks``, ``w_scale``, ``bias``)."""
        if linear.in_features % 32 or linear.out_features % 8:
            raise ValueError("FP4Linear needs in_features a multiple of 32 and out_features a multiple of 8")
        mod = cls(linear.in_features, linear.out_features)
        weight = linear.weight.detach()
        if not weight.is_cuda:
            weight = weight.cuda()
        if weight.dtype not in (torch.bfloat16, torch.float16, torch.float32):
            weight = weight.to(torch.float32)
        for name, t in zip(("w4", "w_blocks", "w_scale"), quantize_fp4(weight)):
            mod.register_buffer(name, t)
        bias = None
        if linear.bias is not None:
            bias = linear.bias.detach().to(device=mod.w4.device, dtype=torch.bfloat16).contiguous()
        mod.register_buffer("bias", bias)
        if isinstance(getattr(linear, "adapters", None), list):
            mod.adapters = list(linear.adapters)
        linear.weight = None
        linear.bias = None
        return mod

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        return fp4_linear(x, self.w4, self.w_blocks, self.w_scale, self.bias, self.adapters).to(x.dtype)


def convert_transformer_to_fp4(transformer: nn.Module, exclude_patterns, keep_edge_blocks: int) -> int:
    """``convert_transformer_to_fp8``'s policy with ``FP4Linear``: in features a multiple of 32, out features of 16."""
    return convert_linears(transformer, exclude_patterns, keep_edge_blocks, FP4Linear.from_linear,
                           lambda m: m.in_features % 32 == 0 and m.out_features % 16 == 0)
