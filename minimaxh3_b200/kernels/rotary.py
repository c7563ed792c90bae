"""Rotary positions with several axes (time, height, width) for video, images and audio.

The model turns Q and K by their tokens' positions between the projection and
attention; the reference's kernels take them already turned, so this has no
counterpart there.  ``rotary_axes`` does both tensors in one launch
(csrc/rotary.cu), on the layouts the attention entry points take, and is
differentiable in Q and K (the gradient is the inverse rotation, the same kernel).
``fp8_attention_varlen(..., rotary=Rotary(...))`` applies it on the way in.
"""
from __future__ import annotations

import math
import typing

import torch

from .. import ops as _ops

_TYPES = (torch.bfloat16, torch.float16, torch.float32)
_POS_TYPES = (torch.int32, torch.int64, torch.float32)
_LIB = torch.library.Library("mh3", "FRAGMENT")
_LIB.define("rotary_axes(Tensor q, Tensor? k, Tensor positions, int[] axes_dim, float[] theta, bool interleaved, "
            "bool inverse) -> (Tensor, Tensor)")


def _rotary_cuda(q, k, positions, axes_dim, theta, interleaved, inverse):
    oq, ok = _ops.rotary(q, k, positions, axes_dim, theta, interleaved, inverse)
    return oq, q.new_empty(0) if ok is None else ok


_LIB.impl("rotary_axes", _rotary_cuda, "CUDA")


def _turn(q, k, positions, *args):  # in or beside a backward pass
    plain = type(positions) is torch.Tensor and _ops.plain_backward(q, k)
    return (_rotary_cuda if plain else torch.ops.mh3.rotary_axes)(q, k, positions, *args)


@torch.library.register_fake("mh3::rotary_axes", lib=_LIB)
def _(q, k, positions, axes_dim, theta, interleaved, inverse):
    return _ops.rotary_like(q), q.new_empty(0) if k is None else _ops.rotary_like(k)


class _RotaryFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, positions, axes_dim, theta, interleaved, inverse):
        ctx.save_for_backward(positions)
        ctx.rest = (axes_dim, theta, interleaved)
        ctx.inverse, ctx.has_k = inverse, k is not None
        return _turn(q, k, positions, axes_dim, theta, interleaved, inverse)

    @staticmethod
    def backward(ctx, gq, gk):
        (positions,) = ctx.saved_tensors
        turn = _RotaryFn.apply if torch.is_grad_enabled() else _turn  # with create_graph: its own gradient
        dq, dk = turn(gq, gk if ctx.has_k else None, positions, *ctx.rest, not ctx.inverse)
        return dq, dk if ctx.has_k else None, None, None, None, None, None


class Rotary(typing.NamedTuple):
    """What ``rotary_axes`` takes beside the tensors."""

    positions: torch.Tensor
    axes_dim: typing.Sequence[int]
    theta: typing.Union[float, typing.Sequence[float]] = 10000.0
    interleaved: bool = True


_AXES = "rotary_axes: axes_dim is 1 to 4 even widths whose sum is positive and at most the head dim"


def _plan(axes_dim, theta, D: int) -> tuple[list[int], list[float]]:
    """The axes' widths and thetas as lists, checked."""
    axes, total = [], 0
    for d in axes_dim:
        d = int(d)
        if d < 0 or d % 2:
            raise ValueError(_AXES)
        axes.append(d)
        total += d
    if not 1 <= len(axes) <= 4 or not 0 < total <= D:
        raise ValueError(_AXES)
    thetas = [float(theta)] * len(axes) if isinstance(theta, (int, float)) else [float(t) for t in theta]
    if len(thetas) != len(axes) or not 0.0 < min(thetas) <= max(thetas) <= 1e300 or math.isnan(sum(thetas)):
        raise ValueError("rotary_axes: theta is one positive number, or one for each axis")
    return axes, thetas


def _shape(name, t):
    if not isinstance(t, torch.Tensor) or t.dim() not in (3, 4):
        raise ValueError(f"rotary_axes: {name} must be a tensor [B, H, S, D] or packed [T, H, D]")
    if t.dtype not in _TYPES:
        raise ValueError(f"rotary_axes: unsupported dtype {t.dtype} (bf16, f16 or f32)")
    return t.shape


def _check(q, k, positions, axes_dim, theta):
    shape, dev = _shape("q", q), q.device
    packed = len(shape) == 3
    tokens, D = shape[0] if packed else shape[2], shape[-1]
    if k is not None:
        ks = _shape("k", k)
        if len(ks) != len(shape) or k.dtype != q.dtype or k.device != dev or ks[-1] != D:
            raise ValueError("rotary_axes: q and k must agree in dimensions, dtype, device and head dim")
        if (ks[0] if packed else ks[2]) != tokens or (not packed and ks[0] != shape[0]):
            raise ValueError("rotary_axes: q and k must have the same tokens")
    axes, thetas = _plan(axes_dim, theta, D)
    if D > 256:
        raise ValueError("rotary_axes: the head dim must be at most 256")
    if not isinstance(positions, torch.Tensor) or positions.dtype not in _POS_TYPES:
        raise ValueError("rotary_axes: positions must be an int32, int64 or float32 tensor")
    ps = positions.shape
    if len(ps) not in (2, 3) or ps[-1] != len(axes) or ps[-2] != tokens or (len(ps) == 3 and (packed or ps[0] not in (1, shape[0]))):
        raise ValueError("rotary_axes: positions must be [S, axes] or [B, S, axes] (packed: [T, axes])")
    if positions.device != dev:
        raise ValueError("rotary_axes: positions must be on q's device")
    if positions.requires_grad and torch.is_grad_enabled():
        raise ValueError("rotary_axes: there is no gradient of the positions (pass positions.detach())")
    if not q.is_cuda:
        raise ValueError("rotary_axes: expected CUDA tensors")
    return axes, thetas


def rotary_axes(
    q: torch.Tensor,
    k: torch.Tensor | None,
    positions: torch.Tensor,
    axes_dim: typing.Sequence[int],
    theta: float | typing.Sequence[float] = 10000.0,
    interleaved: bool = True,
) -> tuple[torch.Tensor, torch.Tensor | None]:
    """Q and K turned by their tokens' positions; new tensors of the same shapes and dtype.

    q [B, H, S, D] and k [B, Hk, S, D] (any strides with contiguous channels; the
    head counts may differ; k may be None), or packed [T, H, D] as
    ``fp8_attention_varlen`` takes them; bf16, f16 or f32, D <= 256.
    ``positions`` [S, axes], [B, S, axes] or packed [T, axes]: int32, int64, or
    float32 for tokens between grid points (audio beside video).  ``axes_dim``:
    the even number of channels each axis turns, in order; channels past their
    sum are copied.  The j-th of an axis's d/2 pairs turns by position *
    theta^(-2j/d).  A pair is two neighbouring channels, or with
    ``interleaved=False`` channels p and p + sum(axes_dim)/2.
    """
    axes, thetas = _check(q, k, positions, axes_dim, theta)
    if _ops.forward_ad._current_level >= 0:
        _ops.refuse_forward_mode("rotary_axes", q, k, positions)
    if torch.is_grad_enabled() and (q.requires_grad or (k is not None and k.requires_grad)):
        oq, ok = _RotaryFn.apply(q, k, positions, axes, thetas, bool(interleaved), False)
    else:
        turn = _rotary_cuda if _ops.plain(q, k, positions) else torch.ops.mh3.rotary_axes
        oq, ok = turn(q, k, positions, axes, thetas, bool(interleaved), False)
    return oq, None if k is None else ok
