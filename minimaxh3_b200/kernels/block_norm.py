"""The norms before and after a transformer block, with modulation, gate and residual.

A diffusion transformer's block normalises its stream, scales and shifts it by
the timestep's modulation, and adds its gated output back; the model does this
between the linears and attention that this package replaces (the reference has
no kernel for it).  ``norm_modulate`` is the norm before a block;
``gated_residual_norm`` joins the norm on a block's output, the gate, the
residual and the next block's ``norm_modulate`` in one pass (csrc/block_norm.cu).
Both are differentiable in every tensor argument.

The modulation belongs to a batch item, to a packed sequence (``cu_seqlens``, as
``fp8_attention_varlen``) or to each token.
"""
from __future__ import annotations

import torch
from torch.autograd.function import once_differentiable

from .. import ops as _ops

_TYPES = (torch.bfloat16, torch.float16, torch.float32)
_MODS = "Tensor x, Tensor? y, Tensor? gate, Tensor? scale, Tensor? shift, Tensor? weight, Tensor? bias, Tensor? y_weight, Tensor? cu"
_CONF = "int norm, int y_norm, float eps, float alpha, bool per_token"
_LIB = torch.library.Library("mh3", "FRAGMENT")
_LIB.define(f"block_norm({_MODS}, {_CONF}, bool want_stats) -> Tensor[]")
_LIB.define(f"block_norm_backward(Tensor? dr, Tensor? dh, {_MODS}, Tensor stats, {_CONF}, bool[] want, "
            "int wide=0) -> Tensor[]")


_LIB.impl("block_norm", _ops.block_norm_fwd, "CUDA")
_LIB.impl("block_norm_backward", _ops.block_norm_bwd, "CUDA")


@torch.library.register_fake("mh3::block_norm", lib=_LIB)
def _(x, y, gate, scale, shift, weight, bias, y_weight, cu, norm, y_norm, eps, alpha, per_token, want_stats):
    rows = 1
    for n in x.shape[:-1]:
        rows = rows * n
    out = [x.new_empty(x.shape) for given in (y is not None, norm) if given]
    return out + ([x.new_empty((rows, 4), dtype=torch.float32)] if want_stats else [])


@torch.library.register_fake("mh3::block_norm_backward", lib=_LIB)
def _(dr, dh, x, y, gate, scale, shift, weight, bias, y_weight, cu, stats, norm, y_norm, eps, alpha, per_token, want, wide=0):
    ts = (x, y, gate, scale, shift, weight, bias, y_weight)
    f32 = [False] * 2 + [bool(wide >> i & 1) for i in range(3)] + [False] * 3
    return [t.new_empty(t.shape, dtype=torch.float32 if f else t.dtype) for t, w, f in zip(ts, want, f32) if w and t is not None]


def _rows(mods, shape):
    """gate, scale and shift with a row for each group or token."""
    return mods if shape is None else [m if m is None or m.shape == shape else m.expand(shape) for m in mods]


def _gradients(ctx, *grads):
    saved = ctx.saved_tensors
    mods, shape = saved[2:5], ctx.shape
    it = iter(grads)
    dr = None if saved[1] is None else next(it)  # r with y, h with a norm
    dh = next(it) if ctx.conf[0] else None
    if dr is None and dh is None:
        return (None,) * 11
    want = ctx.needs_input_grad[:8]  # false for what is not a tensor
    # A modulation shared by groups or tokens: its rows' gradients come in f32 and are summed before they are rounded.
    wide = 0
    if shape is not None:
        for i, m in enumerate(mods):
            if want[2 + i] and m.shape != shape:
                wide |= 1 << i
    plain = ctx.plain and _ops.plain_backward(dr, dh)
    backward = _ops.block_norm_bwd if plain else torch.ops.mh3.block_norm_backward
    it = iter(backward(dr, dh, *saved[:2], *_rows(mods, shape), *saved[5:], *ctx.conf, want, wide))
    out = [next(it) if w else None for w in want]
    if wide:
        for i, m in enumerate(mods):
            if wide >> i & 1:
                out[2 + i] = out[2 + i].sum_to_size(m.shape).to(m.dtype)
    return (*out, None, None, None)


_gradients_once = once_differentiable(_gradients)


class _BlockNormFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, y, gate, scale, shift, weight, bias, y_weight, cu, conf, shape):
        ctx.plain = _ops.plain(x, y, gate, scale, shift, weight, bias, y_weight, cu)
        forward = _ops.block_norm_fwd if ctx.plain else torch.ops.mh3.block_norm
        *out, stats = forward(x, y, *_rows((gate, scale, shift), shape), weight, bias, y_weight, cu, *conf, True)
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(x, y, gate, scale, shift, weight, bias, y_weight, cu, stats)
        ctx.conf, ctx.shape = conf, shape
        return tuple(out)

    @staticmethod
    def backward(ctx, *grads):
        return (_gradients_once if torch.is_grad_enabled() else _gradients)(ctx, *grads)


def _check_stream(what, name, t, like=None):
    if not isinstance(t, torch.Tensor) or t.dim() not in (2, 3) or t.dtype not in _TYPES:
        raise ValueError(f"{what}: {name} must be a bf16, f16 or f32 tensor [B, S, C] or [T, C]")
    if like is not None and (t.shape != like.shape or t.dtype != like.dtype or t.device != like.device):
        raise ValueError(f"{what}: {name} must have x's shape, dtype and device")


def _check_cu(what, x, cu):
    if cu is None:
        return
    if not isinstance(cu, torch.Tensor) or cu.dtype != torch.int32 or cu.dim() != 1 or cu.numel() < 2 or cu.device != x.device:
        raise ValueError(f"{what}: cu_seqlens must be an int32 tensor [nseq+1] on x's device")
    if x.dim() != 2:
        raise ValueError(f"{what}: cu_seqlens needs packed x [T, C]")


def _modulation(what, x, cu, gate, scale, shift):
    """gate, scale and shift in as many dimensions as the shape they broadcast to; that shape, [groups, C], or x's if
    one of them has a row for each token (None: they have it); and whether it is x's."""
    C, device = x.shape[-1], x.device
    groups = cu.numel() - 1 if cu is not None else x.shape[0] if x.dim() == 3 else 1
    for m in (gate, scale, shift):
        if m is not None and not (isinstance(m, torch.Tensor) and m.shape == (groups, C) and m.dtype in _TYPES and m.device == device):
            break
    else:  # the common form
        return gate, scale, shift, None, False
    out, per_token = {}, False
    for name, m in (("gate", gate), ("scale", scale), ("shift", shift)):
        if m is None:
            out[name] = None
            continue
        if not isinstance(m, torch.Tensor) or m.dtype not in _TYPES or m.device != x.device or m.dim() < 1 or m.shape[-1] != C:
            raise ValueError(f"{what}: {name} must be a bf16, f16 or f32 tensor [..., C] on x's device")
        lead = tuple(m.shape[:-1])
        if x.dim() == 3:
            B, S = x.shape[:2]
            if len(lead) == 2 and lead[1] == 1 and lead[0] in (1, B):
                m, kind = m[:, 0], "group"
            elif lead in ((), (1,), (B,)):
                kind = "group"
            elif len(lead) == 2 and lead[0] in (1, B) and lead[1] == S:
                kind = "token"
            else:
                raise ValueError(f"{what}: {name} must be [C], [B, C], [B, 1, C] or [B, S, C]")
        elif lead in ((), (1,), (groups,)):
            kind = "group"
        elif lead == (x.shape[0],):
            kind = "token"
        else:
            raise ValueError(f"{what}: {name} must be [C], [T, C], or with cu_seqlens [nseq, C]")
        per_token = per_token or kind == "token"
        out[name] = (kind, m)
    for name, km in out.items():
        if km is None:
            continue
        kind, m = km
        if per_token and kind == "group" and cu is not None and m.dim() == 2 and m.shape[0] != 1:
            raise ValueError(f"{what}: {name} is per sequence while another modulation is per token")
        if m.dim() == 1:
            m = m.unsqueeze(0)
        if per_token and kind == "group" and x.dim() == 3:
            m = m.unsqueeze(1)
        out[name] = m
    return out["gate"], out["scale"], out["shift"], tuple(x.shape) if per_token else (groups, C), per_token


def _channels(what, x, name, v):
    if not isinstance(v, torch.Tensor) or v.dtype not in _TYPES or v.shape != x.shape[-1:] or v.device != x.device:
        raise ValueError(f"{what}: {name} must be a bf16, f16 or f32 tensor [C] on x's device")


def _run(what, shape, *args):
    if _ops.forward_ad._current_level >= 0:
        _ops.refuse_forward_mode(what, *args[:8])
    if torch.is_grad_enabled():
        for t in args[:8]:
            if t is not None and t.requires_grad:
                return _BlockNormFn.apply(*args[:9], args[9:], shape)
    forward = _ops.block_norm_fwd if _ops.plain(*args[:9]) else torch.ops.mh3.block_norm
    if shape is not None:
        args = (*args[:2], *_rows(args[2:5], shape), *args[5:])
    return forward(*args, False)


def _finish_checks(what, x, eps):
    if not 1 <= x.shape[-1] <= 8192:
        raise ValueError(f"{what}: 1 to 8192 channels")
    if not float(eps) >= 0.0:
        raise ValueError(f"{what}: eps must not be negative")
    if not x.is_cuda:
        raise ValueError(f"{what}: expected CUDA tensors")


def norm_modulate(
    x: torch.Tensor,
    scale: torch.Tensor | None = None,
    shift: torch.Tensor | None = None,
    *,
    weight: torch.Tensor | None = None,
    bias: torch.Tensor | None = None,
    norm: str = "layer",
    eps: float = 1e-6,
    cu_seqlens: torch.Tensor | None = None,
) -> torch.Tensor:
    """``(norm(x) * weight + bias) * (1 + scale) + shift`` over the last dimension, in x's dtype.

    x [B, S, C] or [T, C], bf16, f16 or f32, C <= 8192; ``norm`` "layer" or
    "rms".  scale / shift: [C], [B, C], [B, 1, C], or a row for each token
    ([B, S, C] / [T, C]); with ``cu_seqlens`` (int32 [nseq+1] on the device) also
    [nseq, C] (taken before [T, C] where the two are alike), and rows outside every
    sequence give zeros.  weight / bias [C].
    Modulation and weights may be of other float types than x (kept in f32
    beside a bf16 stream); None leaves that term out.  Statistics and sums are
    f32, the result is rounded once; so is the gradient of a modulation that
    tokens or batch items share (where another one has a row for each token, its
    rows' f32 gradients take 4 bytes an element of x until they are summed).
    """
    what = "norm_modulate"
    _check_stream(what, "x", x)
    _check_cu(what, x, cu_seqlens)
    if norm not in ("layer", "rms"):
        raise ValueError(f"{what}: norm must be 'layer' or 'rms'")
    _, scale, shift, shape, per_token = _modulation(what, x, cu_seqlens, None, scale, shift)
    if weight is not None:
        _channels(what, x, "weight", weight)
    if bias is not None:
        _channels(what, x, "bias", bias)
    _finish_checks(what, x, eps)
    cu = None if cu_seqlens is None else cu_seqlens.contiguous()
    return _run(what, shape, x, None, None, scale, shift, weight, bias, None, cu, _ops.NORM_KINDS[norm], 0, float(eps), 1.0,
                per_token)[0]


def gated_residual_norm(
    x: torch.Tensor,
    y: torch.Tensor,
    gate: torch.Tensor | None = None,
    scale: torch.Tensor | None = None,
    shift: torch.Tensor | None = None,
    *,
    weight: torch.Tensor | None = None,
    bias: torch.Tensor | None = None,
    norm: str = "layer",
    y_norm: str = "none",
    y_weight: torch.Tensor | None = None,
    residual_scale: float = 1.0,
    eps: float = 1e-6,
    cu_seqlens: torch.Tensor | None = None,
) -> tuple[torch.Tensor, torch.Tensor | None]:
    """The stream after a block and the next block's normed input, ``(r, h)``:

    ``r = residual_scale * x + gate * (y_norm(y) * y_weight)`` and
    ``h = (norm(r) * weight + bias) * (1 + scale) + shift``.

    x is the stream, y the block's output (same shape and dtype).  ``y_norm``
    "none", "rms" or "layer" is a norm on the block's output; y_weight [C] needs
    one.  ``norm="none"`` leaves h out (returns ``(r, None)``).  gate takes the
    forms of scale and shift; see ``norm_modulate`` for the rest.  h is computed
    from r before r is rounded to x's dtype.
    """
    what = "gated_residual_norm"
    _check_stream(what, "x", x)
    _check_stream(what, "y", y, x)
    _check_cu(what, x, cu_seqlens)
    if norm not in _ops.NORM_KINDS or y_norm not in _ops.NORM_KINDS:
        raise ValueError(f"{what}: norm and y_norm must be 'none', 'rms' or 'layer'")
    if norm == "none" and not (scale is shift is weight is bias is None):
        raise ValueError(f"{what}: scale, shift, weight and bias need a norm")
    if y_norm == "none" and y_weight is not None:
        raise ValueError(f"{what}: y_weight needs y_norm")
    gate, scale, shift, shape, per_token = _modulation(what, x, cu_seqlens, gate, scale, shift)
    for name, v in (("weight", weight), ("bias", bias), ("y_weight", y_weight)):
        if v is not None:
            _channels(what, x, name, v)
    _finish_checks(what, x, eps)
    cu = None if cu_seqlens is None else cu_seqlens.contiguous()
    out = _run(what, shape, x, y, gate, scale, shift, weight, bias, y_weight, cu, _ops.NORM_KINDS[norm], _ops.NORM_KINDS[y_norm],
               float(eps), float(residual_scale), per_token)
    return out[0], None if norm == "none" else out[1]
