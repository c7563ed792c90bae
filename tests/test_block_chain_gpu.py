"""The operators together, as a block uses them: the modulated norm, 4-bit and FP8 linears with an
adapter, rotary positions, packed attention, and the gated residual with the next norm.

Against the same block in 64 bits, on the weights that the 4-bit and 8-bit layers hold.  What differs
is the rounding of activations: e2m1 leaves at most half a step of 1/2 at 1 (a quarter of the value)
and on average a relative 0.1 of a block's size, e4m3 2^-4.  A linear of independent channels keeps
that relative size, attention's values average it down, and each enters the stream behind a gate of
0.5 beside x itself - so the stream is off by less than 0.2 of its norm, the normed output by less
than 0.2 of its own.
"""
import math

import pytest
import torch
import torch.nn as nn

pytestmark = pytest.mark.gpu
DEV = "cuda"
LENS, H, D = [300, 113], 4, 64
C, AXES = H * D, (16, 24, 24)


def _rand(seed, *shape, scale=1.0, dtype=torch.bfloat16):
    return (torch.randn(*shape, generator=torch.Generator().manual_seed(seed)) * scale).to(dtype).to(DEV)


def _layers():
    from minimaxh3_b200.kernels.fp4_linear import FP4Linear, dequantize_fp4
    from minimaxh3_b200.kernels.fp8_linear import FP8Linear

    made, values = {}, {}
    for i, (name, n, k, kind) in enumerate((("qkv", 3 * C, C, FP4Linear), ("out", C, C, FP4Linear), ("up", 4 * C, C, FP8Linear), ("down", C, 4 * C, FP4Linear))):
        lin = nn.Linear(k, n).to(torch.bfloat16).to(DEV)
        with torch.no_grad():
            lin.weight.copy_(_rand(10 + i, n, k, scale=k ** -0.5))
            lin.bias.copy_(_rand(20 + i, n, scale=0.1))
        bias = lin.bias.detach().double()
        m = made[name] = kind.from_linear(lin)
        w = dequantize_fp4(m.w4, m.w_blocks, m.w_scale).double() if kind is FP4Linear else m.w8.double() * m.w_scale.reshape(-1, 1).double()
        values[name] = (w, bias)
    A, B = _rand(30, 16, C, scale=C ** -0.5), _rand(31, 3 * C, 16, scale=0.05)
    made["qkv"].adapters = [(A, B, 1.0)]
    values["lora"] = (A.double(), B.double())
    return made, values


def _mods(seed):
    return {n: _rand(seed + i, len(LENS), C, scale=0.3, dtype=torch.float32) for i, n in enumerate(("sc1", "sh1", "sc2", "sh2"))} | {
        "g1": torch.full((len(LENS), C), 0.5, device=DEV), "g2": torch.full((len(LENS), C), 0.5, device=DEV)}


def _block(x, layers, mod, cu, pos):
    from minimaxh3_b200.kernels.block_norm import gated_residual_norm, norm_modulate
    from minimaxh3_b200.kernels.fp8_attention import fp8_attention_varlen
    from minimaxh3_b200.kernels.rotary import Rotary

    h = norm_modulate(x, mod["sc1"], mod["sh1"], cu_seqlens=cu)
    q, k, v = layers["qkv"](h).view(-1, 3, H, D).unbind(1)
    a = fp8_attention_varlen(q, k, v, cu, cu, max(LENS), rotary=Rotary(pos, AXES))
    r, h = gated_residual_norm(x, layers["out"](a.reshape(-1, C)), mod["g1"], mod["sc2"], mod["sh2"], cu_seqlens=cu)
    y = layers["down"](torch.nn.functional.gelu(layers["up"](h)))
    return gated_residual_norm(r, y, mod["g2"], y_norm="rms", norm="rms", cu_seqlens=cu)


def _ref(x, val, mod, pos):
    rep = torch.repeat_interleave(torch.arange(len(LENS)), torch.tensor(LENS)).to(DEV)
    m = {n: t.double()[rep] for n, t in mod.items()}
    ln = lambda t: (t - t.mean(-1, keepdim=True)) / (t.var(-1, keepdim=True, unbiased=False) + 1e-6).sqrt()
    rms = lambda t: t / (t.pow(2).mean(-1, keepdim=True) + 1e-6).sqrt()
    lin = lambda n, t: t @ val[n][0].t() + val[n][1]
    x = x.double()
    h = ln(x) * (1 + m["sc1"]) + m["sh1"]
    q, k, v = (lin("qkv", h) + h @ val["lora"][0].t() @ val["lora"][1].t()).view(-1, 3, H, D).unbind(1)
    ang = torch.cat([pos[:, i, None].double() * 10000.0 ** (-2 * torch.arange(d // 2, device=DEV, dtype=torch.float64) / d) for i, d in enumerate(AXES)], -1)[:, None]

    def turn(t):
        a, b = t[..., 0::2], t[..., 1::2]
        return torch.stack([a * ang.cos() - b * ang.sin(), a * ang.sin() + b * ang.cos()], -1).flatten(-2)

    q, k = turn(q), turn(k)
    out, at = [], 0
    for n in LENS:
        s = torch.einsum("qhd,khd->hqk", q[at:at + n], k[at:at + n]) / math.sqrt(D)
        out.append(torch.einsum("hqk,khd->qhd", s.softmax(-1), v[at:at + n]).reshape(n, C))
        at += n
    r = x + m["g1"] * lin("out", torch.cat(out))
    h = ln(r) * (1 + m["sc2"]) + m["sh2"]
    r = r + m["g2"] * rms(lin("down", torch.nn.functional.gelu(lin("up", h))))
    return r, rms(r)


def test_block_matches_and_replays():
    T = sum(LENS)
    cu = torch.tensor([0, LENS[0], T], dtype=torch.int32, device=DEV)
    pos = torch.randint(0, 60, (T, 3), generator=torch.Generator().manual_seed(5), dtype=torch.int32).to(DEV)
    layers, val = _layers()
    x, mod = _rand(1, T, C), _mods(40)
    r, h = _block(x, layers, mod, cu, pos)
    for got, ref in zip((r, h), _ref(x, val, mod, pos)):
        assert float((got.double() - ref).norm() / ref.norm()) < 0.2
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        r2, h2 = _block(x, layers, mod, cu, pos)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(r, r2) and torch.equal(h, h2)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        cap = _block(x, layers, mod, cu, pos)
    x.copy_(_rand(2, T, C))
    graph.replay()
    torch.cuda.synchronize()
    r, h = _block(x, layers, mod, cu, pos)
    assert torch.equal(cap[0], r) and torch.equal(cap[1], h)


def test_one_token_of_a_stream():
    """A block on one token: the smallest call of every operator, the token being the stream's last."""
    from minimaxh3_b200.kernels.block_norm import gated_residual_norm, norm_modulate
    from minimaxh3_b200.kernels.rotary import rotary_axes

    layers, _ = _layers()
    x = _rand(3, 40, C)
    mod = {n: t[:1] for n, t in _mods(50).items()}

    def front(t, pos):
        h = norm_modulate(t, mod["sc1"], mod["sh1"])
        q, k, _ = layers["qkv"](h).view(-1, 3, H, D).unbind(1)
        return (h, *rotary_axes(q, k, pos, AXES), *gated_residual_norm(t, h, mod["g1"], mod["sc2"], mod["sh2"]))

    pos = torch.arange(120, dtype=torch.int32, device=DEV).view(40, 3)
    whole, one = front(x, pos), front(x[39:], pos[39:])
    for a, b in zip(whole, one):
        # the linear's two kernels add in another order (2^-8 of a value and of the row's largest)
        assert bool(((a[39:].double() - b.double()).abs() <= 2.0 ** -7 * b.double().abs() + 2.0 ** -8 * b.double().abs().amax()).all())
    assert torch.equal(whole[0][39:], one[0]) and torch.equal(whole[3][39:], one[3]) and torch.equal(whole[4][39:], one[4])


def test_training_step_on_the_elementwise_operators():
    """Gradients through the chain of norms and rotation equal those of the 64-bit chain."""
    from minimaxh3_b200.kernels.block_norm import gated_residual_norm, norm_modulate
    from minimaxh3_b200.kernels.rotary import rotary_axes

    T = 37
    pos = torch.randint(0, 60, (T, 3), generator=torch.Generator().manual_seed(6), dtype=torch.int32).to(DEV)
    leaf = lambda s, *sh: _rand(s, *sh, dtype=torch.float32).requires_grad_(True)
    t = [leaf(60, T, C), leaf(61, C), leaf(62, C), leaf(63, C), leaf(64, C)]
    dr, dh = _rand(65, T, C, dtype=torch.float32), _rand(66, T, C, dtype=torch.float32)

    def ours(x, sc, sh, g, w):
        h = norm_modulate(x, sc, sh, weight=w)
        q, _ = rotary_axes(h.view(T, H, D), None, pos, AXES)
        return gated_residual_norm(x, q.reshape(T, C), g, sc, sh, y_norm="layer", residual_scale=0.5)

    def plain(x, sc, sh, g, w):
        ln = lambda v: (v - v.mean(-1, keepdim=True)) * ((v - v.mean(-1, keepdim=True)).pow(2).mean(-1, keepdim=True) + 1e-6).rsqrt()
        h = (ln(x) * w * (1 + sc) + sh).view(T, H, D)
        ang = torch.cat([pos[:, i, None].double() * 10000.0 ** (-2 * torch.arange(d // 2, device=DEV, dtype=torch.float64) / d) for i, d in enumerate(AXES)], -1)[:, None]
        a, b = h[..., 0::2], h[..., 1::2]
        y = torch.stack([a * ang.cos() - b * ang.sin(), a * ang.sin() + b * ang.cos()], -1).reshape(T, C)
        r = 0.5 * x + g * ln(y)
        return r, ln(r) * (1 + sc) + sh

    got = torch.autograd.grad(ours(*t), t, (dr, dh))
    t64 = [v.detach().double().requires_grad_(True) for v in t]
    want = torch.autograd.grad(plain(*t64), t64, (dr.double(), dh.double()))
    for a, b in zip(got, want):
        # three norms and a rotation, each within 64 * 2^-24 (1 + max/sigma ~ 5) of its values: 2^-15 of the gradient's norm
        assert float((a.double() - b).norm() / b.norm()) < 2.0 ** -15


def test_training_step_is_captured():
    """Forward and backward in a CUDA graph give the eager gradients, while an eager graph of other leaves lives."""
    from minimaxh3_b200.kernels.block_norm import gated_residual_norm
    from minimaxh3_b200.kernels.rotary import rotary_axes

    T = 50
    pos = torch.randint(0, 60, (T, 3), generator=torch.Generator().manual_seed(7), dtype=torch.int32).to(DEV)

    def step(x, y, g):
        q, _ = rotary_axes(y.view(T, H, D), None, pos, AXES)
        r, h = gated_residual_norm(x, q.reshape(T, C), g, y_norm="rms")
        return torch.autograd.grad((r, h), (x, y, g), (torch.ones_like(r), torch.ones_like(h)))

    make = lambda s: [_rand(s, T, C).requires_grad_(True), _rand(s + 1, T, C).requires_grad_(True), _rand(s + 2, C).requires_grad_(True)]
    alive = make(70)
    r, _ = gated_residual_norm(*alive)  # an eager graph that is not run back
    leaves = make(80)
    ref = step(*leaves)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        cap = step(*leaves)
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(ref, cap)) and r.requires_grad


def test_operators_seen_by_a_dispatch_mode():
    """Under a mode that watches operators they go through the dispatcher, with the same results."""
    from torch.utils._python_dispatch import TorchDispatchMode

    from minimaxh3_b200.kernels.block_norm import gated_residual_norm, norm_modulate
    from minimaxh3_b200.kernels.fp4_linear import fp4_linear, quantize_fp4
    from minimaxh3_b200.kernels.rotary import rotary_axes

    class Watch(TorchDispatchMode):
        def __init__(self):
            super().__init__()
            self.seen = set()

        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            self.seen.add(func.name())
            return func(*args, **(kwargs or {}))

    g = torch.Generator().manual_seed(7)
    rnd = lambda *s: torch.randn(*s, generator=g).to(torch.bfloat16).cuda()  # noqa: E731
    x, y, gate, q, k = rnd(2, 33, 64), rnd(2, 33, 64), rnd(2, 64), rnd(2, 4, 33, 32), rnd(2, 2, 33, 32)
    pos = torch.arange(33, dtype=torch.int32).view(33, 1).cuda()
    w = quantize_fp4(rnd(48, 64))

    def run():
        leaves = [t.detach().clone().requires_grad_(True) for t in (x, y, gate, q, k)]
        a, b, c, d, e = leaves
        r, h = gated_residual_norm(a, b, c)
        outs = (r, norm_modulate(h, c), *rotary_axes(d, e, pos, (32,)))
        grads = torch.autograd.grad(outs, leaves, [torch.ones_like(o) for o in outs])
        with torch.no_grad():
            return [*outs, *grads, fp4_linear(x, *w)]

    plain, watch = run(), Watch()
    with watch:
        seen = run()
    assert all(torch.equal(a, b) for a, b in zip(plain, seen, strict=True))
    assert {"mh3::block_norm", "mh3::rotary_axes", "mh3::fp4_linear"} <= watch.seen
