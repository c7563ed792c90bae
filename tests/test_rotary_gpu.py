"""Rotary positions with several axes against the definition in 64 bits.

Tolerance: the output's half rounding step, and (|x0| + |x1|) 2^-21 for the f32
part: an angle is off by at most 2^-25 turns (2^-22.3 rad), sine and cosine by
about one unit in 2^-23, two products and a sum by 2^-24 each.
"""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"
SUB = {torch.float16: 2.0 ** -25, torch.bfloat16: 0.0, torch.float32: 0.0}  # half a subnormal step


def _ref(x, pos, axes, thetas, inter, sign=1.0):
    """(value, f32 error bound) in 64 bits; x [B,H,S,D], pos [B or 1,S,A]."""
    x, pos = x.double(), pos.double()
    ang = torch.cat([pos[..., a, None] * torch.tensor([t ** (-2.0 * j / d) for j in range(d // 2)], dtype=torch.float64, device=x.device)
                     for a, (d, t) in enumerate(zip(axes, thetas)) if d], -1)[:, None] * sign
    R = sum(axes)
    c, s = torch.cos(ang), torch.sin(ang)
    a, b = (x[..., 0:R:2], x[..., 1:R:2]) if inter else (x[..., :R // 2], x[..., R // 2:R])
    out, err = x.clone(), torch.zeros_like(x)
    e = (a.abs() + b.abs()) * 2.0 ** -21
    idx = (slice(0, R, 2), slice(1, R, 2)) if inter else (slice(0, R // 2), slice(R // 2, R))
    out[..., idx[0]], out[..., idx[1]] = a * c - b * s, a * s + b * c
    err[..., idx[0]], err[..., idx[1]] = e, e
    return out, err


def _close(got, ref, err):
    tol = torch.finfo(got.dtype).eps / 2 * (ref.abs() + err) + err + SUB[got.dtype]
    d = (got.double() - ref).abs()
    assert bool((d <= tol).all()), float((d - tol).max())


def _rand(seed, *shape, dtype=torch.bfloat16):
    return torch.randn(*shape, generator=torch.Generator(device=DEV).manual_seed(seed), device=DEV).to(dtype)


def _pos(seed, *lead, axes, dtype=torch.int32, top=4000):
    g = torch.Generator(device=DEV).manual_seed(seed)
    p = torch.rand(*lead, axes, generator=g, device=DEV) * top - top / 8
    return p if dtype == torch.float32 else p.to(dtype)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("B,H,Hk,S,D,axes,inter", [
    (1, 3, 3, 1, 128, (44, 42, 42), True),
    (2, 4, 1, 37, 128, (32, 48, 48), False),
    (1, 5, 2, 300, 64, (16, 24, 24), True),
    (3, 2, 2, 19, 64, (16, 24), True),          # 24 channels pass
    (2, 2, 1, 65, 80, (20, 30, 30), False),     # half of 80 is no multiple of a vector in 16 bits
    (1, 2, 2, 33, 72, (10, 12, 8, 6), False),   # 36 pass, four axes
    (1, 2, 2, 9, 7, (2, 4), True),              # odd head dim
    (1, 1, 1, 130, 256, (256,), True),
    (1, 40, 40, 1500, 128, (0, 64, 64), True),  # an axis of no channel; several tokens per CTA
    (3, 30, 31, 333, 256, (128, 128), True),    # more heads than a CTA visits; batch items end inside its tokens
    (2, 70, 1, 90, 256, (200,), False),
    (1, 900, 1, 3, 8, (8,), True),
    (2, 1, 0, 700, 16, (4, 4), False),          # one head, 16 tokens per CTA
])
def test_matches_definition(B, H, Hk, S, D, axes, inter, dtype):
    from minimaxh3_b200.kernels.rotary import rotary_axes

    q, k = _rand(1, B, H, S, D, dtype=dtype), _rand(2, B, Hk, S, D, dtype=dtype)
    thetas = [10000.0, 256.0, 50.0, 7.0][:len(axes)]
    for pos in (_pos(3, S, axes=len(axes)), _pos(4, B, S, axes=len(axes), dtype=torch.int64), _pos(5, 1, S, axes=len(axes), dtype=torch.float32)):
        oq, ok = rotary_axes(q, k, pos, axes, theta=thetas, interleaved=inter)
        p3 = pos if pos.dim() == 3 else pos[None]
        _close(oq, *_ref(q, p3, axes, thetas, inter))
        if Hk:
            _close(ok, *_ref(k, p3, axes, thetas, inter))
        R = sum(axes)
        assert torch.equal(oq[..., R:], q[..., R:]) and torch.equal(ok[..., R:], k[..., R:])
        only, none = rotary_axes(q, None, pos, axes, theta=thetas, interleaved=inter)
        assert none is None and torch.equal(only, oq)


@pytest.mark.parametrize("inter", [True, False])
def test_strided_views_and_packed_rows(inter):
    """Views of a fused projection, a transposed layout, odd strides, and packed [T, H, D]."""
    from minimaxh3_b200.kernels.rotary import rotary_axes

    B, H, S, D, axes = 2, 4, 50, 64, (16, 24, 24)
    pos = _pos(6, S, axes=3)
    qkv = _rand(7, B, S, 3 * H, D)
    q, k = qkv[:, :, :H].transpose(1, 2), qkv[:, :, H:2 * H].transpose(1, 2)
    base = rotary_axes(q.contiguous(), k.contiguous(), pos, axes, interleaved=inter)
    got = rotary_axes(q, k, pos, axes, interleaved=inter)
    assert torch.equal(got[0], base[0]) and torch.equal(got[1], base[1]) and got[0].stride(3) == 1
    odd = _rand(8, B, H, S, D + 3)[..., 1:D + 1]  # rows of 67 elements, one element off
    assert torch.equal(rotary_axes(odd, None, pos, axes, interleaved=inter)[0],
                       rotary_axes(odd.contiguous(), None, pos, axes, interleaved=inter)[0])
    chan = _rand(9, B, H, D, S).transpose(2, 3)  # channels not contiguous
    assert torch.equal(rotary_axes(chan, None, pos, axes, interleaved=inter)[0],
                       rotary_axes(chan.contiguous(), None, pos, axes, interleaved=inter)[0])
    shared = _rand(10, B, 1, S, D).expand(B, H, S, D)  # one key head behind every query head
    assert torch.equal(rotary_axes(shared, None, pos, axes, interleaved=inter)[0],
                       rotary_axes(shared.contiguous(), None, pos, axes, interleaved=inter)[0])
    packed = rotary_axes(q[0].transpose(0, 1), k[0].transpose(0, 1), pos, axes, interleaved=inter)
    assert torch.equal(packed[0].transpose(0, 1), base[0][0]) and torch.equal(packed[1].transpose(0, 1), base[1][0])
    tpos = torch.stack([pos[:, 2], pos[:, 1], pos[:, 0]], 0).t().flip(1)  # positions with a stride
    assert torch.equal(rotary_axes(q, None, tpos, axes, interleaved=inter)[0], base[0])


def test_in_place_outputs():
    from minimaxh3_b200 import ops

    for D, axes, inter in ((64, (16, 24, 24), True), (64, (16, 24, 24), False), (30, (10, 8), False)):
        q, pos = _rand(11, 2, 3, 40, D), _pos(12, 40, axes=len(axes))
        ref = ops.rotary(q, None, pos, axes, [1e4] * len(axes), inter)[0]
        got = ops.rotary(q, None, pos, axes, [1e4] * len(axes), inter, out_q=q)[0]
        assert got.data_ptr() == q.data_ptr() and torch.equal(q, ref)


def test_far_positions_keep_their_angle():
    from minimaxh3_b200.kernels.rotary import rotary_axes

    q = _rand(13, 1, 1, 5, 64, dtype=torch.float32)
    pos = torch.tensor([0, 1, 1_000_003, 2 ** 31 - 1, -(2 ** 31)], dtype=torch.int64, device=DEV)[:, None]
    _close(rotary_axes(q, None, pos, (64,))[0], *_ref(q, pos[None], (64,), (10000.0,), True))
    _close(rotary_axes(q, None, pos.to(torch.int32), (64,))[0], *_ref(q, pos[None], (64,), (10000.0,), True))


@pytest.mark.parametrize("inter", [True, False])
def test_infinities_and_nan_stay_in_their_pair(inter):
    from minimaxh3_b200.kernels.rotary import rotary_axes

    D, axes = 32, (8, 4)
    q = _rand(14, 1, 2, 6, D)
    clean = rotary_axes(q, None, _pos(15, 6, axes=2), axes, interleaved=inter)[0]
    bad = q.clone()
    bad[0, 0, 2, 20] = float("inf")  # a passing channel
    bad[0, 1, 3, 13] = float("nan")
    bad[0, 0, 4, 2] = float("nan")   # a rotated one
    got = rotary_axes(bad, None, _pos(15, 6, axes=2), axes, interleaved=inter)[0]
    pair = (2, 3) if inter else (2, 8)
    hit = torch.zeros_like(q, dtype=torch.bool)
    hit[0, 0, 2, 20] = hit[0, 1, 3, 13] = hit[0, 0, 4, pair[0]] = hit[0, 0, 4, pair[1]] = True
    assert torch.equal(got[~hit], clean[~hit]) and bool((~got[hit].isfinite()).all())


def test_empty_and_large_offsets():
    from minimaxh3_b200.kernels.rotary import rotary_axes

    for shape in ((0, 2, 5, 32), (2, 0, 5, 32), (2, 3, 0, 32)):
        q = _rand(16, *shape)
        oq, ok = rotary_axes(q, q, torch.zeros(shape[2], 1, dtype=torch.int32, device=DEV), (32,))
        assert oq.shape == q.shape and ok.shape == q.shape
    far = 2 ** 31 + 64  # elements between the two batch items
    buf = torch.zeros(far + 2 * 5 * 32, dtype=torch.bfloat16, device=DEV)
    q = buf.as_strided((2, 2, 5, 32), (far, 5 * 32, 32, 1))
    q.copy_(_rand(17, 2, 2, 5, 32))
    pos = _pos(18, 5, axes=1)
    assert torch.equal(rotary_axes(q, None, pos, (32,))[0], rotary_axes(q.contiguous(), None, pos, (32,))[0])


@pytest.mark.parametrize("inter", [True, False])
def test_gradient_is_the_inverse_rotation(inter):
    from minimaxh3_b200.kernels.rotary import rotary_axes

    B, H, S, D, axes = 2, 3, 21, 40, (12, 10, 14)
    pos = _pos(19, S, axes=3)
    q, k = (_rand(s, B, H, S, D, dtype=torch.float32).requires_grad_(True) for s in (20, 21))
    dq, dk = _rand(22, B, H, S, D, dtype=torch.float32), _rand(23, B, H, S, D, dtype=torch.float32)
    oq, ok = rotary_axes(q, k, pos, axes, interleaved=inter)
    gq, gk = torch.autograd.grad((oq, ok), (q, k), (dq, dk))
    _close(gq, *_ref(dq, pos[None], axes, (1e4,) * 3, inter, -1.0))
    _close(gk, *_ref(dk, pos[None], axes, (1e4,) * 3, inter, -1.0))
    # against differences of the 64-bit forward: it is linear in q, so a step of any size gives the slope
    v = _rand(24, B, H, S, D, dtype=torch.float32)
    f = lambda t: (_ref(t, pos[None], axes, (1e4,) * 3, inter)[0] * dq.double()).sum()
    slope = (f(q.detach().double() + v.double()) - f(q.detach().double() - v.double())) / 2
    bound = ((v.double().abs() * (gq.double().abs() * 2.0 ** -24 + dq.double().abs().amax() * 2.0 ** -19)).sum())
    assert abs((gq.double() * v.double()).sum() - slope) <= bound
    # only one of the two gradients is asked for, and one input without a gradient
    (only,) = torch.autograd.grad(rotary_axes(q, k.detach(), pos, axes, interleaved=inter)[0], q, dq)
    assert torch.equal(only, gq)
    # twice: the gradient is linear in dq, and its own gradient turns forward
    d1 = dq.clone().requires_grad_(True)
    (g1,) = torch.autograd.grad(rotary_axes(q, k, pos, axes, interleaved=inter)[0], q, d1, create_graph=True)
    assert torch.equal(g1, gq)
    assert torch.equal(torch.autograd.grad(g1, d1, v)[0], rotary_axes(v, None, pos, axes, interleaved=inter)[0])
    # shared key heads: the gradient of the one head is the sum over its copies
    kv = _rand(25, B, 1, S, D, dtype=torch.float32).requires_grad_(True)
    (gs,) = torch.autograd.grad(rotary_axes(kv.expand(B, H, S, D), None, pos, axes, interleaved=inter)[0], kv, dq)
    torch.testing.assert_close(gs, gq.sum(1, keepdim=True), rtol=2.0 ** -22, atol=2.0 ** -20)


def test_captured_replayed_on_other_streams_and_compiled():
    from minimaxh3_b200.kernels.rotary import rotary_axes

    q, k, pos = _rand(26, 1, 4, 100, 64), _rand(27, 1, 2, 100, 64), _pos(28, 100, axes=2)
    ref = rotary_axes(q, k, pos, (32, 32))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = rotary_axes(q, k, pos, (32, 32))
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got[0], ref[0]) and torch.equal(got[1], ref[1])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        cap = rotary_axes(q, k, pos, (32, 32))
    q.copy_(_rand(29, 1, 4, 100, 64))
    graph.replay()
    torch.cuda.synchronize()
    ref = rotary_axes(q, k, pos, (32, 32))
    assert torch.equal(cap[0], ref[0]) and torch.equal(cap[1], ref[1])
    f = torch.compile(lambda a, b: rotary_axes(a, b, pos, (32, 32)), fullgraph=True, backend="aot_eager")
    got = f(q, k)
    assert torch.equal(got[0], ref[0]) and torch.equal(got[1], ref[1])


def test_varlen_attention_takes_the_positions():
    from minimaxh3_b200.kernels.fp8_attention import fp8_attention_varlen
    from minimaxh3_b200.kernels.rotary import Rotary, rotary_axes

    lens, H, D, axes = [200, 57], 2, 64, (16, 24, 24)
    T = sum(lens)
    cu = torch.tensor([0, lens[0], T], dtype=torch.int32, device=DEV)
    q, k, v = (_rand(s, T, H, D) for s in (30, 31, 32))
    pos = _pos(33, T, axes=3)
    got = fp8_attention_varlen(q, k, v, cu, cu, max(lens), rotary=Rotary(pos, axes))
    tq, tk = rotary_axes(q, k, pos, axes)
    assert torch.equal(got, fp8_attention_varlen(tq, tk, v, cu, cu, max(lens)))
    assert not torch.equal(got, fp8_attention_varlen(q, k, v, cu, cu, max(lens)))
