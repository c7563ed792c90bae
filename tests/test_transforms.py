"""The block operators where something traces, transforms or intercepts operators.

Plain calls go to the kernels directly; under ``torch.jit.trace``, ``torch.vmap``, the function
transforms and tensor subclasses they have to go through the dispatcher, which serves those.
"""
import warnings

import pytest
import torch

from minimaxh3_b200 import ops

DEV = "cuda"


class _Sub(torch.Tensor):
    pass


def test_plain_tensors_are_plain():
    x = torch.zeros(2, 3)
    assert ops.plain(x) and ops.plain(x, None, torch.nn.Parameter(x)) and ops.plain() and ops.plain_backward(x, None)
    with torch.no_grad():
        assert ops.plain(x)
    with torch.inference_mode():
        assert ops.plain(x, torch.zeros(2))
    with torch.autocast("cpu"):
        assert ops.plain(x)
    assert not ops.plain(x.as_subclass(_Sub)) and not ops.plain(x, None, x.as_subclass(_Sub))


def test_what_traces_or_transforms_is_not_plain():
    x = torch.zeros(2, 3)
    seen = []

    def f(t):
        seen.append(ops.plain(x) or ops.plain(t))
        return (t * 2).sum()

    with warnings.catch_warnings():
        warnings.simplefilter("ignore")
        torch.jit.trace(f, (x,), check_trace=False)
    torch.vmap(f)(x)
    torch.func.grad(f)(x)
    torch.func.jvp(f, (x,), (x,))
    torch.func.functionalize(f)(x)
    assert seen == [False] * 5


def test_a_batched_backward_is_not_plain():
    seen = []

    class Double(torch.autograd.Function):
        @staticmethod
        def forward(ctx, a):
            return a * 2

        @staticmethod
        def backward(ctx, g):
            seen.append(ops.plain_backward(g, None) or ops.plain_backward(None, g) or ops.plain_backward(x, g))
            return g * 2

    x = torch.zeros(3, requires_grad=True)
    g, = torch.autograd.grad(Double.apply(x), x, torch.eye(3), is_grads_batched=True)
    assert seen == [False] and torch.equal(g, 2 * torch.eye(3))


def _rand(seed, *shape, dtype=torch.bfloat16):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).to(dtype).to(DEV)


def _pos(n):
    return torch.arange(2 * n, dtype=torch.int32, device=DEV).view(n, 2)


def _calls():
    """name -> (function, inputs, other inputs)."""
    from minimaxh3_b200.kernels.block_norm import gated_residual_norm, norm_modulate
    from minimaxh3_b200.kernels.fp4_linear import fp4_linear, quantize_fp4
    from minimaxh3_b200.kernels.rotary import rotary_axes

    w, pos, A, B = quantize_fp4(_rand(1, 48, 64)), _pos(9), _rand(2, 8, 64), _rand(3, 48, 8)
    two = lambda *shapes: [tuple(_rand(10 * s + i, *sh) for i, sh in enumerate(shapes)) for s in (1, 2)]  # noqa: E731
    return {
        "rotary": (lambda q, k: rotary_axes(q, k, pos, (16, 16)), *two((1, 4, 9, 32), (1, 2, 9, 32))),
        "norm": (lambda x, s: norm_modulate(x, s, s), *two((2, 9, 64), (2, 64))),
        "gated": (lambda x, y, g: gated_residual_norm(x, y, g, y_norm="rms"), *two((2, 9, 64), (2, 9, 64), (2, 64))),
        "linear": (lambda x: fp4_linear(x, *w), *two((9, 64))),
        "linear with an adapter": (lambda x: fp4_linear(x, *w, adapters=[(A, B, 0.5)]), *two((9, 64))),
    }


def _same(a, b):
    a, b = ((t,) if isinstance(t, torch.Tensor) else t for t in (a, b))
    assert len(a) == len(b) and all(u.dtype == v.dtype and torch.equal(u.view(torch.uint8), v.view(torch.uint8)) for u, v in zip(a, b))


@pytest.mark.gpu
@pytest.mark.parametrize("name", ["rotary", "norm", "gated", "linear", "linear with an adapter"])
def test_traced_calls_compute(name):
    f, first, second = _calls()[name]
    with torch.no_grad(), warnings.catch_warnings():
        warnings.simplefilter("ignore")
        traced = torch.jit.trace(f, first, check_trace=False)
        assert "mh3::" in str(traced.graph)
        _same(traced(*first), f(*first))
        _same(traced(*second), f(*second))


@pytest.mark.gpu
def test_vmap_turns_each_item():
    from minimaxh3_b200.kernels.rotary import rotary_axes

    q, k, pos = _rand(1, 3, 1, 4, 9, 32), _rand(2, 3, 1, 2, 9, 32), _pos(9)
    got = torch.vmap(lambda a, b: rotary_axes(a, b, pos, (16, 16)))(q, k)
    for i in range(3):
        _same([t[i] for t in got], rotary_axes(q[i], k[i], pos, (16, 16)))
    # the first tensor plain, a later one mapped
    got = torch.vmap(lambda b: rotary_axes(q[0], b, pos, (16, 16))[1])(k)
    _same([got[2]], [rotary_axes(q[0], k[2], pos, (16, 16))[1]])


@pytest.mark.gpu
def test_batched_gradients_of_the_rotation():
    from minimaxh3_b200.kernels.rotary import rotary_axes

    q, g = _rand(1, 1, 2, 5, 32, dtype=torch.float32).requires_grad_(True), _rand(2, 3, 1, 2, 5, 32, dtype=torch.float32)
    out = rotary_axes(q, None, _pos(5), (16, 16))[0]
    got, = torch.autograd.grad(out, q, g, is_grads_batched=True, retain_graph=True)
    for i in range(3):
        assert torch.equal(got[i], torch.autograd.grad(out, q, g[i], retain_graph=True)[0])
    twice, = torch.autograd.grad(out, q, g, is_grads_batched=True, create_graph=True)
    assert torch.equal(twice, got)


@pytest.mark.gpu
def test_a_transform_that_cannot_be_served_raises():
    """An operator that returns a list has no fallback under vmap: an error, not a wrong answer."""
    from minimaxh3_b200.kernels.block_norm import norm_modulate

    with pytest.raises(RuntimeError, match="atching rule"):
        torch.vmap(norm_modulate)(_rand(1, 3, 5, 64))


def test_what_is_no_tensor_is_refused_as_before():
    from minimaxh3_b200.kernels.fp4_linear import quantize_fp4

    with pytest.raises(ValueError, match="2D"):
        quantize_fp4([[1.0] * 32])


def test_four_bit_conversions_are_operators():
    """Their shapes and types without data, as a trace or a compiler asks for them."""
    from torch._subclasses.fake_tensor import FakeTensorMode

    from minimaxh3_b200.kernels.fp4_linear import dequantize_fp4, fp4_matmul, quantize_fp4

    with FakeTensorMode():
        x, w = (torch.empty(m, 96, dtype=torch.bfloat16, device=DEV) for m in (130, 16))
        a, b = quantize_fp4(x), quantize_fp4(w)
        assert [(tuple(t.shape), t.dtype) for t in a] == [((130, 48), torch.uint8), ((2, 2, 32, 4, 4), torch.float8_e4m3fn), ((130, 1), torch.float32)]
        for dt in (torch.bfloat16, torch.float32):
            v = dequantize_fp4(*a, dtype=dt)
            assert tuple(v.shape) == (130, 96) and v.dtype == dt and v.device.type == DEV
        out = fp4_matmul(a, b)
        assert tuple(out.shape) == (130, 16) and out.dtype == torch.bfloat16


@pytest.mark.gpu
def test_traced_and_compiled_four_bit_conversions_compute():
    from minimaxh3_b200.kernels.fp4_linear import dequantize_fp4, fp4_matmul, quantize_fp4

    w = quantize_fp4(_rand(3, 16, 96))

    def f(x):
        a = quantize_fp4(x)
        return (*a, dequantize_fp4(*a), fp4_matmul(a, w))

    x, y = _rand(1, 130, 96), _rand(2, 130, 96)
    with torch.no_grad(), warnings.catch_warnings():
        warnings.simplefilter("ignore")
        for g in (torch.jit.trace(f, (x,), check_trace=False), torch.compile(f, backend="aot_eager", fullgraph=True)):
            _same(g(x), f(x))
            _same(g(y), f(y))


def _dual(t):
    return torch.autograd.forward_ad.make_dual(t, torch.ones_like(t))


def test_forward_mode_is_refused():
    """A tangent, or a function transform inside which one may hide; what carries none is let through."""
    x = torch.zeros(2, 3)
    ops.refuse_forward_mode("f", x, None)
    with torch.autograd.forward_ad.dual_level():
        ops.refuse_forward_mode("f", x, None, 1.0)
        with pytest.raises(RuntimeError, match="f has no forward-mode"):
            ops.refuse_forward_mode("f", x, _dual(x))
    refuse = lambda t: (ops.refuse_forward_mode("f", t), t * 2)[1]  # noqa: E731
    torch.vmap(refuse)(x)
    for g in (refuse, torch.vmap(refuse), torch.func.grad(lambda t: refuse(t).sum())):
        with pytest.raises(RuntimeError, match="f has no forward-mode"):
            torch.func.jvp(g, (x,), (x,))


@pytest.mark.gpu
@pytest.mark.parametrize("name", ["rotary", "norm", "gated", "linear", "linear with an adapter"])
def test_forward_mode_calls_are_refused(name):
    f, inputs, _ = _calls()[name]
    with torch.autograd.forward_ad.dual_level():
        _same(f(*inputs), f(*inputs))
        for i in range(len(inputs)):
            with pytest.raises(RuntimeError, match="has no forward-mode derivative"):
                f(*(_dual(t) if i == j else t for j, t in enumerate(inputs)))


@pytest.mark.gpu
def test_forward_mode_four_bit_conversions_are_refused():
    from minimaxh3_b200.kernels.fp4_linear import dequantize_fp4, fp4_matmul, quantize_fp4

    x = _rand(1, 16, 64)
    v, b, s = quantize_fp4(x)
    with torch.autograd.forward_ad.dual_level():
        for f in (lambda: quantize_fp4(_dual(x)), lambda: dequantize_fp4(v, b, _dual(s)),
                  lambda: fp4_matmul((v, b, s), (v, b, _dual(s))), lambda: fp4_matmul((v, b, s), (v, b, s), _dual(x[:, 0].float()))):
            with pytest.raises(RuntimeError, match="has no forward-mode derivative"):
                f()


LAYOUTS = {  # of q [2, 4, 9, 32]
    "contiguous": lambda t: t(2, 4, 9, 32),
    "tokens first": lambda t: t(2, 9, 4, 32).transpose(1, 2),
    "of a fused projection": lambda t: t(2, 9, 12, 32)[:, :, 4:8].transpose(1, 2),
    "channels before tokens": lambda t: t(2, 4, 32, 9).transpose(2, 3),
    "channels first": lambda t: t(32, 9, 2, 4).permute(2, 3, 1, 0),
    "every other channel": lambda t: t(2, 4, 9, 64)[..., ::2],
    "every other channel, tokens first": lambda t: t(2, 9, 4, 64)[..., ::2].transpose(1, 2),
    "a shared head": lambda t: t(2, 1, 9, 32).expand(2, 4, 9, 32),
    "a padded row": lambda t: t(2, 4, 9, 40)[..., :32],
    "one channel for all": lambda t: t(2, 4, 9, 1).expand(2, 4, 9, 32),
}


def _fake_strides(layout):
    from torch._subclasses.fake_tensor import FakeTensorMode

    from minimaxh3_b200.kernels.rotary import rotary_axes

    with FakeTensorMode():
        q = LAYOUTS[layout](lambda *s: torch.empty(*s, dtype=torch.bfloat16, device=DEV))
        k = LAYOUTS[layout](lambda *s: torch.empty(*s, dtype=torch.bfloat16, device=DEV))
        return [t.stride() for t in rotary_axes(q, k, torch.empty(9, 2, dtype=torch.int32, device=DEV), (16, 16))]


@pytest.mark.parametrize("layout", LAYOUTS)
def test_rotary_strides_that_a_compiler_is_told(layout):
    """Contiguous channels, and the strides of the tensor that the real call makes."""
    t = LAYOUTS[layout](torch.empty)
    real = torch.empty_like(t.contiguous() if t.stride(-1) != 1 else t).stride()
    assert real[-1] == 1 and _fake_strides(layout) == [real, real]


@pytest.mark.gpu
@pytest.mark.parametrize("layout", LAYOUTS)
def test_rotary_strides_and_values_of_a_compiled_call(layout):
    from minimaxh3_b200.kernels.rotary import rotary_axes

    q, k, pos = LAYOUTS[layout](lambda *s: _rand(1, *s)), LAYOUTS[layout](lambda *s: _rand(2, *s)), _pos(9)
    f = lambda a, b: rotary_axes(a, b, pos, (16, 16))  # noqa: E731
    want = f(q, k)
    assert [t.stride() for t in want] == _fake_strides(layout)
    got = torch.compile(f, fullgraph=True, backend="aot_eager")(q, k)
    _same(got, want)
    assert [t.stride() for t in got] == [t.stride() for t in want]


@pytest.mark.gpu
def test_compiled_gradients_of_shared_modulations():
    """A [C] gate beside modulation by token, and [C] scale and shift of several batch items, forward and backward."""
    from minimaxh3_b200.kernels.block_norm import gated_residual_norm, norm_modulate

    def f(x, y, gate, scale, shift):
        r, h = gated_residual_norm(x, y, gate, scale, shift)
        return r, norm_modulate(h, gate, gate)

    leaves = [t.requires_grad_(True) for t in (_rand(1, 2, 9, 64), _rand(2, 2, 9, 64), _rand(3, 64), _rand(4, 2, 9, 64), _rand(5, 2, 64))]
    grads = _rand(6, 2, 9, 64), _rand(7, 2, 9, 64)
    want = f(*leaves)
    want = (*want, *torch.autograd.grad(want, leaves, grads))
    got = torch.compile(f, fullgraph=True, backend="aot_eager")(*leaves)
    _same((*got, *torch.autograd.grad(got, leaves, grads)), want)
