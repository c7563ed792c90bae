"""4-bit rows and their product against the definition.

Rounding is compared bit for bit with a 64-bit restatement.  A product's
tolerance: half a bf16 step (2^-8 of the result), and 2^-22 of the sum of the
products' magnitudes for every 64 elements of K (f32 accumulation on the tensor
cores, which cut off below 2^-23 of the running value).  With adapters the
low-rank operand x A^T / scale is rounded to bf16: 2^-8 of sum_r |a2 b2|, once.
"""
import pytest
import torch
import torch.nn as nn

pytestmark = pytest.mark.gpu
DEV = "cuda"
VALUES = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6], dtype=torch.float64)


def _rand(seed, *shape, dtype=torch.bfloat16, scale=1.0):
    return (torch.randn(*shape, generator=torch.Generator().manual_seed(seed)) * scale).to(dtype)


def _ref(x):
    """(codes [M,K], e4m3 block scales as f64 [M,K/16], row scales f64 [M,1]) in 64 bits."""
    M, K = x.shape
    v = x.double().view(M, -1, 16)
    top = v.abs().amax(2)
    row = torch.tensor([[2.0 ** -100 if a == 0 else max(2.0 ** -100, _ceil_pow2(a / 2688))] for a in top.amax(1).tolist()], dtype=torch.float64)
    blocks = (top / (6 * row)).float().to(torch.float8_e4m3fn).double()
    q = (v / (blocks * row).unsqueeze(2)).abs()
    q = torch.where((blocks > 0).unsqueeze(2), q, torch.zeros_like(q)).clamp(max=6.0)
    step = torch.where(q < 2, 0.5, torch.where(q < 4, 1.0, 2.0)).double()
    code = torch.searchsorted(VALUES, torch.round(q / step) * step)
    return (code + 8 * (v < 0)).view(M, K), blocks, row


def _ceil_pow2(a):
    import math

    m, e = math.frexp(a)
    return 2.0 ** (e - 1 if m == 0.5 else e)


def _codes(x4):
    return torch.stack([x4 & 15, x4 >> 4], 2).view(x4.shape[0], -1).long()


def _rows(blocks, M, nb):
    t = blocks.view(torch.uint8).permute(0, 3, 2, 1, 4)
    return t.reshape(t.shape[0] * 128, -1)[:M, :nb].contiguous().view(torch.float8_e4m3fn).double()


def _values(code, blocks, row):
    v = VALUES[code & 7] * (1 - 2 * (code >> 3)).double()
    return (v.view(*blocks.shape, 16) * blocks.unsqueeze(2)).view(code.shape) * row


@pytest.mark.parametrize("M,K", [(1, 32), (3, 64), (33, 96), (128, 160), (129, 320), (300, 5120), (2, 16384), (5, 16416), (3, 40000)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_rounding_bits(M, K, dtype):
    from minimaxh3_b200.kernels.fp4_linear import dequantize_fp4, quantize_fp4

    x = _rand(1, M, K, dtype=torch.float32)
    x *= torch.where(torch.rand(K, generator=torch.Generator().manual_seed(2)) < 0.01, 8.0, 1.0)
    x[:, :16] *= 1e-4          # block scales in e4m3's subnormals, and below
    if K >= 64:
        x[:, 32:48] *= 1e-7
    x = x.to(dtype)
    x4, blocks, scale = quantize_fp4(x.to(DEV))
    code, b, row = _ref(x)
    assert torch.equal(scale.cpu().double(), row)
    got_b = _rows(blocks.cpu(), M, K // 16)
    assert torch.equal(got_b, b)
    got = _codes(x4.cpu())
    assert torch.equal(got & 7, code & 7)
    assert torch.equal((got >> 3)[(code & 7) > 0], (code >> 3)[(code & 7) > 0])
    # scales that stand for no element are zero
    t = blocks.cpu().view(torch.uint8).permute(0, 3, 2, 1, 4)
    t = t.reshape(t.shape[0] * 128, -1)
    assert int(t[M:].sum()) == 0 and int(t[:, K // 16:].sum()) == 0
    ref = _values(code, b, row)
    assert torch.equal(dequantize_fp4(x4, blocks, scale).cpu().double(), ref)
    assert torch.equal(dequantize_fp4(x4, blocks, scale, torch.float32).cpu().double(), ref)


def test_rounding_borders_and_extremes():
    """Every border between two codes (ties to even), rows of zeros, the range's ends, infinities and NaN."""
    from minimaxh3_b200.kernels.fp4_linear import dequantize_fp4, quantize_fp4

    rows = []
    for s in (448.0, 416.0, 2.0 ** -6, 3 * 2.0 ** -9, 1.0, 13.0):
        t = torch.tensor([6, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, -0.25, -0.75, -1.25, -1.75, -2.5, -3.5, -5.0, 0.0]) * s
        rows.append(torch.cat([t, torch.full((16,), 2688.0)]))
    rows += [torch.zeros(32), torch.full((32,), 2.0 ** -126), torch.full((32,), 3.0e38), torch.full((32,), 2.0 ** -113)]
    x = torch.stack(rows)
    for dtype in (torch.float32, torch.bfloat16):
        y = x.to(dtype)
        x4, blocks, scale = quantize_fp4(y.to(DEV))
        code, b, row = _ref(y)
        assert torch.equal(scale.cpu().double(), row) and torch.equal(_rows(blocks.cpu(), len(rows), 2), b)
        assert torch.equal(_codes(x4.cpu()) & 7, code & 7)
    bad = _rand(3, 6, 64)
    bad[1, 3], bad[3, 40], bad[4, 0] = float("inf"), float("nan"), -float("inf")
    v = dequantize_fp4(*quantize_fp4(bad.to(DEV))).cpu()
    good = [0, 2, 5]
    assert bool(v[[1, 3, 4]].isnan().all())
    assert torch.equal(v[good], dequantize_fp4(*quantize_fp4(bad[good].to(DEV))).cpu())


def test_rounding_strides_and_large_offsets():
    from minimaxh3_b200.kernels.fp4_linear import quantize_fp4

    w = _rand(4, 70, 200).to(DEV)
    for view in (w[:, 8:168], w[:, 3:163], w[::2, :192], _rand(5, 96, 70).to(DEV).t()):
        for a, b in zip(quantize_fp4(view), quantize_fp4(view.contiguous())):
            assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))
    far = 2 ** 30 + 64
    buf = torch.zeros(2 * far + 64, dtype=torch.bfloat16, device=DEV)
    x = buf.as_strided((3, 64), (far, 1))
    x.copy_(_rand(6, 3, 64))
    for a, b in zip(quantize_fp4(x), quantize_fp4(x.contiguous())):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))
    assert quantize_fp4(torch.empty(0, 64, device=DEV))[0].shape == (0, 32)


def _pair(M, N, K, seed=10):
    from minimaxh3_b200.kernels.fp4_linear import quantize_fp4

    x, w = _rand(seed, M, K), _rand(seed + 1, N, K, scale=0.02)
    x[:, ::37] *= 8
    a, b = quantize_fp4(x.to(DEV)), quantize_fp4(w.to(DEV))
    av, bv = _values(*_ref(x)).to(DEV), _values(*_ref(w)).to(DEV)
    return a, b, av, bv


def _check(got, ref, mag, K, extra=0.0):
    err = (K / 64 + 8) * 2.0 ** -22 * mag + extra
    d = (got.double() - ref).abs()
    tol = 2.0 ** -8 * (ref.abs() + err) + err
    assert bool((d <= tol).all()), (float((d - tol).max()), float(d.max()))


@pytest.mark.parametrize("M", [1, 2, 8, 9, 16, 17, 32, 33, 128, 129, 256, 300, 700])
@pytest.mark.parametrize("N,K", [(8, 32), (264, 96), (520, 640), (1000, 4128)])
def test_product(M, N, K):
    from minimaxh3_b200.kernels.fp4_linear import fp4_matmul

    a, b, av, bv = _pair(M, N, K)
    bias = _rand(12, N).to(DEV)
    ref, mag = av @ bv.t(), av.abs() @ bv.abs().t()
    _check(fp4_matmul(a, b), ref, mag, K)
    _check(fp4_matmul(a, b, bias), ref + bias.double(), mag + bias.double().abs(), K)


@pytest.mark.parametrize("M,N,K", [(4097, 1544, 1280), (1, 5120, 13824), (2500, 2568, 5120), (20000, 264, 64)])
def test_product_of_many_tiles(M, N, K):
    """Several tiles per CTA pair: both accumulators, the shared columns and the scale buffers in turn."""
    from minimaxh3_b200.kernels.fp4_linear import fp4_matmul

    a, b, av, bv = _pair(M, N, K)
    _check(fp4_matmul(a, b), av @ bv.t(), av.abs() @ bv.abs().t(), K)
    assert torch.equal(fp4_matmul(a, b), fp4_matmul(a, b))


@pytest.mark.parametrize("M", [3, 32, 40, 600])
@pytest.mark.parametrize("ranks", [(16,), (32, 8), (200,)])
def test_linear_with_adapters(M, ranks):
    from minimaxh3_b200.kernels.fp4_linear import FP4Linear

    K, N = 320, 264
    lin = nn.Linear(K, N).to(torch.bfloat16)
    with torch.no_grad():
        lin.weight.copy_(_rand(20, N, K, scale=0.05))
        lin.bias.copy_(_rand(21, N, scale=0.1))
    w, bias = lin.weight.detach().clone(), lin.bias.detach().clone()
    mod = FP4Linear.from_linear(lin.to(DEV))
    assert lin.weight is None
    x = _rand(22, M, K)
    ad = [(_rand(30 + i, r, K, scale=0.1), _rand(40 + i, N, r, scale=0.1), 0.5 ** i) for i, r in enumerate(ranks)]
    mod.adapters = [(A.to(DEV), B.to(DEV), s) for A, B, s in ad]
    got = mod(x.view(1, M, K).to(DEV))
    assert got.shape == (1, M, N) and got.dtype == torch.bfloat16
    xq, wq = _values(*_ref(x)), _values(*_ref(w))
    ref = xq @ wq.t() + bias.double()
    mag = xq.abs() @ wq.abs().t() + bias.double().abs()
    extra = torch.zeros_like(ref)
    for A, B, s in ad:
        low = x.double() @ A.double().t()
        ref = ref + low @ B.double().t() * s
        m = (x.double().abs() @ A.double().abs().t()) @ B.double().abs().t() * s
        extra += 2.0 ** -8 * (low.abs() @ B.double().abs().t() * s) + (K + 200) * 2.0 ** -23 * m
    _check(got[0].cpu(), ref, mag, K, extra)
    mod.adapters = []
    _check(mod(x.to(DEV)).cpu(), xq @ wq.t() + bias.double(), mag, K)


def test_linear_refuses_gradients():
    from minimaxh3_b200.kernels.fp4_linear import fp4_linear, quantize_fp4

    w = quantize_fp4(_rand(56, 64, 96).to(DEV))
    x = _rand(57, 5, 96).to(DEV).requires_grad_(True)
    A, B = _rand(58, 16, 96).to(DEV), _rand(59, 64, 16).to(DEV).requires_grad_(True)
    for out in (fp4_linear(x, *w), fp4_linear(x.detach(), *w, adapters=[(A, B, 1.0)])):
        with pytest.raises(RuntimeError, match="no gradient"):
            out.float().sum().backward()
    with torch.no_grad():
        assert not fp4_linear(x, *w).requires_grad
    y = fp4_linear(x, *w)
    y += 1  # the result is not a view that must not be written
    assert torch.equal(y, fp4_linear(x, *w) + 1)
    bias = _rand(60, 64).to(DEV).requires_grad_(True)
    assert fp4_linear(x.detach(), *w, bias=bias).requires_grad
    f = torch.compile(lambda t: fp4_linear(t, *w), backend="aot_eager")
    assert torch.equal(f(x), fp4_linear(x, *w)) and torch.equal(f(x.detach()), fp4_linear(x, *w))


def test_linear_types_empty_and_nan_rows():
    from minimaxh3_b200.kernels.fp4_linear import fp4_linear, quantize_fp4

    w = quantize_fp4(_rand(50, 64, 96).to(DEV))
    for M in (5, 50):
        x = _rand(51, M, 96)
        ref = fp4_linear(x.to(DEV), *w)
        assert torch.equal(fp4_linear(x.float().to(DEV), *w), ref)
        assert torch.equal(fp4_linear(x.double().to(DEV), *w), ref)
        bad = x.clone()
        bad[2, 7] = float("nan")
        got = fp4_linear(bad.to(DEV), *w)
        keep = [i for i in range(M) if i != 2]
        assert bool(got[2].isnan().all()) and torch.equal(got[keep], ref[keep])
    A, B = _rand(52, 16, 96).to(DEV), _rand(53, 64, 16).to(DEV)
    for rest in ((), ((A, B, 2.0),)):
        assert fp4_linear(torch.empty(0, 96, device=DEV), *w, adapters=rest).shape == (0, 64)


def test_linear_of_few_rows_strides_and_outputs():
    """The one-launch form (one and two rows) against the two steps it stands for, on rows that vectors fit or not."""
    from minimaxh3_b200 import ops
    from minimaxh3_b200.kernels.fp4_linear import fp4_linear, fp4_matmul, quantize_fp4

    for K, N in ((32, 8), (96, 40), (5120, 264), (40000, 24), (200000, 8)):
        w = quantize_fp4(_rand(54, N, K, scale=0.05).to(DEV))
        for dtype in (torch.bfloat16, torch.float32):
            wide = _rand(55, 3, K + 9, dtype=dtype).to(DEV)
            for x in (wide[:1, 1:K + 1], wide[:2, 8:K + 8], wide[1:, 1:K + 1], wide[:3, :K]):
                got = fp4_linear(x, *w)
                assert torch.equal(got, fp4_matmul(quantize_fp4(x), w))
    for M in (2, 12, 300):  # a strided output, its other elements left as they were
        a, b, av, bv = _pair(M, 264, 96)
        out = torch.full((M, 280), 7.0, dtype=torch.bfloat16, device=DEV)
        ops.fp4_gemm(a, b, out=out[:, :264])
        assert torch.equal(out[:, :264], fp4_matmul(a, b)) and bool((out[:, 264:] == 7).all())


def test_output_offsets_past_32_bits():
    from minimaxh3_b200.kernels.fp4_linear import fp4_matmul, quantize_fp4

    M, N, K = 263000, 8192, 32
    a, b = quantize_fp4(_rand(52, M, K).to(DEV)), quantize_fp4(_rand(53, N, K).to(DEV))
    out = fp4_matmul(a, b)
    lo = 128 * ((M - 600) // 128)
    tail = (a[0][lo:].clone(), a[1][lo // 128:].clone(), a[2][lo:].clone())
    assert torch.equal(out[lo:], fp4_matmul(tail, b))


def test_streams_graphs_and_compile():
    from minimaxh3_b200.kernels.fp4_linear import fp4_linear, quantize_fp4

    w = quantize_fp4(_rand(60, 520, 256).to(DEV))
    for M in (4, 400):
        x, x2 = _rand(61, M, 256).to(DEV), _rand(62, M, 256).to(DEV)
        ref, ref2 = fp4_linear(x, *w), fp4_linear(x2, *w)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            got = fp4_linear(x, *w)
        here = fp4_linear(x2, *w)  # two calls at once
        torch.cuda.current_stream().wait_stream(side)
        assert torch.equal(got, ref) and torch.equal(here, ref2)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            cap = fp4_linear(x, *w)
        x.copy_(x2)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(cap, ref2)
        f = torch.compile(lambda t: fp4_linear(t, *w), fullgraph=True, backend="aot_eager")
        assert torch.equal(f(x2), ref2)


def test_converted_block_and_lora_registry():
    from minimaxh3_b200.kernels.fp4_linear import FP4Linear, convert_transformer_to_fp4
    from minimaxh3_b200.kernels.lora import attach_lora_registry

    class Block(nn.Module):
        def __init__(self):
            super().__init__()
            self.up, self.down, self.odd = nn.Linear(64, 128), nn.Linear(128, 64), nn.Linear(48, 64)

        def forward(self, x):
            return x + self.down(torch.relu(self.up(x)))

    net = nn.Module()
    net.blocks = nn.ModuleList(Block().to(torch.bfloat16) for _ in range(4))
    net.to(DEV)
    assert convert_transformer_to_fp4(net, "", 1) == 4
    assert isinstance(net.blocks[1].up, FP4Linear) and isinstance(net.blocks[0].up, nn.Linear) and isinstance(net.blocks[1].odd, nn.Linear)
    assert isinstance(attach_lora_registry(net)["blocks.1.up"], FP4Linear)
    x = _rand(70, 2, 37, 64).to(DEV)
    for b in net.blocks:
        x = b(x)
    assert x.shape == (2, 37, 64) and bool(x.isfinite().all())
    other = FP4Linear(64, 128)
    for n in ("w4", "w_blocks", "w_scale", "bias"):
        other.register_buffer(n, torch.empty_like(getattr(net.blocks[1].up, n)))
    other.load_state_dict(net.blocks[1].up.state_dict())
    assert torch.equal(other(x), net.blocks[1].up(x))


def test_wait_timeout_sets_error_and_context_survives():
    """A load warp that waits 1 ms on a barrier nothing arrives on: an error code, a clean return, and
    the same bits from the next launch."""
    from minimaxh3_b200 import _lib, ops

    a, b, _, _ = _pair(4096, 2568, 1280)
    err = torch.zeros(1, dtype=torch.int32, device=DEV)
    good = ops.fp4_gemm(a, b, err=err)
    torch.cuda.synchronize()
    assert int(err.item()) == 0
    ops.fp4_gemm(a, b, err=err, timeout_ns=1_000_000, test_flags=_lib.MH3_TEST_STALL_PRODUCER)
    torch.cuda.synchronize()
    assert int(err.item()) == _lib.MH3_DEVERR_WAIT_TIMEOUT
    err.zero_()
    again = ops.fp4_gemm(a, b, err=err)
    torch.cuda.synchronize()
    assert int(err.item()) == 0 and torch.equal(again, good)


def test_every_tensor_that_asks_for_a_gradient_is_refused_one():
    """Scales and biases that ask for a gradient: the values are the same, asking raises (none is cut off)."""
    from minimaxh3_b200.kernels.fp4_linear import dequantize_fp4, fp4_linear, fp4_matmul, quantize_fp4

    x, bias = _rand(80, 5, 64).to(DEV), _rand(81, 16).to(DEV)
    a, w = quantize_fp4(x), quantize_fp4(_rand(82, 16, 64).to(DEV))
    asks = lambda t: t.clone().requires_grad_(True)  # noqa: E731
    for f in (lambda s: fp4_linear(x, *w[:2], s), lambda s: fp4_matmul(a, (*w[:2], s)), lambda s: fp4_matmul((w[0], w[1], s), w),
              lambda s: dequantize_fp4(*w[:2], s)):
        out = f(asks(w[2]))
        assert torch.equal(out, f(w[2]))
        with pytest.raises(RuntimeError, match="no gradient"):
            out.sum().backward()
        with torch.no_grad():
            assert not f(asks(w[2])).requires_grad
    with pytest.raises(RuntimeError, match="no gradient"):
        fp4_matmul(a, w, asks(bias)).sum().backward()


def test_an_adapter_edited_unseen_is_used():
    """Through ``.data`` and by a replayed graph, neither of which counts a tensor's version."""
    from minimaxh3_b200.kernels.fp4_linear import fp4_linear, quantize_fp4

    x, w = _rand(90, 20, 64).to(DEV), quantize_fp4(_rand(91, 32, 64).to(DEV))
    A, B, B2 = _rand(92, 16, 64).to(DEV), _rand(93, 32, 16).to(DEV), _rand(94, 32, 16).to(DEV)
    first, want = fp4_linear(x, *w, adapters=[(A, B, 0.5)]), fp4_linear(x, *w, adapters=[(A, B2, 0.5)])
    keep = B.clone()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        B.copy_(B2)
        cap = fp4_linear(x, *w, adapters=[(A, B, 0.5)])
    assert torch.equal(fp4_linear(x, *w, adapters=[(A, B, 0.5)]), first)
    graph.replay()
    assert torch.equal(cap, want) and torch.equal(fp4_linear(x, *w, adapters=[(A, B, 0.5)]), want)
    B.data.copy_(keep)
    assert torch.equal(fp4_linear(x, *w, adapters=[(A, B, 0.5)]), first)


@pytest.mark.parametrize("M", [1, 3, 40, 300])
def test_products_of_rows_at_the_ends_of_the_range(M):
    """A power of two on x's rows or on the weight goes through to the result exactly, as long as that is in range:
    no product of a sum with one scale alone may overflow or vanish."""
    from minimaxh3_b200.kernels.fp4_linear import fp4_linear, quantize_fp4

    K, N = 128, 64
    x, w = _rand(100, M, K).to(DEV), _rand(101, N, K, scale=0.05).to(DEV)
    A, B = _rand(102, 16, K, scale=0.1).to(DEV), _rand(103, N, 16, scale=0.1).to(DEV)
    ref, low = fp4_linear(x, *quantize_fp4(w)), fp4_linear(x, *quantize_fp4(w), adapters=[(A, B, 0.5)])
    for px, pw in ((0, 0), (118, 0), (110, -40), (-60, 70), (-80, 100), (20, 95), (100, 15)):
        fx, fw = 2.0 ** px, 2.0 ** pw
        want = (ref.double() * fx * fw).to(torch.bfloat16)
        assert bool(want.isfinite().all())
        assert torch.equal(fp4_linear(x * fx, *quantize_fp4(w * fw)), want), (px, pw)
        if M > 2 and px + pw < 110:
            want = (low.double() * fx * fw).to(torch.bfloat16)
            assert torch.equal(fp4_linear(x * fx, *quantize_fp4(w * fw), adapters=[(A, B * fw, 0.5)]), want), (px, pw)


def test_values_at_the_end_of_the_range():
    """Within a twentieth of the largest number a block may round up past it: infinite values, as their definition
    in 64 bits says; the product of such a row is finite where the result is."""
    from minimaxh3_b200.kernels.fp4_linear import dequantize_fp4, fp4_linear, quantize_fp4

    top = torch.finfo(torch.bfloat16).max
    x = torch.full((2, 64), top, dtype=torch.bfloat16)
    x[1] *= 0.95
    ref = _values(*_ref(x))
    assert float(ref[0, 0]) > torch.finfo(torch.float32).max > float(ref[1, 0])
    q = quantize_fp4(x.to(DEV))
    for dt in (torch.bfloat16, torch.float32):
        assert torch.equal(dequantize_fp4(*q, dtype=dt).cpu(), ref.to(dt))
    w = (torch.ones(8, 64) * 2.0 ** -20).to(torch.bfloat16)
    want = ref @ _values(*_ref(w)).t()  # 64 equal products of few bits: exact in f32
    assert torch.equal(fp4_linear(x.to(DEV), *quantize_fp4(w.to(DEV))).cpu(), want.to(torch.bfloat16))
