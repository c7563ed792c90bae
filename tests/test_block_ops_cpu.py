"""Refusals, layouts and conversions of the rotary, norm and 4-bit operators that need no GPU."""
import ctypes
import os
import shutil
import subprocess

import pytest
import torch
import torch.nn as nn

from conftest import ROOT
from minimaxh3_b200 import _lib, ops
from minimaxh3_b200.kernels import fp4_linear as F4
from minimaxh3_b200.kernels.block_norm import gated_residual_norm, norm_modulate
from minimaxh3_b200.kernels.rotary import rotary_axes


def _q(*shape, dtype=torch.bfloat16):
    return torch.zeros(*shape, dtype=dtype)


POS = torch.zeros(5, 2, dtype=torch.int32)


@pytest.mark.parametrize("args,why", [
    ((_q(2, 5, 32), None, POS, (16, 16)), "positions"),                            # packed: 2 tokens
    ((_q(5, 32), None, POS, (16, 16)), "q must be"),
    ((_q(1, 2, 5, 32, dtype=torch.float64), None, POS, (16, 16)), "dtype"),
    ((_q(1, 2, 5, 32), _q(1, 2, 6, 32), POS, (16, 16)), "same tokens"),
    ((_q(2, 2, 5, 32), _q(1, 2, 5, 32), POS, (16, 16)), "same tokens"),
    ((_q(1, 2, 5, 32), _q(1, 2, 5, 16), POS, (16, 16)), "agree"),
    ((_q(1, 2, 5, 32), _q(1, 2, 5, 32, dtype=torch.float16), POS, (16, 16)), "agree"),
    ((_q(1, 2, 5, 32), None, POS, (15, 17)), "even"),
    ((_q(1, 2, 5, 32), None, POS, (16, 18)), "head dim"),
    ((_q(1, 2, 5, 32), None, POS, (0, 0)), "positive"),
    ((_q(1, 2, 5, 32), None, POS, (2,) * 5), "1 to 4"),
    ((_q(1, 2, 5, 512), None, POS, (16, 16)), "256"),
    ((_q(1, 2, 5, 32), None, POS, (16, 16), (1e4,)), "theta"),
    ((_q(1, 2, 5, 32), None, POS, (16, 16), -1.0), "theta"),
    ((_q(1, 2, 5, 32), None, POS, (16, 16), float("nan")), "theta"),
    ((_q(1, 2, 5, 32), None, POS.double(), (16, 16)), "positions"),
    ((_q(1, 2, 5, 32), None, POS[:4], (16, 16)), "positions"),
    ((_q(1, 2, 5, 32), None, POS, (16, 8, 8)), "positions"),
    ((_q(3, 2, 5, 32), None, POS.expand(2, 5, 2), (16, 16)), "positions"),
    ((_q(1, 2, 5, 32), None, POS, (16, 16)), "CUDA"),
])
def test_rotary_refusals(args, why):
    with pytest.raises(ValueError, match=why):
        rotary_axes(*args)


def test_rotary_refuses_positions_that_ask_for_a_gradient():
    q, pos = _q(1, 2, 5, 32), POS.float().requires_grad_(True)
    for t in (q, q.clone().requires_grad_(True)):
        with pytest.raises(ValueError, match="no gradient of the positions"):
            rotary_axes(t, None, pos, (16, 16))
    with torch.no_grad(), pytest.raises(ValueError, match="CUDA"):  # nothing is asked for
        rotary_axes(q, None, pos, (16, 16))


X = _q(2, 5, 16)


@pytest.mark.parametrize("args,kw,why", [
    ((_q(16),), {}, "x must be"),
    ((X.double(),), {}, "x must be"),
    ((X, _q(3, 16)), {}, "scale must be"),
    ((X, _q(2, 4, 16)), {}, "scale must be"),
    ((X, _q(2, 15)), {}, "scale must be"),
    ((X, _q(2, 16).double()), {}, "scale must be"),
    ((X,), dict(norm="batch"), "norm must be"),
    ((X,), dict(norm="none"), "norm must be"),
    ((X,), dict(weight=_q(2, 16)), "weight must be"),
    ((X,), dict(eps=-1.0), "eps"),
    ((X,), dict(eps=float("nan")), "eps"),
    ((X,), dict(cu_seqlens=torch.zeros(3, dtype=torch.int32)), "packed"),
    ((X[0],), dict(cu_seqlens=torch.zeros(3, dtype=torch.int64)), "cu_seqlens"),
    ((X[0],), dict(cu_seqlens=torch.zeros(1, dtype=torch.int32)), "cu_seqlens"),
    ((X[0], _q(3, 16)), dict(cu_seqlens=torch.zeros(3, dtype=torch.int32)), "scale must be"),
    ((X[0], _q(2, 16), _q(5, 16)), dict(cu_seqlens=torch.zeros(3, dtype=torch.int32)), "per sequence"),
    ((_q(2, 8200),), {}, "8192"),
    ((_q(2, 0),), {}, "8192"),
    ((X,), {}, "CUDA"),
])
def test_norm_refusals(args, kw, why):
    with pytest.raises(ValueError, match=why):
        norm_modulate(*args, **kw)


@pytest.mark.parametrize("args,kw,why", [
    ((X, X[:1]), {}, "y must have"),
    ((X, X.float()), {}, "y must have"),
    ((X, X, _q(5, 16)), {}, "gate must be"),
    ((X, X), dict(y_weight=_q(16)), "y_weight needs"),
    ((X, X), dict(norm="none", weight=_q(16)), "need a norm"),
    ((X, X), dict(y_norm="batch"), "y_norm must be"),
    ((X, X), {}, "CUDA"),
])
def test_gated_refusals(args, kw, why):
    with pytest.raises(ValueError, match=why):
        gated_residual_norm(*args, **kw)


def _w4(M=16, K=64):
    return (torch.zeros(M, K // 2, dtype=torch.uint8), torch.zeros(1, (K + 63) // 64, 32, 4, 4).to(torch.float8_e4m3fn), torch.ones(M, 1))


def test_fp4_refusals():
    v, b, s = _w4()
    for bad, why in ((_q(4), "2D"), (_q(4, 48), "multiple of 32"), (_q(4, 0), "multiple of 32"), (_q(4, 64).double(), "dtype"), (_q(4, 64), "CUDA")):
        with pytest.raises(ValueError, match=why):
            F4.quantize_fp4(bad)
    for bad, why in (((v.int(), b, s), "uint8"), ((v, b.float(), s), "e4m3"), ((v, b, s.half()), "float32"), ((v[:, :24], b, s), "multiple of 32"),
                     ((v, b[:, :0], s), "shape"), ((v, b, s[:3]), "row scale"), ((v.t().contiguous().t(), b, s), "contiguous")):
        with pytest.raises(ValueError, match=why):
            F4.dequantize_fp4(*bad)
        with pytest.raises(ValueError, match=why):
            F4.fp4_matmul(bad, (v, b, s))
        with pytest.raises(ValueError, match=why):
            F4.fp4_linear(_q(2, 64), *bad)
    with pytest.raises(ValueError, match="float32"):
        F4.dequantize_fp4(v, b, s, torch.float16)
    with pytest.raises(ValueError, match="aligned"):
        F4.dequantize_fp4(torch.zeros(16 * 32 + 1, dtype=torch.uint8)[1:].view(16, 32), b, s)
    with pytest.raises(ValueError, match=r"b is \[N,K\]"):
        F4.fp4_matmul((v, b, s), _w4(16, 32))
    with pytest.raises(ValueError, match="multiple of 8"):
        F4.fp4_matmul((v, b, s), _w4(12))
    with pytest.raises(ValueError, match="multiple of 8"):
        F4.fp4_linear(_q(2, 64), *_w4(12))
    for x in (_q(2, 32), _q(2, 64).int()):
        with pytest.raises(ValueError, match="float tensor"):
            F4.fp4_linear(x, v, b, s)
    with pytest.raises(ValueError, match="CUDA"):
        F4.fp4_linear(_q(2, 64), v, b, s)
    with pytest.raises(ValueError, match="multiple of 32"):
        F4.FP4Linear.from_linear(nn.Linear(48, 64))


def test_c_entries_refuse_without_a_gpu():
    lib = _lib.load()
    inval, large = _lib.MH3_ERR_INVALID, _lib.MH3_ERR_TOO_LARGE
    assert lib.mh3_rotary(None, None) == lib.mh3_block_norm_fwd(None, None) == lib.mh3_block_norm_bwd(None, None) == inval
    assert lib.mh3_fp4_gemm(None, None) == inval

    def rot(**kw):
        a = _lib.RotaryArgs(batch=1, seqlen=4, heads_q=1, head_dim=32, n_axes=1, q=16, q_out=16, positions=16)
        a.axes_dim[0], a.theta[0] = 32, 1e4
        for n, v in kw.items():
            if n in ("axes_dim", "theta"):
                getattr(a, n)[0] = v
            else:
                setattr(a, n, v)
        return lib.mh3_rotary(a, None)

    for kw in (dict(axes_dim=31), dict(axes_dim=34), dict(axes_dim=-2), dict(axes_dim=0), dict(theta=0.0), dict(theta=float("inf")), dict(dtype=2),
               dict(pos_kind=3), dict(n_axes=0), dict(n_axes=5), dict(q=None), dict(positions=None), dict(seqlen=-1), dict(heads_k=2)):
        assert rot(**kw) == inval, kw
    assert rot(head_dim=300) == large
    assert rot(seqlen=0) == 0

    def norm(bwd=False, **kw):
        a = _lib.BlockNormArgs(rows=4, group_rows=4, channels=64, groups=1, norm=1, x=16, x_stride=64, h=16)
        for n, v in kw.items():
            setattr(a, n, v)
        return (lib.mh3_block_norm_bwd if bwd else lib.mh3_block_norm_fwd)(a, None)

    for kw in (dict(rows=5), dict(channels=0), dict(groups=0), dict(dtype=2), dict(norm=0), dict(norm=3), dict(y_norm=1), dict(y_norm=-1), dict(x=None),
               dict(h=None), dict(r=16), dict(stats=8), dict(bwd=True), dict(bwd=True, dh=16, stats=16), dict(bwd=True, stats=16, workspace=16)):
        assert norm(**kw) == inval, kw
    assert norm(channels=8193) == large
    assert norm(rows=0, group_rows=0) == 0
    assert lib.mh3_block_norm_workspace_bytes(10, 8193, 1) == 0
    assert lib.mh3_block_norm_workspace_bytes(10, 64, 3) == (10 + 6) * 3 * 64 * 4

    assert lib.mh3_fp4_block_bytes(129, 96) == 2 * 2 * 512 and lib.mh3_fp4_block_bytes(0, 96) == 0
    assert lib.mh3_quantize_fp4(16, 64, 0, 4, 48, 16, 16, 16, None) == inval
    assert lib.mh3_quantize_fp4(16, 64, 2, 4, 64, 16, 16, 16, None) == inval
    assert lib.mh3_quantize_fp4(None, 64, 0, 4, 64, 16, 16, 16, None) == inval
    assert lib.mh3_quantize_fp4(16, 64, 0, 4, 64, 8, 16, 16, None) == inval
    assert lib.mh3_quantize_fp4(16, 64, 0, 1 << 40, 64, 16, 16, 16, None) == large
    assert lib.mh3_quantize_fp4(None, 64, 0, 0, 64, None, None, None, None) == 0
    assert lib.mh3_dequantize_fp4(16, 16, 16, 4, 64, 1, 16, None) == inval
    assert lib.mh3_dequantize_fp4(16, 16, 16, 4, 64, 0, 8, None) == inval

    def gemm(**kw):
        a = _lib.Fp4GemmArgs(M=64, N=64, K=64, a=16, a_blocks=16, a_scale=16, b=16, b_blocks=16, b_scale=16, out=16, ldo=64)
        for n, v in kw.items():
            setattr(a, n, v)
        return lib.mh3_fp4_gemm(a, None)

    for kw in (dict(K=48), dict(N=60), dict(ldo=56), dict(ldo=66), dict(a=None), dict(b_scale=None), dict(a=8), dict(R=8), dict(R=-1),
               dict(R=8, a2=16, b2=16, lda2=8, ldb2=4), dict(R=12, a2=16, b2=16, lda2=16, ldb2=16)):
        assert gemm(**kw) == inval, kw
    assert gemm(M=1 << 33) == large
    assert gemm(M=0) == 0


def test_struct_offsets_match_gcc(tmp_path):
    cc = shutil.which("gcc") or shutil.which("cc")
    if cc is None:
        pytest.skip("no C compiler")
    structs = (("mh3_rotary_args", _lib.RotaryArgs), ("mh3_norm_mod", _lib.NormMod), ("mh3_block_norm_args", _lib.BlockNormArgs),
               ("mh3_fp4_gemm_args", _lib.Fp4GemmArgs))
    lines = ['#include <stdio.h>', '#include <stddef.h>', '#include "mh3_b200.h"', "int main(void){"]
    for cname, cls in structs:
        lines.append(f'printf("%zu\\n", sizeof({cname}));')
        lines += [f'printf("%zu\\n", offsetof({cname}, {f[0]}));' for f in cls._fields_]
    src = tmp_path / "probe.c"
    src.write_text("\n".join(lines + ["return 0;}"]))
    subprocess.run([cc, "-I", os.path.join(ROOT, "include"), str(src), "-o", str(tmp_path / "probe")], check=True)
    got = [int(v) for v in subprocess.run([str(tmp_path / "probe")], capture_output=True, text=True, check=True).stdout.split()]
    want = [v for _, cls in structs for v in [ctypes.sizeof(cls)] + [getattr(cls, f[0]).offset for f in cls._fields_]]
    assert got == want


def test_fakes_give_the_outputs_shapes():
    """The registered fakes, as torch.compile sees them."""
    from torch._subclasses.fake_tensor import FakeTensorMode

    with FakeTensorMode():
        q, k = torch.empty(1, 4, 9, 32), torch.empty(1, 2, 9, 32)
        a, b = torch.ops.mh3.rotary_axes(q, k, torch.empty(9, 2, dtype=torch.int32), [16, 16], [1e4, 1e4], True, False)
        assert a.shape == q.shape and b.shape == k.shape
        x = torch.empty(2, 5, 16)
        r, h, st = torch.ops.mh3.block_norm(x, x, None, None, None, None, None, None, None, 1, 0, 1e-6, 1.0, False, True)
        assert r.shape == h.shape == x.shape and st.shape == (10, 4)
        g = torch.ops.mh3.block_norm_backward(r, h, x, x, None, None, None, None, None, None, None, st, 1, 0, 1e-6, 1.0, False,
                                              [True, True] + [False] * 6)
        assert g[0].shape == g[1].shape == x.shape
        o = torch.ops.mh3.fp4_linear(torch.empty(3, 64), torch.empty(16, 32, dtype=torch.uint8), torch.empty(1), torch.empty(16, 1), None, [], [], [])
        assert o.shape == (3, 16) and o.dtype == torch.bfloat16


def test_fp4_conversion_policy(monkeypatch):
    """Blocks at the edges, excluded names and widths that do not fit stay as they are."""
    made = []
    monkeypatch.setattr(F4.FP4Linear, "from_linear", classmethod(lambda cls, lin: made.append(lin) or cls(lin.in_features, lin.out_features)))

    class Block(nn.Module):
        def __init__(self):
            super().__init__()
            self.a, self.keep_me, self.thin, self.odd = nn.Linear(64, 32), nn.Linear(64, 32), nn.Linear(48, 32), nn.Linear(64, 24)

    net = nn.Module()
    net.blocks = nn.ModuleList(Block() for _ in range(5))
    assert F4.convert_transformer_to_fp4(net, "keep_me, other", 1) == 3 and len(made) == 3
    assert all(isinstance(net.blocks[i].a, F4.FP4Linear) for i in (1, 2, 3)) and isinstance(net.blocks[0].a, nn.Linear)
    assert all(type(getattr(b, n)) is nn.Linear for b in net.blocks for n in ("keep_me", "thin", "odd"))


def test_ops_check_is_shared():
    assert ops.check_fp4(*_w4(16, 96)[:1], torch.zeros(1, 2, 32, 4, 4).to(torch.float8_e4m3fn), torch.ones(16), "x") == (16, 96)


@pytest.mark.parametrize("ranks", [(16,), (8,), (0,), (32, 8), (5, 11, 200)])
def test_low_rank_operands_of_a_four_bit_linear(ranks):
    """The adapters side by side, in the bits of the fold that the 8-bit linear makes, anew in each call."""
    K, N = 64, 24
    g = torch.Generator().manual_seed(sum(ranks))
    w_scale = torch.exp2(torch.randint(-20, 5, (N, 1), generator=g).float())
    types = (torch.bfloat16, torch.float32, torch.float16)
    adapters = [(torch.randn(r, K, generator=g).to(types[i]), torch.randn(N, r, generator=g).to(types[i]), 0.3 ** i) for i, r in enumerate(ranks)]
    for _ in range(2):
        got, want = ops._fp4_low_rank(adapters, w_scale, K), ops._fold_lora(adapters, N, K, "cpu", col_scale=w_scale.reshape(-1))
        assert all(a.is_contiguous() and torch.equal(a, b) for a, b in zip(got, want))
        adapters[0][1].data.mul_(2)  # no version counter sees this


def test_low_rank_refusals():
    w_scale = torch.ones(24, 1)
    for A, B in (((8, 32), (24, 8)), ((8, 64), (23, 8)), ((8, 64), (24, 9)), ((8, 1), (24, 8))):
        with pytest.raises(ValueError, match="an adapter is"):
            ops._fp4_low_rank([(torch.zeros(A), torch.zeros(B), 1.0)], w_scale, 64)
