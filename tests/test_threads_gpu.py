"""Host threads that call one operator with sizes of different shared memory at once.

A kernel's limit of dynamic shared memory is shared by the host threads of a process: a thread must not
lower it between another one's setting and launch.  The C entries are called from C++ threads, which
nothing keeps apart (Python's threads mostly take turns)."""
import ctypes
import os
import subprocess

import pytest
import torch

from conftest import ROOT

pytestmark = pytest.mark.gpu
DEV = "cuda"

SOURCE = r"""
#include <atomic>
#include <functional>
#include <thread>
#include <vector>
#include "mh3_b200.h"
using Call = std::function<int()>;
static int run(const Call& a, const Call& b, int n) {
  std::atomic<int> bad{0}, ready{0};
  std::vector<std::thread> ts;
  for (int i = 0; i < 4; ++i)
    ts.emplace_back([&, i] {
      ++ready;
      while (ready < 4) std::this_thread::yield();
      for (int k = 0; k < n; ++k) bad += (i % 2 ? a : b)() != 0;
    });
  for (auto& t : ts) t.join();
  return bad;
}
extern "C" int norms(const mh3_block_norm_args* a, const mh3_block_norm_args* b, int n) {
  return run([=] { return mh3_block_norm_fwd(a, nullptr); }, [=] { return mh3_block_norm_fwd(b, nullptr); }, n);
}
extern "C" int rotations(const mh3_rotary_args* a, const mh3_rotary_args* b, int n) {
  return run([=] { return mh3_rotary(a, nullptr); }, [=] { return mh3_rotary(b, nullptr); }, n);
}
extern "C" int roundings(const void* x, int K0, int K1, void* v, void* blocks, float* scale, int n) {
  auto f = [=](int K) { return mh3_quantize_fp4(x, K, MH3_DTYPE_BF16, 4, K, v, blocks, scale, nullptr); };
  return run([=] { return f(K0); }, [=] { return f(K1); }, n);
}
extern "C" int products(const void* x, int K0, int K1, const void* w, const void* blocks, const float* scale, void* out, int n) {
  auto f = [=](int K) {
    return mh3_fp4_linear(x, K, MH3_DTYPE_BF16, 1, 16, K, w, blocks, scale, nullptr, out, 16, nullptr, nullptr);
  };
  return run([=] { return f(K0); }, [=] { return f(K1); }, n);
}
"""
N = 3000


@pytest.fixture(scope="module")
def threads(tmp_path_factory):
    from minimaxh3_b200 import _lib

    _lib.load()
    d = tmp_path_factory.mktemp("threads")
    (d / "t.cc").write_text(SOURCE)
    so, pkg = str(d / "t.so"), os.path.join(ROOT, "minimaxh3_b200")
    subprocess.run(["g++", "-std=c++17", "-O2", "-shared", "-fPIC", "-pthread", "-I" + os.path.join(ROOT, "include"), str(d / "t.cc"),
                    "-o", so, "-L" + pkg, "-l:libmh3_b200.so", "-Wl,-rpath," + pkg], check=True)
    torch.zeros(1, device=DEV)
    lib = ctypes.CDLL(so)
    torch.cuda.synchronize()
    yield lib
    torch.cuda.synchronize()


def _ptr(t):
    return ctypes.c_void_p(t.data_ptr())


@pytest.mark.parametrize("gated", [False, True])
def test_norms_of_two_widths(threads, gated):
    from minimaxh3_b200 import _lib

    keep, args = [], []
    for C in (5112, 2200):
        x, h, r = (torch.ones(8, C, dtype=torch.bfloat16, device=DEV) for _ in range(3))
        a = _lib.BlockNormArgs()
        a.rows, a.group_rows, a.channels, a.groups, a.dtype, a.norm, a.eps, a.residual_scale = 8, 8, C, 1, _lib.MH3_DTYPE_BF16, 2, 1e-6, 1.0
        a.x, a.x_stride, a.h = x.data_ptr(), C, h.data_ptr()
        if gated:
            a.y, a.y_stride, a.r = x.data_ptr(), C, r.data_ptr()
        keep += [x, h, r]
        args.append(a)
    assert threads.norms(ctypes.byref(args[0]), ctypes.byref(args[1]), N) == 0


def test_rotations_of_two_head_counts(threads):
    from minimaxh3_b200 import _lib

    pos, keep, args = torch.zeros(8, 1, dtype=torch.int32, device=DEV), [], []
    for H in (90, 50):
        q = torch.ones(8, H, 128, dtype=torch.bfloat16, device=DEV)
        a = _lib.RotaryArgs()
        a.batch, a.seqlen, a.heads_q, a.head_dim, a.dtype, a.n_axes, a.interleaved = 1, 8, H, 128, _lib.MH3_DTYPE_BF16, 1, 1
        a.axes_dim[0], a.theta[0], a.positions, a.pos_stride_s = 128, 1e4, pos.data_ptr(), 1
        out = torch.empty_like(q)
        a.q, a.q_stride_h, a.q_stride_s, a.q_out, a.qo_stride_h, a.qo_stride_s = q.data_ptr(), 128, H * 128, out.data_ptr(), 128, H * 128
        keep += [q, out]
        args.append(a)
    assert threads.rotations(ctypes.byref(args[0]), ctypes.byref(args[1]), N) == 0


def test_roundings_of_two_widths(threads):
    from minimaxh3_b200.kernels.fp4_linear import quantize_fp4

    x = torch.ones(4, 13824, dtype=torch.bfloat16, device=DEV)
    assert threads.roundings(_ptr(x), 13824, 6144, *map(_ptr, quantize_fp4(x)), N) == 0


def test_products_of_two_depths(threads):
    from minimaxh3_b200.kernels.fp4_linear import quantize_fp4

    x, out = torch.ones(1, 160000, dtype=torch.bfloat16, device=DEV), torch.empty(1, 16, dtype=torch.bfloat16, device=DEV)
    w = quantize_fp4(torch.ones(16, 160000, dtype=torch.bfloat16, device=DEV))
    assert threads.products(_ptr(x), 160000, 64000, *map(_ptr, w), _ptr(out), N // 6) == 0
