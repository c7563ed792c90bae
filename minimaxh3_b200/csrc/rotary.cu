// Rotary positions with several axes (time, height, width, ...).
//
// Channels [0, R) of a head are rotated in R/2 pairs, R = sum of the axes'
// widths d_a; pair p belongs to one axis a and is its j-th of d_a/2.  At a
// token with positions pos[a] the pair turns by
//   phi = pos[a] * theta_a^(-2j / d_a)
//   (x0, x1) -> (x0 cos phi - x1 sin phi, x0 sin phi + x1 cos phi)
// (phi -> -phi for the inverse, which is the gradient).  Channels [R, D) pass.
//
// Angles: the host computes each pair's rate in turns per position in double;
// the kernel multiplies by the position in double and drops the whole turns
// before it rounds to float, so a token at position 10^6 has the same angle
// error (2^-25 turns) as one at 1.  One sine and cosine per (token, pair) is
// computed into shared memory and used by every head of Q and K, so the two
// double operations and the sincospi are 1/80th of a vector's work at 40 heads.
//
// Bound: HBM.  Q and K are read and written once by 16-byte vectors.  A thread
// keeps the same channels for every (token, head) row it visits and steps through
// the heads by a fixed stride, so a row costs two pointer increments, and a token
// one read of its angles.  Its rows stream through its own part of a ring in shared
// memory (cp.async, no barrier); the first are on their way before the angles are computed.
#include <math.h>

#include <algorithm>

#include "mh3_b200.h"
#include "mh3_internal.h"
#include "ptx.cuh"

namespace mh3 {
namespace rotary {

constexpr int kThreads = 256;    // of the scalar kernel; the most of the streaming one is kMaxThreads
constexpr int kMaxThreads = 384;
constexpr int kMaxPairs = 128;  // head_dim <= 256
constexpr int kMaxTokens = 16;  // tokens per CTA
constexpr int kDepth = 8;       // 16-byte vectors of a thread in the ring

struct Params {
  const char *q, *k;
  char *qo, *ko;
  long long q_sb, q_sh, q_ss, k_sb, k_sh, k_ss;      // element strides
  long long qo_sb, qo_sh, qo_ss, ko_sb, ko_sh, ko_ss;
  long long tokens;  // batch * seqlen
  int S, Hq, Hk, D, R2, tile, side;
  const void* pos;
  int pos_kind;  // 0 int32, 1 int64, 2 float
  long long pos_sb, pos_ss;
  float sign;
  double rate[kMaxPairs];  // turns per unit of position
  uint8_t axis[kMaxPairs];
};

template <typename T>
__device__ __forceinline__ float to_f(T v) {
  if constexpr (std::is_same<T, float>::value) return v;
  else if constexpr (std::is_same<T, __half>::value) return __half2float(v);
  else return __bfloat162float(v);
}
template <typename T>
__device__ __forceinline__ T from_f(float v) {
  if constexpr (std::is_same<T, float>::value) return v;
  else if constexpr (std::is_same<T, __half>::value) return __float2half_rn(v);
  else return __float2bfloat16_rn(v);
}

template <typename T, int V>
struct __align__(sizeof(T) * V) Vec {
  T e[V];
};

// cos and sin of the CTA's tokens, [nt][npair] each; pairs past R/2 have the angle 0.
__device__ __forceinline__ void angles(const Params& p, float* cos_, float* sin_, long long t0, int nt, int npair) {
  for (int i = threadIdx.x; i < nt * npair; i += blockDim.x) {
    const int t = i / npair, j = i - t * npair;
    if (j >= p.R2) {
      cos_[i] = 1.0f;
      sin_[i] = 0.0f;
      continue;
    }
    const long long tok = t0 + t;
    const long long b = tok / p.S, s = tok - b * p.S;
    const long long at = b * p.pos_sb + s * p.pos_ss + p.axis[j];
    const double pos = p.pos_kind == 0   ? (double)static_cast<const int*>(p.pos)[at]
                       : p.pos_kind == 1 ? (double)static_cast<const long long*>(p.pos)[at]
                                         : (double)static_cast<const float*>(p.pos)[at];
    double turn = pos * p.rate[j];
    turn -= rint(turn);
    float sn, c;
    sincospif(2.0f * (float)turn, &sn, &c);
    cos_[i] = c;
    sin_[i] = sn * p.sign;
  }
}

// Addresses of head 0 of the CTA's tokens.
struct Token {
  const char *q, *k;
  char *qo, *ko;
};
__device__ __forceinline__ void token_table(const Params& p, Token* tab, long long t0, int nt, int es) {
  if ((int)threadIdx.x < nt) {
    const long long tok = t0 + threadIdx.x;
    const long long b = tok / p.S, s = tok - b * p.S;
    Token t;
    t.q = p.q + (b * p.q_sb + s * p.q_ss) * es;
    t.k = p.k + (b * p.k_sb + s * p.k_ss) * es;
    t.qo = p.qo + (b * p.qo_sb + s * p.qo_ss) * es;
    t.ko = p.ko + (b * p.ko_sb + s * p.ko_ss) * es;
    tab[threadIdx.x] = t;
  }
  if ((int)threadIdx.x == nt) tab[nt] = Token{};  // read, not followed, past the last token
}

template <typename T>
__device__ __forceinline__ void rotate(T& x0, T& x1, float2 a) {
  const float v0 = to_f(x0), v1 = to_f(x1);
  x0 = from_f<T>(fmaf(v1, -a.y, __fmul_rn(v0, a.x)));  // the streaming kernel's order: the same bits for every layout
  x1 = from_f<T>(fmaf(v1, a.x, __fmul_rn(v0, a.y)));
}

// A thread's way through its rows: tokens t, Q's then K's heads h, h + side, ..
// ``P``: char of the inputs or of the outputs.
template <typename P>
struct Cursor {
  P* at;
  int t, h;
  bool k;
};

// The units of a row: one 16-byte vector when INTER (pairs past R/2 pass), and when
// not the two vectors of V pairs, or V passing channels.
template <typename T, bool INTER>
__global__ void __launch_bounds__(kMaxThreads) stream_kernel(const __grid_constant__ Params p) {
  constexpr int V = 16 / sizeof(T);
  constexpr int W = INTER ? 1 : 2;       // vectors of a unit
  constexpr int D = kDepth / W;          // rows of a thread in the ring
  constexpr int NP = INTER ? V / 2 : V;  // pairs of a unit
  extern __shared__ uint4 smem[];
  uint4* ring = smem + threadIdx.x;  // [D][W][threads]
  const int nthr = blockDim.x;
  float* cos_ = reinterpret_cast<float*>(smem + kDepth * nthr);
  __shared__ Token tab[kMaxTokens + 1];
  const int npair = INTER ? p.D / 2 : p.R2;
  float* sin_ = cos_ + p.tile * npair;
  const long long t0 = (long long)blockIdx.x * p.tile;
  const int nt = (int)min((long long)p.tile, p.tokens - t0);
  const int rot_units = INTER ? p.D / V : p.R2 / V;
  const int units = INTER ? rot_units : rot_units + (p.D - 2 * p.R2) / V;
  const int side = p.side;  // rows visited side by side
  const int row0 = threadIdx.x / units, u = threadIdx.x - row0 * units;
  const bool rot = u < rot_units;
  const int c0 = rot ? u * V : 2 * p.R2 + (u - rot_units) * V;
  const bool has_q = row0 < p.Hq && row0 < side, has_k = row0 < p.Hk && row0 < side;
  // the thread's first Q and K rows, and a step of ``side`` heads, in bytes
  constexpr int ES = sizeof(T);
  const long long q0 = (row0 * p.q_sh + c0) * ES, k0 = (row0 * p.k_sh + c0) * ES;
  const long long qo0 = (row0 * p.qo_sh + c0) * ES, ko0 = (row0 * p.ko_sh + c0) * ES;
  const long long qs = side * p.q_sh * ES, ks = side * p.k_sh * ES, qos = side * p.qo_sh * ES, kos = side * p.ko_sh * ES;
  token_table(p, tab, t0, nt, ES);
  __syncthreads();
  auto enter = [&](auto& c) {  // the first row of c's token and tensor
    c.h = row0;
    if constexpr (std::is_same<std::decay_t<decltype(c)>, Cursor<const char>>::value)
      c.at = c.k ? tab[c.t].k + k0 : tab[c.t].q + q0;
    else
      c.at = c.k ? tab[c.t].ko + ko0 : tab[c.t].qo + qo0;
  };
  auto advance = [&](auto& c, long long qstep, long long kstep) {
    c.h += side;
    c.at += c.k ? kstep : qstep;
    if (c.h >= (c.k ? p.Hk : p.Hq)) {
      if (c.k || !has_k) ++c.t;
      c.k = has_q ? (has_k && !c.k) : true;
      enter(c);  // past the last token: a row of the table that is not followed
    }
  };
  const int per_q = has_q ? (p.Hq - row0 + side - 1) / side : 0, per_k = has_k ? (p.Hk - row0 + side - 1) / side : 0;
  const int n = nt * (per_q + per_k);  // the thread's rows
  Cursor<const char> in{nullptr, 0, 0, !has_q};
  Cursor<char> out{nullptr, 0, 0, !has_q};
  enter(in);
  enter(out);
  int issued = 0;
  auto issue = [&](int slot) {
    if (issued < n) {
      uint4* dst = ring + slot * W * nthr;
      asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(dst)), "l"(in.at) : "memory");
      if (!INTER && rot)
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(dst + nthr)), "l"(in.at + p.R2 * ES) : "memory");
      ++issued;
      advance(in, qs, ks);
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
#pragma unroll
  for (int j = 0; j < D - 1; ++j) issue(j);
  angles(p, cos_, sin_, t0, nt, npair);
  __syncthreads();
  float2 cs[NP / 2], sn[NP / 2];  // of the current token's pairs 2 i, 2 i + 1 of the unit
  const int whole = INTER ? max(0, min(NP, p.R2 - u * NP)) : (rot ? NP : 0);  // rotated pairs of the unit
  int slot = 0, token = -1;
  for (int i = 0; i < n; ++i) {
    issue(slot == 0 ? D - 1 : slot - 1);
    asm volatile("cp.async.wait_group %0;" ::"n"(D - 1) : "memory");
    if (out.t != token) {
      token = out.t;
      if (whole)
#pragma unroll
        for (int q = 0; q < NP / 2; ++q) {
          cs[q] = *reinterpret_cast<const float2*>(cos_ + token * npair + u * NP + 2 * q);
          sn[q] = *reinterpret_cast<const float2*>(sin_ + token * npair + u * NP + 2 * q);
        }
    }
    const uint4* src = ring + slot * W * nthr;
    Vec<T, V> x = *reinterpret_cast<const Vec<T, V>*>(src), y;
    if (!INTER && rot) y = *reinterpret_cast<const Vec<T, V>*>(src + nthr);
    if (whole) {
      const Vec<T, V> keep = x;
#pragma unroll
      for (int q = 0; q < NP / 2; ++q) {
        // pairs 2 q and 2 q + 1, in packed f32
        T &a0 = INTER ? x.e[4 * q] : x.e[2 * q], &a1 = INTER ? x.e[4 * q + 2] : x.e[2 * q + 1];
        T &b0 = INTER ? x.e[4 * q + 1] : y.e[2 * q], &b1 = INTER ? x.e[4 * q + 3] : y.e[2 * q + 1];
        const float2 a = make_float2(to_f(a0), to_f(a1)), b = make_float2(to_f(b0), to_f(b1));
        const float2 ms = make_float2(-sn[q].x, -sn[q].y);
        const float2 r = ffma2(b, ms, fmul2(a, cs[q])), s = ffma2(b, cs[q], fmul2(a, sn[q]));
        a0 = from_f<T>(r.x);
        a1 = from_f<T>(r.y);
        b0 = from_f<T>(s.x);
        b1 = from_f<T>(s.y);
      }
      if (INTER && whole < NP)  // the unit where the rotated channels end: its others pass untouched
#pragma unroll
        for (int q = 0; q < NP; ++q)
          if (q >= whole) {
            x.e[2 * q] = keep.e[2 * q];
            x.e[2 * q + 1] = keep.e[2 * q + 1];
          }
    }
    *reinterpret_cast<Vec<T, V>*>(out.at) = x;
    if (!INTER && rot) *reinterpret_cast<Vec<T, V>*>(out.at + p.R2 * ES) = y;
    advance(out, qos, kos);
    slot = slot + 1 == D ? 0 : slot + 1;
  }
}

// Layouts that 16-byte vectors do not fit: a unit is one pair or one passing channel.
template <typename T>
__global__ void __launch_bounds__(kThreads) scalar_kernel(const __grid_constant__ Params p, int inter) {
  extern __shared__ uint4 smem[];
  float* cos_ = reinterpret_cast<float*>(smem);
  float* sin_ = cos_ + p.tile * p.R2;
  __shared__ Token tab[kMaxTokens + 1];
  const long long t0 = (long long)blockIdx.x * p.tile;
  const int nt = (int)min((long long)p.tile, p.tokens - t0);
  token_table(p, tab, t0, nt, sizeof(T));
  angles(p, cos_, sin_, t0, nt, p.R2);
  __syncthreads();
  const int units = p.D - p.R2;
  const int total = nt * (p.Hq + p.Hk) * units;
  for (int i = threadIdx.x; i < total; i += kThreads) {
    const int row = i / units, u = i - row * units;
    const int t = row / (p.Hq + p.Hk);
    int h = row - t * (p.Hq + p.Hk);
    const bool isq = h < p.Hq;
    h -= isq ? 0 : p.Hq;
    const T* src = reinterpret_cast<const T*>(isq ? tab[t].q : tab[t].k) + h * (isq ? p.q_sh : p.k_sh);
    T* to = reinterpret_cast<T*>(isq ? tab[t].qo : tab[t].ko) + h * (isq ? p.qo_sh : p.ko_sh);
    if (u < p.R2) {
      const int c0 = inter ? 2 * u : u, c1 = inter ? 2 * u + 1 : u + p.R2;
      T x0 = src[c0], x1 = src[c1];
      rotate(x0, x1, make_float2(cos_[t * p.R2 + u], sin_[t * p.R2 + u]));
      to[c0] = x0;
      to[c1] = x1;
    } else {
      to[u + p.R2] = src[u + p.R2];
    }
  }
}

template <typename T>
static cudaError_t launch(const Params& p, bool vec, bool inter, cudaStream_t st) {
  const unsigned grid = (unsigned)((p.tokens + p.tile - 1) / p.tile);
  if (!vec) {
    scalar_kernel<T><<<grid, kThreads, (size_t)p.tile * p.R2 * sizeof(float2), st>>>(p, inter ? 1 : 0);
    return cudaGetLastError();
  }
  constexpr int V = 16 / sizeof(T);
  const int threads = (p.side * (inter ? p.D / V : (p.D - p.R2) / V) + 31) / 32 * 32;
  const size_t smem = (size_t)kDepth * threads * 16 + (size_t)p.tile * (inter ? p.D / 2 : p.R2) * sizeof(float2);
  auto kern = inter ? stream_kernel<T, true> : stream_kernel<T, false>;
  if (smem > 40 * 1024) {  // with the static part, past the 48 KB default
    const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    if (e != cudaSuccess) return e;
  }
  kern<<<grid, threads, smem, st>>>(p);
  return cudaGetLastError();
}

}  // namespace rotary
}  // namespace mh3

using namespace mh3;

extern "C" int mh3_rotary(const mh3_rotary_args* a, void* stream) {
  const mh3::NvtxRange nvtx_range("mh3_rotary");
  if (a == nullptr) return fail(MH3_ERR_INVALID, "mh3_rotary: null args");
  if (a->batch < 0 || a->seqlen < 0 || a->heads_q < 0 || a->heads_k < 0 || a->head_dim <= 0)
    return fail(MH3_ERR_INVALID, "mh3_rotary: negative size");
  if (a->head_dim > 2 * rotary::kMaxPairs) return fail(MH3_ERR_TOO_LARGE, "mh3_rotary: head_dim must be at most 256");
  if (a->dtype != MH3_DTYPE_BF16 && a->dtype != MH3_DTYPE_F16 && a->dtype != MH3_DTYPE_F32)
    return fail(MH3_ERR_INVALID, "mh3_rotary: dtype must be bf16, f16 or f32");
  if (a->pos_kind < 0 || a->pos_kind > 2) return fail(MH3_ERR_INVALID, "mh3_rotary: pos_kind must be 0, 1 or 2");
  if (a->n_axes < 1 || a->n_axes > 4) return fail(MH3_ERR_INVALID, "mh3_rotary: 1 to 4 axes");
  rotary::Params p;
  int r2 = 0;
  for (int x = 0; x < a->n_axes; ++x) {
    const int d = a->axes_dim[x];
    if (d < 0 || (d & 1)) return fail(MH3_ERR_INVALID, "mh3_rotary: axis widths must be even and not negative");
    if (d > a->head_dim - 2 * r2) return fail(MH3_ERR_INVALID, "mh3_rotary: axis widths exceed head_dim");
    if (!(a->theta[x] > 0.0) || !(a->theta[x] <= 1e300)) return fail(MH3_ERR_INVALID, "mh3_rotary: theta must be positive and finite");
    for (int j = 0; j < d / 2; ++j, ++r2) {
      p.rate[r2] = pow(a->theta[x], -2.0 * j / d) / 6.283185307179586476925286766559;
      p.axis[r2] = (uint8_t)x;
    }
  }
  if (r2 == 0) return fail(MH3_ERR_INVALID, "mh3_rotary: no channel to rotate");
  const long long tokens = (long long)a->batch * a->seqlen;
  if (tokens == 0 || a->heads_q + (long long)a->heads_k == 0) return MH3_OK;
  if (!a->positions || (a->heads_q > 0 && (!a->q || !a->q_out)) || (a->heads_k > 0 && (!a->k || !a->k_out)))
    return fail(MH3_ERR_INVALID, "mh3_rotary: null pointer");
  if ((long long)a->heads_q + a->heads_k > 8192 || tokens > (1ll << 34))
    return fail(MH3_ERR_TOO_LARGE, "mh3_rotary: too many heads or tokens");
  const bool inter = a->interleaved != 0;
  const int es = a->dtype == MH3_DTYPE_F32 ? 4 : 2, V = 16 / es;
  bool vec = a->head_dim % V == 0 && (inter || r2 % V == 0);
  auto fits = [&](const void* ptr, int heads, int64_t sb, int64_t sh, int64_t ss) {
    return heads == 0 || (((uintptr_t)ptr & 15u) == 0 && sb % V == 0 && sh % V == 0 && ss % V == 0);
  };
  vec = vec && fits(a->q, a->heads_q, a->q_stride_b, a->q_stride_h, a->q_stride_s) &&
        fits(a->q_out, a->heads_q, a->qo_stride_b, a->qo_stride_h, a->qo_stride_s) &&
        fits(a->k, a->heads_k, a->k_stride_b, a->k_stride_h, a->k_stride_s) &&
        fits(a->k_out, a->heads_k, a->ko_stride_b, a->ko_stride_h, a->ko_stride_s);
  p.q = static_cast<const char*>(a->q);
  p.k = static_cast<const char*>(a->k);
  p.qo = static_cast<char*>(a->q_out);
  p.ko = static_cast<char*>(a->k_out);
  p.q_sb = a->q_stride_b; p.q_sh = a->q_stride_h; p.q_ss = a->q_stride_s;
  p.k_sb = a->k_stride_b; p.k_sh = a->k_stride_h; p.k_ss = a->k_stride_s;
  p.qo_sb = a->qo_stride_b; p.qo_sh = a->qo_stride_h; p.qo_ss = a->qo_stride_s;
  p.ko_sb = a->ko_stride_b; p.ko_sh = a->ko_stride_h; p.ko_ss = a->ko_stride_s;
  p.tokens = tokens;
  p.S = a->seqlen;
  p.Hq = a->heads_q;
  p.Hk = a->heads_k;
  p.D = a->head_dim;
  p.R2 = r2;
  p.pos = a->positions;
  p.pos_kind = a->pos_kind;
  p.pos_sb = a->pos_stride_b;
  p.pos_ss = a->pos_stride_s;
  p.sign = a->inverse ? -1.0f : 1.0f;
  // Tokens per CTA: enough for 80 KB of Q and K (five stages of the ring), while
  // 148 SMs still get four CTAs each.
  const long long token_bytes = ((long long)a->heads_q + a->heads_k) * a->head_dim * es;
  int tile = 1;
  while (tile < rotary::kMaxTokens && tile * token_bytes < 81920 && tokens / (2 * tile) >= 148 * 4) tile *= 2;
  p.tile = tile;
  // Heads side by side: of the counts that fill 192 to 384 threads (fewer where a row
  // has too few heads), the one that leaves the fewest lanes without a row - 20 for
  // 40 heads of 128 channels.
  const int units = inter ? a->head_dim / V : (a->head_dim - r2) / V;
  p.side = 1;
  if (vec) {
    const int most = std::max(1, std::min(rotary::kMaxThreads / units, std::max(a->heads_q, a->heads_k)));
    const int least = std::max(1, std::min(192 / units, most));
    long long best = -1;
    for (int side = most; side >= least; --side) {
      const long long lost = (side - a->heads_q % side) % side + (side - a->heads_k % side) % side;
      if (best < 0 || lost < best) {
        best = lost;
        p.side = side;
      }
    }
  }
  if ((tokens + tile - 1) / tile > 0x7fffffffLL) return fail(MH3_ERR_TOO_LARGE, "mh3_rotary: too many tokens");
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  const cudaError_t e = a->dtype == MH3_DTYPE_BF16  ? rotary::launch<__nv_bfloat16>(p, vec, inter, st)
                        : a->dtype == MH3_DTYPE_F16 ? rotary::launch<__half>(p, vec, inter, st)
                                                    : rotary::launch<float>(p, vec, inter, st);
  return e == cudaSuccess ? MH3_OK : fail_cuda(e, "mh3_rotary launch");
}
