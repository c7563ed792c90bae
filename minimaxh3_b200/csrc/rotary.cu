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
// keeps the same channels for every (token, head) row it visits; its rows stream
// through its own part of a three-stage ring in shared memory (cp.async, no
// barrier), and the first stages are on their way before the angles are computed.
#include <math.h>

#include "mh3_b200.h"
#include "mh3_internal.h"
#include "ptx.cuh"

namespace mh3 {
namespace rotary {

constexpr int kThreads = 256;
constexpr int kMaxPairs = 128;  // head_dim <= 256
constexpr int kMaxTokens = 16;  // tokens per CTA
constexpr int kStages = 3;
constexpr int kVectors = 4;     // 16-byte vectors of a thread in a stage

struct Params {
  const char *q, *k;
  char *qo, *ko;
  long long q_sb, q_sh, q_ss, k_sb, k_sh, k_ss;      // element strides
  long long qo_sb, qo_sh, qo_ss, ko_sb, ko_sh, ko_ss;
  long long tokens;  // batch * seqlen
  int S, Hq, Hk, D, R2, tile;
  unsigned magic;  // 2^32 / (Hq + Hk) + 1; 0 for one head
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

// (cos, sin) of the CTA's tokens, [nt][npair]; pairs past R/2 are not used.
__device__ __forceinline__ void angles(const Params& p, float2* cs, long long t0, int nt, int npair) {
  for (int i = threadIdx.x; i < nt * npair; i += kThreads) {
    const int t = i / npair, j = i - t * npair;
    if (j >= p.R2) continue;
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
    cs[i] = make_float2(c, sn * p.sign);
  }
}

// Row i of the CTA's tokens x heads is head i % rows of token i / rows, Q's heads
// first.  Its addresses come from a table of the CTA's tokens: head 0's address of Q
// and of the output, and for K the address that its first head would have if K's
// heads were numbered from 0 too - so a row costs a division (a multiplication by
// the host's 2^32 / rows + 1, exact below 2^32 / rows), a select and one product.
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
    t.k = p.k + (b * p.k_sb + s * p.k_ss - p.Hq * p.k_sh) * es;
    t.qo = p.qo + (b * p.qo_sb + s * p.qo_ss) * es;
    t.ko = p.ko + (b * p.ko_sb + s * p.ko_ss - p.Hq * p.ko_sh) * es;
    tab[threadIdx.x] = t;
  }
}
__device__ __forceinline__ int row_token(const Params& p, int i, int& h) {
  const int t = p.magic != 0 ? (int)__umulhi((unsigned)i, p.magic) : i;
  h = i - t * (p.Hq + p.Hk);
  return t;
}

template <typename T>
__device__ __forceinline__ void rotate(T& x0, T& x1, float2 a) {
  const float v0 = to_f(x0), v1 = to_f(x1);
  x0 = from_f<T>(v0 * a.x - v1 * a.y);
  x1 = from_f<T>(v0 * a.y + v1 * a.x);
}

// INTER: pairs are neighbouring channels (2p, 2p+1); else (p, p + R/2).
// A thread's unit is one 16-byte vector of the row when INTER (pairs past R/2
// pass), and when not the two vectors of V pairs, or V passing channels.
template <typename T, bool INTER>
__global__ void __launch_bounds__(kThreads) stream_kernel(const __grid_constant__ Params p) {
  constexpr int V = 16 / sizeof(T);
  constexpr int W = INTER ? 1 : 2;       // vectors of a unit
  constexpr int U = kVectors / W;        // rows of a stage
  constexpr int NP = INTER ? V / 2 : V;  // pairs of a unit
  extern __shared__ uint4 smem[];
  uint4* ring = smem + threadIdx.x;  // [kStages][kVectors][kThreads]
  float2* cs = reinterpret_cast<float2*>(smem + kStages * kVectors * kThreads);
  __shared__ Token tab[kMaxTokens];
  const int npair = INTER ? p.D / 2 : p.R2;
  const long long t0 = (long long)blockIdx.x * p.tile;
  const int nt = (int)min((long long)p.tile, p.tokens - t0);
  const int rot_units = INTER ? p.D / V : p.R2 / V;
  const int units = INTER ? rot_units : rot_units + (p.D - 2 * p.R2) / V;
  const int side = kThreads / units;  // rows visited side by side (units <= 64)
  const int row0 = threadIdx.x / units, u = threadIdx.x - row0 * units;
  const bool rot = u < rot_units;
  const int c0 = rot ? u * V : 2 * p.R2 + (u - rot_units) * V;
  const int n = row0 < side ? nt * (p.Hq + p.Hk) : 0;  // rows of the CTA
  auto issue = [&](int i, int st) {
#pragma unroll
    for (int k = 0; k < U; ++k) {
      const int j = i + k * side;
      if (j < n) {
        int h;
        const Token& tk = tab[row_token(p, j, h)];
        const T* src = reinterpret_cast<const T*>(h < p.Hq ? tk.q : tk.k) + h * (h < p.Hq ? p.q_sh : p.k_sh) + c0;
        uint4* dst = ring + (st * kVectors + k * W) * kThreads;
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(dst)), "l"(src) : "memory");
        if (!INTER && rot)
          asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(dst + kThreads)), "l"(src + p.R2) : "memory");
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  token_table(p, tab, t0, nt, sizeof(T));
  __syncthreads();
#pragma unroll
  for (int j = 0; j < kStages - 1; ++j) issue(row0 + j * U * side, j);
  angles(p, cs, t0, nt, npair);
  __syncthreads();
  int st = 0;
  for (int i = row0; i < n; i += U * side) {
    issue(i + (kStages - 1) * U * side, st == 0 ? kStages - 1 : st - 1);
    asm volatile("cp.async.wait_group %0;" ::"n"(kStages - 1) : "memory");
#pragma unroll
    for (int k = 0; k < U; ++k) {
      const int j = i + k * side;
      if (j >= n) break;
      int h;
      const int t = row_token(p, j, h);
      const Token& tk = tab[t];
      T* to = reinterpret_cast<T*>(h < p.Hq ? tk.qo : tk.ko) + h * (h < p.Hq ? p.qo_sh : p.ko_sh) + c0;
      const uint4* src = ring + (st * kVectors + k * W) * kThreads;
      Vec<T, V> x, y;
      x = *reinterpret_cast<const Vec<T, V>*>(src);
      if (rot) {
        if (!INTER) y = *reinterpret_cast<const Vec<T, V>*>(src + kThreads);
        const float4* ap = reinterpret_cast<const float4*>(cs + t * npair + u * NP);
#pragma unroll
        for (int q = 0; q < NP / 2; ++q) {
          const float4 a = ap[q];
          if (INTER) {
            if (u * NP + 2 * q < p.R2) rotate(x.e[4 * q], x.e[4 * q + 1], make_float2(a.x, a.y));
            if (u * NP + 2 * q + 1 < p.R2) rotate(x.e[4 * q + 2], x.e[4 * q + 3], make_float2(a.z, a.w));
          } else {
            rotate(x.e[2 * q], y.e[2 * q], make_float2(a.x, a.y));
            rotate(x.e[2 * q + 1], y.e[2 * q + 1], make_float2(a.z, a.w));
          }
        }
      }
      *reinterpret_cast<Vec<T, V>*>(to) = x;
      if (!INTER && rot) *reinterpret_cast<Vec<T, V>*>(to + p.R2) = y;
    }
    st = st + 1 == kStages ? 0 : st + 1;
  }
}

// Layouts that 16-byte vectors do not fit: a unit is one pair or one passing channel.
template <typename T>
__global__ void __launch_bounds__(kThreads) scalar_kernel(const __grid_constant__ Params p, int inter) {
  extern __shared__ uint4 smem[];
  float2* cs = reinterpret_cast<float2*>(smem);
  __shared__ Token tab[kMaxTokens];
  const long long t0 = (long long)blockIdx.x * p.tile;
  const int nt = (int)min((long long)p.tile, p.tokens - t0);
  token_table(p, tab, t0, nt, sizeof(T));
  angles(p, cs, t0, nt, p.R2);
  __syncthreads();
  const int units = p.D - p.R2;
  const int total = nt * (p.Hq + p.Hk) * units;
  for (int i = threadIdx.x; i < total; i += kThreads) {
    const int row = i / units, u = i - row * units;
    int h;
    const int t = row_token(p, row, h);
    const bool isq = h < p.Hq;
    const T* src = reinterpret_cast<const T*>(isq ? tab[t].q : tab[t].k) + h * (isq ? p.q_sh : p.k_sh);
    T* to = reinterpret_cast<T*>(isq ? tab[t].qo : tab[t].ko) + h * (isq ? p.qo_sh : p.ko_sh);
    if (u < p.R2) {
      const int c0 = inter ? 2 * u : u, c1 = inter ? 2 * u + 1 : u + p.R2;
      T x0 = src[c0], x1 = src[c1];
      rotate(x0, x1, cs[t * p.R2 + u]);
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
  const size_t smem = (size_t)kStages * kVectors * kThreads * 16 + (size_t)p.tile * (inter ? p.D / 2 : p.R2) * sizeof(float2);
  auto kern = inter ? stream_kernel<T, true> : stream_kernel<T, false>;
  if (smem > 40 * 1024) {  // with the static part, past the 48 KB default
    const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    if (e != cudaSuccess) return e;
  }
  kern<<<grid, kThreads, smem, st>>>(p);
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
  // A CTA's rows are divided by their number per token with a 32-bit product: exact
  // while 16 (heads)^2 < 2^32.
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
  p.magic = p.Hq + p.Hk == 1 ? 0u : (unsigned)((1ull << 32) / (unsigned)(p.Hq + p.Hk)) + 1u;
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
  if ((tokens + tile - 1) / tile > 0x7fffffffLL) return fail(MH3_ERR_TOO_LARGE, "mh3_rotary: too many tokens");
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  const cudaError_t e = a->dtype == MH3_DTYPE_BF16  ? rotary::launch<__nv_bfloat16>(p, vec, inter, st)
                        : a->dtype == MH3_DTYPE_F16 ? rotary::launch<__half>(p, vec, inter, st)
                                                    : rotary::launch<float>(p, vec, inter, st);
  return e == cudaSuccess ? MH3_OK : fail_cuda(e, "mh3_rotary launch");
}
