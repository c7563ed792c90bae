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
// Bound: HBM.  Q and K are read and written once by 16-byte vectors; a thread
// keeps the same channels for every head it visits, so it needs one row of
// angles per token, and issues kUnroll rows' loads before it rotates any.
#include <math.h>

#include "mh3_b200.h"
#include "mh3_internal.h"
#include "ptx.cuh"

namespace mh3 {
namespace rotary {

constexpr int kThreads = 256;
constexpr int kMaxPairs = 128;  // head_dim <= 256
constexpr int kUnroll = 5;      // head rows whose loads are in flight per thread
constexpr int kMaxTokens = 8;   // tokens per CTA

struct Params {
  const char *q, *k;
  char *qo, *ko;
  long long q_sb, q_sh, q_ss, k_sb, k_sh, k_ss;      // element strides
  long long qo_sb, qo_sh, qo_ss, ko_sb, ko_sh, ko_ss;
  long long tokens;  // batch * seqlen
  int S, Hq, Hk, D, R2, tile;
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

// V: channels per vector (16 bytes), or 1 for layouts that vectors do not fit.
// INTER: pairs are neighbouring channels (2p, 2p+1); else (p, p + R/2).
// A thread's unit is one vector of the row: V/2 pairs when INTER (those past R/2
// pass), V pairs in two vectors when not, or V passing channels.
template <typename T, int V, bool INTER>
__global__ void __launch_bounds__(kThreads) kernel(const __grid_constant__ Params p) {
  extern __shared__ float2 cs[];  // [tile][npair] (cos, sin)
  const int npair = INTER ? (p.D + 1) / 2 : p.R2;  // INTER: a vector may reach past R/2
  const long long t0 = (long long)blockIdx.x * p.tile;
  const int nt = (int)min((long long)p.tile, p.tokens - t0);
  for (int i = threadIdx.x; i < nt * npair; i += kThreads) {
    const int t = i / npair, j = i - t * npair;
    float2 r = make_float2(1.0f, 0.0f);
    if (j < p.R2) {
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
      r = make_float2(c, sn * p.sign);
    }
    cs[i] = r;
  }
  __syncthreads();

  // units of a row, and the rows that this CTA's threads visit side by side
  const int units = !INTER ? p.R2 / V + (p.D - 2 * p.R2) / V : V > 1 ? p.D / V : npair;
  const int rot_units = INTER ? (V > 1 ? units : p.R2) : p.R2 / V;
  const int lanes = min(units, kThreads);
  const int side = kThreads / lanes;
  const int row0 = threadIdx.x / lanes;
  if (row0 >= side) return;
  const int rows = p.Hq + p.Hk;
  for (int u = threadIdx.x - row0 * lanes; u < units; u += lanes) {
    const bool rot = u < rot_units;
    // first channel of the unit, and the distance to its second vector
    const int c0 = INTER ? (V > 1 ? u * V : 2 * u) : (rot ? u * V : 2 * p.R2 + (u - rot_units) * V);
    const int dist = INTER ? 1 : p.R2;
    const bool two = INTER ? (V == 1 && c0 + 1 < p.D) : rot;  // a second vector (every rotated pair of V == 1 has one)
    for (int t = 0; t < nt; ++t) {
      const long long tok = t0 + t;
      const long long b = tok / p.S, s = tok - b * p.S;
      const T* qp = reinterpret_cast<const T*>(p.q) + b * p.q_sb + s * p.q_ss + c0;
      const T* kp = reinterpret_cast<const T*>(p.k) + b * p.k_sb + s * p.k_ss + c0;
      T* qo = reinterpret_cast<T*>(p.qo) + b * p.qo_sb + s * p.qo_ss + c0;
      T* ko = reinterpret_cast<T*>(p.ko) + b * p.ko_sb + s * p.ko_ss + c0;
      constexpr int NP = INTER ? (V > 1 ? V / 2 : 1) : V;  // pairs of a unit
      float2 a[NP];
#pragma unroll
      for (int j = 0; j < NP; ++j)
        a[j] = rot ? cs[t * npair + u * NP + j] : make_float2(1.0f, 0.0f);
      for (int r = row0; r < rows; r += side * kUnroll) {
        Vec<T, V> x[kUnroll], y[kUnroll];
#pragma unroll
        for (int i = 0; i < kUnroll; ++i) {
          const int h = r + i * side;
          if (h < rows) {
            const T* at = h < p.Hq ? qp + h * p.q_sh : kp + (h - p.Hq) * p.k_sh;
            x[i] = *reinterpret_cast<const Vec<T, V>*>(at);
            if ((V == 1 || !INTER) && two) y[i] = *reinterpret_cast<const Vec<T, V>*>(at + dist);
          }
        }
#pragma unroll
        for (int i = 0; i < kUnroll; ++i) {
          const int h = r + i * side;
          if (h >= rows) break;
          T* to = h < p.Hq ? qo + h * p.qo_sh : ko + (h - p.Hq) * p.ko_sh;
          if constexpr (INTER && V > 1) {
#pragma unroll
            for (int j = 0; j < NP; ++j) {
              if (u * NP + j >= p.R2) break;
              const float v0 = to_f(x[i].e[2 * j]), v1 = to_f(x[i].e[2 * j + 1]);
              x[i].e[2 * j] = from_f<T>(v0 * a[j].x - v1 * a[j].y);
              x[i].e[2 * j + 1] = from_f<T>(v0 * a[j].y + v1 * a[j].x);
            }
          } else if (rot) {
#pragma unroll
            for (int j = 0; j < NP; ++j) {
              const float v0 = to_f(x[i].e[j]), v1 = to_f(y[i].e[j]);
              x[i].e[j] = from_f<T>(v0 * a[j].x - v1 * a[j].y);
              y[i].e[j] = from_f<T>(v0 * a[j].y + v1 * a[j].x);
            }
          }
          *reinterpret_cast<Vec<T, V>*>(to) = x[i];
          if ((V == 1 || !INTER) && two) *reinterpret_cast<Vec<T, V>*>(to + dist) = y[i];
        }
      }
    }
  }
}

template <typename T, int V, bool INTER>
static cudaError_t launch(const Params& p, cudaStream_t st) {
  const int npair = INTER ? (p.D + 1) / 2 : p.R2;
  const unsigned grid = (unsigned)((p.tokens + p.tile - 1) / p.tile);
  kernel<T, V, INTER><<<grid, kThreads, (size_t)p.tile * npair * sizeof(float2), st>>>(p);
  return cudaGetLastError();
}

template <typename T>
static cudaError_t launch_type(const Params& p, bool vec, bool inter, cudaStream_t st) {
  constexpr int V = 16 / sizeof(T);
  if (vec) return inter ? launch<T, V, true>(p, st) : launch<T, V, false>(p, st);
  return inter ? launch<T, 1, true>(p, st) : launch<T, 1, false>(p, st);
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
  if ((long long)a->heads_q + a->heads_k > (1 << 24) || tokens > (1ll << 40))
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
  // Tokens per CTA: enough for 40 KB of Q and K, which hides the angles'
  // latency, while 148 SMs still get several CTAs each.
  const long long token_bytes = ((long long)a->heads_q + a->heads_k) * a->head_dim * es;
  int tile = 1;
  while (tile < rotary::kMaxTokens && tile * token_bytes < 40960 && tokens / (2 * tile) >= 148 * 8) tile *= 2;
  p.tile = tile;
  if ((tokens + tile - 1) / tile > 0x7fffffffLL) return fail(MH3_ERR_TOO_LARGE, "mh3_rotary: too many tokens");
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  const cudaError_t e = a->dtype == MH3_DTYPE_BF16  ? rotary::launch_type<__nv_bfloat16>(p, vec, inter, st)
                        : a->dtype == MH3_DTYPE_F16 ? rotary::launch_type<__half>(p, vec, inter, st)
                                                    : rotary::launch_type<float>(p, vec, inter, st);
  return e == cudaSuccess ? MH3_OK : fail_cuda(e, "mh3_rotary launch");
}
