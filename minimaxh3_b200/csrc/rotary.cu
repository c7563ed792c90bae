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
// keeps the same channels of the same one to four heads for every token of its
// CTA, so a vector costs two pointer increments and about forty instructions in
// all (with the head looked up per vector it was 160, and the kernel issue-bound:
// 326 us at 32760 tokens x 80 heads x 128).  Its vectors stream through its own part
// of a ring in shared memory (cp.async, no barrier); the first tokens are on their
// way before the angles are computed.
#include <math.h>

#include <algorithm>

#include "mh3_b200.h"
#include "mh3_internal.h"
#include "ptx.cuh"

namespace mh3 {
namespace rotary {

constexpr int kThreads = 256;     // of the scalar kernel
constexpr int kMaxThreads = 384;  // of the streaming kernel
constexpr int kMaxPairs = 128;    // head_dim <= 256
constexpr int kMaxTokens = 16;    // tokens per CTA
constexpr int kDepth = 4;         // tokens in the ring
// The most a streaming kernel takes: a ring of four vectors a thread, and the angles.
constexpr size_t kSmemMax = (size_t)kDepth * 4 * kMaxThreads * 16 + (size_t)kMaxTokens * kMaxPairs * sizeof(float2);

struct Params {
  const char *q, *k;
  char *qo, *ko;
  long long q_sb, q_sh, q_ss, k_sb, k_sh, k_ss;      // element strides
  long long qo_sb, qo_sh, qo_ss, ko_sb, ko_sh, ko_ss;
  long long tokens;  // batch * seqlen
  int S, Hq, Hk, D, R2, tile;
  int side;  // rows (heads of Q, then of K) that a CTA visits side by side
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

// Batch item and place of a token.
__device__ __forceinline__ long long split(const Params& p, long long tok, int& s) {
  if (tok < p.S) {
    s = (int)tok;
    return 0;
  }
  const long long b = p.tokens <= 0xffffffffll ? (long long)((unsigned)tok / (unsigned)p.S) : tok / p.S;
  s = (int)(tok - b * p.S);
  return b;
}

// cos and sin of the CTA's tokens, [nt][npair] each; pairs past R/2 have the angle 0.
__device__ __forceinline__ void angles(const Params& p, float* cos_, float* sin_, long long t0, int nt, int npair) {
  for (int i = threadIdx.x; i < nt * npair; i += blockDim.x) {
    const int t = i / npair, j = i - t * npair;
    if (j >= p.R2) {
      cos_[i] = 1.0f;
      sin_[i] = 0.0f;
      continue;
    }
    int s;
    const long long b = split(p, t0 + t, s);
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

template <typename T>
__device__ __forceinline__ void rotate(T& x0, T& x1, float2 a) {
  const float v0 = to_f(x0), v1 = to_f(x1);
  x0 = from_f<T>(fmaf(v1, -a.y, __fmul_rn(v0, a.x)));  // the streaming kernel's order: the same bits for every layout
  x1 = from_f<T>(fmaf(v1, a.x, __fmul_rn(v0, a.y)));
}

// Eight or four values of a vector as pairs (2i, 2i+1), and back.
template <typename T>
struct Pairs {
  static constexpr int N = 8 / sizeof(T);
  float2 e[N];
  __device__ __forceinline__ explicit Pairs(const uint4& u) {
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < N; ++i) {
      if constexpr (sizeof(T) == 4) e[i] = make_float2(__uint_as_float(w[2 * i]), __uint_as_float(w[2 * i + 1]));
      else if constexpr (std::is_same<T, __half>::value) e[i] = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
      else e[i] = make_float2(__uint_as_float(w[i] << 16), __uint_as_float(w[i] & 0xffff0000u));
    }
  }
  __device__ __forceinline__ uint4 vec() const {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < N; ++i) {
      if constexpr (sizeof(T) == 4) {
        w[2 * i] = __float_as_uint(e[i].x);
        w[2 * i + 1] = __float_as_uint(e[i].y);
      } else if constexpr (std::is_same<T, __half>::value) {
        const __half2 h = __floats2half2_rn(e[i].x, e[i].y);
        w[i] = *reinterpret_cast<const uint32_t*>(&h);
      } else {
        const __nv_bfloat162 h = __floats2bfloat162_rn(e[i].x, e[i].y);
        w[i] = *reinterpret_cast<const uint32_t*>(&h);
      }
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
  }
};

// The units of a row: one 16-byte vector when INTER (pairs past R/2 pass), and when
// not the two vectors of V pairs, or V passing channels.  A CTA: ``side`` x M rows of
// ``tile`` tokens.
template <typename T, bool INTER, int M>
__global__ void __launch_bounds__(kMaxThreads) stream_kernel(const __grid_constant__ Params p) {
  constexpr int V = 16 / sizeof(T), ES = sizeof(T);
  constexpr int W = INTER ? 1 : 2;       // vectors of a unit
  constexpr int NP = INTER ? V / 2 : V;  // pairs of a unit
  extern __shared__ uint4 smem[];
  uint4* ring = smem + threadIdx.x;  // [kDepth][M][W][threads]
  const int nthr = blockDim.x;
  float* cos_ = reinterpret_cast<float*>(smem + kDepth * M * W * nthr);
  const int npair = INTER ? p.D / 2 : p.R2;
  float* sin_ = cos_ + p.tile * npair;
  const long long t0 = (long long)blockIdx.x * p.tile;
  const int nt = (int)min((long long)p.tile, p.tokens - t0);
  const int rot_units = INTER ? p.D / V : p.R2 / V;
  const int units = INTER ? rot_units : rot_units + (p.D - 2 * p.R2) / V;
  const int row0 = threadIdx.x / units, u = threadIdx.x - row0 * units;
  const bool rot = u < rot_units;
  const int c0 = rot ? u * V : 2 * p.R2 + (u - rot_units) * V;
  int s_in;
  const long long b0 = split(p, t0, s_in);
  int s_out = s_in;
  const char* in[M];
  char* out[M];
  unsigned own = 0, isq = 0;  // bit j: the thread has row j; it is one of Q's
#pragma unroll
  for (int j = 0; j < M; ++j) {
    const int r = blockIdx.y * (M * p.side) + j * p.side + row0;
    const int h = r < p.Hq ? r : r - p.Hq;
    if (r < p.Hq) {
      isq |= 1u << j;
      in[j] = p.q + (b0 * p.q_sb + s_in * p.q_ss + h * p.q_sh + c0) * ES;
      out[j] = p.qo + (b0 * p.qo_sb + s_in * p.qo_ss + h * p.qo_sh + c0) * ES;
    } else {
      in[j] = p.k + (b0 * p.k_sb + s_in * p.k_ss + h * p.k_sh + c0) * ES;
      out[j] = p.ko + (b0 * p.ko_sb + s_in * p.ko_ss + h * p.ko_sh + c0) * ES;
    }
    if (row0 < p.side && r < p.Hq + p.Hk) own |= 1u << j;
  }
  int ahead = 0;
  auto issue = [&](int slot) {  // the next token's vectors into the ring
    if (ahead < nt) {
      ++ahead;
      const bool wrap = ++s_in == p.S;
      if (wrap) s_in = 0;
#pragma unroll
      for (int j = 0; j < M; ++j) {
        const bool mine = own >> j & 1u, q = isq >> j & 1u;
        uint4* dst = ring + (slot * M + j) * W * nthr;
        if (mine) {
          asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(dst)), "l"(in[j]) : "memory");
          if (!INTER && rot)
            asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(dst + nthr)), "l"(in[j] + p.R2 * ES) : "memory");
        }
        in[j] += (q ? p.q_ss : p.k_ss) * ES;
        if (wrap) in[j] += (q ? p.q_sb - p.S * p.q_ss : p.k_sb - p.S * p.k_ss) * ES;  // the next batch item
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
#pragma unroll
  for (int j = 0; j < kDepth - 1; ++j) issue(j);
  angles(p, cos_, sin_, t0, nt, npair);
  __syncthreads();
  const int whole = INTER ? max(0, min(NP, p.R2 - u * NP)) : (rot ? NP : 0);  // rotated pairs of the unit
  const float *cp = cos_ + u * NP, *sp = sin_ + u * NP;
  int slot = 0;
  for (int t = 0; t < nt; ++t, cp += npair, sp += npair) {
    issue(slot == 0 ? kDepth - 1 : slot - 1);
    float2 cs[NP / 2], sn[NP / 2], ns[NP / 2];  // of pairs 2i and 2i + 1
    if (whole) {
#pragma unroll
      for (int i = 0; i < NP / 2; ++i) {
        cs[i] = *reinterpret_cast<const float2*>(cp + 2 * i);
        sn[i] = *reinterpret_cast<const float2*>(sp + 2 * i);
        ns[i] = make_float2(-sn[i].x, -sn[i].y);
      }
    }
    asm volatile("cp.async.wait_group %0;" ::"n"(kDepth - 1) : "memory");
    const bool wrap = ++s_out == p.S;
    if (wrap) s_out = 0;
#pragma unroll
    for (int j = 0; j < M; ++j) {
      const bool q = isq >> j & 1u;
      if (own >> j & 1u) {
        const uint4* src = ring + (slot * M + j) * W * nthr;
        uint4 x = src[0];
        if (whole) {
          if constexpr (INTER) {
            Pairs<T> v(x);
#pragma unroll
            for (int i = 0; i < NP / 2; ++i) {  // the first and second channels of two pairs, side by side
              const float2 a = make_float2(v.e[2 * i].x, v.e[2 * i + 1].x), b = make_float2(v.e[2 * i].y, v.e[2 * i + 1].y);
              const float2 r = ffma2(b, ns[i], fmul2(a, cs[i])), w = ffma2(b, cs[i], fmul2(a, sn[i]));
              v.e[2 * i] = make_float2(r.x, w.x);
              v.e[2 * i + 1] = make_float2(r.y, w.y);
            }
            const uint4 y = v.vec();
            if (whole == NP) {
              x = y;
            } else {  // the unit where the rotated channels end: its others pass untouched
              constexpr int WP = ES == 4 ? 2 : 1;  // words of a pair
              const uint32_t old[4] = {x.x, x.y, x.z, x.w}, now[4] = {y.x, y.y, y.z, y.w};
              uint32_t w[4];
#pragma unroll
              for (int i = 0; i < 4; ++i) w[i] = i / WP < whole ? now[i] : old[i];
              x = make_uint4(w[0], w[1], w[2], w[3]);
            }
          } else {
            Pairs<T> a(x), b(src[nthr]);
#pragma unroll
            for (int i = 0; i < NP / 2; ++i) {
              const float2 r = ffma2(b.e[i], ns[i], fmul2(a.e[i], cs[i]));
              b.e[i] = ffma2(b.e[i], cs[i], fmul2(a.e[i], sn[i]));
              a.e[i] = r;
            }
            x = a.vec();
            *reinterpret_cast<uint4*>(out[j] + p.R2 * ES) = b.vec();
          }
        }
        *reinterpret_cast<uint4*>(out[j]) = x;
      }
      out[j] += (q ? p.qo_ss : p.ko_ss) * ES;
      if (wrap) out[j] += (q ? p.qo_sb - p.S * p.qo_ss : p.ko_sb - p.S * p.ko_ss) * ES;
    }
    slot = slot + 1 == kDepth ? 0 : slot + 1;
  }
}

// Layouts that 16-byte vectors do not fit: a unit is one pair or one passing channel.
template <typename T>
__global__ void __launch_bounds__(kThreads) scalar_kernel(const __grid_constant__ Params p, int inter) {
  extern __shared__ uint4 smem[];
  float* cos_ = reinterpret_cast<float*>(smem);
  float* sin_ = cos_ + p.tile * p.R2;
  const long long t0 = (long long)blockIdx.x * p.tile;
  const int nt = (int)min((long long)p.tile, p.tokens - t0);
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
    int sq;
    const long long b = split(p, t0 + t, sq);
    const T* src = reinterpret_cast<const T*>(isq ? p.q : p.k) + (isq ? b * p.q_sb + sq * p.q_ss + h * p.q_sh : b * p.k_sb + sq * p.k_ss + h * p.k_sh);
    T* to = reinterpret_cast<T*>(isq ? p.qo : p.ko) + (isq ? b * p.qo_sb + sq * p.qo_ss + h * p.qo_sh : b * p.ko_sb + sq * p.ko_ss + h * p.ko_sh);
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

template <auto K>
static cudaError_t start(const Params& p, dim3 blocks, int threads, size_t smem, cudaStream_t st) {
  if (smem > 40 * 1024) {  // past the 48 KB default
    const cudaError_t e = allow_smem<K>(kSmemMax);
    if (e != cudaSuccess) return e;
  }
  K<<<blocks, threads, smem, st>>>(p);
  return cudaGetLastError();
}

template <typename T>
static cudaError_t launch(const Params& p, bool vec, bool inter, cudaStream_t st) {
  const unsigned grid = (unsigned)((p.tokens + p.tile - 1) / p.tile);
  if (!vec) {
    scalar_kernel<T><<<grid, kThreads, (size_t)p.tile * p.R2 * sizeof(float2), st>>>(p, inter ? 1 : 0);
    return cudaGetLastError();
  }
  // Rows per thread: the fewest of 1, 2 and 4 with which the CTA's threads hold all heads
  // (half as many when a unit is two vectors); more heads than that in further CTAs.
  constexpr int V = 16 / sizeof(T);
  const int units = inter ? p.D / V : (p.D - p.R2) / V, rows = p.Hq + p.Hk, most = inter ? 4 : 2;
  int m = 1;
  while (m < most && (rows + m - 1) / m * units > kMaxThreads) m *= 2;
  Params q = p;
  q.side = std::min((rows + m - 1) / m, kMaxThreads / units);
  const int threads = (q.side * units + 31) / 32 * 32;
  const size_t smem = (size_t)kDepth * m * (inter ? 1 : 2) * threads * 16 + (size_t)p.tile * (inter ? p.D / 2 : p.R2) * sizeof(float2);
  const dim3 blocks(grid, (unsigned)((rows + m * q.side - 1) / (m * q.side)));
  if (inter)
    return m == 1   ? start<stream_kernel<T, true, 1>>(q, blocks, threads, smem, st)
           : m == 2 ? start<stream_kernel<T, true, 2>>(q, blocks, threads, smem, st)
                    : start<stream_kernel<T, true, 4>>(q, blocks, threads, smem, st);
  return m == 1 ? start<stream_kernel<T, false, 1>>(q, blocks, threads, smem, st)
                : start<stream_kernel<T, false, 2>>(q, blocks, threads, smem, st);
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
  // Tokens per CTA: up to 160 KB of Q and K (two rounds of the ring), while 148 SMs
  // still get four CTAs each.
  const long long token_bytes = ((long long)a->heads_q + a->heads_k) * a->head_dim * es;
  int tile = 1;
  while (tile < rotary::kMaxTokens && tile * token_bytes < 163840 && tokens / (2 * tile) >= 148 * 4) tile *= 2;
  p.tile = tile;
  if ((tokens + tile - 1) / tile > 0x7fffffffLL) return fail(MH3_ERR_TOO_LARGE, "mh3_rotary: too many tokens");
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  const cudaError_t e = a->dtype == MH3_DTYPE_BF16  ? rotary::launch<__nv_bfloat16>(p, vec, inter, st)
                        : a->dtype == MH3_DTYPE_F16 ? rotary::launch<__half>(p, vec, inter, st)
                                                    : rotary::launch<float>(p, vec, inter, st);
  return e == cudaSuccess ? MH3_OK : fail_cuda(e, "mh3_rotary launch");
}
