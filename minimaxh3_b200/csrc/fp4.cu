// Microscaled 4-bit rows: rounding to e2m1 with an e4m3 scale for 16 elements and
// a power of two for the row, and back.
//
// Why two levels: an e4m3 scale follows the blocks inside a row over 2^15, but a
// token's activations or a channel's weights may lie anywhere, so the row's
// largest block is put at e4m3's upper end.  The row scale is a power of two: x /
// scale and the row factors of a product are then exact, and it costs at most
// one of e4m3's 18 binades.
//
//   scale  = 2^max(-100, ceil(log2(absmax_row / 2688)))       2688 = 448 * 6
//   block  = e4m3(absmax_16 / (6 scale)),  code = e2m1(x / (block scale))
//
// Both quotients are correctly rounded (the first by Markstein's step, see quant.cu's
// div_rn_by; the second in round_block) and then rounded to nearest even, so the bytes
// are those of the definition.  With M in [1, 2) and absmax = M 2^E, absmax / 2688 = (M / 1.3125)
// 2^(E-11): the exponent is E - 11, one more if M > 1.3125 - integer compares.
//
// Bound: instruction issue (74 % of its slots) beside HBM, 2 bytes in and 0.5625 out
// per 16-bit element: 206 us = 5.6 TB/s at 32760 x 13824.  A thread owns the 16 elements
// of a block, so the block's maximum needs no exchange.  CTAs are persistent and take four rows 32
// apart at a time: their maxima share one barrier, and their block scales for 64
// elements are the 16 neighbouring bytes of the scale layout, written as one
// vector.  The rows stream through a two-stage ring in shared memory (cp.async),
// read once for the maxima and once for the rounding.  A warp copies its blocks as
// neighbouring 16-byte pieces: copied by their owners, two lanes' halves of every
// 32-byte sector came from L2 twice (362 us against 245 before the later steps).  Rows
// too long for that ring (over 14336 elements in 16 bits, 7168 in 32), and rows that
// 16-byte vectors do not fit, are read twice by the general kernel: 680 us = 3.0 TB/s at
// 32760 x 13824 f32, 140 us = 2.4 TB/s at 8192 x 16384 bf16.  Back: HBM, 172 us = 6.7 TB/s.
#include <algorithm>
#include <string>

#include "fp4.cuh"
#include "mh3_b200.h"
#include "mh3_internal.h"
#include "ptx.cuh"

namespace mh3 {
namespace fp4 {

constexpr int kMaxThreads = 1024;

// The four scales of neighbouring lanes as one word (b: the lane's scale index).
__device__ __forceinline__ void put_scales(uint8_t* blocks, uint32_t s8, long long row, int b, int nk64) {
  uint32_t word = s8 << (8 * (b & 3));
  const uint32_t lanes = 0xfu << (threadIdx.x & 28);
  word |= __shfl_xor_sync(lanes, word, 1);
  word |= __shfl_xor_sync(lanes, word, 2);
  if ((b & 3) == 0) *reinterpret_cast<uint32_t*>(blocks + block_offset(row, b, nk64)) = word;
}

// Maximum over a row's threads: all lanes of a warp, then its warps through two
// halves of shared memory in turn (one barrier: the half is written again only
// after the next call's).
__device__ __forceinline__ uint32_t row_max(uint32_t top, uint32_t (*red)[32], int& turn) {
  top = __reduce_max_sync(0xffffffffu, top);
  const int warps = blockDim.x >> 5;
  if (warps == 1) return top;
  const int lane = threadIdx.x & 31;
  uint32_t* r = red[turn] + threadIdx.y * warps;
  if (lane == 0) r[threadIdx.x >> 5] = top;
  __syncthreads();
  top = __reduce_max_sync(0xffffffffu, lane < warps ? r[lane] : 0u);
  turn ^= 1;
  return top;
}

constexpr int kQuad = 4;    // rows r, r + 32, r + 64, r + 96 of a block of 128
constexpr int kStages = 2;
constexpr size_t kRingMax = 224 * 1024;

// Streaming: blockDim.x threads (a multiple of 32, at least the row's scales) per
// row, blockDim.y quads at once.  Rows M.. of the last block of 128 get zero
// scales, so the buffer is the same whatever the memory held.
template <typename T>
__global__ void __launch_bounds__(kMaxThreads) quantize_stream_kernel(const T* __restrict__ x, long long stride, long long M, int K,
                                                                     uint8_t* __restrict__ x4, uint8_t* __restrict__ blocks,
                                                                     float* __restrict__ scale) {
  constexpr int W = sizeof(T);  // 16-byte vectors of a block
  extern __shared__ uint4 ring[];
  __shared__ uint4 red[2][32];  // a warp's four maxima
  const int nb = K / 16, nk64 = (K + 63) / 64, b = threadIdx.x;
  const int nthr = blockDim.x * blockDim.y, warps = blockDim.x >> 5, lane = threadIdx.x & 31;
  // [kStages][kQuad][nthr] blocks of W pieces; the warp's 32 blocks are copied piece
  // by piece, lane after lane, and each lane reads its own block.  Piece p lies at
  // p ^ (p / 8 % W), so that eight lanes W pieces apart read from eight different places
  // of the 128 bytes a cycle delivers.
  uint4* warp_at = ring + (threadIdx.y * blockDim.x + (threadIdx.x & ~31)) * W;
  uint4* put_at = warp_at + (lane ^ ((lane >> 3) & (W - 1)));
  const uint4* get_at[W];
#pragma unroll
  for (int w = 0; w < W; ++w) get_at[w] = warp_at + lane * W + (w ^ ((lane * W >> 3) & (W - 1)));
  const int piece0 = (threadIdx.x & ~31) * W + lane;  // of the row's nb W pieces
  const bool in = b < nb;
  const int quads = (int)((M + 127) / 128 * 32);  // of 32 in each block of 128 rows
  const int step = gridDim.x * blockDim.y;
  auto first_row = [](int q) { return (long long)(q >> 5) * 128 + (q & 31); };
  auto issue = [&](int q, int st) {
    if (q < quads) {
      long long row = first_row(q);
      const T* src = x + row * stride;
#pragma unroll
      for (int i = 0; i < kQuad; ++i, row += 32, src += 32 * stride)
        if (row < M)
#pragma unroll
          for (int w = 0; w < W; ++w)
            if (piece0 + 32 * w < nb * W)
              asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(
                               smem_u32(put_at + (st * kQuad + i) * nthr * W + 32 * w)),
                           "l"(reinterpret_cast<const uint4*>(src) + piece0 + 32 * w)
                           : "memory");
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  const int q0 = blockIdx.x * blockDim.y;
  issue(q0 + threadIdx.y, 0);
  int st = 0;
  for (int base = q0; base < quads; base += step) {  // the same trips for every thread of the CTA
    const int q = base + threadIdx.y;
    issue(q + step, st ^ 1);
    asm volatile("cp.async.wait_group %0;" ::"n"(kStages - 1) : "memory");
    __syncwarp();  // the warp's lanes see one another's pieces
    const long long row0 = first_row(q);
    auto load = [&](int i, uint4(&u)[W]) {
#pragma unroll
      for (int w = 0; w < W; ++w) u[w] = get_at[w][(st * kQuad + i) * nthr * W];
    };
    uint32_t own[kQuad], top[kQuad];
#pragma unroll
    for (int i = 0; i < kQuad; ++i) {
      own[i] = 0;
      if (in && q < quads && row0 + 32 * i < M) {
        uint4 u[W];
        load(i, u);
        own[i] = absmax_raw<T>(u);
      }
      top[i] = __reduce_max_sync(0xffffffffu, own[i]);
    }
    if (warps > 1) {
      uint4* r = red[st] + threadIdx.y * warps;
      if (lane == 0) r[threadIdx.x >> 5] = make_uint4(top[0], top[1], top[2], top[3]);
      __syncthreads();  // one per trip: this half is written again only after the next trip's
      const uint4 t = lane < warps ? r[lane] : make_uint4(0, 0, 0, 0);
      top[0] = __reduce_max_sync(0xffffffffu, t.x);
      top[1] = __reduce_max_sync(0xffffffffu, t.y);
      top[2] = __reduce_max_sync(0xffffffffu, t.z);
      top[3] = __reduce_max_sync(0xffffffffu, t.w);
    }
    if (q < quads) {
      uint32_t words[kQuad];
      uint8_t* xo = x4 + row0 * (K / 2) + (long long)b * 8;
#pragma unroll
      for (int i = 0; i < kQuad; ++i, xo += 16ll * K) {
        const bool live = row0 + 32 * i < M;
        const bool finite = top[i] < 0x7f800000u;
        const int e = row_exponent(top[i]);
        uint2 code = make_uint2(0, 0);
        uint32_t s8 = 0;
        if (live && in) {
          if (finite) {
            uint4 u[W];
            load(i, u);
            float2 v[8];
            pairs16<T>(u, v);
            s8 = round_block(v, own[i], e, code);
          }
          *reinterpret_cast<uint2*>(xo) = code;
          if (b == 0) scale[row0 + 32 * i] = finite ? pow2f(e) : __uint_as_float(0x7fffffffu);
        }
        words[i] = s8 << (8 * (b & 3));
      }
      if (b < nk64 * 4) {  // four lanes hold the four scales of each row's word
        const uint32_t lanes = 0xfu << (lane & 28);
#pragma unroll
        for (int i = 0; i < kQuad; ++i) {
          words[i] |= __shfl_xor_sync(lanes, words[i], 1);
          words[i] |= __shfl_xor_sync(lanes, words[i], 2);
        }
        if ((b & 3) == 0)
          *reinterpret_cast<uint4*>(blocks + ((long long)(q >> 5) * nk64 + (b >> 2)) * 512 + (q & 31) * 16) =
              make_uint4(words[0], words[1], words[2], words[3]);
      }
    }
    st ^= 1;
    __syncwarp();  // every lane has read this stage before one copies into it
  }
}

// General: one row per CTA, read once for its maximum and once for the rounding.
template <typename T>
__global__ void __launch_bounds__(kMaxThreads) quantize_kernel(const T* __restrict__ x, long long stride, long long M, int K,
                                                              uint8_t* __restrict__ x4, uint8_t* __restrict__ blocks,
                                                              float* __restrict__ scale, int vec) {
  __shared__ uint32_t red[2][32];
  const long long row = blockIdx.x;
  const int nb = K / 16, nk64 = (K + 63) / 64;
  const T* xp = x + row * stride;
  const bool live = row < M;
  float2 v[8];
  uint32_t top = 0;
  int turn = 0;
  if (live)
    for (int b = threadIdx.x; b < nb; b += blockDim.x) {
      load16(xp + (long long)b * 16, v, vec != 0);
      top = max(top, absmax16(v));
    }
  top = row_max(top, red, turn);
  const bool finite = top < 0x7f800000u;
  const int e = row_exponent(top);
  if (live && threadIdx.x == 0) scale[row] = finite ? pow2f(e) : __uint_as_float(0x7fffffffu);
  for (int b = threadIdx.x; b < nk64 * 4; b += blockDim.x) {
    uint32_t s8 = 0;
    uint2 code = make_uint2(0, 0);
    if (b < nb && live) {
      if (finite) {
        load16(xp + (long long)b * 16, v, vec != 0);
        s8 = round_block(v, absmax16(v), e, code);
      }
      *reinterpret_cast<uint2*>(x4 + row * (K / 2) + (long long)b * 8) = code;
    }
    put_scales(blocks, s8, row, b, nk64);
  }
}

// Eight elements per thread (16 bytes of bf16, neighbouring threads side by side) of
// the four rows whose scales lie in one vector.
template <typename T>
__global__ void __launch_bounds__(256) dequantize_kernel(const uint8_t* __restrict__ x4, const uint8_t* __restrict__ blocks,
                                                         const float* __restrict__ scale, int n8, long long M, T* __restrict__ out) {
  const int c = blockIdx.x * blockDim.x + threadIdx.x;  // of the row's n8 = K / 8 pieces
  const int nk64 = (n8 + 7) / 8;
  if (c >= n8) return;
  const int quads = (int)((M + 127) / 128 * 32);
  const int byte = 8 * ((c >> 1) & 3);
  for (int q = blockIdx.y * blockDim.y + threadIdx.y; q < quads; q += gridDim.y * blockDim.y) {
    const long long row0 = (long long)(q >> 5) * 128 + (q & 31);
    if (row0 >= M) continue;
    const uint32_t* src = reinterpret_cast<const uint32_t*>(x4) + row0 * n8 + c;
    T* o = out + (row0 * n8 + c) * 8;
    uint32_t code[kQuad];
    float rs[kQuad];
#pragma unroll
    for (int i = 0; i < kQuad; ++i) {
      const bool live = row0 + 32 * i < M;
      code[i] = live ? __ldcs(src + 32ll * i * n8) : 0u;
      rs[i] = live ? scale[row0 + 32 * i] : 0.0f;
    }
    const uint4 s4 = *reinterpret_cast<const uint4*>(blocks + ((long long)(q >> 5) * nk64 + (c >> 3)) * 512 + (q & 31) * 16);
    const uint32_t sw[kQuad] = {s4.x, s4.y, s4.z, s4.w};
#pragma unroll
    for (int i = 0; i < kQuad; ++i) {
      if (row0 + 32 * i >= M) break;
      const float2 s = both(e4m3_value((sw[i] >> byte) & 0xffu) * rs[i]);
      uint32_t h[4];
      e2m1x8_halves(code[i], h);
      float2 v[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) v[k] = fmul2(__half22float2(*reinterpret_cast<const __half2*>(&h[k])), s);
      T* to = o + 256ll * i * n8;
      if constexpr (std::is_same<T, float>::value) {
        reinterpret_cast<float4*>(to)[0] = make_float4(v[0].x, v[0].y, v[1].x, v[1].y);
        reinterpret_cast<float4*>(to)[1] = make_float4(v[2].x, v[2].y, v[3].x, v[3].y);
      } else {
        uint32_t w[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const __nv_bfloat162 p = __floats2bfloat162_rn(v[k].x, v[k].y);
          w[k] = *reinterpret_cast<const uint32_t*>(&p);
        }
        *reinterpret_cast<uint4*>(to) = make_uint4(w[0], w[1], w[2], w[3]);
      }
    }
  }
}

template <typename T>
static cudaError_t launch_quantize(const void* x, long long stride, long long M, int K, void* x4, void* blocks, float* scale,
                                   cudaStream_t st) {
  const int nb4 = (K + 63) / 64 * 4;  // scales of a row, the last word filled up
  const int tx = std::min(kMaxThreads, (nb4 + 31) / 32 * 32);
  const long long padded = (M + 127) / 128 * 128;
  const int vec = ((uintptr_t)x & 15u) == 0 && stride * (long long)sizeof(T) % 16 == 0;
  const T* xp = static_cast<const T*>(x);
  uint8_t *c = static_cast<uint8_t*>(x4), *b = static_cast<uint8_t*>(blocks);
  const int ty = std::max(1, 256 / tx);
  const int nthr = tx * ty;
  const size_t smem = (size_t)kStages * kQuad * sizeof(T) * 16 * nthr;
  if (nb4 > tx || !vec || smem > kRingMax) {
    quantize_kernel<T><<<(unsigned)padded, tx, 0, st>>>(xp, stride, M, K, c, b, scale, vec);
    return cudaGetLastError();
  }
  if (smem > 40 * 1024) {  // with the static part, past the 48 KB default
    const cudaError_t e = allow_smem<quantize_stream_kernel<T>>(kRingMax);
    if (e != cudaSuccess) return e;
  }
  // resident CTAs of 64 registers a thread and their rings
  const long long per = std::max<long long>(1, std::min<long long>(1024 / nthr, (long long)(kRingMax / smem)));
  const long long grid = std::min<long long>((padded / kQuad + ty - 1) / ty, 148 * per);
  quantize_stream_kernel<T><<<(unsigned)grid, dim3((unsigned)tx, (unsigned)ty), smem, st>>>(xp, stride, M, K, c, b, scale);
  return cudaGetLastError();
}

}  // namespace fp4
}  // namespace mh3

using namespace mh3;

extern "C" uint64_t mh3_fp4_block_bytes(int64_t M, int64_t K) {
  if (M <= 0 || K <= 0) return 0;
  return (uint64_t)((M + 127) / 128) * (uint64_t)((K + 63) / 64) * 512;
}

static int check_fp4(const char* what, int64_t M, int64_t K, const void* x4, const void* blocks, const float* scale) {
  static thread_local std::string msg;
  auto bad = [&](int code, const char* why) {
    msg = std::string(what) + ": " + why;
    return fail(code, msg.c_str());
  };
  if (M < 0 || K <= 0 || K % 32) return bad(MH3_ERR_INVALID, "K must be a positive multiple of 32");
  if (M > 0x7fffff00LL || K > (1ll << 30)) return bad(MH3_ERR_TOO_LARGE, "dimension too large");
  if (M > 0 && (!x4 || !blocks || !scale)) return bad(MH3_ERR_INVALID, "null pointer");
  if (((uintptr_t)x4 & 15u) || ((uintptr_t)blocks & 15u))
    return bad(MH3_ERR_INVALID, "the 4-bit buffers must be 16-byte aligned");
  return MH3_OK;
}

extern "C" int mh3_quantize_fp4(const void* x, int64_t x_stride, int32_t in_dtype, int64_t M, int64_t K, void* x4,
                                void* blocks, float* scale, void* stream) {
  const mh3::NvtxRange nvtx_range("mh3_quantize_fp4");
  const int rc = check_fp4("mh3_quantize_fp4", M, K, x4, blocks, scale);
  if (rc) return rc;
  if (in_dtype != MH3_DTYPE_BF16 && in_dtype != MH3_DTYPE_F16 && in_dtype != MH3_DTYPE_F32)
    return fail(MH3_ERR_INVALID, "mh3_quantize_fp4: in_dtype must be bf16, f16 or f32");
  if (M == 0) return MH3_OK;
  if (!x) return fail(MH3_ERR_INVALID, "mh3_quantize_fp4: null x");
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  const cudaError_t e = in_dtype == MH3_DTYPE_BF16 ? fp4::launch_quantize<__nv_bfloat16>(x, x_stride, M, (int)K, x4, blocks, scale, st)
                        : in_dtype == MH3_DTYPE_F16 ? fp4::launch_quantize<__half>(x, x_stride, M, (int)K, x4, blocks, scale, st)
                                                    : fp4::launch_quantize<float>(x, x_stride, M, (int)K, x4, blocks, scale, st);
  return e == cudaSuccess ? MH3_OK : fail_cuda(e, "mh3_quantize_fp4 launch");
}

extern "C" int mh3_dequantize_fp4(const void* x4, const void* blocks, const float* scale, int64_t M, int64_t K,
                                  int32_t out_dtype, void* out, void* stream) {
  const mh3::NvtxRange nvtx_range("mh3_dequantize_fp4");
  const int rc = check_fp4("mh3_dequantize_fp4", M, K, x4, blocks, scale);
  if (rc) return rc;
  if (out_dtype != MH3_DTYPE_BF16 && out_dtype != MH3_DTYPE_F32)
    return fail(MH3_ERR_INVALID, "mh3_dequantize_fp4: out_dtype must be bf16 or f32");
  if (M == 0) return MH3_OK;
  if (!out || ((uintptr_t)out & 15u)) return fail(MH3_ERR_INVALID, "mh3_dequantize_fp4: out must be 16-byte aligned and not null");
  const int n8 = (int)(K / 8);
  const int tx = std::min(256, (n8 + 31) / 32 * 32);
  const dim3 block((unsigned)tx, (unsigned)std::max(1, 256 / tx));
  const int64_t gx = (n8 + tx - 1) / tx;
  const int64_t gy = ((M + 127) / 128 * 32 + block.y - 1) / block.y;  // quads
  const dim3 grid((unsigned)gx, (unsigned)std::min<int64_t>(gy, 65535));
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  const uint8_t *c = static_cast<const uint8_t*>(x4), *b = static_cast<const uint8_t*>(blocks);
  if (out_dtype == MH3_DTYPE_F32)
    fp4::dequantize_kernel<float><<<grid, block, 0, st>>>(c, b, scale, n8, M, static_cast<float*>(out));
  else
    fp4::dequantize_kernel<__nv_bfloat16><<<grid, block, 0, st>>>(c, b, scale, n8, M, static_cast<__nv_bfloat16*>(out));
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? MH3_OK : fail_cuda(e, "mh3_dequantize_fp4 launch");
}
