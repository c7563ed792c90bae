// Product of two microscaled 4-bit matrices (mh3_fp4_gemm) for sm_100a.
//
//   out[m,n] = bf16((sum_k a[m,k] b[n,k] + sum_r a2[m,r] b2[n,r]) * as[m] * bs[n] + bias[n])
//
// a and b are e2m1 codes with an e4m3 scale for 16 of them; as and bs are the
// rows' powers of two, so they factor out of the sum exactly.  Two kernels:
//
// * pair_kernel (M > kSmallM): persistent, a cluster of two CTAs per 256x256 tile,
//   tcgen05.mma.cta_group::2 kind::mxf4nvf4 with the block scales in tensor memory.
//   A stage is 256 elements of K: per CTA 128 rows of A and of B (128 bytes each),
//   2 KB of A's scales and 4 KB of B's (every CTA needs the scales of all 256
//   columns).  Bound: the tensor cores' 4-bit rate and the power limit.
//   Tensor memory (512 columns): one 256-column accumulator and, for each of the
//   five stages, 48 columns of block scales.  A stage's scale columns are rewritten
//   when its shared memory is refilled, which the full barrier already orders after
//   the MMAs that read both; with two accumulators there is room for two scale
//   buffers only, and waiting for the MMAs two stages back cost 11 % (1.18 ms
//   against 1.05 without the wait at 32760 x 13824 x 5120).  Eight epilogue warps take
//   the whole accumulator into registers and hand it over before they scale and
//   store it, so the next tile's MMAs run meanwhile.
// * small_kernel (M <= kSmallM): reads b once.  A CTA takes 16 rows of b, its warps
//   split K; codes are widened to f16 with their block scale (6 significant bits:
//   exact) and multiplied by mma.sync.m16n8k16 with f32 sums.  The weights are the
//   16-row operand, up to 16 tokens the narrow one, and both sides use the same
//   permutation of k, so a lane loads 32 consecutive codes.  Bound: widening the
//   codes (about one instruction each) beside the latency of a chain of a few loads;
//   above 16 rows the pair kernel takes no longer (11.7 us at 17 rows of 5120 x 5120
//   against 9.4 here at 16; 15.6 against 17.3 at 13824 x 5120).

#include <algorithm>
#include <mutex>

#include "fp4.cuh"
#include "mh3_b200.h"
#include "mh3_internal.h"
#include "ptx.cuh"

namespace mh3 {
namespace fp4gemm {

constexpr int NUM_THREADS = 320;
constexpr int EPI_WARPS = 8;
constexpr int STAGES = 5;
constexpr int STAGE_K = 256;                  // elements of K per stage (128 bytes)
constexpr int BM = 256, BN = 256, HALF = 128;  // tile; rows of A and B per CTA
constexpr int TILE_BYTES = HALF * 128;
constexpr int SF_BLOCK = 512;                  // scales of 128 rows x 64 elements
constexpr int EPI_BOX = 32 * 32 * 2;
constexpr int kGroupM = 8;                     // 256-row blocks per raster group
constexpr int SF_COL = 256, SF_COLS = 48;      // scales of a stage: 4 x 4 columns of A, 4 x 8 of B
constexpr int kSmallM = 16;

// A row's scale as the factors before and after the column's, so that no product passes
// f32's range while the result does not: the smaller of 1 and the scale first (a NaN stays in
// the second).  Powers of two: exact.
__device__ __forceinline__ float2 split_scale(float s) { return s <= 1.0f ? make_float2(s, 1.0f) : make_float2(1.0f, s); }

struct Params {
  CUtensorMap tma_a, tma_b;    // bytes (K/2, rows), box (128, 128), 128B swizzle
  CUtensorMap tma_sa, tma_sb;  // words (128, K/64, rows/128), box (128, 4, 1)
  CUtensorMap tma_a2, tma_b2;  // bf16 (R, rows), box (64, 128), 128B swizzle
  CUtensorMap tma_out;         // bf16 (N, M), box (32, 32), 64B swizzle
  int M, N, K, R;
  const float *rs, *cs;
  const __nv_bfloat16* bias;
  int* err;
  unsigned long long timeout_ns;
  int test_flags;
};

struct __align__(1024) Smem {
  uint8_t a[STAGES][TILE_BYTES];
  uint8_t b[STAGES][TILE_BYTES];
  uint8_t sa[STAGES][4 * SF_BLOCK];
  uint8_t sb[STAGES][2][4 * SF_BLOCK];
  uint8_t epi[EPI_WARPS][2][EPI_BOX];
  float col_scale[BN];
  float col_bias[BN];
  uint64_t full[STAGES];  // used in the leader
  uint64_t empty[STAGES];
  uint64_t acc_full;
  uint64_t acc_empty;     // used in the leader: the accumulator is in registers (8 warps x 2 CTAs)
  uint64_t mma_done;
  uint64_t bar_never;     // nothing arrives on it (test hook)
  uint32_t tmem_base;
  int abort_flag;
};

__global__ void __launch_bounds__(NUM_THREADS, 1) pair_kernel(const __grid_constant__ Params p) {
  extern __shared__ uint8_t smem_raw[];
  Smem& sm = *reinterpret_cast<Smem*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const uint32_t crank = cluster_ctarank();
  const int pair = blockIdx.x >> 1;
  const int npairs = gridDim.x >> 1;
  const int num_m = (p.M + BM - 1) / BM;
  const int num_n = (p.N + BN - 1) / BN;
  const int num_tiles = num_m * num_n;
  const int nk64 = (p.K + 63) / 64;
  const int kst_main = (p.K + STAGE_K - 1) / STAGE_K;
  const int kst = kst_main + (p.R + 63) / 64;  // then the low-rank stages, 64 bf16 each

  auto coords = [&](int t, int& mb, int& nb) {
    const int per_group = kGroupM * num_n;
    const int g = t / per_group;
    const int r = t - g * per_group;
    const int gm = min(kGroupM, num_m - g * kGroupM);
    nb = r / gm;
    mb = g * kGroupM + (r - nb * gm);
  };

  if (threadIdx.x == 0) {
    for (int i = 0; i < STAGES; ++i) {
      mbar_init(smem_u32(&sm.full[i]), 1);
      mbar_init(smem_u32(&sm.empty[i]), 1);
    }
    mbar_init(smem_u32(&sm.acc_full), 1);
    mbar_init(smem_u32(&sm.acc_empty), 2 * EPI_WARPS);
    mbar_init(smem_u32(&sm.mma_done), 1);
    mbar_init(smem_u32(&sm.bar_never), 1);
    sm.abort_flag = 0;
    fence_mbar_init();
  }
  if (warp == 1) {
    tmem_alloc_pair(smem_u32(&sm.tmem_base), 512);
    tmem_relinquish_pair();
  }
  tc_fence_before();
  cluster_sync();  // both CTAs' barriers are initialised before any copy or arrive crosses
  tc_fence_after();
  const uint32_t tmem = sm.tmem_base;
  const WaitGuard g{&sm.abort_flag, p.err, p.timeout_ns};

  if (warp == 0) {
    // ---------------------------------------------------------------- producer (both CTAs)
    if (elect_one_sync()) {
      tma_prefetch_desc(&p.tma_a);
      tma_prefetch_desc(&p.tma_b);
      tma_prefetch_desc(&p.tma_sa);
      tma_prefetch_desc(&p.tma_sb);
    }
    __syncwarp();
    int it = 0, last_issued = -1, st = 0;
    uint32_t phase = 1u;
    bool ok = true;
    if (p.test_flags & MH3_TEST_STALL_PRODUCER) {  // a wait that nothing ends runs out first
      bool w = true;
      if (lane == 0) w = mbar_wait(smem_u32(&sm.bar_never), 0, g);
      ok = __shfl_sync(0xffffffffu, w ? 1 : 0, 0) != 0;
    }
    for (int t = pair; t < num_tiles && ok; t += npairs) {
      int mb, nb;
      coords(t, mb, nb);
      const int row_a = mb * BM + (int)crank * HALF;
      const int row_b = nb * BN + (int)crank * HALF;
      for (int s = 0; s < kst; ++s, ++it) {
        bool w = true;
        if (lane == 0) w = mbar_wait(smem_u32(&sm.empty[st]), phase, g);
        if (!__shfl_sync(0xffffffffu, w ? 1 : 0, 0)) {
          ok = false;
          break;
        }
        last_issued = it;
        if (elect_one_sync()) {
          const bool main = s < kst_main;
          // the leader counts both CTAs' copies (clipped boxes are filled and counted whole)
          if (crank == 0)
            mbar_arrive_expect_tx(smem_u32(&sm.full[st]), 2u * (2u * TILE_BYTES + (main ? 12u * SF_BLOCK : 0u)));
          const uint32_t fb = mapa_shared(smem_u32(&sm.full[st]), 0);
          if (main) {
            tma_load_2d_pair(smem_u32(sm.a[st]), &p.tma_a, fb, s * 128, row_a);
            tma_load_2d_pair(smem_u32(sm.b[st]), &p.tma_b, fb, s * 128, row_b);
            tma_load_3d_pair(smem_u32(sm.sa[st]), &p.tma_sa, fb, 0, s * 4, row_a / HALF);
            tma_load_3d_pair(smem_u32(sm.sb[st][0]), &p.tma_sb, fb, 0, s * 4, nb * 2);
            tma_load_3d_pair(smem_u32(sm.sb[st][1]), &p.tma_sb, fb, 0, s * 4, nb * 2 + 1);
          } else {
            tma_load_2d_pair(smem_u32(sm.a[st]), &p.tma_a2, fb, (s - kst_main) * 64, row_a);
            tma_load_2d_pair(smem_u32(sm.b[st]), &p.tma_b2, fb, (s - kst_main) * 64, row_b);
          }
        }
        __syncwarp();
        if (++st == STAGES) {
          st = 0;
          phase ^= 1u;
        }
      }
    }
    // Teardown (leader): the last copies counted on each stage must land.
    if (crank == 0 && lane == 0)
      for (int i = max(0, last_issued - STAGES + 1); i <= last_issued; ++i)
        mbar_wait_teardown(smem_u32(&sm.full[i % STAGES]), (uint32_t)(i / STAGES) & 1u);
  } else if (warp == 1) {
    // ---------------------------------------------------------------- MMA issuer (leader)
    // One thread, and as few instructions per MMA as it takes: its issue is what
    // keeps the tensor cores fed.  With descriptors built per MMA and a division per
    // stage a 512-cycle stage took 750 to 900 cycles; with descriptors that only
    // count up, the twelve scale copies and the commit hide behind the MMAs (513).
    if (crank == 0 && elect_one_sync()) {
      constexpr uint32_t kIdF4 = idesc_nvf4(BM, BN);
      constexpr uint32_t kIdBF = idesc_bf16(BM, BN, false, false);
      const uint64_t da0 = smem_desc(smem_u32(sm.a[0]), 16, 1024, kLayoutSW128);
      const uint64_t db0 = smem_desc(smem_u32(sm.b[0]), 16, 1024, kLayoutSW128);
      const uint64_t dsa0 = smem_desc(smem_u32(sm.sa[0]), 0, 128, kLayoutNone);
      const uint64_t dsb0 = smem_desc(smem_u32(sm.sb[0][0]), 0, 128, kLayoutNone);
      const uint32_t full0 = smem_u32(&sm.full[0]), empty0 = smem_u32(&sm.empty[0]);
      const int tail = nk64 - (kst_main - 1) * 4;  // 64-element steps of the last main stage
      int st = 0;
      uint32_t phase = 0, tphase = 0, fresh = 0;
      uint64_t da = da0, db = db0;  // 16-byte units: 1024 a stage, 2 an MMA
      auto next = [&] {
        mma_commit_pair(empty0 + st * 8, 0x3);
        da += TILE_BYTES / 16;
        db += TILE_BYTES / 16;
        if (++st == STAGES) {
          st = 0;
          phase ^= 1u;
          da = da0;
          db = db0;
        }
      };
      auto main_stage = [&](auto whole, int n, bool first) {
        mbar_wait(full0 + st * 8, phase, g);
        tc_fence_after();
        const uint64_t dsa = dsa0 + (uint64_t)(st * (4 * SF_BLOCK / 16)), dsb = dsb0 + (uint64_t)(st * (8 * SF_BLOCK / 16));
        const uint32_t sfa = tmem + SF_COL + (uint32_t)(st * SF_COLS), sfb = sfa + 16;
#pragma unroll
        for (int kk = 0; kk < 4; ++kk)
          if (decltype(whole)::value || kk < n) {
            tmem_cp_scales_pair(sfa + kk * 4, dsa + kk * (SF_BLOCK / 16));
            tmem_cp_scales_pair(sfb + kk * 8, dsb + kk * (SF_BLOCK / 16));
            tmem_cp_scales_pair(sfb + kk * 8 + 4, dsb + (4 + kk) * (SF_BLOCK / 16));
          }
        if (first && fresh) {  // the epilogue has taken the previous tile
          mbar_wait_cluster(smem_u32(&sm.acc_empty), tphase, g);
          tphase ^= 1u;
          tc_fence_after();
        }
#pragma unroll
        for (int kk = 0; kk < 4; ++kk)
          if (decltype(whole)::value || kk < n)
            mma_nvf4_ss_pair(tmem, da + 2 * kk, db + 2 * kk, kIdF4, sfa + kk * 4, sfb + kk * 8, first && kk == 0 ? 0u : 1u);
        next();
      };
      for (int t = pair; t < num_tiles; t += npairs) {
        const int whole = tail == 4 ? kst_main : kst_main - 1;
        for (int s = 0; s < whole; ++s) main_stage(std::true_type{}, 4, s == 0);
        if (whole < kst_main) main_stage(std::false_type{}, tail, whole == 0);
        for (int s = kst_main; s < kst; ++s) {
          mbar_wait(full0 + st * 8, phase, g);
          tc_fence_after();
#pragma unroll
          for (int kk = 0; kk < 4; ++kk) mma_f16_ss_pair(tmem, da + 2 * kk, db + 2 * kk, kIdBF, 1u);  // 16 bf16 each
          next();
        }
        mma_commit_pair(smem_u32(&sm.acc_full), 0x3);
        fresh = 1u;
      }
      mma_commit_pair(smem_u32(&sm.mma_done), 0x3);
    }
    __syncwarp();
    // Both CTAs: every pair MMA (they write both CTAs' TMEM) must be
    // finished before TMEM is freed, also on the abort path.
    if (lane == 0) mbar_wait_teardown(smem_u32(&sm.mma_done), 0);
    __syncwarp();
  } else {
    // ------------------------------------------------------------------ epilogue (both CTAs)
    const int q = warp & 3;           // TMEM lane quarter of this warp
    const int ew = warp - 2;          // 0..7: warps q and q + 4 of a quarter take a half of the columns each
    const int half = ew >> 2;
    const int et = threadIdx.x - 64;  // 0..255 over the epilogue warps
    const uint32_t base = tmem + ((uint32_t)(q * 32) << 16) + (uint32_t)(half * 128);
    int tcount = 0, buf = 0;
    for (int t = pair; t < num_tiles; t += npairs, ++tcount) {
      int mb, nb;
      coords(t, mb, nb);
      const int n0 = nb * BN;
      named_barrier_sync(1, 32 * EPI_WARPS);  // the last tile's column values have been read
      {
        const int n = n0 + et;
        const bool in = n < p.N;
        sm.col_scale[et] = in ? __ldg(p.cs + n) : 0.0f;
        sm.col_bias[et] = (p.bias != nullptr && in) ? __bfloat162float(p.bias[n]) : 0.0f;
      }
      named_barrier_sync(1, 32 * EPI_WARPS);
      const int m0 = mb * BM + (int)crank * HALF + q * 32;  // first row of this warp's boxes
      const int m = m0 + lane;
      const float2 rsv = split_scale(m < p.M ? __ldg(p.rs + m) : 0.0f);
      mbar_wait(smem_u32(&sm.acc_full), (uint32_t)tcount & 1u, g);
      tc_fence_after();
      uint32_t v[4][32];
#pragma unroll
      for (int c = 0; c < 4; ++c) tmem_ld32(base + (uint32_t)c * 32, v[c]);
      tmem_wait_ld();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive_cluster(mapa_shared(smem_u32(&sm.acc_empty), 0));
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        const int col = half * 128 + c * 32;
        if (n0 + col >= p.N || m0 >= p.M) continue;  // warp-uniform: box wholly outside
        const float* cs = &sm.col_scale[col];
        const float* bs = &sm.col_bias[col];
        uint32_t packed[16];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float4 c4 = *reinterpret_cast<const float4*>(cs + 4 * i);
          const float4 b4 = *reinterpret_cast<const float4*>(bs + 4 * i);
          const __nv_bfloat162 h0 = __floats2bfloat162_rn(fmaf(__uint_as_float(v[c][4 * i + 0]) * rsv.x * c4.x, rsv.y, b4.x),
                                                          fmaf(__uint_as_float(v[c][4 * i + 1]) * rsv.x * c4.y, rsv.y, b4.y));
          const __nv_bfloat162 h1 = __floats2bfloat162_rn(fmaf(__uint_as_float(v[c][4 * i + 2]) * rsv.x * c4.z, rsv.y, b4.z),
                                                          fmaf(__uint_as_float(v[c][4 * i + 3]) * rsv.x * c4.w, rsv.y, b4.w));
          packed[2 * i] = *reinterpret_cast<const uint32_t*>(&h0);
          packed[2 * i + 1] = *reinterpret_cast<const uint32_t*>(&h1);
        }
        if (lane == 0) bulk_wait_group_read<1>();  // the store that last read this box is done
        __syncwarp();
        uint8_t* box = sm.epi[ew][buf];
#pragma unroll
        for (int j = 0; j < 4; ++j)  // 64B swizzle: 16-byte piece j of row ``lane``
          *reinterpret_cast<uint4*>(box + lane * 64 + ((j ^ ((lane >> 1) & 3)) * 16)) =
              make_uint4(packed[4 * j], packed[4 * j + 1], packed[4 * j + 2], packed[4 * j + 3]);
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) {
          tma_store_2d(&p.tma_out, smem_u32(box), n0 + col, m0);
          bulk_commit_group();
        }
        buf ^= 1;
      }
    }
    if (lane == 0) bulk_wait_group<0>();  // stores complete before the CTA's shared memory goes
    __syncwarp();
  }

  tc_fence_before();
  __syncthreads();
  cluster_sync();  // no CTA leaves while its peer may still arrive on or copy into it
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc_pair(tmem, 512);
  }
}

// ---------------------------------------------------------------------------
// Few rows
// ---------------------------------------------------------------------------
// Warps of a CTA, which split K, and its rows of b.  16 rows by 8 warps took 6.9 us at
// one row of 5120 x 5120 (32 rows: 8.1; 4 warps: 10.0) and 13.2 us at 13824 x 5120
// (11.4; 12.4): more rows share a's widening, but leave too few warps per SM.
constexpr int kWarps = 8;
constexpr int kRowsW = 16;

struct SmallParams {
  const void* x;  // FUSED: the rows to round, [M, K] with stride x_s
  long long x_s;
  const uint8_t *a, *sa, *b, *sb;
  const float *rs, *cs;
  const __nv_bfloat16 *bias, *a2, *b2;
  long long lda2, ldb2, ldo;
  __nv_bfloat16* out;
  int M, N, K, R;
};

// 32 codes and their two scales (little endian in ``sf``) as 16 pairs of f16: code * scale, exact.
__device__ __forceinline__ void widen32(const uint4& code, uint32_t sf, uint32_t (&h)[16]) {
  uint32_t s;  // two f16
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(s) : "h"((uint16_t)sf));
  const __half2 s2 = *reinterpret_cast<const __half2*>(&s);
  const __half2 lo = __low2half2(s2), hi = __high2half2(s2);
  const uint32_t w[4] = {code.x, code.y, code.z, code.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    uint32_t t[4];
    fp4::e2m1x8_halves(w[i], t);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const __half2 v = __hmul2(*reinterpret_cast<const __half2*>(&t[j]), i < 2 ? lo : hi);
      h[4 * i + j] = *reinterpret_cast<const uint32_t*>(&v);
    }
  }
}

__device__ __forceinline__ void mma_16x8x16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                            uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// NT: groups of 8 rows of a.  X: void, a is given in 4 bits; or the type of x, which
// every CTA rounds for itself into shared memory while its weights are on their way to
// L2 - one launch and no workspace for the calls where latency counts (8.3 us at one
// row of 5120 x 5120 against 2.3 + 6.9; from three rows on the CTAs' copies of x cost
// more than the launch).
constexpr int kFusedRows = 2;
constexpr int kFusedBytes = 96 * 1024;  // of codes and scales

template <int NT, typename X>
__global__ void __launch_bounds__(kWarps * 32) small_kernel(const __grid_constant__ SmallParams p) {
  constexpr bool FUSED = !std::is_same<X, void>::value;
  __shared__ float red[kWarps][kRowsW][NT * 8 + 1];
  extern __shared__ uint4 own[];  // FUSED: codes [M][K/2], then scales [M][K/16]
  __shared__ uint32_t top[FUSED ? kFusedRows : 1];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int n0 = blockIdx.x * kRowsW;
  const int gr = lane >> 2, q = lane & 3;
  const int units = p.K / 32, nk64 = (p.K + 63) / 64;
  const long long kb = p.K / 2;
  // scale word of 32 codes: two bytes of the row's place in its block of 128
  auto sf_at = [&](int row) { return (long long)(row >> 7) * nk64 * 512 + (row & 31) * 16 + ((row & 127) >> 5) * 4; };
  const uint8_t *w[kRowsW / 8], *sw[kRowsW / 8];  // the lane's rows, 8 apart; those past N are computed and dropped
#pragma unroll
  for (int i = 0; i < kRowsW / 8; ++i) {
    const int r = min(n0 + gr + 8 * i, p.N - 1);
    w[i] = p.b + r * kb;
    sw[i] = p.sb + sf_at(r);
  }
  const uint8_t* xs = reinterpret_cast<const uint8_t*>(own) + p.M * kb;
  float c[kRowsW / 16][NT][4] = {};
  uint4 d[kRowsW / 8];  // a unit's codes and scales
  uint32_t f[kRowsW / 8];
  auto fetch = [&](int u) {
    const long long so = (long long)(u >> 1) * 512 + (u & 1) * 2;
#pragma unroll
    for (int i = 0; i < kRowsW / 8; ++i) {
      d[i] = u < units ? __ldcs(reinterpret_cast<const uint4*>(w[i] + (long long)u * 16)) : make_uint4(0, 0, 0, 0);
      f[i] = u < units ? *reinterpret_cast<const uint16_t*>(sw[i] + so) : 0;
    }
  };
  fetch(warp * 4 + q);
  if constexpr (FUSED) {
    // this CTA's rows of weights towards L2
    const int lines = (int)((kb + 127) / 128);
    for (int i = threadIdx.x; i < kRowsW * lines; i += kWarps * 32) {
      const int row = min(n0 + i / lines, p.N - 1);
      asm volatile("prefetch.global.L2 [%0];" ::"l"(p.b + row * kb + (long long)(i % lines) * 128));
    }
    const int nb = p.K / 16, total = p.M * nb;
    const X* x = static_cast<const X*>(p.x);
    const bool vec = (reinterpret_cast<uintptr_t>(p.x) & 15u) == 0 && p.x_s * (long long)sizeof(X) % 16 == 0;
    if ((int)threadIdx.x < p.M) top[threadIdx.x] = 0;
    __syncthreads();
    uint32_t most[kFusedRows] = {};
    for (int b = threadIdx.x; b < nb; b += kWarps * 32)
#pragma unroll
      for (int m = 0; m < kFusedRows; ++m)
        if (m < p.M) {
          float2 v[8];
          fp4::load16(x + m * p.x_s + b * 16, v, vec);
          most[m] = max(most[m], fp4::absmax16(v));
        }
#pragma unroll
    for (int m = 0; m < kFusedRows; ++m)
      if (m < p.M) {
        most[m] = __reduce_max_sync(0xffffffffu, most[m]);
        if (lane == 0) atomicMax(&top[m], most[m]);
      }
    __syncthreads();
    for (int i = threadIdx.x; i < total; i += kWarps * 32) {
      const int m = i / nb, b = i - m * nb;
      uint2 code = make_uint2(0, 0);
      uint32_t s8 = 0;
      if (top[m] < 0x7f800000u) {
        float2 v[8];
        fp4::load16(x + m * p.x_s + b * 16, v, vec);
        s8 = fp4::round_block(v, fp4::absmax16(v), fp4::row_exponent(top[m]), code);
      }
      reinterpret_cast<uint2*>(own)[i] = code;
      const_cast<uint8_t*>(xs)[i] = (uint8_t)s8;
    }
    __syncthreads();
  }
  for (int u = warp * 4 + q; u - q < units; u += kWarps * 4) {
    uint32_t hx[NT][16];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      uint4 dx = make_uint4(0, 0, 0, 0);
      uint32_t fx = 0;
      const int row = t * 8 + gr;
      if (u < units && row < p.M) {
        if constexpr (FUSED) {
          dx = own[row * units + u];
          fx = *reinterpret_cast<const uint16_t*>(xs + (row * units + u) * 2);
        } else {
          dx = *reinterpret_cast<const uint4*>(p.a + row * kb + (long long)u * 16);
          fx = *reinterpret_cast<const uint16_t*>(p.sa + sf_at(row) + (long long)(u >> 1) * 512 + (u & 1) * 2);
        }
      }
      widen32(dx, fx, hx[t]);
    }
#pragma unroll
    for (int i = 0; i < kRowsW / 16; ++i) {
      uint32_t h0[16], h1[16];
      widen32(d[2 * i], f[2 * i], h0);
      widen32(d[2 * i + 1], f[2 * i + 1], h1);
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int j = 0; j < 8; ++j)
          mma_16x8x16(c[i][t], h0[2 * j], h1[2 * j], h0[2 * j + 1], h1[2 * j + 1], hx[t][2 * j], hx[t][2 * j + 1]);
    }
    fetch(u + kWarps * 4);
  }
#pragma unroll
  for (int i = 0; i < kRowsW / 16; ++i)
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      float* r0 = &red[warp][16 * i + gr][t * 8 + q * 2];
      float* r1 = &red[warp][16 * i + gr + 8][t * 8 + q * 2];
      r0[0] = c[i][t][0];
      r0[1] = c[i][t][1];
      r1[0] = c[i][t][2];
      r1[1] = c[i][t][3];
    }
  __syncthreads();
  for (int i = threadIdx.x; i < kRowsW * NT * 8; i += kWarps * 32) {
    const int j = i % kRowsW, m = i / kRowsW, n = n0 + j;
    if (m >= p.M || n >= p.N) continue;
    float s = 0.0f;
#pragma unroll
    for (int k = 0; k < kWarps; ++k) s += red[k][j][m];
    for (int r = 0; r < p.R; ++r)
      s = fmaf(__bfloat162float(p.a2[m * p.lda2 + r]), __bfloat162float(p.b2[n * p.ldb2 + r]), s);
    float rs;
    if constexpr (FUSED) rs = top[m] < 0x7f800000u ? fp4::pow2f(fp4::row_exponent(top[m])) : __uint_as_float(0x7fffffffu);
    else rs = p.rs[m];
    const float b = p.bias != nullptr ? __bfloat162float(p.bias[n]) : 0.0f;
    const float2 r2 = split_scale(rs);
    p.out[m * p.ldo + n] = __float2bfloat16_rn(fmaf(s * r2.x * p.cs[n], r2.y, b));
  }
}

constexpr uint32_t smem_bytes() { return (uint32_t)sizeof(Smem) + 1024; }
static_assert(smem_bytes() <= 227 * 1024, "shared memory");

static cudaError_t launch_pair(const Params& p, cudaStream_t st) {
  // per device: the attribute and the number of resident pairs belong to it
  constexpr int kMaxDevices = 64;
  static int max_pairs[kMaxDevices] = {};
  static std::mutex mu;
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  if (dev < 0 || dev >= kMaxDevices) return cudaErrorInvalidDevice;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(2, 1, 1);
  cfg.blockDim = dim3(NUM_THREADS, 1, 1);
  cfg.dynamicSmemBytes = smem_bytes();
  cfg.stream = st;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = 2;
  at[0].val.clusterDim.y = 1;
  at[0].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  int pairs_max = 0;
  {
    std::lock_guard<std::mutex> lock(mu);
    if (max_pairs[dev] == 0) {
      e = cudaFuncSetAttribute(pair_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem_bytes());
      if (e != cudaSuccess) return e;
      int nsm = 0;
      e = cudaDeviceGetAttribute(&nsm, cudaDevAttrMultiProcessorCount, dev);
      if (e != cudaSuccess) return e;
      cfg.gridDim = dim3((unsigned)(nsm & ~1), 1, 1);
      // Persistent: no more pairs than can be resident at once (a pair needs two
      // SMs of one GPC, so this can be below nsm/2).
      int n = 0;
      if (cudaOccupancyMaxActiveClusters(&n, pair_kernel, &cfg) != cudaSuccess || n <= 0) {
        cudaGetLastError();
        n = nsm / 2;
      }
      max_pairs[dev] = n;
    }
    pairs_max = max_pairs[dev];
  }
  const long long tiles = (long long)((p.M + BM - 1) / BM) * ((p.N + BN - 1) / BN);
  cfg.gridDim = dim3((unsigned)(2 * std::min<long long>(tiles, pairs_max)), 1, 1);
  return cudaLaunchKernelEx(&cfg, pair_kernel, p);
}

static int map_rows(CUtensorMap* map, CUtensorMapDataType type, int es, const void* base, long long inner, long long rows,
                    long long pitch_bytes) {
  const cuuint64_t dims[2] = {(cuuint64_t)inner, (cuuint64_t)rows};
  const cuuint64_t strides[1] = {(cuuint64_t)pitch_bytes};
  const cuuint32_t box[2] = {(cuuint32_t)(128 / es), (cuuint32_t)HALF};
  const cuuint32_t estr[2] = {1u, 1u};
  return encode_tiled(map, type, 2, const_cast<void*>(base), dims, strides, box, estr, CU_TENSOR_MAP_SWIZZLE_128B);
}

static int map_scales(CUtensorMap* map, const void* base, long long K, long long rows) {
  const long long nk64 = (K + 63) / 64;
  const cuuint64_t dims[3] = {128, (cuuint64_t)nk64, (cuuint64_t)((rows + 127) / 128)};
  const cuuint64_t strides[2] = {SF_BLOCK, (cuuint64_t)(nk64 * SF_BLOCK)};
  const cuuint32_t box[3] = {128, 4, 1};
  const cuuint32_t estr[3] = {1u, 1u, 1u};
  return encode_tiled(map, CU_TENSOR_MAP_DATA_TYPE_UINT32, 3, const_cast<void*>(base), dims, strides, box, estr,
                      CU_TENSOR_MAP_SWIZZLE_NONE);
}

static cudaError_t launch_small(const SmallParams& p, cudaStream_t st) {
  const unsigned grid = (unsigned)((p.N + kRowsW - 1) / kRowsW);
  if (p.M <= 8) small_kernel<1, void><<<grid, kWarps * 32, 0, st>>>(p);
  else small_kernel<2, void><<<grid, kWarps * 32, 0, st>>>(p);
  return cudaGetLastError();
}

// Whether a linear of M rows runs as one launch.
static bool fused(long long M, long long K) { return M <= kFusedRows && M * (K / 2 + K / 16) <= kFusedBytes; }

template <typename X>
static cudaError_t launch_fused(const SmallParams& p, cudaStream_t st) {
  const size_t smem = (size_t)p.M * (p.K / 2 + p.K / 16);
  if (smem > 32 * 1024) {  // with the static part, past the 48 KB default
    const cudaError_t e = allow_smem<small_kernel<1, X>>(kFusedBytes);
    if (e != cudaSuccess) return e;
  }
  small_kernel<1, X><<<(unsigned)((p.N + kRowsW - 1) / kRowsW), kWarps * 32, smem, st>>>(p);
  return cudaGetLastError();
}

}  // namespace fp4gemm
}  // namespace mh3

using namespace mh3;

extern "C" int mh3_fp4_gemm(const mh3_fp4_gemm_args* a, void* stream) {
  const mh3::NvtxRange nvtx_range("mh3_fp4_gemm");
  if (a == nullptr) return fail(MH3_ERR_INVALID, "mh3_fp4_gemm: null args");
  if (a->M < 0 || a->N <= 0 || a->K <= 0 || a->R < 0) return fail(MH3_ERR_INVALID, "mh3_fp4_gemm: sizes must be positive");
  if (a->K % 32) return fail(MH3_ERR_INVALID, "mh3_fp4_gemm: K must be a multiple of 32");
  if (a->N % 8 || a->ldo % 8 || a->ldo < a->N) return fail(MH3_ERR_INVALID, "mh3_fp4_gemm: N and ldo must be multiples of 8, ldo >= N");
  if (a->M > 0x7fffff00LL || a->N > 0x7fffff00LL || a->K > (1ll << 30) || a->R > (1ll << 20))
    return fail(MH3_ERR_TOO_LARGE, "mh3_fp4_gemm: dimension too large");
  if (a->M == 0) return MH3_OK;
  if (((a->M + 255) / 256) * ((a->N + 255) / 256) > 0x7fff0000LL) return fail(MH3_ERR_TOO_LARGE, "mh3_fp4_gemm: too many tiles");
  if (!a->a || !a->a_blocks || !a->a_scale || !a->b || !a->b_blocks || !a->b_scale || !a->out)
    return fail(MH3_ERR_INVALID, "mh3_fp4_gemm: null pointer");
  auto al16 = [](const void* p_) { return ((uintptr_t)p_ & 15u) == 0; };
  if (!al16(a->a) || !al16(a->a_blocks) || !al16(a->b) || !al16(a->b_blocks) || !al16(a->out))
    return fail(MH3_ERR_INVALID, "mh3_fp4_gemm: operands and out must be 16-byte aligned");
  if (a->R > 0) {
    if (!a->a2 || !a->b2) return fail(MH3_ERR_INVALID, "mh3_fp4_gemm: R > 0 needs a2 and b2");
    if (a->R % 8 || a->lda2 % 8 || a->ldb2 % 8 || !al16(a->a2) || !al16(a->b2) || a->lda2 < a->R || a->ldb2 < a->R)
      return fail(MH3_ERR_INVALID, "mh3_fp4_gemm: R and the strides of a2/b2 must be multiples of 8, 16-byte aligned");
  }
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  cudaError_t e;
  if (a->M <= fp4gemm::kSmallM) {
    fp4gemm::SmallParams p = {};
    p.a = static_cast<const uint8_t*>(a->a);
    p.sa = static_cast<const uint8_t*>(a->a_blocks);
    p.b = static_cast<const uint8_t*>(a->b);
    p.sb = static_cast<const uint8_t*>(a->b_blocks);
    p.rs = a->a_scale;
    p.cs = a->b_scale;
    p.bias = static_cast<const __nv_bfloat16*>(a->bias);
    p.a2 = static_cast<const __nv_bfloat16*>(a->a2);
    p.b2 = static_cast<const __nv_bfloat16*>(a->b2);
    p.lda2 = a->lda2;
    p.ldb2 = a->ldb2;
    p.ldo = a->ldo;
    p.out = static_cast<__nv_bfloat16*>(a->out);
    p.M = (int)a->M;
    p.N = (int)a->N;
    p.K = (int)a->K;
    p.R = (int)a->R;
    e = fp4gemm::launch_small(p, st);
  } else {
    fp4gemm::Params p;
    memset(&p, 0, sizeof(p));
    int rc = fp4gemm::map_rows(&p.tma_a, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, a->a, a->K / 2, a->M, a->K / 2);
    if (!rc) rc = fp4gemm::map_rows(&p.tma_b, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, a->b, a->K / 2, a->N, a->K / 2);
    if (!rc) rc = fp4gemm::map_scales(&p.tma_sa, a->a_blocks, a->K, a->M);
    if (!rc) rc = fp4gemm::map_scales(&p.tma_sb, a->b_blocks, a->K, a->N);
    if (!rc && a->R > 0) rc = fp4gemm::map_rows(&p.tma_a2, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, a->a2, a->R, a->M, a->lda2 * 2);
    if (!rc && a->R > 0) rc = fp4gemm::map_rows(&p.tma_b2, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, a->b2, a->R, a->N, a->ldb2 * 2);
    if (rc) return rc;
    const cuuint64_t dims[2] = {(cuuint64_t)a->N, (cuuint64_t)a->M};
    const cuuint64_t strides[1] = {(cuuint64_t)(a->ldo * 2)};
    const cuuint32_t box[2] = {32u, 32u};
    const cuuint32_t estr[2] = {1u, 1u};
    rc = encode_tiled(&p.tma_out, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, a->out, dims, strides, box, estr,
                      CU_TENSOR_MAP_SWIZZLE_64B);
    if (rc) return rc;
    p.M = (int)a->M;
    p.N = (int)a->N;
    p.K = (int)a->K;
    p.R = (int)a->R;
    p.rs = a->a_scale;
    p.cs = a->b_scale;
    p.bias = static_cast<const __nv_bfloat16*>(a->bias);
    p.err = a->err ? a->err : device_error_word();
    p.timeout_ns = a->timeout_ns ? a->timeout_ns : 4000000000ull;
    p.test_flags = a->test_flags;
    e = fp4gemm::launch_pair(p, st);
  }
  return e == cudaSuccess ? MH3_OK : fail_cuda(e, "mh3_fp4_gemm launch");
}

extern "C" uint64_t mh3_fp4_linear_workspace_bytes(int64_t M, int64_t K) {
  if (M <= 0 || K <= 0 || fp4gemm::fused(M, K)) return 0;
  // codes, block scales, row scales, each on a 16-byte boundary
  return (uint64_t)M * (uint64_t)(K / 2) + mh3_fp4_block_bytes(M, K) + ((uint64_t)M * 4 + 15) / 16 * 16;
}

extern "C" int mh3_fp4_linear(const void* x, int64_t x_stride, int32_t in_dtype, int64_t M, int64_t N, int64_t K,
                              const void* w4, const void* w_blocks, const float* w_scale, const void* bias, void* out,
                              int64_t ldo, void* workspace, void* stream) {
  const mh3::NvtxRange nvtx_range("mh3_fp4_linear");
  if (M < 0 || N <= 0 || K <= 0 || K % 32) return fail(MH3_ERR_INVALID, "mh3_fp4_linear: K must be a positive multiple of 32");
  if (in_dtype != MH3_DTYPE_BF16 && in_dtype != MH3_DTYPE_F16 && in_dtype != MH3_DTYPE_F32)
    return fail(MH3_ERR_INVALID, "mh3_fp4_linear: in_dtype must be bf16, f16 or f32");
  mh3_fp4_gemm_args g;
  memset(&g, 0, sizeof(g));
  g.M = M;
  g.N = N;
  g.K = K;
  g.b = w4;
  g.b_blocks = w_blocks;
  g.b_scale = w_scale;
  g.bias = bias;
  g.out = out;
  g.ldo = ldo;
  if (M == 0 || !fp4gemm::fused(M, K)) {
    uint8_t* ws = static_cast<uint8_t*>(workspace);
    if (M > 0 && (!ws || ((uintptr_t)ws & 15u)))
      return fail(MH3_ERR_INVALID, "mh3_fp4_linear: needs a 16-byte aligned workspace");
    g.a = ws;
    g.a_blocks = ws + M * (K / 2);
    g.a_scale = reinterpret_cast<const float*>(ws + M * (K / 2) + mh3_fp4_block_bytes(M, K));
    const int rc = mh3_quantize_fp4(x, x_stride, in_dtype, M, K, ws, ws + M * (K / 2),
                                    reinterpret_cast<float*>(ws + M * (K / 2) + mh3_fp4_block_bytes(M, K)), stream);
    return rc ? rc : mh3_fp4_gemm(&g, stream);
  }
  if (N % 8 || ldo % 8 || ldo < N) return fail(MH3_ERR_INVALID, "mh3_fp4_linear: N and ldo must be multiples of 8, ldo >= N");
  if (N > 0x7fffff00LL || K > (1ll << 30)) return fail(MH3_ERR_TOO_LARGE, "mh3_fp4_linear: dimension too large");
  if (!x || !w4 || !w_blocks || !w_scale || !out) return fail(MH3_ERR_INVALID, "mh3_fp4_linear: null pointer");
  if (((uintptr_t)w4 & 15u) || ((uintptr_t)w_blocks & 15u) || ((uintptr_t)out & 15u))
    return fail(MH3_ERR_INVALID, "mh3_fp4_linear: the weight and out must be 16-byte aligned");
  fp4gemm::SmallParams p = {};
  p.x = x;
  p.x_s = x_stride;
  p.b = static_cast<const uint8_t*>(w4);
  p.sb = static_cast<const uint8_t*>(w_blocks);
  p.cs = w_scale;
  p.bias = static_cast<const __nv_bfloat16*>(bias);
  p.out = static_cast<__nv_bfloat16*>(out);
  p.ldo = ldo;
  p.M = (int)M;
  p.N = (int)N;
  p.K = (int)K;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  const cudaError_t e = in_dtype == MH3_DTYPE_BF16 ? fp4gemm::launch_fused<__nv_bfloat16>(p, st)
                        : in_dtype == MH3_DTYPE_F16 ? fp4gemm::launch_fused<__half>(p, st)
                                                    : fp4gemm::launch_fused<float>(p, st);
  return e == cudaSuccess ? MH3_OK : fail_cuda(e, "mh3_fp4_linear launch");
}
