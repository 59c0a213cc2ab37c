// Block-scaled matrix product of e4m3 operands,
//   y[m][n] = sum_j sa[m][j] * sb[n / 128][j] * sum_{k in block j} a[m][k] b[n][k] + bias[n].
//
// The scales change every 128 k's, so a block's sum leaves the tensor core before
// the next one is added: each block of 128 k's is one accumulation in TMEM, which
// the epilogue warps read, scale and add to a running total in fp32 registers
// while the tensor core works on the next block in another TMEM buffer.
#include <cuda.h>

#include <algorithm>
#include <atomic>

#include "blocks.cuh"
#include "ptx.cuh"

namespace ob2 {
namespace {
// Waits without a result: after a wait that gave up (status and abort flag set) the
// ones behind it return within a millisecond each, and the kernel runs on, over
// whatever its buffers hold, to its end.  No branch on the outcome, and polling before
// sleeping: both sit on the round trip between the MMAs and the epilogue that bounds
// the products.
__device__ __forceinline__ void bar_wait(uint32_t bar, uint32_t parity, volatile int* abort_flag, int* status) {
  for (int i = 0; i < 64; ++i)
    if (mbar_try_wait(bar, parity)) return;
  mbar_wait(bar, parity, abort_flag, status);
}
__device__ __forceinline__ bool elect_one() {
  uint32_t p;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "elect.sync _|p, 0xffffffff;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(p));
  return p != 0;
}


// ---------------------------------------------------------------- CUDA cores
// Operands that TMA cannot read (row strides or pointers off the 16-byte grid):
// 64 x 64 outputs per block, 4 x 4 per thread; the products of a block of 128
// k's are summed in fp32, then scaled and added to the total.  2048 x 2048 x 2049: 762
// us, 22.6 TFLOP/s.
template <typename T>
__global__ void __launch_bounds__(256) matmul_blocks_simt_kernel(const MatmulBlocksArgs p) {
  __shared__ float sa[32][65], sb[32][65];
  pdl_begin();
  const int tiles_n = (p.n + 63) / 64;
  const int m0 = blockIdx.x / tiles_n * 64, n0 = blockIdx.x % tiles_n * 64;
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  float tot[4][4] = {};
  for (int kb = 0; kb * kQBlock < p.k; ++kb) {
    float acc[4][4] = {};
    for (int k0 = kb * kQBlock; k0 < min(p.k, (kb + 1) * kQBlock); k0 += 32) {
      for (int i = threadIdx.x; i < 64 * 32; i += 256) {
        const int r = i >> 5, c = i & 31;
        const int k = k0 + c;
        sa[c][r] = m0 + r < p.m && k < p.k ? from_e4m3(p.a[(int64_t)(m0 + r) * p.lda + k]) : 0.f;
        sb[c][r] = n0 + r < p.n && k < p.k ? from_e4m3(p.b[(int64_t)(n0 + r) * p.ldb + k]) : 0.f;
      }
      __syncthreads();
#pragma unroll 8
      for (int c = 0; c < 32; ++c)
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int j = 0; j < 4; ++j) acc[i][j] = fmaf(sa[c][ty * 4 + i], sb[c][tx * 4 + j], acc[i][j]);
      __syncthreads();
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int m = m0 + ty * 4 + i;
      const float s = m < p.m ? p.as[m * p.as_row + kb * p.as_block] : 0.f;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int n = n0 + tx * 4 + j;
        const float f = n < p.n ? s * p.bs[(n / kQBlock) * p.bs_row + kb * p.bs_block] : 0.f;
        tot[i][j] = fmaf(acc[i][j], f, tot[i][j]);
      }
    }
  }
  T* y = static_cast<T*>(p.y);
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int m = m0 + ty * 4 + i, n = n0 + tx * 4 + j;
      if (m < p.m && n < p.n) {
        float v = tot[i][j] + (p.bias ? p.bias[n] : 0.f);
        if (p.relu) v = v < 0.f ? 0.f : v;  // NaN stays NaN
        y[m * p.ldy + n] = from_f32<T>(v);
      }
    }
}

// ---------------------------------------------------------------- one or two rows
// A single decoding step reads every byte of b once for one or two products per
// byte: CUDA cores nearly keep up with HBM, without the tensor core's set-up or a join
// over CTAs.  A warp takes two rows of b, 16 bytes per lane and load, eight loads in
// flight; a is turned into fp16 (exact) once per block, and products are fused into
// fp32 sums of 16, which are scaled and added.  The mixed fp16 -> fp32 fused
// multiply-adds run at a quarter of the fp32 rate: 1 x 4096 x 4096 takes 6.7 us (17
// MB; 8.1 in the kernel for few rows), 1 x 8192 x 8192 15.0 us (4.5 TB/s), 2 x 4096 x
// 4096 8.2 us, and four rows 10.9, more than below.
constexpr int kVecWarps = 8, kVecRows = 2, kVecUnroll = 4;
template <typename T, int M>
__global__ void __launch_bounds__(kVecWarps * 32) matmul_blocks_vec_kernel(const MatmulBlocksArgs p) {
  extern __shared__ uint4 va[];  // [M][2][chunks] eight fp16 of a; then [M][blocks] scales
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int chunks = (p.k + 15) / 16, kbs = (p.k + kQBlock - 1) / kQBlock;
  float* sc = reinterpret_cast<float*>(va + M * 2 * chunks);
  const int n0 = (blockIdx.x * kVecWarps + warp) * kVecRows;
  pdl_begin();

  // 16 bytes of a row of k, zeros behind its end
  auto load16 = [&](const uint8_t* row, int c) {
    if (c * 16 + 16 <= p.k) return *reinterpret_cast<const uint4*>(row + c * 16);
    uint32_t w[4] = {0, 0, 0, 0};
    for (int i = c * 16; i < p.k; ++i) w[(i & 15) >> 2] |= (uint32_t)row[i] << (8 * (i & 3));
    return make_uint4(w[0], w[1], w[2], w[3]);
  };
  // Steps of 512 k's (16 bytes a lane) that lie whole in a row: a ring of kVecUnroll
  // of them is in flight, refilled as each is used up.
  const int steps = p.k / 512;
  const uint8_t* rows[kVecRows];
#pragma unroll
  for (int r = 0; r < kVecRows; ++r) rows[r] = p.b + (int64_t)min(n0 + r, p.n - 1) * p.ldb;
  uint4 w[kVecUnroll][kVecRows];
  auto fetch = [&](int u, int step) {
#pragma unroll
    for (int r = 0; r < kVecRows; ++r) w[u][r] = *reinterpret_cast<const uint4*>(rows[r] + step * 512 + lane * 16);
  };
#pragma unroll
  for (int u = 0; u < kVecUnroll; ++u)
    if (u < steps) fetch(u, u);
  for (int i = threadIdx.x; i < M * chunks; i += kVecWarps * 32) {
    const int m = i / chunks, c = i - m * chunks;
    const uint4 q = m < p.m ? load16(p.a + m * p.lda, c) : make_uint4(0, 0, 0, 0);
    va[(m * 2) * chunks + c] = make_uint4(e4m3x2_to_f16x2(q.x), e4m3x2_to_f16x2(q.x >> 16), e4m3x2_to_f16x2(q.y),
                                          e4m3x2_to_f16x2(q.y >> 16));
    va[(m * 2 + 1) * chunks + c] = make_uint4(e4m3x2_to_f16x2(q.z), e4m3x2_to_f16x2(q.z >> 16), e4m3x2_to_f16x2(q.w),
                                              e4m3x2_to_f16x2(q.w >> 16));
  }
  const float* bs = p.bs + (int64_t)(blockIdx.x * (kVecWarps * kVecRows) / kQBlock) * p.bs_row;
  for (int i = threadIdx.x; i < M * kbs; i += kVecWarps * 32) {
    const int m = i / kbs, kb = i - m * kbs;
    sc[i] = m < p.m ? p.as[m * p.as_row + kb * p.as_block] * bs[kb * p.bs_block] : 0.f;
  }
  __syncthreads();

  float acc[kVecRows][M] = {};
  auto add = [&](const uint4 (&q4)[kVecRows], int c) {  // chunk c of 16 k's
    uint32_t h[kVecRows][8];
#pragma unroll
    for (int r = 0; r < kVecRows; ++r) {
      const uint32_t q[4] = {q4[r].x, q4[r].y, q4[r].z, q4[r].w};
#pragma unroll
      for (int i = 0; i < 8; ++i) h[r][i] = e4m3x2_to_f16x2(i & 1 ? q[i / 2] >> 16 : q[i / 2]);
    }
#pragma unroll
    for (int m = 0; m < M; ++m) {
      const uint4 lo = va[(m * 2) * chunks + c], hi = va[(m * 2 + 1) * chunks + c];
      const uint32_t x[8] = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
      const float s = sc[m * kbs + c / 8];
#pragma unroll
      for (int r = 0; r < kVecRows; ++r) {
        float d = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) d = fma_f16x2(x[i], h[r][i], d);
        acc[r][m] = fmaf(d, s, acc[r][m]);
      }
    }
  };
  for (int s0 = 0; s0 < steps; s0 += kVecUnroll) {
#pragma unroll
    for (int u = 0; u < kVecUnroll; ++u) {
      if (s0 + u >= steps) break;
      add(w[u], (s0 + u) * 32 + lane);
      if (s0 + u + kVecUnroll < steps) fetch(u, s0 + u + kVecUnroll);
    }
  }
  if (steps * 32 + lane < chunks) {
    uint4 q[kVecRows];
#pragma unroll
    for (int r = 0; r < kVecRows; ++r) q[r] = load16(rows[r], steps * 32 + lane);
    add(q, steps * 32 + lane);
  }
#pragma unroll
  for (int r = 0; r < kVecRows; ++r)
#pragma unroll
    for (int m = 0; m < M; ++m) {
      float v = acc[r][m];
#pragma unroll
      for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
      const int n = n0 + r;
      if (lane == r * M + m && n < p.n && m < p.m) {
        if (p.bias) v += p.bias[n];
        if (p.relu) v = v < 0.f ? 0.f : v;  // NaN stays NaN
        static_cast<T*>(p.y)[m * p.ldy + n] = from_f32<T>(v);
      }
    }
}

// ---------------------------------------------------------------- few rows
// Three to 64 rows of a.  They are the MMA's N and the weights its M: a tile is 128
// rows of b by all rows of a (BN >= m), so a handful of tokens wastes no tensor-core
// rows and y's columns (n) lie along the lanes, whose stores are then contiguous.
// The k range is split over the CTAs of a cluster; each leaves its partial sums in
// shared memory, and the sums are joined in rank order over distributed shared
// memory: one launch, no workspace, the same bits every time.  Bound by HBM with
// many weights (16 x 14336 x 4096, 59 MB: 15.0 us, 3.9 TB/s), by the start of its
// CTAs and the join with few (16 x 4096 x 4096: 8.7 us, of which 2.6 are bytes).
template <int BN>
struct RowsLayout {
  static constexpr int kStages = BN == 16 ? 5 : 4;          // two CTAs per SM: at most 113 KB each
  static constexpr int kW = 128 * 128, kX = BN * 128, kStage = kW + kX;
  static constexpr int kCols = 256;                         // two CTAs per SM share 512
  static constexpr int kBufs = kCols / BN;                  // accumulators: the MMAs rarely wait for the epilogue
  static constexpr int kChunk = 1024 / BN;                  // k-blocks whose scales are staged at once
  static constexpr int kOffScale = kStages * kStage;        // 2 x kChunk x BN floats
  static constexpr int kOffBar = kOffScale + 2 * 4096;
  static constexpr int kBars = 2 * kStages + 2 * kBufs + 1;
  static constexpr int kOffMisc = kOffBar + 8 * kBars;
  static constexpr int kBytes = kOffMisc + 16 + 1024;       // base rounded up to 1024
  static_assert(BN * 128 * 4 <= kStages * kStage, "partial sums reuse the stages");
};
constexpr int kRowsThreads = 192;  // 4 epilogue warps, TMA, MMA

template <typename T, int BN>
__global__ void __launch_bounds__(kRowsThreads, 2)
    matmul_blocks_rows_kernel(const __grid_constant__ MatmulBlocksArgs p, const __grid_constant__ CUtensorMap tm_w,
                              const __grid_constant__ CUtensorMap tm_x, int split) {
  using L = RowsLayout<BN>;
  constexpr int ST = L::kStages, NB = L::kBufs, CH = L::kChunk;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw = smem_u32(smem_raw);
  const uint32_t base = (raw + 1023u) & ~1023u;
  uint8_t* gbase = smem_raw + (base - raw);
  const uint32_t bar0 = base + L::kOffBar;
  auto full = [&](int s) { return bar0 + 8u * s; };
  auto empty = [&](int s) { return bar0 + 8u * (ST + s); };
  auto acc_full = [&](int b) { return bar0 + 8u * (2 * ST + b); };
  auto acc_empty = [&](int b) { return bar0 + 8u * (2 * ST + NB + b); };
  const uint32_t drain = bar0 + 8u * (2 * ST + 2 * NB);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(gbase + L::kOffMisc);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(gbase + L::kOffMisc + 4);

  // (a shuffle tells the compiler that it is the same in all lanes: TMEM addresses and
  // barriers then stay in uniform registers)
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int s = 0; s < ST; ++s) {
      mbar_init(full(s), 1);
      mbar_init(empty(s), 1);
    }
    for (int b = 0; b < NB; ++b) {
      mbar_init(acc_full(b), 1);
      mbar_init(acc_empty(b), 4);
    }
    mbar_init(drain, 1);
    *abort_flag = 0;
    fence_mbarrier_init();
  }
  if (warp == 5) {
    tmem_alloc(smem_u32(tmem_slot), L::kCols);
    tmem_relinquish();
  }
  if (warp == 4 && lane == 0) {
    prefetch_tmap(&tm_w);
    prefetch_tmap(&tm_x);
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  pdl_begin();

  const int rank = blockIdx.x % split;
  const int n0 = blockIdx.x / split * 128;
  const int kbs = (p.k + kQBlock - 1) / kQBlock;
  const int kb0 = (int)((int64_t)kbs * rank / split), kb1 = (int)((int64_t)kbs * (rank + 1) / split);
  const int nkb = kb1 - kb0;

  float acc[BN];  // epilogue threads: row n0 + threadIdx.x, one column per token
  if (warp < 4) {
#pragma unroll
    for (int j = 0; j < BN; ++j) acc[j] = 0.f;
    // Scales of CH k-blocks at a time, sa * sb, 8 values per thread: loaded a
    // chunk ahead into registers, shared through one of two buffers.
    float* sc = reinterpret_cast<float*>(gbase + L::kOffScale);
    const float* bs = p.bs + (n0 / kQBlock) * p.bs_row;
    float nxt[8];
    auto load_scales = [&](int c) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int idx = i * 128 + threadIdx.x;
        const int kb = kb0 + c * CH + idx / BN, m = idx % BN;
        nxt[i] = kb < kb1 && m < p.m ? p.as[m * p.as_row + kb * p.as_block] * bs[kb * p.bs_block] : 0.f;
      }
    };
    load_scales(0);
    const uint32_t lane_addr = tmem + ((uint32_t)(warp * 32) << 16);
    for (int it = 0; it < nkb; ++it) {
      const int c = it / CH;
      float* buf = sc + (c & 1) * 1024;
      if (it % CH == 0) {
        // the buffer's readers of chunk c - 2 passed the barrier of chunk c - 1
#pragma unroll
        for (int i = 0; i < 8; ++i) buf[i * 128 + threadIdx.x] = nxt[i];
        named_bar_sync(128);
        if ((c + 1) * CH < nkb) load_scales(c + 1);
      }
      const int b = it % NB;
      bar_wait(acc_full(b), (it / NB) & 1, abort_flag, p.status);
      __syncwarp();
      tc_fence_after();
      uint32_t r[BN / 16][16];
#pragma unroll
      for (int g = 0; g < BN / 16; ++g) tmem_ld_32x32b_x16(lane_addr + b * BN + g * 16, r[g]);
      const float4* s4 = reinterpret_cast<const float4*>(buf + it % CH * BN);
      tmem_ld_wait();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(acc_empty(b));
#pragma unroll
      for (int q = 0; q < BN / 4; ++q) {
        const float4 s = s4[q];
        const uint32_t* d = r[q / 4] + q % 4 * 4;
        float* a = acc + q * 4;
        a[0] = fmaf(__uint_as_float(d[0]), s.x, a[0]);
        a[1] = fmaf(__uint_as_float(d[1]), s.y, a[1]);
        a[2] = fmaf(__uint_as_float(d[2]), s.z, a[2]);
        a[3] = fmaf(__uint_as_float(d[3]), s.w, a[3]);
      }
    }
  } else if (warp == 4) {
    if (lane == 0) {
      int it = 0;
      for (; it < nkb; ++it) {
        const int s = it % ST;
        if (!mbar_wait(empty(s), ((it / ST) & 1) ^ 1, abort_flag, p.status)) break;
        mbar_arrive_expect_tx(full(s), L::kStage);
        const uint32_t dst = base + s * L::kStage;
        tma_load_2d(dst, &tm_w, (kb0 + it) * kQBlock, n0, full(s));
        tma_load_2d(dst + L::kW, &tm_x, (kb0 + it) * kQBlock, 0, full(s));
      }
      // every copy has landed before the CTA may exit
      volatile int no_abort = 0;
      for (int i = max(0, it - ST); i < it; ++i) mbar_wait(full(i % ST), (i / ST) & 1, &no_abort, p.status);
    }
    __syncwarp();
  } else {
    constexpr uint32_t idesc = make_idesc(0, 128, BN);
    const bool leader = elect_one();
    const uint64_t dw0 = smem_desc_sw128(base);  // a descriptor's address counts 16-byte units
    for (int it = 0; it < nkb; ++it) {
      const int s = it % ST, b = it % NB;
      const uint64_t dw = dw0 + (uint64_t)(s * (L::kStage >> 4)), dx = dw + (L::kW >> 4);
      if (it >= NB) bar_wait(acc_empty(b), ((it / NB) & 1) ^ 1, abort_flag, p.status);
      bar_wait(full(s), (it / ST) & 1, abort_flag, p.status);
      tc_fence_after();
      if (leader) {
#pragma unroll
        for (int kk = 0; kk < 4; ++kk)
          tc_mma_e4m3<1>(tmem + b * BN, dw + (uint64_t)(kk * 2), dx + (uint64_t)(kk * 2), idesc, kk ? 1u : 0u);
        tc_commit(empty(s));
        tc_commit(acc_full(b));
      }
    }
    if (leader) {  // every MMA has completed before TMEM is freed
      tc_commit(drain);
      volatile int no_abort = 0;
      mbar_wait(drain, 0, &no_abort, p.status);
    }
    __syncwarp();
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 5) {
    tc_fence_after();
    tmem_dealloc(tmem, L::kCols);
  }

  T* y = static_cast<T*>(p.y);
  const int n = n0 + (threadIdx.x & 127);
  auto finish = [&](int m, float v, float bias) {
    if (m < p.m && n < p.n) {
      v += bias;
      if (p.relu) v = v < 0.f ? 0.f : v;  // NaN stays NaN
      y[m * p.ldy + n] = from_f32<T>(v);
    }
  };
  const float bias = warp < 4 && p.bias && n < p.n ? p.bias[n] : 0.f;
  if (split == 1) {
    if (warp < 4) {
#pragma unroll
      for (int j = 0; j < BN; ++j) finish(j, acc[j], bias);
    }
    return;
  }
  // partial[j][row] in the stages, which every MMA and copy has left
  float* part = reinterpret_cast<float*>(gbase);
  if (warp < 4) {
#pragma unroll
    for (int j = 0; j < BN; ++j) part[j * 128 + threadIdx.x] = acc[j];
  }
  cluster_sync();
  if (warp < 4) {
    const int j0 = BN * rank / split, j1 = BN * (rank + 1) / split;
    const uint32_t mine = smem_u32(part) + threadIdx.x * 4;
    uint32_t from[8];
#pragma unroll
    for (int q = 0; q < 8; ++q) from[q] = map_to_rank(mine, q < split ? q : 0);
    for (int j = j0; j < j1; ++j) {
      float v[8];
#pragma unroll
      for (int q = 0; q < 8; ++q) v[q] = ld_cluster_f32(from[q] + j * 512);  // all in flight at once
#pragma unroll
      for (int q = 1; q < 8; ++q) v[0] = q < split ? v[0] + v[q] : v[0];
      finish(j, v[0], bias);
    }
  }
  cluster_sync_relaxed();  // no CTA leaves while another reads its partial sums
}

// ---------------------------------------------------------------- many rows
// A pair of CTAs computes 256 rows of a by BN rows of b (cta_group::2: each CTA
// loads its 128 rows of a and half of the rows of b, and holds its 128 rows of
// the accumulator).  The tile's columns are worked on 128 at a time: each half is
// an accumulator of its own, so its sums are read while the other half's MMAs
// run, and 128 columns share one scale of b.  Eight warps of each CTA keep the
// running totals in registers, thread = row of y; a further warp multiplies the
// scales of a and b and hands them over four blocks at a time.  Persistent: pairs
// walk the tiles, and a tile's stores (TMA, from shared memory) run under the
// next tile's loads and MMAs.
//
// What bounds it: at 256 x 256 a block of 128 k's takes 690 cycles, of which the MMAs
// need 512 (a pure stream of them measured 512, at 1.4 GHz under the power cap 3.3
// PFLOP/s).  With a quarter of the MMAs it still takes 685, with a quarter of the
// columns read and added 520: the epilogue warps set it, by latencies (a wait that is
// answered at once 95 cycles, the reads of two times 64 columns 190, the last additions
// 105) that two warps per scheduler do not cover, and the clock, 1.2 to 1.4 GHz at the
// power cap.  TMEM is full, and so are the registers: with sixteen columns in flight
// instead of 64 8192^3 took 523 instead of 503 us, with the next block's first columns
// loaded under the last additions 527 to 600 (register moves), with sixteen warps and
// half the totals each 580 (spills); a second warp to issue the MMAs changed nothing.
// Run without a pause (1.16 to 1.5 GHz under the power cap): 8192^3 bf16 500 to 530 us,
// 2.07 to 2.2 PFLOP/s; 4096^3 70 to 73 us; 8192 x 8192 x 1024 80 to 82 us (its tiles'
// output is a sixth); after idle, at higher clocks, 8192^3 435 to 458 us, 4096^3 62.  200
// x 8192 x 4096 (256 x 128 tiles, 36 MB) 15 us, its loop at 4.7 TB/s.
//
// 8 epilogue warps, then a warpgroup with the TMA, MMA and scale warps.  Launched
// with 168 registers a thread (384 x 168 = 64512), split as 208 for the totals and
// 88 for the rest (256 x 208 + 128 x 88 = 64512).
constexpr int kPairEpiWarps = 8;
constexpr int kPairThreads = 384;
constexpr int kGroupM = 8;  // tile order: columns of 8 tiles, so that pairs running together share operands

template <int BN>
struct PairLayout {
  static constexpr int kHalves = BN / 128;
  static constexpr int kBufs = 4 / kHalves;            // accumulators per half: 512 TMEM columns in all
  static constexpr int kA = 128 * 128, kB = BN / 2 * 128, kStage = kA + kB;
  static constexpr int kStages = BN == 256 ? 4 : 6;
  static constexpr int kOutBufs = 2;                   // staging: 32 rows of 128 bytes, two per warp
  static constexpr int kOutWarp = kOutBufs * 32 * 128;
  static constexpr int kOffOut = kStages * kStage;
  static constexpr int kOffScale = kOffOut + kPairEpiWarps * kOutWarp;  // two groups: [halves][128] rows of four blocks
  static constexpr int kScaleGroup = 4 * kHalves * 128;
  static constexpr int kCW = BN * 4 / kPairEpiWarps;   // columns per epilogue warp
  static constexpr int kOffBias = kOffScale + 2 * kScaleGroup * 4;      // per epilogue warp: its columns' bias
  static constexpr int kOffBar = kOffBias + kPairEpiWarps * kCW * 4;
  static constexpr int kBars = 2 * kStages + 13;
  static constexpr int kOffMisc = kOffBar + 8 * kBars;
  static constexpr int kBytes = kOffMisc + 16 + 1024;
};

template <typename T, int BN, bool SPLIT>
__global__ void __launch_bounds__(kPairThreads, 1)
    matmul_blocks_pair_kernel(const __grid_constant__ MatmulBlocksArgs p, const __grid_constant__ CUtensorMap tm_a,
                              const __grid_constant__ CUtensorMap tm_b, const __grid_constant__ CUtensorMap tm_y,
                              int tma_out, int split) {
  static_assert(!SPLIT || BN == 128, "the partial sums of a half would overwrite operands of the other's MMAs");
  using L = PairLayout<BN>;
  constexpr int ST = L::kStages, CW = L::kCW, NH = L::kHalves, NB = L::kBufs;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw = smem_u32(smem_raw);
  const uint32_t base = (raw + 1023u) & ~1023u;
  uint8_t* gbase = smem_raw + (base - raw);
  const uint32_t bar0 = base + L::kOffBar;
  auto full = [&](int s) { return bar0 + 8u * s; };           // leader's: both CTAs' bytes
  auto empty = [&](int s) { return bar0 + 8u * (ST + s); };   // own
  auto acc_full = [&](int b) { return bar0 + 8u * (2 * ST + b); };       // b = buffer * halves + half
  auto acc_empty = [&](int b) { return bar0 + 8u * (2 * ST + 4 + b); };  // leader's: both CTAs' warps
  auto sc_full = [&](int g) { return bar0 + 8u * (2 * ST + 8 + g); };
  auto sc_empty = [&](int g) { return bar0 + 8u * (2 * ST + 10 + g); };
  const uint32_t drain = bar0 + 8u * (2 * ST + 12);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(gbase + L::kOffMisc);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(gbase + L::kOffMisc + 4);

  // (a shuffle tells the compiler that it is the same in all lanes: TMEM addresses and
  // barriers then stay in uniform registers)
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  // rank in the pair, the pair's leader, and its slice of k (SPLIT: the pairs of a
  // cluster share a tile)
  const uint32_t crank = cluster_ctarank(), rank = SPLIT ? crank & 1 : crank, lead = SPLIT ? crank & ~1u : 0;
  const uint16_t both = (uint16_t)(3u << lead);
  if (threadIdx.x == 0) {
    for (int s = 0; s < ST; ++s) {
      mbar_init(full(s), 1);
      mbar_init(empty(s), 1);
    }
    for (int b = 0; b < 4; ++b) {
      mbar_init(acc_full(b), 1);
      mbar_init(acc_empty(b), 2 * kPairEpiWarps / NH);
    }
    for (int g = 0; g < 2; ++g) {
      mbar_init(sc_full(g), 32);
      mbar_init(sc_empty(g), kPairEpiWarps);
    }
    mbar_init(drain, 1);
    *abort_flag = 0;
    fence_mbarrier_init();
  }
  if (warp == kPairEpiWarps + 1) tmem_alloc_pair(smem_u32(tmem_slot), 512);
  if (warp == kPairEpiWarps && lane == 0) {
    prefetch_tmap(&tm_a);
    prefetch_tmap(&tm_b);
    if (tma_out) prefetch_tmap(&tm_y);
  }
  tc_fence_before();
  __syncthreads();
  cluster_sync();  // both CTAs' barriers are initialised
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  pdl_begin();

  const int tm = (p.m + 255) / 256, tn = (p.n + BN - 1) / BN;
  const int tiles = tm * tn, per_tile = SPLIT ? 2 * split : 2, pairs = gridDim.x / per_tile, tile0 = blockIdx.x / per_tile;
  const int kbs = (p.k + kQBlock - 1) / kQBlock;
  const int kb0 = SPLIT ? (int)((int64_t)kbs * (crank >> 1) / split) : 0;
  const int nkb = SPLIT ? (int)((int64_t)kbs * ((crank >> 1) + 1) / split) - kb0 : kbs;
  auto tile_at = [&](int t, int& mt, int& nt) {
    const int per = kGroupM * tn, g = t / per, rem = t - g * per;
    const int rows = min(kGroupM, tm - g * kGroupM);
    mt = g * kGroupM + rem % rows;
    nt = rem / rows;
  };

  if (warp < kPairEpiWarps) {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 208;");
    constexpr int GPH = kPairEpiWarps / 4 / NH;  // groups of four warps per half
    const int sub = warp & 3, half = (warp >> 2) / GPH, within = (warp >> 2) % GPH * CW;
    const uint32_t lane_addr = tmem + ((uint32_t)(sub * 32) << 16) + half * 128 + within;
    const uint32_t remote_empty = map_to_rank(acc_empty(half), lead);
    const uint32_t sc = base + L::kOffScale + (half * 128 + sub * 32 + lane) * 16;
    uint32_t it = 0, group = 0;
    for (int t = tile0; t < tiles; t += pairs) {
      int mt, nt;
      tile_at(t, mt, nt);
      const int row0 = mt * 256 + (int)rank * 128 + sub * 32;
      const int col0 = nt * BN + half * 128 + within;
      if (!SPLIT && p.bias) {  // here, where the first block is waited for anyway
        float* bias = reinterpret_cast<float*>(gbase + L::kOffBias) + warp * CW;
#pragma unroll
        for (int j = 0; j < CW; j += 32) bias[j + lane] = col0 + j + lane < p.n ? p.bias[col0 + j + lane] : 0.f;
      }
      uint64_t acc[CW / 2];
#pragma unroll
      for (int j = 0; j < CW / 2; ++j) acc[j] = 0;
      for (int left = nkb; left > 0; left -= 4, ++group) {
        const uint32_t g1 = group & 1;
        bar_wait(sc_full(g1), (group >> 1) & 1, abort_flag, p.status);
#pragma unroll 1
        for (int i = 0; i < min(4, left); ++i) {
          float s;
          asm volatile("ld.shared.f32 %0, [%1];" : "=f"(s) : "r"(sc + g1 * (L::kScaleGroup * 4) + i * 4) : "memory");
          const uint32_t buf = it % NB;
          bar_wait(acc_full(buf * NH + half), (it / NB) & 1, abort_flag, p.status);
          ++it;
          __syncwarp();
          tc_fence_after();
          const uint64_t s2 = pack_f2(s, s);
          const uint32_t src = lane_addr + buf * (NH * 128);
          // 64 columns arrive per wait (the wait is for every load before it); of 128,
          // each 16 of the second half are loaded into the registers of the 16 just added
          uint32_t r[4][16];
          auto add = [&](int g) {
            const uint32_t* q = r[g % 4];
#pragma unroll
            for (int j = 0; j < 8; ++j)
              acc[g * 8 + j] =
                  fma_f2(pack_f2(__uint_as_float(q[2 * j]), __uint_as_float(q[2 * j + 1])), s2, acc[g * 8 + j]);
          };
#pragma unroll
          for (int g = 0; g < 4; ++g) tmem_ld_32x32b_x16(src + g * 16, r[g]);
          tmem_ld_wait();
          if constexpr (CW == 128) {
#pragma unroll
            for (int g = 0; g < 4; ++g) {
              add(g);
              tmem_ld_32x32b_x16(src + 64 + g * 16, r[g]);
            }
            tmem_ld_wait();
          }
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive_remote(remote_empty + buf * (NH * 8));
#pragma unroll
          for (int g = CW / 16 - 4; g < CW / 16; ++g) add(g);
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(sc_empty(g1));
      }
      if constexpr (SPLIT) {
        // partial[column][row] in the stages: the last block's sums are here, so every
        // MMA has run and every copy has landed
        float* part = reinterpret_cast<float*>(gbase) + within * 128 + sub * 32 + lane;
#pragma unroll
        for (int j = 0; j < CW / 2; ++j) {
          const float2 f = unpack_f2(acc[j]);
          part[(2 * j) * 128] = f.x;
          part[(2 * j + 1) * 128] = f.y;
        }
        break;
      }
      // Bias, Relu, rounding; then a warp's 32 rows go through its own staging
      // rows (swizzled as the TMA map wants them, which is also free of bank
      // conflicts) to TMA stores that clip the tile's edges; where TMA cannot
      // write (y, or its last column, off the 16-byte grid), element by element.
      constexpr int ES = sizeof(T), PER = 16 / ES, CPR = 128 / ES;  // columns of a 16-byte unit, of a staging row
      constexpr int NC = CW / CPR, OB = NC < L::kOutBufs ? NC : L::kOutBufs;
      const uint32_t out = base + L::kOffOut + warp * L::kOutWarp;
#pragma unroll
      for (int c0 = 0; c0 < NC; c0 += OB) {
        if (lane == 0) bulk_wait_group_read<0>();  // the last stores have read the buffers
        __syncwarp();
        auto stage = [&](auto extras) {  // with bias and Relu, or without either
#pragma unroll
          for (int c = c0; c < c0 + OB; ++c) {
            const uint32_t mine = out + (c - c0) * 4096 + lane * 128;
#pragma unroll
            for (int u = 0; u < 8; ++u) {
              float f[PER];
#pragma unroll
              for (int q = 0; q < PER; q += 2) {
                const float2 v = unpack_f2(acc[(c * CPR + u * PER + q) / 2]);
                f[q] = v.x;
                f[q + 1] = v.y;
              }
              if constexpr (decltype(extras)::value) {
                if (p.bias) {
                  const float4* b4 = reinterpret_cast<const float4*>(gbase + L::kOffBias) + (warp * CW + c * CPR + u * PER) / 4;
#pragma unroll
                  for (int q = 0; q < PER; q += 4) {
                    const float4 b = b4[q / 4];
                    f[q] += b.x;
                    f[q + 1] += b.y;
                    f[q + 2] += b.z;
                    f[q + 3] += b.w;
                  }
                }
#pragma unroll
                for (int q = 0; q < PER; ++q)
                  if (p.relu) f[q] = f[q] < 0.f ? 0.f : f[q];  // NaN stays NaN
              }
              uint32_t w[4];
#pragma unroll
              for (int q = 0; q < 4; ++q) {
                if constexpr (ES == 4)
                  w[q] = __float_as_uint(f[q]);
                else
                  w[q] = pack_rounded<T>(f[2 * q], f[2 * q + 1]);
              }
              asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(mine + ((u ^ (lane & 7)) * 16)), "r"(w[0]),
                           "r"(w[1]), "r"(w[2]), "r"(w[3])
                           : "memory");
            }
          }
        };
        if (p.bias || p.relu)
          stage(std::true_type{});
        else
          stage(std::false_type{});
        // a store's box is cut in units of 16 bytes: an edge inside one is written by elements
        if (tma_out && (p.n % PER == 0 || col0 + (c0 + OB) * CPR <= p.n)) {
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) {
#pragma unroll
            for (int c = c0; c < c0 + OB; ++c)
              if (row0 < p.m && col0 + c * CPR < p.n) tma_store_2d(&tm_y, col0 + c * CPR, row0, out + (c - c0) * 4096);
            bulk_commit_group();
          }
        } else {
          __syncwarp();
#pragma unroll 1
          for (int q = 0; q < OB * 8; ++q) {
            const int rr = q % 8 * 4 + (lane >> 3), u = lane & 7, col = col0 + (c0 + q / 8) * CPR + u * PER;
            uint32_t w[4];
            asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
                         : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3])
                         : "r"(out + q / 8 * 4096 + rr * 128 + ((u ^ (rr & 7)) * 16))
                         : "memory");
            if (row0 + rr < p.m) {
              T* dst = static_cast<T*>(p.y) + (row0 + rr) * p.ldy + col;
              const T* e = reinterpret_cast<const T*>(w);
#pragma unroll
              for (int k = 0; k < PER; ++k)
                if (col + k < p.n) dst[k] = e[k];
            }
          }
          __syncwarp();
        }
      }
    }
    if (lane == 0) bulk_wait_group<0>();  // every store is complete before the CTA exits
    __syncwarp();
  } else {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 88;");
  }
  if (warp == kPairEpiWarps) {
    if (lane == 0) {
      uint32_t it = 0;
      bool ok = true;
      for (int t = tile0; t < tiles && ok; t += pairs) {
        int mt, nt;
        tile_at(t, mt, nt);
        const int ra = mt * 256 + (int)rank * 128, rb = nt * BN + (int)rank * 64;
        for (int kb = 0; kb < nkb; ++kb, ++it) {
          const int s = it % ST;
          ok = mbar_wait(empty(s), ((it / ST) & 1) ^ 1, abort_flag, p.status);
          if (!ok) break;
          const uint32_t bar = map_to_rank(full(s), lead);
          if (rank == 0) mbar_arrive_expect_tx(full(s), 2 * L::kStage);
          const uint32_t dst = base + s * L::kStage;
          tma_load_2d_pair(dst, &tm_a, (kb0 + kb) * kQBlock, ra, bar);
#pragma unroll
          for (int hf = 0; hf < NH; ++hf)  // this CTA's 64 rows of each half
            tma_load_2d_pair(dst + L::kA + hf * 8192, &tm_b, (kb0 + kb) * kQBlock, rb + hf * 128, bar);
        }
      }
      // every copy has landed before the CTA may exit: the MMA of its stage has
      // run (only the leader sees the arrivals themselves)
      volatile int no_abort = 0;
      for (uint32_t i = it > ST ? it - ST : 0; i < it; ++i) mbar_wait(empty(i % ST), (i / ST) & 1, &no_abort, p.status);
    }
    __syncwarp();
  } else if (warp == kPairEpiWarps + 1) {
    constexpr uint32_t idesc = make_idesc(0, 256, 128);
    if (rank == 0) {
      const bool leader = elect_one();
      const uint64_t da0 = smem_desc_sw128(base);  // a descriptor's address counts 16-byte units
      int s = 0, buf = 0;
      uint32_t sp = 0, bp = 1;  // parities: of the stage's use, of the buffer's release
      const int total = nkb * ((tiles - tile0 + pairs - 1) / pairs);
      for (int it = 0; it < total; ++it) {
        const uint64_t da = da0 + (uint64_t)(s * (L::kStage >> 4)), db = da + (L::kA >> 4);
        bar_wait(full(s), sp, abort_flag, p.status);
#pragma unroll
        for (int hf = 0; hf < NH; ++hf) {
          bar_wait(acc_empty(buf * NH + hf), bp, abort_flag, p.status);
          tc_fence_after();
          if (leader) {
#pragma unroll
            for (int kk = 0; kk < 4; ++kk)
              tc_mma_e4m3<2>(tmem + (buf * NH + hf) * 128, da + (uint64_t)(kk * 2), db + (uint64_t)(hf * 512 + kk * 2),
                             idesc, kk ? 1u : 0u);
            if (hf == NH - 1) tc_commit_pair(empty(s), both);
            tc_commit_pair(acc_full(buf * NH + hf), both);
          }
        }
        if (++s == ST) {
          s = 0;
          sp ^= 1;
        }
        if (++buf == NB) {
          buf = 0;
          bp ^= 1;
        }
      }
      // every MMA has completed before TMEM is freed
      if (leader) {
        tc_commit_pair(drain, both);
        volatile int no_abort = 0;
        mbar_wait(drain, 0, &no_abort, p.status);
      }
    }
    __syncwarp();
  } else if (warp == kPairEpiWarps + 2) {
    // sa * sb of this CTA's 128 rows and each half's block of b, four blocks of k
    // ahead: loaded before the buffer is waited for
    uint32_t group = 0;
    bool ok = true;
    for (int t = tile0; t < tiles && ok; t += pairs) {
      int mt, nt;
      tile_at(t, mt, nt);
      const int row = mt * 256 + (int)rank * 128 + lane;
      for (int kb = 0; kb < nkb; kb += 4, ++group) {
        float va[4][4], vb[4][NH];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int k = kb0 + min(kb + i, nkb - 1);
#pragma unroll
          for (int j = 0; j < 4; ++j) va[i][j] = p.as[(int64_t)min(row + j * 32, p.m - 1) * p.as_row + k * p.as_block];
#pragma unroll
          for (int hf = 0; hf < NH; ++hf)
            vb[i][hf] = p.bs[(int64_t)(min(nt * BN + hf * 128, p.n - 1) / kQBlock) * p.bs_row + k * p.bs_block];
        }
        ok = __all_sync(0xffffffffu, mbar_wait(sc_empty(group & 1), ((group >> 1) & 1) ^ 1, abort_flag, p.status));
        if (!ok) break;
        float4* dst = reinterpret_cast<float4*>(gbase + L::kOffScale) + (group & 1) * (L::kScaleGroup / 4) + lane;
#pragma unroll
        for (int hf = 0; hf < NH; ++hf)
#pragma unroll
          for (int j = 0; j < 4; ++j)
            dst[hf * 128 + j * 32] = make_float4(va[0][j] * vb[0][hf], va[1][j] * vb[1][hf], va[2][j] * vb[2][hf], va[3][j] * vb[3][hf]);
        mbar_arrive(sc_full(group & 1));  // every lane: its own stores
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  cluster_sync();  // the pair's MMAs read both CTAs' shared memory and write both TMEMs; partial sums
  if (warp == kPairEpiWarps + 1) {
    tc_fence_after();
    tmem_dealloc_pair(tmem, 512);
  }
  if constexpr (SPLIT) {
    // Each pair finishes its share of the tile's columns, 8 at a time per thread (row):
    // the slices' sums over distributed shared memory, in order.
    if (warp < kPairEpiWarps) {
      int mt, nt;
      tile_at(tile0, mt, nt);
      const int r = (warp & 3) * 32 + lane, row = mt * 256 + (int)rank * 128 + r;
      const int share = BN / split, c0 = (int)(crank >> 1) * share + (warp >> 2) * (share / 2);
      uint32_t from[4];
#pragma unroll
      for (int q = 0; q < 4; ++q) from[q] = map_to_rank(base + r * 4, q < split ? 2 * q + rank : crank);
      constexpr int PER = 16 / sizeof(T);
      const bool vec = (reinterpret_cast<uintptr_t>(p.y) & 15) == 0 && p.ldy % PER == 0;
      for (int c = c0; c < c0 + share / 2; c += 8) {
        float v[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          float s[4];
#pragma unroll
          for (int q = 0; q < 4; ++q) s[q] = ld_cluster_f32(from[q] + (c + j) * 512);
          v[j] = s[0] + s[1];
          if (split == 4) v[j] = v[j] + s[2] + s[3];
        }
        const int col = nt * BN + c;
        if (row < p.m && col < p.n) {
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            if (p.bias) v[j] += p.bias[min(col + j, p.n - 1)];
            if (p.relu) v[j] = v[j] < 0.f ? 0.f : v[j];  // NaN stays NaN
          }
          T* dst = static_cast<T*>(p.y) + row * p.ldy + col;
          if (vec && col + 8 <= p.n) {
#pragma unroll
            for (int u = 0; u < 8 / PER; ++u) {
              uint32_t w[4];
#pragma unroll
              for (int q = 0; q < 4; ++q) {
                if constexpr (sizeof(T) == 4)
                  w[q] = __float_as_uint(v[u * 4 + q]);
                else
                  w[q] = pack_rounded<T>(v[2 * q], v[2 * q + 1]);
              }
              reinterpret_cast<uint4*>(dst)[u] = make_uint4(w[0], w[1], w[2], w[3]);
            }
          } else {
#pragma unroll
            for (int j = 0; j < 8; ++j)
              if (col + j < p.n) dst[j] = from_f32<T>(v[j]);
          }
        }
      }
    }
    cluster_sync_relaxed();  // no CTA leaves while another reads its partial sums
  }
}

// ---------------------------------------------------------------- host
typedef CUresult (*EncodeFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                             const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                             CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
EncodeFn encode_fn() {
  static EncodeFn fn = [] {
    void* f = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &f, 12000, cudaEnableDefault, &q) != cudaSuccess ||
        q != cudaDriverEntryPointSuccess)
      f = nullptr;
    return reinterpret_cast<EncodeFn>(f);
  }();
  return fn;
}

// Boxes of `box` rows by 128 bytes of a [rows][k] byte matrix, zeros outside.
bool encode_rows(const uint8_t* q, int rows, int k, int64_t ld, int box, CUtensorMap* map) {
  EncodeFn fn = encode_fn();
  if (!fn) return false;
  const cuuint64_t dims[2] = {(cuuint64_t)k, (cuuint64_t)rows}, strides[1] = {(cuuint64_t)ld};
  const cuuint32_t boxes[2] = {128, (cuuint32_t)box}, es[2] = {1, 1};
  return fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<uint8_t*>(q), dims, strides, boxes, es,
            CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

cudaLaunchConfig_t cluster_config(unsigned grid, unsigned cluster, int threads, int smem, cudaLaunchAttribute (&attr)[2]) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3((unsigned)threads);
  cfg.dynamicSmemBytes = (size_t)smem;
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = cluster;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  return cfg;
}

// Clusters of 4 or 8 CTAs that run at once: a cluster does not cross the groups of SMs that
// the GPU is made of, so that fewer fit than its SMs would hold.  A device's answer never
// changes: asked once, of a kernel that does nothing in CTAs of the same size (of one that
// takes tensor memory it is given for one CTA per SM, though two run).
template <int THREADS, int PER_SM, int TAG>
__global__ void __launch_bounds__(THREADS, PER_SM) same_size_kernel() {}
template <auto KERNEL>
int clusters_at_once(unsigned cluster, int threads, int smem) {
  constexpr int kMaxDevices = 64;
  static std::atomic<int> known[kMaxDevices][2];  // plus one; 0: not asked yet
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= kMaxDevices) return 0;
  std::atomic<int>& k = known[dev][cluster == 8];
  int v = k.load(std::memory_order_relaxed);
  if (v == 0) {
    cudaLaunchAttribute attr[2];
    cudaLaunchConfig_t cfg = cluster_config(cluster, cluster, threads, smem, attr);
    cfg.numAttrs = 1;
    int n = 0;
    if (opt_in<KERNEL>(smem) != 0 || cudaOccupancyMaxActiveClusters(&n, KERNEL, &cfg) != cudaSuccess) {
      cudaGetLastError();  // no reason for the launch of smaller clusters to fail
      return 0;
    }
    v = n + 1;
    k.store(v, std::memory_order_relaxed);
  }
  return v - 1;
}

template <typename T, int M>
int launch_vec(const MatmulBlocksArgs& a, cudaStream_t st) {
  const size_t smem = (size_t)matmul_vec_smem(M, a.k);
  if (smem > 48 * 1024) {
    const int rc = opt_in<matmul_blocks_vec_kernel<T, M>>((int)kVecMaxSmem);
    if (rc) return rc;
  }
  const unsigned per = kVecWarps * kVecRows;
  return launch_pdl(matmul_blocks_vec_kernel<T, M>, (a.n + per - 1) / per, kVecWarps * 32, smem, st, a);
}

template <typename T, int BN>
int launch_rows(const MatmulBlocksArgs& a, int split, cudaStream_t st) {
  using L = RowsLayout<BN>;
  CUtensorMap w, x;
  if (!encode_rows(a.b, a.n, a.k, a.ldb, 128, &w) || !encode_rows(a.a, a.m, a.k, a.lda, BN, &x))
    return (int)cudaErrorInvalidValue;
  int rc = opt_in<matmul_blocks_rows_kernel<T, BN>>(L::kBytes);
  if (rc) return rc;
  cudaLaunchAttribute attr[2];
  cudaLaunchConfig_t cfg = cluster_config((unsigned)((a.n + 127) / 128) * split, (unsigned)split, kRowsThreads, L::kBytes, attr);
  cfg.stream = st;
  return (int)cudaLaunchKernelEx(&cfg, matmul_blocks_rows_kernel<T, BN>, a, w, x, split);
}

// Split k over CTAs until they fill the GPU's SMs once or twice, two blocks each at
// least; the first split also pays for the clusters (16 x 4096 x 4096 with 32
// tiles: 12.9, 10.8, 8.9 and 8.7 us with 1, 2, 4 and 8 CTAs a tile; 16 x 14336 x
// 4096 with 112: 15.1, 16.4, 19.9; 17 x 1000 x 2048 with 8: 9.1, 9.2, 7.2, 5.9), and
// no further than the clusters run at once (16 x 9472 x 4096, whose 74 clusters of
// four take two turns: 13.0, 13.2, 16.6).
template <typename T, int BN>
int rows_split(const MatmulBlocksArgs& a, int num_sms) {
  const int tiles = (a.n + 127) / 128, kbs = (a.k + kQBlock - 1) / kQBlock;
  int split = tiles * 4 <= num_sms * 3 && kbs >= 4 ? 2 : 1;
  while (split > 1 && split < 8 && tiles * split <= num_sms && kbs >= split * 4 &&
         tiles <= clusters_at_once<same_size_kernel<kRowsThreads, 2, BN>>(2u * split, kRowsThreads, RowsLayout<BN>::kBytes))
    split *= 2;
  return split;
}

// Boxes of 32 rows by 128 bytes of y, for the stores; false where TMA cannot write.
template <typename T>
bool encode_out(const MatmulBlocksArgs& a, CUtensorMap* map) {
  EncodeFn fn = encode_fn();
  if (!fn || (reinterpret_cast<uintptr_t>(a.y) & 15) || a.ldy * sizeof(T) % 16) return false;
  const cuuint64_t dims[2] = {(cuuint64_t)a.n, (cuuint64_t)a.m}, strides[1] = {(cuuint64_t)a.ldy * sizeof(T)};
  const cuuint32_t boxes[2] = {(cuuint32_t)(128 / sizeof(T)), 32}, es[2] = {1, 1};
  return fn(map, sizeof(T) == 2 ? CU_TENSOR_MAP_DATA_TYPE_UINT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT32, 2, a.y, dims, strides,
            boxes, es, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
            CU_TENSOR_MAP_L2_PROMOTION_NONE, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// split: pairs that share a tile (1, 2 or 4; BN == 128).
template <typename T, int BN, bool SPLIT = false>
int launch_pair(const MatmulBlocksArgs& a, int num_sms, cudaStream_t st, int split = 1) {
  using L = PairLayout<BN>;
  CUtensorMap ma, mb, my{};
  if (!encode_rows(a.a, a.m, a.k, a.lda, 128, &ma) || !encode_rows(a.b, a.n, a.k, a.ldb, 64, &mb))
    return (int)cudaErrorInvalidValue;
  const int tma_out = SPLIT ? 0 : encode_out<T>(a, &my);
  int rc = opt_in<matmul_blocks_pair_kernel<T, BN, SPLIT>>(L::kBytes);
  if (rc) return rc;
  const int tiles = ((a.m + 255) / 256) * ((a.n + BN - 1) / BN);
  cudaLaunchAttribute attr[2];
  cudaLaunchConfig_t cfg =
      cluster_config(2u * split * (SPLIT ? tiles : std::min(tiles, num_sms / 2)), 2u * split, kPairThreads, L::kBytes, attr);
  cfg.stream = st;
  return (int)cudaLaunchKernelEx(&cfg, matmul_blocks_pair_kernel<T, BN, SPLIT>, a, ma, mb, my, tma_out, split);
}

}  // namespace

int matmul_blocks_launch(const MatmulBlocksArgs& a, int num_sms, cudaStream_t st) {
  const bool tma = a.k > 0 && a.lda % 16 == 0 && a.ldb % 16 == 0 &&
                   ((reinterpret_cast<uintptr_t>(a.a) | reinterpret_cast<uintptr_t>(a.b)) & 15) == 0;
  return with_type(a.out_type, [&](auto* t) {
    using T = std::remove_pointer_t<decltype(t)>;
    if (!tma) {
      return launch_pdl(matmul_blocks_simt_kernel<T>, (unsigned)((a.n + 63) / 64) * ((a.m + 63) / 64), 256, 0, st, a);
    }
    const int kbs = (a.k + kQBlock - 1) / kQBlock;
    // 33 to 64 rows with few columns stay with the kernel for few rows, whose clusters
    // split k eight ways (64 x 4096 x 4096: 10.7 us, 12.5 on pairs; with 64 tiles of
    // columns, 64 x 8192 x 4096, 18.7 and 15.4).
    if (a.m > 64 || (a.m > 32 && (a.n + 127) / 128 * 4 > num_sms)) {
      const int64_t tm = (a.m + 255) / 256, pairs = num_sms / 2;
      // Few tiles: two or four pairs share one, where all run at once (with one, two and
      // four: 256 x 1024 x 4096 13.2, 12.3 and 10.6 us; 100 x 1000 x 14336 30.9, 21.6 and
      // 15.5; but 200 x 2048 x 4096, whose 16 clusters of eight CTAs take two turns, 13.3,
      // 12.5 and 19.2, and 256 x 4608 x 4096 13.8, 23.1 and 28.6) and k is long enough to
      // pay for the join (256 x 1280 x 2048: 9.0, 9.7 and 9.0; 256 x 2560 x 2560 10.8 and
      // 11.3 with one and two).
      const int64_t tiles = tm * ((a.n + 127) / 128);
      auto at_once = [&](int s) {
        return clusters_at_once<same_size_kernel<kPairThreads, 1, 128>>(2u * s, kPairThreads, PairLayout<128>::kBytes);
      };
      if (tiles * 4 <= pairs && kbs >= 16 && tiles <= at_once(4)) return launch_pair<T, 128, true>(a, num_sms, st, 4);
      if (tiles * 2 <= pairs && kbs >= 28 && tiles <= at_once(2)) return launch_pair<T, 128, true>(a, num_sms, st, 2);
      return matmul_takes_wide(a.m, a.n, num_sms) ? launch_pair<T, 256>(a, num_sms, st) : launch_pair<T, 128>(a, num_sms, st);
    }
    if (matmul_takes_vec(a.m, a.k)) return a.m == 1 ? launch_vec<T, 1>(a, st) : launch_vec<T, 2>(a, st);
    return a.m <= 16   ? launch_rows<T, 16>(a, rows_split<T, 16>(a, num_sms), st)
           : a.m <= 32 ? launch_rows<T, 32>(a, rows_split<T, 32>(a, num_sms), st)
                       : launch_rows<T, 64>(a, rows_split<T, 64>(a, num_sms), st);
  });
}

}  // namespace ob2
