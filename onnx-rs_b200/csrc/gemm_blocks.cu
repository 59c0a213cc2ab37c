// Block-scaled matrix product of e4m3 operands.
#include "blocks.cuh"

namespace ob2 {
namespace {

// CUDA cores: 64 x 64 outputs per block, 4 x 4 per thread; the products of a
// block of 128 k's are summed in fp32, then scaled and added to the total.
template <typename T>
__global__ void __launch_bounds__(256) matmul_blocks_simt_kernel(const MatmulBlocksArgs p) {
  __shared__ float sa[32][65], sb[32][65];
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

}  // namespace

int matmul_blocks_launch(const MatmulBlocksArgs& a, int num_sms, cudaStream_t st) {
  (void)num_sms;
  return with_type(a.out_type, [&](auto* t) {
    using T = std::remove_pointer_t<decltype(t)>;
    matmul_blocks_simt_kernel<T><<<(unsigned)((a.n + 63) / 64) * ((a.m + 63) / 64), 256, 0, st>>>(a);
    return (int)cudaGetLastError();
  });
}

}  // namespace ob2
