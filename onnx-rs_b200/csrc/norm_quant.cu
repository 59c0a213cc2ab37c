// Root-mean-square normalisation (with the residual's addition in front and the
// quantisation behind it) and block quantisation to e4m3.
#include "blocks.cuh"

namespace ob2 {
namespace {

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
__device__ __forceinline__ float warp_max_nan(float v) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v = max_nan(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}

// One row per block, the row's fp32 sum x + residual held in shared memory.
template <typename T, typename W>
__global__ void __launch_bounds__(256) rmsnorm_row_kernel(const RmsNormArgs p) {
  extern __shared__ float row[];
  __shared__ float part[8];
  const int64_t r = blockIdx.x;
  const T* x = static_cast<const T*>(p.x) + r * p.ldx;
  const T* res = p.res ? static_cast<const T*>(p.res) + r * p.ldr : nullptr;
  T* sum = p.sum ? static_cast<T*>(p.sum) + r * p.lds : nullptr;
  const W* w = static_cast<const W*>(p.weight);
  float ss = 0.f;
  for (int i = threadIdx.x; i < p.cols; i += 256) {
    float v = to_f32(x[i]);
    if (res) v += to_f32(res[i]);
    if (sum) sum[i] = from_f32<T>(v);
    row[i] = v;
    ss = fmaf(v, v, ss);
  }
  ss = warp_sum(ss);
  if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = ss;
  __syncthreads();
  float tot = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) tot += part[i];
  const float rstd = 1.f / sqrtf(tot / (float)p.cols + p.eps);
  if (p.out_type != kE4M3) {
    T* y = static_cast<T*>(p.y) + r * p.ldy;
    for (int i = threadIdx.x; i < p.cols; i += 256) y[i] = from_f32<T>(row[i] * rstd * to_f32(w[i]));
    return;
  }
  uint8_t* q = static_cast<uint8_t*>(p.y) + r * p.ldy;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  for (int b = warp; b * kQBlock < p.cols; b += 8) {
    float v[4], amax = 0.f;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int i = b * kQBlock + j * 32 + lane;
      v[j] = i < p.cols ? row[i] * rstd * to_f32(w[i]) : 0.f;
      amax = max_nan(amax, fabsf(v[j]));
    }
    float scale, inv;
    block_scale(warp_max_nan(amax), scale, inv);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int i = b * kQBlock + j * 32 + lane;
      if (i < p.cols) q[i] = to_e4m3(v[j] * inv);
    }
    if (lane == 0) p.y_scale[r * p.ys_row + b * p.ys_block] = scale;
  }
}

// block_rows = 1: one warp per block of 128 columns of a row.
template <typename T>
__global__ void __launch_bounds__(256) quantize_row_kernel(const QuantizeArgs p, int64_t cb, int64_t units) {
  const int lane = threadIdx.x & 31;
  const int64_t u = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
  if (u >= units) return;
  const int64_t r = u / cb, b = u - r * cb;
  const T* x = static_cast<const T*>(p.x) + r * p.ldx;
  float v[4], amax = 0.f;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int64_t i = b * kQBlock + j * 32 + lane;
    v[j] = i < p.cols ? to_f32(x[i]) : 0.f;
    amax = max_nan(amax, fabsf(v[j]));
  }
  float scale, inv;
  block_scale(warp_max_nan(amax), scale, inv);
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int64_t i = b * kQBlock + j * 32 + lane;
    if (i < p.cols) p.q[r * p.ldq + i] = to_e4m3(v[j] * inv);
  }
  if (lane == 0) p.scale[r * p.s_row + b * p.s_block] = scale;
}

// block_rows = 128: one thread block per block of 128 x 128.
template <typename T>
__global__ void __launch_bounds__(256) quantize_tile_kernel(const QuantizeArgs p, int64_t cb) {
  __shared__ float part[8];
  const int64_t rb = blockIdx.x / cb, b = blockIdx.x - rb * cb;
  const int64_t c = b * kQBlock + (threadIdx.x & 127);
  const T* x = static_cast<const T*>(p.x);
  float amax = 0.f;
  for (int i = threadIdx.x >> 7; i < 128; i += 2) {
    const int64_t r = rb * 128 + i;
    if (r < p.rows && c < p.cols) amax = max_nan(amax, fabsf(to_f32(x[r * p.ldx + c])));
  }
  amax = warp_max_nan(amax);
  if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = amax;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 8; ++i) amax = max_nan(amax, part[i]);
  float scale, inv;
  block_scale(amax, scale, inv);
  for (int i = threadIdx.x >> 7; i < 128; i += 2) {
    const int64_t r = rb * 128 + i;
    if (r < p.rows && c < p.cols) p.q[r * p.ldq + c] = to_e4m3(to_f32(x[r * p.ldx + c]) * inv);
  }
  if (threadIdx.x == 0) p.scale[rb * p.s_row + b * p.s_block] = scale;
}

}  // namespace

int rmsnorm_launch(const RmsNormArgs& a, cudaStream_t st) {
  return with_type(a.type, [&](auto* t) {
    using T = std::remove_pointer_t<decltype(t)>;
    return with_type(a.weight_type, [&](auto* wt) {
      using W = std::remove_pointer_t<decltype(wt)>;
      const int smem = a.cols * (int)sizeof(float);
      if (smem > 48 * 1024 - 64) {
        cudaError_t e = cudaFuncSetAttribute(rmsnorm_row_kernel<T, W>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
        if (e != cudaSuccess) return (int)e;
      }
      rmsnorm_row_kernel<T, W><<<(unsigned)a.rows, 256, smem, st>>>(a);
      return (int)cudaGetLastError();
    });
  });
}

int quantize_launch(const QuantizeArgs& a, cudaStream_t st) {
  const int64_t cb = (a.cols + kQBlock - 1) / kQBlock;
  return with_type(a.type, [&](auto* t) {
    using T = std::remove_pointer_t<decltype(t)>;
    if (a.block_rows == 1) {
      const int64_t units = a.rows * cb;
      quantize_row_kernel<T><<<(unsigned)((units + 7) / 8), 256, 0, st>>>(a, cb, units);
    } else {
      quantize_tile_kernel<T><<<(unsigned)((a.rows + 127) / 128 * cb), 256, 0, st>>>(a, cb);
    }
    return (int)cudaGetLastError();
  });
}

}  // namespace ob2
