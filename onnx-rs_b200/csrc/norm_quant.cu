// Root-mean-square normalisation (with the residual's addition in front and the
// quantisation behind it) and block quantisation to e4m3.
#include <algorithm>

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

// Eight consecutive elements of a type that starts on a 16-byte boundary (fp32:
// two 16-byte accesses, 16-bit types: one).
template <typename T>
struct Vec8 {
  uint4 v[sizeof(T) / 2];
  __device__ __forceinline__ void load(const T* p) {
#pragma unroll
    for (int i = 0; i < (int)sizeof(T) / 2; ++i) v[i] = reinterpret_cast<const uint4*>(p)[i];
  }
  __device__ __forceinline__ void store(T* p) const {
#pragma unroll
    for (int i = 0; i < (int)sizeof(T) / 2; ++i) reinterpret_cast<uint4*>(p)[i] = v[i];
  }
  __device__ __forceinline__ float get(int i) const { return to_f32(reinterpret_cast<const T*>(v)[i]); }
  __device__ __forceinline__ void set(int i, float f) { reinterpret_cast<T*>(v)[i] = from_f32<T>(f); }
};

// Largest magnitude over the 16 lanes (of 8 elements each) that share a block of 128.
__device__ __forceinline__ float lanes16_max_nan(float v) {
#pragma unroll
  for (int o = 8; o; o >>= 1) v = max_nan(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}

// Rows whose every vector is aligned: one row per block, CH vectors of eight
// columns per thread, read once and kept in registers; the weight is on its way
// before the row's one reduction (a shuffle and a barrier).  Bound by HBM with
// several blocks per SM taking turns; blocks that walk rows with the next two rows
// copied ahead were slower (107 against 84 us below: fewer blocks, and the same
// chain of reductions).  8192 x 8192 bf16 with residual and e4m3 output (470 MB):
// %NORM%.
template <typename T, typename W, int CH>
__global__ void __launch_bounds__(CH == 4 ? 512 : 1024, CH == 4 && sizeof(T) == 2 ? 2 : 1)
    rmsnorm_vec_kernel(const RmsNormArgs p) {
  __shared__ float part[32];
  pdl_begin();
  const int64_t r = blockIdx.x;
  const int n8 = p.cols / 8, nt = blockDim.x;
  const T* x = static_cast<const T*>(p.x) + r * p.ldx;
  Vec8<T> v[CH];
#pragma unroll
  for (int c = 0; c < CH; ++c)
    if (c * nt + threadIdx.x < n8) v[c].load(x + (c * nt + threadIdx.x) * 8);
  float h[CH][8];
  if (p.res) {
    const T* res = static_cast<const T*>(p.res) + r * p.ldr;
    Vec8<T> vr[CH];
#pragma unroll
    for (int c = 0; c < CH; ++c)
      if (c * nt + threadIdx.x < n8) vr[c].load(res + (c * nt + threadIdx.x) * 8);
#pragma unroll
    for (int c = 0; c < CH; ++c)
#pragma unroll
      for (int j = 0; j < 8; ++j) h[c][j] = c * nt + threadIdx.x < n8 ? v[c].get(j) + vr[c].get(j) : 0.f;
  } else {
#pragma unroll
    for (int c = 0; c < CH; ++c)
#pragma unroll
      for (int j = 0; j < 8; ++j) h[c][j] = c * nt + threadIdx.x < n8 ? v[c].get(j) : 0.f;
  }
  Vec8<W> vw[CH];
#pragma unroll
  for (int c = 0; c < CH; ++c)
    if (c * nt + threadIdx.x < n8) vw[c].load(static_cast<const W*>(p.weight) + (c * nt + threadIdx.x) * 8);
  float ss = 0.f;
#pragma unroll
  for (int c = 0; c < CH; ++c)
#pragma unroll
    for (int j = 0; j < 8; ++j) ss = fmaf(h[c][j], h[c][j], ss);
  ss = warp_sum(ss);
  if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = ss;
  if (p.sum) {
    T* sum = static_cast<T*>(p.sum) + r * p.lds;
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      Vec8<T> o;
#pragma unroll
      for (int j = 0; j < 8; ++j) o.set(j, h[c][j]);
      if (c * nt + threadIdx.x < n8) o.store(sum + (c * nt + threadIdx.x) * 8);
    }
  }
  __syncthreads();
  ss = (threadIdx.x & 31) < nt / 32 ? part[threadIdx.x & 31] : 0.f;
  ss = warp_sum(ss);
  const float rstd = 1.f / sqrtf(ss / (float)p.cols + p.eps);
#pragma unroll
  for (int c = 0; c < CH; ++c) {
    const int i = c * nt + threadIdx.x;
    float amax = 0.f;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      h[c][j] = i < n8 ? h[c][j] * rstd * vw[c].get(j) : 0.f;
      amax = max_nan(amax, fabsf(h[c][j]));
    }
    if (p.out_type != kE4M3) {
      Vec8<T> o;
#pragma unroll
      for (int j = 0; j < 8; ++j) o.set(j, h[c][j]);
      if (i < n8) o.store(static_cast<T*>(p.y) + r * p.ldy + i * 8);
    } else {
      float scale, inv;
      block_scale(lanes16_max_nan(amax), scale, inv);
      if (i < n8) {
        const float* f = h[c];
        *reinterpret_cast<uint2*>(static_cast<uint8_t*>(p.y) + r * p.ldy + i * 8) =
            make_uint2(to_e4m3x4(f[0] * inv, f[1] * inv, f[2] * inv, f[3] * inv),
                       to_e4m3x4(f[4] * inv, f[5] * inv, f[6] * inv, f[7] * inv));
        if ((threadIdx.x & 15) == 0) p.y_scale[r * p.ys_row + (i / 16) * p.ys_block] = scale;
      }
    }
  }
}

// Any alignment and width: one row per block, the row's fp32 sum x + residual held
// in shared memory.
constexpr int kRowThreads = 512;
template <typename T, typename W>
__global__ void __launch_bounds__(kRowThreads) rmsnorm_row_kernel(const RmsNormArgs p) {
  extern __shared__ float row[];
  __shared__ float part[kRowThreads / 32];
  pdl_begin();
  const int64_t r = blockIdx.x;
  const T* x = static_cast<const T*>(p.x) + r * p.ldx;
  const T* res = p.res ? static_cast<const T*>(p.res) + r * p.ldr : nullptr;
  T* sum = p.sum ? static_cast<T*>(p.sum) + r * p.lds : nullptr;
  const W* w = static_cast<const W*>(p.weight);
  float ss = 0.f;
  for (int i0 = threadIdx.x; i0 < p.cols; i0 += 8 * kRowThreads) {
    float v[8];  // eight loads in flight (a store to sum would keep the next load behind it)
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = i0 + j * kRowThreads < p.cols ? to_f32(x[i0 + j * kRowThreads]) : 0.f;
    if (res) {
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] += i0 + j * kRowThreads < p.cols ? to_f32(res[i0 + j * kRowThreads]) : 0.f;
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int i = i0 + j * kRowThreads;
      if (i >= p.cols) break;
      if (sum) sum[i] = from_f32<T>(v[j]);
      row[i] = v[j];
      ss = fmaf(v[j], v[j], ss);
    }
  }
  ss = warp_sum(ss);
  if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = ss;
  __syncthreads();
  float tot = 0.f;
#pragma unroll
  for (int i = 0; i < kRowThreads / 32; ++i) tot += part[i];
  const float rstd = 1.f / sqrtf(tot / (float)p.cols + p.eps);
  if (p.out_type != kE4M3) {
    T* y = static_cast<T*>(p.y) + r * p.ldy;
    for (int i = threadIdx.x; i < p.cols; i += kRowThreads) y[i] = from_f32<T>(row[i] * rstd * to_f32(w[i]));
    return;
  }
  uint8_t* q = static_cast<uint8_t*>(p.y) + r * p.ldy;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  for (int b = warp; b * kQBlock < p.cols; b += kRowThreads / 32) {
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

// block_rows = 1, aligned rows: a warp takes UNROLL x 256 columns of a row, eight
// per lane and vector (2 or 4 KB a warp), all loads in flight before the first is used; 16 lanes
// share a block's scale.  Bound by HBM: 8192 x 4096 fp32 (169 MB) in %QROW%.
template <typename T>
constexpr int kQuantUnroll = 4;
template <typename T>
__global__ void __launch_bounds__(256) quantize_row_vec_kernel(const QuantizeArgs p, unsigned segments, unsigned units) {
  pdl_begin();
  const unsigned u = blockIdx.x * 8 + (threadIdx.x >> 5);
  if (u >= units) return;
  const int64_t r = u / segments;
  const int n8 = (int)(p.cols / 8), i0 = (int)(u % segments) * (kQuantUnroll<T> * 32) + (threadIdx.x & 31);
  const T* x = static_cast<const T*>(p.x) + r * p.ldx;
  Vec8<T> v[kQuantUnroll<T>];
#pragma unroll
  for (int c = 0; c < kQuantUnroll<T>; ++c)
    if (i0 + c * 32 < n8) v[c].load(x + (int64_t)(i0 + c * 32) * 8);
#pragma unroll
  for (int c = 0; c < kQuantUnroll<T>; ++c) {
    const int i = i0 + c * 32;
    float amax = 0.f;
    if (i < n8) {
#pragma unroll
      for (int j = 0; j < 8; ++j) amax = max_nan(amax, fabsf(v[c].get(j)));
    }
    float scale, inv;
    block_scale(lanes16_max_nan(amax), scale, inv);
    if (i < n8) {
      *reinterpret_cast<uint2*>(p.q + r * p.ldq + (int64_t)i * 8) =
          make_uint2(to_e4m3x4(v[c].get(0) * inv, v[c].get(1) * inv, v[c].get(2) * inv, v[c].get(3) * inv),
                     to_e4m3x4(v[c].get(4) * inv, v[c].get(5) * inv, v[c].get(6) * inv, v[c].get(7) * inv));
      if ((threadIdx.x & 15) == 0) p.scale[r * p.s_row + (i / 16) * p.s_block] = scale;
    }
  }
}

// block_rows = 1, any alignment: one warp per block of 128 columns of a row.
template <typename T>
__global__ void __launch_bounds__(256) quantize_row_kernel(const QuantizeArgs p, unsigned cb, unsigned units) {
  pdl_begin();
  const int lane = threadIdx.x & 31;
  const unsigned u = blockIdx.x * 8 + (threadIdx.x >> 5);
  if (u >= units) return;
  const int64_t r = u / cb, b = u % cb;
  const T* x = static_cast<const T*>(p.x) + r * p.ldx;
  float v[4], amax = 0.f;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int64_t i = b * kQBlock + j * 32 + lane;
    v[j] = i < p.cols ? to_f32(x[i]) : 0.f;
  }
#pragma unroll
  for (int j = 0; j < 4; ++j) amax = max_nan(amax, fabsf(v[j]));
  float scale, inv;
  block_scale(warp_max_nan(amax), scale, inv);
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int64_t i = b * kQBlock + j * 32 + lane;
    if (i < p.cols) p.q[r * p.ldq + i] = to_e4m3(v[j] * inv);
  }
  if (lane == 0) p.scale[r * p.s_row + b * p.s_block] = scale;
}

// The largest magnitude over a thread block of 256.
__device__ __forceinline__ float block_max_nan(float v) {
  __shared__ float part[8];
  v = warp_max_nan(v);
  if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = v;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 8; ++i) v = max_nan(v, part[i]);
  return v;
}

// block_rows = 128, aligned rows: one thread block per block of 128 x 128, which it
// reads once (8 vectors of 8 columns per thread) and keeps in registers.
template <typename T>
__global__ void __launch_bounds__(256, sizeof(T) == 2 ? 3 : 2) quantize_tile_vec_kernel(const QuantizeArgs p, unsigned cb) {
  pdl_begin();
  const int64_t rb = blockIdx.x / cb, b = blockIdx.x % cb;
  const int64_t c = b * kQBlock + (threadIdx.x & 15) * 8, r0 = rb * 128 + (threadIdx.x >> 4);
  const T* x = static_cast<const T*>(p.x);
  Vec8<T> v[8];
#pragma unroll
  for (int i = 0; i < 8; ++i)
    if (c < p.cols && r0 + i * 16 < p.rows) v[i].load(x + (r0 + i * 16) * p.ldx + c);
  float amax = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i)
    if (c < p.cols && r0 + i * 16 < p.rows) {
#pragma unroll
      for (int j = 0; j < 8; ++j) amax = max_nan(amax, fabsf(v[i].get(j)));
    }
  float scale, inv;
  block_scale(block_max_nan(amax), scale, inv);
#pragma unroll
  for (int i = 0; i < 8; ++i)
    if (c < p.cols && r0 + i * 16 < p.rows)
      *reinterpret_cast<uint2*>(p.q + (r0 + i * 16) * p.ldq + c) =
          make_uint2(to_e4m3x4(v[i].get(0) * inv, v[i].get(1) * inv, v[i].get(2) * inv, v[i].get(3) * inv),
                     to_e4m3x4(v[i].get(4) * inv, v[i].get(5) * inv, v[i].get(6) * inv, v[i].get(7) * inv));
  if (threadIdx.x == 0) p.scale[rb * p.s_row + b * p.s_block] = scale;
}

// block_rows = 128, any alignment: V elements per access (2 where rows start on
// multiples of two elements).  The block is read twice, the second time from L2:
// keeping it in registers left too few of them for more than one block per SM.
template <typename T, int V>
__global__ void __launch_bounds__(256) quantize_tile_kernel(const QuantizeArgs p, unsigned cb) {
  pdl_begin();
  struct alignas(sizeof(T) * V) Elems { T e[V]; };
  struct alignas(V) Bytes { uint8_t e[V]; };
  constexpr int kAcross = 128 / V, kDown = 256 / kAcross;
  const int64_t rb = blockIdx.x / cb, b = blockIdx.x % cb;
  const int64_t c = b * kQBlock + threadIdx.x % kAcross * V, r0 = rb * 128 + threadIdx.x / kAcross;
  const T* x = static_cast<const T*>(p.x) + r0 * p.ldx + c;
  const int rows = c < p.cols ? (int)min((int64_t)128, p.rows - rb * 128) - (int)(threadIdx.x / kAcross) : 0;
  float amax = 0.f;
#pragma unroll 8
  for (int i = 0; i < rows; i += kDown) {
    const Elems v = *reinterpret_cast<const Elems*>(x + i * p.ldx);
#pragma unroll
    for (int j = 0; j < V; ++j) amax = max_nan(amax, fabsf(to_f32(v.e[j])));
  }
  float scale, inv;
  block_scale(block_max_nan(amax), scale, inv);
  uint8_t* q = p.q + r0 * p.ldq + c;
  for (int i0 = 0; i0 < rows; i0 += 8 * kDown) {
    Elems v[8];
#pragma unroll
    for (int k = 0; k < 8; ++k)
      if (i0 + k * kDown < rows) v[k] = *reinterpret_cast<const Elems*>(x + (i0 + k * kDown) * p.ldx);
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      if (i0 + k * kDown >= rows) break;
      Bytes w;
#pragma unroll
      for (int j = 0; j < V; ++j) w.e[j] = to_e4m3(to_f32(v[k].e[j]) * inv);
      *reinterpret_cast<Bytes*>(q + (i0 + k * kDown) * p.ldq) = w;
    }
  }
  if (threadIdx.x == 0) p.scale[rb * p.s_row + b * p.s_block] = scale;
}

bool on_grid(const void* p, int64_t ld, int es, int bytes) {
  return (reinterpret_cast<uintptr_t>(p) & (bytes - 1)) == 0 && ld * es % bytes == 0;
}

}  // namespace

int rmsnorm_launch(const RmsNormArgs& a, int num_sms, cudaStream_t st) {
  return with_type(a.type, [&](auto* t) {
    using T = std::remove_pointer_t<decltype(t)>;
    return with_type(a.weight_type, [&](auto* wt) {
      using W = std::remove_pointer_t<decltype(wt)>;
      const bool quant = a.out_type == kE4M3;
      const bool vec = a.cols % 8 == 0 && a.cols <= 4 * 512 * 8 && on_grid(a.x, a.ldx, sizeof(T), 16) &&
                       (!a.res || on_grid(a.res, a.ldr, sizeof(T), 16)) && (!a.sum || on_grid(a.sum, a.lds, sizeof(T), 16)) &&
                       on_grid(a.weight, 0, sizeof(W), 16) && on_grid(a.y, a.ldy, quant ? 1 : sizeof(T), quant ? 8 : 16);
      if (!vec) {
        const int smem = a.cols * (int)sizeof(float);
        if (smem > 48 * 1024 - 64) {
          cudaError_t e =
              cudaFuncSetAttribute(rmsnorm_row_kernel<T, W>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
          if (e != cudaSuccess) return (int)e;
        }
        return launch_pdl(rmsnorm_row_kernel<T, W>, (unsigned)a.rows, kRowThreads, smem, st, a);
      }
      // vectors per thread: 256 threads a row when there are rows enough to fill the
      // GPU (more loads in flight per thread, cheaper reductions), as many threads as
      // there are vectors when there are not
      const int n8 = a.cols / 8;
      const int want = a.rows <= 2 * num_sms ? 1024 : 256;
      const int ch = n8 <= want ? 1 : n8 <= 2 * want ? 2 : 4;
      const int threads = std::min(1024, ((n8 + ch - 1) / ch + 31) / 32 * 32);
      if (ch == 1) return launch_pdl(rmsnorm_vec_kernel<T, W, 1>, (unsigned)a.rows, threads, 0, st, a);
      if (ch == 2) return launch_pdl(rmsnorm_vec_kernel<T, W, 2>, (unsigned)a.rows, threads, 0, st, a);
      return launch_pdl(rmsnorm_vec_kernel<T, W, 4>, (unsigned)a.rows, threads, 0, st, a);
    });
  });
}

int quantize_launch(const QuantizeArgs& a, cudaStream_t st) {
  const unsigned cb = (unsigned)((a.cols + kQBlock - 1) / kQBlock);
  return with_type(a.type, [&](auto* t) {
    using T = std::remove_pointer_t<decltype(t)>;
    const bool vec = a.cols % 8 == 0 && on_grid(a.x, a.ldx, sizeof(T), 16) && on_grid(a.q, a.ldq, 1, 8);
    if (a.block_rows == 1) {
      if (vec) {
        const unsigned per = kQuantUnroll<T> * 256, segments = (unsigned)((a.cols + per - 1) / per);
        const unsigned units = (unsigned)a.rows * segments;
        return launch_pdl(quantize_row_vec_kernel<T>, (units + 7) / 8, 256, 0, st, a, segments, units);
      }
      const unsigned units = (unsigned)a.rows * cb;
      return launch_pdl(quantize_row_kernel<T>, (units + 7) / 8, 256, 0, st, a, cb, units);
    }
    const unsigned tiles = (unsigned)((a.rows + 127) / 128) * cb;
    if (vec) return launch_pdl(quantize_tile_vec_kernel<T>, tiles, 256, 0, st, a, cb);
    const bool two = a.cols % 2 == 0 && on_grid(a.x, a.ldx, sizeof(T), 2 * sizeof(T)) && on_grid(a.q, a.ldq, 1, 2);
    return two ? launch_pdl(quantize_tile_kernel<T, 2>, tiles, 256, 0, st, a, cb)
               : launch_pdl(quantize_tile_kernel<T, 1>, tiles, 256, 0, st, a, cb);
  });
}

}  // namespace ob2
