// Root-mean-square normalisation (with the residual's addition in front and the
// quantisation behind it) and block quantisation to e4m3.
#include <algorithm>

#include "../../include/onnxb200.h"
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
  uint32_t v[2 * sizeof(T)];
  __device__ __forceinline__ void load(const T* p, bool in_range) {
#pragma unroll
    for (int i = 0; i < (int)sizeof(T) / 2; ++i) {
      const uint4 u = in_range ? reinterpret_cast<const uint4*>(p)[i] : make_uint4(0, 0, 0, 0);
      v[i * 4] = u.x;
      v[i * 4 + 1] = u.y;
      v[i * 4 + 2] = u.z;
      v[i * 4 + 3] = u.w;
    }
  }
  __device__ __forceinline__ void unpack(float (&f)[8]) const {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      if constexpr (std::is_same_v<T, float>)
        f[i] = __uint_as_float(v[i]);
      else if constexpr (std::is_same_v<T, __nv_bfloat16>)
        f[i] = __uint_as_float(i & 1 ? v[i / 2] & 0xffff0000u : v[i / 2] << 16);
      else
        f[i] = __half2float(__ushort_as_half((unsigned short)(v[i / 2] >> (i & 1 ? 16 : 0))));
    }
  }
  __device__ __forceinline__ void pack(const float (&f)[8]) {
    if constexpr (std::is_same_v<T, float>) {
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = __float_as_uint(f[i]);
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] = pack_rounded<T>(f[2 * i], f[2 * i + 1]);
    }
  }
  __device__ __forceinline__ void store(T* p) const {
#pragma unroll
    for (int i = 0; i < (int)sizeof(T) / 2; ++i)
      reinterpret_cast<uint4*>(p)[i] = make_uint4(v[i * 4], v[i * 4 + 1], v[i * 4 + 2], v[i * 4 + 3]);
  }
  // Largest magnitude; 16-bit types two at a time, in their own type (it is exact).
  __device__ __forceinline__ float amax() const {
    if constexpr (std::is_same_v<T, float>) {
      float m = 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) m = max_abs_nan(m, __uint_as_float(v[i]));
      return m;
    } else {
      uint32_t m = v[0] & 0x7fff7fffu;
#pragma unroll
      for (int i = 1; i < 4; ++i) {
        if constexpr (std::is_same_v<T, __half>)
          asm("max.NaN.f16x2 %0, %0, %1;" : "+r"(m) : "r"(v[i] & 0x7fff7fffu));
        else
          asm("max.NaN.bf16x2 %0, %0, %1;" : "+r"(m) : "r"(v[i] & 0x7fff7fffu));
      }
      const unsigned short lo = (unsigned short)m, hi = (unsigned short)(m >> 16);
      if constexpr (std::is_same_v<T, __half>)
        return max_nan(__half2float(__ushort_as_half(lo)), __half2float(__ushort_as_half(hi)));
      else
        return max_nan(__uint_as_float((uint32_t)lo << 16), __uint_as_float((uint32_t)hi << 16));
    }
  }
};

// f(row r of y) in y's type: x's, or the weight's.
template <typename T, typename W, typename F>
__device__ __forceinline__ void with_out(const RmsNormArgs& p, int64_t r, F f) {
  if (std::is_same_v<T, W> || p.out_type == p.type)
    f(static_cast<T*>(p.y) + r * p.ldy);
  else
    f(static_cast<W*>(p.y) + r * p.ldy);
}

// Eight values times inv, in e4m3.
__device__ __forceinline__ void store_e4m3(uint8_t* p, const float (&f)[8], float inv) {
  *reinterpret_cast<uint2*>(p) = make_uint2(to_e4m3x4(f[0] * inv, f[1] * inv, f[2] * inv, f[3] * inv),
                                            to_e4m3x4(f[4] * inv, f[5] * inv, f[6] * inv, f[7] * inv));
}

// The scales of N vectors (1, 2 or 4) per lane, each vector's block being spread
// over the 16 lanes of a half warp: `amax` holds a lane's largest magnitudes, inv[c]
// receives the factor of vector c's block.  The maxima are exchanged so that each
// lane ends with one block's, and the two divisions of a block are done by one lane
// in four or so instead of by all 16: they were a quarter of all instructions of
// kernels whose instructions, not bytes, set the time.  The block that a lane ended
// with is returned, and its scale.
template <int N>
__device__ __forceinline__ int half_warp_scales(const float (&amax)[N], float (&inv)[N], float& scale) {
  const int lane = threadIdx.x & 31;
  float m;
  int mine;
  if constexpr (N == 4) {
    const bool up = lane & 8, up2 = lane & 4;
    float a = up ? amax[2] : amax[0], b = up ? amax[3] : amax[1];
    a = max_nan(a, __shfl_xor_sync(0xffffffffu, up ? amax[0] : amax[2], 8));
    b = max_nan(b, __shfl_xor_sync(0xffffffffu, up ? amax[1] : amax[3], 8));
    m = max_nan(up2 ? b : a, __shfl_xor_sync(0xffffffffu, up2 ? a : b, 4));
    mine = (lane >> 2) & 3;
  } else if constexpr (N == 2) {
    const bool up = lane & 8;
    m = max_nan(up ? amax[1] : amax[0], __shfl_xor_sync(0xffffffffu, up ? amax[0] : amax[1], 8));
    m = max_nan(m, __shfl_xor_sync(0xffffffffu, m, 4));
    mine = (lane >> 3) & 1;
  } else {
    m = max_nan(amax[0], __shfl_xor_sync(0xffffffffu, amax[0], 8));
    m = max_nan(m, __shfl_xor_sync(0xffffffffu, m, 4));
    mine = 0;
  }
  m = max_nan(m, __shfl_xor_sync(0xffffffffu, m, 2));
  m = max_nan(m, __shfl_xor_sync(0xffffffffu, m, 1));
  float f;
  block_scale(m, scale, f);
#pragma unroll
  for (int c = 0; c < N; ++c)
    inv[c] = N == 1 ? f : __shfl_sync(0xffffffffu, f, (lane & 16) | c * (16 / N));
  return mine;
}
// Whether this lane writes the scale it ended with.
template <int N>
__device__ __forceinline__ bool writes_scale() {
  return (threadIdx.x & (16 / N - 1)) == 0;
}

// Rows whose every vector is aligned: one row per block, or (WARP) per warp of a block
// of 256 threads, CH vectors of eight columns per thread, read once and kept in
// registers; the weight is on its way
// before the row's one reduction (a shuffle and a barrier).  Bound by HBM with
// several blocks per SM taking turns; blocks that walk rows with the next two rows
// copied ahead were slower (107 against 84 us then: fewer blocks, and the same chain
// of reductions).  8192 x 8192 bf16 with residual and e4m3 output (470 MB): 73 us,
// 6.4 TB/s (run without a pause, at 1.6 GHz under the power cap, 78 to 80); one row of
// 4096 2.6 to 2.9 us.
template <typename T, typename W, int CH, bool WARP = false>
__global__ void __launch_bounds__(WARP ? 256 : CH == 4 ? 512 : 1024, CH == 4 && sizeof(T) == 2 ? (WARP ? 4 : 2) : 1)
    rmsnorm_vec_kernel(const RmsNormArgs p) {
  __shared__ float part[32];
  pdl_begin();
  const int64_t r = WARP ? (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5) : blockIdx.x;
  if (WARP && r >= p.rows) return;
  const int n8 = p.cols / 8, nt = WARP ? 32 : blockDim.x, tid = WARP ? threadIdx.x & 31 : threadIdx.x;
  // vector c of this thread; threads past the row's end work on zeros
  auto at = [&](int c) { return c * nt + tid; };
  const T* x = static_cast<const T*>(p.x) + r * p.ldx;
  float h[CH][8];
  {
    Vec8<T> v[CH];
#pragma unroll
    for (int c = 0; c < CH; ++c) v[c].load(x + at(c) * 8, at(c) < n8);
    if (p.res) {
      const T* res = static_cast<const T*>(p.res) + r * p.ldr;
      Vec8<T> vr[CH];
#pragma unroll
      for (int c = 0; c < CH; ++c) vr[c].load(res + at(c) * 8, at(c) < n8);
#pragma unroll
      for (int c = 0; c < CH; ++c) {
        float f[8];
        v[c].unpack(h[c]);
        vr[c].unpack(f);
#pragma unroll
        for (int j = 0; j < 8; ++j) h[c][j] += f[j];
      }
    } else {
#pragma unroll
      for (int c = 0; c < CH; ++c) v[c].unpack(h[c]);
    }
  }
  Vec8<W> vw[CH];
#pragma unroll
  for (int c = 0; c < CH; ++c) vw[c].load(static_cast<const W*>(p.weight) + at(c) * 8, at(c) < n8);
  // A sum per vector, then pairs: 8 + log2(CH) + 5 roundings lie on the way of a square
  // (and 5 over the warps of a block), where one sum per thread has up to 32 + 5 and was
  // wrong by as much for a row of one large element and many small ones.
  float ss, sq[CH];
#pragma unroll
  for (int c = 0; c < CH; ++c) {
    sq[c] = 0.f;
#pragma unroll
    for (int j = 0; j < 8; ++j) sq[c] = fmaf(h[c][j], h[c][j], sq[c]);
  }
  if constexpr (CH == 4)
    ss = (sq[0] + sq[1]) + (sq[2] + sq[3]);
  else if constexpr (CH == 2)
    ss = sq[0] + sq[1];
  else
    ss = sq[0];
  ss = warp_sum(ss);
  if (!WARP && (threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = ss;
  if (p.sum) {
    T* sum = static_cast<T*>(p.sum) + r * p.lds;
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      Vec8<T> o;
      o.pack(h[c]);
      if (at(c) < n8) o.store(sum + at(c) * 8);
    }
  }
  if (!WARP) {
    __syncthreads();
    ss = (threadIdx.x & 31) < nt / 32 ? part[threadIdx.x & 31] : 0.f;
    ss = warp_sum(ss);
  }
  const float rstd = 1.f / sqrtf(ss / (float)p.cols + p.eps);
  float amax[CH];
#pragma unroll
  for (int c = 0; c < CH; ++c) {
    float f[8];
    vw[c].unpack(f);
#pragma unroll
    for (int j = 0; j < 8; ++j) h[c][j] = h[c][j] * rstd * f[j];
  }
  if (p.out_type != kE4M3) {
    with_out<T, W>(p, r, [&](auto* y) {
#pragma unroll
      for (int c = 0; c < CH; ++c) {
        Vec8<std::remove_pointer_t<decltype(y)>> o;
        o.pack(h[c]);
        if (at(c) < n8) o.store(y + at(c) * 8);
      }
    });
    return;
  }
#pragma unroll
  for (int c = 0; c < CH; ++c) {
    amax[c] = 0.f;
#pragma unroll
    for (int j = 0; j < 8; ++j) amax[c] = max_abs_nan(amax[c], h[c][j]);
  }
  float inv[CH], scale;
  const int mine = at(half_warp_scales<CH>(amax, inv, scale)) / 16;
  if (writes_scale<CH>() && mine * 16 < n8) p.y_scale[r * p.ys_row + mine * p.ys_block] = scale;
  uint8_t* q = static_cast<uint8_t*>(p.y) + r * p.ldy;
#pragma unroll
  for (int c = 0; c < CH; ++c)
    if (at(c) < n8) store_e4m3(q + at(c) * 8, h[c], inv[c]);
}

// Any alignment, up to 4096 columns: one row per thread block, blocks of 128 columns
// dealt to its warps (NB each, four columns a lane), all elements of x, the residual
// and the weight on their way before the first is used; h stays in registers.  Bound
// by instructions, an element each (80% of the issue slots): 4096 x 1001 fp16 with
// residual and e4m3 output (29 MB) 13.7 us, fp32 without (33 MB) 9.4 us.
constexpr int kRowThreads = 512;
template <typename T, typename W, int NB>
__global__ void __launch_bounds__(kRowThreads, NB == 1 ? 4 : 2) rmsnorm_elem_kernel(const RmsNormArgs p) {
  __shared__ float part[kRowThreads / 32];
  pdl_begin();
  const int64_t r = blockIdx.x;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, warps = blockDim.x >> 5;
  const T* x = static_cast<const T*>(p.x) + r * p.ldx;
  const W* w = static_cast<const W*>(p.weight);
  auto block = [&](int c) { return c * warps + warp; };
  auto at = [&](int c, int j) { return block(c) * kQBlock + j * 32 + lane; };
  float h[NB][4];
  {
    T a[NB][4];
#pragma unroll
    for (int c = 0; c < NB; ++c)
#pragma unroll
      for (int j = 0; j < 4; ++j) a[c][j] = at(c, j) < p.cols ? x[at(c, j)] : from_f32<T>(0.f);
    if (p.res) {
      const T* res = static_cast<const T*>(p.res) + r * p.ldr;
      T b[NB][4];
#pragma unroll
      for (int c = 0; c < NB; ++c)
#pragma unroll
        for (int j = 0; j < 4; ++j) b[c][j] = at(c, j) < p.cols ? res[at(c, j)] : from_f32<T>(0.f);
#pragma unroll
      for (int c = 0; c < NB; ++c)
#pragma unroll
        for (int j = 0; j < 4; ++j) h[c][j] = to_f32(a[c][j]) + to_f32(b[c][j]);
    } else {
#pragma unroll
      for (int c = 0; c < NB; ++c)
#pragma unroll
        for (int j = 0; j < 4; ++j) h[c][j] = to_f32(a[c][j]);
    }
  }
  W g[NB][4];
#pragma unroll
  for (int c = 0; c < NB; ++c)
#pragma unroll
    for (int j = 0; j < 4; ++j) g[c][j] = at(c, j) < p.cols ? w[at(c, j)] : from_f32<W>(0.f);
  float ss = 0.f;
#pragma unroll
  for (int c = 0; c < NB; ++c)
#pragma unroll
    for (int j = 0; j < 4; ++j) ss = fmaf(h[c][j], h[c][j], ss);
  ss = warp_sum(ss);
  if (lane == 0) part[warp] = ss;
  if (p.sum) {
    T* sum = static_cast<T*>(p.sum) + r * p.lds;
#pragma unroll
    for (int c = 0; c < NB; ++c)
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (at(c, j) < p.cols) sum[at(c, j)] = from_f32<T>(h[c][j]);
  }
  __syncthreads();
  float tot = 0.f;
  for (int i = 0; i < warps; ++i) tot += part[i];
  const float rstd = 1.f / sqrtf(tot / (float)p.cols + p.eps);
  float amax[NB];
#pragma unroll
  for (int c = 0; c < NB; ++c) {
    amax[c] = 0.f;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      h[c][j] = h[c][j] * rstd * to_f32(g[c][j]);
      if (at(c, j) < p.cols) amax[c] = max_nan(amax[c], fabsf(h[c][j]));
    }
  }
  if (p.out_type != kE4M3) {
    with_out<T, W>(p, r, [&](auto* y) {
#pragma unroll
      for (int c = 0; c < NB; ++c)
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (at(c, j) < p.cols) y[at(c, j)] = from_f32<std::remove_pointer_t<decltype(y)>>(h[c][j]);
    });
    return;
  }
  uint8_t* q = static_cast<uint8_t*>(p.y) + r * p.ldy;
#pragma unroll
  for (int c = 0; c < NB; ++c) amax[c] = warp_max_nan(amax[c]);
#pragma unroll
  for (int c = 0; c < NB; ++c) {
    float scale, inv;
    block_scale(amax[c], scale, inv);
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (at(c, j) < p.cols) q[at(c, j)] = to_e4m3(h[c][j] * inv);
    if (lane == 0 && block(c) * kQBlock < p.cols) p.y_scale[r * p.ys_row + block(c) * p.ys_block] = scale;
  }
}

// Any alignment and width: one row per block, the row's fp32 sum x + residual held
// in shared memory.  Bound by instructions, an element each (82% of the issue slots):
// 333 x 5001 fp16 with residual and e4m3 output (12 MB) 8.0 us, 8192 x 8001 bf16 (459
// MB) 136 to 143 us; aligned rows of more than 16384 columns take it too (1024 x 20000
// bf16 64 us, 2.2 TB/s).
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
    with_out<T, W>(p, r, [&](auto* y) {
      for (int i = threadIdx.x; i < p.cols; i += kRowThreads)
        y[i] = from_f32<std::remove_pointer_t<decltype(y)>>(row[i] * rstd * to_f32(w[i]));
    });
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
// share a block's scale.  Bound by HBM: 8192 x 4096 fp32 (168 MB) in 27.3 us, 6.2 TB/s;
// 8192 x 8192 bf16 in 32.8 us, 6.1 TB/s (34.7 run without a pause, at 1.75 GHz).
constexpr int kQuantUnroll = 4;
template <typename T>
__global__ void __launch_bounds__(256) quantize_row_vec_kernel(const QuantizeArgs p, unsigned segments, unsigned units) {
  pdl_begin();
  const unsigned u = blockIdx.x * 8 + (threadIdx.x >> 5);
  if (u >= units) return;
  const int64_t r = u / segments;
  const int n8 = (int)(p.cols / 8), i0 = (int)(u % segments) * (kQuantUnroll * 32) + (threadIdx.x & 31);
  const T* x = static_cast<const T*>(p.x) + r * p.ldx;
  Vec8<T> v[kQuantUnroll];
#pragma unroll
  for (int c = 0; c < kQuantUnroll; ++c) v[c].load(x + (int64_t)(i0 + c * 32) * 8, i0 + c * 32 < n8);
  float amax[kQuantUnroll], inv[kQuantUnroll], scale;
#pragma unroll
  for (int c = 0; c < kQuantUnroll; ++c) amax[c] = v[c].amax();
  const int mine = (i0 + half_warp_scales<kQuantUnroll>(amax, inv, scale) * 32) / 16;
  if (writes_scale<kQuantUnroll>() && mine * 16 < n8) p.scale[r * p.s_row + mine * p.s_block] = scale;
  uint8_t* q = p.q + r * p.ldq;
#pragma unroll
  for (int c = 0; c < kQuantUnroll; ++c) {
    float f[8];
    v[c].unpack(f);
    if (i0 + c * 32 < n8) store_e4m3(q + (int64_t)(i0 + c * 32) * 8, f, inv[c]);
  }
}

// block_rows = 1, any alignment: one warp per block of 128 columns of a row.  Bound by
// instructions, an element each (81% of the issue slots): 4096 x 4099 bf16 (50 MB) and
// fp32 (84 MB) 28 us.
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
// reads once (8 vectors of 8 columns per thread) and keeps in registers.  8192 x 8192
// fp32 51.3 us (6.5 TB/s), bf16 34.6 us (5.8 TB/s); 52.3 and 35.6 run without a pause.
template <typename T>
__global__ void __launch_bounds__(256, sizeof(T) == 2 ? 3 : 2) quantize_tile_vec_kernel(const QuantizeArgs p, unsigned cb) {
  pdl_begin();
  const int64_t rb = blockIdx.x / cb, b = blockIdx.x % cb;
  const int64_t c = b * kQBlock + (threadIdx.x & 15) * 8, r0 = rb * 128 + (threadIdx.x >> 4);
  const T* x = static_cast<const T*>(p.x);
  Vec8<T> v[8];
  auto in_range = [&](int i) { return c < p.cols && r0 + i * 16 < p.rows; };
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i].load(x + (r0 + i * 16) * p.ldx + c, in_range(i));
  float amax = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) amax = max_nan(amax, v[i].amax());
  float scale, inv;
  block_scale(block_max_nan(amax), scale, inv);
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    float f[8];
    v[i].unpack(f);
    if (in_range(i)) store_e4m3(p.q + (r0 + i * 16) * p.ldq + c, f, inv);
  }
  if (threadIdx.x == 0) p.scale[rb * p.s_row + b * p.s_block] = scale;
}

// block_rows = 128, any alignment: V elements per access (2 where rows start on
// multiples of two elements), eight rows of loads in flight; the block is read a
// second time, from L2 (in registers it left room for one block per SM, or was
// slower by its guards).  5000 x 2050 bf16 (31 MB): 9.8 us, 3.1 TB/s.
template <typename T, int V>
__global__ void __launch_bounds__(256) quantize_tile_kernel(const QuantizeArgs p, unsigned cb) {
  pdl_begin();
  struct alignas(sizeof(T) * V) Elems { T e[V]; };
  struct alignas(V) Bytes { uint8_t e[V]; };
  constexpr int kAcross = 128 / V, kDown = 256 / kAcross, kBatch = 8;
  const int64_t rb = blockIdx.x / cb, b = blockIdx.x % cb;
  const int64_t c = b * kQBlock + threadIdx.x % kAcross * V, r0 = rb * 128 + threadIdx.x / kAcross;
  const char* x = reinterpret_cast<const char*>(static_cast<const T*>(p.x) + r0 * p.ldx + c);
  const int64_t step = kDown * p.ldx * (int64_t)sizeof(T), qstep = kDown * p.ldq;
  uint8_t* q = p.q + r0 * p.ldq + c;
  // rows of this thread: r0 + i * kDown for i < mine
  const int left = c < p.cols ? (int)min((int64_t)128, p.rows - rb * 128) - (int)(threadIdx.x / kAcross) : 0;
  const int mine = left > 0 ? (left + kDown - 1) / kDown : 0;
  auto amax_of = [](const Elems& v) {
    float m = 0.f;
#pragma unroll
    for (int j = 0; j < V; ++j) m = max_abs_nan(m, to_f32(v.e[j]));
    return m;
  };
  auto put = [&](uint8_t* to, const Elems& v, float inv) {
    Bytes w;
    if constexpr (V == 2) {
      uint16_t two;
      asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(two) : "f"(to_f32(v.e[1]) * inv), "f"(to_f32(v.e[0]) * inv));
      *reinterpret_cast<uint16_t*>(to) = two;
    } else {
      w.e[0] = to_e4m3(to_f32(v.e[0]) * inv);
      *reinterpret_cast<Bytes*>(to) = w;
    }
  };
  // f(pointer, row index) over this thread's rows, kBatch at a time
  auto walk = [&](auto batch, auto single) {
    const char* at = x;
    int i = 0;
    for (; i + kBatch <= mine; i += kBatch) {
      Elems v[kBatch];
#pragma unroll
      for (int k = 0; k < kBatch; ++k, at += step) v[k] = *reinterpret_cast<const Elems*>(at);
      batch(v);
    }
    for (; i < mine; ++i, at += step) single(*reinterpret_cast<const Elems*>(at));
  };
  float amax = 0.f;
  walk(
      [&](const Elems (&v)[kBatch]) {
#pragma unroll
        for (int k = 0; k < kBatch; ++k) amax = max_nan(amax, amax_of(v[k]));
      },
      [&](const Elems& v) { amax = max_nan(amax, amax_of(v)); });
  float scale, inv;
  block_scale(block_max_nan(amax), scale, inv);
  walk(
      [&](const Elems (&v)[kBatch]) {
#pragma unroll
        for (int k = 0; k < kBatch; ++k, q += qstep) put(q, v[k], inv);
      },
      [&](const Elems& v) {
        put(q, v, inv);
        q += qstep;
      });
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
                       on_grid(a.weight, 0, sizeof(W), 16) && on_grid(a.y, a.ldy, elem_size(a.out_type), quant ? 8 : 16);
      // Short rows off the grid stay in registers, a warp for one or two blocks of columns
      // (4096 x 1001 fp16: 13.7 us, 22.6 in shared memory; 4096 x 3001 bf16 28.4 and 30.0);
      // with four a warp the registers left too few warps (8192 x 8001: 167 us and 138).
      const int nb = (a.cols + kQBlock - 1) / kQBlock;
      if (!vec && nb <= 16) return launch_pdl(rmsnorm_elem_kernel<T, W, 1>, (unsigned)a.rows, nb * 32, 0, st, a);
      if (!vec && nb <= 32) return launch_pdl(rmsnorm_elem_kernel<T, W, 2>, (unsigned)a.rows, (nb + 1) / 2 * 32, 0, st, a);
      if (!vec) {
        const int smem = a.cols * (int)sizeof(float);
        if (smem > 48 * 1024 - 64) {
          const int rc = opt_in<rmsnorm_row_kernel<T, W>>(ONNXB200_RMSNORM_MAX_COLS * (int)sizeof(float));
          if (rc) return rc;
        }
        return launch_pdl(rmsnorm_row_kernel<T, W>, (unsigned)a.rows, kRowThreads, smem, st, a);
      }
      // With rows enough to fill the GPU: a warp a row up to 1024 columns (8192 x 128
      // bf16: 3.3 us against 10.0 with a block a row), then few threads with more
      // loads in flight each and cheaper reductions (8192 x 2048 with residual and e4m3
      // output: 20.9 us with 128 threads, 23.2 with 256).  Otherwise as many threads as there are vectors.
      const int n8 = a.cols / 8;
      const bool many = a.rows > 2 * num_sms;
      if (many && n8 <= 128) {
        const unsigned grid = (unsigned)((a.rows + 7) / 8);
        if (n8 <= 32) return launch_pdl(rmsnorm_vec_kernel<T, W, 1, true>, grid, 256, 0, st, a);
        if (n8 <= 64) return launch_pdl(rmsnorm_vec_kernel<T, W, 2, true>, grid, 256, 0, st, a);
        return launch_pdl(rmsnorm_vec_kernel<T, W, 4, true>, grid, 256, 0, st, a);
      }
      const int want = many ? 128 : 1024;
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
        const unsigned per = kQuantUnroll * 256, segments = (unsigned)((a.cols + per - 1) / per);
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
