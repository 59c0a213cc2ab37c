// The 8-bit linear path: what its entry points (blocks_api.cu) and kernels
// (norm_quant.cu, gemm_blocks.cu) share.
#pragma once
#include <cuda_runtime.h>

#include <cstdint>

namespace ob2 {

constexpr int kQBlock = 128;           // columns (and weight rows) of one scale
constexpr float kE4m3Max = 448.f;
constexpr float kAmaxFloor = 0x1p-96f;  // keeps 448 / amax finite

// Element types, as ONNXB200_TYPE_*.
enum ElemType { kF32 = 0, kF16 = 1, kBF16 = 2, kE4M3 = 3 };
inline int elem_size(int t) { return t == kF32 ? 4 : t == kE4M3 ? 1 : 2; }

struct RmsNormArgs {
  const void* x;
  const void* res;     // null: none
  const void* weight;
  void* sum;           // null: not wanted
  void* y;
  float* y_scale;      // out_type == kE4M3
  int64_t rows;
  int cols;
  int64_t ldx, ldr, lds, ldy, ys_row, ys_block;
  int type, weight_type, out_type;
  float eps;
};
// Return a cudaError_t.
int rmsnorm_launch(const RmsNormArgs& a, int num_sms, cudaStream_t stream);

struct QuantizeArgs {
  const void* x;
  uint8_t* q;
  float* scale;
  int64_t rows, cols, ldx, ldq, s_row, s_block;
  int type, block_rows;
};
int quantize_launch(const QuantizeArgs& a, cudaStream_t stream);

struct MatmulBlocksArgs {
  const uint8_t* a;
  const uint8_t* b;
  const float* as;
  const float* bs;
  const float* bias;   // null: none
  void* y;
  int m, n, k;
  int64_t lda, ldb, ldy, as_row, as_block, bs_row, bs_block;
  int out_type, relu;
  int* status;         // device status word (ONNXB200_ERR_* on failure)
};
// The CUDA-core product for one or two rows of a keeps them whole in shared memory, as
// fp16 and with a scale per block of k.  Bytes in 64 bits: k goes up to 2^31.
constexpr int64_t kVecMaxSmem = 100 * 1024;  // two thread blocks per SM; longer rows go to the tensor cores
constexpr int64_t matmul_vec_smem(int m, int k) {
  return m * (((int64_t)k + 15) / 16 * 32 + ((int64_t)k + kQBlock - 1) / kQBlock * 4);
}
constexpr bool matmul_takes_vec(int m, int k) { return m <= 2 && matmul_vec_smem(m, k) <= kVecMaxSmem; }
// Many rows: tiles of 256 x 256 or 256 x 128 on num_sms / 2 pairs of thread blocks.  A
// wave of the narrow ones takes ~0.6 of a wave of the wide ones (8.5 and 16 us at k =
// 4096; 200 x 8192: 15.3 and 20.4 us, 512 x 8192: 23.4 and 21.4 us, 4096 x 4096: 70.6 and
// 67.2 us).
constexpr bool matmul_takes_wide(int m, int n, int num_sms) {
  const int64_t tm = ((int64_t)m + 255) / 256, pairs = num_sms / 2;
  const int64_t wide = (tm * (((int64_t)n + 255) / 256) + pairs - 1) / pairs;
  const int64_t narrow = (tm * (((int64_t)n + 127) / 128) + pairs - 1) / pairs;
  return 3 * narrow >= 5 * wide;
}
int matmul_blocks_launch(const MatmulBlocksArgs& a, int num_sms, cudaStream_t stream);

}  // namespace ob2
