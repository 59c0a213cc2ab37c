// C-ABI entry points of the 8-bit linear path (onnxb200_rmsnorm,
// onnxb200_quantize_blocks, onnxb200_matmul_blocks): argument checks and
// launches.  The arguments are checked before the handle is looked at, so that a
// host without a GPU can check a descriptor (with a null handle, a call whose
// arguments are all valid returns ONNXB200_ERR_INVALID_ARGUMENT).  No workspace and no device memory of the handle's is used besides
// its status word.
#include <cuda_runtime.h>

#include <climits>

#include "blocks.h"
#include "internal.h"

using namespace ob2;

namespace {

// Makes the handle's device current for a call and puts the caller's back.
struct DeviceGuard {
  int prev = -1;
  explicit DeviceGuard(int dev) {
    if (cudaGetDevice(&prev) == cudaSuccess && prev == dev)
      prev = -1;
    else
      cudaSetDevice(dev);
  }
  ~DeviceGuard() {
    if (prev >= 0) cudaSetDevice(prev);
  }
};

// An error whose message cannot be stored still has its code.
int fail(onnxb200_handle* h, int code, const char* msg) noexcept {
  try {
    return set_error(h, code, msg);
  } catch (...) {
    return code;
  }
}
int cuda_fail(onnxb200_handle* h, int e, const char* what) noexcept {
  try {
    return cuda_check(h, (cudaError_t)e, what);
  } catch (...) {
    return e == cudaErrorMemoryAllocation ? ONNXB200_ERR_RESOURCE_EXHAUSTED : ONNXB200_ERR_EXECUTION;
  }
}

constexpr int64_t kMaxDim = INT_MAX - 256;     // one dimension of a matrix
constexpr int64_t kMaxStride = int64_t(1) << 37;  // elements; keeps byte strides below 2^40

bool wide_type(int t) { return t == kF32 || t == kF16 || t == kBF16; }
bool aligned(const void* p, int bytes) { return (reinterpret_cast<uintptr_t>(p) & (bytes - 1)) == 0; }

// 0 -> dense; false if the rows would overlap or the stride is absurd.
bool resolve_ld(int64_t* ld, int64_t cols) {
  if (*ld == 0) *ld = cols;
  return *ld >= cols && *ld <= kMaxStride;
}
// Strides of a [rows][blocks] array of scales; written ones must not overlap.
bool resolve_scale(int64_t* row, int64_t* block, int64_t rows, int64_t blocks, bool written) {
  if (*row == 0 && *block == 0) {
    *row = blocks;
    *block = 1;
  }
  if (*row < 0 || *block < 0 || *row > kMaxStride || *block > kMaxStride) return false;
  if (!written || rows == 0 || blocks == 0) return true;
  const bool one_row = rows <= 1, one_block = blocks <= 1;
  if ((!one_row && *row == 0) || (!one_block && *block == 0)) return false;
  if (one_row || one_block) return true;
  return *row / blocks >= *block || *block / rows >= *row;  // products of the two pass 64 bits
}
int64_t blocks_of(int64_t v) { return (v + kQBlock - 1) / kQBlock; }

}  // namespace

extern "C" {

int onnxb200_rmsnorm(onnxb200_handle* h, const onnxb200_rmsnorm_desc* d, const void* x, const void* residual,
                     const void* weight, void* sum, void* y, float* y_scale) {
  if (!d) return fail(h, ONNXB200_ERR_INVALID_ARGUMENT, "RMSNormalization: null descriptor");
  if (!wide_type(d->type) || !wide_type(d->weight_type) ||
      (d->out_type != d->type && d->out_type != d->weight_type && d->out_type != kE4M3))
    return fail(h, ONNXB200_ERR_VALIDATION, "RMSNormalization: unsupported element type");
  if (d->rows < 0 || d->rows > kMaxDim || d->cols <= 0)
    return fail(h, ONNXB200_ERR_VALIDATION, "RMSNormalization: invalid shape");
  if (d->cols > ONNXB200_RMSNORM_MAX_COLS)
    return fail(h, ONNXB200_ERR_UNSUPPORTED, "RMSNormalization: rows longer than ONNXB200_RMSNORM_MAX_COLS");
  if (!(d->epsilon >= 0.f)) return fail(h, ONNXB200_ERR_VALIDATION, "RMSNormalization: epsilon must not be negative");
  RmsNormArgs a{x,          residual,    weight, sum,    y,      y_scale, d->rows,          (int)d->cols,
                d->ldx,     d->ldr,      d->lds, d->ldy, d->y_scale_row, d->y_scale_block, d->type,
                d->weight_type, d->out_type, d->epsilon};
  if (!resolve_ld(&a.ldx, d->cols) || !resolve_ld(&a.ldr, d->cols) || !resolve_ld(&a.lds, d->cols) ||
      !resolve_ld(&a.ldy, d->cols))
    return fail(h, ONNXB200_ERR_VALIDATION, "RMSNormalization: row stride shorter than a row");
  if (d->out_type == kE4M3 && !resolve_scale(&a.ys_row, &a.ys_block, d->rows, blocks_of(d->cols), true))
    return fail(h, ONNXB200_ERR_VALIDATION, "RMSNormalization: scale strides overlap");
  if (d->rows == 0) return h ? ONNXB200_OK : ONNXB200_ERR_INVALID_ARGUMENT;
  if (!x || !weight || !y || (d->out_type == kE4M3 && !y_scale))
    return fail(h, ONNXB200_ERR_INVALID_ARGUMENT, "RMSNormalization: null argument");
  const int es = elem_size(d->type);
  if (!aligned(x, es) || !aligned(residual, es) || !aligned(sum, es) || !aligned(weight, elem_size(d->weight_type)) ||
      !aligned(y, elem_size(d->out_type)) || !aligned(y_scale, 4))
    return fail(h, ONNXB200_ERR_VALIDATION, "RMSNormalization: pointer not aligned to its type");
  if (!h) return ONNXB200_ERR_INVALID_ARGUMENT;
  DeviceGuard g(h->device);
  const int rc = rmsnorm_launch(a, h->num_sms, h->stream);
  h->launches++;
  return rc ? cuda_fail(h, rc, "RMSNormalization") : ONNXB200_OK;
}

int onnxb200_quantize_blocks(onnxb200_handle* h, const onnxb200_quantize_desc* d, const void* x, void* q,
                             float* scale) {
  if (!d) return fail(h, ONNXB200_ERR_INVALID_ARGUMENT, "QuantizeBlocks: null descriptor");
  if (!wide_type(d->type)) return fail(h, ONNXB200_ERR_VALIDATION, "QuantizeBlocks: unsupported element type");
  if (d->block_rows != 1 && d->block_rows != kQBlock)
    return fail(h, ONNXB200_ERR_VALIDATION, "QuantizeBlocks: block_rows must be 1 or 128");
  if (d->rows < 0 || d->cols < 0 || d->rows > kMaxDim || d->cols > kMaxDim)
    return fail(h, ONNXB200_ERR_VALIDATION, "QuantizeBlocks: invalid shape");
  QuantizeArgs a{x, static_cast<uint8_t*>(q), scale, d->rows, d->cols, d->ldx, d->ldq, d->scale_row,
                 d->scale_block, d->type, d->block_rows};
  if (!resolve_ld(&a.ldx, d->cols) || !resolve_ld(&a.ldq, d->cols))
    return fail(h, ONNXB200_ERR_VALIDATION, "QuantizeBlocks: row stride shorter than a row");
  const int64_t rb = d->block_rows == 1 ? d->rows : blocks_of(d->rows), cb = blocks_of(d->cols);
  if (!resolve_scale(&a.s_row, &a.s_block, rb, cb, true))
    return fail(h, ONNXB200_ERR_VALIDATION, "QuantizeBlocks: scale strides overlap");
  if (d->rows == 0 || d->cols == 0) return h ? ONNXB200_OK : ONNXB200_ERR_INVALID_ARGUMENT;
  if (rb * cb > kMaxDim) return fail(h, ONNXB200_ERR_UNSUPPORTED, "QuantizeBlocks: matrix too large");
  if (!x || !q || !scale) return fail(h, ONNXB200_ERR_INVALID_ARGUMENT, "QuantizeBlocks: null argument");
  if (!aligned(x, elem_size(d->type)) || !aligned(scale, 4))
    return fail(h, ONNXB200_ERR_VALIDATION, "QuantizeBlocks: pointer not aligned to its type");
  if (!h) return ONNXB200_ERR_INVALID_ARGUMENT;
  DeviceGuard g(h->device);
  const int rc = quantize_launch(a, h->stream);
  h->launches++;
  return rc ? cuda_fail(h, rc, "QuantizeBlocks") : ONNXB200_OK;
}

int onnxb200_matmul_blocks(onnxb200_handle* h, const onnxb200_matmul_blocks_desc* d, const void* a,
                           const float* a_scale, const void* b, const float* b_scale, const float* bias, void* y) {
  if (!d) return fail(h, ONNXB200_ERR_INVALID_ARGUMENT, "MatMulBlockScaled: null descriptor");
  if (!wide_type(d->out_type)) return fail(h, ONNXB200_ERR_VALIDATION, "MatMulBlockScaled: unsupported element type");
  if (d->flags & ~ONNXB200_EPI_RELU) return fail(h, ONNXB200_ERR_VALIDATION, "MatMulBlockScaled: unknown flag");
  if (d->m < 0 || d->n < 0 || d->k < 0 || d->m > kMaxDim || d->n > kMaxDim || d->k > kMaxDim)
    return fail(h, ONNXB200_ERR_VALIDATION, "MatMulBlockScaled: invalid shape");
  MatmulBlocksArgs p{static_cast<const uint8_t*>(a), static_cast<const uint8_t*>(b), a_scale, b_scale, bias, y,
                     (int)d->m, (int)d->n, (int)d->k, d->lda, d->ldb, d->ldy, d->a_scale_row, d->a_scale_block,
                     d->b_scale_row, d->b_scale_block, d->out_type, (d->flags & ONNXB200_EPI_RELU) ? 1 : 0,
                     h ? h->d_status : nullptr};
  if (!resolve_ld(&p.lda, d->k) || !resolve_ld(&p.ldb, d->k) || !resolve_ld(&p.ldy, d->n))
    return fail(h, ONNXB200_ERR_VALIDATION, "MatMulBlockScaled: row stride shorter than a row");
  if (!resolve_scale(&p.as_row, &p.as_block, d->m, blocks_of(d->k), false) ||
      !resolve_scale(&p.bs_row, &p.bs_block, blocks_of(d->n), blocks_of(d->k), false))
    return fail(h, ONNXB200_ERR_VALIDATION, "MatMulBlockScaled: invalid scale strides");
  if (d->m == 0 || d->n == 0) return h ? ONNXB200_OK : ONNXB200_ERR_INVALID_ARGUMENT;
  // the product's tiles are counted in 32 bits
  if (blocks_of(d->n) * blocks_of(d->m) > kMaxDim / 16)
    return fail(h, ONNXB200_ERR_UNSUPPORTED, "MatMulBlockScaled: matrix too large");
  if (!y || (d->k > 0 && (!a || !a_scale || !b || !b_scale)))
    return fail(h, ONNXB200_ERR_INVALID_ARGUMENT, "MatMulBlockScaled: null argument");
  if (!aligned(a_scale, 4) || !aligned(b_scale, 4) || !aligned(bias, 4) || !aligned(y, elem_size(d->out_type)))
    return fail(h, ONNXB200_ERR_VALIDATION, "MatMulBlockScaled: pointer not aligned to its type");
  if (!h) return ONNXB200_ERR_INVALID_ARGUMENT;
  DeviceGuard g(h->device);
  // the stride of a single row is never used: the one its bytes would have
  if (d->m == 1) p.lda = (d->k + 15) / 16 * 16;
  if (d->n == 1) p.ldb = (d->k + 15) / 16 * 16;
  const int rc = matmul_blocks_launch(p, h->num_sms, h->stream);
  h->launches++;
  return rc ? cuda_fail(h, rc, "MatMulBlockScaled") : ONNXB200_OK;
}

}  // extern "C"
