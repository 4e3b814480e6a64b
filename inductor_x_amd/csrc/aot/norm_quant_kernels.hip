// Instantiations of the residual add + RMS norm with an 8-bit result (norm_quant.h): element type, threads per
// row and pieces per thread, one scale per row or per 128 columns, aligned or unaligned access.
#include "../mi/norm_quant.h"

using namespace mi;

#define NORM_QUANT(TN, T, BLOCK, TPR, ITERS, GN, GROUPED, WN, WIDE)                                        \
  extern "C" __global__ __launch_bounds__(BLOCK) void add_rmsnorm_quant_##TN##_b##BLOCK##_t##TPR##_i##ITERS##GN##WN( \
      const T* h, const T* r, const T* w, uint8_t* q, float* scales, T* s, int rows, int cols,             \
      long long h_stride, long long r_stride, float eps) {                                                 \
    add_rmsnorm_quant<T, BLOCK, TPR, ITERS, GROUPED, WIDE>(h, r, w, q, scales, s, rows, cols, h_stride, r_stride, eps); \
  }
#define NORM_QUANT_FORMS(TN, T, BLOCK, TPR, ITERS)             \
  NORM_QUANT(TN, T, BLOCK, TPR, ITERS, , false, , true)        \
  NORM_QUANT(TN, T, BLOCK, TPR, ITERS, _g128, true, , true)    \
  NORM_QUANT(TN, T, BLOCK, TPR, ITERS, , false, _odd, false)   \
  NORM_QUANT(TN, T, BLOCK, TPR, ITERS, _g128, true, _odd, false)
#define NORM_QUANT_SIZES(TN, T)            \
  NORM_QUANT_FORMS(TN, T, 256, 16, 1)      \
  NORM_QUANT_FORMS(TN, T, 256, 32, 1)      \
  NORM_QUANT_FORMS(TN, T, 256, 64, 1)      \
  NORM_QUANT_FORMS(TN, T, 256, 64, 2)      \
  NORM_QUANT_FORMS(TN, T, 256, 256, 1)     \
  NORM_QUANT_FORMS(TN, T, 512, 512, 1)     \
  NORM_QUANT_FORMS(TN, T, 512, 512, 2)     \
  NORM_QUANT_FORMS(TN, T, 1024, 1024, 2)   \
  NORM_QUANT_FORMS(TN, T, 1024, 1024, 4)

NORM_QUANT_SIZES(bf16, bf16_t)
NORM_QUANT_SIZES(f16, f16_t)
