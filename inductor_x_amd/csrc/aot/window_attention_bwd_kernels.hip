// Instantiations of the gradients of attention with a sliding window and visible first tokens (window_attention_bwd.h).
#include "../mi/window_attention_bwd.h"

using namespace mi;

#define WINDOW_BWD(TN, T, DH)                                                                                       \
  extern "C" __global__ __launch_bounds__(512, 1) void window_attention_bwd_dq_##TN##_d##DH(WindowBwdArgs args) {   \
    window_bwd_dq<T, DH>(args);                                                                                     \
  }                                                                                                                 \
  /* gridDim.y = 2: dK, dV */                                                                                       \
  extern "C" __global__ __launch_bounds__(512, 1) void window_attention_bwd_dkv_##TN##_d##DH(WindowBwdArgs args) {  \
    if (blockIdx.y == 0)                                                                                            \
      window_bwd_dkv<T, DH, 0>(args);                                                                               \
    else                                                                                                            \
      window_bwd_dkv<T, DH, 1>(args);                                                                               \
  }                                                                                                                 \
  extern "C" __global__ __launch_bounds__(256, 1) void window_attention_bwd_sinks_##TN##_d##DH(WindowBwdArgs args) { \
    window_bwd_sinks<T, DH>(args);                                                                                  \
  }                                                                                                                 \
  extern "C" __global__ __launch_bounds__(2 * DH) void window_attention_bwd_join_##TN##_d##DH(WindowBwdArgs args) { \
    window_bwd_join<T, DH>(args);                                                                                   \
  }
#define WINDOW_BWD_TYPE(TN, T)                                                                                      \
  extern "C" __global__ __launch_bounds__(256) void window_attention_bwd_stats_##TN(WindowBwdArgs args) {           \
    window_bwd_stats<T>(args);                                                                                      \
  }                                                                                                                 \
  WINDOW_BWD(TN, T, 64)                                                                                             \
  WINDOW_BWD(TN, T, 128)

WINDOW_BWD_TYPE(bf16, bf16_t)
WINDOW_BWD_TYPE(f16, f16_t)
