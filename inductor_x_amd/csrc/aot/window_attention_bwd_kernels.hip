// Instantiations of the gradients of attention with a sliding window and visible first tokens (window_attention_bwd.h).
// dQ: as in the forward, two workgroups of four wavefronts per CU, 1219 against 1264 us for the backward pass with eight at
// [4,32/8,4096,128], window 1024.  dK and dV: one workgroup of eight wavefronts per CU, whose 99 KB of LDS (128 columns) leave
// no room for another; the bound of two wavefronts per SIMD is those eight.
#include "../mi/window_attention_bwd.h"

using namespace mi;

#define WINDOW_BWD(TN, T, DH)                                                                                            \
  extern "C" __global__ __launch_bounds__(kWinThreads, 2) void window_attention_bwd_dq_##TN##_d##DH(WindowBwdArgs args) { \
    window_bwd_dq<T, DH>(args);                                                                                          \
  }                                                                                                                      \
  extern "C" __global__ __launch_bounds__(128 * kPairs, 2) void window_attention_bwd_dkv_##TN##_d##DH(WindowBwdArgs args) { \
    window_bwd_dkv<T, DH>(args);                                                                                         \
  }                                                                                                                      \
  extern "C" __global__ __launch_bounds__(64 * kSinkWaves, 1) void window_attention_bwd_sinks_##TN##_d##DH(WindowBwdArgs args) { \
    window_bwd_sinks<T, DH>(args);                                                                                       \
  }                                                                                                                      \
  extern "C" __global__ __launch_bounds__(2 * DH) void window_attention_bwd_join_##TN##_d##DH(WindowBwdArgs args) {      \
    window_bwd_join<T, DH>(args);                                                                                        \
  }

WINDOW_BWD(bf16, bf16_t, 64)
WINDOW_BWD(bf16, bf16_t, 128)
WINDOW_BWD(f16, f16_t, 64)
WINDOW_BWD(f16, f16_t, 128)
