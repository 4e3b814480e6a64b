// Instantiations of the forward of attention with a sliding window and visible first tokens (window_attention.h).
// Four wavefronts, two workgroups per CU: the two wavefronts of a SIMD then belong to different workgroups, whose first
// loads and last stores hide behind each other's products.  Eight wavefronts that share their tiles measured 374
// against 318 us at [4,32/8,4096,128] with a window of 1024, 640 against 566 us at [1,32/8,8192,128] without one.
#include "../mi/window_attention.h"

using namespace mi;

#define WINDOW_FWD(TN, T, DH)                                                                                        \
  extern "C" __global__ __launch_bounds__(kWinThreads, 2) void window_attention_fwd_##TN##_d##DH(WindowFwdArgs args) { \
    window_attention_fwd<T, DH>(args);                                                                               \
  }

WINDOW_FWD(bf16, bf16_t, 64)
WINDOW_FWD(bf16, bf16_t, 128)
WINDOW_FWD(f16, f16_t, 64)
WINDOW_FWD(f16, f16_t, 128)
