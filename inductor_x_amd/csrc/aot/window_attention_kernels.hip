// Instantiations of the forward of attention with a sliding window and visible first tokens (window_attention.h).
// 512 threads, one workgroup per CU.
#include "../mi/window_attention.h"

using namespace mi;

#define WINDOW_FWD(TN, T, DH)                                                                                      \
  extern "C" __global__ __launch_bounds__(512, 1) void window_attention_fwd_##TN##_d##DH(WindowFwdArgs args) {     \
    window_attention_fwd<T, DH>(args);                                                                             \
  }

WINDOW_FWD(bf16, bf16_t, 64)
WINDOW_FWD(bf16, bf16_t, 128)
WINDOW_FWD(f16, f16_t, 64)
WINDOW_FWD(f16, f16_t, 128)
