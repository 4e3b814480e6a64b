// Instantiations of the rotary positions (rotary.h): element type, wide or element-wise access, pair layout.
#include "../mi/rotary.h"

using namespace mi;

#define ROTARY(NAME, T, VEC, INTERLEAVED)                                                                       \
  extern "C" __global__ __launch_bounds__(kRotaryThreads) void NAME(                                            \
      const T* q, T* q_out, const T* k, T* k_out, const void* positions, const void* inv_freq, long long qb,    \
      long long qt, long long qh, long long qob, long long qot, long long qoh, long long kb, long long kt,      \
      long long kh, long long kob, long long kot, long long koh, int q_heads, int k_heads, int positions_wide,  \
      int freq_wide, int tokens, int length, int dim, int rotary, int end0, int end1, int end2, int per_block,  \
      float sign) {                                                                                             \
    const RotaryTensor tq{q, q_out, q_heads, qb, qt, qh, qob, qot, qoh};                                        \
    const RotaryTensor tk{k, k_out, k_heads, kb, kt, kh, kob, kot, koh};                                        \
    rotary_axes<T, VEC, INTERLEAVED>(tq, tk, positions, positions_wide, inv_freq, freq_wide, tokens, length,    \
                                     dim, rotary, end0, end1, end2, per_block, sign);                           \
  }
#define ROTARY_TYPE(TN, T, VEC)                              \
  ROTARY(rotary_axes_##TN##_half, T, VEC, false)             \
  ROTARY(rotary_axes_##TN##_beside, T, VEC, true)            \
  ROTARY(rotary_axes_##TN##_half_odd, T, 1, false)           \
  ROTARY(rotary_axes_##TN##_beside_odd, T, 1, true)

ROTARY_TYPE(bf16, bf16_t, 8)
ROTARY_TYPE(f16, f16_t, 8)
ROTARY_TYPE(f32, float, 4)
