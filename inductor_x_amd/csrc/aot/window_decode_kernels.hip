// Instantiations of single-token attention over a cache (window_decode.h): element type, columns of a tile.
#include "../mi/window_decode.h"

using namespace mi;

#define WINDOW_DECODE(TN, T, DH)                                                                               \
  extern "C" __global__ __launch_bounds__(256) void window_decode_##TN##_d##DH(                                \
      const T* q, const T* k, const T* v, T* out, float* part, const int* lengths, long long qb, long long qh, \
      long long kb, long long kh, long long kt, long long vb, long long vh, long long vt, long long ob,        \
      long long oh, int kv_heads, int group, int splits, int capacity, int dim, int window, int sinks, float scale_log2e) { \
    const DecodeArgs a{q,  k,  v,  out, part, lengths, qb, qh, kb, kh, kt, vb, vh, vt, ob, oh,                 \
                       kv_heads, group, splits, capacity, dim, window, sinks, scale_log2e};                            \
    window_decode<T, DH>(a);                                                                                   \
  }                                                                                                            \
  extern "C" __global__ __launch_bounds__(DH) void window_decode_join_##TN##_d##DH(                            \
      const float* part, T* out, const int* lengths, int heads, int splits, int dim, long long ob, long long oh) { \
    window_decode_join<T, DH>(part, out, lengths, heads, splits, dim, ob, oh);                                 \
  }

WINDOW_DECODE(bf16, bf16_t, 64)
WINDOW_DECODE(bf16, bf16_t, 128)
WINDOW_DECODE(f16, f16_t, 64)
WINDOW_DECODE(f16, f16_t, 128)
