// Rotary positions over several axes: pair p of the first `rotary` columns of every head turns by the angle
// position[axis(p)] * inv_freq[p]; the columns behind them are copied.
//   a' = a cos - b sin,   b' = b cos + a sin       (sin negated for the inverse, which is the gradient)
// A pair is (column p, column p + rotary / 2) or, interleaved, (column 2 p, column 2 p + 1).
//
// A workgroup takes a few tokens.  Their sines and cosines are made once, in LDS, and serve all query and key
// heads of the token.  The angle is formed and reduced in 64 bits as a number of turns (a position of 10^6 in
// 32 bits would lose half the digits of the angle); from the fraction of a turn on, 32 bits hold the
// rounding of the result.
//
// Bound by memory: every element is read and written once.  128 angles a workgroup (two tokens of 64 pairs) rather
// than one a thread, for more workgroups in flight: 59 against 63 us at [4,4096,32+8,128]; results leave with the
// streaming hint, 59 against 63 us there (5.7 TB/s) and 23 against 29 us at [3,2047,24+24,96].  The element-wise form for
// heads off the 16-byte grid takes 158 us where the wide one takes 50 (126 and 128 columns, one input set replayed).
#pragma once

#include "common.h"

namespace mi {

struct RotaryTensor {
  const void* in;
  void* out;
  int heads;
  long long in_batch, in_token, in_head, out_batch, out_token, out_head;  // strides in elements
};

constexpr int kRotaryThreads = 256;
constexpr int kRotaryMaxPairs = 1024;  // (token, pair) angles a workgroup holds: 8 KiB of LDS

// VEC: elements per access (16 bytes wide, or 1 where strides, columns or addresses do not allow it).
template <typename T, int VEC, bool INTERLEAVED>
__device__ __forceinline__ void rotary_axes(const RotaryTensor& q, const RotaryTensor& k, const void* __restrict__ positions,
                                            int positions_wide, const void* __restrict__ inv_freq, int freq_wide, int tokens,
                                            int length, int dim, int rotary, int end0, int end1, int end2, int per_block,
                                            float sign) {
  __shared__ float cosine[kRotaryMaxPairs], sine[kRotaryMaxPairs];
  const int pairs = rotary / 2;
  const int t0 = blockIdx.x * per_block;
  const int here = min(per_block, tokens - t0);
  for (int i = threadIdx.x; i < here * pairs; i += kRotaryThreads) {
    const int p = i % pairs;
    const int axis = (p >= end0) + (p >= end1) + (p >= end2);
    const size_t at = static_cast<size_t>(axis) * tokens + t0 + i / pairs;
    const double where = positions_wide ? static_cast<double>(static_cast<const long long*>(positions)[at])
                                        : static_cast<double>(static_cast<const int*>(positions)[at]);
    const double f = freq_wide ? static_cast<const double*>(inv_freq)[p] : static_cast<double>(static_cast<const float*>(inv_freq)[p]);
    const double turns = where * f * 0.15915494309189533577;
    float s, c;
    sincospif(2.0f * static_cast<float>(turns - rint(turns)), &s, &c);
    cosine[i] = c;
    sine[i] = s * sign;
  }
  __syncthreads();
  // one item: VEC pairs (interleaved and wide: the VEC / 2 pairs of one access), or VEC copied columns
  constexpr int PAIRS = INTERLEAVED ? (VEC > 1 ? VEC / 2 : 1) : VEC;
  const int turned = pairs / PAIRS;
  const int per_head = turned + (dim - rotary) / VEC;
  const int heads = q.heads + k.heads;
  for (int i = threadIdx.x; i < here * heads * per_head; i += kRotaryThreads) {
    const int j = i % per_head;
    const int rest = i / per_head;
    const int head = rest % heads, tok = rest / heads;
    const int token = t0 + tok;
    const bool is_q = head < q.heads;
    const RotaryTensor& x = is_q ? q : k;
    const int hd = is_q ? head : head - q.heads;
    const int b = token / length, s = token % length;
    const T* __restrict__ in = static_cast<const T*>(x.in) + b * x.in_batch + s * x.in_token + hd * x.in_head;
    T* __restrict__ out = static_cast<T*>(x.out) + b * x.out_batch + s * x.out_token + hd * x.out_head;
    if (j >= turned) {
      const int c = rotary + (j - turned) * VEC;
      store_vec<T, VEC, true>(out + c, load_vec<T, VEC>(in + c));
      continue;
    }
    const float* cs = cosine + tok * pairs + j * PAIRS;
    const float* sn = sine + tok * pairs + j * PAIRS;
    if constexpr (INTERLEAVED && VEC > 1) {
      const Vec<T, VEC> v = load_vec<T, VEC>(in + j * VEC);
      Vec<T, VEC> o;
#pragma unroll
      for (int e = 0; e < PAIRS; ++e) {
        const float a = to_f32(v[2 * e]), d = to_f32(v[2 * e + 1]);
        o[2 * e] = from_f32<T>(a * cs[e] - d * sn[e]);
        o[2 * e + 1] = from_f32<T>(d * cs[e] + a * sn[e]);
      }
      store_vec<T, VEC, true>(out + j * VEC, o);
    } else {
      const int ca = INTERLEAVED ? 2 * j : j * VEC;
      const int cb = INTERLEAVED ? ca + 1 : ca + pairs;
      const Vec<T, VEC> va = load_vec<T, VEC>(in + ca), vb = load_vec<T, VEC>(in + cb);
      Vec<T, VEC> oa, ob;
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        const float a = to_f32(va[e]), d = to_f32(vb[e]);
        oa[e] = from_f32<T>(a * cs[e] - d * sn[e]);
        ob[e] = from_f32<T>(d * cs[e] + a * sn[e]);
      }
      store_vec<T, VEC, true>(out + ca, oa);
      store_vec<T, VEC, true>(out + cb, ob);
    }
  }
}

}  // namespace mi
