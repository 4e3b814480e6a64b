// Residual add + RMS norm with an 8-bit result:
//   s = h + r,   y = s * rsqrt(mean(s^2) + eps) * w,   scale = max |y| / 448,   q = e4m3(y / scale)
// with one scale per row or per 128 columns.  Sums and y are fp32 (s enters them unrounded, as in
// add_rmsnorm); the only roundings are those of the outputs s (input type) and q.
//
// The norm's factor is positive and common to a row, so max |y| = factor * max |s w|: the maximum is
// collected in the same sweep as the sum of squares and a row costs one workgroup reduction, its elements
// stay in registers and memory is touched once.  A thread holds ITERS pieces of eight consecutive
// columns, so 128 columns are 16 neighbouring lanes and their maximum four DPP steps.
//
// Bound by memory, 7 bytes an element.  [16384, 4096] bf16 with 128-column scales, three input sets in turn: 85 us a call,
// 5.5 TB/s (a plain copy of 4 GiB reaches 4.7); one input set replayed: 77 us.  A few rows cost the launch: 3.5 us.
// Rows off the 16-byte grid move in the same pieces by unaligned accesses and only a row's last columns one by one: 57 us
// where the aligned form takes 43 ([8192, 4095] and 4096; 142 with every element on its own).  A row of up to 128 or
// 256 columns takes 16 or 32 lanes: [65536, 128] 12 us, 30 with a wavefront a row; [65536, 256] 20 and 31.
#pragma once

#include "common.h"

namespace mi {

constexpr float kE4m3Max = 448.0f;

// A maximum that carries the sum of squares along, so that one pass through LDS folds both.
struct SumMax {
  float sum, max;
};

template <int BLOCK, int GROUP>
__device__ __forceinline__ SumMax group_sum_max(SumMax v, float* lds) {
  constexpr int WIDTH = GROUP < kWave ? GROUP : kWave;
  v.sum = wave_reduce<WIDTH>(v.sum, SumOp());
  v.max = wave_reduce<WIDTH>(v.max, MaxOp());
  if constexpr (GROUP > kWave) {
    constexpr int WAVES = GROUP / kWave;
    const int wave = threadIdx.x / kWave;
    if ((threadIdx.x & (kWave - 1)) == 0) {
      lds[2 * wave] = v.sum;
      lds[2 * wave + 1] = v.max;
    }
    __syncthreads();
    const int from = (wave / WAVES) * WAVES + (threadIdx.x & (WAVES - 1));
    v.sum = wave_reduce<WAVES>(lds[2 * from], SumOp());
    v.max = wave_reduce<WAVES>(lds[2 * from + 1], MaxOp());
  }
  return v;
}

// Scale of a group whose largest |y| is `largest`: 1 for a group of zeros, and never below the smallest
// normal number, where the division by it would lose all precision or overflow.
__device__ __forceinline__ float e4m3_scale(float largest) {
  const float scale = largest / kE4m3Max;
  return largest == 0.f ? 1.f : (scale < 1.17549435e-38f ? 1.17549435e-38f : scale);
}

// GROUPED: a scale for every 128 columns (the last group may be short), otherwise one per row.
// WIDE: rows are 16-byte aligned and a multiple of eight columns long.
template <typename T, int BLOCK, int TPR, int ITERS, bool GROUPED, bool WIDE>
__device__ __forceinline__ void add_rmsnorm_quant(const T* __restrict__ h, const T* __restrict__ r,
                                                  const T* __restrict__ w, uint8_t* __restrict__ q,
                                                  float* __restrict__ scales, T* __restrict__ s_out, int rows,
                                                  int cols, long long h_stride, long long r_stride, float eps) {
  constexpr int VEC = 8;
  constexpr int ROWS = BLOCK / TPR;
  __shared__ float lds[2 * (BLOCK / kWave)];
  const int row = blockIdx.x * ROWS + threadIdx.x / TPR;
  const int lane = threadIdx.x % TPR;
  const bool live = row < rows;
  const size_t at = static_cast<size_t>(live ? row : 0);

  float y[ITERS][VEC];   // s * w
  float group_max[ITERS];
  SumMax total{0.f, 0.f};
#pragma unroll
  for (int it = 0; it < ITERS; ++it) {
    const int c = (it * TPR + lane) * VEC;
    group_max[it] = 0.f;
    Vec<T, VEC> hv, rv, wv, sv;
    const int n = live ? min(VEC, cols - c) : 0;  // columns of this piece that exist (may be negative)
    if (WIDE) {
      if (n > 0) {
        hv = load_vec<T, VEC, true>(h + at * h_stride + c);
        rv = load_vec<T, VEC, true>(r + at * r_stride + c);
        wv = load_vec<T, VEC>(w + c);
      }
    } else if (n >= VEC) {
      __builtin_memcpy(&hv, h + at * h_stride + c, sizeof(hv));
      __builtin_memcpy(&rv, r + at * r_stride + c, sizeof(rv));
      __builtin_memcpy(&wv, w + c, sizeof(wv));
    } else {
#pragma unroll
      for (int k = 0; k < VEC; ++k)
        if (k < n) {
          hv[k] = h[at * h_stride + c + k];
          rv[k] = r[at * r_stride + c + k];
          wv[k] = w[c + k];
        }
    }
#pragma unroll
    for (int k = 0; k < VEC; ++k) {
      if (WIDE ? n > 0 : k < n) {
        const float t = to_f32(hv[k]) + to_f32(rv[k]);
        sv[k] = from_f32<T>(t);
        total.sum = fmaf(t, t, total.sum);
        y[it][k] = t * to_f32(wv[k]);
        group_max[it] = MaxOp()(group_max[it], fabsf(y[it][k]));
      } else {
        y[it][k] = 0.f;
      }
    }
    if (WIDE) {
      if (n > 0) store_vec<T, VEC, true>(s_out + at * cols + c, sv);
    } else if (n >= VEC) {
      __builtin_memcpy(s_out + at * cols + c, &sv, sizeof(sv));
    } else {
#pragma unroll
      for (int k = 0; k < VEC; ++k)
        if (k < n) s_out[at * cols + c + k] = sv[k];
    }
    total.max = MaxOp()(total.max, group_max[it]);
  }
  total = group_sum_max<BLOCK, TPR>(total, lds);
  const float factor = rsqrtf(total.sum / static_cast<float>(cols) + eps);
  float scale = e4m3_scale(total.max * factor);
  if (!GROUPED && live && lane == 0) scales[at] = scale;
  const int groups = (cols + 127) / 128;
#pragma unroll
  for (int it = 0; it < ITERS; ++it) {
    const int c = (it * TPR + lane) * VEC;
    if (GROUPED) {
      scale = e4m3_scale(wave_reduce<16>(group_max[it], MaxOp()) * factor);
      if (live && c < cols && (lane & 15) == 0) scales[at * groups + c / 128] = scale;
    }
    uint32_t word[2] = {0u, 0u};
#pragma unroll
    for (int k = 0; k < VEC; k += 4) {
      word[k / 4] = __builtin_amdgcn_cvt_pk_fp8_f32(y[it][k] * factor / scale, y[it][k + 1] * factor / scale, word[k / 4], false);
      word[k / 4] = __builtin_amdgcn_cvt_pk_fp8_f32(y[it][k + 2] * factor / scale, y[it][k + 3] * factor / scale, word[k / 4], true);
    }
    if (WIDE) {
      if (live && c < cols) {
        Vec<uint32_t, 2> v;
        v[0] = word[0];
        v[1] = word[1];
        store_vec<uint32_t, 2, true>(reinterpret_cast<uint32_t*>(q + at * cols + c), v);
      }
    } else if (live && c + VEC <= cols) {
      __builtin_memcpy(q + at * cols + c, word, sizeof(word));
    } else {
      const int n = live ? cols - c : 0;
#pragma unroll
      for (int k = 0; k < VEC; ++k)
        if (k < n) q[at * cols + c + k] = static_cast<uint8_t>(word[k / 4] >> (8 * (k & 3)));
    }
  }
}

}  // namespace mi
