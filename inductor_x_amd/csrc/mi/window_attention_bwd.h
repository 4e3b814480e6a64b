// Gradients of window_attention.h.  With P = exp(S - lse) recomputed from the forward's row statistic, D = rowsum(dO * O)
// and dS = P * (dO V^T - D) over the visible pairs:
//     dV = P^T dO        dK = scale * dS^T Q        dQ = scale * dS K        (dK, dV summed over the heads of a group)
//
//   dQ          blocks and key tiles of the forward: wavefronts of 32 queries of heads that share a key head.  It
//               also forms the row statistics -lse / scale and -D, the values that the accumulators of Q K^T and
//               dO V^T start from in the kernels after it, so that P = exp2(S' scale log2 e) and dS = P dP' need no
//               subtraction there; a row that does not exist gets -1e30 and 0, which makes its P zero.
//               D takes O with what its rounding lost, where the forward kept that; blocks with at most two key tiles,
//               and any whose rows see at most kFewKeys, add it up from P and dP: in rows that see few keys dO V^T and
//               D nearly cancel, and the roundings of O, and of P in the forward, would be the largest errors of dS.
//               P and dS are rounded to the operand type for the products they enter (half a step each; the
//               products take 16 bits), everything else is fp32.
//   dK, dV      32 keys are a pair of wavefronts, a workgroup four pairs, 128 keys of one key head; it walks the query
//               tiles of 64 that see them through the window, head after head of the group.  One wavefront of a pair
//               makes S and P and adds to dV; it hands P to the other through LDS, in fp32, lane to lane (both hold the
//               same rows and keys), which has made dP meanwhile and adds to dK.  Neither holds more than one
//               gradient's sums and one operand, each product is made once and each tile is copied once; two
//               separate kernels (five products, two copies of each tile) took 670 us where this took 567 us on the same card
//               ([4,32/8,4096,128], window 1024; 565 to 572 us on average in later traces, 840 TFLOP/s over the four products).
//               Where there are few blocks of keys several workgroups share a walk (the host's rule); their sums go to
//               fp32 slots and the join kernel adds those in order and rounds once: [1,8/1,2048,128] causal 106 us for
//               the whole backward pass with 16 shares, 485 without.
//   first keys  the keys j < sinks are also seen by every query beyond their window, hundreds of tiles for a few keys
//               in a long text.  There that part is a kernel of its own: a workgroup takes 32 such keys and a share of
//               those queries, each wavefront streams its own tiles of 32 queries, and the sums go to fp32 slots; the
//               dK / dV kernel puts its part of these keys in slot 0 and a last kernel adds the slots in order and
//               rounds once.  Where those queries are few, or the first keys many, the dK / dV kernel walks them
//               itself (the host's rule has both sides measured).
// No atomics: results do not depend on the order of execution.
//
// fp16 has five bits of exponent: P of 2^-15 (one of 32768 keys) is below its normal numbers, and so is dS = P (dP - D) where dO
// is small, as in the mean of a loss over many tokens; and dS past 65504 is infinite.  There P enters its product times 2^14, and dS
// times a power of two which the sums are divided by at the end:
//   dK   per key, from bounds: |dP| <= max |dO| sum |V| and |D|, over the rows of the walk, reach 2^15 at most.  dQ's
//        kernel leaves the two maxima of each 32 rows behind the row statistics.
//   dQ   per row, from max |dO| alone, which becomes 2^7 to 2^8: that takes |dP - D| of up to 2^8 max |dO|, and a
//        row with more becomes infinite, which starts the workgroup over (win_any_lost) with the bound from max |V|.
// bf16 has the exponents of fp32 and no such factors.  Backward pass of [4,32/8,4096,128] window 1024 in fp16: 1093 us, 1061
// without them (bf16 1022); of [3,8/8,777,96] window 256 56 and 54.
#pragma once

#include "window_attention.h"

namespace mi {

struct WindowBwdArgs {
  const void *q, *k, *v, *o, *low, *dout;  // low may be null
  void *dq, *dk, *dv;
  const float* lse;  // [B, N, Sq]
  float* stats;      // [2][B, N, Sq]: -lse / scale, -D; for fp16 behind them [B, N, ceil(Sq / 32)][2]: largest |dO|, |D|
  float* slots;      // [B * Nk][n_slots][2][slot_rows][DH] (dK without its scale, dV) of the first `joined` keys, or null
  WindowShape shape;
  int n_slots, slot_rows;  // slot_rows: `joined` rounded up to 32
  int shares, joined;      // workgroups of a block of keys in the dK / dV kernel
  WindowStride qs, ks, vs, os, dos, dqs, dks, dvs;
};

// Matrix steps between an LDS fragment's read and its use; one to four measured alike.
constexpr int kAhead = 2;

// Visible keys up to which a row's D is added up from P and dP in any block, at the price of two more products: with n
// keys D from O adds about 1 / n to the two squared roundings that dQ and dK have otherwise (1.53 roundings of the
// outputs at 4 keys, 1.45 so).
constexpr int kFewKeys = 8;

template <typename T>
constexpr bool kWinScaled = std::is_same_v<T, f16_t>;
constexpr int kWinPShift = 14;  // P <= 1 and a little from rounding

// The power of two that brings `bound` to less than 2^top
__device__ __forceinline__ int win_shift(float bound, int top) { return top - __builtin_amdgcn_frexp_expf(bound); }

// Largest |dO| and |D| of the 32 rows of head `head` that tile t of 32 holds
__device__ __forceinline__ float* win_maxima(const WindowBwdArgs& a, int b, int head, int t) {
  const WindowShape& s = a.shape;
  const size_t rows = static_cast<size_t>(s.batch) * s.heads;
  return a.stats + 2 * (rows * s.Sq + (static_cast<size_t>(b) * s.heads + head) * ((s.Sq + 31) / 32) + t);
}

// ---- dQ, and the row statistics for the kernels after it ----
template <typename T, int DH>
__device__ __forceinline__ void window_bwd_dq(const WindowBwdArgs& a) {
  typedef AttnElem<T> E;
  typedef typename E::x8 x8_t;
  constexpr int DS = DH / 16, DB = DH / 32, TILE = kWinTile * DH;
  extern __shared__ __attribute__((aligned(16))) unsigned char attn_lds[];
  const WindowShape& s = a.shape;
  const int lane = threadIdx.x & 63, li = lane & 31, g = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int per_block = kWinRows >> s.hb_shift;
  const WindowBlock w = window_block(s, (s.Sq + per_block - 1) / per_block, s.group >> s.hb_shift);
  if (!w.any) return;
  const int length = s.length(w.b), query_end = s.query_end(w.b);
  const WindowWave me = window_wave(s, w, wave, query_end);
  T* dQ = static_cast<T*>(a.dq) + w.b * a.dqs.batch + me.head * a.dqs.head + me.q0 * a.dqs.token;
  T* stage = reinterpret_cast<T*>(attn_lds) + wave * (32 * DH);
  f32x16_t acc[DB];
  win_zero(acc);
  const int block_q0 = w.qb * per_block;
  if (block_q0 >= query_end) {
    win_store<T, DH>(dQ, a.dqs.token, acc, 0.f, stage, lane, 0, me.rows, s.dim);
    if (g == 0 && li < me.rows) {
      const size_t row = (static_cast<size_t>(w.b) * s.heads + me.head) * s.Sq + me.q0 + li;
      a.stats[row] = -1e30f;
      a.stats[static_cast<size_t>(s.batch) * s.heads * s.Sq + row] = 0.f;
    }
    if (kWinScaled<T> && lane < 2 && me.rows > 0) win_maxima(a, w.b, me.head, me.q0 / 32)[lane] = 0.f;
    return;
  }
  const WindowKeys keys = window_keys(block_q0 + s.offset(), min(block_q0 + per_block, query_end) - 1 + s.offset(), s.window, s.sinks,
                                      max(a.ks.token, a.vs.token));
  const int qi = min(me.q0 + li, s.Sq - 1);
  x8_t qf[DS], dof[DS];
  win_load_row<T>(qf, static_cast<const T*>(a.q) + w.b * a.qs.batch + me.head * a.qs.head + qi * a.qs.token, s.dim, g);
  win_load_row<T>(dof, static_cast<const T*>(a.dout) + w.b * a.dos.batch + me.head * a.dos.head + qi * a.dos.token, s.dim, g);
  const float c2 = s.scale2;
  const size_t row = (static_cast<size_t>(w.b) * s.heads + me.head) * s.Sq + me.q0;  // the first of the 32
  const bool exists = li < me.exist;
  const float m2 = (exists ? -a.lse[row + li] : -1e30f) * kWinLog2e;
  float delta = 0.f;  // -D
  const bool few = keys.n <= 2, add_up = few || s.window + s.sinks <= kFewKeys;
  if (!add_up) {
    const long long o_at = w.b * a.os.batch + me.head * a.os.head + qi * a.os.token;
    x8_t of[DS];
    auto add = [&]() {
#pragma unroll
      for (int d = 0; d < DS; ++d)
#pragma unroll
        for (int e = 0; e < 8; ++e) delta = fmaf(-static_cast<float>(of[d][e]), static_cast<float>(dof[d][e]), delta);
    };
    win_load_row<T>(of, static_cast<const T*>(a.o) + o_at, s.dim, g);
    add();
    if (a.low != nullptr) {
      win_load_row<T>(of, static_cast<const T*>(a.low) + o_at, s.dim, g);
      add();
    }
  }
  const int p = me.p_lo + li;
  float largest = 0.f;  // |dO| of the row
  if constexpr (kWinScaled<T>) {
#pragma unroll
    for (int d = 0; d < DS; ++d)
#pragma unroll
      for (int e = 0; e < 8; ++e) largest = fmaxf(largest, __builtin_fabsf(static_cast<float>(dof[d][e])));
    largest = exists ? win_half_max(largest) : 0.f;
    if (!win_is_number(largest)) largest = 0.f;  // a row that is lost
  }
  int shift = kWinScaled<T> ? win_shift(largest, 8) : 0;
  float m2s = m2;  // with the shift

  const T* K = static_cast<const T*>(a.k) + w.b * a.ks.batch + w.kvh * a.ks.head;
  const T* V = static_cast<const T*>(a.v) + w.b * a.vs.batch + w.kvh * a.vs.head;
  T* buffers = reinterpret_cast<T*>(attn_lds);
  auto request = [&](int i) {
    T* dst = buffers + (i & 1) * 2 * TILE;
    win_copy_keys<T, DH>(K, a.ks.token, keys, i, length, s.dim, dst, wave, lane);
    win_copy_keys<T, DH>(V, a.vs.token, keys, i, length, s.dim, dst + TILE, wave, lane);
  };
  auto clear = [&](int i) {
    win_clear<T, kWinThreads>(buffers + (i & 1) * 2 * TILE, 2 * TILE, threadIdx.x);
    __syncthreads();
  };
  const WinBases lane_bases = win_lane_bases<DH>(attn_lds, lane);
  // One tile.  Its matrix steps (per key block the d slices of S and dP, then the updates) read their LDS fragments
  // kAhead steps ahead, across the phases, with the order pinned by scheduling fences; `whole`: no pair is hidden.
  auto compute = [&](int i, bool whole) {
    constexpr int N1 = 2 * DS, N2 = 4 * DB;
    const WinBases at = win_bases(lane_bases, (i & 1) * 4 * TILE);
    x8_t dsf[4], ka[N1], va[N1], ta[N2];
    auto issue = [&](auto ic) {
      constexpr int n = decltype(ic)::value;
      if constexpr (n < N1) {
        ka[n] = win_row_frag<T, DH>(at, 0, n / DS, n % DS);
        va[n] = win_row_frag<T, DH>(at, 2 * TILE, n / DS, n % DS);
      } else if constexpr (n < N1 + N2) {
        ta[n - N1] = win_tr_frag<T, DH>(at, 0, (n - N1) % DB, (n - N1) / DB);
      }
    };
    static_for<kAhead>([&](auto ic) { issue(ic); });
    f32x16_t sp[2];
    static_for<N1 + N2>([&](auto ic) {
      constexpr int n = decltype(ic)::value;
      issue(std::integral_constant<int, n + kAhead>{});
      __builtin_amdgcn_sched_barrier(0);
      if constexpr (n < N1) {
        constexpr int kb = n / DS, d = n % DS;
        if constexpr (d == 0) win_zero(sp);
        sp[0] = E::mfma(ka[n], qf[d], sp[0]);
        sp[1] = E::mfma(va[n], dof[d], sp[1]);
        __builtin_amdgcn_sched_barrier(0);
        if constexpr (d == DS - 1) {
          if (!whole) me.hide(keys, i * kWinTile + 32 * kb, p, g, sp[0]);
#pragma unroll
          for (int r = 0; r < 16; ++r) {
            const float e = __builtin_amdgcn_exp2f(fmaf(sp[0][r], c2, m2s));
            dsf[2 * kb + (r >> 3)][r & 7] = static_cast<T>(e * (sp[1][r] + delta));
          }
          win_pin(dsf[2 * kb]);
          win_pin(dsf[2 * kb + 1]);
          __builtin_amdgcn_sched_barrier(0);
        }
      } else {
        constexpr int j = n - N1;
        acc[j % DB] = E::mfma(ta[j], dsf[j / DB], acc[j % DB]);
        __builtin_amdgcn_sched_barrier(0);
      }
    });
  };
  for (bool guarded = false;; guarded = true) {
    request(win_first());
    if (keys.n == 2) request(win_first() + 1);
    __builtin_amdgcn_s_waitcnt(0x0F70);  // vmcnt(0)
    __syncthreads();
    if (add_up) {
      // D = sum of P dP itself, free of the roundings that P and O took in the forward
      for (int i = 0; i < keys.n; ++i) {
        if (!few) {
          if (i > 0) {
            __builtin_amdgcn_s_waitcnt(0x0F70);  // vmcnt(0): tile i has landed, and nobody reads the buffer of the next
            __syncthreads();
          }
          if (i + 1 < keys.n) request(i + 1);
        }
        if (guarded) clear(i);
        if (!me.active(keys, i)) continue;
        const WinBases at = win_bases(lane_bases, (i & 1) * 4 * TILE);
#pragma nounroll
        for (int kb = 0; kb < 2; ++kb) {
          f32x16_t sp[2];
          win_zero(sp);
#pragma unroll
          for (int d = 0; d < DS; ++d) {
            sp[0] = E::mfma(win_row_frag<T, DH>(at, 0, kb, d), qf[d], sp[0]);
            sp[1] = E::mfma(win_row_frag<T, DH>(at, 2 * TILE, kb, d), dof[d], sp[1]);
          }
          me.hide(keys, i * kWinTile + 32 * kb, p, g, sp[0]);
#pragma unroll
          for (int r = 0; r < 16; ++r) delta = fmaf(-__builtin_amdgcn_exp2f(fmaf(sp[0][r], c2, m2)), sp[1][r], delta);
        }
      }
      if (!few) {  // from the first tile again
        __syncthreads();
        request(win_first());
        __builtin_amdgcn_s_waitcnt(0x0F70);  // vmcnt(0)
        __syncthreads();
      }
    }
    if (add_up || !guarded) delta = exists ? win_half_sum(delta) : 0.f;
    if (g == 0 && li < me.rows) {
      a.stats[row + li] = exists ? m2 / s.scale2 : -1e30f;
      a.stats[static_cast<size_t>(s.batch) * s.heads * s.Sq + row + li] = delta;
    }
    if constexpr (kWinScaled<T>) {
      const float all = wave_reduce<kWave>(largest, MaxOp()), d = wave_reduce<kWave>(win_largest(0.f, delta), MaxOp());
      if (lane < 2 && me.rows > 0) win_maxima(a, w.b, me.head, me.q0 / 32)[lane] = lane == 0 ? all : d;
      m2s = m2 + static_cast<float>(shift);
    }
    for (int i = 0; i < keys.n; ++i) {
      if (guarded) clear(i);
      if (i + 1 < keys.n && !few) request(i + 1);
      if (me.active(keys, i)) compute(i, me.whole(keys, i));
      __builtin_amdgcn_s_waitcnt(0x0F70);  // vmcnt(0): the next tile has landed
      __syncthreads();
    }
    if (guarded) {
      // a key that is no number in a column makes its score or dP none, and so the whole row of whoever sees it
      for (int i = 0; i < keys.n; ++i) {
        request(i);
        __builtin_amdgcn_s_waitcnt(0x0F70);  // vmcnt(0)
        __syncthreads();
        const T* K = buffers + (i & 1) * 2 * TILE;
        uint64_t bad = win_all_lost(acc, exists) ? 0 : __ballot(win_bad_row<T, DH>(K, lane) | win_bad_row<T, DH>(K + TILE, lane));
        bool reached = false;
        for (; bad != 0; bad &= bad - 1) reached |= me.sees(keys, i * kWinTile + __builtin_ctzll(bad), p);
        win_reach_all(acc, reached);
        if (reached && g == 0 && exists) a.stats[static_cast<size_t>(s.batch) * s.heads * s.Sq + row + li] = __builtin_nanf("");
        __syncthreads();
      }
      break;
    }
    // the words lie behind the wavefronts' pieces for the store
    if (!win_any_lost<kWinWaves>(acc, exists, reinterpret_cast<int*>(attn_lds + 4 * TILE * sizeof(T) - 64), wave, lane)) break;
    __syncthreads();
    win_zero(acc);
    if (add_up) delta = 0.f;
    if constexpr (kWinScaled<T>) {  // |dP| and |D| are at most DH max |dO| max |V|
      float most = 0.f;
      for (int i = 0; i < keys.n; ++i) {
        request(i);
        __builtin_amdgcn_s_waitcnt(0x0F70);  // vmcnt(0)
        __syncthreads();
        const T* V = buffers + (i & 1) * 2 * TILE + TILE;
#pragma nounroll
        for (int c = threadIdx.x; c < TILE; c += kWinThreads) most = win_largest(most, static_cast<float>(V[c]));
        __syncthreads();
      }
      float* words = reinterpret_cast<float*>(attn_lds);
      most = wave_reduce<kWave>(most, MaxOp());
      if (lane == 0) words[wave] = most;
      __syncthreads();
#pragma unroll
      for (int v = 0; v < kWinWaves; ++v) most = fmaxf(most, words[v]);
      __syncthreads();
      shift = win_shift(2.f * DH * largest * most, 15);
    }
  }
  win_store<T, DH>(dQ, a.dqs.token, acc, __builtin_ldexpf(s.scale, -shift), stage, lane, me.exist, me.rows, s.dim);
}

// ---- dK and dV: the pairs inside the window ----
constexpr int kPairs = 4;                      // 32 keys each: two wavefronts, one for P and dV, one for dP and dK
constexpr int kPairKeys = 32 * kPairs;
constexpr int kPairBytes = kWinTile / 2 * 64 * 4;  // P of a tile in fp32, as its lanes hold it

// All wavefronts meet; unlike __syncthreads this leaves copies into the other buffer under way.
__device__ __forceinline__ void win_meet() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");  // writes to LDS have landed
  __builtin_amdgcn_s_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
}

template <typename T, int DH>
__device__ __forceinline__ void window_bwd_dkv(const WindowBwdArgs& a) {
  typedef AttnElem<T> E;
  typedef typename E::x8 x8_t;
  constexpr int DS = DH / 16, DB = DH / 32, TILE = kWinTile * DH;
  constexpr int BUF = 2 * TILE * 2 + kWinTile * 8;  // bytes: Q, dO, statistics of the tile
  extern __shared__ __attribute__((aligned(16))) unsigned char attn_lds[];
  const WindowShape& s = a.shape;
  const int lane = threadIdx.x & 63, li = lane & 31, g = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int pair = wave % kPairs;
  const bool for_dk = wave >= kPairs;  // the two wavefronts of a pair share a SIMD
  const int blocks = (s.Sk + kPairKeys - 1) / kPairKeys;
  const WindowBlock w = window_block(s, blocks, a.shares);
  if (!w.any) return;
  const int length = s.length(w.b), query_end = s.query_end(w.b), off = s.offset();
  const int k0 = (blocks - 1 - w.qb) * kPairKeys, kw = k0 + 32 * pair;  // the first keys, seen by the most queries, first
  const int exist = min(32, length - kw), rows = min(32, s.Sk - kw);
  f32x16_t acc[DB];
  win_zero(acc);

  // query tiles that see a key of the block: through the window, or all from its first key on where the block holds
  // first keys and there is no kernel for them
  const int t_lo = max(0, k0 - off) / kWinTile;
  const int sinks = a.slots == nullptr || a.shares > 1 ? s.sinks : 0;
  const int q_last = min(query_end - 1, k0 < sinks ? query_end : min(k0 + kPairKeys, length) - 2 + s.window - off);
  const int nt = k0 < length && q_last >= 0 ? max(0, q_last / kWinTile - t_lo + 1) : 0;
  // this share of the walk
  const long long walk = static_cast<long long>(nt) * s.group;
  const int begin = static_cast<int>(walk * w.hg / a.shares), steps = static_cast<int>(walk * (w.hg + 1) / a.shares) - begin;
  const int first_h = nt > 0 ? begin / nt : 0, first_t = t_lo + begin - first_h * nt;
  const int kj = kw + li, kc = min(kj, s.Sk - 1);
  x8_t kf[DS];  // the lane's key for P, its value for dP
  win_load_row<T>(kf, for_dk ? static_cast<const T*>(a.v) + w.b * a.vs.batch + w.kvh * a.vs.head + kc * a.vs.token
                             : static_cast<const T*>(a.k) + w.b * a.ks.batch + w.kvh * a.ks.head + kc * a.ks.token, s.dim, g);
  float factor = kWinScaled<T> ? __builtin_ldexpf(1.f, kWinPShift) : 1.f;  // of P, in one kind of wavefront
  auto ds_factor = [&]() {  // of dS beside P's, in the other; every such wavefront for itself
    float largest = 0.f, d = 0.f, sum = 0.f;
    const int tiles = (s.Sq + 31) / 32;
    for (int j = lane; j < 2 * steps; j += 64) {
      const int at = begin + j / 2, t = 2 * (t_lo + at % nt) + j % 2;
      if (t < tiles) {
        const float* m = win_maxima(a, w.b, w.kvh * s.group + at / nt, t);
        largest = fmaxf(largest, m[0]);
        d = fmaxf(d, m[1]);
      }
    }
    largest = wave_reduce<kWave>(largest, MaxOp());
    d = wave_reduce<kWave>(d, MaxOp());
#pragma unroll
    for (int i = 0; i < DS; ++i)
#pragma unroll
      for (int e = 0; e < 8; ++e) sum += __builtin_fabsf(static_cast<float>(kf[i][e]));  // no number: a key that is lost
    return __builtin_ldexpf(1.f, win_shift(fmaf(largest, win_half_sum(sum), d), 15) - kWinPShift);
  };
  const float c2 = s.scale2;
  const WinBases lane_bases = win_lane_bases<DH>(attn_lds, lane);
  float* handed = reinterpret_cast<float*>(attn_lds + 2 * BUF + pair * kPairBytes) + 4 * lane;

  float sst;
  int next_h = first_h, next_t = first_t;  // head of the group and query tile of the next request
  auto request = [&](int i) {
    const int head = w.kvh * s.group + next_h;
    T* dst = reinterpret_cast<T*>(attn_lds + (i & 1) * BUF);
    const long long q0 = static_cast<long long>(next_t) * kWinTile;
    win_copy<T, DH, kWinTile, 2 * kPairs>(static_cast<const T*>(a.q) + w.b * a.qs.batch + head * a.qs.head + q0 * a.qs.token, a.qs.token,
                                          query_end - static_cast<int>(q0), s.dim, dst, wave, lane);
    win_copy<T, DH, kWinTile, 2 * kPairs>(static_cast<const T*>(a.dout) + w.b * a.dos.batch + head * a.dos.head + q0 * a.dos.token, a.dos.token,
                                          query_end - static_cast<int>(q0), s.dim, dst + TILE, wave, lane);
    if (threadIdx.x < 2 * kWinTile) {  // the first wavefront fetches -lse / scale of the 64 rows, the second -D
      const int q = static_cast<int>(q0) + lane;
      sst = wave == 0 ? -1e30f : 0.f;
      if (q < s.Sq) sst = a.stats[((static_cast<size_t>(wave) * s.batch + w.b) * s.heads + head) * s.Sq + q];
    }
    if (++next_t == t_lo + nt) {
      next_t = t_lo;
      ++next_h;
    }
  };
  // the requested tile has landed and its statistics go behind it
  auto finish = [&](int i) {
    if (threadIdx.x < 2 * kWinTile) reinterpret_cast<float*>(attn_lds + (i & 1) * BUF + 4 * TILE)[threadIdx.x] = sst;
    __builtin_amdgcn_s_waitcnt(0x0F70);  // vmcnt(0)
  };
  // the loop of one kind of wavefront; both kinds run it over the same tiles and meet at the same places
  auto run = [&](auto for_dk_c, bool guarded) {
    constexpr bool FOR_DK = decltype(for_dk_c)::value;
    f32x16_t sp[2];  // S and then P, or dP, of the two blocks of 32 queries
    x8_t bf[4];      // P or dS as operands
    int t = first_t;
    for (int i = 0; i < steps; ++i) {
      if (guarded) {
        unsigned char* buffer = attn_lds + (i & 1) * BUF;
        win_clear<T, 128 * kPairs>(reinterpret_cast<T*>(buffer), 2 * TILE, threadIdx.x);
        float* d = reinterpret_cast<float*>(buffer + 4 * TILE) + kWinTile;  // -D; without -lse there is no probability
        if (threadIdx.x < kWinTile && !win_is_number(d[threadIdx.x])) d[threadIdx.x] = 0.f;
        __syncthreads();
      }
      if (i + 1 < steps) request(i + 1);
      const int p0 = t * kWinTile + off;  // positions p0 .. p0 + 63
      const bool active = exist > 0 && p0 + kWinTile > kw && (p0 < kw + 32 - 1 + s.window || kw < sinks);
      const WinBases at = win_bases(lane_bases, (i & 1) * BUF);
      if (active) {
        // sp = start values + (Q or dO) (K or V)^T, fragments kAhead steps ahead, the order pinned by scheduling fences
        constexpr int N = 2 * DS, tile = FOR_DK ? 2 * TILE : 0;
        x8_t qa[N];
        static_for<kAhead>([&](auto ic) { qa[ic.value] = win_row_frag<T, DH>(at, tile, ic.value / DS, ic.value % DS); });
        const float* st = reinterpret_cast<const float*>(attn_lds + (i & 1) * BUF + 4 * TILE) + (FOR_DK ? kWinTile : 0) + 4 * g;
#pragma unroll
        for (int qb = 0; qb < 2; ++qb)
#pragma unroll
          for (int rq = 0; rq < 4; ++rq) {
            const Vec<float, 4> v = load_vec<float, 4>(st + 32 * qb + 8 * rq);
#pragma unroll
            for (int e = 0; e < 4; ++e) sp[qb][4 * rq + e] = v[e];
          }
        static_for<N>([&](auto ic) {
          constexpr int n = decltype(ic)::value;
          if constexpr (n + kAhead < N) qa[n + kAhead] = win_row_frag<T, DH>(at, tile, (n + kAhead) / DS, (n + kAhead) % DS);
          __builtin_amdgcn_sched_barrier(0);
          sp[n / DS] = E::mfma(qa[n], kf[n % DS], sp[n / DS]);
          __builtin_amdgcn_sched_barrier(0);
        });
        if constexpr (FOR_DK && kWinScaled<T>) {  // here, where this wavefront waits for P
#pragma unroll
          for (int qb = 0; qb < 2; ++qb) {
#pragma unroll
            for (int r = 0; r < 16; ++r) sp[qb][r] *= factor;
            asm volatile("" : "+v"(sp[qb]));
          }
        }
        if constexpr (!FOR_DK) {
          if (!(p0 >= kw + 31 && (p0 + kWinTile - 1 < kw + s.window || kw + 32 <= sinks))) {
#pragma unroll
            for (int qb = 0; qb < 2; ++qb) {
              // row r sees the key if d0 <= its offset < d1
              const int d0 = kj - (p0 + 32 * qb + 4 * g), d1 = kj < sinks ? kWinTile : d0 + s.window;
#pragma unroll
              for (int r = 0; r < 16; ++r) {
                const int o = 8 * (r >> 2) + (r & 3);
                sp[qb][r] = (o < d0) | (o >= d1) ? -__builtin_inff() : sp[qb][r];
              }
            }
          }
#pragma unroll
          for (int qb = 0; qb < 2; ++qb)
#pragma unroll
            for (int rq = 0; rq < 4; ++rq) {
              Vec<float, 4> v;
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                const float x = sp[qb][4 * rq + e];
                v[e] = __builtin_amdgcn_exp2f(kWinScaled<T> ? fmaf(x, c2, static_cast<float>(kWinPShift)) : x * c2);
                bf[2 * qb + (rq >> 1)][4 * (rq & 1) + e] = static_cast<T>(v[e]);
              }
              store_vec<float, 4>(handed + 256 * (4 * qb + rq), v);
            }
        }
      }
      win_meet();  // P is handed over
      if (active) {
        if constexpr (FOR_DK) {
#pragma unroll
          for (int qb = 0; qb < 2; ++qb)
#pragma unroll
            for (int rq = 0; rq < 4; ++rq) {
              const Vec<float, 4> v = load_vec<float, 4>(handed + 256 * (4 * qb + rq));
#pragma unroll
              for (int e = 0; e < 4; ++e) bf[2 * qb + (rq >> 1)][4 * (rq & 1) + e] = static_cast<T>(v[e] * sp[qb][4 * rq + e]);
            }
        }
        // acc += (dO or Q)^T (P or dS)
        constexpr int N = 4 * DB, tile = FOR_DK ? 0 : 2 * TILE;
        x8_t ta[N];
        static_for<kAhead>([&](auto ic) { ta[ic.value] = win_tr_frag<T, DH>(at, tile, ic.value % DB, ic.value / DB); });
        static_for<N>([&](auto ic) {
          constexpr int n = decltype(ic)::value;
          if constexpr (n + kAhead < N) ta[n + kAhead] = win_tr_frag<T, DH>(at, tile, (n + kAhead) % DB, (n + kAhead) / DB);
          __builtin_amdgcn_sched_barrier(0);
          acc[n % DB] = E::mfma(ta[n], bf[n / DB], acc[n % DB]);
          __builtin_amdgcn_sched_barrier(0);
        });
      }
      // one register set for the sums on both ways here: the compiler otherwise copies all of them in every tile
#pragma unroll
      for (int db = 0; db < DB; ++db) asm volatile("" : "+v"(acc[db]));
      if (i + 1 < steps) finish(i + 1);
      __syncthreads();
      if (++t == t_lo + nt) t = t_lo;
    }
  };
  for (bool guarded = false;; guarded = true) {
    if (steps > 0) {
      const int first = win_first();
      request(first);
      if (kWinScaled<T> && for_dk) factor = ds_factor();
      finish(first);
    }
    __syncthreads();
    if (for_dk)
      run(std::true_type(), guarded);
    else
      run(std::false_type(), guarded);
    if (guarded) {
      next_h = first_h;
      next_t = first_t;
      for (int i = 0, t = first_t; i < steps; ++i) {
        request(i);
        finish(i);
        __syncthreads();
        const T* Q = reinterpret_cast<const T*>(attn_lds + (i & 1) * BUF);
        const float* d = reinterpret_cast<const float*>(attn_lds + (i & 1) * BUF + 4 * TILE) + kWinTile;
        auto sees = [&](int row) {
          const int q = t * kWinTile + row, behind = q + off - kj;
          return q < query_end && behind >= 0 && (behind < s.window || kj < sinks);
        };
        if (!win_all_lost(acc, li < exist)) {
          const bool bad = win_bad_row<T, DH>(Q + TILE, lane);
          if (for_dk) {  // dS is no number wherever Q, dO or D is none
            uint64_t left = __ballot(bad | win_bad_row<T, DH>(Q, lane) | !win_is_number(d[lane]));
            bool reached = false;
            for (; left != 0; left &= left - 1) reached |= sees(__builtin_ctzll(left));
            win_reach_all(acc, reached);
          } else if (__any(bad)) {
            win_reach<T, DH, 4>(acc, win_bases(lane_bases, (i & 1) * BUF), 2 * TILE, g, sees);
          }
        }
#pragma unroll
        for (int db = 0; db < DB; ++db) asm volatile("" : "+v"(acc[db]));  // as in the loop above
        __syncthreads();
        if (++t == t_lo + nt) t = t_lo;
      }
      break;
    }
    // the words lie behind the wavefronts' pieces for the store
    if (!win_any_lost<2 * kPairs>(acc, li < exist, reinterpret_cast<int*>(attn_lds + 2 * BUF + kPairs * kPairBytes - 64), wave, lane)) break;
    __syncthreads();
    win_zero(acc);
    next_h = first_h;
    next_t = first_t;
    if (for_dk) win_clear_row<T>(kf);  // whoever sees such a value has no D
  }
  // the sums without their factor, a power of two
  const float unscale = !kWinScaled<T> ? 1.f : for_dk ? __builtin_ldexpf(1.f, -kWinPShift) / factor : 1.f / factor;
  const int which = for_dk ? 0 : 1;
  if (a.slots != nullptr && kw < a.slot_rows) {  // kw and slot_rows are multiples of 32
    float* slot = a.slots + ((static_cast<size_t>(w.b * s.kv_heads + w.kvh) * a.n_slots + w.hg) * 2 + which) * a.slot_rows * DH;
#pragma unroll
    for (int db = 0; db < DB; ++db)
#pragma unroll
      for (int rq = 0; rq < 4; ++rq) {
        Vec<float, 4> v;
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = li < exist ? acc[db][4 * rq + e] * unscale : 0.f;
        store_vec<float, 4>(slot + static_cast<size_t>(kj) * DH + 32 * db + 8 * rq + 4 * g, v);
      }
  }
  if (a.shares > 1) return;  // every key is joined
  const WindowStride& ds = for_dk ? a.dks : a.dvs;
  T* out = static_cast<T*>(for_dk ? a.dk : a.dv) + w.b * ds.batch + w.kvh * ds.head + kw * ds.token;
  win_store<T, DH>(out, ds.token, acc, for_dk ? s.scale * unscale : unscale, reinterpret_cast<T*>(attn_lds) + wave * (32 * DH), lane, exist, rows, s.dim);
}

// ---- dK and dV of the first keys from the queries beyond their window ----
constexpr int kSinkWaves = 4;
constexpr int kSinkTile = 32;  // queries of a tile

template <typename T, int DH>
__device__ __forceinline__ void window_bwd_sinks(const WindowBwdArgs& a) {
  typedef AttnElem<T> E;
  typedef typename E::x8 x8_t;
  constexpr int DS = DH / 16, DB = DH / 32, TILE = kSinkTile * DH;
  extern __shared__ __attribute__((aligned(16))) unsigned char attn_lds[];
  const WindowShape& s = a.shape;
  const int lane = threadIdx.x & 63, li = lane & 31, g = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  // workgroups: [sequence and key head][32 keys][split]
  const int splits = a.n_slots - 1, key_blocks = a.slot_rows / 32;
  const int split = blockIdx.x % splits, rest = blockIdx.x / splits;
  const int k0 = rest % key_blocks * 32, unit = rest / key_blocks;
  const int b = unit / s.kv_heads, kvh = unit % s.kv_heads;
  const int length = s.length(b), query_end = s.query_end(b), off = s.offset();
  const int keys = min(min(s.sinks, length) - k0, 32);  // of these 32, the ones that exist and stay visible
  const int t_lo = max(0, k0 + s.window - off) / kSinkTile;
  const int nt = keys > 0 && query_end > 0 ? max(0, (query_end - 1) / kSinkTile - t_lo + 1) : 0;
  const long long total = static_cast<long long>(nt) * s.group;
  const int begin = static_cast<int>(total * split / splits), end = static_cast<int>(total * (split + 1) / splits);

  const int kj = k0 + li, kc = min(kj, s.Sk - 1);
  x8_t kf[DS], vf[DS];
  win_load_row<T>(kf, static_cast<const T*>(a.k) + b * a.ks.batch + kvh * a.ks.head + kc * a.ks.token, s.dim, g);
  win_load_row<T>(vf, static_cast<const T*>(a.v) + b * a.vs.batch + kvh * a.vs.head + kc * a.vs.token, s.dim, g);
  const float c2 = s.scale2;
  const WinBases lane_bases = win_lane_bases<DH>(attn_lds, lane);
  float factor = 1.f;  // of dS beside P's
  if constexpr (kWinScaled<T>) {
    float largest = 0.f, d = 0.f, sum = 0.f;
    for (int j = begin + lane; j < end; j += 64) {
      const float* m = win_maxima(a, b, kvh * s.group + j / nt, t_lo + j % nt);
      largest = fmaxf(largest, m[0]);
      d = fmaxf(d, m[1]);
    }
    largest = wave_reduce<kWave>(largest, MaxOp());
    d = wave_reduce<kWave>(d, MaxOp());
#pragma unroll
    for (int i = 0; i < DS; ++i)
#pragma unroll
      for (int e = 0; e < 8; ++e) sum += __builtin_fabsf(static_cast<float>(vf[i][e]));
    factor = __builtin_ldexpf(1.f, win_shift(fmaf(largest, win_half_sum(sum), d), 15) - kWinPShift);
  }
  f32x16_t dk[DB], dv[DB];
  win_zero(dk);
  win_zero(dv);
  T* mine = reinterpret_cast<T*>(attn_lds) + wave * 4 * TILE;  // two buffers of Q and dO
  auto request = [&](int i, int buf) {
    const int head = kvh * s.group + i / nt;
    const long long q0 = static_cast<long long>(t_lo + i % nt) * kSinkTile;
    win_copy<T, DH, kSinkTile, 1>(static_cast<const T*>(a.q) + b * a.qs.batch + head * a.qs.head + q0 * a.qs.token, a.qs.token,
                                  query_end - static_cast<int>(q0), s.dim, mine + buf * 2 * TILE, 0, lane);
    win_copy<T, DH, kSinkTile, 1>(static_cast<const T*>(a.dout) + b * a.dos.batch + head * a.dos.head + q0 * a.dos.token, a.dos.token,
                                  query_end - static_cast<int>(q0), s.dim, mine + buf * 2 * TILE + TILE, 0, lane);
  };
  for (bool guarded = false;; guarded = true) {
    int i = begin + wave;
    if (i < end) request(i, 0);
    for (int buf = 0; i < end; i += kSinkWaves, buf ^= 1) {
      const int head = kvh * s.group + i / nt;
      const int q0 = (t_lo + i % nt) * kSinkTile;
      // statistics of the lane's sixteen rows, requested before the next tile's copies
      f32x16_t sp[2];
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const int q = min(q0 + 8 * (r >> 2) + 4 * g + (r & 3), s.Sq - 1);
#pragma unroll
        for (int k = 0; k < 2; ++k) sp[k][r] = a.stats[((static_cast<size_t>(k) * s.batch + b) * s.heads + head) * s.Sq + q];
      }
      __builtin_amdgcn_s_waitcnt(0x0F70);  // vmcnt(0): this tile has landed
      __builtin_amdgcn_sched_barrier(0);
      if (i + kSinkWaves < end) request(i + kSinkWaves, buf ^ 1);
      if (guarded) {
        win_clear<T, 64>(mine + buf * 2 * TILE, 2 * TILE, lane);
#pragma unroll
        for (int r = 0; r < 16; ++r) sp[1][r] = win_is_number(sp[1][r]) ? sp[1][r] : 0.f;
      }
      const WinBases at = win_bases(lane_bases, (wave * 4 + buf * 2) * TILE * 2);
#pragma unroll
      for (int d = 0; d < DS; ++d) {
        sp[0] = E::mfma(win_row_frag<T, DH>(at, 0, 0, d), kf[d], sp[0]);
        sp[1] = E::mfma(win_row_frag<T, DH>(at, 2 * TILE, 0, d), vf[d], sp[1]);
      }
      x8_t pf[2], dsf[2];
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const int q = q0 + 8 * (r >> 2) + 4 * g + (r & 3);
        float x = __builtin_amdgcn_exp2f(kWinScaled<T> ? fmaf(sp[0][r], c2, static_cast<float>(kWinPShift)) : sp[0][r] * c2);
        x = (q < query_end) & (q + off - kj >= s.window) & (li < keys) ? x : 0.f;
        pf[r >> 3][r & 7] = static_cast<T>(x);
        dsf[r >> 3][r & 7] = static_cast<T>(kWinScaled<T> ? x * sp[1][r] * factor : x * sp[1][r]);
      }
#pragma unroll
      for (int q2 = 0; q2 < 2; ++q2)
#pragma unroll
        for (int db = 0; db < DB; ++db) {
          dv[db] = E::mfma(win_tr_frag<T, DH>(at, 2 * TILE, db, q2), pf[q2], dv[db]);
          dk[db] = E::mfma(win_tr_frag<T, DH>(at, 0, db, q2), dsf[q2], dk[db]);
        }
      __builtin_amdgcn_s_waitcnt(0xC07F);  // lgkmcnt(0): the reads of this buffer are done before it is refilled
      __builtin_amdgcn_sched_barrier(0);
    }
    if (guarded) {
      for (i = begin + wave; i < end; i += kSinkWaves) {
        request(i, 0);
        const int head = kvh * s.group + i / nt, q0 = (t_lo + i % nt) * kSinkTile;
        const float d = a.stats[((static_cast<size_t>(s.batch) + b) * s.heads + head) * s.Sq + min(q0 + li, s.Sq - 1)];
        __builtin_amdgcn_s_waitcnt(0x0F70);  // vmcnt(0)
        __builtin_amdgcn_sched_barrier(0);
        const bool bad_do = win_bad_row<T, DH>(mine + TILE, li), bad = win_bad_row<T, DH>(mine, li) | bad_do | !win_is_number(d);
        auto sees = [&](int row) { return q0 + row < query_end && q0 + row + off - kj >= s.window && li < keys; };
        bool reached = false;
        for (uint32_t left = static_cast<uint32_t>(__ballot(bad)); left != 0; left &= left - 1) reached |= sees(__builtin_ctz(left));
        win_reach_all(dk, reached);
        if (__any(bad_do) && !win_all_lost(dv, li < keys)) win_reach<T, DH, 2>(dv, win_bases(lane_bases, wave * 4 * TILE * 2), 2 * TILE, g, sees);
        __builtin_amdgcn_s_waitcnt(0xC07F);  // lgkmcnt(0): the reads are done before the next request
        __builtin_amdgcn_sched_barrier(0);
      }
      break;
    }
    if (!(win_lost(dk, li < keys) | win_lost(dv, li < keys))) break;
    win_zero(dk);
    win_zero(dv);
    win_clear_row<T>(vf);  // whoever sees such a value has no D
  }
  const float unscale_v = kWinScaled<T> ? __builtin_ldexpf(1.f, -kWinPShift) : 1.f, unscale_k = kWinScaled<T> ? unscale_v / factor : 1.f;
  // the four wavefronts' sums meet in LDS, [wave][dK, dV][key][DH]
  __syncthreads();
  float* all = reinterpret_cast<float*>(attn_lds);
#pragma unroll
  for (int db = 0; db < DB; ++db)
#pragma unroll
    for (int rq = 0; rq < 4; ++rq) {
      Vec<float, 4> x, y;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        x[e] = li < keys ? dk[db][4 * rq + e] * unscale_k : 0.f;
        y[e] = li < keys ? dv[db][4 * rq + e] * unscale_v : 0.f;
      }
      const int at = li * DH + 32 * db + 8 * rq + 4 * g;
      store_vec<float, 4>(all + wave * 64 * DH + at, x);
      store_vec<float, 4>(all + wave * 64 * DH + 32 * DH + at, y);
    }
  __syncthreads();
  float* slot = a.slots + (static_cast<size_t>(unit) * a.n_slots + 1 + split) * 2 * a.slot_rows * DH;
  for (int j = threadIdx.x; j < 64 * DH; j += 64 * kSinkWaves) {
    float sum = 0.f;
#pragma unroll
    for (int v = 0; v < kSinkWaves; ++v) sum += all[v * 64 * DH + j];
    const int which = j / (32 * DH), in = j % (32 * DH);
    slot[static_cast<size_t>(which) * a.slot_rows * DH + static_cast<size_t>(k0) * DH + in] = sum;
  }
}

// Adds the slots of one joined key row (blockIdx: sequence and key head, key) in order: a thread per column, dK then dV.
template <typename T, int DH>
__device__ __forceinline__ void window_bwd_join(const WindowBwdArgs& a) {
  const WindowShape& s = a.shape;
  const int unit = blockIdx.x / a.joined, j = blockIdx.x % a.joined;
  const int b = unit / s.kv_heads, kvh = unit % s.kv_heads;
  const int which = threadIdx.x / DH, d = threadIdx.x % DH;
  float sum = 0.f;
  for (int n = 0; n < a.n_slots; ++n)
    sum += a.slots[(((static_cast<size_t>(unit) * a.n_slots + n) * 2 + which) * a.slot_rows + j) * DH + d];
  if (d < s.dim) {
    if (which == 0)
      static_cast<T*>(a.dk)[b * a.dks.batch + kvh * a.dks.head + j * a.dks.token + d] = static_cast<T>(sum * s.scale);
    else
      static_cast<T*>(a.dv)[b * a.dvs.batch + kvh * a.dvs.head + j * a.dvs.token + d] = static_cast<T>(sum);
  }
}

}  // namespace mi
