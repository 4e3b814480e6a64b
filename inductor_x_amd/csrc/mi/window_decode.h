// Attention of one new token per sequence against a cache, with a sliding window and first tokens that stay
// visible: of a sequence that holds `length` keys, the keys j < sinks and j >= length - window are seen.
//
// Bound by reading those rows of the cache once, so everything is built around loads in flight: a workgroup
// serves one key head of one sequence and up to 16 query heads that share it (they are the 16 columns of the
// matrix products, so a key row is read once for all of them), and takes a contiguous share of the visible
// keys; few sequences are spread over the chip by splitting the keys, and window_decode_join puts the
// shares together.  Each of the four wavefronts streams its own tiles of 32 keys through a private double
// buffer in LDS by direct 16-byte loads, with no barrier until the end.
//
//   S^T [key, head] = K [key, d] Q^T           v_mfma 16x16x32, A = K from LDS, B = Q in registers
//   O^T [d, head]  += V^T [d, key] P^T         A = V read transposed from LDS, B = P as the first product left it
//
// Accumulator element r of lane (column n = lane % 16, group g = lane / 16) is key 4 g + r of its block of
// 16.  The B operand of the second product wants eight keys a lane: the two blocks' four each, and the
// transposing reads of V deliver their keys in the same order.
// Rows past the visible end are never read (the buffer descriptor ends there), so what lies in the unused
// part of the cache, NaN included, has no effect.
//
// Measured: 64 sequences of up to 16384 keys, window 4096, 8 key heads of 128: 168 us, 5.7 TB/s of the 0.95 GB of visible
// rows; one sequence, window 1024: 5.8 us and 2.8 us for the join, both mostly latency.
#pragma once

#include "attention.h"

namespace mi {

typedef float f32x4_t __attribute__((ext_vector_type(4)));

constexpr int kDecodeWaves = 4;
constexpr int kDecodeKeys = 32;   // keys of a tile
constexpr int kDecodeHeads = 16;  // query heads of a workgroup

template <typename T>
struct DecodeElem;
template <>
struct DecodeElem<bf16_t> {
  static __device__ __forceinline__ f32x4_t mfma(AttnElem<bf16_t>::x8 a, AttnElem<bf16_t>::x8 b, f32x4_t c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
  }
};
template <>
struct DecodeElem<f16_t> {
  static __device__ __forceinline__ f32x4_t mfma(AttnElem<f16_t>::x8 a, AttnElem<f16_t>::x8 b, f32x4_t c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
  }
};

struct DecodeArgs {
  const void *q, *k, *v;
  void* out;           // [B, N, D], written when there is one split
  float* part;         // [B * N][splits][DH + 2]: O, maximum, sum; written when there are several
  const int* lengths;  // keys of each sequence, the new token's among them
  long long q_batch, q_head, k_batch, k_head, k_token, v_batch, v_head, v_token, out_batch, out_head;
  int kv_heads, group, splits, capacity, dim, window, sinks;
  float scale_log2e;
};

// DH: columns the tiles carry, 64 or 128; dim of them hold data (a multiple of 8), the others read as zeros.
template <typename T, int DH>
__device__ __forceinline__ void window_decode(const DecodeArgs& a) {
  typedef AttnElem<T> E;
  typedef typename E::x8 x8_t;
  constexpr int CHUNKS = DH / 8;         // 16-byte chunks of a row
  constexpr int TILE = kDecodeKeys * DH;  // elements of a K or V tile
  constexpr int STEPS = DH / 32, DB = DH / 16;
  extern __shared__ __attribute__((aligned(16))) unsigned char decode_lds[];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int n = lane & 15, g = lane >> 4;
  // workgroups of one key head are neighbours: [sequence][key head][16 query heads][split]
  const int splits = a.splits, parts = (a.group + kDecodeHeads - 1) / kDecodeHeads;
  const int split = blockIdx.x % splits, unit = blockIdx.x / splits;
  const int h0 = unit % parts * kDecodeHeads;  // first query head of this workgroup within the group
  const int b = unit / parts / a.kv_heads, kvh = unit / parts % a.kv_heads;
  const int heads = min(kDecodeHeads, a.group - h0);

  const int length = min(max(a.lengths[b], 0), a.capacity);
  const int first = max(0, length - a.window);  // first key of the window
  const int sinks = min(a.sinks, first);        // keys before it that stay visible
  const int sink_tiles = (sinks + kDecodeKeys - 1) / kDecodeKeys;
  const int tiles = sink_tiles + (length - first + kDecodeKeys - 1) / kDecodeKeys;
  const int t_begin = static_cast<int>(static_cast<long long>(tiles) * split / splits);
  const int t_end = static_cast<int>(static_cast<long long>(tiles) * (split + 1) / splits);

  const T* __restrict__ K = static_cast<const T*>(a.k) + b * a.k_batch + kvh * a.k_head;
  const T* __restrict__ V = static_cast<const T*>(a.v) + b * a.v_batch + kvh * a.v_head;
  T* Kt = reinterpret_cast<T*>(decode_lds) + wave * 4 * TILE;  // two buffers of K and V
  auto first_key = [&](int t) { return t < sink_tiles ? t * kDecodeKeys : first + (t - sink_tiles) * kDecodeKeys; };
  auto keys_of = [&](int t) { return min(kDecodeKeys, t < sink_tiles ? sinks - t * kDecodeKeys : length - first_key(t)); };
  auto copy = [&](const T* src, long long stride, int rows, T* dst) {
    // one instruction fills 64 chunks of LDS; the chunk a lane fetches is XOR-swizzled by its row
    const int bytes = static_cast<int>((rows - 1) * stride * 2 + a.dim * 2);
#pragma unroll
    for (int u = 0; u < TILE / 512; ++u) {
      const int row = (u * 64 + lane) / CHUNKS;
      const int chunk = (lane % CHUNKS) ^ (row % CHUNKS);
      const int voff = 8 * chunk < a.dim ? static_cast<int>(row * stride * 2) + 16 * chunk : 0x7ffffff0;
      __builtin_amdgcn_raw_ptr_buffer_load_lds(
          __builtin_amdgcn_make_buffer_rsrc(const_cast<T*>(src), 0, bytes, 0x00020000),
          (__attribute__((address_space(3))) void*)(dst + u * 512), 16, voff, 0, 0, 0);
    }
  };
  auto request = [&](int t, int buf) {
    const long long key = first_key(t);
    const int rows = keys_of(t);
    copy(K + key * a.k_token, a.k_token, rows, Kt + buf * 2 * TILE);
    copy(V + key * a.v_token, a.v_token, rows, Kt + buf * 2 * TILE + TILE);
  };

  x8_t qf[STEPS];
  {
    const T* q = static_cast<const T*>(a.q) + b * a.q_batch + (kvh * a.group + h0 + min(n, heads - 1)) * a.q_head;
#pragma unroll
    for (int s = 0; s < STEPS; ++s) {
      const int c = 32 * s + 8 * g;
      if (c < a.dim) {
        qf[s] = *reinterpret_cast<const x8_t*>(q + c);
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) qf[s][e] = static_cast<T>(0.f);
      }
    }
  }
  f32x4_t o[DB];
#pragma unroll
  for (int db = 0; db < DB; ++db) o[db] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  float m = -1e30f, l = 0.f;  // a finite start keeps lanes whose keys do not exist free of inf - inf

  int t = t_begin + wave;
  if (t < t_end) request(t, 0);
  for (int buf = 0; t < t_end; t += kDecodeWaves, buf ^= 1) {
    const bool more = t + kDecodeWaves < t_end;
    if (more) request(t + kDecodeWaves, buf ^ 1);
    // the tile's own 2 * TILE / 512 loads have landed; those just issued may be under way
    if (more) {
      static_assert(2 * (TILE / 512) == 16 || 2 * (TILE / 512) == 8, "loads of a tile");
      if constexpr (2 * (TILE / 512) == 16)
        __builtin_amdgcn_s_waitcnt(0x4F70);  // vmcnt(16)
      else
        __builtin_amdgcn_s_waitcnt(0x0F78);  // vmcnt(8)
    } else {
      __builtin_amdgcn_s_waitcnt(0x0F70);  // vmcnt(0)
    }
    __builtin_amdgcn_sched_barrier(0);
    const T* Ks = Kt + buf * 2 * TILE;
    const T* Vs = Ks + TILE;
    f32x4_t s[2];
#pragma unroll
    for (int kb = 0; kb < 2; ++kb) {
      s[kb] = f32x4_t{0.f, 0.f, 0.f, 0.f};
      const int row = 16 * kb + n;
#pragma unroll
      for (int st = 0; st < STEPS; ++st) {
        const x8_t kf = *reinterpret_cast<const x8_t*>(Ks + row * DH + 8 * ((4 * st + g) ^ (row % CHUNKS)));
        s[kb] = DecodeElem<T>::mfma(kf, qf[st], s[kb]);
      }
    }
    const int rows = keys_of(t);
    float mx = -1e30f;
#pragma unroll
    for (int kb = 0; kb < 2; ++kb)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        s[kb][r] = 16 * kb + 4 * g + r < rows ? s[kb][r] * a.scale_log2e : -__builtin_inff();
        mx = fmaxf(mx, s[kb][r]);
      }
    mx = fmaxf(mx, __shfl_xor(mx, 16, kWave));
    mx = fmaxf(mx, __shfl_xor(mx, 32, kWave));
    const float m_new = fmaxf(m, mx);
    const float alpha = __builtin_amdgcn_exp2f(m - m_new);
    m = m_new;
    x8_t p;
    float sum = 0.f;
#pragma unroll
    for (int kb = 0; kb < 2; ++kb)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const float e = __builtin_amdgcn_exp2f(s[kb][r] - m);
        sum += e;
        p[4 * kb + r] = static_cast<T>(e);  // the product with V takes 16 bits; the sum keeps 32
      }
    l = fmaf(l, alpha, sum);
    if (__any(alpha != 1.f)) {
#pragma unroll
      for (int db = 0; db < DB; ++db) o[db] *= alpha;
    }
    const int vr = 4 * g + (n >> 2);
#pragma unroll
    for (int db = 0; db < DB; ++db) {
      const int c = 2 * db + ((n & 3) >> 1);
      const typename E::x4 lo = E::read_tr(Vs + vr * DH + 8 * (c ^ (vr % CHUNKS)) + 4 * (n & 1));
      const typename E::x4 hi = E::read_tr(Vs + (vr + 16) * DH + 8 * (c ^ ((vr + 16) % CHUNKS)) + 4 * (n & 1));
      x8_t vf;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        vf[e] = lo[e];
        vf[4 + e] = hi[e];
      }
      o[db] = DecodeElem<T>::mfma(vf, p, o[db]);
    }
    // the reads of this buffer are done before the next request refills it
    __builtin_amdgcn_s_waitcnt(0xC07F);  // lgkmcnt(0)
    __builtin_amdgcn_sched_barrier(0);
  }
  l += __shfl_xor(l, 16, kWave);
  l += __shfl_xor(l, 32, kWave);

  // ---- the four wavefronts' shares meet in LDS: [wave][head][DH + 4], O and behind it maximum and sum ----
  __syncthreads();
  constexpr int PITCH = DH + 4;
  float* mine = reinterpret_cast<float*>(decode_lds) + (wave * kDecodeHeads + n) * PITCH;
#pragma unroll
  for (int db = 0; db < DB; ++db) *reinterpret_cast<f32x4_t*>(mine + 16 * db + 4 * g) = o[db];
  if (g == 0) {
    mine[DH] = m;
    mine[DH + 1] = l;
  }
  __syncthreads();
  const float* all = reinterpret_cast<const float*>(decode_lds);
  for (int i = threadIdx.x; i < heads * DH; i += 64 * kDecodeWaves) {
    const int h = i / DH, d = i % DH;
    float top = -1e30f;
#pragma unroll
    for (int w = 0; w < kDecodeWaves; ++w) top = fmaxf(top, all[(w * kDecodeHeads + h) * PITCH + DH]);
    float sum = 0.f, acc = 0.f;
#pragma unroll
    for (int w = 0; w < kDecodeWaves; ++w) {
      const float* x = all + (w * kDecodeHeads + h) * PITCH;
      const float f = __builtin_amdgcn_exp2f(x[DH] - top);
      sum = fmaf(x[DH + 1], f, sum);
      acc = fmaf(x[d], f, acc);
    }
    const int head = kvh * a.group + h0 + h;
    if (splits == 1) {
      if (d < a.dim)
        static_cast<T*>(a.out)[b * a.out_batch + head * a.out_head + d] = static_cast<T>(length > 0 ? acc / sum : 0.f);
    } else {
      float* part = a.part + ((static_cast<size_t>(b) * a.kv_heads * a.group + head) * splits + split) * (DH + 2);
      part[d] = acc;
      if (d == 0) {
        part[DH] = top;
        part[DH + 1] = sum;
      }
    }
  }
}

constexpr int kDecodeSplits = 64;  // most shares the keys of a sequence are cut into

// Joins the splits of one (sequence, head): a thread per split finds its weight, then a thread per column adds up.
template <typename T, int DH>
__device__ __forceinline__ void window_decode_join(const float* __restrict__ part, T* __restrict__ out,
                                                   const int* __restrict__ lengths, int heads, int splits, int dim,
                                                   long long out_batch, long long out_head) {
  static_assert(DH >= kDecodeSplits, "a thread per split");
  __shared__ float weight[kDecodeSplits], share[kDecodeSplits];
  const int b = blockIdx.x / heads, h = blockIdx.x % heads, d = threadIdx.x;
  const float* p = part + static_cast<size_t>(blockIdx.x) * splits * (DH + 2);
  const int length = lengths[b];
  if (d < kDecodeSplits) {  // the first wavefront
    const bool mine = d < splits;
    const float m = mine ? p[d * (DH + 2) + DH] : -1e30f;
    const float l = mine ? p[d * (DH + 2) + DH + 1] : 0.f;
    const float f = __builtin_amdgcn_exp2f(m - wave_reduce<kWave>(m, MaxOp()));
    weight[d] = mine ? f : 0.f;
    share[d] = wave_reduce<kWave>(l * f, SumOp());
  }
  __syncthreads();
  float acc = 0.f;
#pragma unroll 8
  for (int s = 0; s < splits; ++s) acc = fmaf(p[s * (DH + 2) + d], weight[s], acc);
  if (d < dim) out[b * out_batch + h * out_head + d] = static_cast<T>(length > 0 ? acc / share[0] : 0.f);
}

}  // namespace mi
