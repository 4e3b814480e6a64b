// Attention with a sliding window and first tokens that stay visible (sinks), for heads that share keys.
//
//   position of query i:  p = i + (Sk - Sq)          (the queries are the last Sq of Sk positions)
//   key j is visible:     j <= p  and  (p - j < window  or  j < sinks)
//   O = softmax(Q K^T * scale over the visible keys) V,   lse = log sum exp of the scaled scores
//
// Positions from lengths[b] on do not exist (right padding): their keys are hidden and not read, their rows are
// zero, lse -inf.
//
// Work of a workgroup: four wavefronts of 32 queries on one key head.  They are HB = 1, 2 or 4 query heads
// that share the key head times 128 / HB consecutive queries, so that heads in a group read a key tile once
// between them, and a block visits the keys of a window plus 128 / HB - 1 others, in tiles of 64 (window_keys).
// No mask exists in memory: a wavefront compares positions in the few tiles that are neither wholly visible nor
// wholly hidden to it.
//
// Measured on MI355X (bf16, 32 query heads on 8 key heads, 128 columns; several cards): 4096 queries at the end of 32768
// keys, window 8192, 128 first keys: 532 to 552 us, 1012 to 1050 TFLOP/s over the visible pairs, 87 to 90 % of what a large
// library product reaches (1165); 8192 queries, window 1024: 162 to 166 us, 780 to 800 TFLOP/s.  The matrix pipe is busy 52 %
// and 42 % of the cycles: beside it run 6 (8) vector instructions per product, and every product reads one operand from
// LDS.  A block of 18 tiles takes about 37 us at the long rows' pace and 42 as it is: its first loads and last stores, which the
// second workgroup of the CU covers in part.  Blocks are not split over their keys: few blocks of long rows leave CUs idle, and
// their time is one block's chain, 50 us for [1,8/1,2048,128] causal (floor 7).  A two-phase software
// pipeline like attention_v5.h's was 4 % faster in rows of thousands of keys and 25 % slower in windows of 256.
//
// Operand layouts and the transposed products are those of attention.h.  Tiles travel memory -> LDS by direct
// 16-byte loads, [64][DH] as they lie in memory with the chunks of a row swizzled; rows past the end and
// columns past the head dimension arrive as zeros (bounds of the buffer descriptor).
#pragma once

#include "attention.h"

namespace mi {

constexpr int kWinWaves = 4;
constexpr int kWinThreads = 64 * kWinWaves;
constexpr int kWinRows = 32 * kWinWaves;  // (head, query) rows or keys of a workgroup
constexpr int kWinTile = 64;              // keys (queries) of a tile
constexpr float kWinLog2e = 1.4426950408889634f;
constexpr float kWinLn2 = 0.69314718055994530942f;
constexpr float kWinFloor = -1e30f;       // below every score: keeps rows without a visible key so far free of inf - inf

// Strides in elements of a [batch, head, token, column] tensor with contiguous columns.
struct WindowStride {
  long long batch, head, token;
};

// Problem description that every kernel takes behind its operands' pointers.
struct WindowShape {
  const int* lengths;  // may be null: every position exists
  int batch, heads, kv_heads, group, Sq, Sk, dim, window, sinks, hb_shift;
  float scale, scale2;  // scale2 = scale log2 e

  __device__ __forceinline__ int offset() const { return Sk - Sq; }
  __device__ __forceinline__ int length(int b) const { return lengths ? min(max(lengths[b], 0), Sk) : Sk; }
  // queries that exist (may be <= 0)
  __device__ __forceinline__ int query_end(int b) const { return min(Sq, length(b) - offset()); }
};

static_assert(sizeof(WindowShape) == 56, "the host packs it without padding");

// The keys a block visits, as one run of slots cut into tiles of 64: slots below `turn` are the first keys, slot u
// from there on is key u - turn + lo, up to the position of the last query.  No tile is spent on the gap between them,
// and the window starts at the very first key that a query of the block sees.  In a cache so long that a tile with
// keys of both kinds would span 2^31 bytes, `turn` is rounded up to a whole tile.
struct WindowKeys {
  int sinks, lo, turn, n;  // n: tiles
  __device__ __forceinline__ int jump() const { return lo - turn; }
};
__device__ __forceinline__ WindowKeys window_keys(int p_lo, int p_hi, int window, int sinks, long long stride) {
  WindowKeys k;
  k.sinks = min(sinks, p_hi + 1);
  k.lo = max(k.sinks, p_lo - window + 1);
  const bool near = 2 * stride * (k.lo + kWinTile) < 0x7fffffffLL;
  k.turn = near ? k.sinks : (k.sinks + kWinTile - 1) / kWinTile * kWinTile;
  k.n = (k.turn + p_hi + 1 - k.lo + kWinTile - 1) / kWinTile;
  return k;
}

// Chunk swizzle of a tile row: the 16-byte chunk c of row r lies at position c ^ win_swz(r).  One swizzle serves the
// reads along the rows (one row per lane) and the transposing reads (four rows x 64 bytes per 32 lanes).
template <int DH>
__device__ __forceinline__ int win_swz(int row) {
  const int r0 = row & 1, r1 = (row >> 1) & 1, r2 = (row >> 2) & 1, r3 = (row >> 3) & 1;
  if constexpr (DH == 128) return (r0 << 1) | (r1 << 2) | r2 | ((r0 ^ r3) << 3);
  return r0 | (r1 << 2) | (r2 << 1);
}

// ROWS rows of DH columns, memory -> LDS, by WAVES wavefronts.  `rows` of them exist (<= 0: none), `dim` columns hold data,
// the rest arrives as zeros.  Byte offsets stay inside the tile: the caller's pointer is the tile's first row.  Rows from
// `turn` on lie `jump` rows further.
template <typename T, int DH, int ROWS, int WAVES>
__device__ __forceinline__ void win_copy(const T* src, long long stride, int rows, int dim, T* dst, int wave, int lane,
                                         int turn = ROWS, int jump = 0) {
  constexpr int CH = DH / 8;            // chunks of a row
  constexpr int PER = 64 / CH;          // rows of one instruction
  constexpr int N = ROWS / PER / WAVES;  // instructions of a wavefront
  const int step = 2 * static_cast<int>(stride);
  const int bytes = rows > 0 ? (min(rows, ROWS) - 1 + jump) * step + dim * 2 : 0;
#pragma unroll
  for (int u = 0; u < N; ++u) {
    const int blk = wave * N + u;
    const int row = blk * PER + lane / CH;
    const int chunk = (lane % CH) ^ win_swz<DH>(row);
    const int at = row >= turn ? row + jump : row;
    const int voff = 8 * chunk < dim ? at * step + 16 * chunk : 0x7ffffff0;
    __builtin_amdgcn_raw_ptr_buffer_load_lds(
        __builtin_amdgcn_make_buffer_rsrc(const_cast<T*>(src), 0, bytes, 0x00020000),
        (__attribute__((address_space(3))) void*)(dst + blk * 512), 16, voff, 0, 0, 0);
  }
}
// Tile t of a block's keys: rows of the key or value matrix `src` that starts at key 0 and has `length` rows
template <typename T, int DH>
__device__ __forceinline__ void win_copy_keys(const T* src, long long stride, const WindowKeys& k, int t, int length, int dim, T* dst,
                                              int wave, int lane) {
  const int slot = t * kWinTile;
  if (slot >= k.turn) {  // a path of its own: with the turn's selects in every tile a long prefill took 5 % longer
    const int key = slot + k.jump();
    win_copy<T, DH, kWinTile, kWinWaves>(src + key * stride, stride, length - key, dim, dst, wave, lane);
  } else {
    const bool both = slot + kWinTile > k.turn;
    win_copy<T, DH, kWinTile, kWinWaves>(src + slot * stride, stride, length - slot - (both ? k.jump() : 0), dim, dst, wave, lane,
                                     both ? k.turn - slot : kWinTile, both ? k.jump() : 0);
  }
}

// Fragment addresses.  With the swizzle, the place of a fragment is the lane's base with a constant XORed into its chunk
// bits and a constant added above them: two registers address every fragment of every tile, where one register per
// distinct fragment (which is what the compiler makes of loop-invariant addresses) pushed accumulators into scratch.
// `win_bases` gives the bases for a buffer and keeps the compiler from hoisting what follows from them.
struct WinBases {
  uint32_t row, tr;
};
// `lds`: the kernel's dynamic LDS, in which the buffers start.
template <int DH>
__device__ __forceinline__ WinBases win_lane_bases(unsigned char* lds, int lane) {
  const int li = lane & 31, g = lane >> 5;
  const int sl = lane & 15, grp = lane >> 4;
  const int tr_row = 4 * (grp >> 1) + (sl >> 2);
  const int tr_chunk = 2 * (grp & 1) + ((sl & 3) >> 1);
  const uint32_t start = (uint32_t)(__attribute__((address_space(3))) unsigned char*)lds;
  WinBases b;
  b.row = start + li * DH * 2 + 16 * (g ^ win_swz<DH>(li));
  b.tr = start + tr_row * DH * 2 + 16 * (tr_chunk ^ win_swz<DH>(tr_row)) + 8 * (sl & 1);
  return b;
}
__device__ __forceinline__ WinBases win_bases(WinBases lane_bases, uint32_t buffer) {
  WinBases b{lane_bases.row + buffer, lane_bases.tr + buffer};
  asm volatile("" : "+v"(b.row), "+v"(b.tr));
  return b;
}
// A operand along the rows: row 32 block + lane % 32, d slice s, half lane / 32, of the tile `at` bytes into the buffer
template <typename T, int DH>
__device__ __forceinline__ typename AttnElem<T>::x8 win_row_frag(const WinBases& b, int at, int block, int s) {
  return *(const __attribute__((address_space(3))) typename AttnElem<T>::x8*)((b.row ^ (32 * s)) + at + 64 * DH * block);
}
// A operand across the rows (the tile transposed): columns 32 db + lane % 32, row slice t of 16.  In every group of 16
// lanes, lane s points at four consecutive d of row 4 g + s / 4 (+ 8 for the second read) and receives, for its own d,
// the four rows: the order in which the accumulators of the first product hold them.
template <typename T, int DH>
__device__ __forceinline__ typename AttnElem<T>::x8 win_tr_frag(const WinBases& b, int at, int db, int t) {
  typedef AttnElem<T> E;
  typedef __attribute__((address_space(3))) typename E::x4v lds_x4;
  const typename E::x4 lo = E::read_tr_lds((lds_x4*)((b.tr ^ (64 * db)) + at + 32 * DH * t));
  const typename E::x4 hi = E::read_tr_lds((lds_x4*)((b.tr ^ (64 * db) ^ (16 * win_swz<DH>(8))) + at + 32 * DH * t + 16 * DH));
  typename E::x8 r;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    r[e] = lo[e];
    r[4 + e] = hi[e];
  }
  return r;
}

// B operand fragments of one row in memory: zeros past the head dimension
template <typename T, int DS>
__device__ __forceinline__ void win_load_row(typename AttnElem<T>::x8 (&f)[DS], const T* row, int dim, int g) {
#pragma unroll
  for (int s = 0; s < DS; ++s) {
    const int c = 16 * s + 8 * g;
    if (c < dim) {
      f[s] = *reinterpret_cast<const typename AttnElem<T>::x8*>(row + c);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) f[s][e] = static_cast<T>(0.f);
    }
  }
}

// maximum and sum over the two halves of a wavefront that hold a row, by a register swap
__device__ __forceinline__ float win_half_max(float x) {
  const auto sw = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return fmaxf(__uint_as_float(sw[0]), __uint_as_float(sw[1]));
}
__device__ __forceinline__ float win_half_sum(float x) {
  const auto sw = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __uint_as_float(sw[0]) + __uint_as_float(sw[1]);
}

// keeps the computation of a fragment in its place: the compiler otherwise moves it to the fragment's use, behind the
// products of the next block, and holds the fp32 scores until then
template <typename X8>
__device__ __forceinline__ void win_pin(X8& f) {
  u32x4_t w = __builtin_bit_cast(u32x4_t, f);
  asm volatile("" : "+v"(w));
  f = __builtin_bit_cast(X8, w);
}

// zero, but nothing the compiler can compute with: what follows from it stays in the walk that it is used in
__device__ __forceinline__ int win_first() {
  int zero = 0;
  asm volatile("" : "+s"(zero));
  return zero;
}

template <int DB>
__device__ __forceinline__ void win_zero(f32x16_t (&acc)[DB]) {
#pragma unroll
  for (int db = 0; db < DB; ++db)
#pragma unroll
    for (int r = 0; r < 16; ++r) acc[db][r] = 0.f;
}

// Hidden pairs and what is no number.  The matrix instruction multiplies hidden pairs too, by a factor of zero, and zero
// times a NaN or an infinity is NaN: a row that holds one would reach everything that shares a tile with it.  That always
// leaves NaN in a sum, so nobody looks for it in the tiles: a workgroup that finds something else than numbers in its
// sums starts over, clears such elements in every tile before it enters the products (win_clear), and walks the tiles once more
// to give what it cleared to those who see it (win_reach).  Sums that hold NaN by right cost the same three walks.  The
// check takes a meeting of the workgroup: 12.1 against 11.6 us for a short padded prefill, nothing measurable for long ones.

__device__ __forceinline__ bool win_is_number(float x) { return __builtin_fabsf(x) < __builtin_inff(); }

// max(m, |x|) over what is a number
__device__ __forceinline__ float win_largest(float m, float x) { return win_is_number(x) ? fmaxf(m, __builtin_fabsf(x)) : m; }

// Whether any wavefront of the workgroup has something else than numbers in its sums (of the lanes `mine`).  `words`: LDS that
// nobody else uses until the workgroup meets again.
template <int DB>
__device__ __forceinline__ bool win_lost(const f32x16_t (&acc)[DB], bool mine) {
  float zero = 0.f;
#pragma unroll
  for (int db = 0; db < DB; ++db)
#pragma unroll
    for (int r = 0; r < 16; ++r) zero = fmaf(acc[db][r], 0.f, zero);
  return __any(mine && zero != 0.f);  // NaN compares unequal
}
// Whether there is nothing left to lose: every sum is NaN
template <int DB>
__device__ __forceinline__ bool win_all_lost(const f32x16_t (&acc)[DB], bool mine) {
  bool number = false;
#pragma unroll
  for (int db = 0; db < DB; ++db)
#pragma unroll
    for (int r = 0; r < 16; ++r) number |= acc[db][r] == acc[db][r];
  return !__any(mine && number);
}
template <int WAVES, int DB>
__device__ __forceinline__ bool win_any_lost(const f32x16_t (&acc)[DB], bool mine, int* words, int wave, int lane) {
  const bool lost = win_lost(acc, mine);
  if (lane == 0) words[wave] = lost;
  __syncthreads();
  int any = 0;
#pragma unroll
  for (int w = 0; w < WAVES; ++w) any |= words[w];
  return __builtin_amdgcn_readfirstlane(any) != 0;
}
// Zeros for what is no number in a tile of `elements` in LDS, by THREADS threads
template <typename T, int THREADS>
__device__ __forceinline__ void win_clear(T* tile, int elements, int thread) {
  typedef typename AttnElem<T>::x8 x8_t;
#pragma nounroll
  for (int c = 8 * thread; c < elements; c += 8 * THREADS) {
    x8_t f = *reinterpret_cast<const x8_t*>(tile + c);
    bool clear = false;
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (!win_is_number(static_cast<float>(f[e]))) {
        f[e] = static_cast<T>(0.f);
        clear = true;
      }
    if (clear) *reinterpret_cast<x8_t*>(tile + c) = f;
  }
}
// The same for the fragments of a row
template <typename T, int DS>
__device__ __forceinline__ void win_clear_row(typename AttnElem<T>::x8 (&f)[DS]) {
#pragma unroll
  for (int i = 0; i < DS; ++i)
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (!win_is_number(static_cast<float>(f[i][e]))) f[i][e] = static_cast<T>(0.f);
}
// Whether row `row` of a tile holds something else than numbers
template <typename T, int DH>
__device__ __forceinline__ bool win_bad_row(const T* tile, int row) {
  typedef typename AttnElem<T>::x8 x8_t;
  bool bad = false;
#pragma nounroll
  for (int c = 0; c < DH; c += 8) {
    const x8_t f = *reinterpret_cast<const x8_t*>(tile + row * DH + c);
#pragma unroll
    for (int e = 0; e < 8; ++e) bad |= !win_is_number(static_cast<float>(f[e]));
  }
  return bad;
}
// Adds what is no number in a tile of 16 SLICES rows to the transposed sums (lane = who sees a row or not, registers =
// columns) of those who see it: an infinity times a positive weight is itself.  Ones in its place times ones for the
// pairs that sees(row) says are seen, first for what goes up and then for what goes down; a NaN goes both ways.
template <typename T, int DH, int SLICES, int DB, class Sees>
__device__ __forceinline__ void win_reach(f32x16_t (&acc)[DB], const WinBases& at, int tile, int g, Sees&& sees) {
  typedef AttnElem<T> E;
  typedef typename E::x8 x8_t;
#pragma nounroll
  for (int t = 0; t < SLICES; ++t) {
    x8_t seen;
#pragma unroll
    for (int e = 0; e < 8; ++e) seen[e] = static_cast<T>(sees(16 * t + 8 * (e >> 2) + 4 * g + (e & 3)) ? 1.f : 0.f);
#pragma unroll
    for (int db = 0; db < DB; ++db) {
      const x8_t f = win_tr_frag<T, DH>(at, tile + 32 * DH * t, db, 0);
#pragma unroll
      for (int up = 0; up < 2; ++up) {
        x8_t goes;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float x = static_cast<float>(f[e]);
          goes[e] = static_cast<T>((up ? x < __builtin_inff() : x > -__builtin_inff()) ? 0.f : 1.f);
        }
        f32x16_t reached;
#pragma unroll
        for (int r = 0; r < 16; ++r) reached[r] = 0.f;
        reached = E::mfma(goes, seen, reached);
#pragma unroll
        for (int r = 0; r < 16; ++r) acc[db][r] += reached[r] > 0.f ? (up ? __builtin_inff() : -__builtin_inff()) : 0.f;
        __builtin_amdgcn_sched_barrier(0);
      }
    }
  }
}
// The same where the weights have no sign to go by: all that such a row reaches is NaN.
template <int DB>
__device__ __forceinline__ void win_reach_all(f32x16_t (&acc)[DB], bool sees) {
#pragma unroll
  for (int db = 0; db < DB; ++db)
#pragma unroll
    for (int r = 0; r < 16; ++r) acc[db][r] = sees ? __builtin_nanf("") : acc[db][r];
}

// Transposed accumulators (lane = row, registers = columns) of a wavefront's 32 rows -> memory, through the
// wavefront's own 32 x DH piece of LDS so that whole rows leave.  Rows below `exist` get the values times the lane's
// factor, those from there to `rows` zeros.  REMAINDER stores what the rounding of that value lost instead.
template <typename T, int DH, bool REMAINDER = false, int DB>
__device__ __forceinline__ void win_store(T* dst, long long stride, const f32x16_t (&acc)[DB], float factor, T* stage,
                                          int lane, int exist, int rows, int dim) {
  typedef typename AttnElem<T>::x4 x4_t;
  constexpr int CH = DH / 8;
  const int li = lane & 31, g = lane >> 5;
#pragma unroll
  for (int db = 0; db < DB; ++db)
#pragma unroll
    for (int rq = 0; rq < 4; ++rq) {
      x4_t o4;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        float x = li < exist ? acc[db][4 * rq + e] * factor : 0.f;
        // the product is rounded to fp32 here: fused into a conversion or the subtraction it would round another
        // way near a tie, and value and remainder would not belong together
        asm volatile("" : "+v"(x));
        o4[e] = static_cast<T>(REMAINDER ? x - static_cast<float>(static_cast<T>(x)) : x);
      }
      *reinterpret_cast<x4_t*>(stage + li * DH + 8 * ((4 * db + rq) ^ (li % CH)) + 4 * g) = o4;
    }
  const int c = lane % CH;
#pragma unroll
  for (int j = 0; j < CH / 2; ++j) {
    const int row = j * (64 / CH) + lane / CH;
    const u32x4_t v16 = *reinterpret_cast<const u32x4_t*>(stage + row * DH + 8 * (c ^ (row % CH)));
    if (row < rows && 8 * c < dim) *reinterpret_cast<u32x4_t*>(dst + row * stride + 8 * c) = v16;
  }
}

// Where a workgroup works.  Consecutive ids go round-robin to the eight dies, each with its own L2: a die takes a
// contiguous eighth of the items, which run through one key head's query blocks before the next, from the last to the
// first (a block without a full window before it is shorter).
struct WindowBlock {
  int b, kvh, qb, hg;
  bool any;
};
__device__ __forceinline__ WindowBlock window_block(const WindowShape& s, int blocks, int parts) {
  const int per_kv = blocks * parts;
  const int total = s.batch * s.kv_heads * per_kv;
  const int share = (total + 7) / 8;
  const int item = (blockIdx.x % 8) * share + blockIdx.x / 8;
  WindowBlock w;
  w.any = static_cast<int>(blockIdx.x / 8) < share && item < total;
  const int unit = item / per_kv, rest = item % per_kv;
  w.b = unit / s.kv_heads;
  w.kvh = unit % s.kv_heads;
  const int at = rest / parts;
  w.hg = rest % parts;
  w.qb = blocks - 1 - at;
  return w;
}

// What one wavefront sees of the block: 32 queries of one head.
struct WindowWave {
  int head, q0, exist, rows;  // first query, how many of the 32 exist, how many lie inside Sq
  int p_lo, p_hi;             // positions of the first and last that exist
  int window;
  // some query sees some key of tile t / every query sees every key
  __device__ __forceinline__ bool active(const WindowKeys& k, int t) const {
    const int slot = t * kWinTile, key = slot + k.jump();
    const bool first = slot < k.sinks && slot <= p_hi;
    const bool rest = slot + kWinTile > k.turn && key <= p_hi && key + kWinTile - 1 > p_lo - window;
    return exist > 0 && (first || rest);
  }
  __device__ __forceinline__ bool whole(const WindowKeys& k, int t) const {
    const int slot = t * kWinTile, key = slot + k.jump();
    if (slot >= k.turn) return key + kWinTile - 1 <= p_lo && key > p_hi - window;
    return slot + kWinTile <= k.sinks && slot + kWinTile - 1 <= p_lo;
  }
  // sets x[r] (key rows 8 (r / 4) + 4 g + r % 4 of the 32 slots from `slot` on) to -inf where position p does not see it
  __device__ __forceinline__ void hide(const WindowKeys& k, int slot, int p, int g, f32x16_t& x) const {
    const int near = p - (slot + k.jump() + 4 * g);  // offset o is behind p by near - o, if o is a window slot
    const int far = near - window;
    const int turn = k.turn - slot - 4 * g;
    const int first = min(k.sinks, p + 1) - slot - 4 * g;  // first keys: offsets below it are seen
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      const int o = 8 * (r >> 2) + (r & 3);
      // without short circuits: each would be a branch around two compares
      const bool hidden = ((o < turn) & (o >= first)) | ((o >= turn) & ((o > near) | (o <= far)));
      x[r] = hidden ? -__builtin_inff() : x[r];
    }
  }
  // whether position p sees slot `slot`
  __device__ __forceinline__ bool sees(const WindowKeys& k, int slot, int p) const {
    const int key = slot + k.jump();
    return slot < k.turn ? slot < min(k.sinks, p + 1) : key <= p && key > p - window;
  }
};
__device__ __forceinline__ WindowWave window_wave(const WindowShape& s, const WindowBlock& w, int wave, int query_end) {
  WindowWave v;
  const int per_head = kWinWaves >> s.hb_shift;  // wavefronts of a head
  v.head = w.kvh * s.group + (w.hg << s.hb_shift) + wave / per_head;
  v.q0 = w.qb * (32 * per_head) + 32 * (wave % per_head);
  v.exist = min(32, query_end - v.q0);
  v.rows = min(32, s.Sq - v.q0);
  v.p_lo = v.q0 + s.offset();
  v.p_hi = v.p_lo + v.exist - 1;
  v.window = s.window;
  return v;
}

// ---------------------------------------------------------------------------------------------
// forward
// ---------------------------------------------------------------------------------------------
struct WindowFwdArgs {
  const void *q, *k, *v;
  void* o;
  void* low;   // may be null: what rounding o lost, laid out like o
  float* lse;  // [B, N, Sq]
  WindowShape shape;
  WindowStride qs, ks, vs, os;
};

template <typename T, int DH>
__device__ __forceinline__ void window_attention_fwd(const WindowFwdArgs& a) {
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
  const long long o_at = w.b * a.os.batch + me.head * a.os.head + me.q0 * a.os.token;
  T* O = static_cast<T*>(a.o) + o_at;
  float* lse = a.lse + (static_cast<size_t>(w.b) * s.heads + me.head) * s.Sq + me.q0;
  T* stage = reinterpret_cast<T*>(attn_lds) + wave * (32 * DH);
  f32x16_t oacc[DB];
  win_zero(oacc);
  const int block_q0 = w.qb * per_block;
  if (block_q0 >= query_end) {  // nothing here exists
    win_store<T, DH>(O, a.os.token, oacc, 0.f, stage, lane, 0, me.rows, s.dim);
    if (a.low != nullptr) win_store<T, DH>(static_cast<T*>(a.low) + o_at, a.os.token, oacc, 0.f, stage, lane, 0, me.rows, s.dim);
    if (g == 0 && li < me.rows) lse[li] = -__builtin_inff();
    return;
  }
  const int p_lo = block_q0 + s.offset();
  const int p_hi = min(block_q0 + per_block, query_end) - 1 + s.offset();
  const WindowKeys keys = window_keys(p_lo, p_hi, s.window, s.sinks, max(a.ks.token, a.vs.token));

  x8_t qf[DS];
  const int qi = min(me.q0 + li, s.Sq - 1);  // rows past the end work on a copy of the last row and are not stored
  win_load_row<T>(qf, static_cast<const T*>(a.q) + w.b * a.qs.batch + me.head * a.qs.head + qi * a.qs.token, s.dim, g);
  const int p = me.p_lo + li;
  const float scale2 = s.scale2;

  const T* K = static_cast<const T*>(a.k) + w.b * a.ks.batch + w.kvh * a.ks.head;
  const T* V = static_cast<const T*>(a.v) + w.b * a.vs.batch + w.kvh * a.vs.head;
  T* buffers = reinterpret_cast<T*>(attn_lds);  // two of K and V
  auto request = [&](int i) {
    T* dst = buffers + (i & 1) * 2 * TILE;
    win_copy_keys<T, DH>(K, a.ks.token, keys, i, length, s.dim, dst, wave, lane);
    win_copy_keys<T, DH>(V, a.vs.token, keys, i, length, s.dim, dst + TILE, wave, lane);
  };
  const WinBases lane_bases = win_lane_bases<DH>(attn_lds, lane);
  float m, l;
  for (bool guarded = false;; guarded = true) {
    m = kWinFloor, l = 0.f;
    request(win_first());
    __builtin_amdgcn_s_waitcnt(0x0F70);  // vmcnt(0)
    __syncthreads();
    for (int i = 0; i < keys.n; ++i) {
      if (guarded) {
        win_clear<T, kWinThreads>(buffers + (i & 1) * 2 * TILE + TILE, TILE, threadIdx.x);
        __syncthreads();
      }
      if (i + 1 < keys.n) request(i + 1);
      if (me.active(keys, i)) {
        const WinBases at = win_bases(lane_bases, (i & 1) * 4 * TILE);
        f32x16_t sacc[2];
        win_zero(sacc);
#pragma unroll
        for (int kb = 0; kb < 2; ++kb)
#pragma unroll
          for (int d = 0; d < DS; ++d) sacc[kb] = E::mfma(win_row_frag<T, DH>(at, 0, kb, d), qf[d], sacc[kb]);
        if (!me.whole(keys, i)) {
#pragma unroll
          for (int kb = 0; kb < 2; ++kb) me.hide(keys, i * kWinTile + 32 * kb, p, g, sacc[kb]);
        }
        float mx = sacc[0][0];
#pragma unroll
        for (int kb = 0; kb < 2; ++kb)
#pragma unroll
          for (int r = 0; r < 16; ++r) mx = fmaxf(mx, sacc[kb][r]);
        mx = fmaxf(win_half_max(mx) * scale2, kWinFloor);
        const float m_new = mx > m + kAttnSlack ? mx : m;
        const float alpha = __builtin_amdgcn_exp2f(m - m_new);
        m = m_new;
        x8_t pf[4];
        float sum = 0.f;
#pragma unroll
        for (int kb = 0; kb < 2; ++kb)
#pragma unroll
          for (int r = 0; r < 16; ++r) {
            const float e = __builtin_amdgcn_exp2f(fmaf(sacc[kb][r], scale2, -m));
            sum += e;
            pf[2 * kb + (r >> 3)][r & 7] = static_cast<T>(e);  // the product with V takes 16 bits; the sum keeps 32
          }
        l = fmaf(l, alpha, sum);
        if (__any(alpha != 1.f)) {
#pragma unroll
          for (int db = 0; db < DB; ++db)
#pragma unroll
            for (int r = 0; r < 16; ++r) oacc[db][r] *= alpha;
        }
#pragma unroll
        for (int k4 = 0; k4 < 4; ++k4)
#pragma unroll
          for (int db = 0; db < DB; ++db) oacc[db] = E::mfma(win_tr_frag<T, DH>(at, 2 * TILE, db, k4), pf[k4], oacc[db]);
      }
      __builtin_amdgcn_s_waitcnt(0x0F70);  // vmcnt(0): the next tile has landed
      __syncthreads();
    }
    if (guarded) {
      for (int i = 0; i < keys.n; ++i) {
        request(i);
        __builtin_amdgcn_s_waitcnt(0x0F70);  // vmcnt(0)
        __syncthreads();
        const T* V = buffers + (i & 1) * 2 * TILE + TILE;
        if (!win_all_lost(oacc, li < me.exist) && __any(win_bad_row<T, DH>(V, lane)))
          win_reach<T, DH, 4>(oacc, win_bases(lane_bases, (i & 1) * 4 * TILE), 2 * TILE, g,
                              [&](int row) { return me.sees(keys, i * kWinTile + row, p); });
        __syncthreads();
      }
      break;
    }
    // the words lie behind the wavefronts' pieces for the store
    if (!win_any_lost<kWinWaves>(oacc, li < me.exist, reinterpret_cast<int*>(attn_lds + 4 * TILE * sizeof(T) - 64), wave, lane)) break;
    __syncthreads();
    win_zero(oacc);
  }
  l = win_half_sum(l);
  win_store<T, DH>(O, a.os.token, oacc, 1.0f / l, stage, lane, me.exist, me.rows, s.dim);
  if (a.low != nullptr)
    win_store<T, DH, true>(static_cast<T*>(a.low) + o_at, a.os.token, oacc, 1.0f / l, stage, lane, me.exist, me.rows, s.dim);
  if (g == 0 && li < me.rows)
    lse[li] = li < me.exist ? (m + __builtin_amdgcn_logf(l)) * kWinLn2 : -__builtin_inff();
}

}  // namespace mi
