// Attention whose scores and masks go by positions (fl_attention_scores).
#include <cmath>
#include <type_traits>

#include "decoder_common.h"

using namespace fl;

namespace {

struct AttentionView {
  void *base;
  int64_t strides[4];  // batch, head, position, column
};

struct AttentionArgs {
  AttentionView q, k, v, out;
  const float *slopes;
  const int32_t *prefix_lengths, *query_documents, *key_documents, *query_starts, *query_lengths, *key_lengths;
  int64_t slope_stride, prefix_stride, query_document_strides[2], key_document_strides[2], query_start_stride, query_length_stride, key_length_stride;
  int64_t window;
  int32_t batch, heads, kv_heads, group, queries, keys, columns, causal;
  int32_t rows;  // of a key head: queries * group
  float scale2;  // |scale|, in powers of two; its sign is Q's
  float sign, cap, cap2, scale_by_cap, scale_by_cap2;
  int32_t q_aligned, out_aligned, by_xcd;
  FastDiv group_div, kv_div, tiles_div, heads_div;  // query heads of a key head, key heads, tiles of rows, key heads of all sequences
  int2 *ranges;  // documents of every kBlock keys [batch, blocks], or NULL
  int32_t blocks, splits;
  float *partial;  // [splits, batch * kv_heads * rows, columns]
  float2 *stats;   // maximum and sum [splits, batch * kv_heads * rows]
};

constexpr float kLog2e = 1.4426950408889634f;
constexpr int kBlock = 64;         // keys whose documents the ranges cover
constexpr float kLazy = 8.0f;      // a maximum may be behind by this many powers of two before the sums are scaled
constexpr int64_t kFar = 1 << 30;  // distances to queries further from the keys than this are taken as to here: to a softmax they are the same

typedef _Float16 halfx8 __attribute__((ext_vector_type(8)));
typedef float floatx4 __attribute__((ext_vector_type(4)));
typedef int32_t intx4 __attribute__((ext_vector_type(4)));
typedef short shortx4 __attribute__((ext_vector_type(4)));

// What one sequence looks like to a query of it.
struct Sequence {
  int32_t n_queries, n_keys, start, prefix;  // prefix <= n_keys
};

__device__ __forceinline__ Sequence SequenceOf(const AttentionArgs &a, int b) {
  Sequence s;
  s.n_keys = a.key_lengths == nullptr ? a.keys : min(max(a.key_lengths[b * a.key_length_stride], 0), a.keys);
  s.n_queries = a.query_lengths == nullptr ? a.queries : min(max(a.query_lengths[b * a.query_length_stride], 0), a.queries);
  s.start = a.query_starts == nullptr ? s.n_keys - s.n_queries : a.query_starts[b * a.query_start_stride];
  s.prefix = a.prefix_lengths == nullptr ? 0 : min(max(a.prefix_lengths[b * a.prefix_stride], 0), s.n_keys);
  return s;
}

// The keys [lo, hi) that query i sees beside the prefix, 0 <= lo, hi <= n_keys.  (Starts may be any 32-bit number and windows any 64-bit one.)
__device__ __forceinline__ int32_t Within(const Sequence &s, int64_t j) { return static_cast<int32_t>(min(max(j, int64_t{0}), static_cast<int64_t>(s.n_keys))); }
__device__ __forceinline__ int32_t FirstKey(const AttentionArgs &a, const Sequence &s, int32_t i) {
  return a.window == 0 ? 0 : Within(s, static_cast<int64_t>(s.start) + i - a.window + 1);
}
__device__ __forceinline__ int32_t LastKey(const AttentionArgs &a, const Sequence &s, int32_t i) {
  const int64_t at = static_cast<int64_t>(s.start) + i;
  int64_t hi = s.n_keys;
  if (a.causal) hi = min(hi, at + 1);
  if (a.window != 0) hi = min(hi, at + a.window);
  return Within(s, hi);
}

// The row of a tile that a lane works for: row r of a key head is head r % group of query r / group.
struct Row {
  int32_t i, head;  // query and head
  int32_t at, lo, hi, prefix, document;
  float slope;  // in powers of two
  bool there;   // has a result
};

__device__ __forceinline__ Row RowOf(const AttentionArgs &a, const Sequence &s, int b, int kv, int32_t r) {
  Row row;
  row.i = static_cast<int32_t>(a.group_div.Div(static_cast<uint32_t>(r)));
  row.head = kv * a.group + (r - row.i * a.group);
  row.there = row.i < s.n_queries;
  const int32_t i = min(row.i, a.queries - 1);  // (what is read for rows that are not there)
  row.at = static_cast<int32_t>(min(max(static_cast<int64_t>(s.start) + row.i, -kFar), kFar));
  row.document = a.query_documents == nullptr ? 0 : a.query_documents[b * a.query_document_strides[0] + i * a.query_document_strides[1]];
  const bool sees = row.there && row.document >= 0;
  if (row.document < 0) row.document = -2;
  row.lo = sees ? FirstKey(a, s, row.i) : 0;
  row.hi = sees ? max(LastKey(a, s, row.i), row.lo) : 0;
  row.prefix = sees ? s.prefix : 0;
  row.slope = a.slopes == nullptr ? 0.0f : a.slopes[row.head * a.slope_stride] * kLog2e;
  return row;
}

// (-1: padding, which no row's document is)
__device__ __forceinline__ int32_t KeyDocument(const AttentionArgs &a, int b, int32_t j) {
  return max(a.key_documents[b * a.key_document_strides[0] + static_cast<int64_t>(j) * a.key_document_strides[1]], -1);
}

__device__ __forceinline__ bool Sees(const AttentionArgs &a, const Row &row, int b, int32_t j) {
  bool sees = (j >= row.lo && j < row.hi) || j < row.prefix;
  if (sees && a.key_documents != nullptr) sees = KeyDocument(a, b, j) == row.document;
  return sees;
}

// cap tanh(scale (q . k) / cap), in powers of two
__device__ __forceinline__ float Capped(const AttentionArgs &a, float dot) { return a.cap2 * tanhf(dot * a.scale_by_cap); }

// One row by one wave, key by key as the definition has it: what a row gets whose sums are not finite.  (A tile's products take in
// every value of its keys, 0 * infinity among them; here what a query does not see is not read.)
template <typename T>
__device__ __forceinline__ void CarefulRow(const AttentionArgs &a, int b, int kv, int32_t r) {
  const int lane = threadIdx.x % kWave;
  const Sequence seq = SequenceOf(a, b);
  const Row row = RowOf(a, seq, b, kv, r);
  const T *const q = static_cast<const T *>(a.q.base) + b * a.q.strides[0] + row.head * a.q.strides[1] + row.i * a.q.strides[2];
  const T *const k = static_cast<const T *>(a.k.base) + b * a.k.strides[0] + kv * a.k.strides[1];
  const T *const v = static_cast<const T *>(a.v.base) + b * a.v.strides[0] + kv * a.v.strides[1];
  float most = -INFINITY, sum = 0.0f, acc[FL_ATTENTION_MAX_HEAD / kWave] = {};
  for (int32_t j0 = 0; j0 < seq.n_keys; j0 += kWave) {
    const int32_t j = j0 + lane;
    const bool sees = Sees(a, row, b, j);
    const uint64_t which = __ballot(sees);
    if (which == 0) continue;
    float s = -INFINITY;
    if (sees) {
      s = 0.0f;
      for (int d = 0; d < a.columns; ++d) s += static_cast<float>(q[d * a.q.strides[3]]) * a.sign * static_cast<float>(k[j * a.k.strides[2] + d * a.k.strides[3]]);
      s = a.cap == 0.0f ? s * a.scale2 : Capped(a, s);
      if (a.slopes != nullptr) s -= row.slope * fabsf(static_cast<float>(row.at - j));
    }
    const float now = fmaxf(most, WaveReduce(s, MaxOp{}));
    const float from = now == -INFINITY ? 0.0f : now;
    const float kept = most == -INFINITY ? 0.0f : exp2f(most - from);
    const float p = exp2f(s - from);
    sum = sum * kept + GroupSum<64>(p);
    most = now;
#pragma unroll
    for (float &x : acc) x *= kept;
    for (uint64_t rest = which; rest != 0; rest &= rest - 1) {
      const int e = __builtin_ctzll(rest);
      const float w = __shfl(p, e);
#pragma unroll
      for (int c = 0; c < FL_ATTENTION_MAX_HEAD / kWave; ++c) {
        const int d = c * kWave + lane;
        if (d < a.columns) acc[c] += w * static_cast<float>(v[(j0 + e) * a.v.strides[2] + d * a.v.strides[3]]);
      }
    }
  }
  T *const to = static_cast<T *>(a.out.base) + b * a.out.strides[0] + row.head * a.out.strides[1] + row.i * a.out.strides[2];
#pragma unroll
  for (int c = 0; c < FL_ATTENTION_MAX_HEAD / kWave; ++c) {
    const int d = c * kWave + lane;
    if (d < a.columns) to[d * a.out.strides[3]] = static_cast<T>(sum == 0.0f ? 0.0f : acc[c] / sum);
  }
}

// The smallest and the largest document of every kBlock keys, so that tiles of other documents are passed over unread.
__global__ __launch_bounds__(256) void DocumentRangesKernel(const AttentionArgs a) {
  const int lane = threadIdx.x % kWave;
  const int32_t block = blockIdx.x * 4 + threadIdx.x / kWave, b = blockIdx.y;
  if (block >= a.blocks) return;
  const int32_t id = KeyDocument(a, b, min(block * kBlock + lane, a.keys - 1));
  const int32_t least = WaveReduce(id, [](int32_t x, int32_t y) { return min(x, y); });
  const int32_t most = WaveReduce(id, [](int32_t x, int32_t y) { return max(x, y); });
  if (lane == 0) a.ranges[static_cast<int64_t>(b) * a.blocks + block] = make_int2(least, most);
}

// Walks the tiles of BK keys that some row of a tile of rows sees, 64 candidates at a time: a lane looks at one.
template <int BK>
struct Tiles {
  int32_t lo, hi, prefix;    // keys that some row may see
  int32_t least, most;       // documents of the rows
  int32_t first, step, end;  // candidates: first, first + step, .. below end
  int32_t base;
  uint64_t mask;
  int32_t own_document;      // of the lane's candidate: the one document of its keys, or -1

  __device__ __forceinline__ void Fill(const AttentionArgs &a, int b) {
    mask = 0;
    while (base < end) {
      const int32_t tile = base + static_cast<int32_t>(threadIdx.x % kWave) * step, j = tile * BK;
      bool some = tile < end && ((j < hi && j + BK > lo) || j < prefix);
      if (some && a.ranges != nullptr) {
        const int2 r = a.ranges[static_cast<int64_t>(b) * a.blocks + j / kBlock];
        some = r.y >= least && r.x <= most;
        own_document = r.x == r.y ? r.x : -1;
      }
      mask = __ballot(some);
      if (mask != 0) return;
      base += kWave * step;
    }
  }
  // the next tile, or -1; `document`: of all its keys, or -1
  __device__ __forceinline__ int32_t Next(const AttentionArgs &a, int b, int32_t &document) {
    if (mask == 0) {
      if (base >= end) return -1;
      base += kWave * step;
      Fill(a, b);
      if (mask == 0) return -1;
    }
    const int32_t at = __builtin_ctzll(mask);
    mask &= mask - 1;
    document = __builtin_amdgcn_readlane(own_document, at);
    return base + at * step;
  }
  __device__ __forceinline__ void Start(const AttentionArgs &a, int b) {
    own_document = -1;
    base = first;
    Fill(a, b);
  }
};

// Applies scale, cap and bias to the dot products of one row with N keys and hides those it does not see.  `key(e)`: the e-th key;
// `document(e)`: its document.  Returns what the values still are to be multiplied by: scores without bias keep their scale until the
// exponential, which has a multiplication to spare.  Scores that are the same amount too small are the same to a softmax.
// PRECISE: the cap to a few roundings of the score itself.  Else cap tanh(x) = cap - 2 cap / (1 + exp(2 x)) without its first
// term, which is good to a few roundings of the cap: far below what 16-bit operands carry.
template <bool PRECISE, int N, typename K, typename D>
__device__ __forceinline__ float Finish(const AttentionArgs &a, const Row &row, bool prefixed, bool whole, bool one_document, float (&s)[N], K key, D document) {
  float by = a.scale2;
  if (a.cap != 0.0f) {
    if constexpr (PRECISE) {
      by = 1.0f;
#pragma unroll
      for (int e = 0; e < N; ++e) s[e] = Capped(a, s[e]);
    } else {
      by = 2.0f * a.cap2;
#pragma unroll
      for (int e = 0; e < N; ++e) s[e] = __builtin_amdgcn_exp2f(s[e] * a.scale_by_cap2);
#pragma unroll
      for (int e = 0; e < N; ++e) s[e] = __builtin_amdgcn_rcpf(-1.0f - s[e]);
    }
  }
  if (a.slopes != nullptr || by == 0.0f) {  // (no scale: an infinite product is no number, and one that is not seen minus infinity)
#pragma unroll
    for (int e = 0; e < N; ++e) s[e] = s[e] * by - row.slope * fabsf(static_cast<float>(row.at - key(e)));
    by = 1.0f;
  }
  if (!whole) {
    const uint32_t width = static_cast<uint32_t>(row.hi - row.lo);  // (never negative: a window holds a key or the row sees none)
    if (prefixed) {
#pragma unroll
      for (int e = 0; e < N; ++e) s[e] = static_cast<uint32_t>(key(e) - row.lo) < width || key(e) < row.prefix ? s[e] : -INFINITY;
    } else {
#pragma unroll
      for (int e = 0; e < N; ++e) s[e] = static_cast<uint32_t>(key(e) - row.lo) < width ? s[e] : -INFINITY;
    }
  }
  if (!one_document) {
#pragma unroll
    for (int e = 0; e < N; ++e) s[e] = document(e) == row.document ? s[e] : -INFINITY;
  }
  return by;
}

// The matrix instructions of a type: 32 x 32 results of sixteen products
template <typename E>
__device__ __forceinline__ floatx16 Mfma32(u32x4 x, u32x4 y, floatx16 acc) {
  if constexpr (std::is_same_v<E, _Float16>) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(halfx8, x), __builtin_bit_cast(halfx8, y), acc, 0, 0, 0);
  } else {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, x), __builtin_bit_cast(bf16x8, y), acc, 0, 0, 0);
  }
}
template <typename E>
__device__ __forceinline__ u32x4 Pack8(const float *x) {
  typedef E Vec __attribute__((ext_vector_type(8)));
  Vec v;
#pragma unroll
  for (int e = 0; e < 8; ++e) v[e] = static_cast<E>(x[e]);
  return __builtin_bit_cast(u32x4, v);
}

// Asks the compiler for this order of the products that stand before it and of the LDS reads of their operands, READS each: those of the
// first AHEAD products, then a product and the reads of a later one in turn.  Left alone it reads each operand right before its product.
template <int AHEAD, int READS, int PRODUCTS>
__device__ __forceinline__ void ReadAhead() {
  constexpr int kProduct = 0x8, kRead = 0x100;
  __builtin_amdgcn_sched_group_barrier(kRead, AHEAD * READS, 0);
  StaticFor<PRODUCTS - AHEAD>([](auto) __attribute__((always_inline)) {
    __builtin_amdgcn_sched_group_barrier(kProduct, 1, 0);
    __builtin_amdgcn_sched_group_barrier(kRead, READS, 0);
  });
  __builtin_amdgcn_sched_group_barrier(kProduct, AHEAD, 0);
}

// Eight neighbouring values of a row from column d on, zeros behind the last column.  (No branch around a load: what is not there is read as the
// last column.)
template <typename T>
__device__ __forceinline__ void Load8(const T *row, int64_t stride, int d, int columns, float (&x)[8]) {
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const float v = static_cast<float>(row[min(d + e, columns - 1) * stride]);
    x[e] = d + e < columns ? v : 0.0f;
  }
}

// ... of a query, whose first of eight is there
template <typename T>
__device__ __forceinline__ void LoadQuery(const AttentionArgs &a, const T *row, int d, float (&x)[8]) {
  if (!a.q_aligned) return Load8(row, a.q.strides[3], d, a.columns, x);
  typedef T Vec __attribute__((ext_vector_type(16 / sizeof(T))));
  constexpr int kVec = 16 / sizeof(T);
#pragma unroll
  for (int n = 0; n < 8 / kVec; ++n) {
    const Vec v = *reinterpret_cast<const Vec *>(row + d + n * kVec);
#pragma unroll
    for (int e = 0; e < kVec; ++e) x[n * kVec + e] = static_cast<float>(v[e]);
  }
}

// --------------------------------------------------------------------------------------------------------------------
// Many rows.  A workgroup owns 128 rows of one key head, 32 a wave, and walks the keys in tiles of BK.  Everything is transposed: the scores
// are K Q^T, so that a lane holds BK / 2 scores of ONE row (lane % 32): maximum and sum stay in the lane but for one exchange between
// the halves of the wave, and what is a row's own (position, slope, document) is one register.  The result is V^T P^T; the
// key that a lane's score stands for and the slot that the instruction reads need only agree with V's, so P goes from registers to registers
// as it lies, and V's columns come out of LDS through the transposing read.
// 16-bit: K and V of the next tile are on their way into LDS (two of each) while one is worked on; one barrier a tile.
// fp32: three bf16 parts of each value (six products, see fl_common.h), split once per workgroup on the way into LDS; the next
// tile waits in registers.  The parts of small terms are summed apart, tile by tile.
// LDS rows are DP values without padding (the loads land side by side), groups of 16 bytes permuted within a row against bank conflicts.
// 4096 queries and keys, 32 heads of 128 columns in bf16, no mask: 307 us, 895 TFLOP/s; causal 182 us; 96 columns 238 us; 64 columns 184 us (746); in
// fp32 with 64 columns 851 us (161 TFLOP/s, where the fp32 instruction reaches 154 in a large product).  Bound by issue: of the cycles 32 % are
// matrix instructions, 46 % the softmax's vector instructions, and 72 % issue something; no LDS conflicts.
template <typename T, int DP, int BK, bool PARTED = std::is_same_v<T, float>>
struct RowsShape {
  static constexpr int kParts = PARTED ? 3 : 1;
  static constexpr int kBuffers = PARTED ? 1 : 2;
  static constexpr int kPlane = BK * DP;                       // values of one part of a tile
  static constexpr int kValues = kBuffers * 2 * kParts * kPlane;  // of K and V
  // LDS serves 256 bytes at a time: sixteen lanes' 16 bytes of one column group of sixteen keys of K, 64 bytes of four keys of V.  A group of a
  // row lies in the place whose number is its own, turned so that those fall on different banks, however many rows lie in 256 bytes.
  static constexpr int kTurns = DP % 128 == 0 ? 16 : DP == 64 ? 8 : 4;  // K: places that a row's number chooses from
  static constexpr int kVTurns = DP % 128 == 0 ? 4 : DP == 64 ? 2 : 1;  // V: in fours
  static __host__ __device__ __forceinline__ constexpr int TurnK(int key) { return DP % 128 == 0 ? key & 15 : DP == 64 ? key >> 1 & 7 : key >> 2 & 3; }
  static __host__ __device__ __forceinline__ constexpr int TurnV(int key) { return DP % 128 == 0 ? (key & 3) * 4 : DP == 64 ? (key >> 1 & 1) * 4 : 0; }
  static constexpr int kGroups = BK * DP / 8;                  // of eight values
  static constexpr int kLoads = kGroups / 256;                 // a thread's, per matrix
};

template <typename T, int DP, int BK, int WAVES>
__global__ __launch_bounds__(256, WAVES) void AttentionRowsKernel(const AttentionArgs a) {
  using Shape = RowsShape<T, DP, BK>;
  constexpr bool kParted = Shape::kParts == 3;
  using E = std::conditional_t<kParted, __bf16, T>;
  constexpr int kParts = Shape::kParts, kSteps = DP / 16, kColumns = DP / 32, kKeyTiles = BK / 32;
  // operands read ahead of the products: 4096 queries and keys of 32 heads of 128, 330 -> 321 us; at 64 columns the registers cost the third wave
  // (114 -> 130), at 256 there are none to spare (16 heads 527 -> 568)
  constexpr bool kAhead = !kParted && (DP == 96 || DP == 128);
  __shared__ alignas(16) uint16_t lds[Shape::kValues];

  // which rows: a key head's workgroups run on one XCD where that comes out even, its last (with a causal mask: longest) rows first
  uint32_t head, tile;
  if (a.by_xcd) {
    const uint32_t xcd = blockIdx.x % 8, at = blockIdx.x / 8;
    head = a.tiles_div.Div(at);
    tile = at - head * a.tiles_div.divisor;
    head = head * 8 + xcd;
  } else {
    tile = a.heads_div.Div(blockIdx.x);
    head = blockIdx.x - tile * a.heads_div.divisor;
  }
  tile = a.tiles_div.divisor - 1 - tile;
  const int b = static_cast<int>(a.kv_div.Div(head)), kv = static_cast<int>(head) - b * a.kv_heads;
  const Sequence seq = SequenceOf(a, b);
  const int lane = threadIdx.x % kWave, half = lane / 32, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int32_t row0 = static_cast<int32_t>(tile) * 128, first_query = static_cast<int32_t>(a.group_div.Div(row0));
  if (first_query >= seq.n_queries) return;
  const int32_t last_query = min(static_cast<int32_t>(a.group_div.Div(min(row0 + 127, a.rows - 1))), seq.n_queries - 1);
  const int32_t wave_row = row0 + wave * 32;
  const Row row = RowOf(a, seq, b, kv, wave_row + lane % 32);
  const bool there = row.there && wave_row + lane % 32 < a.rows;
  const int32_t wave_first = min(static_cast<int32_t>(a.group_div.Div(wave_row)), last_query);
  const int32_t wave_last = min(static_cast<int32_t>(a.group_div.Div(wave_row + 31)), last_query);
  const bool wave_there = wave_row < a.rows && static_cast<int32_t>(a.group_div.Div(wave_row)) < seq.n_queries;
  // keys that all rows of the wave see, and that some do
  const int32_t all_lo = FirstKey(a, seq, wave_last), all_hi = LastKey(a, seq, wave_first);
  const int32_t some_lo = FirstKey(a, seq, wave_first), some_hi = LastKey(a, seq, wave_last);

  // Q^T: sixteen columns a step, eight of them in each half
  u32x4 q[kSteps][kParts];
  {
    const T *const from = static_cast<const T *>(a.q.base) + b * a.q.strides[0] + row.head * a.q.strides[1] + row.i * a.q.strides[2];
#pragma unroll
    for (int s = 0; s < kSteps; ++s) {
      float x[8] = {};
      const int d = s * 16 + half * 8;
      if (there && d < a.columns) {
        LoadQuery(a, from, d, x);
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e] *= a.sign;
      if constexpr (kParted) {
        SplitParts<3>(x, q[s]);
      } else {
        q[s][0] = Pack8<E>(x);
      }
    }
  }

  Tiles<BK> tiles;
  tiles.lo = FirstKey(a, seq, first_query);
  tiles.hi = LastKey(a, seq, last_query);
  tiles.prefix = seq.prefix;
  tiles.first = 0, tiles.step = 1, tiles.end = (seq.n_keys + BK - 1) / BK;
  tiles.least = 0, tiles.most = INT32_MAX;
  int32_t wave_document = -1;  // the document of all rows of the wave, or -1
  if (a.ranges != nullptr) {
    int32_t *const shared = reinterpret_cast<int32_t *>(lds);
    const bool counts = there && row.document >= 0;
    const int32_t least = WaveReduce(counts ? row.document : INT32_MAX, [](int32_t x, int32_t y) { return min(x, y); });
    const int32_t most = WaveReduce(counts ? row.document : -1, [](int32_t x, int32_t y) { return max(x, y); });
    if (least == most && __all(counts || !there)) wave_document = least;
    if (lane == 0) shared[wave] = least, shared[4 + wave] = most;
    __syncthreads();
    tiles.least = min(min(shared[0], shared[1]), min(shared[2], shared[3]));
    tiles.most = max(max(shared[4], shared[5]), max(shared[6], shared[7]));
    __syncthreads();
  }
  if (tiles.most >= 0) {
    tiles.Start(a, b);
  } else {
    tiles.base = tiles.end, tiles.mask = 0, tiles.own_document = -1;
  }

  // a thread's groups of eight values: key and column group, the same of every tile
  const T *const k_head = static_cast<const T *>(a.k.base) + b * a.k.strides[0] + kv * a.k.strides[1];
  const T *const v_head = static_cast<const T *>(a.v.base) + b * a.v.strides[0] + kv * a.v.strides[1];
  const int last_group = (a.columns - 1) / 8;
  floatx4 staged[kParted ? 2 : 1][kParted ? Shape::kLoads : 1][2];
  uint32_t offset[kParted ? 1 : 2][kParted ? 1 : Shape::kLoads];  // bytes from a tile's first key, where that fits
  const bool near = max(a.k.strides[2], a.v.strides[2]) < (1 << 23);
  if constexpr (!kParted) {
#pragma unroll
    for (int m = 0; m < 2; ++m) {
#pragma unroll
      for (int n = 0; n < Shape::kLoads; ++n) {
        const int place = (wave * Shape::kLoads + n) * kWave + lane, key = place / (DP / 8);
        const int group = place % (DP / 8) ^ (m == 0 ? Shape::TurnK(key) : Shape::TurnV(key));
        offset[m][n] = static_cast<uint32_t>(key) * static_cast<uint32_t>(m == 0 ? a.k.strides[2] : a.v.strides[2]) * 2 + min(group, last_group) * 16;
      }
    }
  }
  auto fetch = [&](int32_t t, int buffer) __attribute__((always_inline)) {
    if constexpr (!kParted) {
      if (near && t * BK + BK <= seq.n_keys) {
#pragma unroll
        for (int m = 0; m < 2; ++m) {
          const char *const from = reinterpret_cast<const char *>((m == 0 ? k_head : v_head) + static_cast<int64_t>(t * BK) * (m == 0 ? a.k.strides[2] : a.v.strides[2]));
#pragma unroll
          for (int n = 0; n < Shape::kLoads; ++n) {
            const int32_t to = ((buffer * 2 + m) * Shape::kGroups + (wave * Shape::kLoads + n) * kWave) * 8;
            LoadToLds(from + offset[m][n], lds + to);
          }
        }
        return;
      }
    }
#pragma unroll
    for (int m = 0; m < 2; ++m) {
      const T *const from = m == 0 ? k_head : v_head;
      const int64_t stride = m == 0 ? a.k.strides[2] : a.v.strides[2];
#pragma unroll
      for (int n = 0; n < Shape::kLoads; ++n) {
        const int place = (wave * Shape::kLoads + n) * kWave + lane, key = place / (DP / 8);
        const int group = place % (DP / 8) ^ (m == 0 ? Shape::TurnK(key) : Shape::TurnV(key));
        // (columns behind the last and keys behind the last are read as the last: Q is zero there, and the weight of such a key)
        const T *const at = from + min(t * BK + key, seq.n_keys - 1) * stride + min(group, last_group) * 8;
        if constexpr (kParted) {
          staged[m][n][0] = *reinterpret_cast<const floatx4 *>(at);
          staged[m][n][1] = *reinterpret_cast<const floatx4 *>(at + (min(group, last_group) * 8 + 4 < a.columns ? 4 : 0));
        } else {
          const int32_t to = ((buffer * 2 + m) * Shape::kGroups + (wave * Shape::kLoads + n) * kWave) * 8;
          LoadToLds(at, lds + to);
        }
      }
    }
  };
  auto store = [&]() __attribute__((always_inline)) {
    if constexpr (kParted) {
#pragma unroll
      for (int m = 0; m < 2; ++m) {
#pragma unroll
        for (int n = 0; n < Shape::kLoads; ++n) {
          const int place = (wave * Shape::kLoads + n) * kWave + lane;
          float x[8];
#pragma unroll
          for (int e = 0; e < 8; ++e) x[e] = staged[m][n][e / 4][e % 4];
          u32x4 part[3];
          SplitParts<3>(x, part);
#pragma unroll
          for (int p = 0; p < 3; ++p) *reinterpret_cast<u32x4 *>(lds + (m * 3 + p) * Shape::kPlane + place * 8) = part[p];
        }
      }
    }
  };

  floatx16 acc[kColumns];
#pragma unroll
  for (int c = 0; c < kColumns; ++c) {
#pragma unroll
    for (int e = 0; e < 16; ++e) acc[c][e] = 0.0f;
  }
  float most = -INFINITY, sum = 0.0f;

  const int k_row = lane % 32 * DP;                                            // K: key lane % 32 ..
  const int v_key = 4 * half + lane % 16 / 4;                                  // V: key ..
  const int v_group = lane / 16 % 2 * 2 + lane % 4 / 2, v_swizzle = Shape::TurnV(lane % 16 / 4);

  int32_t now_document = -1, next_document = -1, now = tiles.Next(a, b, now_document);
  int buffer = 0;
  if (now >= 0) fetch(now, 0);
  while (now >= 0) {
    const int32_t next = tiles.Next(a, b, next_document);
    if constexpr (kParted) {
      __syncthreads();  // everyone is done with the tile before
      store();
      if (next >= 0) fetch(next, 0);
      __syncthreads();
    } else {
      asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
      __builtin_amdgcn_s_barrier();  // this tile has landed for all, and everyone is done with the other buffer
      asm volatile("" ::: "memory");
      if (next >= 0) fetch(next, buffer ^ 1);
    }
    const int32_t j0 = now * BK;
    const bool some = wave_there && ((j0 < some_hi && j0 + BK > some_lo) || j0 < seq.prefix);
    if (some) {
      const uint16_t *const k_tile = lds + buffer * 2 * kParts * Shape::kPlane, *const v_tile = k_tile + kParts * Shape::kPlane;
      float s[kKeyTiles * 16];
      floatx16 dots[kKeyTiles], lows[kParted ? kKeyTiles : 1];
#pragma unroll
      for (int t = 0; t < kKeyTiles; ++t) {
#pragma unroll
        for (int e = 0; e < 16; ++e) dots[t][e] = 0.0f, lows[kParted ? t : 0][e] = 0.0f;
      }
      // (neighbouring products go to different sums: one that waits for the one before it leaves the matrix pipe idle)
#pragma unroll
      for (int st = 0; st < kSteps; ++st) {
        u32x4 k[kKeyTiles][kParts];
#pragma unroll
        for (int t = 0; t < kKeyTiles; ++t) {
          const int at = t * 32 * DP + k_row + ((2 * st + half) ^ Shape::TurnK(lane % 32)) * 8;
#pragma unroll
          for (int p = 0; p < kParts; ++p) k[t][p] = *reinterpret_cast<const u32x4 *>(k_tile + p * Shape::kPlane + at);
        }
        if constexpr (kParted) {
          ForParts([&](auto i, auto j, auto small) __attribute__((always_inline)) {
#pragma unroll
            for (int t = 0; t < kKeyTiles; ++t) {
              floatx16 &to = small ? lows[t] : dots[t];
              to = Mfma32<E>(k[t][i], q[st][j], to);
            }
          });
        } else {
#pragma unroll
          for (int t = 0; t < kKeyTiles; ++t) dots[t] = Mfma32<E>(k[t][0], q[st][0], dots[t]);
        }
      }
      if constexpr (kAhead) ReadAhead<4, 1, kKeyTiles * kSteps>();
      Settle(dots);
      if constexpr (kParted) Settle(lows);
#pragma unroll
      for (int e = 0; e < kKeyTiles * 16; ++e) s[e] = kParted ? dots[e / 16][e % 16] + lows[kParted ? e / 16 : 0][e % 16] : dots[e / 16][e % 16];
      const bool whole = (j0 >= all_lo && j0 + BK <= all_hi) || j0 + BK <= seq.prefix;
      const bool one_document = a.ranges == nullptr || (now_document >= 0 && now_document == wave_document);
      const int32_t j_lane = j0 + 4 * half, ids = one_document ? 0 : KeyDocument(a, b, min(j0 + lane, a.keys - 1));
      const float by = Finish<kParted>(a, row, seq.prefix > 0, whole, one_document, s, [&](int e) { return j_lane + e / 16 * 32 + e % 16 / 4 * 8 + e % 4; },
                                       [&](int e) {
                                         const int from = e / 16 * 32 + e % 16 / 4 * 8 + e % 4;
                                         const int32_t lower = __builtin_amdgcn_readlane(ids, from), upper = __builtin_amdgcn_readlane(ids, from + 4);
                                         return half == 0 ? lower : upper;
                                       });
      float top = s[0];
#pragma unroll
      for (int e = 1; e < kKeyTiles * 16; ++e) top = fmaxf(top, s[e]);
      top = AcrossHalves(top, MaxOp{}) * by;
      if (__any(top > most + kLazy)) {
        const float higher = fmaxf(most, top), from = higher == -INFINITY ? 0.0f : higher;
        const float kept = __builtin_amdgcn_exp2f(most - from);
        most = higher;
        sum *= kept;
#pragma unroll
        for (int c = 0; c < kColumns; ++c) {
#pragma unroll
          for (int e = 0; e < 16; ++e) acc[c][e] *= kept;
        }
      }
      const float from = most == -INFINITY ? 0.0f : most;
      float part_sum = 0.0f;
#pragma unroll
      for (int e = 0; e < kKeyTiles * 16; ++e) {
        s[e] = __builtin_amdgcn_exp2f(fmaf(s[e], by, -from));
        part_sum += s[e];
      }
      sum += part_sum;
      u32x4 weights[kKeyTiles * 2][kParts];
#pragma unroll
      for (int n = 0; n < kKeyTiles * 2; ++n) {
        if constexpr (kParted) {
          float x[8];
#pragma unroll
          for (int e = 0; e < 8; ++e) x[e] = s[n * 8 + e];
          SplitParts<3>(x, weights[n]);
        } else {
          weights[n][0] = Pack8<E>(s + n * 8);
        }
      }
      auto read_v = [&](int n, int c, int p) __attribute__((always_inline)) {
        const int at = (n * 16 + v_key) * DP + ((c * 4 + v_group) ^ v_swizzle) * 8 + lane % 2 * 4;
        uint16_t *const from16 = const_cast<uint16_t *>(v_tile) + p * Shape::kPlane + at;
        typedef __attribute__((address_space(3))) shortx4 *Lds;
        const uint64_t first = __builtin_bit_cast(uint64_t, __builtin_amdgcn_ds_read_tr16_b64_v4i16((Lds)(from16)));
        const uint64_t second = __builtin_bit_cast(uint64_t, __builtin_amdgcn_ds_read_tr16_b64_v4i16((Lds)(from16 + 8 * DP)));
        return u32x4{static_cast<uint32_t>(first), static_cast<uint32_t>(first >> 32), static_cast<uint32_t>(second), static_cast<uint32_t>(second >> 32)};
      };
      if constexpr (kParted) {
#pragma unroll
        for (int c0 = 0; c0 < kColumns; c0 += 2) {  // two at a time
          floatx16 low[2];
#pragma unroll
          for (int e = 0; e < 16; ++e) low[0][e] = 0.0f, low[1][e] = 0.0f;
#pragma unroll
          for (int n = 0; n < kKeyTiles * 2; ++n) {
            u32x4 v[2][kParts];
#pragma unroll
            for (int c = 0; c < 2; ++c) {
#pragma unroll
              for (int p = 0; p < kParts; ++p) v[c][p] = read_v(n, c0 + c, p);
            }
            ForParts([&](auto i, auto j, auto small) __attribute__((always_inline)) {
#pragma unroll
              for (int c = 0; c < 2; ++c) {
                floatx16 &to = small ? low[c] : acc[c0 + c];
                to = Mfma32<E>(v[c][i], weights[n][j], to);
              }
            });
          }
#pragma unroll
          for (int e = 0; e < 16; ++e) acc[c0][e] += low[0][e], acc[c0 + 1][e] += low[1][e];
        }
      } else {
#pragma unroll
        for (int n = 0; n < kKeyTiles * 2; ++n) {
#pragma unroll
          for (int c = 0; c < kColumns; ++c) acc[c] = Mfma32<E>(read_v(n, c, 0), weights[n][0], acc[c]);
        }
      }
      if constexpr (kAhead) ReadAhead<4, 2, kColumns * kKeyTiles * 2>();
    }
    now = next, now_document = next_document;
    if constexpr (!kParted) buffer ^= 1;
  }

  SettleAcrossBranch();
  Settle(acc);
  sum = AcrossHalves(sum, SumOp{});
  const float inverse = sum == 0.0f ? 0.0f : 1.0f / sum;
  bool bad = !(sum < INFINITY);
#pragma unroll
  for (int c = 0; c < kColumns; ++c) {
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      acc[c][e] = sum == 0.0f ? 0.0f : acc[c][e] * inverse;
      bad = bad || (c * 32 + e / 4 * 8 + 4 * half + e % 4 < a.columns && !(fabsf(acc[c][e]) < INFINITY));
    }
  }
  const uint64_t which = __ballot(bad && there);
  uint32_t careful = static_cast<uint32_t>(which) | static_cast<uint32_t>(which >> 32);
  if (there && !(careful >> (lane % 32) & 1)) {
    T *const to = static_cast<T *>(a.out.base) + b * a.out.strides[0] + row.head * a.out.strides[1] + row.i * a.out.strides[2];
#pragma unroll
    for (int c = 0; c < kColumns; ++c) {
#pragma unroll
      for (int e = 0; e < 16; e += 4) {
        const int d = c * 32 + e / 4 * 8 + 4 * half;
        if (d >= a.columns) continue;
        typedef T Vec __attribute__((ext_vector_type(4)));
        if (a.out_aligned) {
          Vec v;
#pragma unroll
          for (int n = 0; n < 4; ++n) v[n] = static_cast<T>(acc[c][e + n]);
          *reinterpret_cast<Vec *>(to + d) = v;
        } else {
#pragma unroll
          for (int n = 0; n < 4; ++n) {
            if (d + n < a.columns) to[(d + n) * a.out.strides[3]] = static_cast<T>(acc[c][e + n]);
          }
        }
      }
    }
  }
  for (; careful != 0; careful &= careful - 1) CarefulRow<T>(a, b, kv, wave_row + __builtin_ctz(careful));
}

// Writes one row by one wave: lane l has the sums of columns l, l + 64, ..
template <typename T>
__device__ __forceinline__ void StoreRow(const AttentionArgs &a, int b, int kv, int32_t r, const float (&sums)[FL_ATTENTION_MAX_HEAD / kWave], float sum) {
  const int lane = threadIdx.x % kWave;
  const float inverse = sum == 0.0f ? 0.0f : 1.0f / sum;
  float x[FL_ATTENTION_MAX_HEAD / kWave];
  bool bad = !(sum < INFINITY);
#pragma unroll
  for (int c = 0; c < FL_ATTENTION_MAX_HEAD / kWave; ++c) {
    x[c] = sum == 0.0f ? 0.0f : sums[c] * inverse;
    bad = bad || (c * kWave + lane < a.columns && !(fabsf(x[c]) < INFINITY));
  }
  if (__any(bad)) return CarefulRow<T>(a, b, kv, r);
  const int32_t i = static_cast<int32_t>(a.group_div.Div(static_cast<uint32_t>(r)));
  T *const to = static_cast<T *>(a.out.base) + b * a.out.strides[0] + (kv * a.group + (r - i * a.group)) * a.out.strides[1] + i * a.out.strides[2];
#pragma unroll
  for (int c = 0; c < FL_ATTENTION_MAX_HEAD / kWave; ++c) {
    const int d = c * kWave + lane;
    if (d < a.columns) to[d * a.out.strides[3]] = static_cast<T>(x[c]);
  }
}

// --------------------------------------------------------------------------------------------------------------------
// Few rows (a step of decoding: `group` rows a token).  Bound by the bytes of K and V, so what counts is how many are on their way: a workgroup
// has 16 rows and its waves, and those of the other workgroups of the same rows (`splits`), take the tiles of keys in turn, each tile straight
// into registers, K's while V's of the tile before are multiplied and the other way round.  No LDS until the waves' sums are joined.
// Transposed as above, with 16 x 16 instructions.  A lane's scores are those of row lane % 16 with keys 4 (lane / 16) + e (and 16 more),
// and it loads the same keys of V, DP / 16 columns each, for which it then has a small square to turn around: two registers make two.
// fp32 stays fp32 (v_mfma_f32_16x16x4_f32): at sixteen rows its products cost less than the bytes.
// 8 sequences of 8 key heads of 128 columns in bf16, 8192 keys, one token: 53 us for 268 MB, 5.1 TB/s, and 5 us to join the splits.
template <typename T, int DP>
struct FewShape {
  static constexpr bool kWide = std::is_same_v<T, float>;
  static constexpr int kKeys = kWide ? 16 : 32;          // of a tile
  static constexpr int kGroup = 16 / sizeof(T);          // values of a 16-byte load
  static constexpr int kSteps = DP / (4 * kGroup);       // loads of a row of K by the four lanes that share it
  static constexpr int kKeyTiles = kKeys / 16;
  static constexpr int kColumns = DP / 16;               // a lane's of V
  static constexpr int kOwn = kKeys / 4;                 // a lane's keys of V
  static constexpr int kRaw = kColumns * sizeof(T) / 4;  // registers of a key's columns
};

template <typename T, int DP, bool ALIGNED>
__global__ __launch_bounds__(256, DP == 256 ? 1 : 2) void AttentionFewKernel(const AttentionArgs a) {
  using Shape = FewShape<T, DP>;
  constexpr bool kWide = Shape::kWide;
  constexpr int kKeys = Shape::kKeys, kSteps = Shape::kSteps, kKeyTiles = Shape::kKeyTiles, kColumns = Shape::kColumns, kOwn = Shape::kOwn, kGroup = Shape::kGroup;
  typedef T Group __attribute__((ext_vector_type(kGroup)));
  __shared__ float joined[4][16][DP];
  __shared__ float2 joined_stats[4][16];
  const int lane = threadIdx.x % kWave, own = lane % 16, quarter = lane / 16, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  uint32_t at = blockIdx.x / a.splits;
  const int split = static_cast<int>(blockIdx.x - at * a.splits);
  const uint32_t head = a.tiles_div.Div(at);
  const int32_t row0 = static_cast<int32_t>(at - head * a.tiles_div.divisor) * 16;
  const int b = static_cast<int>(a.kv_div.Div(head)), kv = static_cast<int>(head) - b * a.kv_heads;
  const Sequence seq = SequenceOf(a, b);
  const int32_t first_query = static_cast<int32_t>(a.group_div.Div(row0));
  if (first_query >= seq.n_queries) return;
  const int32_t last_query = min(static_cast<int32_t>(a.group_div.Div(min(row0 + 15, a.rows - 1))), seq.n_queries - 1);
  const Row row = RowOf(a, seq, b, kv, row0 + own);
  const bool there = row.there && row0 + own < a.rows;
  const int32_t all_lo = FirstKey(a, seq, last_query), all_hi = LastKey(a, seq, first_query);

  Group q[kSteps];
  {
    const T *const from = static_cast<const T *>(a.q.base) + b * a.q.strides[0] + row.head * a.q.strides[1] + row.i * a.q.strides[2];
#pragma unroll
    for (int s = 0; s < kSteps; ++s) {
      float x[8] = {};
      const int d = (s * 4 + quarter) * kGroup;
      if (a.q_aligned) {  // (no branch around a load: what is not there is read elsewhere in q and made zero)
        const Group g = *reinterpret_cast<const Group *>((there ? from : static_cast<const T *>(a.q.base)) + min(d, a.columns - kGroup));
#pragma unroll
        for (int e = 0; e < kGroup; ++e) x[e] = there && d < a.columns ? static_cast<float>(g[e]) : 0.0f;
      } else if (there) {
        Load8(from, a.q.strides[3], d, min(a.columns, d + kGroup), x);
      }
#pragma unroll
      for (int e = 0; e < kGroup; ++e) q[s][e] = static_cast<T>(x[e] * a.sign);
    }
  }

  Tiles<kKeys> tiles;
  tiles.lo = FirstKey(a, seq, first_query);
  tiles.hi = LastKey(a, seq, last_query);
  tiles.prefix = seq.prefix;
  // (from the first tile that may be seen on, so that the tiles spread evenly over the waves whatever the mask)
  const int32_t front = seq.prefix > 0 ? 0 : min(tiles.lo, seq.n_keys) / kKeys;
  tiles.first = front + split * 4 + wave, tiles.step = a.splits * 4, tiles.end = (seq.n_keys + kKeys - 1) / kKeys;
  tiles.least = 0, tiles.most = INT32_MAX;
  int32_t row_document = -1;
  if (a.ranges != nullptr) {
    const bool counts = there && row.document >= 0;
    tiles.least = WaveReduce(counts ? row.document : INT32_MAX, [](int32_t x, int32_t y) { return min(x, y); });
    tiles.most = WaveReduce(counts ? row.document : -1, [](int32_t x, int32_t y) { return max(x, y); });
    if (tiles.least == tiles.most && __all(counts || !there)) row_document = tiles.least;
  }
  if (tiles.most >= 0) {
    tiles.Start(a, b);
  } else {
    tiles.base = tiles.end, tiles.mask = 0, tiles.own_document = -1;
  }

  const T *const k_head = static_cast<const T *>(a.k.base) + b * a.k.strides[0] + kv * a.k.strides[1];
  const T *const v_head = static_cast<const T *>(a.v.base) + b * a.v.strides[0] + kv * a.v.strides[1];
  Group k[kKeyTiles][kSteps];
  uint32_t v[kOwn][Shape::kRaw];
  auto load_k = [&](int32_t tile) __attribute__((always_inline)) {
#pragma unroll
    for (int t = 0; t < kKeyTiles; ++t) {
      const T *const from = k_head + min(tile * kKeys + t * 16 + own, seq.n_keys - 1) * a.k.strides[2];
#pragma unroll
      for (int s = 0; s < kSteps; ++s) {
        const int d = (s * 4 + quarter) * kGroup;
        if constexpr (ALIGNED) {  // (columns behind the last: the last ones again, where Q is zero)
          k[t][s] = *reinterpret_cast<const Group *>(from + min(d, a.columns - kGroup));
        } else {
          float x[8];
          Load8(from, a.k.strides[3], d, min(a.columns, d + kGroup), x);
#pragma unroll
          for (int e = 0; e < kGroup; ++e) k[t][s][e] = static_cast<T>(x[e]);
        }
      }
    }
  };
  auto load_v = [&](int32_t tile) __attribute__((always_inline)) {
#pragma unroll
    for (int n = 0; n < kOwn; ++n) {
      const int32_t j = tile * kKeys + n / 4 * 16 + quarter * 4 + n % 4;
      const T *const from = v_head + min(j, seq.n_keys - 1) * a.v.strides[2];
      if constexpr (ALIGNED) {
        constexpr int kRun = kColumns < kGroup ? kColumns : kGroup;  // values of a load
        typedef uint32_t Run __attribute__((ext_vector_type(kRun * sizeof(T) / 4)));
#pragma unroll
        for (int g = 0; g < kColumns / kRun; ++g) {
          const Run x = *reinterpret_cast<const Run *>(from + min(own * kColumns + g * kRun, a.columns - kRun));
#pragma unroll
          for (int e = 0; e < kRun * static_cast<int>(sizeof(T)) / 4; ++e) v[n][g * (kRun * sizeof(T) / 4) + e] = x[e];
        }
      } else {
#pragma unroll
        for (int e = 0; e < kColumns; e += 4 / sizeof(T)) {
          T x[4 / sizeof(T)];
#pragma unroll
          for (int m = 0; m < static_cast<int>(4 / sizeof(T)); ++m) {
            const int d = own * kColumns + e + m;
            x[m] = d < a.columns ? from[d * a.v.strides[3]] : static_cast<T>(0.0f);
          }
          v[n][e * sizeof(T) / 4] = __builtin_bit_cast(uint32_t, x);
        }
      }
    }
  };

  floatx4 acc[kColumns];
#pragma unroll
  for (int c = 0; c < kColumns; ++c) acc[c] = floatx4{0.0f, 0.0f, 0.0f, 0.0f};
  float most = -INFINITY, sum = 0.0f;
  auto work = [&](int32_t tile, int32_t document, int32_t next, auto more) __attribute__((always_inline)) {
    const int32_t j0 = tile * kKeys;
    float s[kOwn];
    floatx4 dots[kKeyTiles];
#pragma unroll
    for (int t = 0; t < kKeyTiles; ++t) {
      floatx4 &dot = dots[t];
      dot = floatx4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int st = 0; st < kSteps; ++st) {
        if constexpr (kWide) {
#pragma unroll
          for (int e = 0; e < 4; ++e) dot = __builtin_amdgcn_mfma_f32_16x16x4f32(k[t][st][e], q[st][e], dot, 0, 0, 0);
        } else if constexpr (std::is_same_v<T, _Float16>) {
          dot = __builtin_amdgcn_mfma_f32_16x16x32_f16(k[t][st], q[st], dot, 0, 0, 0);
        } else {
          dot = __builtin_amdgcn_mfma_f32_16x16x32_bf16(k[t][st], q[st], dot, 0, 0, 0);
        }
      }
    }
    Settle(dots);
#pragma unroll
    for (int e = 0; e < kOwn; ++e) s[e] = dots[e / 4][e % 4];
    if constexpr (decltype(more)::value) load_k(next);
    const bool whole = (j0 >= all_lo && j0 + kKeys <= all_hi) || j0 + kKeys <= seq.prefix;
    const bool one_document = a.ranges == nullptr || (document >= 0 && document == row_document);
    const int32_t j_lane = j0 + 4 * quarter, ids = one_document ? 0 : KeyDocument(a, b, min(j0 + lane % kKeys, a.keys - 1));
    const float by = Finish<kWide>(a, row, seq.prefix > 0, whole, one_document, s, [&](int e) { return j_lane + e / 4 * 16 + e % 4; },
                                   [&](int e) { return __shfl(ids, e / 4 * 16 + 4 * quarter + e % 4); });
    float top = s[0];
#pragma unroll
    for (int e = 1; e < kOwn; ++e) top = fmaxf(top, s[e]);
    top = AcrossRows(AcrossHalves(top, MaxOp{}), MaxOp{}) * by;
    if (__any(top > most + kLazy)) {
      const float higher = fmaxf(most, top), from = higher == -INFINITY ? 0.0f : higher;
      const float kept = __builtin_amdgcn_exp2f(most - from);
      most = higher;
      sum *= kept;
#pragma unroll
      for (int c = 0; c < kColumns; ++c) acc[c] *= kept;
    }
    const float from = most == -INFINITY ? 0.0f : most;
#pragma unroll
    for (int e = 0; e < kOwn; ++e) {
      s[e] = __builtin_amdgcn_exp2f(fmaf(s[e], by, -from));
      sum += s[e];
    }
    if constexpr (kWide) {
#pragma unroll
      for (int c = 0; c < kColumns; ++c) {
#pragma unroll
        for (int n = 0; n < kOwn; ++n) acc[c] = __builtin_amdgcn_mfma_f32_16x16x4f32(__builtin_bit_cast(float, v[n][c]), s[n], acc[c], 0, 0, 0);
      }
    } else {
      typedef T Vec __attribute__((ext_vector_type(8)));
      const Vec weights = __builtin_bit_cast(Vec, Pack8<T>(s));
#pragma unroll
      for (int c = 0; c < kColumns; ++c) {
        u32x4 turned;  // column c of the lane's eight keys
#pragma unroll
        for (int n = 0; n < 4; ++n) turned[n] = __builtin_amdgcn_perm(v[2 * n + 1][c / 2], v[2 * n][c / 2], c % 2 == 0 ? 0x05040100u : 0x07060302u);
        if constexpr (std::is_same_v<T, _Float16>) {
          acc[c] = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(Vec, turned), weights, acc[c], 0, 0, 0);
        } else {
          acc[c] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(Vec, turned), weights, acc[c], 0, 0, 0);
        }
      }
    }
    if constexpr (decltype(more)::value) load_v(next);
  };
  int32_t now_document = -1, next_document = -1, now = tiles.Next(a, b, now_document);
  if (now >= 0) {
    load_k(now);
    load_v(now);
    for (int32_t next; (next = tiles.Next(a, b, next_document)) >= 0; now = next, now_document = next_document) work(now, now_document, next, std::true_type{});
    work(now, now_document, -1, std::false_type{});
  }

  SettleAcrossBranch();
  Settle(acc);
  // the waves' sums, each as far behind the common maximum as its own
  sum = AcrossRows(AcrossHalves(sum, SumOp{}), SumOp{});
#pragma unroll
  for (int c = 0; c < kColumns; ++c) {
#pragma unroll
    for (int e = 0; e < 4; ++e) joined[wave][own][(4 * quarter + e) * kColumns + c] = acc[c][e];
  }
  if (quarter == 0) joined_stats[wave][own] = make_float2(most, sum);
  __syncthreads();
  const int64_t all_rows = static_cast<int64_t>(a.batch) * a.kv_heads * a.rows;
  for (int n = 0; n < 4; ++n) {
    const int32_t at_row = wave * 4 + n, r = row0 + at_row;
    if (r >= a.rows || static_cast<int32_t>(a.group_div.Div(r)) >= seq.n_queries) break;
    float2 stats[4];
    float higher = -INFINITY, total = 0.0f, x[FL_ATTENTION_MAX_HEAD / kWave] = {};
#pragma unroll
    for (int w = 0; w < 4; ++w) stats[w] = joined_stats[w][at_row], higher = fmaxf(higher, stats[w].x);
    const float from = higher == -INFINITY ? 0.0f : higher;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      const float kept = __builtin_amdgcn_exp2f(stats[w].x - from);
      total += stats[w].y * kept;
#pragma unroll
      for (int c = 0; c < (DP + kWave - 1) / kWave; ++c) {
        if (c * kWave + lane < DP) x[c] += joined[w][at_row][c * kWave + lane] * kept;
      }
    }
    if (a.splits == 1) {
      StoreRow<T>(a, b, kv, r, x, total);
    } else {
      const int64_t place = split * all_rows + static_cast<int64_t>(head) * a.rows + r;
      if (lane == 0) a.stats[place] = make_float2(higher, total);
#pragma unroll
      for (int c = 0; c < (DP + kWave - 1) / kWave; ++c) {
        if (c * kWave + lane < a.columns) a.partial[place * a.columns + c * kWave + lane] = x[c];
      }
    }
  }
}

// Joins the splits, a wave a row, in their order.  What counts is how many loads are on their way: those of kRun splits at a time (32 rows of 128
// columns in 64 splits: one at a time 23.5 us, sixteen 5.1).
template <typename T, int DP>
__global__ __launch_bounds__(256) void AttentionJoinKernel(const AttentionArgs a) {
  constexpr int kColumns = DP / kWave, kRun = 16;
  const int lane = threadIdx.x % kWave;
  const int64_t all_rows = static_cast<int64_t>(a.batch) * a.kv_heads * a.rows;
  const int64_t at = static_cast<int64_t>(blockIdx.x) * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  if (at >= all_rows) return;
  const uint32_t head = static_cast<uint32_t>(at / a.rows);
  const int32_t r = static_cast<int32_t>(at - static_cast<int64_t>(head) * a.rows);
  const int b = static_cast<int>(a.kv_div.Div(head)), kv = static_cast<int>(head) - b * a.kv_heads;
  if (static_cast<int32_t>(a.group_div.Div(r)) >= SequenceOf(a, b).n_queries) return;
  // (at most 64 splits: a lane reads the figures of one)
  const float2 own = lane < a.splits ? a.stats[lane * all_rows + at] : make_float2(-INFINITY, 0.0f);
  const float higher = WaveReduce(own.x, MaxOp{});
  const float kept = __builtin_amdgcn_exp2f(own.x - (higher == -INFINITY ? 0.0f : higher));
  const float total = GroupSum<64>(own.y * kept);
  float x[FL_ATTENTION_MAX_HEAD / kWave] = {};
  for (int s0 = 0; s0 < a.splits; s0 += kRun) {
    float part[kRun][kColumns];
#pragma unroll
    for (int n = 0; n < kRun; ++n) {  // (no branch around a load: splits and columns that are not there are the last ones again)
      const float *const from = a.partial + (min(s0 + n, a.splits - 1) * all_rows + at) * a.columns;
#pragma unroll
      for (int c = 0; c < kColumns; ++c) part[n][c] = from[min(c * kWave + lane, a.columns - 1)];
    }
#pragma unroll
    for (int n = 0; n < kRun; ++n) {
      const float by = __shfl(kept, min(s0 + n, a.splits - 1));
#pragma unroll
      for (int c = 0; c < kColumns; ++c) x[c] = s0 + n < a.splits ? x[c] + part[n][c] * by : x[c];
    }
  }
  StoreRow<T>(a, b, kv, r, x, total);
}

constexpr int64_t kPartialBytes = 16 << 20;  // of the splits' sums
constexpr int64_t kSplitWorkgroups = 768;

int CheckLengths(const fl_tensor *t, int64_t batch) { return CheckOptionalVector(t, FL_INT32, batch); }

int CheckDocuments(const fl_tensor *t, int64_t batch, int64_t length) {
  FL_CHECK(CheckWideView(t));
  if (t->rank != 2) return FL_ERR_RANK;
  if (t->dtype != FL_INT32) return FL_ERR_DTYPE;
  return t->shape[0] == batch && t->shape[1] == length ? FL_OK : FL_ERR_SHAPE;
}

int CheckScores(const fl_tensor *q, const fl_tensor *k, const fl_attention_scores *s) {
  FL_CHECK(CheckWideView(q));
  FL_CHECK(CheckWideView(k));
  if (q->rank != 4 || k->rank != 4) return FL_ERR_RANK;
  if (!IsDecoderType(q->dtype) || k->dtype != q->dtype) return FL_ERR_DTYPE;
  if (k->shape[0] != q->shape[0] || k->shape[3] != q->shape[3] || q->shape[1] % k->shape[1] != 0) return FL_ERR_SHAPE;
  if (q->shape[3] > FL_ATTENTION_MAX_HEAD) return FL_ERR_UNSUPPORTED;
  if (s == nullptr) return FL_ERR_NULL;
  const int64_t B = q->shape[0];
  // (what the kernels multiply by is finite: both by log2(e), and their quotient by twice that)
  if (!(1.45 * std::fabs(s->scale) < 3e38) || !(2.9 * s->cap < 3e38) || s->cap < 0.0) return FL_ERR_ATTR;
  if (s->cap > 0.0 && !(2.9 * std::fabs(s->scale) / s->cap < 3e38)) return FL_ERR_ATTR;
  if ((s->causal != 0 && s->causal != 1) || s->window < 0) return FL_ERR_ATTR;
  // what a grid of workgroups counts: tiles of rows of all key heads, sequences
  const __int128 tiles = (q->shape[2] * (q->shape[1] / k->shape[1]) + 15) / 16;
  if (tiles * q->shape[0] * k->shape[1] > kMostWorkgroups - kSplitWorkgroups || q->shape[0] > 65535) return FL_ERR_TOO_LARGE;
  FL_CHECK(CheckOptionalVector(s->slopes, FL_FLOAT32, q->shape[1]));
  FL_CHECK(CheckLengths(s->prefix_lengths, B));
  FL_CHECK(CheckLengths(s->query_starts, B));
  FL_CHECK(CheckLengths(s->query_lengths, B));
  FL_CHECK(CheckLengths(s->key_lengths, B));
  if ((s->query_documents == nullptr) != (s->key_documents == nullptr)) return FL_ERR_NULL;
  if (s->query_documents != nullptr) {
    FL_CHECK(CheckDocuments(s->query_documents, B, q->shape[2]));
    FL_CHECK(CheckDocuments(s->key_documents, B, k->shape[2]));
  }
  return FL_OK;
}

AttentionView View(const fl_tensor *t) { return {t->base, {t->strides[0], t->strides[1], t->strides[2], t->strides[3]}}; }

const int32_t *Lengths(const fl_tensor *t, int64_t *stride) {
  *stride = t == nullptr ? 0 : t->strides[0];
  return t == nullptr ? nullptr : static_cast<const int32_t *>(t->base);
}

const int32_t *Documents(const fl_tensor *t, int64_t (&strides)[2]) {
  for (int i = 0; i < 2; ++i) strides[i] = t == nullptr ? 0 : t->strides[i];
  return t == nullptr ? nullptr : static_cast<const int32_t *>(t->base);
}

// How a call runs.
struct Plan {
  bool many;       // AttentionRowsKernel, else AttentionFewKernel
  int32_t splits;  // workgroups that share the keys of a tile of rows
  size_t ranges_at, partial_at, stats_at, bytes;
};

bool Aligned(const fl_tensor *t) {
  const size_t item = t->dtype == FL_FLOAT32 ? 4 : 2;
  const int64_t group = static_cast<int64_t>(16 / item);
  if (!IsAligned(t->base, 16) || t->shape[3] % group != 0 || (t->strides[3] != 1 && t->shape[3] > 1)) return false;
  for (int i = 0; i < 3; ++i) {
    if (t->shape[i] > 1 && t->strides[i] % group != 0) return false;
  }
  return true;
}

// (of K and V only the extents and K's alignment are known here; `aligned`: that of both)
Plan MakePlan(const fl_tensor *q, const fl_tensor *k, const fl_attention_scores *s, bool aligned) {
  const int64_t B = q->shape[0], KV = k->shape[1], Skv = k->shape[2], D = q->shape[3], rows = q->shape[2] * (q->shape[1] / KV);
  Plan p{};
  // Tiles of 128 rows where there are enough of them to fill the chip, else of 16 whose keys are split.  32 heads of 128 columns in bf16, 4096 keys:
  // 96 tiles of 128 rows 112 us (split tiles of 16: 145), 64 tiles 111 (111), 32 tiles 110 (72); in fp32, 64 columns, 128 tiles 36 (52), 48 tiles
  // 217 (102).  Up to 32 rows of a key head most of 128 would be empty: 115 us where tiles of 128 take 264.
  p.many = aligned && rows > 32 && B * KV * ((rows + 127) / 128) >= 96;
  p.splits = 1;
  if (!p.many) {
    const int64_t tiles = B * KV * ((rows + 15) / 16);
    int64_t reach = Skv;
    if (s->window > 0 && s->prefix_lengths == nullptr) reach = std::min(reach, std::min(s->window, Skv) * (s->causal ? 1 : 2) + 16);
    const int64_t keys = q->dtype == FL_FLOAT32 ? 16 : 32;
    // three workgroups for each compute unit, each wave with two tiles of keys or more: 8 sequences of 8 key heads, 8192 keys, 12 splits 53.0 us and
    // 5.1 to join them, 24 splits 52.8 and 5.8, 48 splits 58 and more; 16 heads of fp32, 128 queries, 39 and 4.8 with 6 splits, 44 and 4.7 with 12
    int64_t splits = std::min<int64_t>((kSplitWorkgroups + tiles - 1) / tiles, reach / (4 * 2 * keys));
    splits = std::min(splits, kPartialBytes / (B * KV * rows * (D + 2) * 4));
    p.splits = static_cast<int32_t>(std::max<int64_t>(1, std::min<int64_t>(splits, 64)));
  }
  auto place = [&](size_t bytes) {
    const size_t at = p.bytes;
    p.bytes += (bytes + 15) / 16 * 16;
    return at;
  };
  if (s->key_documents != nullptr) p.ranges_at = place(static_cast<size_t>(B) * ((Skv + kBlock - 1) / kBlock) * sizeof(int2));
  if (p.splits > 1) {
    p.partial_at = place(static_cast<size_t>(p.splits) * B * KV * rows * D * sizeof(float));
    p.stats_at = place(static_cast<size_t>(p.splits) * B * KV * rows * sizeof(float2));
  }
  return p;
}

// Key tiles of 64, of 32 where the columns of 64 keys leave no registers for a second operand: 4096 queries and keys of 16 heads of 256 columns in
// bf16 take 537 us with 64 keys in a tile and 511 with 32, with a window of 1024 keys 283 and 247. The last argument is the waves of a SIMD that the
// registers are shared out for: what the tile of that width needs without spilling.
template <typename T>
int LaunchRows(const AttentionArgs &a, hipStream_t stream) {
  const dim3 grid(a.tiles_div.divisor * a.heads_div.divisor), block(256);
  if constexpr (std::is_same_v<T, float>) {
    if (a.columns <= 64) {
      FL_LAUNCH((AttentionRowsKernel<T, 64, 64, 1>), grid, block, 0, stream, a);
    } else if (a.columns <= 128) {
      FL_LAUNCH((AttentionRowsKernel<T, 128, 64, 1>), grid, block, 0, stream, a);
    } else {
      FL_LAUNCH((AttentionRowsKernel<T, 256, 32, 1>), grid, block, 0, stream, a);
    }
  } else {
    if (a.columns <= 64) {
      FL_LAUNCH((AttentionRowsKernel<T, 64, 64, 3>), grid, block, 0, stream, a);
    } else if (a.columns <= 96) {
      FL_LAUNCH((AttentionRowsKernel<T, 96, 64, 2>), grid, block, 0, stream, a);
    } else if (a.columns <= 128) {
      FL_LAUNCH((AttentionRowsKernel<T, 128, 64, 2>), grid, block, 0, stream, a);
    } else {
      FL_LAUNCH((AttentionRowsKernel<T, 256, 32, 1>), grid, block, 0, stream, a);
    }
  }
  return LaunchStatus();
}

template <typename T, int DP>
int LaunchFew(const AttentionArgs &a, bool aligned, hipStream_t stream) {
  const dim3 grid(a.tiles_div.divisor * a.heads_div.divisor * a.splits), block(256);
  if (aligned) {
    FL_LAUNCH((AttentionFewKernel<T, DP, true>), grid, block, 0, stream, a);
  } else {
    FL_LAUNCH((AttentionFewKernel<T, DP, false>), grid, block, 0, stream, a);
  }
  FL_CHECK(LaunchStatus());
  if (a.splits > 1) {
    const int64_t rows = static_cast<int64_t>(a.heads_div.divisor) * a.rows;
    FL_LAUNCH((AttentionJoinKernel<T, DP>), dim3(static_cast<uint32_t>((rows + 3) / 4)), block, 0, stream, a);
  }
  return LaunchStatus();
}

}  // namespace

extern "C" {

int fluidml_hip_attention_positions_scratch(const fl_tensor *q, const fl_tensor *k, const fl_attention_scores *scores, size_t *bytes) {
  if (bytes == nullptr) return FL_ERR_NULL;
  FL_CHECK(CheckScores(q, k, scores));
  // (V's alignment may make the call go either way)
  *bytes = std::max(MakePlan(q, k, scores, true).bytes, MakePlan(q, k, scores, false).bytes);
  return FL_OK;
}

int fluidml_hip_attention_positions(const fl_tensor *q, const fl_tensor *k, const fl_tensor *v, const fl_tensor *out, const fl_attention_scores *scores,
                                    void *scratch, size_t scratch_bytes, void *stream) {
  FL_CHECK(CheckScores(q, k, scores));
  FL_CHECK(CheckWideView(v));
  FL_CHECK(CheckWideResult(out));
  if (v->rank != 4 || out->rank != 4) return FL_ERR_RANK;
  if (v->dtype != q->dtype || out->dtype != q->dtype) return FL_ERR_DTYPE;
  if (!SameShape(k, v) || !SameShape(q, out)) return FL_ERR_SHAPE;
  const bool aligned = Aligned(k) && Aligned(v);
  const Plan plan = MakePlan(q, k, scores, aligned);
  if (plan.bytes > 0) {
    if (scratch == nullptr) return FL_ERR_NULL;
    if (plan.bytes > scratch_bytes || !IsAligned(scratch, 16)) return FL_ERR_SCRATCH;
  }
  AttentionArgs a;
  std::memset(&a, 0, sizeof(a));
  a.q = View(q), a.k = View(k), a.v = View(v), a.out = View(out);
  a.slopes = scores->slopes == nullptr ? nullptr : static_cast<const float *>(scores->slopes->base);
  a.slope_stride = scores->slopes == nullptr ? 0 : scores->slopes->strides[0];
  a.prefix_lengths = Lengths(scores->prefix_lengths, &a.prefix_stride);
  a.query_starts = Lengths(scores->query_starts, &a.query_start_stride);
  a.query_lengths = Lengths(scores->query_lengths, &a.query_length_stride);
  a.key_lengths = Lengths(scores->key_lengths, &a.key_length_stride);
  a.query_documents = Documents(scores->query_documents, a.query_document_strides);
  a.key_documents = Documents(scores->key_documents, a.key_document_strides);
  a.batch = static_cast<int32_t>(q->shape[0]);
  a.heads = static_cast<int32_t>(q->shape[1]);
  a.kv_heads = static_cast<int32_t>(k->shape[1]);
  a.group = a.heads / a.kv_heads;
  a.queries = static_cast<int32_t>(q->shape[2]);
  a.keys = static_cast<int32_t>(k->shape[2]);
  a.columns = static_cast<int32_t>(q->shape[3]);
  a.rows = a.queries * a.group;
  a.causal = scores->causal;
  a.window = std::min<int64_t>(scores->window, INT64_C(1) << 33);  // (no two positions are further apart)
  a.sign = scores->scale < 0.0 ? -1.0f : 1.0f;
  const double scale = std::fabs(scores->scale), log2e = 1.4426950408889634;
  a.scale2 = static_cast<float>(scale * log2e);
  a.cap = static_cast<float>(scores->cap);
  if (scores->cap > 0.0) {
    a.cap2 = static_cast<float>(scores->cap * log2e);
    a.scale_by_cap = static_cast<float>(scale / scores->cap);
    a.scale_by_cap2 = static_cast<float>(2.0 * log2e * scale / scores->cap);
  }
  a.q_aligned = Aligned(q) && q->shape[3] % 8 == 0;
  const size_t item = q->dtype == FL_FLOAT32 ? 4 : 2;
  a.out_aligned = IsAligned(out->base, 4 * item) && out->shape[3] % 4 == 0 && out->strides[3] == 1;
  for (int i = 0; i < 3; ++i) a.out_aligned = a.out_aligned && (out->shape[i] == 1 || out->strides[i] % 4 == 0);
  const uint32_t heads = static_cast<uint32_t>(a.batch) * static_cast<uint32_t>(a.kv_heads);
  const uint32_t tiles = static_cast<uint32_t>(plan.many ? (a.rows + 127) / 128 : (a.rows + 15) / 16);
  a.by_xcd = heads % 8 == 0;
  a.group_div = FastDiv(static_cast<uint32_t>(a.group));
  a.kv_div = FastDiv(static_cast<uint32_t>(a.kv_heads));
  a.tiles_div = FastDiv(tiles);
  a.heads_div = FastDiv(heads);
  a.splits = plan.splits;
  uint8_t *const at = static_cast<uint8_t *>(scratch);
  if (scores->key_documents != nullptr) {
    a.blocks = (a.keys + kBlock - 1) / kBlock;
    a.ranges = reinterpret_cast<int2 *>(at + plan.ranges_at);
    FL_LAUNCH(DocumentRangesKernel, dim3((a.blocks + 3) / 4, a.batch), dim3(256), 0, AsStream(stream), a);
    FL_CHECK(LaunchStatus());
  }
  if (plan.splits > 1) {
    a.partial = reinterpret_cast<float *>(at + plan.partial_at);
    a.stats = reinterpret_cast<float2 *>(at + plan.stats_at);
  }
  return ForDecoderType(q->dtype, [&](auto type) {
    using T = decltype(type);
    if (plan.many) return LaunchRows<T>(a, AsStream(stream));
    if (a.columns <= 64) return LaunchFew<T, 64>(a, aligned, AsStream(stream));
    if (a.columns <= 128) return LaunchFew<T, 128>(a, aligned, AsStream(stream));
    return LaunchFew<T, 256>(a, aligned, AsStream(stream));
  });
}

}  // extern "C"
