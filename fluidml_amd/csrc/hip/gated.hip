// The gated feed-forward block: products = act(x . gate + gate_bias) * (x . up + up_bias), out = products . down + down_bias + addend.
#include <cmath>
#include <type_traits>

#include "decoder_common.h"

using namespace fl;

namespace {

struct GatedArgs {
  const void *x, *gate, *up, *gate_bias, *up_bias, *addend;
  void *out;
  int64_t x_strides[2], gate_strides[2], up_strides[2], out_strides[2], addend_strides[2], gate_bias_stride, up_bias_stride;
  int32_t rows, depth, columns, activation;
  FastDiv row_tiles, column_tiles, group;  // tiles of x, of the weights; tiles of x that are walked together times those of the weights
  int32_t out_vectors;  // four results of a row in one store
  int32_t x_near, weights_near;      // runs of whole words, near enough for 32-bit offsets ..
  int32_t x_direct, weights_direct;  // .. and 16-byte aligned: straight into LDS
  int32_t x_run, gate_run, up_run;   // values of the layout's long side lie side by side: 2 in whole words, 1 at any address, 0 not
};

typedef _Float16 halfx8 __attribute__((ext_vector_type(8)));
typedef float floatx4 __attribute__((ext_vector_type(4)));
typedef short shortx4 __attribute__((ext_vector_type(4)));

// 1 / (1 + exp(-v)), from exp2 and the reciprocal instruction: a few roundings of itself
__device__ __forceinline__ float Logistic(float v) { return __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(v * -1.4426950408889634f)); }

__device__ __forceinline__ float Activated(int activation, float v) {
  switch (activation) {
    case FL_GATE_SILU: return v * Logistic(v);
    case FL_GATE_GELU: return 0.5f * v * (1.0f + erff(v * 0.70710678118654752f));
    case FL_GATE_GELU_TANH: return v * Logistic(1.5957691216057308f * (v + 0.044715f * v * v * v));  // 1 + tanh y = 2 / (1 + exp(-2 y))
    case FL_GATE_RELU: return v != v ? v : fmaxf(v, 0.0f);
    case FL_GATE_SIGMOID: return Logistic(v);
    default: return v;
  }
}

template <typename T>
__device__ __forceinline__ float BiasAt(const void *bias, int64_t stride, int64_t n) {
  return bias == nullptr ? 0.0f : static_cast<float>(static_cast<const T *>(bias)[n * stride]);
}

// The epilogue of one result: biases, the activation and the product, or a bias and an addend.
template <typename T, bool GATED>
__device__ __forceinline__ void StoreOne(const GatedArgs &a, int32_t m, int32_t n, float g, float u) {
  g += BiasAt<T>(a.gate_bias, a.gate_bias_stride, n);
  if constexpr (GATED) {
    g = Activated(a.activation, g) * (u + BiasAt<T>(a.up_bias, a.up_bias_stride, n));
  } else if (a.addend != nullptr) {
    g += static_cast<float>(static_cast<const T *>(a.addend)[m * a.addend_strides[0] + n * a.addend_strides[1]]);
  }
  static_cast<T *>(a.out)[m * a.out_strides[0] + n * a.out_strides[1]] = static_cast<T>(g);
}

// ... of four neighbouring columns of a row
template <typename T, bool GATED>
__device__ __forceinline__ void StoreFour(const GatedArgs &a, int32_t m, int32_t n, floatx4 g, floatx4 u) {
  if (m >= a.rows || n >= a.columns) return;
  T *const to = static_cast<T *>(a.out) + m * a.out_strides[0] + n * a.out_strides[1];
  typedef T Vec __attribute__((ext_vector_type(4)));
  Vec v;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const int32_t at = min(n + e, a.columns - 1);
    float x = g[e] + BiasAt<T>(a.gate_bias, a.gate_bias_stride, at);
    if constexpr (GATED) {
      x = Activated(a.activation, x) * (u[e] + BiasAt<T>(a.up_bias, a.up_bias_stride, at));
    } else if (a.addend != nullptr) {
      x += static_cast<float>(static_cast<const T *>(a.addend)[m * a.addend_strides[0] + at * a.addend_strides[1]]);
    }
    v[e] = static_cast<T>(x);
  }
  if (a.out_vectors) {
    *reinterpret_cast<Vec *>(to) = v;
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      if (n + e < a.columns) to[e * a.out_strides[1]] = v[e];
    }
  }
}

// A sum of fp32 products that three bf16 parts cannot carry (an infinity minus itself is no number; parts of the smallest values vanish), again
// with fp32 products, by the whole wave.
__device__ __forceinline__ float CarefulDot(const GatedArgs &a, const void *weights, const int64_t (&strides)[2], int32_t m, int32_t n) {
  const float *const x = static_cast<const float *>(a.x) + m * a.x_strides[0], *const w = static_cast<const float *>(weights) + n * strides[1];
  float sum = 0.0f;
  for (int32_t k = threadIdx.x % kWave; k < a.depth; k += kWave) sum += x[k * a.x_strides[1]] * w[k * strides[0]];
  return GroupSum<64>(sum);
}

// --------------------------------------------------------------------------------------------------------------------
// Tiles.  A workgroup owns BM rows of x and BW columns of weights: half of them the gate's and half the up projection's same ones, so that both
// sums of a result meet in one lane, or (not GATED) BW of one matrix.  Computed transposed, W^T x^T: a lane has one row of the result and
// four neighbouring columns at a time.  WM x WN x WK waves; WK waves share the depth of a stage and add their sums through LDS.
// A stage is BK of the depth, in two buffers: the next one is on its way while one is multiplied, one barrier a stage.  Direct: from memory
// into LDS without a register; otherwise (odd strides and addresses, the last part of a depth that BK does not divide, and fp32,
// which is split into three bf16 parts on the way) through registers, zeros behind the ends.
// Weights lie in LDS as they lie in memory, a row for each column of the product (ROWS: a checkpoint's [N, K]) or a row for each of the
// depth ([K, N], turned by the transposing read).  Groups of 16 bytes are permuted within a row against bank conflicts.
// bf16, 8192 rows of 4096, 14336 columns: 1650 us gated (1166 TFLOP/s), 800 us back (1202); a library's plain product of that kind reaches 1378, at
// which both would take 2094.  Bound by the matrix pipe and the power it leaves the clock.  fp32 in three parts: 4096^3 165 TFLOP/s.
template <typename T, int BM_, int BW_, int WM_, int WN_, int WK_, int BK_, bool GATED_, bool ROWS_>
struct TileShape {
  static constexpr int BM = BM_, BW = BW_, WM = WM_, WN = WN_, WK = WK_, BK = BK_;
  static constexpr bool GATED = GATED_, ROWS = ROWS_, kParted = std::is_same_v<T, float>;
  static constexpr int kParts = kParted ? 3 : 1, kWaves = WM * WN * WK, kThreads = kWaves * kWave;
  static constexpr int BN = GATED ? BW / 2 : BW;           // columns of the result
  static constexpr int kXGroups = BM * BK / 8, kWGroups = BW * BK / 8;
  static constexpr int kXLoads = kXGroups / kThreads, kWLoads = kWGroups / kThreads;  // a thread's, in groups of eight values
  static constexpr int kRowTiles = BM / WM / 32, kWTiles = BW / WN / 32;
  static constexpr int kXValues = BM * BK, kWValues = BW * BK;
  static constexpr int kStage = kParts * (kXValues + kWValues);
  static constexpr int kBuffers = kParted ? 1 : 2;       // two workgroups of the one hide more than two buffers of one workgroup
  static constexpr int kLds = kStage * kBuffers;
  static constexpr bool kLarge = BM == 256;             // direct loads only
  static constexpr int kAhead = WK > 1 || (kParted && BM < 128) ? 2 : 1;  // stages on their way in registers
  static_assert(kXGroups % kThreads == 0 && kWGroups % kThreads == 0 && BK % (16 * WK) == 0 && (!GATED || BW / WN == 64), "every thread and wave has the same to do");
};

// The group of eight values in the place of group `group` of row `row`.  LDS serves 256 bytes at a time: sixteen lanes' 16 bytes of one group of sixteen
// rows of x and of ROWS weights (BK values a row), 64 bytes of four rows of the others (BW values a row).  Turned by the row's number those
// fall on different banks, however many rows lie in 256 bytes.
template <int BK>
__device__ __forceinline__ int SwizzledLong(int row, int group) {
  constexpr int kGroups = BK / 8;
  static_assert(kGroups <= 16, "a row is at most 256 bytes");
  return group ^ (row / (16 / kGroups) & (kGroups - 1));
}
template <int BW>
__device__ __forceinline__ int SwizzledWide(int row, int group) {
  static_assert(BW == 64 || BW % 128 == 0, "half of 256 bytes or whole ones");
  return group ^ (BW == 64 ? (row / 2 & 1) * 4 : (row & 3) * 4);
}

template <typename E>
__device__ __forceinline__ floatx16 Mfma32(u32x4 x, u32x4 y, floatx16 acc) {
  if constexpr (std::is_same_v<E, _Float16>) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(halfx8, x), __builtin_bit_cast(halfx8, y), acc, 0, 0, 0);
  } else {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, x), __builtin_bit_cast(bf16x8, y), acc, 0, 0, 0);
  }
}

// Values at .. at + 7 of a row whose values lie `stride` apart, zeros from `limit` on (which is at least 1).  No branch around a load: what is not
// there is read as the last one.
template <typename T>
struct Eight {
  T v[8];
};
template <typename T>
__device__ __forceinline__ Eight<T> LoadEight(const T *row, int64_t stride, int32_t at, int32_t limit, bool there = true) {
  Eight<T> x;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const T v = row[min(at + e, limit - 1) * stride];
    x.v[e] = there && at + e < limit ? v : static_cast<T>(0.0f);
  }
  return x;
}

// The same for values side by side at any address, `limit` at least N, without a branch around a load: the last N of the row where at + N > limit,
// shifted.  16-bit values at odd addresses: whole words and the next one, turned (16 bytes at an odd address take the load three
// times as long: 333 rows of 2731 by 1000 columns 65 us, of 2732 23).
template <int N, typename T>
struct Row {
  typedef T Vec __attribute__((ext_vector_type(N)));
  typedef uint32_t Words __attribute__((ext_vector_type(N * sizeof(T) / 4)));
  typedef uint32_t LooseWords __attribute__((ext_vector_type(N * sizeof(T) / 4), aligned(4)));
  static __device__ __forceinline__ Vec Load(const T *row, int32_t at, int32_t limit) {
    const int32_t from = min(at, limit - N), shift = at - from;
    Vec v, x;
    if constexpr (sizeof(T) == 4) {
      v = __builtin_bit_cast(Vec, Words(*reinterpret_cast<const LooseWords *>(row + from)));
    } else {
      constexpr int kWords = N / 2;
      const uintptr_t where = reinterpret_cast<uintptr_t>(row + from);
      const uint32_t odd = where & 2;
      const uint32_t *const word = reinterpret_cast<const uint32_t *>(where - odd);
      Words w = *reinterpret_cast<const LooseWords *>(word);
      const uint32_t next = word[odd ? kWords : kWords - 1];  // (every word read holds a value of the row)
#pragma unroll
      for (int n = 0; n < kWords; ++n) w[n] = __builtin_amdgcn_alignbit(n + 1 < kWords ? w[(n + 1) % kWords] : next, w[n], odd * 8);
      v = __builtin_bit_cast(Vec, w);
    }
    if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int e = 0; e < N; ++e) {
        x[e] = static_cast<T>(0.0f);
#pragma unroll
        for (int n = e; n < N; ++n) x[e] = shift == n - e ? v[n] : x[e];
      }
    } else {
      typedef uint64_t Longs __attribute__((ext_vector_type(N / 4)));
      Longs w = __builtin_bit_cast(Longs, v);
      const int bits = 16 * (shift & 3);
      if constexpr (N == 8) {
        const uint64_t low = shift < 4 ? w[0] : w[1], high = shift < 4 ? w[1] : 0;
        w[0] = low >> bits | (bits == 0 ? 0 : high << (64 - bits));
        w[1] = high >> bits;
      } else {
        w[0] >>= bits;
      }
      x = __builtin_bit_cast(Vec, w);
#pragma unroll
      for (int e = 0; e < N; ++e) x[e] = shift < N ? x[e] : static_cast<T>(0.0f);
    }
    return x;
  }
};

template <typename T, typename Shape>
__global__ __launch_bounds__(Shape::kThreads, Shape::WK > 2 ? 3 : 2) void GatedTileKernel(const GatedArgs a) {
  using S = Shape;
  constexpr int BK = S::BK, BW = S::BW, BN = S::BN, kParts = S::kParts;
  constexpr bool kParted = S::kParted, GATED = S::GATED, ROWS = S::ROWS;
  using E = std::conditional_t<kParted, __bf16, T>;
  __shared__ alignas(16) uint16_t lds[S::kLds];
  const int lane = threadIdx.x % kWave, half = lane / 32, own = lane % 32, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int wk = wave % S::WK, wn = wave / S::WK % S::WN, wm = wave / S::WK / S::WN;

  // workgroups of an XCD (every eighth) work on neighbouring tiles: `group` tiles of rows by all columns, one after the other
  uint32_t id = blockIdx.x;
  const uint32_t total = a.row_tiles.divisor * a.column_tiles.divisor, even = total / 8 * 8;
  if (id < even) id = id % 8 * (total / 8) + id / 8;
  uint32_t row_tile, column_tile;
  {
    const uint32_t g = a.group.Div(id), rest = id - g * a.group.divisor, high = a.group.divisor / a.column_tiles.divisor;
    const uint32_t here = min(high, a.row_tiles.divisor - g * high);
    column_tile = rest / here;
    row_tile = g * high + (rest - column_tile * here);
  }
  const int32_t m0 = static_cast<int32_t>(row_tile) * S::BM, n0 = static_cast<int32_t>(column_tile) * BN;

  const T *const x_tile = static_cast<const T *>(a.x) + m0 * a.x_strides[0];
  const T *const gate_tile = static_cast<const T *>(a.gate) + n0 * a.gate_strides[1];
  const T *const up_tile = GATED ? static_cast<const T *>(a.up) + n0 * a.up_strides[1] : nullptr;

  // where a thread's groups come from.  x: row and group of the depth.  Weights: column and group of the depth (ROWS), or depth and group of columns
  uint32_t x_offset[S::kXLoads], w_offset[S::kWLoads];  // bytes, where 32 bits hold them
  constexpr uint32_t kItem = sizeof(T);
#pragma unroll
  for (int n = 0; n < S::kXLoads; ++n) {
    const int place = (wave * S::kXLoads + n) * kWave + lane, row = place / (BK / 8), group = SwizzledLong<BK>(row, place % (BK / 8));
    x_offset[n] = (static_cast<uint32_t>(min(row, a.rows - 1 - m0)) * static_cast<uint32_t>(a.x_strides[0]) + group * 8) * kItem;
  }
#pragma unroll
  for (int n = 0; n < S::kWLoads; ++n) {
    const int place = (wave * S::kWLoads + n) * kWave + lane;
    if constexpr (ROWS) {
      const int row = place / (BK / 8), group = SwizzledLong<BK>(row, place % (BK / 8));
      const bool up = GATED && row >= BN;
      w_offset[n] = (static_cast<uint32_t>(min(up ? row - BN : row, a.columns - 1 - n0)) * static_cast<uint32_t>(up ? a.up_strides[1] : a.gate_strides[1]) + group * 8) * kItem;
    } else {
      const int row = place / (BW / 8), group = SwizzledWide<BW>(row, place % (BW / 8));
      const bool up = GATED && group >= BN / 8;
      // (columns behind the last: the last group again, whose results are not stored)
      w_offset[n] = (static_cast<uint32_t>(row) * static_cast<uint32_t>(up ? a.up_strides[0] : a.gate_strides[0]) +
                     min(up ? group - BN / 8 : group, (a.columns - 1 - n0) / 8) * 8) * kItem;
    }
  }
  // (a group is the gate's or the up projection's by its place alone: the same for a whole load of a wave where ROWS, else by lane)
  auto direct = [&](int32_t k0) __attribute__((always_inline)) { return S::kLarge || (!kParted && S::kAhead == 1 && k0 + BK <= a.depth); };
  auto weights_from = [&](int32_t k0, int n) __attribute__((always_inline)) {
    const T *from = gate_tile + (ROWS ? k0 : k0 * a.gate_strides[0]);
    if constexpr (GATED) {
      const int place = (wave * S::kWLoads + n) * kWave + lane;
      const bool up = ROWS ? (wave * S::kWLoads + n) * kWave / (BK / 8) >= BN : SwizzledWide<BW>(place / (BW / 8), place % (BW / 8)) >= BN / 8;
      if (up) from = up_tile + (ROWS ? k0 : k0 * a.up_strides[0]);
    }
    return reinterpret_cast<const char *>(from) + w_offset[n];
  };
  auto fetch_direct = [&](int32_t k0, int stage, bool x, bool weights) __attribute__((always_inline)) {
    if constexpr (!kParted) {
      uint16_t *const x_to = lds + stage * S::kStage, *const w_to = x_to + kParts * S::kXValues;
      if (x) {
        const char *const from = reinterpret_cast<const char *>(x_tile + k0);
#pragma unroll
        for (int n = 0; n < S::kXLoads; ++n) LoadToLds(from + x_offset[n], x_to + (wave * S::kXLoads + n) * kWave * 8);
      }
      if (weights) {
#pragma unroll
        for (int n = 0; n < S::kWLoads; ++n) LoadToLds(weights_from(k0, n), w_to + (wave * S::kWLoads + n) * kWave * 8);
      }
    }
  };
  // through registers: whole runs of eight where they lie side by side, without a branch around a load; else value by value, zeros behind the ends
  struct Held {
    Eight<T> x[S::kXLoads], w[S::kWLoads];
  };
  auto fetch = [&](Held &held, int32_t k0, bool x, bool weights) __attribute__((always_inline)) {
    const bool whole = k0 + BK <= a.depth;
    if (x) {
#pragma unroll
      for (int n = 0; n < S::kXLoads; ++n) {
        const int place = (wave * S::kXLoads + n) * kWave + lane, row = place / (BK / 8), k = k0 + SwizzledLong<BK>(row, place % (BK / 8)) * 8;
        const T *const from = x_tile + min(row, a.rows - 1 - m0) * a.x_strides[0];
        if (whole && a.x_near) {
          __builtin_memcpy(&held.x[n], __builtin_assume_aligned(reinterpret_cast<const char *>(x_tile + k0) + x_offset[n], 4), sizeof(Eight<T>));
        } else if (a.x_run && a.depth >= 8) {
          held.x[n] = __builtin_bit_cast(Eight<T>, Row<8, T>::Load(from, k, a.depth));
        } else {
          held.x[n] = LoadEight<T>(from, a.x_strides[1], k, a.depth);
        }
      }
    }
    if (weights) {
      const bool runs = a.gate_run && (!GATED || a.up_run), run = a.weights_near && whole && (ROWS || n0 + BN <= a.columns);
#pragma unroll
      for (int n = 0; n < S::kWLoads; ++n) {
        const int place = (wave * S::kWLoads + n) * kWave + lane;
        const int row = ROWS ? place / (BK / 8) : place / (BW / 8);
        const int group = ROWS ? SwizzledLong<BK>(row, place % (BK / 8)) : SwizzledWide<BW>(row, place % (BW / 8));
        const bool up = GATED && (ROWS ? row >= BN : group >= BN / 8);
        const int64_t along = up ? a.up_strides[0] : a.gate_strides[0], across = up ? a.up_strides[1] : a.gate_strides[1];
        const T *from = up ? up_tile : gate_tile;
        if constexpr (ROWS) {
          const int32_t k = k0 + group * 8;
          from += min(up ? row - BN : row, a.columns - 1 - n0) * across;
          if (run) {
            __builtin_memcpy(&held.w[n], __builtin_assume_aligned(weights_from(k0, n), 4), sizeof(Eight<T>));
          } else if (runs && a.depth >= 8) {
            held.w[n] = __builtin_bit_cast(Eight<T>, Row<8, T>::Load(from, k, a.depth));
          } else {
            held.w[n] = LoadEight<T>(from, along, k, a.depth);
          }
        } else {
          const int32_t k = k0 + row, c = (up ? group - BN / 8 : group) * 8;
          from += min(k, a.depth - 1) * along;
          if (run) {
            __builtin_memcpy(&held.w[n], __builtin_assume_aligned(weights_from(k0, n), 4), sizeof(Eight<T>));
          } else if (runs && a.columns - n0 >= 8) {
            held.w[n] = __builtin_bit_cast(Eight<T>, Row<8, T>::Load(from, c, k < a.depth ? a.columns - n0 : 8));
            if (k >= a.depth) held.w[n] = Eight<T>{};
          } else {
            held.w[n] = LoadEight<T>(from, across, c, a.columns - n0, k < a.depth);
          }
        }
      }
    }
  };
  auto store = [&](const Held &held, int stage, bool x, bool weights) __attribute__((always_inline)) {
    uint16_t *const x_to = lds + stage * S::kStage, *const w_to = x_to + kParts * S::kXValues;
    auto put = [&](const Eight<T> &v, uint16_t *to, int values, int place) __attribute__((always_inline)) {
      if constexpr (kParted) {
        float f[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) f[e] = v.v[e];
        u32x4 part[3];
        SplitParts<3>(f, part);
#pragma unroll
        for (int p = 0; p < 3; ++p) *reinterpret_cast<u32x4 *>(to + p * values + place * 8) = part[p];
      } else {
        *reinterpret_cast<u32x4 *>(to + place * 8) = __builtin_bit_cast(u32x4, v);
      }
    };
    if (x) {
#pragma unroll
      for (int n = 0; n < S::kXLoads; ++n) put(held.x[n], x_to, S::kXValues, (wave * S::kXLoads + n) * kWave + lane);
    }
    if (weights) {
#pragma unroll
      for (int n = 0; n < S::kWLoads; ++n) put(held.w[n], w_to, S::kWValues, (wave * S::kWLoads + n) * kWave + lane);
    }
  };

  floatx16 acc[S::kRowTiles][S::kWTiles], low[kParted ? S::kRowTiles : 1][kParted ? S::kWTiles : 1];
#pragma unroll
  for (int i = 0; i < S::kRowTiles; ++i) {
#pragma unroll
    for (int j = 0; j < S::kWTiles; ++j) {
#pragma unroll
      for (int e = 0; e < 16; ++e) acc[i][j][e] = 0.0f, low[kParted ? i : 0][kParted ? j : 0][e] = 0.0f;
    }
  }
  // column (in LDS) of the wave's j-th tile of weights
  auto w_column = [&](int j) __attribute__((always_inline)) { return GATED ? j * BN + wn * 32 : wn * S::kWTiles * 32 + j * 32; };
  struct Operands {
    u32x4 x[S::kRowTiles][kParts], w[S::kWTiles][kParts];
  };
  auto read = [&](Operands &o, int stage, int step) __attribute__((always_inline)) {
    const uint16_t *const x_from = lds + stage * S::kStage, *const w_from = x_from + kParts * S::kXValues;
    const int st = step * S::WK + wk;
#pragma unroll
    for (int j = 0; j < S::kWTiles; ++j) {
#pragma unroll
      for (int p = 0; p < kParts; ++p) {
        if constexpr (ROWS) {
          const int row = w_column(j) + own;
          o.w[j][p] = *reinterpret_cast<const u32x4 *>(w_from + p * S::kWValues + row * BK + SwizzledLong<BK>(row, 2 * st + half) * 8);
        } else {
          // sixteen lanes read four of the depth by sixteen columns, and each gets one column's four
          const int row = st * 16 + half * 8 + lane % 16 / 4, group = w_column(j) / 8 + lane / 16 % 2 * 2 + lane % 4 / 2;
          uint16_t *const from = const_cast<uint16_t *>(w_from) + p * S::kWValues + row * BW + SwizzledWide<BW>(row, group) * 8 + lane % 2 * 4;
          typedef __attribute__((address_space(3))) shortx4 *Lds;
          const uint64_t first = __builtin_bit_cast(uint64_t, __builtin_amdgcn_ds_read_tr16_b64_v4i16((Lds)(from)));
          const uint64_t second = __builtin_bit_cast(uint64_t, __builtin_amdgcn_ds_read_tr16_b64_v4i16((Lds)(from + 4 * BW)));
          o.w[j][p] = u32x4{static_cast<uint32_t>(first), static_cast<uint32_t>(first >> 32), static_cast<uint32_t>(second), static_cast<uint32_t>(second >> 32)};
        }
      }
    }
#pragma unroll
    for (int i = 0; i < S::kRowTiles; ++i) {
      const int row = (wm * S::kRowTiles + i) * 32 + own;
#pragma unroll
      for (int p = 0; p < kParts; ++p) o.x[i][p] = *reinterpret_cast<const u32x4 *>(x_from + p * S::kXValues + row * BK + SwizzledLong<BK>(row, 2 * st + half) * 8);
    }
  };
  auto multiply = [&](int stage) __attribute__((always_inline)) {
    constexpr int kSteps = BK / 16 / S::WK, kSets = kParted ? 1 : 2;
    Operands o[kSets];
    if constexpr (!kParted) read(o[0], stage, 0);
#pragma unroll
    for (int step = 0; step < kSteps; ++step) {
      if constexpr (kParted) {
        read(o[0], stage, step);
      } else {
        if (step + 1 < kSteps) read(o[(step + 1) % kSets], stage, step + 1);
      }
      const Operands &now = o[step % kSets];
      if constexpr (kParted) {
        ForParts([&](auto p, auto q, auto small) __attribute__((always_inline)) {
#pragma unroll
          for (int i = 0; i < S::kRowTiles; ++i) {
#pragma unroll
            for (int j = 0; j < S::kWTiles; ++j) {
              floatx16 &to = small ? low[kParted ? i : 0][kParted ? j : 0] : acc[i][j];
              to = Mfma32<E>(now.w[j][p], now.x[i][q], to);
            }
          }
        });
      } else {
#pragma unroll
        for (int i = 0; i < S::kRowTiles; ++i) {
#pragma unroll
          for (int j = 0; j < S::kWTiles; ++j) acc[i][j] = Mfma32<E>(now.w[j][0], now.x[i][0], acc[i][j]);
        }
      }
    }
    if constexpr (!kParted && S::WK == 1) {
      // the order asked for: a step's operands are read between the products of the step before
      constexpr int kProducts = S::kRowTiles * S::kWTiles, kReads = S::kRowTiles + S::kWTiles * (ROWS ? 1 : 2);
      __builtin_amdgcn_sched_group_barrier(0x100, kReads, 0);
      StaticFor<kSteps>([&](auto step) __attribute__((always_inline)) {
        constexpr int left = decltype(step)::value + 1 < kSteps ? kReads : 0, each = (left + kProducts - 1) / kProducts;
        StaticFor<kProducts>([&](auto n) __attribute__((always_inline)) {
          constexpr int some = left - decltype(n)::value * each < 0 ? 0 : left - decltype(n)::value * each < each ? left - decltype(n)::value * each : each;
          __builtin_amdgcn_sched_group_barrier(0x8, 1, 0);
          if constexpr (some > 0) __builtin_amdgcn_sched_group_barrier(0x100, some, 0);
        });
      });
    }
  };
  auto ready = [&]() __attribute__((always_inline)) {  // the stage is there for all, and everyone is done with the one before
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    if constexpr (!kParted && S::kAhead == 1) asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
  };

  if constexpr (kParted) {
    Held held[S::kAhead];
    StaticFor<S::kAhead>([&](auto n) __attribute__((always_inline)) {
      if (n * BK < a.depth) fetch(held[n], n * BK, true, true);
    });
    for (int32_t k0 = 0; k0 < a.depth; k0 += S::kAhead * BK) {
      StaticFor<S::kAhead>([&](auto n) __attribute__((always_inline)) {
        const int32_t k = k0 + n * BK;
        if (k >= a.depth) return;
        ready();
        store(held[n], 0, true, true);
        if (k + S::kAhead * BK < a.depth) fetch(held[n], k + S::kAhead * BK, true, true);
        ready();
        multiply(0);
      });
    }
  } else if constexpr (S::kAhead > 1) {
    // few products to a stage: the time is that of the loads, so several stages are on their way
    Held held[S::kAhead];
    StaticFor<S::kAhead>([&](auto n) __attribute__((always_inline)) {
      if (n * BK < a.depth) fetch(held[n], n * BK, true, true);
    });
    store(held[0], 0, true, true);
    for (int32_t k0 = 0; k0 < a.depth; k0 += S::kAhead * BK) {
      StaticFor<S::kAhead>([&](auto n) __attribute__((always_inline)) {
        const int32_t k = k0 + n * BK;
        if (k >= a.depth) return;
        ready();
        if (k + S::kAhead * BK < a.depth) fetch(held[n], k + S::kAhead * BK, true, true);
        multiply(n % 2);
        if (k + BK < a.depth) store(held[(n + 1) % S::kAhead], (n + 1) % 2, true, true);
      });
    }
  } else {
    Held held;
    auto begin = [&](int32_t k0, int stage) __attribute__((always_inline)) {
      const bool near = direct(k0);
      fetch_direct(k0, stage, near && (S::kLarge || a.x_direct), near && (S::kLarge || a.weights_direct));
      if constexpr (!S::kLarge) fetch(held, k0, !(near && a.x_direct), !(near && a.weights_direct));
    };
    auto end = [&](int32_t k0, int stage) __attribute__((always_inline)) {
      const bool near = direct(k0);
      if constexpr (!S::kLarge) store(held, stage, !(near && a.x_direct), !(near && a.weights_direct));
    };
    begin(0, 0);
    end(0, 0);
    int stage = 0;
    for (int32_t k0 = 0; k0 < a.depth; k0 += BK) {
      ready();
      const bool more = k0 + BK < a.depth;
      if (more) begin(k0 + BK, stage ^ 1);
      multiply(stage);
      if (more) end(k0 + BK, stage ^ 1);
      stage ^= 1;
    }
  }
  SettleAcrossBranch();
#pragma unroll
  for (int i = 0; i < S::kRowTiles; ++i) {
#pragma unroll
    for (int j = 0; j < S::kWTiles; ++j) {
      asm volatile("" : "+v"(acc[i][j]));
      if constexpr (kParted) {
        asm volatile("" : "+v"(low[i][j]));
#pragma unroll
        for (int e = 0; e < 16; ++e) acc[i][j][e] += low[i][j][e];
      }
    }
  }

  if constexpr (S::WK > 1) {  // the waves that share the depth: the first adds the others' sums, in their order
    constexpr int kSums = S::kRowTiles * S::kWTiles * 16 * kWave;
    static_assert(S::kLds >= S::WM * S::WN * kSums * 2, "sums fit");
    float *const sums = reinterpret_cast<float *>(lds) + wave / S::WK * kSums;
    for (int w = 1; w < S::WK; ++w) {
      __syncthreads();
      if (wk == w) {
#pragma unroll
        for (int i = 0; i < S::kRowTiles; ++i) {
#pragma unroll
          for (int j = 0; j < S::kWTiles; ++j) {
#pragma unroll
            for (int e = 0; e < 16; ++e) sums[((i * S::kWTiles + j) * 16 + e) * kWave + lane] = acc[i][j][e];
          }
        }
      }
      __syncthreads();
      if (wk == 0) {
#pragma unroll
        for (int i = 0; i < S::kRowTiles; ++i) {
#pragma unroll
          for (int j = 0; j < S::kWTiles; ++j) {
#pragma unroll
            for (int e = 0; e < 16; ++e) acc[i][j][e] += sums[((i * S::kWTiles + j) * 16 + e) * kWave + lane];
          }
        }
      }
    }
    if (wk != 0) return;
  }

  constexpr int kResults = GATED ? 1 : S::kWTiles;
#pragma unroll
  for (int i = 0; i < S::kRowTiles; ++i) {
    const int32_t row0 = m0 + (wm * S::kRowTiles + i) * 32;
#pragma unroll
    for (int j = 0; j < kResults; ++j) {
      const int32_t column0 = n0 + (GATED ? wn * 32 : w_column(j));
      if constexpr (kParted) {
#pragma unroll
        for (int w = 0; w < (GATED ? 2 : 1); ++w) {
          bool bad = false;
#pragma unroll
          for (int e = 0; e < 16; ++e) bad = bad || BadSum(acc[i][j + w][e], false);
          if (!__any(bad)) continue;
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            const int32_t column = column0 + e / 4 * 8 + half * 4 + e % 4;
            for (uint64_t rest = __ballot(BadSum(acc[i][j + w][e], false) && row0 + own < a.rows && column < a.columns); rest != 0; rest &= rest - 1) {
              const int who = __builtin_ctzll(rest);
              const float again = CarefulDot(a, w == 0 ? a.gate : a.up, w == 0 ? a.gate_strides : a.up_strides, row0 + who % 32, column0 + e / 4 * 8 + who / 32 * 4 + e % 4);
              if (lane == who) acc[i][j + w][e] = again;
            }
          }
        }
      }
#pragma unroll
      for (int e = 0; e < 16; e += 4) {
        const floatx4 g = {acc[i][j][e], acc[i][j][e + 1], acc[i][j][e + 2], acc[i][j][e + 3]};
        floatx4 u = {};
        if constexpr (GATED) u = floatx4{acc[i][1][e], acc[i][1][e + 1], acc[i][1][e + 2], acc[i][1][e + 3]};
        StoreFour<T, GATED>(a, row0 + own, column0 + e / 4 * 8 + half * 4, g, u);
      }
    }
  }
}

// --------------------------------------------------------------------------------------------------------------------
// Few rows (a step of decoding): bound by the bytes of the weights, which go straight into registers, 16 x 16 instructions behind them; the rows
// of x are the instruction's columns, up to sixteen of them RT times.  A workgroup owns 16 columns of the product (ROWS) or 64, and its eight
// waves share the depth, each a run of kDepth at a time; their sums meet in LDS, in the order of the waves.  The next run is on
// its way while one is multiplied.
// ROWS: a lane loads 16 bytes of the depth of column lane % 16.  Otherwise four columns of each of the depth's values of its quarter of the wave,
// and turns them around in registers.  fp32 stays fp32: at few rows its products cost less than the bytes.
// bf16, 4 rows of 4096, 11008 columns: 34 us gated (180 MB, 5.4 TB/s), 19 us back (90 MB, 4.8 TB/s).
template <typename T, bool GATED_, bool ROWS_, int RT_>
struct FewShape {
  static constexpr bool GATED = GATED_, ROWS = ROWS_, kWide = std::is_same_v<T, float>;
  static constexpr int RT = RT_, kMatrices = GATED ? 2 : 1;
  static constexpr int kGroup = 16 / sizeof(T);                       // values of the depth of a lane in a step
  static constexpr int kStep = 4 * kGroup;                            // of the depth
  static constexpr int kSteps = ROWS ? (GATED || RT == 2 ? 4 : 8) : (GATED ? 1 : 2);
  static constexpr int kDepth = kSteps * kStep;                       // a wave's run
  static constexpr int kTiles = ROWS ? 1 : 4, kColumns = 16 * kTiles; // tiles of sixteen columns
  static constexpr int kWaves = 8;
};

template <typename T, typename Shape>
__global__ __launch_bounds__(512, 2) void GatedFewKernel(const GatedArgs a) {
  using S = Shape;
  constexpr bool GATED = S::GATED, ROWS = S::ROWS, kWide = S::kWide;
  constexpr int RT = S::RT, kMatrices = S::kMatrices, kGroup = S::kGroup, kSteps = S::kSteps, kTiles = S::kTiles;
  typedef T Group __attribute__((ext_vector_type(kGroup)));
  typedef T Four __attribute__((ext_vector_type(4)));
  typedef T Loose __attribute__((ext_vector_type(kGroup), aligned(4)));   // at any word
  typedef T LooseFour __attribute__((ext_vector_type(4), aligned(4)));
  __shared__ float joined[S::kWaves][kMatrices][RT][256];
  const int lane = threadIdx.x % kWave, own = lane % 16, quarter = lane / 16, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  // (the tiles of rows of the same columns one after the other on one XCD, which has the weights then)
  uint32_t id = blockIdx.x;
  const uint32_t total = a.row_tiles.divisor * a.column_tiles.divisor, even = total / 8 * 8;
  if (id < even) id = id % 8 * (total / 8) + id / 8;
  const uint32_t column_tile = a.row_tiles.Div(id);
  const int32_t n0 = static_cast<int32_t>(column_tile) * S::kColumns, m0 = static_cast<int32_t>(id - column_tile * a.row_tiles.divisor) * RT * 16;
  const T *const x_own = static_cast<const T *>(a.x);
  const T *const matrix[2] = {static_cast<const T *>(a.gate), static_cast<const T *>(GATED ? a.up : a.gate)};
  const int64_t along[2] = {a.gate_strides[0], a.up_strides[0]}, across[2] = {a.gate_strides[1], a.up_strides[1]};

  struct Run {
    Group x[kSteps][RT];
    Group w[ROWS ? kMatrices : 1][ROWS ? kSteps : 1];
    Four v[ROWS ? 1 : kMatrices][ROWS ? 1 : kSteps][ROWS ? 1 : kGroup];  // [depth][columns]
  };
  const bool runs = a.x_run && a.gate_run && (!GATED || a.up_run) && a.depth >= kGroup && (ROWS || a.columns >= 4);
  const bool inside = (ROWS || n0 + S::kColumns <= a.columns) && a.x_run == 2 && a.gate_run == 2 && (!GATED || a.up_run == 2);
  auto load = [&](Run &r, int32_t k0) __attribute__((always_inline)) {
    if (inside && k0 + S::kDepth <= a.depth) {
#pragma unroll
      for (int s = 0; s < kSteps; ++s) {
        const int32_t k = k0 + s * S::kStep + quarter * kGroup;
#pragma unroll
        for (int m = 0; m < kMatrices; ++m) {
          if constexpr (ROWS) {
            r.w[m][s] = *reinterpret_cast<const Loose *>(matrix[m] + min(n0 + own, a.columns - 1) * across[m] + k);
          } else {
#pragma unroll
            for (int e = 0; e < kGroup; ++e) r.v[m][s][e] = *reinterpret_cast<const LooseFour *>(matrix[m] + (k + e) * along[m] + n0 + own * 4);
          }
        }
#pragma unroll
        for (int t = 0; t < RT; ++t) r.x[s][t] = *reinterpret_cast<const Loose *>(x_own + min(m0 + t * 16 + own, a.rows - 1) * a.x_strides[0] + k);
      }
    } else if (runs) {  // the same at the ends, and at odd addresses
#pragma unroll
      for (int s = 0; s < kSteps; ++s) {
        const int32_t k = k0 + s * S::kStep + quarter * kGroup;
#pragma unroll
        for (int m = 0; m < kMatrices; ++m) {
          if constexpr (ROWS) {
            r.w[m][s] = Row<kGroup, T>::Load(matrix[m] + min(n0 + own, a.columns - 1) * across[m], k, a.depth);
          } else {
#pragma unroll
            for (int e = 0; e < kGroup; ++e) {
              const Four v = Row<4, T>::Load(matrix[m] + min(k + e, a.depth - 1) * along[m], n0 + own * 4, a.columns);
              r.v[m][s][e] = k + e < a.depth ? v : Four{};
            }
          }
        }
#pragma unroll
        for (int t = 0; t < RT; ++t) r.x[s][t] = Row<kGroup, T>::Load(x_own + min(m0 + t * 16 + own, a.rows - 1) * a.x_strides[0], k, a.depth);
      }
    } else {  // value by value, zeros behind the ends (no branch around a load)
#pragma unroll
      for (int s = 0; s < kSteps; ++s) {
        const int32_t k = k0 + s * S::kStep + quarter * kGroup;
#pragma unroll
        for (int m = 0; m < kMatrices; ++m) {
          if constexpr (ROWS) {
            const T *const from = matrix[m] + min(n0 + own, a.columns - 1) * across[m];
#pragma unroll
            for (int e = 0; e < kGroup; ++e) {
              const T v = from[min(k + e, a.depth - 1) * along[m]];
              r.w[m][s][e] = k + e < a.depth ? v : static_cast<T>(0.0f);
            }
          } else {
#pragma unroll
            for (int e = 0; e < kGroup; ++e) {
#pragma unroll
              for (int c = 0; c < 4; ++c) {
                const int32_t n = n0 + own * 4 + c;
                const T v = matrix[m][min(k + e, a.depth - 1) * along[m] + min(n, a.columns - 1) * across[m]];
                r.v[m][s][e][c] = k + e < a.depth && n < a.columns ? v : static_cast<T>(0.0f);
              }
            }
          }
        }
#pragma unroll
        for (int t = 0; t < RT; ++t) {
          const T *const from = x_own + min(m0 + t * 16 + own, a.rows - 1) * a.x_strides[0];
#pragma unroll
          for (int e = 0; e < kGroup; ++e) {
            const T v = from[min(k + e, a.depth - 1) * a.x_strides[1]];
            r.x[s][t][e] = k + e < a.depth ? v : static_cast<T>(0.0f);
          }
        }
      }
    }
  };
  floatx4 acc[kMatrices][kTiles][RT];
#pragma unroll
  for (int m = 0; m < kMatrices; ++m) {
#pragma unroll
    for (int c = 0; c < kTiles; ++c) {
#pragma unroll
      for (int t = 0; t < RT; ++t) acc[m][c][t] = floatx4{0.0f, 0.0f, 0.0f, 0.0f};
    }
  }
  auto multiply = [&](const Run &r) __attribute__((always_inline)) {
#pragma unroll
    for (int s = 0; s < kSteps; ++s) {
#pragma unroll
      for (int m = 0; m < kMatrices; ++m) {
#pragma unroll
        for (int c = 0; c < kTiles; ++c) {
          if constexpr (kWide) {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const float w = ROWS ? r.w[ROWS ? m : 0][ROWS ? s : 0][e] : r.v[ROWS ? 0 : m][ROWS ? 0 : s][ROWS ? 0 : e][c];
#pragma unroll
              for (int t = 0; t < RT; ++t) acc[m][c][t] = __builtin_amdgcn_mfma_f32_16x16x4f32(w, r.x[s][t][e], acc[m][c][t], 0, 0, 0);
            }
          } else {
            Group w;
            if constexpr (ROWS) {
              w = r.w[m][s];
            } else {  // column c of eight of the depth
              typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
              u32x4 turned;
#pragma unroll
              for (int n = 0; n < 4; ++n) {
                const u32x2 first = __builtin_bit_cast(u32x2, r.v[m][s][2 * n]), second = __builtin_bit_cast(u32x2, r.v[m][s][2 * n + 1]);
                turned[n] = __builtin_amdgcn_perm(second[c / 2], first[c / 2], c % 2 == 0 ? 0x05040100u : 0x07060302u);
              }
              w = __builtin_bit_cast(Group, turned);
            }
#pragma unroll
            for (int t = 0; t < RT; ++t) {
              if constexpr (std::is_same_v<T, _Float16>) {
                acc[m][c][t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(w, r.x[s][t], acc[m][c][t], 0, 0, 0);
              } else {
                acc[m][c][t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(w, r.x[s][t], acc[m][c][t], 0, 0, 0);
              }
            }
          }
        }
      }
    }
  };

  constexpr int32_t kAll = S::kWaves * S::kDepth;
  Run r;
  int32_t k0 = wave * S::kDepth;
  if (k0 < a.depth) {
    load(r, k0);
    for (; k0 + kAll < a.depth; k0 += kAll) {
      Run next;
      load(next, k0 + kAll);
      multiply(r);
      r = next;
    }
    multiply(r);
  }
  SettleAcrossBranch();
#pragma unroll
  for (int c = 0; c < kTiles; ++c) {
    if (c > 0) __syncthreads();
#pragma unroll
    for (int m = 0; m < kMatrices; ++m) {
#pragma unroll
      for (int t = 0; t < RT; ++t) {
        asm volatile("" : "+v"(acc[m][c][t]));
        *reinterpret_cast<floatx4 *>(&joined[wave][m][t][lane * 4]) = acc[m][c][t];
      }
    }
    __syncthreads();
    for (int at = threadIdx.x; at < RT * 256; at += 512) {
      // row `row` of x by column `place` of the tile: register place % 4 of lane (place / 4) * 16 + row
      const int t = at / 256, row = at % 256 / 16, place = at % 16, from = ((place / 4) * 16 + row) * 4 + place % 4;
      const int32_t m = m0 + t * 16 + row, n = n0 + (ROWS ? place : place * 4 + c);
      if (m >= a.rows || n >= a.columns) continue;
      float g = 0.0f, u = 0.0f;
#pragma unroll
      for (int w = 0; w < S::kWaves; ++w) {
        g += joined[w][0][t][from];
        if constexpr (GATED) u += joined[w][kMatrices - 1][t][from];
      }
      StoreOne<T, GATED>(a, m, n, g, u);
    }
  }
}

int CheckMatrix(const fl_tensor *t, int32_t dtype, int64_t rows, int64_t columns, bool result = false) {
  FL_CHECK(result ? CheckWideResult(t) : CheckWideView(t));
  if (t->rank != 2) return FL_ERR_RANK;
  if (t->dtype != dtype) return FL_ERR_DTYPE;
  return t->shape[0] == rows && t->shape[1] == columns ? FL_OK : FL_ERR_SHAPE;
}

// a result that any of the kernels' grids counts: its tiles have 16 columns or more, 8192 places or more where there are many
int CheckExtents(int64_t rows, int64_t columns) { return columns > (1 << 26) || rows * columns > (INT64_C(1) << 36) ? FL_ERR_TOO_LARGE : FL_OK; }

int CheckGated(const fl_tensor *x, const fl_tensor *gate, const fl_tensor *up, const fl_tensor *gate_bias, const fl_tensor *up_bias,
               const fl_tensor *products, int32_t activation) {
  FL_CHECK(CheckWideView(x));
  FL_CHECK(CheckWideView(gate));
  if (x->rank != 2 || gate->rank != 2) return FL_ERR_RANK;
  if (!IsDecoderType(x->dtype)) return FL_ERR_DTYPE;
  const int64_t M = x->shape[0], K = x->shape[1], N = gate->shape[1];
  FL_CHECK(CheckMatrix(gate, x->dtype, K, N));
  FL_CHECK(CheckMatrix(up, x->dtype, K, N));
  FL_CHECK(CheckMatrix(products, x->dtype, M, N, true));
  FL_CHECK(CheckOptionalVector(gate_bias, x->dtype, N));
  FL_CHECK(CheckOptionalVector(up_bias, x->dtype, N));
  if (activation < FL_GATE_SILU || activation > FL_GATE_IDENTITY) return FL_ERR_ATTR;
  return CheckExtents(M, N);
}

void Set(const fl_tensor *t, int64_t (&strides)[2]) {
  for (int i = 0; i < 2; ++i) strides[i] = t == nullptr ? 0 : t->strides[i];
}

int Run(const fl_tensor *t, int unit) {
  if (t->strides[unit] != 1) return 0;
  return t->dtype == FL_FLOAT32 || (IsAligned(t->base, 4) && (t->strides[1 - unit] % 2 == 0 || t->shape[1 - unit] == 1)) ? 2 : 1;
}

template <typename T, typename Shape>
int LaunchTiles(GatedArgs &a, hipStream_t stream) {
  const int64_t rows = (a.rows + Shape::BM - 1) / Shape::BM, columns = (a.columns + Shape::BN - 1) / Shape::BN;
  a.row_tiles = FastDiv(static_cast<uint32_t>(rows));
  a.column_tiles = FastDiv(static_cast<uint32_t>(columns));
  a.group = FastDiv(static_cast<uint32_t>(std::min<int64_t>(rows, 8) * columns));
  FL_LAUNCH((GatedTileKernel<T, Shape>), dim3(static_cast<uint32_t>(rows * columns)), dim3(Shape::kThreads), 0, stream, a);
  return LaunchStatus();
}

template <typename T, typename Shape>
int LaunchFew(GatedArgs &a, hipStream_t stream) {
  const int64_t rows = (a.rows + Shape::RT * 16 - 1) / (Shape::RT * 16), columns = (a.columns + Shape::kColumns - 1) / Shape::kColumns;
  a.row_tiles = FastDiv(static_cast<uint32_t>(rows));
  a.column_tiles = FastDiv(static_cast<uint32_t>(columns));
  FL_LAUNCH((GatedFewKernel<T, Shape>), dim3(static_cast<uint32_t>(rows * columns)), dim3(512), 0, stream, a);
  return LaunchStatus();
}

// The largest tiles that still fill the chip.  Gated, weights as [N, K], in us (other choice):
//   16-bit, depth 4096: 256 x 256 in 208 tiles 125 (128 x 128: 152), in 160 tiles 125 (130); 128 x 128 in 128 tiles 57 (64 x 64: 57), in 96 tiles 53
//   (55); 64 x 64 in 256 tiles 50 (32 rows, few: 66), in 128 tiles 40 (33)
//   fp32, depth 1024: 128 x 128 in 256 tiles 75 (64 x 128: 76), in 128 tiles 69 (39); 64 x 128 in 128 tiles 35 (few: 43), in 64 tiles 34 (23)
//   few rows: 32 of them in 512 workgroups 33 (16: 47), in 128 workgroups 17.6 (13.7)
template <typename T, bool GATED, bool ROWS>
int LaunchLayout(GatedArgs &a, hipStream_t stream) {
  auto tiles = [&](int64_t bm, int64_t bw) { return (a.rows + bm - 1) / bm * ((a.columns + bw / (GATED ? 2 : 1) - 1) / (bw / (GATED ? 2 : 1))); };
  if (a.rows <= 16) return LaunchFew<T, FewShape<T, GATED, ROWS, 1>>(a, stream);
  if (a.rows <= 32) return LaunchFew<T, FewShape<T, GATED, ROWS, 2>>(a, stream);
  if constexpr (std::is_same_v<T, float>) {
    if (tiles(128, 128) >= 256) return LaunchTiles<T, TileShape<T, 128, 128, 2, 2, 1, 32, GATED, ROWS>>(a, stream);
    if (tiles(64, 128) >= 128) return LaunchTiles<T, TileShape<T, 64, 128, 2, 2, 2, 64, GATED, ROWS>>(a, stream);
  } else {
    if (tiles(256, 256) >= 160 && a.x_direct && a.weights_direct && a.depth % 64 == 0) return LaunchTiles<T, TileShape<T, 256, 256, 2, 4, 1, 64, GATED, ROWS>>(a, stream);
    if (tiles(128, 128) >= 128) return LaunchTiles<T, TileShape<T, 128, 128, 2, 2, 1, 64, GATED, ROWS>>(a, stream);
    if (tiles(64, 64) >= 256) return LaunchTiles<T, TileShape<T, 64, 64, 1, 1, 4, 64, GATED, ROWS>>(a, stream);
  }
  // few tiles: sixteen rows a workgroup where thirty-two leave compute units without one
  constexpr int kColumns = FewShape<T, GATED, ROWS, 1>::kColumns;
  if ((a.rows + 31) / 32 * ((a.columns + kColumns - 1) / kColumns) < 256) return LaunchFew<T, FewShape<T, GATED, ROWS, 1>>(a, stream);
  return LaunchFew<T, FewShape<T, GATED, ROWS, 2>>(a, stream);
}

// out = act(x . gate + gate_bias) * (x . up + up_bias), or with `up` NULL: x . gate + gate_bias + addend
int Contract(const fl_tensor *x, const fl_tensor *gate, const fl_tensor *up, const fl_tensor *gate_bias, const fl_tensor *up_bias, const fl_tensor *addend,
             const fl_tensor *out, int32_t activation, hipStream_t stream) {
  GatedArgs a;
  std::memset(&a, 0, sizeof(a));
  a.x = x->base, a.gate = gate->base, a.up = up == nullptr ? nullptr : up->base, a.out = out->base;
  a.gate_bias = gate_bias == nullptr ? nullptr : gate_bias->base;
  a.up_bias = up_bias == nullptr ? nullptr : up_bias->base;
  a.addend = addend == nullptr ? nullptr : addend->base;
  Set(x, a.x_strides), Set(gate, a.gate_strides), Set(up, a.up_strides), Set(out, a.out_strides), Set(addend, a.addend_strides);
  a.gate_bias_stride = gate_bias == nullptr ? 0 : gate_bias->strides[0];
  a.up_bias_stride = up_bias == nullptr ? 0 : up_bias->strides[0];
  a.rows = static_cast<int32_t>(x->shape[0]), a.depth = static_cast<int32_t>(x->shape[1]), a.columns = static_cast<int32_t>(gate->shape[1]);
  a.activation = activation;
  // the layout that the weights share, or that of a checkpoint; a matrix that has another is read value by value
  const bool wide = gate->strides[1] == 1 && (up == nullptr || up->strides[1] == 1) && !(gate->strides[0] == 1 && gate->shape[1] > 1 && gate->shape[0] == 1);
  const int unit = wide ? 1 : 0;
  a.x_run = Run(x, 1);
  a.gate_run = Run(gate, unit);
  a.up_run = up == nullptr ? 0 : Run(up, unit);
  auto near = [](const fl_tensor *t, int u) { return Run(t, u) == 2 && t->strides[1 - u] < (1 << 21); };
  const int64_t group = x->dtype == FL_FLOAT32 ? 4 : 8;
  auto aligned = [&](const fl_tensor *t, int u) { return near(t, u) && IsAligned(t->base, 16) && t->strides[1 - u] % group == 0; };
  a.x_near = near(x, 1);
  a.weights_near = near(gate, unit) && (up == nullptr || near(up, unit));
  a.x_direct = aligned(x, 1);
  a.weights_direct = aligned(gate, unit) && (up == nullptr || aligned(up, unit)) && (!wide || a.columns % 8 == 0);
  const size_t item = x->dtype == FL_FLOAT32 ? 4 : 2;
  a.out_vectors = out->strides[1] == 1 && out->strides[0] % 4 == 0 && a.columns % 4 == 0 && IsAligned(out->base, 4 * item);
  return ForDecoderType(x->dtype, [&](auto type) {
    using T = decltype(type);
    if (up != nullptr) return wide ? LaunchLayout<T, true, false>(a, stream) : LaunchLayout<T, true, true>(a, stream);
    return wide ? LaunchLayout<T, false, false>(a, stream) : LaunchLayout<T, false, true>(a, stream);
  });
}

}  // namespace

extern "C" {

int fluidml_hip_gated_matmul(const fl_tensor *x, const fl_tensor *gate, const fl_tensor *up, const fl_tensor *gate_bias, const fl_tensor *up_bias,
                             const fl_tensor *products, int32_t activation, void *stream) {
  FL_CHECK(CheckGated(x, gate, up, gate_bias, up_bias, products, activation));
  return Contract(x, gate, up, gate_bias, up_bias, nullptr, products, activation, AsStream(stream));
}

int fluidml_hip_gated_feed_forward(const fl_tensor *x, const fl_tensor *gate, const fl_tensor *up, const fl_tensor *gate_bias, const fl_tensor *up_bias,
                                   const fl_tensor *down, const fl_tensor *down_bias, const fl_tensor *addend, const fl_tensor *products,
                                   const fl_tensor *out, int32_t activation, void *stream) {
  FL_CHECK(CheckGated(x, gate, up, gate_bias, up_bias, products, activation));
  FL_CHECK(CheckWideView(down));
  if (down->rank != 2) return FL_ERR_RANK;
  const int64_t M = x->shape[0], N = gate->shape[1], O = down->shape[1];
  FL_CHECK(CheckMatrix(down, x->dtype, N, O));
  FL_CHECK(CheckMatrix(out, x->dtype, M, O, true));
  FL_CHECK(CheckOptionalVector(down_bias, x->dtype, O));
  if (addend != nullptr) FL_CHECK(CheckMatrix(addend, x->dtype, M, O));
  FL_CHECK(CheckExtents(M, O));
  FL_CHECK(Contract(x, gate, up, gate_bias, up_bias, nullptr, products, activation, AsStream(stream)));
  return Contract(products, down, nullptr, down_bias, nullptr, addend, out, FL_GATE_IDENTITY, AsStream(stream));
}

}  // extern "C"
