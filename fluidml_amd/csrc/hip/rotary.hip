// Rotary positions whose angles are computed where they are used, from the tokens' positions: queries and keys of a layer in one launch.
//   (a, b) -> (a c - b s, b c + a s),  c = amplitude cos(p f_j), s = amplitude sin(p f_j)
// Bound by memory: every value is read once and written once, three operations a value.  A workgroup owns a run of tokens and all their
// heads: it computes the runs' angles once, into LDS, and every head reads them there, so that the 64-bit arithmetic (an exponential and
// the whole turns of p f_j taken off, some 150 instructions) is paid once per token and pair instead of once per value.  The first loads
// are on their way meanwhile.  A thread moves two vectors of up to 16 bytes at a time, the two halves of V pairs.
// bf16, 40 heads of 128 columns: 16384 tokens 53 us (6.3 TB/s read and written; a large copy reaches 5.1), 64 tokens 5.2 us, which is a launch and
// one chain of positions, exponential and sine.
#include <cmath>

#include "decoder_common.h"

using namespace fl;

namespace {

constexpr int kRotaryThreads = 256;
constexpr int kRotaryItems = 4;      // items a thread has in flight
constexpr int kRotaryAngles = 1024;  // pairs whose angles a workgroup keeps

struct RotaryTensor {
  const void *x;
  void *out;
  int64_t x_strides[4], out_strides[4];  // batch, head, token, column
};

struct RotaryArgs {
  RotaryTensor t[2];
  const void *positions;
  int64_t position_strides[2];  // batch, token
  FastDiv length, items, chunks;  // tokens of a sequence; items of a token; chunks of a head
  uint32_t tokens, heads0, rotated_chunks, half;
  int32_t wide_positions, group, interleaved, scaling, streaming;
  double log_step;   // ln f_(j+1) - ln f_j
  double share_at, share_slope;  // the share of f_j that stays is clamp((t_j or j - share_at) * share_slope)
  double turns;      // t_j = turns * f_j
  double inv_factor;
  float amplitude;
};

template <typename T, int V>
using RotaryVec = T __attribute__((ext_vector_type(V)));

__device__ __forceinline__ float2 RotaryAngle(const RotaryArgs &a, uint32_t token, uint32_t j) {
  uint32_t b, s;
  a.length.DivMod(token, b, s);
  const int64_t at = b * a.position_strides[0] + s * a.position_strides[1];
  const double p = a.wide_positions ? static_cast<double>(static_cast<const int64_t *>(a.positions)[at])
                                    : static_cast<double>(static_cast<const int32_t *>(a.positions)[at]);
  double f = exp(a.log_step * j);
  if (a.scaling == FL_ROTARY_LINEAR) f *= a.inv_factor;
  if (a.scaling == FL_ROTARY_WAVELENGTH || a.scaling == FL_ROTARY_DIMENSION) {
    const double of = a.scaling == FL_ROTARY_WAVELENGTH ? a.turns * f : static_cast<double>(j);
    const double stays = fmin(fmax((of - a.share_at) * a.share_slope, 0.0), 1.0);
    f *= stays + (1.0 - stays) * a.inv_factor;
  }
  // whole turns come off in 64 bits; what is left is at most half a turn and needs 32
  const double turns = p * (f * 0.15915494309189533577);
  float sine, cosine;
  sincospif(2.0f * static_cast<float>(turns - rint(turns)), &sine, &cosine);
  return make_float2(a.amplitude * cosine, a.amplitude * sine);
}

// what a thread moves at a time: V pairs, or V columns that are copied
template <typename T, int V>
struct RotaryItem {
  RotaryVec<T, V> first, second;
  T *to;
  int64_t step;   // elements from the first vector to the second, in the result
  uint32_t pair;  // where the item's angles start; ~0: columns that are copied
};

template <typename T, int V>
__device__ __forceinline__ RotaryItem<T, V> LoadItem(const RotaryArgs &a, uint32_t token0, uint32_t item) {
  using Vec = RotaryVec<T, V>;
  RotaryItem<T, V> r;
  uint32_t t, rest, head, chunk, b, s;
  a.items.DivMod(item, t, rest);
  a.chunks.DivMod(rest, head, chunk);
  a.length.DivMod(token0 + t, b, s);
  const bool other = head >= a.heads0;
  const RotaryTensor &m = a.t[other];
  if (other) head -= a.heads0;
  const bool rotated = chunk < a.rotated_chunks;
  const uint32_t column = !rotated ? 2 * a.half + (chunk - a.rotated_chunks) * V : a.interleaved ? chunk * 2 * V : chunk * V;
  const uint32_t next = !rotated ? 0 : a.interleaved ? V : a.half;
  const T *from = static_cast<const T *>(m.x) + b * m.x_strides[0] + head * m.x_strides[1] + s * m.x_strides[2] + column * m.x_strides[3];
  r.to = static_cast<T *>(m.out) + b * m.out_strides[0] + head * m.out_strides[1] + s * m.out_strides[2] + column * m.out_strides[3];
  r.step = next * m.out_strides[3];
  r.pair = rotated ? t * a.half + chunk * V : ~0u;
  r.first = *reinterpret_cast<const Vec *>(from);
  r.second = *reinterpret_cast<const Vec *>(from + next * m.x_strides[3]);  // (columns that are copied: the same again)
  return r;
}

template <typename T, int V>
__device__ __forceinline__ void StoreVec(T *to, RotaryVec<T, V> v, bool streaming) {
  RotaryVec<T, V> *const at = reinterpret_cast<RotaryVec<T, V> *>(to);
  if constexpr (sizeof(v) >= 4) {
    StoreMaybeStreaming(at, v, streaming);
  } else {
    *at = v;
  }
}

template <typename T, int V>
__device__ __forceinline__ void TurnItem(const RotaryArgs &a, const RotaryItem<T, V> &item, const float2 *angles) {
  if (item.pair == ~0u) {
    StoreVec<T, V>(item.to, item.first, a.streaming);
    return;
  }
  RotaryVec<T, V> u = item.first, w = item.second;
  angles += item.pair;
  if (V > 1 && a.interleaved) {
#pragma unroll
    for (int e = 0; e < V; e += 2) {
      const float u0 = static_cast<float>(u[e]), u1 = static_cast<float>(u[(e + 1) % V]), w0 = static_cast<float>(w[e]), w1 = static_cast<float>(w[(e + 1) % V]);
      const float2 c = angles[e / 2], d = angles[V / 2 + e / 2];
      u[e] = static_cast<T>(u0 * c.x - u1 * c.y);
      u[(e + 1) % V] = static_cast<T>(u1 * c.x + u0 * c.y);
      w[e] = static_cast<T>(w0 * d.x - w1 * d.y);
      w[(e + 1) % V] = static_cast<T>(w1 * d.x + w0 * d.y);
    }
  } else {
#pragma unroll
    for (int e = 0; e < V; ++e) {
      const float u0 = static_cast<float>(u[e]), w0 = static_cast<float>(w[e]);
      const float2 c = angles[e];
      u[e] = static_cast<T>(u0 * c.x - w0 * c.y);
      w[e] = static_cast<T>(w0 * c.x + u0 * c.y);
    }
  }
  StoreVec<T, V>(item.to, u, a.streaming);
  StoreVec<T, V>(item.to + item.step, w, a.streaming);
}

template <typename T, int V>
__global__ __launch_bounds__(kRotaryThreads) void RotaryPositionsKernel(const RotaryArgs a) {
  __shared__ float2 angles[kRotaryAngles];
  const uint32_t token0 = blockIdx.x * a.group, n_tokens = min(static_cast<uint32_t>(a.group), a.tokens - token0);
  const uint32_t n_items = n_tokens * a.items.divisor, last = n_items - 1;
  RotaryItem<T, V> items[kRotaryItems];
  // (no branch around a load: an item that is not there is the last one again, and not stored)
#pragma unroll
  for (int i = 0; i < kRotaryItems; ++i) items[i] = LoadItem<T, V>(a, token0, min(threadIdx.x + i * kRotaryThreads, last));
  for (uint32_t i = threadIdx.x; i < n_tokens * a.half; i += kRotaryThreads) {
    const uint32_t t = i / a.half;
    angles[i] = RotaryAngle(a, token0 + t, i - t * a.half);
  }
  __syncthreads();
  for (uint32_t item = threadIdx.x;;) {
#pragma unroll
    for (int i = 0; i < kRotaryItems; ++i) {
      if (item + i * kRotaryThreads <= last) TurnItem<T, V>(a, items[i], angles);
    }
    item += kRotaryItems * kRotaryThreads;
    if (item > last) break;
#pragma unroll
    for (int i = 0; i < kRotaryItems; ++i) items[i] = LoadItem<T, V>(a, token0, min(item + i * kRotaryThreads, last));
  }
}

int CheckPlan(const fl_rotary_plan *p, int64_t columns) {
  if (p == nullptr) return FL_ERR_NULL;
  if (p->interleaved != 0 && p->interleaved != 1) return FL_ERR_ATTR;
  if (p->dims < 2 || p->dims % 2 != 0 || p->dims > columns) return FL_ERR_ATTR;
  if (p->dims > FL_ROTARY_MAX_DIMS) return FL_ERR_UNSUPPORTED;
  if (!(p->base > 1.0) || !std::isfinite(p->base) || !std::isfinite(static_cast<float>(p->amplitude))) return FL_ERR_ATTR;
  if (p->scaling < FL_ROTARY_PLAIN || p->scaling > FL_ROTARY_DIMENSION) return FL_ERR_ATTR;
  if (p->scaling != FL_ROTARY_PLAIN && (!(p->factor >= 1.0) || !std::isfinite(p->factor))) return FL_ERR_ATTR;
  if (p->scaling == FL_ROTARY_WAVELENGTH || p->scaling == FL_ROTARY_DIMENSION) {
    if (!(p->original_length > 0.0) || !std::isfinite(p->original_length)) return FL_ERR_ATTR;
    if (!(p->low > 0.0) || !(p->high > p->low) || !std::isfinite(p->high)) return FL_ERR_ATTR;
  }
  return FL_OK;
}

bool Multiple(const fl_tensor *t, int v, size_t item) {
  if (!IsAligned(t->base, v * item)) return false;
  for (int i = 0; i < 3; ++i) {
    if (t->shape[i] > 1 && t->strides[i] % v != 0) return false;
  }
  return t->strides[3] == 1 || t->shape[3] == 1;
}

int Rotate(int n, const fl_tensor *const *x, const fl_tensor *const *out, const fl_tensor *positions, const fl_rotary_plan *plan, void *stream) {
  for (int i = 0; i < n; ++i) {
    FL_CHECK(CheckWideView(x[i]));
    FL_CHECK(CheckWideResult(out[i]));
    if (x[i]->rank != 4 || out[i]->rank != 4) return FL_ERR_RANK;
    if (!IsDecoderType(x[i]->dtype) || x[i]->dtype != x[0]->dtype || out[i]->dtype != x[0]->dtype) return FL_ERR_DTYPE;
    if (!SameShape(x[i], out[i])) return FL_ERR_SHAPE;
    for (int d : {0, 2, 3}) {
      if (x[i]->shape[d] != x[0]->shape[d]) return FL_ERR_SHAPE;
    }
  }
  const int64_t B = x[0]->shape[0], S = x[0]->shape[2], D = x[0]->shape[3];
  FL_CHECK(CheckWideView(positions));
  if (positions->dtype != FL_INT32 && positions->dtype != FL_INT64) return FL_ERR_DTYPE;
  if (positions->rank != 1 && positions->rank != 2) return FL_ERR_RANK;
  if (positions->shape[positions->rank - 1] != S) return FL_ERR_SHAPE;
  if (positions->rank == 2 && positions->shape[0] != B && positions->shape[0] != 1) return FL_ERR_SHAPE;
  FL_CHECK(CheckPlan(plan, D));

  RotaryArgs a;
  std::memset(&a, 0, sizeof(a));
  const size_t item = x[0]->dtype == FL_FLOAT32 ? 4 : 2;
  const int64_t half = plan->dims / 2;
  int v = static_cast<int>(16 / item);
  auto fits = [&](int w) {
    bool ok = half % w == 0 && D % w == 0;
    for (int i = 0; i < n; ++i) ok = ok && Multiple(x[i], w, item) && Multiple(out[i], w, item);
    return ok;
  };
  while (v > 1 && !fits(v)) v /= 2;

  int64_t heads = 0;
  size_t bytes = 0;
  bool in_place = true;
  for (int i = 0; i < n; ++i) {
    a.t[i].x = x[i]->base;
    a.t[i].out = out[i]->base;
    bool same = x[i]->base == out[i]->base;
    for (int d = 0; d < 4; ++d) {
      a.t[i].x_strides[d] = x[i]->strides[d];
      a.t[i].out_strides[d] = out[i]->strides[d];
      same = same && (x[i]->strides[d] == out[i]->strides[d] || x[i]->shape[d] == 1);
    }
    in_place = in_place && same;
    heads += x[i]->shape[1];
    bytes += static_cast<size_t>(B) * S * x[i]->shape[1] * D * item;
  }
  // columns that are only copied need nothing where the result is the operand
  const int64_t rotated = half / v, chunks = rotated + (in_place ? 0 : (D - plan->dims) / v), per_token = heads * chunks;
  if (B * S > INT32_MAX || per_token > INT32_MAX / 8) return FL_ERR_TOO_LARGE;
  // Tokens of a workgroup: one where there are few, so that they spread over the chip; else as many as give each thread four items
  // twice (and as their angles fit), so that the angles and the start of a workgroup are paid for less often.
  int64_t group = 1;
  if (B * S >= 2048) group = std::max<int64_t>(1, std::min<int64_t>(2 * kRotaryItems * kRotaryThreads / per_token, kRotaryAngles / half));
  a.positions = positions->base;
  a.wide_positions = positions->dtype == FL_INT64;
  a.position_strides[0] = positions->rank == 2 && positions->shape[0] == B ? positions->strides[0] : 0;
  a.position_strides[1] = positions->strides[positions->rank - 1];
  a.length = FastDiv(static_cast<uint32_t>(S));
  a.items = FastDiv(static_cast<uint32_t>(per_token));
  a.chunks = FastDiv(static_cast<uint32_t>(chunks));
  a.tokens = static_cast<uint32_t>(B * S);
  a.heads0 = static_cast<uint32_t>(x[0]->shape[1]);
  a.rotated_chunks = static_cast<uint32_t>(rotated);
  a.half = static_cast<uint32_t>(half);
  a.group = static_cast<int32_t>(group);
  a.interleaved = plan->interleaved;
  a.scaling = plan->scaling;
  a.streaming = StreamingOutput(bytes);
  const double R = static_cast<double>(plan->dims), two_pi = 6.283185307179586477;
  double log_base = std::log(plan->base);
  if (plan->scaling == FL_ROTARY_BASE && plan->dims > 2) log_base += std::log(plan->factor) * R / (R - 2.0);
  a.log_step = -2.0 * log_base / R;
  a.inv_factor = plan->scaling == FL_ROTARY_PLAIN ? 1.0 : 1.0 / plan->factor;
  if (plan->scaling == FL_ROTARY_WAVELENGTH) {
    a.turns = plan->original_length / two_pi;
    a.share_at = plan->low;
    a.share_slope = 1.0 / (plan->high - plan->low);
  } else if (plan->scaling == FL_ROTARY_DIMENSION) {
    const double from = std::max(0.0, std::floor(R * std::log(plan->original_length / (two_pi * plan->high)) / (2.0 * log_base)));
    const double to = std::min(R - 1.0, std::ceil(R * std::log(plan->original_length / (two_pi * plan->low)) / (2.0 * log_base)));
    a.share_slope = -1.0 / std::max(to - from, 0.001);  // the share that stays falls from one at `from` to none at `to`
    a.share_at = from - 1.0 / a.share_slope;
  }
  a.amplitude = static_cast<float>(plan->amplitude);

  if ((B * S + group - 1) / group > kMostWorkgroups) return FL_ERR_TOO_LARGE;
  const dim3 grid(static_cast<uint32_t>((B * S + group - 1) / group));
  FL_CHECK(ForDecoderType(x[0]->dtype, [&](auto type) {
    using T = decltype(type);
    auto launch = [&](auto width) {
      FL_LAUNCH((RotaryPositionsKernel<T, decltype(width)::value>), grid, dim3(kRotaryThreads), 0, AsStream(stream), a);
      return FL_OK;
    };
    if constexpr (sizeof(T) == 2) {
      if (v == 8) return launch(std::integral_constant<int, 8>{});
    }
    if (v == 4) return launch(std::integral_constant<int, 4>{});
    if (v == 2) return launch(std::integral_constant<int, 2>{});
    return launch(std::integral_constant<int, 1>{});
  }));
  return LaunchStatus();
}

}  // namespace

extern "C" {

int fluidml_hip_rotary_positions(const fl_tensor *x, const fl_tensor *positions, const fl_tensor *out, const fl_rotary_plan *plan, void *stream) {
  return Rotate(1, &x, &out, positions, plan, stream);
}

int fluidml_hip_rotary_positions_pair(const fl_tensor *x0, const fl_tensor *out0, const fl_tensor *x1, const fl_tensor *out1, const fl_tensor *positions,
                                      const fl_rotary_plan *plan, void *stream) {
  const fl_tensor *x[2] = {x0, x1}, *out[2] = {out0, out1};
  return Rotate(2, x, out, positions, plan, stream);
}

}  // extern "C"
