// Attention whose scores and masks go by positions (fl_attention_scores).
#include <cmath>

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
  int32_t batch, heads, kv_heads, group, queries, keys, columns, causal, window;
  float scale, cap;
};

// One wave per query and head: 64 keys at a time, a lane a key; then the weights go around and a lane is a column.
template <typename T>
__global__ __launch_bounds__(64) void AttentionSimpleKernel(const AttentionArgs a) {
  __shared__ float q[FL_ATTENTION_MAX_HEAD];
  const int i = blockIdx.x, h = blockIdx.y, b = blockIdx.z, lane = threadIdx.x;
  auto clamped = [&](const int32_t *p, int64_t stride, int32_t most) { return p == nullptr ? most : min(max(p[b * stride], 0), most); };
  const int n_queries = clamped(a.query_lengths, a.query_length_stride, a.queries), n_keys = clamped(a.key_lengths, a.key_length_stride, a.keys);
  if (i >= n_queries) return;
  const int prefix = a.prefix_lengths == nullptr ? 0 : a.prefix_lengths[b * a.prefix_stride];
  const int64_t at = (a.query_starts == nullptr ? n_keys - n_queries : static_cast<int64_t>(a.query_starts[b * a.query_start_stride])) + i;
  const T *const k = static_cast<const T *>(a.k.base) + b * a.k.strides[0] + (h / a.group) * a.k.strides[1];
  const T *const v = static_cast<const T *>(a.v.base) + b * a.v.strides[0] + (h / a.group) * a.v.strides[1];
  const T *const from = static_cast<const T *>(a.q.base) + b * a.q.strides[0] + h * a.q.strides[1] + i * a.q.strides[2];
  for (int d = lane; d < a.columns; d += 64) q[d] = static_cast<float>(from[d * a.q.strides[3]]);
  __syncthreads();
  const float slope = a.slopes == nullptr ? 0.0f : a.slopes[h * a.slope_stride];
  const int document = a.query_documents == nullptr ? 0 : a.query_documents[b * a.query_document_strides[0] + i * a.query_document_strides[1]];
  float most = -INFINITY, sum = 0.0f, acc[FL_ATTENTION_MAX_HEAD / 64] = {};
  for (int j0 = 0; j0 < n_keys; j0 += 64) {
    const int j = j0 + lane;
    const int64_t distance = at - j;
    bool seen = (!a.causal || distance >= 0) && (a.window == 0 || (distance < a.window && -distance < a.window));
    seen = (seen || j < prefix) && j < n_keys && document >= 0;
    if (seen && a.key_documents != nullptr) seen = a.key_documents[b * a.key_document_strides[0] + j * a.key_document_strides[1]] == document;
    if (!__any(seen)) continue;
    float s = -INFINITY;
    if (seen) {
      s = 0.0f;
      for (int d = 0; d < a.columns; ++d) s += q[d] * static_cast<float>(k[j * a.k.strides[2] + d * a.k.strides[3]]);
      s *= a.scale;
      if (a.cap > 0.0f) s = a.cap * tanhf(s / a.cap);
      if (a.slopes != nullptr) s -= slope * static_cast<float>(distance < 0 ? -distance : distance);
    }
    const float now = fmaxf(most, WaveReduce(s, MaxOp{}));
    const float kept = now == -INFINITY ? 1.0f : expf(most - now);
    const float p = s == -INFINITY ? 0.0f : expf(s - now);
    sum = sum * kept + GroupSum<64>(p);
    most = now;
#pragma unroll
    for (float &x : acc) x *= kept;
    const uint64_t which = __ballot(seen);
    for (uint64_t rest = which; rest != 0; rest &= rest - 1) {
      const int e = __builtin_ctzll(rest);
      const float w = __shfl(p, e);
#pragma unroll
      for (int c = 0; c < FL_ATTENTION_MAX_HEAD / 64; ++c) {
        const int d = c * 64 + lane;
        if (d < a.columns) acc[c] += w * static_cast<float>(v[(j0 + e) * a.v.strides[2] + d * a.v.strides[3]]);
      }
    }
  }
  T *const to = static_cast<T *>(a.out.base) + b * a.out.strides[0] + h * a.out.strides[1] + i * a.out.strides[2];
#pragma unroll
  for (int c = 0; c < FL_ATTENTION_MAX_HEAD / 64; ++c) {
    const int d = c * 64 + lane;
    if (d < a.columns) to[d * a.out.strides[3]] = static_cast<T>(sum == 0.0f ? 0.0f : acc[c] / sum);
  }
}

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
  if (!std::isfinite(static_cast<float>(s->scale)) || !std::isfinite(static_cast<float>(s->cap)) || s->cap < 0.0) return FL_ERR_ATTR;
  if ((s->causal != 0 && s->causal != 1) || s->window < 0) return FL_ERR_ATTR;
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

}  // namespace

extern "C" {

int fluidml_hip_attention_positions_scratch(const fl_tensor *q, const fl_tensor *k, const fl_attention_scores *scores, size_t *bytes) {
  if (bytes == nullptr) return FL_ERR_NULL;
  FL_CHECK(CheckScores(q, k, scores));
  *bytes = 0;
  return FL_OK;
}

int fluidml_hip_attention_positions(const fl_tensor *q, const fl_tensor *k, const fl_tensor *v, const fl_tensor *out, const fl_attention_scores *scores,
                                    void *scratch, size_t scratch_bytes, void *stream) {
  (void)scratch, (void)scratch_bytes;
  FL_CHECK(CheckScores(q, k, scores));
  FL_CHECK(CheckWideView(v));
  FL_CHECK(CheckWideResult(out));
  if (v->rank != 4 || out->rank != 4) return FL_ERR_RANK;
  if (v->dtype != q->dtype || out->dtype != q->dtype) return FL_ERR_DTYPE;
  if (!SameShape(k, v) || !SameShape(q, out)) return FL_ERR_SHAPE;
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
  a.causal = scores->causal;
  // (no two positions are further apart than this, so a wider window is none)
  a.window = static_cast<int32_t>(std::min<int64_t>(scores->window, INT32_MAX));
  a.scale = static_cast<float>(scores->scale);
  a.cap = static_cast<float>(scores->cap);
  if (a.heads > 65535 || a.batch > 65535) return FL_ERR_TOO_LARGE;
  FL_CHECK(ForDecoderType(q->dtype, [&](auto type) {
    FL_LAUNCH(AttentionSimpleKernel<decltype(type)>, dim3(a.queries, a.heads, a.batch), dim3(64), 0, AsStream(stream), a);
    return FL_OK;
  }));
  return LaunchStatus();
}

}  // extern "C"
