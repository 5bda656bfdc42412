// The gated feed-forward block: products = act(x . gate + gate_bias) * (x . up + up_bias), out = products . down + down_bias + addend.
#include <cmath>

#include "decoder_common.h"

using namespace fl;

namespace {

struct GatedArgs {
  const void *x, *gate, *up, *gate_bias, *up_bias, *addend;
  void *out;
  int64_t x_strides[2], gate_strides[2], up_strides[2], out_strides[2], addend_strides[2], gate_bias_stride, up_bias_stride;
  int32_t rows, depth, columns, activation;
};

__device__ __forceinline__ float Activated(int activation, float v) {
  switch (activation) {
    case FL_GATE_SILU: return v / (1.0f + expf(-v));
    case FL_GATE_GELU: return 0.5f * v * (1.0f + erff(v * 0.70710678118654752f));
    case FL_GATE_GELU_TANH: return 0.5f * v * (1.0f + tanhf(0.79788456080286536f * (v + 0.044715f * v * v * v)));
    case FL_GATE_RELU: return v != v ? v : fmaxf(v, 0.0f);
    case FL_GATE_SIGMOID: return 1.0f / (1.0f + expf(-v));
    default: return v;
  }
}

// A thread per result.  GATED: two sums and their product; else one sum, a bias and an addend.
template <typename T, bool GATED>
__global__ __launch_bounds__(256) void GatedSimpleKernel(const GatedArgs a) {
  const int64_t n = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x, m = blockIdx.y;
  if (n >= a.columns) return;
  const T *const x = static_cast<const T *>(a.x) + m * a.x_strides[0];
  const T *const gate = static_cast<const T *>(a.gate) + n * a.gate_strides[1], *const up = static_cast<const T *>(a.up) + n * a.up_strides[1];
  float g = 0.0f, u = 0.0f;
  for (int64_t k = 0; k < a.depth; ++k) {
    const float v = static_cast<float>(x[k * a.x_strides[1]]);
    g += v * static_cast<float>(gate[k * a.gate_strides[0]]);
    if constexpr (GATED) u += v * static_cast<float>(up[k * a.up_strides[0]]);
  }
  if (a.gate_bias != nullptr) g += static_cast<float>(static_cast<const T *>(a.gate_bias)[n * a.gate_bias_stride]);
  if constexpr (GATED) {
    if (a.up_bias != nullptr) u += static_cast<float>(static_cast<const T *>(a.up_bias)[n * a.up_bias_stride]);
    g = Activated(a.activation, g) * u;
  } else if (a.addend != nullptr) {
    g += static_cast<float>(static_cast<const T *>(a.addend)[m * a.addend_strides[0] + n * a.addend_strides[1]]);
  }
  static_cast<T *>(a.out)[m * a.out_strides[0] + n * a.out_strides[1]] = static_cast<T>(g);
}

int CheckMatrix(const fl_tensor *t, int32_t dtype, int64_t rows, int64_t columns, bool result = false) {
  FL_CHECK(result ? CheckWideResult(t) : CheckWideView(t));
  if (t->rank != 2) return FL_ERR_RANK;
  if (t->dtype != dtype) return FL_ERR_DTYPE;
  return t->shape[0] == rows && t->shape[1] == columns ? FL_OK : FL_ERR_SHAPE;
}

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
  return FL_OK;
}

void Set(const fl_tensor *t, int64_t (&strides)[2]) {
  for (int i = 0; i < 2; ++i) strides[i] = t == nullptr ? 0 : t->strides[i];
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
  if (a.rows > 65535) return FL_ERR_TOO_LARGE;
  const dim3 grid((a.columns + 255) / 256, a.rows);
  FL_CHECK(ForDecoderType(x->dtype, [&](auto type) {
    using T = decltype(type);
    if (up != nullptr) {
      FL_LAUNCH((GatedSimpleKernel<T, true>), grid, dim3(256), 0, stream, a);
    } else {
      FL_LAUNCH((GatedSimpleKernel<T, false>), grid, dim3(256), 0, stream, a);
    }
    return FL_OK;
  }));
  return LaunchStatus();
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
  FL_CHECK(Contract(x, gate, up, gate_bias, up_bias, nullptr, products, activation, AsStream(stream)));
  return Contract(products, down, nullptr, down_bias, nullptr, addend, out, FL_GATE_IDENTITY, AsStream(stream));
}

}  // extern "C"
