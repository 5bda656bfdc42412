// Shared by the decoder operators (rotary.hip, attention_positions.hip, gated.hip): views that may reach beyond 2^31 elements and the three types
// they compute on.
#ifndef FLUIDML_AMD_CSRC_HIP_DECODER_COMMON_H_
#define FLUIDML_AMD_CSRC_HIP_DECODER_COMMON_H_

#include <type_traits>

#include "fl_common.h"

namespace fl {

// of 256 threads: a grid has fewer than 2^32 threads
constexpr int64_t kMostWorkgroups = (INT64_C(1) << 24) - 1;

inline bool IsDecoderType(int32_t dtype) { return dtype == FL_FLOAT32 || dtype == FL_FLOAT16 || dtype == FL_BFLOAT16; }

// CheckView for these operators: 64-bit offsets, FL_BFLOAT16 among the types
inline int CheckWideView(const fl_tensor *t) {
  if (t == nullptr || t->base == nullptr) return FL_ERR_NULL;
  if (t->rank < 0 || t->rank > kMaxRank) return FL_ERR_RANK;
  if (DtypeSize(t->dtype) == 0 && t->dtype != FL_BFLOAT16) return FL_ERR_DTYPE;
  __int128 span = 0;
  for (int i = 0; i < t->rank; ++i) {
    if (t->shape[i] <= 0 || t->strides[i] < 0) return FL_ERR_SHAPE;
    if (t->shape[i] > FL_DECODER_MAX_EXTENT) return FL_ERR_TOO_LARGE;
    span += static_cast<__int128>(t->shape[i] - 1) * t->strides[i];
    if (span > (static_cast<__int128>(1) << 48)) return FL_ERR_TOO_LARGE;
  }
  return FL_OK;
}

// ... of a result: no two elements in one place along a dim
inline int CheckWideResult(const fl_tensor *t) {
  FL_CHECK(CheckWideView(t));
  for (int i = 0; i < t->rank; ++i) {
    if (t->shape[i] > 1 && t->strides[i] == 0) return FL_ERR_SHAPE;
  }
  return FL_OK;
}

// [n] of type `dtype`, or [n] that is NULL
inline int CheckOptionalVector(const fl_tensor *t, int32_t dtype, int64_t n) {
  if (t == nullptr) return FL_OK;
  FL_CHECK(CheckWideView(t));
  if (t->rank != 1) return FL_ERR_RANK;
  if (t->dtype != dtype) return FL_ERR_DTYPE;
  return t->shape[0] == n ? FL_OK : FL_ERR_SHAPE;
}

// body(a value of the C++ type of `dtype`)
template <typename F>
inline int ForDecoderType(int32_t dtype, F &&body) {
  switch (dtype) {
    case FL_FLOAT32: return body(float{});
    case FL_FLOAT16: return body(static_cast<_Float16>(0));
    case FL_BFLOAT16: return body(static_cast<__bf16>(0.0f));
    default: return FL_ERR_DTYPE;
  }
}

#if defined(__HIPCC__)
// 16 bytes from a lane's own address to 16 * lane bytes behind `to` (the same for all lanes, in LDS), without a register between.
// Not waited for by the compiler: s_waitcnt vmcnt.  (In the host pass the builtin makes a template kernel lose its launch stub.)
__device__ __forceinline__ void LoadToLds(const void *from, void *to) {
#if defined(__HIP_DEVICE_COMPILE__)
  __builtin_amdgcn_global_load_lds(from, (__attribute__((address_space(3))) void *)to, 16, 0, 0);
#endif
}

// body(part of the left operand, part of the right one, whether the product is one of the small ones) for the six products of fl_common.h's
// MfmaParts, so that several sums can take turns: products of one sum after the other wait for each other.
template <typename F>
__device__ __forceinline__ void ForParts(F &&body) {
  using std::integral_constant;
  using Small = std::true_type;
  body(integral_constant<int, 2>{}, integral_constant<int, 0>{}, Small{});
  body(integral_constant<int, 0>{}, integral_constant<int, 2>{}, Small{});
  body(integral_constant<int, 1>{}, integral_constant<int, 1>{}, Small{});
  body(integral_constant<int, 1>{}, integral_constant<int, 0>{}, Small{});
  body(integral_constant<int, 0>{}, integral_constant<int, 1>{}, Small{});
  body(integral_constant<int, 0>{}, integral_constant<int, 0>{}, std::false_type{});
}

// Waits until matrix instructions (of up to 16 passes) have written their results.  The compiler does this where it sees them read in the same basic
// block; across a branch (scores that are capped or not, the end of a loop) it has left it out, and the last results were read
// before they were there.  For the block behind such a branch:
__device__ __forceinline__ void SettleAcrossBranch() {
  asm volatile("s_nop 10");
  __builtin_amdgcn_sched_barrier(0);
}
// ... and for results of this block that are read behind the next branch
template <int N, typename Acc>
__device__ __forceinline__ void Settle(Acc (&acc)[N]) {
#pragma unroll
  for (int n = 0; n < N; ++n) asm volatile("" : "+v"(acc[n]));  // behind the products ..
  asm volatile("s_nop 10");
#pragma unroll
  for (int n = 0; n < N; ++n) asm volatile("" : "+v"(acc[n]));  // .. and before what reads them
}
#endif

}  // namespace fl

#endif  // FLUIDML_AMD_CSRC_HIP_DECODER_COMMON_H_
