// f8_common.h -- what the kernels and entry points of the 8-bit operators (bof_f8.h) share.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "bof_f8.h"
#include "bof_internal.h"

namespace bof {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef int i32x8 __attribute__((ext_vector_type(8)));

// ---- dense elements -----------------------------------------------------------------
__device__ __forceinline__ float bf16_bits_to_f32(uint32_t b) { return __uint_as_float(b << 16); }
template <int T>
__device__ __forceinline__ float load_dense(const void *p, int64_t i) {
  if constexpr (T == BOF_F32) return ((const float *) p)[i];
  if constexpr (T == BOF_BF16) return bf16_bits_to_f32(((const uint16_t *) p)[i]);
  return (float) ((const _Float16 *) p)[i];
}
// one rounding, to nearest even
template <int T>
__device__ __forceinline__ void store_dense(void *p, int64_t i, float v) {
  if constexpr (T == BOF_F32) ((float *) p)[i] = v;
  else if constexpr (T == BOF_BF16) ((__bf16 *) p)[i] = (__bf16) v;
  else ((_Float16 *) p)[i] = (_Float16) v;
}
constexpr int dense_bytes(int type) { return type == BOF_F32 ? 4 : 2; }

// ---- 8-bit elements and their scales ------------------------------------------------
// Both types end at 0.875 * 2^TOP (448 = 0.875 * 2^9, 57344 = 0.875 * 2^16).
constexpr int f8_top(int f8_type) { return f8_type == BOF_E4M3 ? 9 : 16; }
// the magnitude's bits if it is finite, else 0: what a block's largest magnitude is taken over (magnitudes of floats
// order like their bits)
__device__ __forceinline__ uint32_t finite_magnitude(float v) {
  const uint32_t b = __float_as_uint(v) & 0x7fffffffu;
  return b < 0x7f800000u ? b : 0u;
}
// E8M0 code of the smallest power of two, at least 2^-126, that brings a magnitude (its bits) into the type's range.
// amax = 1.f * 2^(E-127) = (1.f / 2) * 2^(E-126) fits 0.875 * 2^(TOP + e) from e = E - 126 - TOP on, one more where
// 1.f > 1.75.  The codes lie in [1, 247]: a scale and its reciprocal are both normal floats.
template <int F8>
__device__ __forceinline__ uint32_t scale_code(uint32_t amax_bits) {
  const int c = (int) (amax_bits >> 23) + 1 - f8_top(F8) + ((amax_bits & 0x7fffffu) > 0x600000u ? 1 : 0);
  return amax_bits == 0 ? 127u : (uint32_t) max(c, 1);
}
__device__ __forceinline__ float scale_inverse(uint32_t code) { return __uint_as_float((254u - code) << 23); }
// two floats, already divided by their scale, to two bytes (nearest even; a NaN stays NaN, an infinity becomes the
// type's NaN or infinity: the conversion instructions do that)
template <int F8, bool HI>
__device__ __forceinline__ uint32_t f8_pair(float a, float b, uint32_t old) {
  if constexpr (F8 == BOF_E4M3) return (uint32_t) __builtin_amdgcn_cvt_pk_fp8_f32(a, b, (int) old, HI);
  return (uint32_t) __builtin_amdgcn_cvt_pk_bf8_f32(a, b, (int) old, HI);
}
template <int F8>
__device__ __forceinline__ uint32_t f8_quad(float a, float b, float c, float d) {
  return f8_pair<F8, true>(c, d, f8_pair<F8, false>(a, b, 0u));
}

// ---- entry points -------------------------------------------------------------------
// Every launch of a call goes to the stream's device: it becomes the thread's current one for the call's duration.
class LaunchDevice {
 public:
  explicit LaunchDevice(hipStream_t st);
  ~LaunchDevice();
  int status() const { return rc_; }
  // BOF_EINVAL (with a message) unless the device can reach p: its own memory, or host memory that HIP knows
  int reaches(const void *p, const char *call, const char *name);

 private:
  int rc_ = BOF_OK, before_ = 0, dev_ = 0;
};
int refuse(const char *call, const char *why);

}  // namespace bof
