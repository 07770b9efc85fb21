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
// Eight neighbours as they lie in memory.  Any alignment of the element type: the loads and stores are 16 bytes wide whatever
// the address (gfx950 takes them unaligned).  `valid` elements exist (any number; the others read as 0 and are not written).
template <int T>
struct Eight {
  u32x4 w[T == BOF_F32 ? 2 : 1];
  __device__ __forceinline__ float at(int e) const {
    if constexpr (T == BOF_F32) return __uint_as_float(w[e >> 2][e & 3]);
    const uint32_t u = w[0][e >> 1];
    if constexpr (T == BOF_BF16) return __uint_as_float(e & 1 ? u & 0xffff0000u : u << 16);
    const uint16_t b = (uint16_t) (e & 1 ? u >> 16 : u);
    return (float) __builtin_bit_cast(_Float16, b);
  }
};
template <int T>
__device__ __forceinline__ Eight<T> load_eight(const void *p, int64_t i, int64_t valid) {
  Eight<T> r;
  constexpr int z = T == BOF_F32 ? 4 : 2;
  const uint8_t *from = (const uint8_t *) p + i * z;
  if (valid >= 8) {
    __builtin_memcpy(&r, from, 8 * z);
  } else {
    r.w[0] = u32x4{0u, 0u, 0u, 0u};
    if constexpr (T == BOF_F32) r.w[1] = r.w[0];
#pragma unroll
    for (int e = 0; e < 8; e++)
      if (e < valid) {
        if constexpr (T == BOF_F32) r.w[e >> 2][e & 3] = ((const uint32_t *) from)[e];
        else r.w[0][e >> 1] |= (uint32_t) ((const uint16_t *) from)[e] << (16 * (e & 1));
      }
  }
  return r;
}
template <int T>
__device__ __forceinline__ void store_eight(void *p, int64_t i, const float (&v)[8], int64_t valid) {
  if (valid >= 8) {
    if constexpr (T == BOF_F32) {
      __builtin_memcpy((float *) p + i, v, 32);
    } else if constexpr (T == BOF_BF16) {
      __bf16 o[8];
#pragma unroll
      for (int e = 0; e < 8; e++) o[e] = (__bf16) v[e];
      __builtin_memcpy((__bf16 *) p + i, o, 16);
    } else {
      _Float16 o[8];
#pragma unroll
      for (int e = 0; e < 8; e++) o[e] = (_Float16) v[e];
      __builtin_memcpy((_Float16 *) p + i, o, 16);
    }
  } else {
#pragma unroll
    for (int e = 0; e < 8; e++)
      if (e < valid) store_dense<T>(p, i + e, v[e]);
  }
}
// eight bytes, of which `valid` are written
__device__ __forceinline__ void store_bytes(uint8_t *p, uint64_t v, int64_t valid) {
  if (valid >= 8) {
    __builtin_memcpy(p, &v, 8);
  } else {
#pragma unroll
    for (int e = 0; e < 8; e++)
      if (e < valid) p[e] = (uint8_t) (v >> (8 * e));
  }
}

// ---- reductions over lanes ----------------------------------------------------------
template <int CTRL>
__device__ __forceinline__ uint32_t lanes(uint32_t v) { return (uint32_t) __builtin_amdgcn_update_dpp(0, (int) v, CTRL, 0xf, 0xf, true); }
// over each 16 neighbouring lanes, for all of them: lane ^ 1, lane ^ 2, then the mirrors of 8 and of 16
__device__ __forceinline__ uint32_t max_of_16(uint32_t m) {
  m = max(m, lanes<0xB1>(m));
  m = max(m, lanes<0x4E>(m));
  m = max(m, lanes<0x141>(m));
  return max(m, lanes<0x140>(m));
}
__device__ __forceinline__ float sum_of_wave(float v) {
  v += __uint_as_float(lanes<0xB1>(__float_as_uint(v)));
  v += __uint_as_float(lanes<0x4E>(__float_as_uint(v)));
  v += __uint_as_float(lanes<0x141>(__float_as_uint(v)));
  v += __uint_as_float(lanes<0x140>(__float_as_uint(v)));
  v += __shfl_xor(v, 16);
  return v + __shfl_xor(v, 32);
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
__device__ __forceinline__ uint32_t scale_code(uint32_t amax_bits, int top) {
  const int c = (int) (amax_bits >> 23) + 1 - top + ((amax_bits & 0x7fffffu) > 0x600000u ? 1 : 0);
  return amax_bits == 0 ? 127u : (uint32_t) max(c, 1);
}
__device__ __forceinline__ float scale_inverse(uint32_t code) { return __uint_as_float((254u - code) << 23); }
// eight floats times inv to eight bytes (nearest even; a NaN stays NaN, an infinity becomes the type's NaN or infinity:
// the conversion instructions do that).  top = f8_top(type) names the type.
__device__ __forceinline__ uint64_t f8_eight(const float (&v)[8], float inv, int top) {
  uint32_t o[2];
#pragma unroll
  for (int h = 0; h < 2; h++) {
    const float a = v[4 * h] * inv, b = v[4 * h + 1] * inv, c = v[4 * h + 2] * inv, d = v[4 * h + 3] * inv;
    if (top == 9) o[h] = (uint32_t) __builtin_amdgcn_cvt_pk_fp8_f32(c, d, __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false), true);
    else o[h] = (uint32_t) __builtin_amdgcn_cvt_pk_bf8_f32(c, d, __builtin_amdgcn_cvt_pk_bf8_f32(a, b, 0, false), true);
  }
  return o[0] | (uint64_t) o[1] << 32;
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
