// Eight values on their way to MXFP4: what the quantisation of weights, activations and a cache's keys and values share.
#pragma once
#include "common.h"

namespace tllm {

typedef __attribute__((__vector_size__(4 * sizeof(unsigned)))) unsigned u32x4;

template <class T>
struct Eight;                        // eight values as loaded; the largest of their magnitudes as an fp32's bits; eight codes
template <>
struct Eight<bf16> {
  u32x4 v;
  __device__ void load(const void* p) { v = *static_cast<const u32x4*>(p); }
  __device__ unsigned largest() const {
    unsigned m = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) m = max(m, max(v[i] << 16 & 0x7fff0000u, v[i] & 0x7fff0000u));
    return m;
  }
  template <int I>
  __device__ unsigned pair(unsigned old, float scale) const {
    const unsigned two = v[I];       // (a scalar of its own: __builtin_bit_cast of a vector's element takes element 0 with this compiler)
    return __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(old, __builtin_bit_cast(bf16x2, two), scale, I);
  }
};
template <>
struct Eight<_Float16> {
  typedef __attribute__((__vector_size__(2 * sizeof(_Float16)))) _Float16 f16x2;
  u32x4 v;
  __device__ void load(const void* p) { v = *static_cast<const u32x4*>(p); }
  __device__ unsigned largest() const {
    unsigned m = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) m = max(m, max(v[i] & 0x7fffu, v[i] >> 16 & 0x7fffu));
    return __builtin_bit_cast(unsigned, static_cast<float>(__builtin_bit_cast(_Float16, static_cast<unsigned short>(m))));
  }
  template <int I>
  __device__ unsigned pair(unsigned old, float scale) const {
    const unsigned two = v[I];
    return __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(old, __builtin_bit_cast(f16x2, two), scale, I);
  }
};
template <>
struct Eight<float> {
  f32x4 v[2];
  __device__ void load(const void* p) {
    v[0] = static_cast<const f32x4*>(p)[0];
    v[1] = static_cast<const f32x4*>(p)[1];
  }
  __device__ unsigned largest() const {
    unsigned m = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float one = v[i / 4][i % 4];
      m = max(m, __builtin_bit_cast(unsigned, one) & 0x7fffffffu);
    }
    return m;
  }
  template <int I>
  __device__ unsigned pair(unsigned old, float scale) const { return __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(old, v[I / 2][I % 2 * 2], v[I / 2][I % 2 * 2 + 1], scale, I); }
};

// The eight values' codes and the scale byte of their block of 32, which four neighbouring lanes share (blocks begin at lanes that are
// multiples of four, all four of them active). The maximum is one of the values' bits: without the sign they order as integers, and the
// exponent field less 2 is the scale byte; a field of 255 -- a NaN or an infinity in the block -- gives 255 and codes of 0.
template <class T>
__device__ __forceinline__ unsigned mx_quantize8(const Eight<T>& e, unsigned* scale_byte) {
  unsigned m = e.largest();
  m = max(m, static_cast<unsigned>(__builtin_amdgcn_update_dpp(0, static_cast<int>(m), 0xB1, 0xf, 0xf, true)));   // lane ^ 1
  m = max(m, static_cast<unsigned>(__builtin_amdgcn_update_dpp(0, static_cast<int>(m), 0x4E, 0xf, 0xf, true)));   // lane ^ 2
  const unsigned field = m >> 23, byte = field == 255 ? 255 : field > 2 ? field - 2 : 0;
  const float scale = __builtin_bit_cast(float, byte << 23);                 // (a field of 0 is 2^-127 to the conversion)
  unsigned codes = e.template pair<0>(0u, scale);
  codes = e.template pair<1>(codes, scale);
  codes = e.template pair<2>(codes, scale);
  codes = e.template pair<3>(codes, scale);
  *scale_byte = byte;
  return field == 255 ? 0 : codes;
}

}  // namespace tllm
