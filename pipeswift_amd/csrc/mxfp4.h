// The 4-bit KV cache's row and its conversions, for the kernels that write it
// (mxfp4_cache.hip, norm_rope.hip) and read it (mxfp4_cache.hip, mxfp4_attention.hip,
// mxfp4_prefill.hip).
//
// A row is one head of one token's K or V, D elements in groups of 32:
//   [0, D / 2)              codes: element 2 i in the low half of byte i, 2 i + 1 in the high
//   [D / 2, D / 2 + D / 32) scales: byte j stands for 2^(byte - 127), 0xFF for NaN
//   then zeros up to a multiple of 4 bytes.
// A code is E2M1 (sign, two bits of exponent, one of fraction): 0, 0.5, 1, 1.5, 2, 3,
// 4, 6 and their negatives.  A group's scale s is the smallest power of two, 2^-126 at
// least, with max |x| < 7 s (1 for a group of zeros), its codes are x / s rounded to
// nearest, ties to even.  Below 7 the nearest values are 6 and less, so nothing is
// clipped and every value is off by half a step at most: 2^-2 of it, or s / 4 below s.
// (The other usual rule, max |x| < 8 s, has the finer step for a maximum between 6 s
// and 8 s but clips it to 6 s, 2^-2 of the maximum and never recovered.)  A group
// that holds an infinity or a NaN has no scale: it reads as NaN.
//
// v_cvt_scalef32_pk_fp4_* and *_pk_*_fp4 compute exactly this for every scale byte
// (round to nearest even, denormals kept, NaN for 0xFF, and 2^-127 for byte 0, which is handed
// to them as 0.0): checked on all bf16 values and on all codes under all scale bytes.
#pragma once

#include "psk_common.h"

namespace psk_detail {

typedef __bf16 mx_bf16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 mx_f16x2 __attribute__((ext_vector_type(2)));

constexpr int kMxGroup = 32;
constexpr uint32_t kMxNan = 255;

__host__ __device__ constexpr int64_t mx_entry_bytes(int64_t head_size) {
  return (head_size / 2 + head_size / kMxGroup + 3) / 4 * 4;
}

// The scale byte of a group from the bits of its largest |x|.
__device__ __forceinline__ uint32_t mx_scale_byte(uint32_t amax_bits) {
  // a fraction of 1.75 or more carries into the exponent
  const uint32_t e = (amax_bits + 0x200000u) >> 23;
  const uint32_t byte = amax_bits == 0 ? 127u : e > 3u ? e - 2u : 1u;
  return amax_bits >= 0x7F800000u ? kMxNan : byte;
}

__device__ __forceinline__ float mx_scale(uint32_t byte) { return __uint_as_float(byte << 23); }

// Largest |x| of eight elements as float bits; NaN and infinity come out at or above 0x7F800000.
template <int DT>
__device__ __forceinline__ uint32_t mx_amax8(const typename Elt<DT>::Bits (&e)[8]) {
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) m = max(m, __float_as_uint(Elt<DT>::to_f32(e[i])) & 0x7FFFFFFFu);
  return m;
}
// bf16 magnitudes order as integers, two to an instruction.
typedef unsigned short mx_u16x2 __attribute__((ext_vector_type(2)));
__device__ __forceinline__ uint32_t mx_amax8_bf16(u32x4 x) {
  mx_u16x2 m = {0, 0};
#pragma unroll
  for (int i = 0; i < 4; ++i) m = __builtin_elementwise_max(m, __builtin_bit_cast(mx_u16x2, x[i] & 0x7FFF7FFFu));
  return uint32_t(m[0] > m[1] ? m[0] : m[1]) << 16;
}

// The maximum over a quad of lanes (a group: 8 elements a lane).
__device__ __forceinline__ uint32_t mx_quad_max(uint32_t v) {
  v = max(v, uint32_t(__builtin_amdgcn_update_dpp(0, int(v), 0xB1, 0xF, 0xF, false)));  // lanes 1, 0, 3, 2
  return max(v, uint32_t(__builtin_amdgcn_update_dpp(0, int(v), 0x4E, 0xF, 0xF, false)));  // lanes 2, 3, 0, 1
}

// Eight elements (a lane's part of a group whose four lanes are a quad) -> their
// codes and the group's scale byte.
template <int DT>
__device__ __forceinline__ uint32_t mx_quantize8(const typename Elt<DT>::Bits (&e)[8], uint32_t& byte) {
  uint32_t w = 0;
  if constexpr (DT == PSK_DTYPE_BF16) {
    u32x4 x;
    __builtin_memcpy(&x, e, 16);
    byte = mx_scale_byte(mx_quad_max(mx_amax8_bf16(x)));
    const float s = mx_scale(byte);
    mx_bf16x2 p[4];
    __builtin_memcpy(p, e, 16);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(w, p[0], s, 0);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(w, p[1], s, 1);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(w, p[2], s, 2);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(w, p[3], s, 3);
  } else {
    byte = mx_scale_byte(mx_quad_max(mx_amax8<DT>(e)));
    const float s = mx_scale(byte);
    float x[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = Elt<DT>::to_f32(e[i]);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[0], x[1], s, 0);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[2], x[3], s, 1);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[4], x[5], s, 2);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[6], x[7], s, 3);
  }
  return byte == kMxNan ? 0u : w;
}

// Whether any of a group's values (16 code bytes) is NaN or, as 4 and 6 times 2^126 and
// 2 and more times 2^127 are, past the largest finite one.
__device__ __forceinline__ bool mx_not_finite(u32x4 codes, uint32_t byte) {
  if (byte < 253) return false;
  uint32_t four = 0, six = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t high = codes[i] & 0x44444444u;
    four |= high;
    six |= high & (codes[i] << 1);
  }
  return byte == kMxNan || (byte == 254 ? four : six) != 0;
}

// Eight codes -> eight elements.
__device__ __forceinline__ u32x4 mx_bf16x8(uint32_t w, float s) {
  return u32x4{__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, s, 0)),
               __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, s, 1)),
               __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, s, 2)),
               __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, s, 3))};
}
__device__ __forceinline__ u32x4 mx_f16x8(uint32_t w, float s) {
  return u32x4{__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, s, 0)),
               __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, s, 1)),
               __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, s, 2)),
               __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, s, 3))};
}
__device__ __forceinline__ void mx_f32x8(uint32_t w, float s, u32x4& lo, u32x4& hi) {
  const f32x2 a = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, s, 0), b = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, s, 1);
  const f32x2 c = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, s, 2), d = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, s, 3);
  lo = u32x4{__float_as_uint(a.x), __float_as_uint(a.y), __float_as_uint(b.x), __float_as_uint(b.y)};
  hi = u32x4{__float_as_uint(c.x), __float_as_uint(c.y), __float_as_uint(d.x), __float_as_uint(d.y)};
}

// Eight elements of a row at p: one or two 16-byte loads where every row is so
// aligned, else element by element.
template <int DT>
__device__ __forceinline__ void load8(const char* p, bool wide, typename Elt<DT>::Bits (&e)[8]) {
  using Bits = typename Elt<DT>::Bits;
  if (wide) {
#pragma unroll
    for (int i = 0; i < int(sizeof(Bits)) / 2; ++i) {
      const u32x4 x = vload<16>(p + 16 * i);
      __builtin_memcpy(reinterpret_cast<char*>(e) + 16 * i, &x, 16);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) e[i] = reinterpret_cast<const Bits*>(p)[i];
  }
}

// A lane's codes and, from the group's first lane, the scale byte into a row: lane
// `chunk` of the row holds elements 8 chunk .. 8 chunk + 7.  The lane of the row's
// last scale writes the padding.
__device__ __forceinline__ void mx_store8(char* row, int chunk, int head_size, uint32_t codes, uint32_t byte) {
  vstore<4>(row + 4 * chunk, codes);
  if ((chunk & 3) == 0) {
    const int groups = head_size / kMxGroup, g = chunk >> 2;
    char* scales = row + head_size / 2;
    scales[g] = char(byte);
    if (g == groups - 1)
      for (int i = groups; i & 3; ++i) scales[i] = 0;
  }
}

}  // namespace psk_detail
