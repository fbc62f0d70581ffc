// Shared device-side definitions of the MXFP4 kernels (gfx950).
//
// Weight format (OCP Microscaling formats v1.0, MXFP4):
//   w       uint32 [N, K/8], code j of word i is element 8 i + j at bit 4 j
//           (low bits first): E2M1, sign in bit 3, magnitudes 0, 0.5, 1, 1.5,
//           2, 3, 4, 6
//   scales  uint8 [N, K/32], one E8M0 byte e per 32 codes: 2^(e - 127), 255 NaN
//   deq     T(code * 2^(e - 127)), rounded to nearest even (in bf16 always
//           exact but for e at the ends of the range)
//
// gfx950 converts both ways in one instruction per two codes:
// v_cvt_scalef32_pk_{bf16,f16,f32}_fp4 multiplies by the power of two in the
// exponent field of a float (field 0: 2^-127, 255: NaN, the E8M0 reading), and
// v_cvt_scalef32_pk_fp4_* divides by it, rounds to nearest even and saturates
// at 6.  Checked over every code, byte and rounding case of all three types.
#pragma once
#include "stream_tile.cuh"

namespace mq {

typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef int i32x8 __attribute__((ext_vector_type(8)));

// The float whose exponent field is the scale byte e.
__device__ __forceinline__ float mx_scale(uint32_t e) { return __uint_as_float(e << 23); }

template <int DT, int SEL>
__device__ __forceinline__ uint32_t mx_pair(uint32_t w, float s) {
  if constexpr (DT == kBF16)
    return bitcast<uint32_t>(__builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, s, SEL));
  else
    return bitcast<uint32_t>(__builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, s, SEL));
}

// The 8 codes of a word as four packed T pairs.
template <int DT>
__device__ __forceinline__ u32x4 mx_word(uint32_t w, float s) {
  return (u32x4){mx_pair<DT, 0>(w, s), mx_pair<DT, 1>(w, s), mx_pair<DT, 2>(w, s),
                 mx_pair<DT, 3>(w, s)};
}

// Scale byte of a group whose largest magnitude has the bits `top` (of T,
// sign cleared): floor(log2) less E2M1's largest exponent, 2; 255 where top
// is infinite or NaN.  A bf16 subnormal's field is 0 and clamps as it should;
// a half is normalised by its conversion to float.
template <int DT>
__device__ __forceinline__ uint32_t mx_scale_byte(uint32_t top) {
  const float f = DT == kF32 ? __uint_as_float(top) : T16<DT == kF32 ? kBF16 : DT>::to_f32((uint16_t)top);
  const uint32_t field = __float_as_uint(f) >> 23;
  return field == 255 ? 255u : field < 2 ? 0u : field - 2;
}

// Codes SEL of a word from a packed T pair; groups of scale 255 are given
// zero codes by the caller.
template <int DT, int SEL>
__device__ __forceinline__ uint32_t mx_code_pair(uint32_t old, uint32_t v, float s) {
  if constexpr (DT == kBF16)
    return __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(old, bitcast<bf16x2>(v), s, SEL);
  else
    return __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(old, bitcast<f16x2>(v), s, SEL);
}

// Four packed T pairs -> a word of 8 codes.
template <int DT>
__device__ __forceinline__ uint32_t mx_code_word(const u32x4& v, float s) {
  uint32_t w = 0;
  w = mx_code_pair<DT, 0>(w, v[0], s);
  w = mx_code_pair<DT, 1>(w, v[1], s);
  w = mx_code_pair<DT, 2>(w, v[2], s);
  return mx_code_pair<DT, 3>(w, v[3], s);
}

// Largest of two packed pairs of 16-bit magnitudes.
__device__ __forceinline__ uint32_t mx_max2(uint32_t a, uint32_t b) {
  typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
  return bitcast<uint32_t>(__builtin_elementwise_max(bitcast<u16x2>(a), bitcast<u16x2>(b)));
}

// Largest of the four lanes of a quad, in each of them.
__device__ __forceinline__ uint32_t mx_quad_max(uint32_t v) {
  // quad_perm [1,0,3,2], then [2,3,0,1]
  v = max(v, (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0xB1, 0xf, 0xf, true));
  return max(v, (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0x4E, 0xf, 0xf, true));
}

// Scales of an expert or tile as a byte range: [first, first + bytes) of an
// array whose base is 16-byte aligned, as a descriptor from the 16-byte
// boundary before it to the end of the 4-byte word that holds its last byte,
// and in `skew` the bytes before it.
__device__ __forceinline__ __amdgpu_buffer_rsrc_t mx_scale_rsrc(const uint8_t* first,
                                                                int64_t bytes, uint32_t& skew) {
  const uintptr_t a = reinterpret_cast<uintptr_t>(first);
  skew = (uint32_t)(a & 15);
  return wide_rsrc(reinterpret_cast<const void*>(a - skew), (bytes + skew + 3) & ~(int64_t)3);
}

// Whether a grid of n workgroups of `threads` has a launch's 32-bit thread count.
inline bool mx_grid_ok(int64_t n, int64_t threads) { return n <= (int64_t)UINT32_MAX / threads; }

}  // namespace mq
