// Rows and weights in e4m3 with a power-of-two scale for each block of 128
// values, on the device.
//
// A block whose largest finite magnitude is a has the scale 2^e, e the least
// integer >= -127 with a <= 448 * 2^e (448 = 1.75 * 2^8 is e4m3's largest
// value).  With a = 1.m * 2^(E - 127) in f32 that is e + 127 = E - 8, one more
// where 1.m > 1.75: adding 0x1fffff to the bits carries into E for exactly
// those m.  A power of two costs e4m3 no significant bit, x * 2^-e is exact
// in f32 (far below the block's largest value it may be subnormal, which
// rounds to 0 in e4m3 either way), and the matrix cores take the scale as it
// is stored: e + 127 in a byte (e8m0).
#pragma once
#include <initializer_list>

#include "cev_device.h"
#include "cev_internal.h"

constexpr int kFp8Block = 128;    // values of a row under one scale
constexpr int kFp8Group = 32;     // weight rows of one matrix-core operand
constexpr int kFp8GroupBytes = kFp8Group * kFp8Block;
constexpr int kFp8TileGroups = 8;  // weight rows are padded to 8 groups

// A launch counts its threads in 32 bits.
inline bool fp8_grid_fits(int64_t grid, int threads) { return grid <= (int64_t)(UINT32_MAX / (uint32_t)threads); }

// Whether a call's outputs overlap neither each other nor an input.
inline bool fp8_apart(std::initializer_list<CevRows> outs, std::initializer_list<CevRows> ins) {
  for (const CevRows& o : outs) {
    for (const CevRows& other : outs)
      if (&o < &other && cev_overlap(&o, &other)) return false;
    for (const CevRows& in : ins)
      if (cev_overlap(&o, &in)) return false;
  }
  return true;
}

typedef uint32_t u32x4_t __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2_t __attribute__((ext_vector_type(2)));
typedef int i32x8 __attribute__((ext_vector_type(8)));

// |x| as an integer that orders like it; 0 where x is not finite.
__device__ __forceinline__ uint32_t fp8_size(float x) {
  const uint32_t u = __float_as_uint(x) & 0x7fffffffu;
  return u < 0x7f800000u ? u : 0u;
}

// The scale's byte for a block whose largest size is `top`, and the factor
// 2^-e that goes with it.
__device__ __forceinline__ uint32_t fp8_code(uint32_t top) {
  const int c = (int)((top + 0x1fffffu) >> 23) - 8;
  return (uint32_t)(c > 0 ? c : 0);
}
__device__ __forceinline__ float fp8_inverse(uint32_t code) { return __uint_as_float((254u - code) << 23); }

// Four values, scaled, as e4m3 bytes (nearest even; what is not finite
// becomes NaN).
__device__ __forceinline__ uint32_t fp8_pack4(float a, float b, float c, float d) {
  int w = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
  return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(c, d, w, true);
}

// The largest of 16 adjacent lanes' values, in all of them.
__device__ __forceinline__ uint32_t max_of_16(uint32_t v) {
  v = max(v, dpp_u<0xB1>(v));   // lane ^ 1
  v = max(v, dpp_u<0x4E>(v));   // lane ^ 2
  v = max(v, dpp_u<0x141>(v));  // the other four of eight lanes (half-row mirror)
  return max(v, dpp_u<0x140>(v));  // the other eight (row mirror)
}

// Eight elements of a row at p, of which `have` lie within it (the others
// are 0): two 16-byte loads of f32, one of bf16, single ones at a row's end.
template <typename T>
__device__ __forceinline__ void load8(const T* p, int have, float* v) {
  if (have >= 8) {
    if constexpr (sizeof(T) == 2) {
      const u32x4_t c = *(const u32x4_t*)p;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        v[2 * i] = __uint_as_float(c[i] << 16);
        v[2 * i + 1] = __uint_as_float(c[i] & 0xffff0000u);
      }
    } else {
      const f32x4 a = *(const f32x4*)p, b = *(const f32x4*)(p + 4);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        v[i] = a[i];
        v[4 + i] = b[i];
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = i < have ? (float)p[i] : 0.0f;
  }
}

// 16 adjacent lanes' 8 values each, one block: its largest size.
__device__ __forceinline__ uint32_t fp8_top16(const float* v) {
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) top = max(top, __float_as_uint(v[i]) & 0x7fffffffu);
  if (top >= 0x7f800000u) {  // (what is not finite does not count)
    top = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) top = max(top, fp8_size(v[i]));
  }
  return max_of_16(top);
}

// The lane's 8 bytes under the block's scale.
__device__ __forceinline__ u32x2_t fp8_pack8(const float* v, uint32_t code) {
  const float f = fp8_inverse(code);
  return u32x2_t{fp8_pack4(v[0] * f, v[1] * f, v[2] * f, v[3] * f), fp8_pack4(v[4] * f, v[5] * f, v[6] * f, v[7] * f)};
}

// Both.
__device__ __forceinline__ u32x2_t fp8_block16(const float* v, uint32_t& code) {
  code = fp8_code(fp8_top16(v));
  return fp8_pack8(v, code);
}
