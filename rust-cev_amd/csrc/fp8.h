// What the kernels of a product of e4m3 rows and weights share (fp8_linear.hip
// plans a call and launches them, fp8_tile.hip holds the kernel for many rows).
#pragma once
#include "cev_internal.h"
#include "fp8_device.h"

struct Fp8Args {
  const void* x;          // rows
  const uint8_t* xs;      // their scales (e4m3 rows)
  const uint8_t* w;       // packed weight
  const uint8_t* ws;      // its scales: f32, or bytes in rows of ws_pitch
  void* out;
  uint8_t* out_s;
  float* part;            // sums over parts of the columns, nullptr: none
  int64_t t, x_st, out_st, n;
  int32_t k, kb;          // columns, blocks of them
  int32_t groups;         // groups of 32 weight rows
  int32_t parts, blocks_part;
  int32_t ws_pitch;       // scales of a group
};

// The kernel for many rows, 16 tt of them a workgroup (tt 4 or 8, with scales
// in e8m0 also 16; exact, for f32 outputs: 4) of one team of waves or two (tt
// 4, with f32 scales also 8).
int32_t fp8_launch_tile(const Fp8Args& a, int tt, int teams, bool exact, bool e8m0, bool gate_up, hipStream_t s);

__device__ __forceinline__ f32x4 fp8_mfma(const i32x8& a, const i32x8& b, const f32x4& c, int sa, int sb) {
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b, c, 0, 0, 0, sa, 0, sb);
}

// 32 values of a lane in bf16, which holds e4m3's exactly, times `by`, a power of
// two: 8 for each of four products.
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
__device__ __forceinline__ bf16x8 fp8_widen(int lo, int hi, float by = 1.0f) {
  const bf16x2 a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((unsigned)lo, by, false), b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((unsigned)lo, by, true);
  const bf16x2 c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((unsigned)hi, by, false), d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((unsigned)hi, by, true);
  return bf16x8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

// A weight's scale as 2^(code - 127) times the rest: 1 of an e8m0 byte, of an
// f32 (whose exponent the matrix cores then apply) its significand, 1 to 2, so
// that a product under the code alone leaves f32's range only where the result
// does.  0 keeps code 0; infinities and NaN keep themselves as the rest.
struct Fp8Scale {
  int code;
  float rest;
};
template <bool E8M0>
__device__ __forceinline__ Fp8Scale fp8_scale(uint32_t s) {
  if constexpr (E8M0) return {(int)s, s == 255 ? __builtin_nanf("") : 1.0f};
  const int code = min((int)(s >> 23 & 255), 254);
  return {code, __builtin_ldexpf(__uint_as_float(s), 127 - code)};
}

// A row's scale 2^e in two: `values` widens the row with, 2^-100 to 2^100, so
// that bf16 holds them and f32 the sums of their products exactly, and 2^rest
// goes to the weight's scale (code 255: NaN).
struct Fp8RowScale {
  float values;
  int rest;
  bool nan;
};
__device__ __forceinline__ Fp8RowScale fp8_row_scale(int code) {
  const int c = min(max(code, 27), 227);
  return {__uint_as_float((uint32_t)c << 23), code - c, code == 255};
}
// What multiplies such a sum: in range wherever the result is.  (More than 127
// comes with values of 2^100: infinite, but for a sum of 0.)
__device__ __forceinline__ float fp8_factor(const Fp8RowScale& row, const Fp8Scale& w) {
  const float f = __builtin_ldexpf(w.rest, min(w.code - 127 + row.rest, 127));
  return row.nan ? __builtin_nanf("") : f;
}

__device__ __forceinline__ i32x8 fp8_join(const u32x4_t& a, const u32x4_t& b) {
  return i32x8{(int)a[0], (int)a[1], (int)a[2], (int)a[3], (int)b[0], (int)b[1], (int)b[2], (int)b[3]};
}

// Four neighbouring columns of a row of the output; the row's last ones and
// rows that are not aligned to four go one by one.
template <typename O>
__device__ __forceinline__ void fp8_store4(O* row, int64_t n, int64_t col, const f32x4& v) {
  O* const p = row + col;
  if (col + 4 <= n && ((uintptr_t)p & (4 * sizeof(O) - 1)) == 0) {
    if constexpr (sizeof(O) == 2)
      *(u32x2_t*)p = u32x2_t{(uint32_t)bf16_bits(v[0]) | (uint32_t)bf16_bits(v[1]) << 16, (uint32_t)bf16_bits(v[2]) | (uint32_t)bf16_bits(v[3]) << 16};
    else
      *(f32x4*)p = v;
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (col + i < n) p[i] = (O)v[i];
  }
}

// silu(g) u in f32, by the hardware's exp2 and reciprocal: within 2^-20 of the
// value, and below g = 0 within |g| 2^-23 more (the exponent's own rounding);
// e4m3 keeps 4 bits of it.
__device__ __forceinline__ float fp8_swiglu(float g, float u) {
  return g * __builtin_amdgcn_rcpf(1.0f + fast_exp2(-1.44269504f * g)) * u;
}
