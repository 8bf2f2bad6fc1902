// Products of rows and weights in e4m3 (see fp8_device.h for the scales):
//
//   y[t, n] = sum over blocks b of 128 columns:  2^e[t, b] s[n / 128, b] (q[t, b] . w[n, b])
//
// Two kinds of matrix product, by the output's type:
//
//   bf16, e4m3  v_mfma_scale_f32_32x32x64_f8f6f4, which takes 2^e as an operand
//               (and s where it is a power of two; an f32 s multiplies the
//               block's 32 x 32 results).  It adds eight neighbouring columns'
//               products after cutting each towards zero to a multiple of
//               2^(E - 13), 2^E the largest one's power of two (measured bit by
//               bit); what follows is f32.  A sum is therefore up to 7 * 2^-13
//               of its largest products off; on normal data it is 4.5e-5 of
//               the result, a fortieth of bf16's rounding.
//   f32         v_mfma_f32_32x32x16_bf16 on the same values in bf16, which holds
//               them exactly: products and sums in f32, at half the rate.
#include <algorithm>

#include "cev_internal.h"
#include "fp8_device.h"

namespace {

constexpr int kWaves = 8;  // waves of a workgroup of the small-row kernel, each with its share of the column blocks

struct ProductArgs {
  const void* x;          // rows
  const uint8_t* xs;      // their scales (e4m3 rows)
  const uint8_t* w;       // packed weight
  const uint32_t* ws;     // its scales
  void* out;
  float* part;            // sums over parts of the columns
  int64_t t, x_st, out_st, n;
  int32_t k, kb;          // columns, blocks of them
  int32_t groups;         // groups of 32 weight rows
  int32_t parts, blocks_part;
};

__device__ __forceinline__ f32x16 mfma(const i32x8& a, const i32x8& b, const f32x16& c, int sa, int sb) {
  return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(a, b, c, 0, 0, 0, sa, 0, sb);
}

// The two operands' 64 columns in bf16 (8 columns of each half of the lanes at
// a time; any order of columns that both share will do).
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
__device__ __forceinline__ bf16x8 widen(int lo, int hi) {
  const bf16x2 a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((unsigned)lo, 1.0f, false), b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((unsigned)lo, 1.0f, true);
  const bf16x2 c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((unsigned)hi, 1.0f, false), d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((unsigned)hi, 1.0f, true);
  return bf16x8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}
__device__ __forceinline__ f32x16 mfma_exact(const i32x8& a, const i32x8& b, f32x16 c) {
#pragma unroll
  for (int i = 0; i < 4; ++i)
    c = __builtin_amdgcn_mfma_f32_32x32x16_bf16(widen(a[2 * i], a[2 * i + 1]), widen(b[2 * i], b[2 * i + 1]), c, 0, 0, 0);
  return c;
}

// 2^(code - 127); 2^-127 is subnormal.
__device__ __forceinline__ float e8m0_value(uint32_t code) {
  return __uint_as_float(code == 0 ? 0x400000u : code == 255 ? 0x7fc00000u : code << 23);
}

__device__ __forceinline__ i32x8 join8(const u32x4_t& a, const u32x4_t& b) {
  return i32x8{(int)a[0], (int)a[1], (int)a[2], (int)a[3], (int)b[0], (int)b[1], (int)b[2], (int)b[3]};
}

// The lane's share of block kb of its row: bytes 32 (lane / 32) .. + 31 of
// each half of the block, as two operands; sc the row's scale.  Rows in the
// model's type are brought into e4m3 on the way (the two lanes of a row hold
// the whole block).
template <typename T>
__device__ __forceinline__ void load_x(const ProductArgs& a, int64_t row, int kb, i32x8* o, int& sc) {
  const int up = (threadIdx.x >> 5) & 1;
  if constexpr (sizeof(T) == 1) {
    const uint8_t* const p = (const uint8_t*)a.x + (row * a.kb + kb) * kFp8Block + up * 32;
#pragma unroll
    for (int s = 0; s < 2; ++s) o[s] = join8(*(const u32x4_t*)(p + s * 64), *(const u32x4_t*)(p + s * 64 + 16));
    sc = a.xs[row * a.kb + kb];
  } else {
    float v[8][8];
    uint32_t top = 0;
#pragma unroll
    for (int c = 0; c < 8; ++c) {
      const int col = kb * kFp8Block + (c >> 2) * 64 + up * 32 + (c & 3) * 8;
      load8((const T*)a.x + row * a.x_st + (col < a.k ? col : 0), a.k - col, v[c]);
#pragma unroll
      for (int j = 0; j < 8; ++j) top = max(top, fp8_size(v[c][j]));
    }
    top = max(top, (uint32_t)__shfl_xor((int)top, 32, 64));
    const uint32_t code = fp8_code(top);
    const float f = fp8_inverse(code);
#pragma unroll
    for (int c = 0; c < 8; ++c) {
      o[c >> 2][(c & 3) * 2] = (int)fp8_pack4(v[c][0] * f, v[c][1] * f, v[c][2] * f, v[c][3] * f);
      o[c >> 2][(c & 3) * 2 + 1] = (int)fp8_pack4(v[c][4] * f, v[c][5] * f, v[c][6] * f, v[c][7] * f);
    }
    sc = (int)code;
  }
}

// Four neighbouring columns of a row of the output; the row's last ones and
// rows that are not aligned to four go one by one.
template <typename O>
__device__ __forceinline__ void store4(O* row, int64_t n, int64_t col, const f32x4& v) {
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

// 32 rows times a group of 32 weight rows, the column blocks dealt to the
// workgroup's waves, their sums joined in LDS in the waves' order.
template <typename T, typename O, bool E8M0>
__global__ __launch_bounds__(kWaves * 64) void fp8_small_kernel(ProductArgs a) {
  __shared__ f32x4 sums[kWaves][4][64];
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const int group = (int)(blockIdx.x % a.groups);
  const int64_t tile = blockIdx.x / a.groups / a.parts;
  const int part = (int)(blockIdx.x / a.groups % a.parts);
  const int64_t row = min(tile * 32 + (lane & 31), a.t - 1);
  const int end = min(a.kb, (part + 1) * a.blocks_part);
  f32x16 acc = {};
  for (int kb = part * a.blocks_part + wave; kb < end; kb += kWaves) {
    const uint8_t* const wp = a.w + ((int64_t)group * a.kb + kb) * kFp8GroupBytes + lane * 16;
    i32x8 w[2], x[2];
#pragma unroll
    for (int s = 0; s < 2; ++s) w[s] = join8(*(const u32x4_t*)(wp + s * 2048), *(const u32x4_t*)(wp + s * 2048 + 1024));
    const uint32_t sw = a.ws[(int64_t)group * a.kb + kb];
    int sx;
    load_x<T>(a, row, kb, x, sx);
    if constexpr (sizeof(O) == 4) {
      f32x16 b = {};
      b = mfma_exact(w[0], x[0], b);
      b = mfma_exact(w[1], x[1], b);
      const float f = (E8M0 ? e8m0_value(sw) : __uint_as_float(sw)) * e8m0_value(sx);
#pragma unroll
      for (int i = 0; i < 16; ++i) acc[i] = __builtin_fmaf(b[i], f, acc[i]);
    } else if constexpr (E8M0) {
      acc = mfma(w[0], x[0], acc, (int)sw, sx);
      acc = mfma(w[1], x[1], acc, (int)sw, sx);
    } else {
      f32x16 b = {};
      b = mfma(w[0], x[0], b, 127, sx);
      b = mfma(w[1], x[1], b, 127, sx);
      const float f = __uint_as_float(sw);
#pragma unroll
      for (int i = 0; i < 16; ++i) acc[i] = __builtin_fmaf(b[i], f, acc[i]);
    }
  }
  // lane l holds row l % 32, columns 8 i + 4 (l / 32) .. + 3 of the group in registers 4 i .. 4 i + 3
#pragma unroll
  for (int i = 0; i < 4; ++i) sums[wave][i][lane] = f32x4{acc[4 * i], acc[4 * i + 1], acc[4 * i + 2], acc[4 * i + 3]};
  __syncthreads();
  if (threadIdx.x < 256) {
    const int i = threadIdx.x >> 6;
    f32x4 v = sums[0][i][lane];
#pragma unroll
    for (int w = 1; w < kWaves; ++w) v += sums[w][i][lane];
    const int64_t out_row = tile * 32 + (lane & 31);
    const int64_t col = (int64_t)group * kFp8Group + 8 * i + 4 * (lane >> 5);
    if (out_row < a.t) {
      if (a.part)
        *(f32x4*)(a.part + ((int64_t)part * a.t + out_row) * ((int64_t)a.groups * kFp8Group) + col) = v;
      else
        store4((O*)a.out + out_row * a.out_st, a.n, col, v);
    }
  }
}

// The sums of the parts of the columns, into the output's type: four columns a thread.
struct JoinArgs {
  const float* part;
  void* out;
  uint8_t* out_s;
  int64_t t, n, out_st, width;  // width: padded columns of a row of sums
  int32_t parts, quads;         // quads (gate and up: chunks of 8 columns) of a row
};

template <typename O>
__global__ __launch_bounds__(256) void fp8_join_kernel(JoinArgs a) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int64_t row = i / a.quads;
  if (row >= a.t) return;
  const int64_t col = (i - row * a.quads) * 4;
  const float* p = a.part + row * a.width + col;
  f32x4 v = *(const f32x4*)p;
  for (int s = 1; s < a.parts; ++s) v += *(const f32x4*)(p + (int64_t)s * a.t * a.width);
  store4((O*)a.out + row * a.out_st, a.n, col, v);
}

// silu(g) u in f32 (the hardware's exp2 and reciprocal, within 2^-20 of the
// value: e4m3 keeps 4 bits of it).
__device__ __forceinline__ float swiglu(float g, float u) {
  return g * __builtin_amdgcn_rcpf(1.0f + fast_exp2(-1.44269504f * g)) * u;
}

// Sums of gate and up (groups of 32 columns in turn) into rows in e4m3: 8
// columns a thread, 16 threads a block.
__global__ __launch_bounds__(256) void fp8_join_gate_up_kernel(JoinArgs a) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int64_t row = i / a.quads;
  if (row >= a.t) return;  // (16 threads of a block leave together)
  const int col = (int)(i - row * a.quads) * 8;
  const float* p = a.part + row * a.width + col / kFp8Group * 2 * kFp8Group + col % kFp8Group;
  f32x4 g[2] = {}, u[2] = {};
  for (int s = 0; s < a.parts; ++s, p += a.t * a.width)
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      g[j] += *(const f32x4*)(p + 4 * j);
      u[j] += *(const f32x4*)(p + kFp8Group + 4 * j);
    }
  float v[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) v[j] = col + j < a.n ? swiglu(g[j >> 2][j & 3], u[j >> 2][j & 3]) : 0.0f;
  uint32_t code;
  const u32x2_t q = fp8_block16(v, code);
  *(u32x2_t*)((uint8_t*)a.out + (row * a.quads + col / 8) * 8) = q;
  if ((col & 127) == 0) a.out_s[row * (a.quads >> 4) + (col >> 7)] = (uint8_t)code;
}

int32_t launched(const char* what) {
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? CEV_OK : cev_fail(CEV_ERR_HIP, "%s launch: %s", what, hipGetErrorString(e));
}

// How a product runs.
struct Form {
  bool pack_x;  // rows of the model's type go into e4m3 in a launch of their own
  int32_t groups, kb, parts, blocks_part;
  size_t rows_bytes, scales_bytes, part_bytes;
};

size_t up256(size_t n) { return (n + 255) & ~(size_t)255; }

Form form_of(const cev_fp8_desc& d) {
  Form f{};
  f.kb = (int32_t)((d.k + 127) / 128);
  f.groups = (int32_t)(d.gate_up ? (d.n + 127) / 128 * 8 : (d.n + 255) / 256 * 8);
  const int64_t tiles = (d.t + 31) / 32;
  f.pack_x = d.x_dtype != CEV_E4M3 && tiles > 1;
  if (f.pack_x) {
    f.rows_bytes = up256((size_t)d.t * f.kb * kFp8Block);
    f.scales_bytes = up256((size_t)d.t * f.kb);
  }
  f.parts = 1;
  f.blocks_part = f.kb;
  if (d.gate_up) f.part_bytes = (size_t)f.parts * d.t * f.groups * kFp8Group * 4;
  return f;
}

int32_t check_desc(const char* what, const cev_fp8_desc* d) {
  CEV_CHECK_ARG(d != nullptr, "%s: null descriptor", what);
  if (d->x_dtype != CEV_F32 && d->x_dtype != CEV_BF16 && d->x_dtype != CEV_E4M3) return cev_fail(CEV_ERR_UNSUPPORTED, "%s: x dtype %d", what, d->x_dtype);
  if (d->gate_up ? d->out_dtype != CEV_E4M3 : d->out_dtype != CEV_F32 && d->out_dtype != CEV_BF16)
    return cev_fail(CEV_ERR_UNSUPPORTED, "%s: out dtype %d", what, d->out_dtype);
  if (d->scales != CEV_FP8_SCALES_E8M0 && d->scales != CEV_FP8_SCALES_F32) return cev_fail(CEV_ERR_UNSUPPORTED, "%s: scale kind %d", what, d->scales);
  CEV_CHECK_ARG(d->t >= 0 && d->t <= INT32_MAX && d->n >= 1 && d->n <= INT32_MAX - 256 && d->k >= 1 && d->k <= INT32_MAX - 128,
                "%s: %lld rows, %lld x %lld weight", what, (long long)d->t, (long long)d->n, (long long)d->k);
  // (the workspace's bytes stay within 64 bits)
  CEV_CHECK_ARG(d->t <= ((int64_t)1 << 46) / std::max(d->n, d->k), "%s: %lld rows are too large", what, (long long)d->t);
  return CEV_OK;
}

template <typename T, typename O>
int32_t launch_small(const ProductArgs& a, bool e8m0, hipStream_t s) {
  const int64_t grid = (a.t + 31) / 32 * a.parts * a.groups;
  if (grid > INT32_MAX) return cev_fail(CEV_ERR_UNSUPPORTED, "cev_fp8_product: grid too large");
  if (e8m0)
    hipLaunchKernelGGL((fp8_small_kernel<T, O, true>), dim3((unsigned)grid), dim3(kWaves * 64), 0, s, a);
  else
    hipLaunchKernelGGL((fp8_small_kernel<T, O, false>), dim3((unsigned)grid), dim3(kWaves * 64), 0, s, a);
  return launched("cev_fp8_product");
}

template <typename O>
int32_t launch_small(const ProductArgs& a, int x_dtype, bool e8m0, hipStream_t s) {
  if (x_dtype == CEV_E4M3) return launch_small<uint8_t, O>(a, e8m0, s);
  if (x_dtype == CEV_BF16) return launch_small<__bf16, O>(a, e8m0, s);
  return launch_small<float, O>(a, e8m0, s);
}

}  // namespace

extern "C" int32_t cev_fp8_work_size(const cev_fp8_desc* d, size_t* bytes) {
  if (const int32_t rc = check_desc("cev_fp8_work_size", d)) return rc;
  CEV_CHECK_ARG(bytes != nullptr, "cev_fp8_work_size: null output");
  const Form f = form_of(*d);
  *bytes = f.rows_bytes + f.scales_bytes + f.part_bytes;
  return CEV_OK;
}

extern "C" int32_t cev_fp8_product(const cev_fp8_desc* d, const void* x, const void* x_scales, const void* weight, size_t weight_bytes,
                                   void* out, void* out_scales, void* work, size_t work_bytes, cev_stream stream) {
  const char* const me = "cev_fp8_product";
  if (const int32_t rc = check_desc(me, d)) return rc;
  size_t need = 0;
  if (const int32_t rc = cev_fp8_weight_size(d->n, d->k, d->gate_up, &need)) return rc;
  if (weight_bytes < need) return cev_fail(CEV_ERR_SPACE, "%s: a weight of %zu bytes, %zu needed", me, weight_bytes, need);
  if (d->t == 0) return CEV_OK;
  CEV_CHECK_ARG(x && weight && out, "%s: null buffer", me);
  CEV_CHECK_ARG((((uintptr_t)x | (uintptr_t)weight) & 15) == 0, "%s: x and the weight must be 16-byte aligned", me);
  CEV_CHECK_ARG((d->x_dtype == CEV_E4M3) == (x_scales != nullptr) && (d->gate_up != 0) == (out_scales != nullptr), "%s: rows in e4m3 come with their scales", me);
  if (d->x_dtype != CEV_E4M3 && d->t > 1) {
    const int vec = d->x_dtype == CEV_BF16 ? 8 : 4;
    CEV_CHECK_ARG(d->x_stride >= d->k && d->x_stride % vec == 0 && cev_stride_fits(d->x_stride, d->t),
                  "%s: the row stride of x must cover a row and be a multiple of %d elements", me, vec);
  }
  if (!d->gate_up) {
    CEV_CHECK_ARG(d->t <= 1 || (d->out_stride >= d->n && cev_stride_fits(d->out_stride, d->t)), "%s: the row stride of out must cover a row", me);
    CEV_CHECK_ARG(((uintptr_t)out & (d->out_dtype == CEV_BF16 ? 1 : 3)) == 0, "%s: misaligned out", me);
  } else {
    CEV_CHECK_ARG(((uintptr_t)out & 15) == 0, "%s: rows in e4m3 must be 16-byte aligned", me);
  }
  const Form f = form_of(*d);
  need = f.rows_bytes + f.scales_bytes + f.part_bytes;
  if (work_bytes < need) return cev_fail(CEV_ERR_SPACE, "%s: a workspace of %zu bytes, %zu needed", me, work_bytes, need);
  CEV_CHECK_ARG(need == 0 || (work && ((uintptr_t)work & 255) == 0), "%s: the workspace must be 256-byte aligned", me);
  const hipStream_t s = (hipStream_t)stream;
  uint8_t* const space = (uint8_t*)work;
  int x_dtype = d->x_dtype;
  ProductArgs a{};
  a.x = x, a.xs = (const uint8_t*)x_scales;
  a.x_st = d->t > 1 ? d->x_stride : 0;
  if (f.pack_x) {
    if (const int32_t rc = cev_fp8_rows(d->x_dtype, d->t, d->k, x, d->x_stride, space, space + f.rows_bytes, stream)) return rc;
    a.x = space, a.xs = space + f.rows_bytes;
    x_dtype = CEV_E4M3;
  }
  a.w = (const uint8_t*)weight;
  a.ws = (const uint32_t*)(a.w + (int64_t)f.groups * f.kb * kFp8GroupBytes);
  a.out = out, a.out_st = d->t > 1 ? d->out_stride : 0;
  a.t = d->t, a.n = d->n, a.k = (int32_t)d->k, a.kb = f.kb, a.groups = f.groups, a.parts = f.parts, a.blocks_part = f.blocks_part;
  if (f.part_bytes) a.part = (float*)(space + f.rows_bytes + f.scales_bytes);
  const bool e8m0 = d->scales == CEV_FP8_SCALES_E8M0;
  const int32_t rc = d->out_dtype == CEV_F32 ? launch_small<float>(a, x_dtype, e8m0, s) : launch_small<__bf16>(a, x_dtype, e8m0, s);
  if (rc || !a.part) return rc;
  JoinArgs j{a.part, out, (uint8_t*)out_scales, d->t, d->n, a.out_st, (int64_t)f.groups * kFp8Group, f.parts, 0};
  j.quads = (int32_t)(d->gate_up ? (d->n + 127) / 128 * 16 : (d->n + 3) / 4);
  const int64_t grid = (d->t * j.quads + 255) / 256;
  if (grid > INT32_MAX) return cev_fail(CEV_ERR_UNSUPPORTED, "%s: too many rows", me);
  if (d->gate_up)
    hipLaunchKernelGGL(fp8_join_gate_up_kernel, dim3((unsigned)grid), dim3(256), 0, s, j);
  else if (d->out_dtype == CEV_BF16)
    hipLaunchKernelGGL(fp8_join_kernel<__bf16>, dim3((unsigned)grid), dim3(256), 0, s, j);
  else
    hipLaunchKernelGGL(fp8_join_kernel<float>, dim3((unsigned)grid), dim3(256), 0, s, j);
  return launched(me);
}
