// Rows of activations and weights into e4m3 with a scale for each block of
// 128 values, and weights laid out for the products of fp8_linear.hip.
//
//   rows    q = e4m3(x / 2^e), a scale for 128 columns of a row
//   norm    the same of the RMS norm of x (+ h): from the rounded residual on
//           as good as exact (the sum in f64, products in f32 only where that
//           rounds the same way) up to the one rounding
//   blocks  the same of a weight, a scale for 128 x 128 values
//   pack    an e4m3 weight in the order in which the matrix cores read it
//
// All of them move bytes and compute next to nothing: one pass, 16 lanes of 8
// values for a block, the largest value by lane moves.
#include "cev_internal.h"
#include "fp8_device.h"

namespace {

constexpr int kThreads = 256;

struct RowsArgs {
  const void* x;
  uint8_t* q;
  uint8_t* s;
  int64_t t, x_st;
  int32_t k, chunks;  // chunks of 8 columns of a padded row
  int32_t rows_wg;    // rows of a workgroup (1: a part of a wide row)
};

// 8 columns a thread (8192 x 4096 bf16: 18.0 us, 5.6 TB/s; 32 columns a thread
// take 20.4 there and 3.5 instead of 2.4 for one row).
template <typename T>
__global__ __launch_bounds__(kThreads) void fp8_rows_kernel(RowsArgs a, int parts) {
  const int i = (int)(blockIdx.x % parts) * kThreads + (int)threadIdx.x;
  const int rr = a.rows_wg > 1 ? i / a.chunks : 0, col = i - rr * a.chunks;
  const int64_t row = (int64_t)(blockIdx.x / parts) * a.rows_wg + rr;
  const bool on = rr < a.rows_wg && col < a.chunks && row < a.t;  // (16 lanes of a block alike)
  float v[8];
  load8((const T*)a.x + (on ? row * a.x_st + (int64_t)col * 8 : 0), on ? a.k - col * 8 : 0, v);
  uint32_t code;
  const u32x2_t q = fp8_block16(v, code);
  if (!on) return;
  *(u32x2_t*)(a.q + (row * a.chunks + col) * 8) = q;
  if ((col & 15) == 0) a.s[row * (a.chunks >> 4) + (col >> 4)] = (uint8_t)code;
}

struct NormArgs {
  const void* x;
  const void* h;
  void* x_out;
  const void* w;
  uint8_t* q;
  uint8_t* s;
  int64_t rows, x_st, h_st, xo_st;
  int32_t k, chunks, plus_one;
  float eps;
  double inv_k;
};

template <typename T>
__device__ __forceinline__ void store8(T* p, int have, const float* v) {
  if (have >= 8) {
    if constexpr (sizeof(T) == 2) {
      u32x4_t c;
#pragma unroll
      for (int i = 0; i < 4; ++i) c[i] = (uint32_t)bf16_bits(v[2 * i]) | (uint32_t)bf16_bits(v[2 * i + 1]) << 16;
      *(u32x4_t*)p = c;
    } else {
      *(f32x4*)p = f32x4{v[0], v[1], v[2], v[3]};
      *(f32x4*)(p + 4) = f32x4{v[4], v[5], v[6], v[7]};
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i < have) p[i] = (T)v[i];
  }
}

// v * inv * w in f64, then in f32 rounded to odd: what is rounded to fewer bits
// after it comes out as the f64 product's own rounding would.  (Beyond f32's
// range it is infinite, far below it 2^-149.)
__device__ __forceinline__ float scaled_odd(float v, double inv, float w) {
  asm("" : "+v"(v));  // (or the f64 values of the sum of squares are kept for it, in the registers of three waves a SIMD)
  const double exact = (double)v * inv * (double)w;
  const float p = (float)exact;
  if (__builtin_fabsf(p) < __builtin_inff() && (double)p != exact) {
    const uint32_t u = __float_as_uint(p), sign = (uint32_t)(__double_as_longlong(exact) >> 32) & 0x80000000u;
    const uint32_t size = u & 0x7fffffffu, down = __builtin_fabs((double)p) > __builtin_fabs(exact);  // p is the larger one
    return __uint_as_float(sign | (size - down) | 1u);
  }
  return p;
}

// The scale of a block that holds kSmallTop is more than 2^-57, and what is less than 2^-10 of it becomes 0.
constexpr float kLargeWeight = 0x1p56f, kSmallTop = 0x1p-48f;

// One row for WAVES waves, NCH chunks of 8 columns a lane in registers; a
// row wider than that reads its residual a second time.
template <typename T, int WAVES, int NCH, bool RES>
__global__ __launch_bounds__(WAVES > 4 ? WAVES * 64 : kThreads) void fp8_norm_kernel(NormArgs a) {
  constexpr int LANES = WAVES * 64, ROWS = WAVES > 4 ? 1 : kThreads / LANES;
  __shared__ double part[ROWS * WAVES];
  const int64_t r = (int64_t)blockIdx.x * ROWS + threadIdx.x / LANES;
  const int lane = threadIdx.x % LANES;
  const bool live = r < a.rows;
  const T* const x = (const T*)a.x + (live ? r : 0) * a.x_st;
  const T* const h = RES ? (const T*)a.h + (live ? r : 0) * a.h_st : nullptr;
  T* const xo = RES ? (T*)a.x_out + (live ? r : 0) * a.xo_st : nullptr;
  float v[NCH][8];
  double sum = 0.0;
  auto take = [&](int c, float* o) {  // chunk c of the row, the residual added and rounded
    const int have = live ? a.k - c * 8 : 0;
    load8(x + (have > 0 ? c * 8 : 0), have, o);
    if constexpr (RES) {
      float add[8];
      load8(h + (have > 0 ? c * 8 : 0), have, add);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        o[j] += add[j];
        if constexpr (sizeof(T) == 2) o[j] = bf16_round(o[j]);
      }
      if (have > 0) store8(xo + c * 8, have, o);
    }
  };
#pragma unroll
  for (int b = 0; b < NCH; ++b) take(lane + b * LANES, v[b]);
#pragma unroll
  for (int b = 0; b < NCH; ++b)
#pragma unroll
    for (int j = 0; j < 8; ++j) sum = __builtin_fma((double)v[b][j], (double)v[b][j], sum);
  for (int c = lane + NCH * LANES; c < a.chunks; c += LANES) {
    float o[8];
    take(c, o);
#pragma unroll
    for (int j = 0; j < 8; ++j) sum = __builtin_fma((double)o[j], (double)o[j], sum);
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) sum += __shfl_xor(sum, o, 64);
  if constexpr (WAVES > 1) {
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = sum;
    __syncthreads();
    sum = 0.0;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) sum += part[threadIdx.x / LANES * WAVES + w];
  }
  // 1 / root to 2^-43: the f32 one and a step of Newton's, where f32 holds the mean
  const double mean = __builtin_fma(sum, a.inv_k, (double)a.eps);
  double inv;
  if (mean > 1e-30 && mean < 1e30) {
    const double y = rsqrtf((float)mean);
    inv = __builtin_fma(0.5 * y, __builtin_fma(-mean * y, y, 1.0), y);
  } else {
    inv = 1.0 / sqrt(mean);
  }
  const float inv_high = (float)inv;
  const bool odd_row = !(inv_high >= 0x1p-126f && inv_high <= 0x1p126f);
  auto give = [&](int c, float* o) {  // the row's chunk c, normalised, into e4m3
    float w[8];
    const int have = a.k - c * 8;
    load8((const T*)a.w + (have > 0 ? c * 8 : 0), have, w);
    // Of normal numbers the f32 products, three roundings with that of inv_high,
    // are within 3 * 2^-24 of the exact ones, less than 3 units of their last
    // place.  e4m3's borders (between two of its values, and of its scale) are
    // multiples of 2^19 units: within 4 units of one the f64 product decides.
    uint32_t near = ~0u;
    float p[8], w_top = 0.0f;
    auto from_border = [](float f) { return (__float_as_uint(f) << 13) + (4u << 13); };  // less than 8 << 13: that near
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      if (a.plus_one) w[j] += 1.0f;
      p[j] = o[j] * inv_high * w[j];
      near = min(near, from_border(p[j]));
      w_top = fmaxf(w_top, __builtin_fabsf(w[j]));
    }
    bool redo = odd_row || w_top >= kLargeWeight;
    if (near < 8u << 13)
#pragma unroll
      for (int j = 0; j < 8; ++j) redo |= p[j] != 0.0f && from_border(p[j]) < 8u << 13;  // (0 is no border)
    auto in_f64 = [&] {
#pragma unroll
      for (int j = 0; j < 8; ++j) p[j] = j < have ? scaled_odd(o[j], inv, w[j]) : 0.0f;
    };
    if (redo) in_f64();
    // Where x * inv or the product is no normal number, the product with a
    // smaller weight is less than 2^-126 * kLargeWeight = 2^-70: 0 in a block that
    // holds kSmallTop.
    uint32_t top = fp8_top16(p);
    if (top - 1 < __builtin_bit_cast(uint32_t, kSmallTop) - 1) {  // (16 lanes alike; not a block of zeros)
      in_f64();
      top = fp8_top16(p);
    }
    const uint32_t code = fp8_code(top);
    const u32x2_t q = fp8_pack8(p, code);
    if (live && c < a.chunks) {
      *(u32x2_t*)(a.q + (r * a.chunks + c) * 8) = q;
      if ((c & 15) == 0) a.s[r * (a.chunks >> 4) + (c >> 4)] = (uint8_t)code;
    }
  };
#pragma unroll
  for (int b = 0; b < NCH; ++b) give(lane + b * LANES, v[b]);
  // (chunks is a multiple of 16: the 16 lanes of a block go on together)
  for (int c = lane + NCH * LANES; c < a.chunks; c += LANES) {
    float o[8];
    const int have = live ? a.k - c * 8 : 0;
    load8((RES ? (const T*)xo : x) + (have > 0 ? c * 8 : 0), have, o);
    give(c, o);
  }
}

struct BlocksArgs {
  const void* w;
  uint8_t* q;
  uint8_t* s;
  int64_t n, ldw;
  int32_t k, kb;
};

constexpr int kBlockThreads = 1024;

// One 128 x 128 block a workgroup, 16 columns a thread: all of a block's loads
// are under way together (4096 x 12288 bf16 29.2 us, 5.2 TB/s; 1021 x 2056 f32 4.5.
// With 256 threads 31.9 and 6.2).
template <typename T>
__global__ __launch_bounds__(kBlockThreads) void fp8_blocks_kernel(BlocksArgs a) {
  __shared__ uint32_t part[kBlockThreads / 64];
  const int64_t rb = blockIdx.x / a.kb;
  const int cb = (int)(blockIdx.x % a.kb);
  constexpr int CH = 2048 / kBlockThreads, STEP = kBlockThreads / 16;  // chunks of 8 columns of a thread, rows apart
  float v[CH][8];
  const int col = cb * kFp8Block + (int)(threadIdx.x & 15) * 8, have = a.k - col;
  const int64_t r0 = rb * kFp8Block + (threadIdx.x >> 4);
  uint32_t top = 0;
#pragma unroll
  for (int b = 0; b < CH; ++b) {
    const int64_t r = r0 + b * STEP;
    const bool on = r < a.n && have > 0;
    load8((const T*)a.w + (on ? r * a.ldw + col : 0), on ? have : 0, v[b]);
  }
#pragma unroll
  for (int b = 0; b < CH; ++b)
#pragma unroll
    for (int j = 0; j < 8; ++j) top = max(top, fp8_size(v[b][j]));
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) top = max(top, (uint32_t)__shfl_xor((int)top, o, 64));
  if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = top;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kBlockThreads / 64; ++w) top = max(top, part[w]);
  const uint32_t code = fp8_code(top);
  const float f = fp8_inverse(code);
  if (threadIdx.x == 0) a.s[rb * a.kb + cb] = (uint8_t)code;
#pragma unroll
  for (int b = 0; b < CH; ++b) {
    const int64_t r = r0 + b * STEP;
    if (r >= a.n || have <= 0) continue;
    const u32x2_t q = {fp8_pack4(v[b][0] * f, v[b][1] * f, v[b][2] * f, v[b][3] * f), fp8_pack4(v[b][4] * f, v[b][5] * f, v[b][6] * f, v[b][7] * f)};
    uint8_t* const p = a.q + r * a.k + col;
    if (a.k % 8 == 0) {  // rows of q start 8-byte aligned
      *(u32x2_t*)p = q;
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (j < have) p[j] = (uint8_t)(q[j >> 2] >> (8 * (j & 3)));
    }
  }
}

struct PackArgs {
  const uint8_t* q[2];
  const void* s[2];
  int64_t ldq[2], lds[2];
  uint8_t* out;
  uint32_t* out_s;
  int64_t n, groups;
  int32_t k, kb, gate_up, f32_scales;
};

// One 4 KB piece of the layout (32 rows, 128 columns) a workgroup, 16 bytes a
// thread; thread 0 its scale.
__global__ __launch_bounds__(kThreads) void fp8_pack_kernel(PackArgs a) {
  const int64_t group = blockIdx.x / a.kb;
  const int kb = (int)(blockIdx.x % a.kb);
  const int which = a.gate_up ? (int)(group & 1) : 0;
  const int64_t row0 = (a.gate_up ? group >> 1 : group) * kFp8Group;
  // thread = ((sub * 2 + half) * 64 + lane): row lane % 32, columns 64 sub + 32 (lane / 32) + 16 half
  const int lane = threadIdx.x & 63, sub = threadIdx.x >> 7, half = (threadIdx.x >> 6) & 1;
  const int64_t row = row0 + (lane & 31);
  const int col = kb * kFp8Block + sub * 64 + (lane >> 5) * 32 + half * 16, have = a.k - col;
  u32x4_t v = {0, 0, 0, 0};
  if (row < a.n && have > 0) {
    const uint8_t* const p = a.q[which] + row * a.ldq[which] + col;
    if (have >= 16 && ((uintptr_t)p & 15) == 0) {
      v = *(const u32x4_t*)p;
    } else {
#pragma unroll
      for (int j = 0; j < 16; ++j)
        if (j < have) v[j >> 2] |= (uint32_t)p[j] << (8 * (j & 3));
    }
  }
  *(u32x4_t*)(a.out + (group * a.kb + kb) * kFp8GroupBytes + threadIdx.x * 16) = v;
  if (threadIdx.x == 0) {
    uint32_t s = a.f32_scales ? 0x3f800000u : 127u;  // rows behind the last: 1
    if (row0 < a.n) {
      const int64_t at = (row0 / kFp8Block) * a.lds[which] + kb;
      s = a.f32_scales ? ((const uint32_t*)a.s[which])[at] : ((const uint8_t*)a.s[which])[at];
    }
    if (a.f32_scales)
      a.out_s[group * a.kb + kb] = s;
    else  // bytes, a group's blocks up to a multiple of 4
      ((uint8_t*)a.out_s)[group * ((a.kb + 3) & ~3) + kb] = (uint8_t)s;
  }
}

bool aligned(const void* p, uintptr_t n) { return ((uintptr_t)p & (n - 1)) == 0; }

int32_t launched(const char* what) {
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? CEV_OK : cev_fail(CEV_ERR_HIP, "%s launch: %s", what, hipGetErrorString(e));
}

int64_t size_of(int32_t dtype) { return dtype == CEV_BF16 ? 2 : 4; }

// The checks of a call's rows in the model's type.
int32_t check_rows(const char* what, int32_t dtype, int64_t t, int64_t k, const char* name, const void* p, int64_t stride) {
  const int vec = dtype == CEV_BF16 ? 8 : 4;
  CEV_CHECK_ARG(p != nullptr, "%s: null %s", what, name);
  CEV_CHECK_ARG(aligned(p, 16), "%s: %s must be 16-byte aligned", what, name);
  CEV_CHECK_ARG(t <= 1 || (stride >= k && stride % vec == 0 && cev_stride_fits(stride, t)),
                "%s: the row stride of %s must cover a row and be a multiple of %d elements", what, name, vec);
  return CEV_OK;
}

}  // namespace

extern "C" int32_t cev_fp8_rows(int32_t dtype, int64_t t, int64_t k, const void* x, int64_t x_stride, void* q, void* scales, cev_stream stream) {
  if (dtype != CEV_F32 && dtype != CEV_BF16) return cev_fail(CEV_ERR_UNSUPPORTED, "cev_fp8_rows: dtype %d", dtype);
  CEV_CHECK_ARG(t >= 0 && t <= INT32_MAX && k >= 1 && k <= INT32_MAX - 128, "cev_fp8_rows: %lld rows of %lld values", (long long)t, (long long)k);
  if (t == 0) return CEV_OK;
  if (const int32_t rc = check_rows("cev_fp8_rows", dtype, t, k, "x", x, x_stride)) return rc;
  CEV_CHECK_ARG(q && scales && aligned(q, 16), "cev_fp8_rows: null or misaligned output");
  RowsArgs a{x, (uint8_t*)q, (uint8_t*)scales, t, x_stride, (int32_t)k, (int32_t)((k + 127) / 128 * 16), 1};
  a.rows_wg = a.chunks >= kThreads ? 1 : kThreads / a.chunks;
  const int parts = a.chunks > kThreads ? (a.chunks + kThreads - 1) / kThreads : 1;
  const int64_t grid = (t + a.rows_wg - 1) / a.rows_wg * parts;
  if (!fp8_grid_fits(grid, kThreads)) return cev_fail(CEV_ERR_UNSUPPORTED, "cev_fp8_rows: too many rows");
  CEV_CHECK_ARG(fp8_apart({{q, 1, 0, t * a.chunks * 8}, {scales, 1, 0, t * (a.chunks / 16)}}, {cev_rows(x, t, x_stride, k, size_of(dtype))}),
                "cev_fp8_rows: the outputs must have memory of their own");
  hipLaunchKernelGGL(dtype == CEV_BF16 ? fp8_rows_kernel<__bf16> : fp8_rows_kernel<float>, dim3((unsigned)grid), dim3(kThreads), 0, (hipStream_t)stream, a, parts);
  return launched("cev_fp8_rows");
}

namespace {

template <typename T, int WAVES, int NCH>
int32_t launch_norm(const NormArgs& a, hipStream_t s) {
  constexpr int ROWS = WAVES > 4 ? 1 : 4 / WAVES;
  const int64_t grid = (a.rows + ROWS - 1) / ROWS;
  if (!fp8_grid_fits(grid, ROWS * WAVES * 64)) return cev_fail(CEV_ERR_UNSUPPORTED, "cev_fp8_rms_norm: too many rows");
  if (a.h)
    hipLaunchKernelGGL((fp8_norm_kernel<T, WAVES, NCH, true>), dim3((unsigned)grid), dim3(ROWS * WAVES * 64), 0, s, a);
  else
    hipLaunchKernelGGL((fp8_norm_kernel<T, WAVES, NCH, false>), dim3((unsigned)grid), dim3(ROWS * WAVES * 64), 0, s, a);
  return launched("cev_fp8_rms_norm");
}

template <typename T>
int32_t launch_norm(const NormArgs& a, hipStream_t s) {
  // A row's chunks of 8 columns go to one lane each; where there are more rows
  // than fill the card, to as few waves as hold them in registers (us, bf16 with
  // the residual, launches over three inputs in turn: 64 x 4096 with 8 waves 3.7,
  // with 4 4.1; 8192 x 4096 42.8 and 41.5; 64 x 12288 with 16 waves 5.0, with 8
  // 5.8; 4096 x 1024 with 4 waves 10.0, with 2 8.0.  Over inputs that change with
  // every call 8192 x 4096 takes 47.4, 5.0 TB/s).
  if (a.chunks <= 64) return launch_norm<T, 1, 1>(a, s);
  const bool few = a.rows <= 512;
  if (a.chunks <= 128 && !few) return launch_norm<T, 2, 1>(a, s);
  if (a.chunks <= 256) return launch_norm<T, 4, 1>(a, s);
  if (a.chunks <= 512) return few ? launch_norm<T, 8, 1>(a, s) : launch_norm<T, 4, 2>(a, s);
  return few ? launch_norm<T, 16, 1>(a, s) : launch_norm<T, 8, 2>(a, s);
}

}  // namespace

extern "C" int32_t cev_fp8_rms_norm(int32_t dtype, int64_t rows, int64_t k, const void* x, int64_t x_stride, const void* h, int64_t h_stride,
                                    void* x_out, int64_t x_out_stride, const void* w, float eps, int32_t weight_plus_one, void* q,
                                    void* scales, cev_stream stream) {
  if (dtype != CEV_F32 && dtype != CEV_BF16) return cev_fail(CEV_ERR_UNSUPPORTED, "cev_fp8_rms_norm: dtype %d", dtype);
  CEV_CHECK_ARG(rows >= 0 && rows <= INT32_MAX && k >= 1 && k <= INT32_MAX - 128, "cev_fp8_rms_norm: %lld rows of %lld values", (long long)rows,
                (long long)k);
  CEV_CHECK_ARG(eps >= 0.0f && eps <= 3.0e38f, "cev_fp8_rms_norm: eps must be finite and not negative");
  if (rows == 0) return CEV_OK;
  if (const int32_t rc = check_rows("cev_fp8_rms_norm", dtype, rows, k, "x", x, x_stride)) return rc;
  if (const int32_t rc = check_rows("cev_fp8_rms_norm", dtype, 1, k, "w", w, 0)) return rc;
  if (h) {
    if (const int32_t rc = check_rows("cev_fp8_rms_norm", dtype, rows, k, "h", h, h_stride)) return rc;
    if (const int32_t rc = check_rows("cev_fp8_rms_norm", dtype, rows, k, "x_out", x_out, x_out_stride)) return rc;
  }
  CEV_CHECK_ARG(q && scales && aligned(q, 16), "cev_fp8_rms_norm: null or misaligned output");
  const int64_t e = size_of(dtype), kb = (k + 127) / 128;
  const CevRows rx = cev_rows(x, rows, x_stride, k, e), rh = cev_rows(h, rows, h_stride, k, e), ro = cev_rows(h ? x_out : nullptr, rows, x_out_stride, k, e),
                rw = cev_rows(w, 1, 0, k, e);
  CEV_CHECK_ARG(fp8_apart({{q, 1, 0, rows * kb * 128}, {scales, 1, 0, rows * kb}}, {rx, rh, ro, rw}),
                "cev_fp8_rms_norm: the rows in e4m3 must have memory of their own");
  CEV_CHECK_ARG((cev_same(ro, rx) || !cev_overlap(&ro, &rx)) && (cev_same(ro, rh) || !cev_overlap(&ro, &rh)) && !cev_overlap(&ro, &rw),
                "cev_fp8_rms_norm: x_out must be x or h, or have memory of its own");
  const NormArgs a{x, h, x_out, w, (uint8_t*)q, (uint8_t*)scales, rows, x_stride, h_stride, x_out_stride, (int32_t)k, (int32_t)((k + 127) / 128 * 16),
                   weight_plus_one, eps, 1.0 / (double)k};
  return dtype == CEV_BF16 ? launch_norm<__bf16>(a, (hipStream_t)stream) : launch_norm<float>(a, (hipStream_t)stream);
}

extern "C" int32_t cev_fp8_blocks(int32_t dtype, int64_t n, int64_t k, const void* w, int64_t ldw, void* q, void* scales, cev_stream stream) {
  if (dtype != CEV_F32 && dtype != CEV_BF16) return cev_fail(CEV_ERR_UNSUPPORTED, "cev_fp8_blocks: dtype %d", dtype);
  CEV_CHECK_ARG(n >= 1 && n <= INT32_MAX - 256 && k >= 1 && k <= INT32_MAX - 128, "cev_fp8_blocks: a weight of %lld x %lld", (long long)n, (long long)k);
  if (const int32_t rc = check_rows("cev_fp8_blocks", dtype, n, k, "w", w, ldw)) return rc;
  CEV_CHECK_ARG(q && scales && aligned(q, 16), "cev_fp8_blocks: null or misaligned output");
  const BlocksArgs a{w, (uint8_t*)q, (uint8_t*)scales, n, ldw, (int32_t)k, (int32_t)((k + 127) / 128)};
  const int64_t grid = (n + 127) / 128 * a.kb;
  if (!fp8_grid_fits(grid, kBlockThreads)) return cev_fail(CEV_ERR_UNSUPPORTED, "cev_fp8_blocks: weight too large");
  CEV_CHECK_ARG(fp8_apart({{q, 1, 0, n * k}, {scales, 1, 0, grid}}, {cev_rows(w, n, ldw, k, size_of(dtype))}),
                "cev_fp8_blocks: the outputs must have memory of their own");
  if (dtype == CEV_BF16)
    hipLaunchKernelGGL(fp8_blocks_kernel<__bf16>, dim3((unsigned)grid), dim3(kBlockThreads), 0, (hipStream_t)stream, a);
  else
    hipLaunchKernelGGL(fp8_blocks_kernel<float>, dim3((unsigned)grid), dim3(kBlockThreads), 0, (hipStream_t)stream, a);
  return launched("cev_fp8_blocks");
}

extern "C" int32_t cev_fp8_weight_size(int64_t n, int64_t k, int32_t gate_up, size_t* bytes) {
  CEV_CHECK_ARG(bytes != nullptr, "cev_fp8_weight_size: null output");
  CEV_CHECK_ARG(n >= 1 && n <= INT32_MAX - 256 && k >= 1 && k <= INT32_MAX - 128, "cev_fp8_weight_size: a weight of %lld x %lld", (long long)n,
                (long long)k);
  const size_t tile = (size_t)kFp8Group * kFp8TileGroups, rows = (size_t)n * (gate_up ? 2 : 1);
  const size_t columns = gate_up ? ((size_t)n + 127) / 128 * 256 : (rows + tile - 1) / tile * tile;
  const size_t pieces = columns / kFp8Group * (((size_t)k + 127) / 128);
  *bytes = pieces * (kFp8GroupBytes + 4);
  return CEV_OK;
}

extern "C" int32_t cev_fp8_weight_pack(int64_t n, int64_t k, int32_t scale_kind, const void* q, int64_t ldq, const void* scales, int64_t lds,
                                       const void* up_q, int64_t up_ldq, const void* up_scales, int64_t up_lds, void* weight,
                                       size_t weight_bytes, cev_stream stream) {
  const int gate_up = up_q != nullptr;
  size_t need = 0;
  if (const int32_t rc = cev_fp8_weight_size(n, k, gate_up, &need)) return rc;
  if (scale_kind != CEV_FP8_SCALES_E8M0 && scale_kind != CEV_FP8_SCALES_F32)
    return cev_fail(CEV_ERR_UNSUPPORTED, "cev_fp8_weight_pack: scale kind %d", scale_kind);
  const int64_t kb = (k + 127) / 128, nb = (n + 127) / 128;
  CEV_CHECK_ARG(q && scales && (!gate_up || up_scales) && (gate_up || !up_scales), "cev_fp8_weight_pack: null buffer");
  CEV_CHECK_ARG((n <= 1 || (ldq >= k && cev_stride_fits(ldq, n))) && (nb <= 1 || (lds >= kb && cev_stride_fits(lds, nb))) &&
                    (!gate_up || ((n <= 1 || (up_ldq >= k && cev_stride_fits(up_ldq, n))) && (nb <= 1 || (up_lds >= kb && cev_stride_fits(up_lds, nb))))),
                "cev_fp8_weight_pack: row strides must cover a row");
  CEV_CHECK_ARG(scale_kind == CEV_FP8_SCALES_E8M0 || (aligned(scales, 4) && aligned(up_scales, 4)), "cev_fp8_weight_pack: misaligned scales");
  CEV_CHECK_ARG(weight && aligned(weight, 256), "cev_fp8_weight_pack: the weight must be 256-byte aligned");
  if (weight_bytes < need) return cev_fail(CEV_ERR_SPACE, "cev_fp8_weight_pack: %zu bytes, %zu needed", weight_bytes, need);
  PackArgs a{};
  a.q[0] = (const uint8_t*)q, a.q[1] = (const uint8_t*)up_q;
  a.s[0] = scales, a.s[1] = up_scales;
  a.ldq[0] = ldq, a.ldq[1] = up_ldq, a.lds[0] = lds, a.lds[1] = up_lds;
  a.n = n, a.k = (int32_t)k, a.kb = (int32_t)kb;
  a.groups = (int64_t)(need / (kFp8GroupBytes + 4)) / kb;
  a.out = (uint8_t*)weight;
  a.out_s = (uint32_t*)(a.out + a.groups * kb * kFp8GroupBytes);
  a.gate_up = gate_up, a.f32_scales = scale_kind == CEV_FP8_SCALES_F32;
  const int64_t grid = a.groups * kb;
  if (!fp8_grid_fits(grid, kThreads)) return cev_fail(CEV_ERR_UNSUPPORTED, "cev_fp8_weight_pack: weight too large");
  const int64_t e = a.f32_scales ? 4 : 1;
  CEV_CHECK_ARG(fp8_apart({{weight, 1, 0, (int64_t)need}},
                          {cev_rows(q, n, ldq, k, 1), cev_rows(scales, nb, lds, kb, e), cev_rows(up_q, n, up_ldq, k, 1), cev_rows(up_scales, nb, up_lds, kb, e)}),
                "cev_fp8_weight_pack: the weight must have memory of its own");
  hipLaunchKernelGGL(fp8_pack_kernel, dim3((unsigned)grid), dim3(kThreads), 0, (hipStream_t)stream, a);
  return launched("cev_fp8_weight_pack");
}
