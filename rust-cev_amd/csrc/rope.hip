// Rotary positions of q and k with the stores of k and v into a paged cache.
//
// A pair (a, b) of a row becomes f (a cos t - b sin t, b cos t + a sin t) at
// t = position * inv.  The angle is kept as a fraction of a turn: the host
// gives inv / 2 pi as an integer of 2^-64 turns, and position * step modulo
// 2^64 is the fraction exactly, where a float angle at position 10^6 is off by
// 0.03 rad.  Its two leading bits (rounded) pick the quadrant and the rest, at
// most an eighth of a turn, goes through a polynomial, so no table is read and
// no position is too far.
//
// Each value is read and written once: HBM bounds it.  8192 bf16 tokens of 48
// heads of 128 take 32.9 us, 6.1 TB/s of reads and writes (much of them in the
// MALL); one token 3.0 us, a launch.
#include "cev_device.h"
#include "cev_internal.h"

namespace {

constexpr int kThreads = 256;

struct RopeArgs {
  const void *q_in, *k_in, *v_in;
  void *q_out, *k_out, *v_out;
  const int32_t *pos, *slots;
  const uint64_t* steps;
  int64_t qi_st, qi_sh, ki_st, ki_sh, vi_st, vi_sh, qo_st, qo_sh, ko_sp, ko_st, ko_sh, vo_sp, vo_st, vo_sh;
  int32_t t, hq, hkv, heads, rot, units, interleaved, transposed, page_shift, n_slots;
  int32_t lanes, groups;  // lanes of a token in a workgroup, groups of heads a token is split into
  float factor;
};

// cos and sin of a fraction x / 2^64 of a turn, within 2^-23.  |r| <= pi / 4: the
// first terms that the Taylor sums drop, r^10 / 10! of cos and r^11 / 11! of sin,
// are below 2^-25.
__device__ __forceinline__ void turn_cos_sin(uint64_t x, float& c, float& s) {
  const uint32_t quad = (uint32_t)((x + (1ull << 61)) >> 62);
  const int32_t part = (int32_t)((int64_t)(x - ((uint64_t)quad << 62)) >> 32);  // of 2^-32 turns
  const float r = (float)part * 1.46291807926715968105e-9f;                     // 2 pi / 2^32
  const float r2 = r * r;
  const float cr = 1.0f + r2 * (-0.5f + r2 * (4.16666666666667e-2f + r2 * (-1.38888888888889e-3f + r2 * 2.48015873015873e-5f)));
  const float sr = r + r * r2 * (-1.66666666666667e-1f + r2 * (8.33333333333333e-3f + r2 * (-1.98412698412698e-4f + r2 * 2.75573192239859e-6f)));
  const bool odd = quad & 1;
  const float a = odd ? sr : cr, b = odd ? cr : sr;
  c = ((quad + 1) & 2) ? -a : a;
  s = (quad & 2) ? -b : b;
}

template <typename T>
using Vec = typename std::conditional<sizeof(T) == 2, bf16x8, f32x4>::type;

// A thread turns one unit (two 16-byte vectors: VEC pairs) of a token's
// rows: its angles are made once for all of the thread's heads.  The lanes of
// a token are `units` units of `lanes / units` heads side by side.
template <typename T>
__global__ __launch_bounds__(kThreads) void rope_kernel(RopeArgs a) {
  constexpr int VEC = 16 / sizeof(T);
  const int per_wg = kThreads / a.lanes;
  const int64_t item = (int64_t)blockIdx.x * per_wg + threadIdx.x / a.lanes;
  const int64_t token = item / a.groups;
  const int group = (int)(item - token * a.groups);
  if ((int)threadIdx.x >= per_wg * a.lanes || token >= a.t) return;
  const int lane = threadIdx.x % a.lanes;
  const int side = a.lanes / a.units, unit = lane % a.units;  // heads side by side
  // first values of the unit's two vectors within a row
  const bool turned = unit < a.rot / (2 * VEC);
  int e0 = 2 * VEC * unit, e1 = e0 + VEC;
  if (turned && !a.interleaved) {
    e0 = VEC * unit;
    e1 = e0 + a.rot / 2;
  }
  float c[VEC], s[VEC];
  if (turned) {
    const int64_t p = a.pos[token];
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
      turn_cos_sin((uint64_t)p * a.steps[VEC * unit + i], c[i], s[i]);
      c[i] *= a.factor;
      s[i] *= a.transposed ? -a.factor : a.factor;
    }
  }
  int64_t page = 0, row = token;
  bool store = true;
  if (a.slots) {
    const int32_t slot = a.slots[token];
    store = (uint32_t)slot < (uint32_t)a.n_slots;
    page = slot >> a.page_shift;
    row = slot & ((1 << a.page_shift) - 1);
  }
  for (int h = group * side + lane / a.units; h < a.heads; h += side * a.groups) {
    const T* in;
    T* out;
    bool turn = turned;
    if (h < a.hq) {
      in = (const T*)a.q_in + token * a.qi_st + h * a.qi_sh;
      out = (T*)a.q_out + token * a.qo_st + h * a.qo_sh;
    } else if (h < a.hq + a.hkv) {
      const int k = h - a.hq;
      in = (const T*)a.k_in + token * a.ki_st + k * a.ki_sh;
      out = (T*)a.k_out + page * a.ko_sp + row * a.ko_st + k * a.ko_sh;
      if (!store) continue;
    } else {
      const int k = h - a.hq - a.hkv;
      in = (const T*)a.v_in + token * a.vi_st + k * a.vi_sh;
      out = (T*)a.v_out + page * a.vo_sp + row * a.vo_st + k * a.vo_sh;
      turn = false;
      if (!store) continue;
    }
    Vec<T> x = *(const Vec<T>*)(in + e0), y = *(const Vec<T>*)(in + e1);
    if (turn) {
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        // interleaved: pair i is values 2i, 2i + 1 of the unit
        const int j = 2 * i % VEC;
        if (a.interleaved) {
          Vec<T>& v = i < VEC / 2 ? x : y;
          const float p = (float)v[j], q = (float)v[j + 1];
          v[j] = (T)(p * c[i] - q * s[i]);
          v[j + 1] = (T)(q * c[i] + p * s[i]);
        } else {
          const float p = (float)x[i], q = (float)y[i];
          x[i] = (T)(p * c[i] - q * s[i]);
          y[i] = (T)(q * c[i] + p * s[i]);
        }
      }
    }
    *(Vec<T>*)(out + e0) = x;
    *(Vec<T>*)(out + e1) = y;
  }
}

template <typename T>
int32_t launch(RopeArgs a, int d, hipStream_t stream) {
  constexpr int VEC = 16 / sizeof(T);
  a.units = d / (2 * VEC);
  const int rows = a.heads;
  int side = kThreads / a.units;
  if (side > rows) side = rows;
  if (side > 64 / a.units && a.units <= 64) side = 64 / a.units;
  if (side < 1) side = 1;
  a.lanes = side * a.units;
  const int rounds = (rows + side - 1) / side;
  // Every round of heads is a group of its own, so that they run side by side; for
  // many tokens in bf16 one thread makes a unit's angles for all heads.  48 heads
  // of 128, groups of their own and one group, us: bf16 16 tokens 3.5 and 6.2, 512
  // 5.5 and 7.2, 1024 (65536 threads) 7.9 and 7.7, 8192 39.0 and 32.9; f32, with
  // twice the bytes for an angle, 1024 tokens 10.6 and 11.2, 8192 72.7 and 79.4.
  a.groups = sizeof(T) == 2 && (int64_t)a.t * a.lanes >= 65536 ? 1 : rounds;
  const int per_wg = kThreads / a.lanes;
  const int64_t grid = ((int64_t)a.t * a.groups + per_wg - 1) / per_wg;
  if (grid > INT32_MAX) return cev_fail(CEV_ERR_UNSUPPORTED, "rope grid too large");
  hipLaunchKernelGGL((rope_kernel<T>), dim3((unsigned)grid), dim3(kThreads), 0, stream, a);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return cev_fail(CEV_ERR_HIP, "rope launch: %s", hipGetErrorString(e));
  return CEV_OK;
}

}  // namespace

extern "C" int32_t cev_rope(const cev_rope_desc* d, const void* q_in, const void* k_in, const void* v_in, const int32_t* pos,
                            const uint64_t* steps, const int32_t* slots, void* q_out, void* k_out, void* v_out, cev_stream stream) {
  CEV_CHECK_ARG(d != nullptr, "cev_rope: null descriptor");
  if (d->dtype != CEV_F32 && d->dtype != CEV_BF16) return cev_fail(CEV_ERR_UNSUPPORTED, "cev_rope: dtype %d", d->dtype);
  CEV_CHECK_ARG(d->t >= 0 && d->n_q_heads >= 0 && d->n_kv_heads >= 0 && (int64_t)d->n_q_heads + 2 * (int64_t)d->n_kv_heads <= 65536,
                "cev_rope: t %d, %d q heads, %d kv heads", d->t, d->n_q_heads, d->n_kv_heads);
  if (d->head_dim < 16 || d->head_dim > 256 || d->head_dim % 16)
    return cev_fail(CEV_ERR_UNSUPPORTED, "cev_rope: head_dim %d (a multiple of 16 up to 256)", d->head_dim);
  if (d->rotary_dim < 16 || d->rotary_dim > d->head_dim || d->rotary_dim % 16)
    return cev_fail(CEV_ERR_UNSUPPORTED, "cev_rope: rotary_dim %d (a multiple of 16 up to head_dim %d)", d->rotary_dim, d->head_dim);
  CEV_CHECK_ARG(d->factor == d->factor && d->factor >= -3.0e38f && d->factor <= 3.0e38f, "cev_rope: factor must be finite");
  const int64_t t = d->t, hq = d->n_q_heads, hkv = d->n_kv_heads, al = d->dtype == CEV_BF16 ? 8 : 4;
  // rows of a k or v output: the tokens', or a page's
  const int64_t rows = slots ? d->page_size : t, pages = slots && d->page_size > 0 ? ((int64_t)d->n_slots + d->page_size - 1) / d->page_size : 1;
  const int64_t st[][2] = {{d->qi_stride_t, t},    {d->qi_stride_h, hq},  {d->ki_stride_t, t},     {d->ki_stride_h, hkv}, {d->vi_stride_t, t},
                           {d->vi_stride_h, hkv},  {d->qo_stride_t, t},   {d->qo_stride_h, hq},    {d->ko_stride_p, pages}, {d->ko_stride_t, rows},
                           {d->ko_stride_h, hkv},  {d->vo_stride_p, pages}, {d->vo_stride_t, rows}, {d->vo_stride_h, hkv}};
  for (const auto& s : st) {
    CEV_CHECK_ARG(cev_stride_fits(s[0], s[1]), "cev_rope: stride %lld of %lld rows", (long long)s[0], (long long)s[1]);
    if (s[1] > 1 && s[0] % al) return cev_fail(CEV_ERR_UNSUPPORTED, "cev_rope: strides must be multiples of %lld elements", (long long)al);
  }
  if (slots) {
    CEV_CHECK_ARG(d->n_slots >= 0, "cev_rope: %d slots", d->n_slots);
    CEV_CHECK_ARG(d->page_size >= 1 && (d->page_size & (d->page_size - 1)) == 0, "cev_rope: page_size %d is not a power of two", d->page_size);
  }
  const int64_t outs[][2] = {{d->qo_stride_t, t}, {d->qo_stride_h, hq}, {d->ko_stride_p, pages}, {d->ko_stride_t, rows}, {d->ko_stride_h, hkv},
                             {v_out ? d->vo_stride_p : INT64_MAX, pages}, {v_out ? d->vo_stride_t : INT64_MAX, rows}, {v_out ? d->vo_stride_h : INT64_MAX, hkv}};
  for (const auto& s : outs)
    CEV_CHECK_ARG(s[1] <= 1 || s[0] >= d->head_dim, "cev_rope: rows of an output overlap");
  if (d->t == 0 || d->n_q_heads + d->n_kv_heads == 0) return CEV_OK;
  CEV_CHECK_ARG(pos && steps, "cev_rope: null pos or steps");
  CEV_CHECK_ARG(d->n_q_heads == 0 || (q_in && q_out), "cev_rope: null q buffers");
  CEV_CHECK_ARG(d->n_kv_heads == 0 || (k_in && k_out), "cev_rope: null k buffers");
  CEV_CHECK_ARG((v_in == nullptr) == (v_out == nullptr) && (!v_in || d->n_kv_heads > 0), "cev_rope: v_in and v_out go together, with kv heads");
  CEV_CHECK_ARG((((uintptr_t)q_in | (uintptr_t)k_in | (uintptr_t)v_in | (uintptr_t)q_out | (uintptr_t)k_out | (uintptr_t)v_out) & 15) == 0 &&
                    ((uintptr_t)steps & 7) == 0 && (((uintptr_t)pos | (uintptr_t)slots) & 3) == 0,
                "cev_rope: rows must be 16-byte aligned");
  RopeArgs a{};
  a.q_in = q_in;
  a.k_in = k_in;
  a.v_in = v_in;
  a.q_out = q_out;
  a.k_out = k_out;
  a.v_out = v_out;
  a.pos = pos;
  a.slots = slots;
  a.steps = steps;
  a.qi_st = d->qi_stride_t;
  a.qi_sh = d->qi_stride_h;
  a.ki_st = d->ki_stride_t;
  a.ki_sh = d->ki_stride_h;
  a.vi_st = d->vi_stride_t;
  a.vi_sh = d->vi_stride_h;
  a.qo_st = d->qo_stride_t;
  a.qo_sh = d->qo_stride_h;
  a.ko_sp = d->ko_stride_p;
  a.ko_st = d->ko_stride_t;
  a.ko_sh = d->ko_stride_h;
  a.vo_sp = d->vo_stride_p;
  a.vo_st = d->vo_stride_t;
  a.vo_sh = d->vo_stride_h;
  a.t = d->t;
  a.hq = d->n_q_heads;
  a.hkv = d->n_kv_heads;
  a.heads = a.hq + a.hkv * (v_in ? 2 : 1);
  a.rot = d->rotary_dim;
  a.interleaved = d->interleaved;
  a.transposed = d->transposed;
  a.page_shift = slots ? __builtin_ctz((unsigned)d->page_size) : 0;
  a.n_slots = d->n_slots;
  a.factor = d->factor;
  const hipStream_t s = (hipStream_t)stream;
  return d->dtype == CEV_BF16 ? launch<__bf16>(a, d->head_dim, s) : launch<float>(a, d->head_dim, s);
}
