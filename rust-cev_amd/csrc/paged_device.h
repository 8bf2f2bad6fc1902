// Device side of the paged attention's work list.
#pragma once
#include "attn_device.h"
#include "paged.h"

namespace {

// A workgroup's walk over the items of its run.  Lane l loads word l of an
// item, ahead of its use; the values go to scalar registers.
struct PagedWalk {
  const PagedArgs& a;
  int32_t word;
  __device__ __forceinline__ void load(const PagedItem* from) {
    word = ((const int32_t*)from)[min((int)(threadIdx.x & 63), (int)(sizeof(PagedItem) / 4) - 1)];
  }
  __device__ __forceinline__ PagedWalk(const PagedArgs& args, int run) : a(args) { load((const PagedItem*)(a.work + a.first_off) + run); }
  // The item that was loaded; the one behind it is loaded next.
  __device__ __forceinline__ PagedItem item() {
    PagedItem it;
    int32_t* const to = (int32_t*)&it;
#pragma unroll
    for (int i = 0; i < 11; ++i) to[i] = __builtin_amdgcn_readlane(word, i);
    it.reserved = 0;
    load((const PagedItem*)(a.work + a.items_off) + max(it.next, 0));
    return it;
  }
};

// Whether the header is that of the descriptor's plan, without a fault.
__device__ __forceinline__ bool paged_plan_ok(const PagedArgs& a, int list, int& n_parts) {
  const PagedHeader h = *(const PagedHeader*)a.work;
  n_parts = uniform_i32(h.n_parts[list]);
  return uniform_i32((h.sig == a.sig) & (h.bad == 0));
}

// Cache policy of loads and stores that go past the XCD's own L2 (sc1): partial
// results go between workgroups of any XCD.  Fences in their place write back
// and drop the whole L2: a decoding batch's attention took 334 us with 512
// workgroups and 1019 with 4096.
constexpr int kPastL2 = 16;

__device__ __forceinline__ void put_past_l2(__amdgpu_buffer_rsrc_t rs, int at, const f32x4& v, int scalar_at = 0) {
  __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(decltype(__builtin_amdgcn_raw_buffer_load_b128(rs, 0, 0, 0)), v), rs, at, scalar_at, kPastL2);
}
__device__ __forceinline__ void put_past_l2(__amdgpu_buffer_rsrc_t rs, int at, const float2& v) {
  __builtin_amdgcn_raw_buffer_store_b64(__builtin_bit_cast(decltype(__builtin_amdgcn_raw_buffer_load_b64(rs, 0, 0, 0)), v), rs, at, 0, kPastL2);
}
__device__ __forceinline__ void put_past_l2(__amdgpu_buffer_rsrc_t rs, int at, float v) {
  __builtin_amdgcn_raw_buffer_store_b32(__builtin_bit_cast(decltype(__builtin_amdgcn_raw_buffer_load_b32(rs, 0, 0, 0)), v), rs, at, 0, kPastL2);
}
__device__ __forceinline__ f32x4 get4_past_l2(__amdgpu_buffer_rsrc_t rs, int at, int scalar_at = 0) {
  return __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(rs, at, scalar_at, kPastL2));
}
__device__ __forceinline__ float2 get2_past_l2(__amdgpu_buffer_rsrc_t rs, int at) {
  return __builtin_bit_cast(float2, __builtin_amdgcn_raw_buffer_load_b64(rs, at, 0, kPastL2));
}

// An infinity or NaN of V makes its column of every row that sees it the sum of all
// such values, whatever their weights.  (A weight may come out as 0, for which the
// products have NaN, and which weights do depends on how the keys were shared out.)
// The kernels keep what they have found of a value's sum as a bit of `up` (+inf) and
// one of `down` (-inf), both for NaN.
__device__ __forceinline__ void note_odd(float x, bool seen, uint32_t bit, uint32_t& up, uint32_t& down) {
  const bool odd = seen & !__builtin_isfinite(x);
  up |= (odd & !(x < 0.0f)) ? bit : 0u;
  down |= (odd & !(x > 0.0f)) ? bit : 0u;
}
// x, or the sum that was found.
__device__ __forceinline__ float odd_or(float x, uint32_t bit, uint32_t up, uint32_t down) {
  x = (down & bit) ? -INFINITY : x;
  return (up & bit) ? ((down & bit) ? __builtin_nanf("") : INFINITY) : x;
}
__device__ __forceinline__ bool finite4(const f32x4& x) {
  return __builtin_isfinite(x[0]) & __builtin_isfinite(x[1]) & __builtin_isfinite(x[2]) & __builtin_isfinite(x[3]);
}

}  // namespace
