// Device side of the paged attention's work list.
#pragma once
#include "attn_device.h"
#include "paged.h"

namespace {

// The first item of workgroup run `run`, and the one behind its last.  (The
// work buffer is written by the kernels too, so its loads are vector loads; the
// values are the same in every lane and go to scalar registers.)
__device__ __forceinline__ int paged_first_item(const PagedArgs& a, int run, int& end) {
  const int32_t* const first = (const int32_t*)(a.work + a.first_off) + run;
  end = uniform_i32(first[1]);
  return uniform_i32(first[0]);
}

__device__ __forceinline__ PagedItem paged_item(const PagedArgs& a, int item) {
  const int32_t* const w = (const int32_t*)((const PagedItem*)(a.work + a.items_off) + item);
  PagedItem it;
  int32_t* const to = (int32_t*)&it;
#pragma unroll
  for (int i = 0; i < 10; ++i) to[i] = uniform_i32(w[i]);
  it.reserved0 = it.reserved1 = 0;
  return it;
}

}  // namespace
