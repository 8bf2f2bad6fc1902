// What the paged-cache code shares: the work buffer of an attention pass
// (written on the device by the plan kernel, read by the attention kernels)
// and the host's bounds on it.
#pragma once
#include <stddef.h>
#include <stdint.h>

#include "cev_internal.h"

// The work buffer: a header, the lists of work items, one arrival counter
// for every (split tile, KV head), then the split tiles' partial results.
struct PagedHeader {
  uint32_t sig;     // signature of the descriptor that the plan was made for
  int32_t bad;      // not 0: a length, offset or count was out of its bounds
  int32_t n_items;  // items of the list
  int32_t reserved;
};

// One work item: a run of query rows of one request and a part of the key
// sub-tiles that they see.
struct PagedItem {
  int32_t row0, n_rows, pos0, req;         // first packed row, rows, position of the first
  int32_t c_begin, c_end, part, n_parts;   // key sub-tiles [c_begin, c_end) of the rows' stream
  int32_t rec, split, reserved0, reserved1;  // first partial record and counter of a split tile
};
static_assert(sizeof(PagedHeader) == 16 && sizeof(PagedItem) == 48, "work buffer layout");

constexpr int kPagedSlots = 32;     // query slots (rows x heads of a group) of an item
constexpr int kPagedKeys = 32;      // keys of a sub-tile
constexpr int kPagedTarget = 4096;   // workgroups that a launch is split into (two for each CU)
constexpr int kPagedMaxRequests = 4096;

// What a descriptor bounds: sizes and offsets of the work buffer's parts.
struct PagedBounds {
  int32_t rows;        // query rows of an item
  int32_t target;      // parts that the whole launch's keys are cut into, per KV head
  int32_t items;       // most items
  int32_t max_len;     // most keys of a request
  uint32_t sig;
  size_t items_off, counters_off, records_off, bytes;
};

// Checks d and gives its bounds.
int32_t cev_paged_bounds(const cev_paged_desc* d, PagedBounds* b);

// The key sub-tiles that query rows at positions [pos0, pos1] see, in stream
// order: `sinks` sub-tiles from key 0, then those from `first` on.  Keys from
// skip_lo to skip_hi (between the first tokens that stay visible and the
// window) are seen by none of the rows.
struct PagedSpan {
  int32_t sinks, first, total, skip_lo, skip_hi, end;
};
#ifdef __HIPCC__
#define PAGED_HD __host__ __device__
#else
#define PAGED_HD
#endif
template <int KEYS>
PAGED_HD inline PagedSpan paged_span(int32_t pos0, int32_t pos1, int32_t window, int32_t sinks) {
  PagedSpan s{0, 0, 0, 0, 0, pos1 + 1};
  if (window > 0 && pos0 >= window) {
    const int32_t lo = pos0 - window + 1;
    if (sinks < lo) {
      s.skip_lo = sinks;
      s.skip_hi = lo;
      s.sinks = (sinks + KEYS - 1) / KEYS;
      s.first = lo / KEYS;
      if (s.first < s.sinks) s.sinks = s.first = 0;  // the gap lies inside one sub-tile
    }
  }
  s.total = s.sinks + (s.end + KEYS - 1) / KEYS - s.first;
  return s;
}
