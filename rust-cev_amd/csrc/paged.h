// What the paged-cache code shares: the work buffer of an attention pass
// (written on the device by the plan kernel, read by the attention kernels)
// and the host's bounds on it.
#pragma once
#include <stddef.h>
#include <stdint.h>

#include "cev_internal.h"

constexpr int kPagedMaxRequests = 4096;

// The two kernels and their work lists: requests with few new rows go to the
// first, those with many to the second where the plan kernel finds enough work in
// them (few_work in paged_tables.hip; cev_paged_bounds says whether a shape has a
// second list at all).
constexpr int kPagedFew = 0, kPagedMany = 1, kPagedLists = 2;
// Query slots (rows x heads of a group) of a tile and keys of a sub-tile of heads of d.
constexpr int paged_slots(int list) { return list == kPagedFew ? 32 : 256; }
constexpr int paged_keys(int list, int d) { return list == kPagedMany && d == 128 ? 64 : 32; }

// The work buffer: this header, then for each list the first item of every
// workgroup's run, all items, one arrival counter for every (split tile, KV
// head), and the split tiles' partial results.
struct PagedHeader {
  uint32_t sig;                   // signature of the descriptor that the plan was made for
  int32_t bad;                    // not 0: a length, offset or count was out of its bounds
  int32_t n_parts[kPagedLists];   // workgroups (for each KV head) with work
};

// One work item: a run of query rows of one request (a tile) and a run of the
// key sub-tiles that they see.  A workgroup walks its run's items in order.
struct PagedItem {
  int32_t row0, n_rows, pos0, req;         // first packed row, rows, position of the first
  int32_t c_begin, c_end, piece, n_pieces; // key sub-tiles [c_begin, c_end) of the tile's stream
  int32_t rec, split;                      // first partial result and counter of a split tile
  int32_t next;                            // the run's next item, -1 behind the last
  int32_t reserved;
};
static_assert(sizeof(PagedHeader) == 16 && sizeof(PagedItem) == 48, "work buffer layout");

struct PagedListBounds {
  int32_t rows;      // query rows of a tile
  int32_t keys;      // keys of a sub-tile
  int32_t target;    // most workgroups, for each KV head (0: no request can be in the list)
  int32_t items;     // most items
  size_t first_off, items_off, counters_off, records_off;
};
// What a descriptor bounds: sizes and offsets of the work buffer's parts.
struct PagedBounds {
  int32_t max_len;     // most keys of a request
  uint32_t sig;
  size_t bytes;
  PagedListBounds list[kPagedLists];
};

// Checks d and gives its bounds.
int32_t cev_paged_bounds(const cev_paged_desc* d, PagedBounds* b);

// Launch arguments of the attention kernels.
struct PagedArgs {
  const void *q, *kc, *vc;
  const int32_t* bt;
  void* out;
  char* work;
  size_t first_off, items_off, counters_off, records_off;
  int64_t q_st, q_sh, kc_sp, kc_st, kc_sh, vc_sp, vc_st, vc_sh, o_st, o_sh, bt_stride;
  int32_t hkv, g, t, page_shift, n_pages, max_pages, window, sinks;
  float scale_log2;
  uint32_t sig;
};
// The kernel of tiles of 256 query slots (paged_tile.hip).
int32_t cev_paged_tile_launch(const PagedArgs& a, int32_t d, int32_t target, void* stream);

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
PAGED_HD inline PagedSpan paged_span(int32_t keys, int32_t pos0, int32_t pos1, int32_t window, int32_t sinks) {
  PagedSpan s{0, 0, 0, 0, 0, pos1 + 1};
  if (window > 0 && pos0 >= window) {
    const int32_t lo = pos0 - window + 1;
    if (sinks < lo) {
      s.skip_lo = sinks;
      s.skip_hi = lo;
      s.sinks = (sinks + keys - 1) / keys;
      s.first = lo / keys;
      if (s.first < s.sinks) s.sinks = s.first = 0;  // the gap lies inside one sub-tile
    }
  }
  s.total = s.sinks + (s.end + keys - 1) / keys - s.first;
  return s;
}
