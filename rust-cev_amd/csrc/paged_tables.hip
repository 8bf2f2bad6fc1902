// A serving step's bookkeeping on the device: pages, block tables, positions
// and slots from the requests' lengths, and the attention's work list.
#include "cev_device.h"
#include "paged.h"

namespace {

// Sums of lower lanes' values by lane moves within rows of 16 lanes and then
// across rows (a bpermute a step takes ten times as long).  Sums saturate, so
// that counts out of their bounds stay so.
__device__ __forceinline__ uint32_t add_sat(uint32_t a, uint32_t b) { return __builtin_elementwise_add_sat(a, b); }
template <typename Op>
__device__ __forceinline__ uint32_t wave_inclusive(uint32_t x, Op op) {
  x = op(x, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x111, 0xF, 0xF, false));  // row_shr:1
  x = op(x, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x112, 0xF, 0xF, false));  // row_shr:2
  x = op(x, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x114, 0xF, 0xF, false));  // row_shr:4
  x = op(x, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x118, 0xF, 0xF, false));  // row_shr:8
  x = op(x, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x142, 0xA, 0xF, false));  // row_bcast:15 to rows 1 and 3
  x = op(x, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x143, 0xC, 0xF, false));  // row_bcast:31 to rows 2 and 3
  return x;
}

// The largest of the workgroup's values.  `part` holds a value a wave; two barriers.
template <int W>
__device__ __forceinline__ uint32_t largest(uint32_t x, uint32_t* part) {
  x = (uint32_t)__builtin_amdgcn_readlane((int)wave_inclusive(x, [](uint32_t a, uint32_t b) { return max(a, b); }), 63);
  if constexpr (W > 1) {
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = x;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < W; ++w) x = max(x, part[w]);
    __syncthreads();
  }
  return x;
}

// N values at once: each becomes the sum of those of all lower threads, total
// that of the whole workgroup.  `part` holds N values a wave; two barriers.
template <int W, int N>
__device__ __forceinline__ void exclusive_sums(uint32_t (&x)[N], uint32_t (&total)[N], uint32_t* part) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  uint32_t own[N];
#pragma unroll
  for (int k = 0; k < N; ++k) {
    own[k] = x[k];
    x[k] = wave_inclusive(x[k], add_sat);
    if constexpr (W == 1)
      total[k] = (uint32_t)__builtin_amdgcn_readlane((int)x[k], 63);
    else if (lane == 63)
      part[wave * N + k] = x[k];
  }
  if constexpr (W > 1) {
    __syncthreads();
#pragma unroll
    for (int k = 0; k < N; ++k) {
      uint32_t before = 0, all = 0;
#pragma unroll
      for (int w = 0; w < W; ++w) {
        const uint32_t p = part[w * N + k];
        before = add_sat(before, w < wave ? p : 0);
        all = add_sat(all, p);
      }
      x[k] = add_sat(x[k], before);
      total[k] = all;
    }
    __syncthreads();
  }
#pragma unroll
  for (int k = 0; k < N; ++k) x[k] = x[k] == UINT32_MAX ? x[k] : x[k] - own[k];
}

// Workgroups of W waves for up to 64 W PER requests.  One wave where it can hold
// them and has little else to do: no barriers (the plan of one request 4.0 us, with
// eight waves 5.0; of 64 decoding ones 4.6 and 5.7).
template <typename Fn>
int32_t by_requests(int32_t n_requests, bool small, Fn&& launch) {
  if (n_requests <= 64 && small) return launch(std::integral_constant<int, 1>{}, std::integral_constant<int, 1>{});
  if (n_requests <= 512) return launch(std::integral_constant<int, 8>{}, std::integral_constant<int, 1>{});
  return launch(std::integral_constant<int, 8>{}, std::integral_constant<int, kPagedMaxRequests / 512>{});
}

constexpr int kTokens = 4;  // packed rows of a thread and round

struct TablesArgs {
  const int32_t *lengths, *new_len, *ring;
  int32_t *block_table, *free_pages, *lengths_out, *ring_out, *cu, *pos, *slots;
  int32_t* arrived;  // workgroups that have read the inputs; null: no output lies in an input's place
  int64_t bt_stride;
  int32_t n_requests, page_shift, n_pages, max_pages, max_tokens;
};

// Every workgroup sums the requests (a few KB that stay in L2) and then
// fills its share of the rows, so no workgroup waits for another and one
// launch does.  What the workgroups read is what no workgroup writes: block
// table entries of cached tokens, ring places [head, head + taken) (places
// [head + count, ...) receive the pages given back: pages are distinct, so
// the two ranges never meet in a ring of n_pages places).  Only the new
// lengths and the new ring state may lie in their inputs' place; the last
// workgroup to have read the inputs writes those then (counted in ring[3], which
// the caller sets up with the rest of the ring).
//
// Of an ended request only the entries that are pages go back (its holder enters
// another value for what the request does not hold), so every workgroup counts
// them first, in steps that end one: 1.8 us for 50 that end among 512.
//
// Bound by the launch and a chain of three trips to memory, four where requests
// end: 3.5 us for 64 requests of one token, 9.0 for 20000 tokens of 512 requests
// (10 workgroups).
template <int W, int PER>
__global__ __launch_bounds__(64 * W) void paged_tables_kernel(TablesArgs a) {
  constexpr int kThreads = 64 * W, kMax = kThreads * PER;
  __shared__ int32_t cu_s[kMax + 1];
  __shared__ int32_t len_s[kMax];
  __shared__ int32_t first_s[kMax];  // pages taken before this request's; ended: -1 - (pages given back before)
  __shared__ uint32_t part[W * 3];
  __shared__ int32_t status_s, last_s;
  const int tid = threadIdx.x, lane = tid & 63;
  const int R = a.n_requests;
  const int page = 1 << a.page_shift;
  if (tid == 0) status_s = 0;
  const int32_t head = a.ring[0], count = a.ring[1];
  int32_t len[PER], add[PER], back[PER];
  uint32_t x[3] = {0, 0, 0};  // new tokens, pages taken, pages given back
  int bad = 0;
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int r = tid * PER + i;
    len[i] = r < R ? a.lengths[r] : 0;
    add[i] = r < R ? a.new_len[r] : 0;
    back[i] = 0;
  }
  const int32_t max_len = a.max_pages << a.page_shift;
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    if (len[i] < 0 || len[i] > max_len || add[i] < -1) {
      bad |= 8;
      len[i] = add[i] = 0;
    }
    if (add[i] > max_len - len[i]) {
      bad |= 2;
      add[i] = 0;
    }
    const int32_t have = (len[i] + page - 1) >> a.page_shift;
    if (add[i] >= 0) {
      x[0] = add_sat(x[0], add[i]);
      x[1] = add_sat(x[1], a.free_pages ? ((len[i] + add[i] + page - 1) >> a.page_shift) - have : 0);
    }
  }
  // What ended requests give back: a wave counts for its own lanes' requests, the
  // entries of kAtOnce of them in a trip to memory.
  constexpr int kAtOnce = 8, kBlocks = 4;
  // Entries j0 + lane, j0 + 64 + lane, ... of a row of n, -1 behind its last one
  // (loads without a branch, or each would be waited for by itself).
  auto entries = [&](const int32_t* row, int j0, int n, int32_t* e) {
#pragma unroll
    for (int b = 0; b < kBlocks; ++b) e[b] = row[max(min(j0 + 64 * b + lane, n - 1), 0)];
  };
  auto is_page = [&](int32_t e, int j, int n) { return j < n && (uint32_t)e < (uint32_t)a.n_pages; };
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    uint64_t ended = a.free_pages ? __ballot(add[i] < 0 && len[i] > 0) : 0;
    while (ended) {
      int from[kAtOnce], n[kAtOnce], longest = 0;
      int32_t count_of[kAtOnce];
#pragma unroll
      for (int k = 0; k < kAtOnce; ++k) {
        // (behind the last one: none of the entries of the one before)
        from[k] = ended ? __builtin_ctzll(ended) : from[k > 0 ? k - 1 : 0];
        n[k] = ended ? (__builtin_amdgcn_readlane(len[i], from[k]) + page - 1) >> a.page_shift : 0;
        count_of[k] = 0;
        longest = max(longest, n[k]);
        ended &= ended - 1;
      }
      for (int j0 = 0; j0 < longest; j0 += 64 * kBlocks) {
        int32_t e[kAtOnce][kBlocks];
#pragma unroll
        for (int k = 0; k < kAtOnce; ++k)
          entries(a.block_table + (int64_t)(((tid & ~63) + from[k]) * PER + i) * a.bt_stride, j0, n[k], e[k]);
#pragma unroll
        for (int k = 0; k < kAtOnce; ++k)
#pragma unroll
          for (int b = 0; b < kBlocks; ++b) count_of[k] += __popcll(__ballot(is_page(e[k][b], j0 + 64 * b + lane, n[k])));
      }
#pragma unroll
      for (int k = 0; k < kAtOnce; ++k) back[i] += lane == from[k] ? count_of[k] : 0;
    }
    x[2] = add_sat(x[2], back[i]);
  }
  uint32_t total[3];
  exclusive_sums<W>(x, total, part);
  if (total[0] > (uint32_t)a.max_tokens) bad |= 1;
  if (a.free_pages) {
    if (head < 0 || head >= a.n_pages || count < 0 || count > a.n_pages)
      bad |= 8;
    else if (total[1] > (uint32_t)count)
      bad |= 4;
    else if (total[2] > (uint32_t)(a.n_pages - count))
      bad |= 8;
  }
  if (W == 1) __syncthreads();  // (status_s is clear; the sums' barriers do it otherwise)
  if (bad) atomicOr(&status_s, bad);
  __syncthreads();
  const int status = status_s;
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int r = tid * PER + i;
    if (r < R) {
      const int32_t have = (len[i] + page - 1) >> a.page_shift;
      cu_s[r] = status ? 0 : (int32_t)x[0];
      len_s[r] = len[i];
      if (add[i] < 0) {
        first_s[r] = (int32_t)(-1 - (int32_t)x[2]);
        x[2] += back[i];
      } else {
        first_s[r] = (int32_t)x[1];
        x[0] += add[i];
        x[1] += a.free_pages ? ((len[i] + add[i] + page - 1) >> a.page_shift) - have : 0;
      }
    }
  }
  const int32_t n = status ? 0 : (int32_t)total[0];
  if (tid == 0) cu_s[R] = n;
  __syncthreads();

  if (blockIdx.x == 0)
    for (int r = tid; r <= R; r += kThreads) a.cu[r] = cu_s[r];
  // Place i of the ring, counted from its head: i < 2 n_pages - head.
  auto place = [&](uint32_t i) {
    const uint32_t at = (uint32_t)head + i;
    return at >= (uint32_t)a.n_pages ? at - (uint32_t)a.n_pages : at;
  };

  // Rows: kTokens in a row to a thread; its first one's request by bisection.
  const int64_t step = (int64_t)gridDim.x * kThreads * kTokens;
  for (int64_t i0 = ((int64_t)blockIdx.x * kThreads + tid) * kTokens; i0 < a.max_tokens; i0 += step) {
    int r = 0;
    if (i0 < n) {
      int hi = R;  // cu_s[r] <= i0 < cu_s[hi]
      while (hi - r > 1) {
        const int mid = (r + hi) >> 1;
        if (cu_s[mid] <= i0) r = mid; else hi = mid;
      }
    }
    int32_t p[kTokens], id[kTokens];
    int32_t* entry[kTokens];  // of a new page's first token
#pragma unroll
    for (int k = 0; k < kTokens; ++k) {
      const int i = (int)i0 + k;
      p[k] = 0;
      id[k] = -1;
      entry[k] = nullptr;
      if (i0 + k < n) {
        while (cu_s[r + 1] <= i) ++r;
        p[k] = len_s[r] + i - cu_s[r];
        const int32_t j = p[k] >> a.page_shift, have = (len_s[r] + page - 1) >> a.page_shift;
        int32_t* const e = a.block_table + r * a.bt_stride + j;
        const bool fresh = a.free_pages && j >= have;
        id[k] = *(fresh ? a.free_pages + place((uint32_t)(first_s[r] + (j - have))) : e);
        entry[k] = fresh && (p[k] & (page - 1)) == 0 ? e : nullptr;
      }
    }
#pragma unroll
    for (int k = 0; k < kTokens; ++k)
      if (i0 + k < a.max_tokens) {
        a.pos[i0 + k] = p[k];
        a.slots[i0 + k] = (uint32_t)id[k] < (uint32_t)a.n_pages ? (id[k] << a.page_shift) + (p[k] & (page - 1)) : -1;
        if (entry[k]) *entry[k] = id[k];
      }
  }

  // Pages of the requests that ended: a wave to a request.
  if (status == 0 && a.free_pages && total[2] > 0)
    for (int r = blockIdx.x * W + (tid >> 6); r < R; r += gridDim.x * W)
      if (first_s[r] < 0) {
        const int32_t have = (len_s[r] + page - 1) >> a.page_shift;
        uint32_t to = (uint32_t)count + (uint32_t)(-1 - first_s[r]);
        for (int j0 = 0; j0 < have; j0 += 64 * kBlocks) {
          int32_t e[kBlocks];
          entries(a.block_table + r * a.bt_stride, j0, have, e);
#pragma unroll
          for (int b = 0; b < kBlocks; ++b) {
            const bool ok = is_page(e[b], j0 + 64 * b + lane, have);
            const uint64_t pages = __ballot(ok);
            if (ok) a.free_pages[place(to + (uint32_t)__popcll(pages & ((1ull << lane) - 1)))] = e[b];
            to += (uint32_t)__popcll(pages);
          }
        }
      }

  if (a.arrived) {
    __syncthreads();
    if (tid == 0) last_s = atomicAdd(a.arrived, 1) == (int)gridDim.x - 1;
    __syncthreads();
    if (!last_s) return;
  } else if (blockIdx.x > 0) {
    return;
  }
  for (int r = tid; r < R; r += kThreads) {
    // (a status leaves the lengths as they were, also those out of bounds)
    if (status)
      a.lengths_out[r] = a.lengths[r];
    else
      a.lengths_out[r] = first_s[r] < 0 ? 0 : len_s[r] + cu_s[r + 1] - cu_s[r];
  }
  if (tid == 0) {
    if (a.arrived) *a.arrived = 0;
    const bool same = status || !a.free_pages;
    a.ring_out[0] = same ? head : (int32_t)place(total[1]);
    a.ring_out[1] = same ? count : count - (int32_t)total[1] + (int32_t)total[2];
    a.ring_out[2] = status;
    a.ring_out[3] = 0;
  }
}

// --------------------------------------------------------------------------
// The attention's work lists.

struct PlanArgs {
  const int32_t *cu, *lengths;
  char* work;
  PagedListBounds list[kPagedLists];
  int32_t n_requests, t, max_new, max_len, window, sinks, hkv;
  uint32_t sig;
  bool bf16, d128;
};

// Requests of more rows than a tile of the first kernel (32 slots) go to the
// second from this many of the first kernel's sub-tiles for each of its
// workgroups on.  With fewer the first has more workgroups at work; with more it
// is bound by reading the keys once for every 32 slots.  First and second kernel,
// d = 128 (32 query over 8 KV heads, us):
//   1 request of 256 slots and  2048 keys (8 sub-tiles a workgroup)   20.6  35.5
//   4 requests of  64 slots and  4096 keys (16)                       25.5  31.7
//   12 requests of 128 slots and 1024 keys (24)                       25.1  26.3
//   16 requests of 64 slots and  2048 keys (32)                       34.9  33.9
//   64 requests of 48 slots and   512 keys (32)                       49.7  36.1
//   64 requests of 64 slots and  2048 keys (128)                       195   117
// d = 256 (16 over 4):
//   16 requests of  64 slots and  2048 keys (32)                      39.7  43.4
//   16 requests of 128 slots and  2048 keys (64)                      48.8  48.2
//   6 requests of 70 to 164 slots and 4000 to 8000 keys (71)          93.7  80.2
//   16 requests of 256 slots and  2048 keys (128)                     92.6  68.1
//   64 requests of 256 slots and  2048 keys (512)                      740   155
//   1 request of 1024 slots and   8192 keys (126), the other way        90   102
constexpr int few_work(bool d128) { return d128 ? 32 : 64; }
static_assert(few_work(true) * 512 < 1 << 18 && few_work(false) * 256 < 1 << 18, "the sum's clip");
// What an item costs beside its sub-tiles (its start, and its partial or final
// result), in sub-tiles.  With 4, 8 and 12 (us): 12 f32 chunks 59.7, 60.4, 60.5; 32
// requests of d = 256 95.6, 92.1, 95.0; 12 f32 chunks of 17 to 41 rows of 4 heads
// 57.5, 53.2, 54.4.
constexpr int kItemCost = 8;
// Pieces of a tile of n_sub sub-tiles where there are workgroups enough for all.
// A piece's sub-tiles take r us each, and joining the pieces takes j us for each
// of them (the last workgroup reads them past its L2), so the best length is near
// sqrt(n_sub j / r); the waves of the kernel of few rows take four sub-tiles at
// once, and up to two of those a wave are not worth a join.  Of a tile that fills
// at most half of its slots less is read.  piece_rate: one over the length.  One
// request, us, against pieces of 16 sub-tiles of the first kernel, 32 of the second:
//   one row, 4 heads a KV head, after  1023 / 4095 keys
//     bf16 d = 128   8.3 (11.4) / 11.0 (12.1)
//     bf16 d = 256  11.1 (16.5) / 14.8 (17.2)    f32  12.5 (23.4) / 15.7 (23.6)
//   32 slots of bf16 d = 128 in 1024 / 4096 keys   13.5 (16.1) / 18.0 (18.1)
//   256 slots of the second kernel                 30.8 (35.9) / 44.9 (69.0)
__device__ __forceinline__ float piece_rate(int list, bool bf16, bool d128, bool half_filled, uint32_t n_sub) {
  const float root = __builtin_amdgcn_sqrtf((float)n_sub);
  float len;
  if (list == kPagedMany)
    len = (d128 ? 2.0f : 2.8f) * root;
  else
    len = n_sub <= 8 ? 8.0f : fmaxf(4.0f, 4.0f * rintf((half_filled ? 0.125f : 0.25f) * (bf16 ? 1.4f : 0.7f) * root));
  return __builtin_amdgcn_rcpf(len);
}
__device__ __forceinline__ uint32_t piece_count(uint32_t n_sub, float rate) { return 1 + (uint32_t)((float)(n_sub - 1) * rate); }

// One workgroup.  A list's tiles are runs of query rows of a request.  When
// there are workgroups enough for every tile in pieces of a good length, each
// piece is a run of its own.  Otherwise the tiles, one after the other, each
// kItemCost longer than its sub-tiles, are cut into as many runs of equal length
// as workgroups run at once, and every piece of a tile that lies in one run is
// an item: all workgroups end together whatever the lengths, and a tile is split
// only where a cut falls.
//
// Sums of sub-tiles are 32-bit: cev_paged_bounds refuses shapes beyond.  4.0 us for
// one request, 4.6 for 64 of one token, 5.6 for 119 tiles of two prompts: a launch,
// a trip to memory, and the sums' lane moves.
template <int W, int PER>
__global__ __launch_bounds__(64 * W) void paged_plan_kernel(PlanArgs a) {
  constexpr int kThreads = 64 * W, kMax = kThreads * PER;
  __shared__ int32_t tiles_s[kMax + 1];  // tiles before each request's
  __shared__ int32_t row_s[kMax], n_s[kMax], pos_s[kMax];
  __shared__ uint32_t part[W * 4];
  __shared__ int32_t bad_s;
  const int tid = threadIdx.x;
  const int R = a.n_requests;
  if (tid == 0) bad_s = 0;
  __syncthreads();
  int32_t rows[PER];
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int r = tid * PER + i;
    rows[i] = 0;
    if (r < R) {
      const int32_t row = a.cu[r], end = a.cu[r + 1], len = a.lengths[r];
      const int64_t n = (int64_t)end - row;
      const bool bad = row < 0 || end > a.t || n < 0 || n > a.max_new || len < n || len > a.max_len;
      if (bad) bad_s = 1;
      rows[i] = bad ? 0 : (int32_t)n;
      row_s[r] = row;
      n_s[r] = rows[i];
      pos_s[r] = bad ? 0 : len - rows[i];
    }
  }
  PagedHeader* const h = (PagedHeader*)a.work;
  int32_t n_parts[kPagedLists];
  // Requests of more rows than a tile of the first kernel go to the second one,
  // which reads their keys once for 256 slots, unless the first one's workgroups
  // have little work with them: it shares a request out to many more.
  int32_t few_rows = INT32_MAX;
  if (a.list[kPagedMany].target > 0) {
    const PagedListBounds& l = a.list[kPagedFew];
    uint32_t work[1] = {0}, all_work[1];
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      if (rows[i] <= l.rows) continue;
      const int32_t pos0 = pos_s[tid * PER + i], pos1 = pos0 + rows[i] - 1;
      const int64_t n_sub = (int64_t)paged_span(l.keys, pos0, pos0 + l.rows - 1, a.window, a.sinks).total +
                            paged_span(l.keys, pos1 - l.rows + 1, pos1, a.window, a.sinks).total;
      work[0] += (uint32_t)min((int64_t)1 << 18, ((rows[i] + l.rows - 1) / l.rows * n_sub) >> 1);
    }
    exclusive_sums<W>(work, all_work, part);
    if (all_work[0] >= (uint32_t)(few_work(a.d128) * l.target)) few_rows = l.rows;
  }
#pragma unroll
  for (int list = 0; list < kPagedLists; ++list) {
    const PagedListBounds& l = a.list[list];
    n_parts[list] = 0;
    if (l.target == 0) continue;
    uint32_t x[3] = {0, 0, 0}, total[3];  // tiles, requests, rows
    int32_t n_tiles[PER];
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      n_tiles[i] = (rows[i] <= few_rows) == (list == kPagedFew) ? (rows[i] + l.rows - 1) / l.rows : 0;
      x[0] += n_tiles[i];
      x[1] += n_tiles[i] > 0;
      x[2] += n_tiles[i] > 0 ? rows[i] : 0;
    }
    exclusive_sums<W>(x, total, part);
    int32_t before = (int32_t)x[0];
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int r = tid * PER + i;
      if (r < R) tiles_s[r] = before;
      before += n_tiles[i];
    }
    const int32_t all = (int32_t)total[0];
    if (tid == 0) tiles_s[R] = all;
    __syncthreads();
    if (bad_s) break;  // (rows of a request beyond its bounds)
    if (all == 0) continue;

    // tile i of the list; its sub-tiles in c_end
    auto tile = [&](int i) {
      int lo = 0, hi = R;  // tiles_s[lo] <= i < tiles_s[hi]
      while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (tiles_s[mid] <= i) lo = mid; else hi = mid;
      }
      // (requests without tiles share their start with the one that has it)
      const int32_t at = (i - tiles_s[lo]) * l.rows;
      PagedItem t{};
      t.row0 = row_s[lo] + at;
      t.n_rows = min(l.rows, n_s[lo] - at);
      t.pos0 = pos_s[lo] + at;
      t.req = lo;
      t.c_end = paged_span(l.keys, t.pos0, t.pos0 + t.n_rows - 1, a.window, a.sinks).total;
      return t;
    };
    // length of all tiles; pieces of them, of twice and of four times the length
    uint32_t sum[4] = {0, 0, 0, 0}, sums[4], longest = 0;
    for (int i = tid; i < all; i += kThreads) {
      const PagedItem t = tile(i);
      const uint32_t n_sub = (uint32_t)t.c_end;
      sum[0] += n_sub + kItemCost;
      longest = max(longest, n_sub);
      const float rate = piece_rate(list, a.bf16, a.d128, 2 * t.n_rows <= l.rows, n_sub);
#pragma unroll
      for (int k = 0; k < 3; ++k) sum[1 + k] += piece_count(n_sub, rate / (float)(1 << k));
    }
    exclusive_sums<W>(sum, sums, part);
    // Two workgroups of few rows of bf16 d = 128 share a CU: short pieces are made
    // longer before that (16 requests of one token after 1023: 15.5 us, 18.1 with
    // two a CU), long ones are not (4 requests of 32 rows after 4064: 29.4 us with
    // two a CU, 35.6 in longer pieces).
    const bool two = list == kPagedFew && a.d128;
    const uint32_t target = (uint32_t)l.target, alone = two ? target / 2 : target;
    const int by = sums[1] <= alone ? 0 : sums[2] <= alone ? 1 : two && sums[3] <= alone && sums[0] <= 24 * sums[3] ? 2 : 1;
    const uint32_t n_pieces = by == 0 ? sums[1] : by == 1 ? sums[2] : sums[3];
    const float shorter = by == 0 ? 1.0f : by == 1 ? 0.5f : 0.25f;
    bool pieces = n_pieces <= target;
    // Length of a run in cuts (longer than a tile's cost, so sub-tiles lie in every
    // one).  Tiles of few rows stream their keys as fast with one run a CU and have
    // fewer joins (64 decoding requests of 64 to 8192 keys 186 us, 196 with two a
    // CU), fuller ones do not (64 requests of 8 rows of 4 heads in 512 keys 30.1 us,
    // 27.4 with two).
    const uint32_t runs = 2 * total[2] <= (uint32_t)(all * l.rows) ? alone : target;
    const uint32_t len = max((sums[0] + runs - 1) / runs, (uint32_t)kItemCost + 1);
    // Tiles of one request that walk the same keys at once read them from memory
    // once.  Where requests have several tiles, pieces of one length for all tiles
    // are taken before cuts, if they are at most half as long again as the runs
    // (d = 128, 12 requests of 9 to 24 rows in 256 to 2048 keys: 26.4 us, 32.9 in
    // cuts; d = 256, 4 requests of 40 rows in 4096 keys: 42.6 us, 63.8 in cuts).
    // f32 is bound by its arithmetic and loses by the longer pieces (6 requests of
    // 9 to 24 rows in 500 to 8000 keys: 68.5 us, 62.0 in cuts).
    uint32_t same = 0;
    if (!pieces && list == kPagedFew && a.bf16 && (uint32_t)all <= target && (uint32_t)all > total[1]) {
      longest = largest<W>(longest, part);
      const uint32_t spare = target - (uint32_t)all, n_sub = sums[0] - (uint32_t)(all * kItemCost);
      same = spare ? min((n_sub + spare - 1) / spare, longest) : longest;
      pieces = 2 * same <= 3 * len;
      if (!pieces) same = 0;
    }

    PagedItem* const first = (PagedItem*)(a.work + l.first_off);
    PagedItem* const items = (PagedItem*)(a.work + l.items_off);
    uint32_t units = 0, base[3] = {0, 0, 0};  // length so far; items, partial results and split tiles
    for (int i0 = 0; i0 < all; i0 += kThreads) {
      const int i = i0 + tid;
      PagedItem t{};
      if (i < all) t = tile(i);
      const uint32_t n_sub = (uint32_t)t.c_end;
      uint32_t u[1] = {n_sub ? n_sub + kItemCost : 0}, u_all[1];
      exclusive_sums<W>(u, u_all, part);
      // run r is [r len, (r + 1) len); a tile's cost comes before its sub-tiles
      const uint32_t from = units + u[0], keys = from + kItemCost, to = keys + n_sub;
      const uint32_t r0 = keys / len, r1 = n_sub ? (to - 1) / len : 0;
      uint32_t n = 0;
      if (n_sub && !pieces)
        n = r1 - r0 + 1;
      else if (n_sub && same)
        n = (n_sub + same - 1) / same;
      else if (n_sub)
        n = piece_count(n_sub, piece_rate(list, a.bf16, a.d128, 2 * t.n_rows <= l.rows, n_sub) * shorter);
      uint32_t y[3] = {n, n > 1 ? n : 0, n > 1 ? 1u : 0u}, y_all[3];
      exclusive_sums<W>(y, y_all, part);
      t.n_pieces = (int32_t)n;
      t.rec = (int32_t)(base[1] + y[1]);
      t.split = (int32_t)(base[2] + y[2]);
      const float step = (float)n_sub * __builtin_amdgcn_rcpf((float)n);
      for (uint32_t k = 0; k < n; ++k) {
        const uint32_t at = base[0] + y[0] + k, begin = (r0 + k) * len, end = begin + len;
        t.piece = (int32_t)k;
        if (pieces) {
          t.c_begin = k ? t.c_end : 0;
          t.c_end = (int32_t)(k + 1 < n ? (uint32_t)((float)(k + 1) * step) : n_sub);
          t.next = -1;
        } else {
          t.c_begin = (int32_t)(max(begin, keys) - keys);
          t.c_end = (int32_t)(min(end, to) - keys);
          // the run goes on with the next tile when that tile's sub-tiles begin in it
          t.next = to + kItemCost < end && i + 1 < all ? (int32_t)at + 1 : -1;
        }
        if (at < (uint32_t)l.items) {
          items[at] = t;
          // a run begins here when no tile before has sub-tiles in it
          if (pieces)
            first[at] = t;
          else if (begin >= from)
            first[r0 + k] = t;
        }
      }
      units += u_all[0];
#pragma unroll
      for (int k = 0; k < 3; ++k) base[k] += y_all[k];
    }
    if (tid == 0 && base[0] > (uint32_t)l.items) bad_s = 1;
    for (int i = tid; i < (int)base[2] * a.hkv; i += kThreads) ((int32_t*)(a.work + l.counters_off))[i] = 0;
    n_parts[list] = (int32_t)(pieces ? base[0] : (sums[0] + len - 1) / len);
    __syncthreads();
  }
  if (tid == 0) *h = PagedHeader{a.sig, bad_s, {bad_s ? 0 : n_parts[0], bad_s ? 0 : n_parts[1]}};
}

}  // namespace

extern "C" int32_t cev_paged_tables(int32_t n_requests, int32_t page_size, int32_t n_pages, int32_t max_pages, int32_t max_tokens,
                                    const int32_t* lengths, const int32_t* new_len, int32_t* block_table, int64_t bt_stride,
                                    int32_t* free_pages, int32_t* ring, int32_t* lengths_out, int32_t* ring_out, int32_t* cu,
                                    int32_t* pos, int32_t* slots, cev_stream stream) {
  CEV_CHECK_ARG(n_requests >= 1, "cev_paged_tables: %d requests", n_requests);
  if (n_requests > kPagedMaxRequests)
    return cev_fail(CEV_ERR_UNSUPPORTED, "cev_paged_tables: %d requests (at most %d)", n_requests, kPagedMaxRequests);
  CEV_CHECK_ARG(page_size >= 1 && (page_size & (page_size - 1)) == 0, "cev_paged_tables: page_size %d is not a power of two", page_size);
  CEV_CHECK_ARG(n_pages >= 1 && max_pages >= 1 && max_tokens >= 0, "cev_paged_tables: n_pages %d, max_pages %d, max_tokens %d", n_pages,
                max_pages, max_tokens);
  CEV_CHECK_ARG((int64_t)n_pages * page_size <= INT32_MAX && (int64_t)max_pages * page_size <= INT32_MAX - page_size,
                "cev_paged_tables: %d pages (%d a request) of %d slots overflow the slot index", n_pages, max_pages, page_size);
  CEV_CHECK_ARG(bt_stride >= 0 && (n_requests == 1 || bt_stride >= max_pages), "cev_paged_tables: block table stride %lld",
                (long long)bt_stride);
  CEV_CHECK_ARG(lengths && new_len && block_table && ring && lengths_out && ring_out && cu, "cev_paged_tables: null argument");
  CEV_CHECK_ARG(max_tokens == 0 || (pos && slots), "cev_paged_tables: null pos or slots");
  auto cut = [](const int32_t* x, const int32_t* y, int32_t n) {  // the same place, or apart
    const int64_t by = (int64_t)((uintptr_t)x - (uintptr_t)y);
    return by != 0 && by < 4 * (int64_t)n && -by < 4 * (int64_t)n;
  };
  CEV_CHECK_ARG(!cut(lengths, lengths_out, n_requests) && !cut(ring, ring_out, 4),
                "cev_paged_tables: an output overlaps its input without being the same");
  TablesArgs a;
  a.lengths = lengths;
  a.new_len = new_len;
  a.ring = ring;
  a.block_table = block_table;
  a.free_pages = free_pages;
  a.lengths_out = lengths_out;
  a.ring_out = ring_out;
  a.cu = cu;
  a.pos = pos;
  a.slots = slots;
  a.bt_stride = bt_stride;
  a.n_requests = n_requests;
  a.page_shift = __builtin_ctz((unsigned)page_size);
  a.n_pages = n_pages;
  a.max_pages = max_pages;
  a.max_tokens = max_tokens;
  return by_requests(n_requests, max_tokens <= 64 * kTokens, [&](auto w_c, auto per_c) {
    constexpr int W = decltype(w_c)::value, PER = decltype(per_c)::value, rows = 64 * W * kTokens;
    const int64_t grid = ((int64_t)max_tokens + rows - 1) / rows;
    a.arrived = grid > 1 && (lengths == lengths_out || ring == ring_out) ? ring + 3 : nullptr;
    hipLaunchKernelGGL((paged_tables_kernel<W, PER>), dim3((unsigned)(grid < 1 ? 1 : grid > 256 ? 256 : grid)), dim3(64 * W), 0,
                       (hipStream_t)stream, a);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return cev_fail(CEV_ERR_HIP, "paged tables launch: %s", hipGetErrorString(e));
    return (int32_t)CEV_OK;
  });
}

extern "C" int32_t cev_paged_plan(const cev_paged_desc* d, const int32_t* cu, const int32_t* lengths, void* work, size_t work_bytes,
                                  cev_stream stream) {
  PagedBounds b;
  const int32_t rc = cev_paged_bounds(d, &b);
  if (rc) return rc;
  CEV_CHECK_ARG(cu && lengths && work, "cev_paged_plan: null argument");
  CEV_CHECK_ARG(((uintptr_t)work & 15) == 0, "cev_paged_plan: the work buffer must be 16-byte aligned");
  if (work_bytes < b.bytes) return cev_fail(CEV_ERR_SPACE, "cev_paged_plan: work buffer of %zu bytes, %zu needed", work_bytes, b.bytes);
  PlanArgs a;
  a.cu = cu;
  a.lengths = lengths;
  a.work = (char*)work;
  for (int i = 0; i < kPagedLists; ++i) a.list[i] = b.list[i];
  a.n_requests = d->n_requests;
  a.t = d->t;
  a.max_new = d->max_new;
  a.max_len = b.max_len;
  a.window = d->window;
  a.sinks = d->sinks;
  a.hkv = d->n_kv_heads;
  a.sig = b.sig;
  a.bf16 = d->dtype == CEV_BF16;
  a.d128 = a.bf16 && d->head_dim == 128;
  // one wave where a lane has a few tiles at most
  const PagedListBounds& most = b.list[b.list[kPagedMany].target ? kPagedMany : kPagedFew];
  const int64_t tiles = (int64_t)most.items - most.target;
  return by_requests(d->n_requests, tiles <= 256, [&](auto w_c, auto per_c) {
    constexpr int W = decltype(w_c)::value, PER = decltype(per_c)::value;
    hipLaunchKernelGGL((paged_plan_kernel<W, PER>), dim3(1), dim3(64 * W), 0, (hipStream_t)stream, a);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return cev_fail(CEV_ERR_HIP, "paged plan launch: %s", hipGetErrorString(e));
    return (int32_t)CEV_OK;
  });
}
