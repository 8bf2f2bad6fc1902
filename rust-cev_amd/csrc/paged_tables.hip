// A serving step's bookkeeping on the device: pages, block tables, positions
// and slots from the requests' lengths, and the attention's work list.
#include "cev_device.h"
#include "paged.h"

namespace {

constexpr int kThreads = 512;
constexpr int kWaves = kThreads / 64;
constexpr int kPerThread = kPagedMaxRequests / kThreads;  // requests of a thread
constexpr int kTokens = 4;                                // packed rows of a thread and round

// Sums of the values of all lower lanes and waves (and of the whole
// workgroup), N values at once.  `part` holds kWaves * N values; two barriers.
template <int N>
__device__ __forceinline__ void exclusive_sums(int64_t (&x)[N], int64_t (&total)[N], int64_t* part) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  int64_t own[N];
#pragma unroll
  for (int k = 0; k < N; ++k) {
    own[k] = x[k];
#pragma unroll
    for (int s = 1; s < 64; s <<= 1) {
      const int64_t y = __shfl_up(x[k], s, 64);
      if (lane >= s) x[k] += y;
    }
    if (lane == 63) part[wave * N + k] = x[k];
  }
  __syncthreads();
#pragma unroll
  for (int k = 0; k < N; ++k) {
    int64_t before = 0, all = 0;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
      const int64_t p = part[w * N + k];
      before += w < wave ? p : 0;
      all += p;
    }
    x[k] += before - own[k];
    total[k] = all;
  }
  __syncthreads();
}

struct TablesArgs {
  const int32_t *lengths, *new_len, *ring;
  int32_t *block_table, *free_pages, *lengths_out, *ring_out, *cu, *pos, *slots;
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
// workgroup to have read the inputs writes those.
__global__ __launch_bounds__(kThreads) void paged_tables_kernel(TablesArgs a) {
  __shared__ int32_t cu_s[kPagedMaxRequests + 1];
  __shared__ int32_t len_s[kPagedMaxRequests];
  __shared__ int32_t first_s[kPagedMaxRequests];  // pages taken before this request's; ended: -1 - (pages given back before)
  __shared__ int64_t part[kWaves * 3];
  __shared__ int32_t status_s, last_s;
  const int tid = threadIdx.x, lane = tid & 63;
  const int R = a.n_requests, per = (R + kThreads - 1) / kThreads;
  const int page = 1 << a.page_shift;
  if (tid == 0) status_s = 0;
  const int64_t head = a.ring[0], count = a.ring[1];
  int32_t len[kPerThread], add[kPerThread];
  int64_t x[3] = {0, 0, 0};  // new tokens, pages taken, pages given back
  int bad = 0;
#pragma unroll
  for (int i = 0; i < kPerThread; ++i) {
    const int r = tid * per + i;
    const bool ok = i < per && r < R;
    len[i] = ok ? a.lengths[r] : 0;
    add[i] = ok ? a.new_len[r] : 0;
  }
  const int32_t max_len = a.max_pages << a.page_shift;
#pragma unroll
  for (int i = 0; i < kPerThread; ++i) {
    if (len[i] < 0 || len[i] > max_len || add[i] < -1) {
      bad |= 8;
      len[i] = add[i] = 0;
    }
    if (add[i] > max_len - len[i]) {
      bad |= 2;
      add[i] = 0;
    }
    const int32_t have = (len[i] + page - 1) >> a.page_shift;
    if (add[i] < 0) {
      x[2] += a.free_pages ? have : 0;
    } else {
      x[0] += add[i];
      x[1] += a.free_pages ? ((len[i] + add[i] + page - 1) >> a.page_shift) - have : 0;
    }
  }
  int64_t total[3];
  exclusive_sums(x, total, part);
  if (total[0] > a.max_tokens) bad |= 1;
  if (a.free_pages) {
    if (head < 0 || head >= a.n_pages || count < 0 || count > a.n_pages)
      bad |= 8;
    else if (total[1] > count)
      bad |= 4;
    else if (count + total[2] > a.n_pages)
      bad |= 8;
  }
  if (bad) atomicOr(&status_s, bad);
  __syncthreads();
  const int status = status_s;
#pragma unroll
  for (int i = 0; i < kPerThread; ++i) {
    const int r = tid * per + i;
    if (i < per && r < R) {
      const int32_t have = (len[i] + page - 1) >> a.page_shift;
      cu_s[r] = status ? 0 : (int32_t)x[0];
      len_s[r] = len[i];
      if (add[i] < 0) {
        first_s[r] = (int32_t)(-1 - x[2]);
        x[2] += a.free_pages ? have : 0;
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
    int32_t p[kTokens], sl[kTokens];
#pragma unroll
    for (int k = 0; k < kTokens; ++k) {
      const int i = (int)i0 + k;
      p[k] = 0;
      sl[k] = -1;
      if (i0 + k < n) {
        while (cu_s[r + 1] <= i) ++r;
        p[k] = len_s[r] + i - cu_s[r];
        const int32_t j = p[k] >> a.page_shift, have = (len_s[r] + page - 1) >> a.page_shift;
        int32_t* const entry = a.block_table + r * a.bt_stride + j;
        int32_t id;
        if (a.free_pages && j >= have) {
          id = a.free_pages[(head + first_s[r] + (j - have)) % a.n_pages];
          if ((p[k] & (page - 1)) == 0) *entry = id;
        } else {
          id = *entry;
        }
        sl[k] = (uint32_t)id < (uint32_t)a.n_pages ? (id << a.page_shift) + (p[k] & (page - 1)) : -1;
      }
    }
#pragma unroll
    for (int k = 0; k < kTokens; ++k)
      if (i0 + k < a.max_tokens) {
        a.pos[i0 + k] = p[k];
        a.slots[i0 + k] = sl[k];
      }
  }

  // Pages of the requests that ended: a wave to a request.
  if (status == 0 && a.free_pages && total[2] > 0)
    for (int r = blockIdx.x * kWaves + (tid >> 6); r < R; r += gridDim.x * kWaves)
      if (first_s[r] < 0) {
        const int32_t have = (len_s[r] + page - 1) >> a.page_shift;
        for (int j = lane; j < have; j += 64)
          a.free_pages[(head + count + (-1 - first_s[r]) + j) % a.n_pages] = a.block_table[r * a.bt_stride + j];
      }

  if (gridDim.x > 1) {
    __syncthreads();
    if (tid == 0) last_s = atomicAdd(&a.ring_out[3], 1) == (int)gridDim.x - 1;
    __syncthreads();
    if (!last_s) return;
  }
  for (int r = tid; r < R; r += kThreads) {
    // (a status leaves the lengths as they were, also those out of bounds)
    if (status)
      a.lengths_out[r] = a.lengths[r];
    else
      a.lengths_out[r] = first_s[r] < 0 ? 0 : len_s[r] + cu_s[r + 1] - cu_s[r];
  }
  if (tid == 0) {
    a.ring_out[0] = (int32_t)(status || !a.free_pages ? head : (head + total[1]) % a.n_pages);
    a.ring_out[1] = (int32_t)(status || !a.free_pages ? count : count - total[1] + total[2]);
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
};

// What an item costs beside its sub-tiles (its start, and its partial or final
// result), in sub-tiles; and the least that a run is worth, in the same.
constexpr int kItemCost = 8, kMinRun = 16;
static_assert(kMinRun > kItemCost, "no run without a sub-tile");

// One workgroup.  A list's tiles (runs of query rows of a request), one after
// the other, are a row of key sub-tiles, each tile kItemCost longer than its
// own; it is cut into as many runs of equal length as workgroups run at once,
// and every piece of a tile that lies in one run is an item.  So all workgroups
// end together whatever the lengths, and a tile is split only where a cut
// falls.
__global__ __launch_bounds__(kThreads) void paged_plan_kernel(PlanArgs a) {
  __shared__ int32_t tiles_s[kPagedMaxRequests + 1];  // tiles before each request's
  __shared__ int32_t row_s[kPagedMaxRequests], n_s[kPagedMaxRequests], pos_s[kPagedMaxRequests];
  __shared__ int64_t part[kWaves * 3];
  __shared__ int32_t bad_s;
  const int tid = threadIdx.x;
  const int R = a.n_requests, per = (R + kThreads - 1) / kThreads;
  if (tid == 0) bad_s = 0;
  __syncthreads();
  int32_t rows[kPerThread];
#pragma unroll
  for (int i = 0; i < kPerThread; ++i) {
    const int r = tid * per + i;
    rows[i] = 0;
    if (i < per && r < R) {
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
#pragma unroll
  for (int list = 0; list < kPagedLists; ++list) {
    const PagedListBounds& l = a.list[list];
    n_parts[list] = 0;
    if (l.max_new < l.min_new) continue;
    int64_t x[1] = {0}, total[1];
    int32_t n_tiles[kPerThread];
#pragma unroll
    for (int i = 0; i < kPerThread; ++i) {
      n_tiles[i] = rows[i] >= l.min_new && rows[i] <= l.max_new ? (rows[i] + l.rows - 1) / l.rows : 0;
      x[0] += n_tiles[i];
    }
    exclusive_sums(x, total, part);
    int32_t before = (int32_t)x[0];
#pragma unroll
    for (int i = 0; i < kPerThread; ++i) {
      const int r = tid * per + i;
      if (i < per && r < R) tiles_s[r] = before;
      before += n_tiles[i];
    }
    const int32_t all = (int32_t)total[0];
    if (tid == 0) tiles_s[R] = all;
    __syncthreads();
    if (bad_s) break;  // (rows of a request beyond its bounds)

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
      t.c_end = paged_span(kPagedKeys[list], t.pos0, t.pos0 + t.n_rows - 1, a.window, a.sinks).total;
      return t;
    };
    int64_t sum[1] = {0};
    for (int i = tid; i < all; i += kThreads) sum[0] += tile(i).c_end + kItemCost;
    exclusive_sums(sum, total, part);
    // (a run is longer than a tile's cost, so sub-tiles lie in every run)
    const int64_t T = total[0], P = T == 0 ? 0 : max(min(T / kMinRun, (int64_t)l.target), (int64_t)1);

    PagedItem* const first = (PagedItem*)(a.work + l.first_off);
    PagedItem* const items = (PagedItem*)(a.work + l.items_off);
    int64_t units = 0, base[3] = {0, 0, 0};  // length so far; items, partial results and split tiles
    for (int i0 = 0; i0 < all; i0 += kThreads) {
      const int i = i0 + tid;
      PagedItem t{};
      if (i < all) t = tile(i);
      const int32_t n_sub = t.c_end;
      int64_t u[1] = {n_sub ? n_sub + kItemCost : 0}, u_all[1];
      exclusive_sums(u, u_all, part);
      // run r is [r T / P, (r + 1) T / P); a tile's cost comes before its sub-tiles
      const int64_t from = units + u[0], keys = from + kItemCost, to = keys + n_sub;
      const int64_t r0 = n_sub ? ((keys + 1) * P - 1) / T : 0, r1 = n_sub ? (to * P - 1) / T : -1;
      const int64_t n = r1 - r0 + 1;
      int64_t y[3] = {n, n > 1 ? n : 0, n > 1 ? 1 : 0}, sums[3];
      exclusive_sums(y, sums, part);
      t.n_pieces = (int32_t)n;
      t.rec = (int32_t)(base[1] + y[1]);
      t.split = (int32_t)(base[2] + y[2]);
      for (int64_t r = r0; r <= r1; ++r) {
        const int64_t begin = r * T / P, end = (r + 1) * T / P, at = base[0] + y[0] + (r - r0);
        t.c_begin = (int32_t)(max(begin, keys) - keys);
        t.c_end = (int32_t)(min(end, to) - keys);
        t.piece = (int32_t)(r - r0);
        // the run goes on with the next tile when that tile's sub-tiles begin in it
        t.next = to + kItemCost < end && i + 1 < all ? (int32_t)at + 1 : -1;
        // it begins here when no tile before has sub-tiles in it
        if (at < l.items) {
          items[at] = t;
          if (begin >= from) first[r] = t;
        }
      }
      units += u_all[0];
#pragma unroll
      for (int k = 0; k < 3; ++k) base[k] += sums[k];
    }
    if (tid == 0 && base[0] > l.items) bad_s = 1;
    for (int i = tid; i < (int)base[2] * a.hkv; i += kThreads) ((int32_t*)(a.work + l.counters_off))[i] = 0;
    n_parts[list] = (int32_t)P;
    __syncthreads();
  }
  if (tid == 0) *h = PagedHeader{a.sig, bad_s, {bad_s ? 0 : n_parts[0], bad_s ? 0 : n_parts[1]}};
}

}  // namespace

extern "C" int32_t cev_paged_tables(int32_t n_requests, int32_t page_size, int32_t n_pages, int32_t max_pages, int32_t max_tokens,
                                    const int32_t* lengths, const int32_t* new_len, int32_t* block_table, int64_t bt_stride,
                                    int32_t* free_pages, const int32_t* ring, int32_t* lengths_out, int32_t* ring_out, int32_t* cu,
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
  const int64_t grid = ((int64_t)max_tokens + kThreads * kTokens - 1) / (kThreads * kTokens);
  hipLaunchKernelGGL(paged_tables_kernel, dim3((unsigned)(grid < 1 ? 1 : grid > 256 ? 256 : grid)), dim3(kThreads), 0, (hipStream_t)stream, a);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return cev_fail(CEV_ERR_HIP, "paged tables launch: %s", hipGetErrorString(e));
  return CEV_OK;
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
  hipLaunchKernelGGL(paged_plan_kernel, dim3(1), dim3(kThreads), 0, (hipStream_t)stream, a);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return cev_fail(CEV_ERR_HIP, "paged plan launch: %s", hipGetErrorString(e));
  return CEV_OK;
}
