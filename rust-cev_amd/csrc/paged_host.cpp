// Host side of the paged-cache operators: descriptors, the bounds of an
// attention pass's work buffer and the rotary angles.
#include <math.h>
#include <string.h>

#include "paged.h"

namespace {

bool power_of_two(int32_t x) { return x > 0 && (x & (x - 1)) == 0; }

// Workgroups that the keys of a launch are shared out to: as many as run at
// once (256 CUs; two workgroups of the first kernel share one for bf16 heads
// of 128, by their LDS).  With twice as many, us: 48 decoding requests 49.1 for 46.2,
// d = 256 113.7 for 91.8, f32 69.3 for 58.3, a window's chunk 201.9 for 185.5.
constexpr int32_t kFewWorkgroups128 = 512, kFewWorkgroups = 256, kManyWorkgroups = 256;

size_t align_up(size_t x) { return (x + 255) & ~(size_t)255; }

// FNV-1a over the fields that a plan depends on.
uint32_t signature(const cev_paged_desc* d) {
  const int32_t words[] = {d->dtype,   d->n_q_heads, d->n_kv_heads, d->head_dim,  d->n_requests, d->t,
                           d->max_new, d->page_size, d->n_pages,    d->max_pages, d->window,     d->sinks};
  uint32_t h = 2166136261u;
  for (int32_t w : words)
    for (int b = 0; b < 4; ++b) h = (h ^ ((uint32_t)w >> (8 * b) & 255u)) * 16777619u;
  return h ? h : 1u;
}

}  // namespace

extern "C" int32_t cev_paged_desc_init(cev_paged_desc* d, int32_t dtype, int32_t hq, int32_t hkv, int32_t hd, int32_t n_requests, int32_t t,
                                       int32_t page_size, int32_t n_pages, int32_t max_pages) {
  CEV_CHECK_ARG(d != nullptr, "cev_paged_desc_init: null descriptor");
  memset(d, 0, sizeof *d);
  d->dtype = dtype;
  d->n_q_heads = hq;
  d->n_kv_heads = hkv;
  d->head_dim = hd;
  d->n_requests = n_requests;
  d->t = t;
  d->max_new = t;
  d->page_size = page_size;
  d->n_pages = n_pages;
  d->max_pages = max_pages;
  d->scale = hd > 0 ? (float)(1.0 / sqrt((double)hd)) : 0.0f;
  d->q_stride_t = d->o_stride_t = (int64_t)hq * hd;
  d->q_stride_h = d->o_stride_h = hd;
  d->kc_stride_h = d->vc_stride_h = hd;
  d->kc_stride_t = d->vc_stride_t = (int64_t)hkv * hd;
  d->kc_stride_p = d->vc_stride_p = (int64_t)page_size * hkv * hd;
  d->bt_stride = max_pages;
  return CEV_OK;
}

int32_t cev_paged_bounds(const cev_paged_desc* d, PagedBounds* b) {
  CEV_CHECK_ARG(d != nullptr, "paged attention: null descriptor");
  if (d->dtype != CEV_F32 && d->dtype != CEV_BF16) return cev_fail(CEV_ERR_UNSUPPORTED, "paged attention: dtype %d", d->dtype);
  if (d->head_dim != 128 && !(d->head_dim == 256 && d->dtype == CEV_BF16))
    return cev_fail(CEV_ERR_UNSUPPORTED, "paged attention: head_dim %d (128, in bf16 also 256)", d->head_dim);
  CEV_CHECK_ARG(d->n_q_heads > 0 && d->n_kv_heads > 0 && d->n_q_heads % d->n_kv_heads == 0, "paged attention: %d q heads over %d kv heads",
                d->n_q_heads, d->n_kv_heads);
  const int32_t g = d->n_q_heads / d->n_kv_heads;
  if (g != 1 && g != 2 && g != 4 && g != 8) return cev_fail(CEV_ERR_UNSUPPORTED, "paged attention: GQA group %d (1, 2, 4, 8)", g);
  if (d->n_kv_heads > 4096) return cev_fail(CEV_ERR_UNSUPPORTED, "paged attention: %d kv heads", d->n_kv_heads);
  CEV_CHECK_ARG(d->n_requests >= 1, "paged attention: %d requests", d->n_requests);
  if (d->n_requests > kPagedMaxRequests)
    return cev_fail(CEV_ERR_UNSUPPORTED, "paged attention: %d requests (at most %d)", d->n_requests, kPagedMaxRequests);
  CEV_CHECK_ARG(d->t >= 1 && d->max_new >= 1 && d->max_new <= d->t, "paged attention: t %d, max_new %d", d->t, d->max_new);
  CEV_CHECK_ARG(power_of_two(d->page_size) && d->page_size >= 16 && d->page_size <= 1024,
                "paged attention: page_size %d (a power of two, 16 to 1024)", d->page_size);
  CEV_CHECK_ARG(d->n_pages >= 1 && d->max_pages >= 1, "paged attention: n_pages %d, max_pages %d", d->n_pages, d->max_pages);
  // key sub-tiles are rounded up to whole ones in 32 bits
  CEV_CHECK_ARG((int64_t)d->max_pages * d->page_size <= INT32_MAX - 1024, "paged attention: %d pages of %d keys overflow the key index",
                d->max_pages, d->page_size);
  CEV_CHECK_ARG(d->window >= 0 && d->sinks >= 0, "paged attention: window %d, sinks %d", d->window, d->sinks);
  CEV_CHECK_ARG(d->sinks == 0 || d->window > 0, "paged attention: first tokens that stay visible need a window");
  CEV_CHECK_ARG(d->scale > 0.0f && isfinite(d->scale), "paged attention: scale must be finite and positive");
  const int64_t esz = d->dtype == CEV_BF16 ? 2 : 4, al = 16 / esz;
  const int64_t hq = d->n_q_heads, hkv = d->n_kv_heads;
  const int64_t st[][2] = {{d->q_stride_t, d->t},        {d->q_stride_h, hq},           {d->kc_stride_p, d->n_pages}, {d->kc_stride_t, d->page_size},
                           {d->kc_stride_h, hkv},        {d->vc_stride_p, d->n_pages},  {d->vc_stride_t, d->page_size}, {d->vc_stride_h, hkv},
                           {d->o_stride_t, d->t},        {d->o_stride_h, hq}};
  for (const auto& s : st) {
    CEV_CHECK_ARG(cev_stride_fits(s[0], s[1]), "paged attention: stride %lld of %lld rows", (long long)s[0], (long long)s[1]);
    if (s[1] > 1 && s[0] % al) return cev_fail(CEV_ERR_UNSUPPORTED, "paged attention: strides must be multiples of %lld elements", (long long)al);
  }
  CEV_CHECK_ARG((hq == 1 || d->o_stride_h >= d->head_dim) && (d->t == 1 || d->o_stride_t >= d->head_dim), "paged attention: rows of out overlap");
  // a buffer resource spans 16 rows of a page
  const int64_t row_max = (INT32_MAX / 2) / 16 / esz;
  const int64_t rows[] = {d->kc_stride_t, d->vc_stride_t};
  for (int64_t s : rows)
    if (s < d->head_dim || s > row_max)
      return cev_fail(CEV_ERR_UNSUPPORTED, "paged attention: cache token stride %lld outside [head_dim, %lld]", (long long)s, (long long)row_max);
  CEV_CHECK_ARG(d->bt_stride >= 0 && (d->n_requests == 1 || d->bt_stride >= d->max_pages), "paged attention: block table stride %lld",
                (long long)d->bt_stride);
  b->max_len = d->max_pages * d->page_size;
  b->sig = signature(d);
  // bf16 heads have a kernel for requests of more rows than one tile of
  // the first kernel holds; the plan decides which kernel takes them.
  const bool tiles = d->dtype == CEV_BF16, two = tiles && d->head_dim == 128;
  size_t at = 256;
  for (int i = 0; i < kPagedLists; ++i) {
    PagedListBounds& l = b->list[i];
    l.rows = paged_slots(i) / g;
    l.keys = paged_keys(i, d->head_dim);
    l.target = 0;
    int64_t items = 0;
    if (i == kPagedFew || (tiles && d->max_new > paged_slots(kPagedFew) / g)) {
      const int32_t cus = i == kPagedMany ? kManyWorkgroups : two ? kFewWorkgroups128 : kFewWorkgroups;
      l.target = cus / d->n_kv_heads > 0 ? cus / d->n_kv_heads : 1;
      // whole tiles, and a cut for each workgroup after the first (no request has
      // more new tokens than tokens)
      auto most = [&](int32_t max_new) {
        const int64_t new_rows = max_new < b->max_len ? max_new : b->max_len;
        const int64_t by_request = d->n_requests * ((new_rows + l.rows - 1) / l.rows);
        const int64_t by_rows = d->t / l.rows + (int64_t)d->n_requests;
        return by_request < by_rows ? by_request : by_rows;
      };
      items = most(d->max_new) + l.target;
      // the plan counts the tiles' sub-tiles, and eight more for each, in 32 bits
      // (much work in requests of many rows is not left to the first kernel)
      const int64_t counted = most(i == kPagedFew && tiles && d->max_new > l.rows ? l.rows : d->max_new);
      if (counted * ((int64_t)b->max_len / l.keys + 16) > INT32_MAX)
        return cev_fail(CEV_ERR_UNSUPPORTED, "paged attention: %lld tiles of query rows over %d keys are too many for one call",
                        (long long)counted, b->max_len);
    }
    l.items = (int32_t)items;
    l.first_off = at;
    l.items_off = align_up(l.first_off + sizeof(PagedItem) * (size_t)l.target);
    l.counters_off = align_up(l.items_off + sizeof(PagedItem) * (size_t)items);
    // a cut makes at most one more split tile and two more pieces
    l.records_off = align_up(l.counters_off + 4 * (size_t)l.target * d->n_kv_heads);
    at = align_up(l.records_off + 2 * (size_t)l.target * d->n_kv_heads * paged_slots(i) * (d->head_dim + 2) * sizeof(float));
  }
  b->bytes = at;
  return CEV_OK;
}

extern "C" int32_t cev_paged_work_size(const cev_paged_desc* d, size_t* bytes) {
  CEV_CHECK_ARG(bytes != nullptr, "cev_paged_work_size: null output");
  PagedBounds b;
  const int32_t rc = cev_paged_bounds(d, &b);
  if (rc) return rc;
  *bytes = b.bytes;
  return CEV_OK;
}

// ---------------------------------------------------------------------
// Rotary angles

extern "C" int32_t cev_rope_angles(const cev_rope_scaling* s, uint64_t* steps, float* factor) {
  CEV_CHECK_ARG(s && steps && factor, "cev_rope_angles: null argument");
  CEV_CHECK_ARG(s->rotary_dim >= 2 && s->rotary_dim % 2 == 0 && s->rotary_dim <= 65536, "cev_rope_angles: rotary_dim %d", s->rotary_dim);
  CEV_CHECK_ARG(s->theta > 1.0 && isfinite(s->theta), "cev_rope_angles: theta must be finite and above 1");
  CEV_CHECK_ARG(s->attention_factor >= 0.0 && isfinite(s->attention_factor), "cev_rope_angles: attention_factor must be finite and not negative");
  if (s->kind < CEV_ROPE_PLAIN || s->kind > CEV_ROPE_WAVELENGTH) return cev_fail(CEV_ERR_UNSUPPORTED, "cev_rope_angles: scaling %d", s->kind);
  if (s->kind != CEV_ROPE_PLAIN) CEV_CHECK_ARG(s->factor >= 1.0 && isfinite(s->factor), "cev_rope_angles: factor must be at least 1");
  const long double turn = 2.0L * acosl(-1.0L);
  long double lo = 0, hi = 0;
  if (s->kind == CEV_ROPE_YARN || s->kind == CEV_ROPE_WAVELENGTH) {
    CEV_CHECK_ARG(s->original > 0.0 && isfinite(s->original), "cev_rope_angles: the original context must be positive");
    CEV_CHECK_ARG(s->low > 0.0 && s->high > s->low && isfinite(s->high), "cev_rope_angles: turns %g to %g", s->low, s->high);
  }
  if (s->kind == CEV_ROPE_YARN) {
    // the (fractional) pair that turns n times in the original context
    auto pair = [&](double n) { return (long double)s->rotary_dim * logl(s->original / (n * turn)) / (2 * logl(s->theta)); };
    lo = fmaxl(0, floorl(pair(s->high)));
    hi = fminl(s->rotary_dim - 1, ceill(pair(s->low)));
  }
  for (int i = 0; i < s->rotary_dim / 2; ++i) {
    const long double inv = powl(s->theta, -2.0L * i / s->rotary_dim);
    long double r = 0;  // share of the stretched angle
    if (s->kind == CEV_ROPE_LINEAR) r = 1;
    if (s->kind == CEV_ROPE_YARN) r = fminl(1, fmaxl(0, (i - lo) / fmaxl(hi - lo, 1e-3L)));
    if (s->kind == CEV_ROPE_WAVELENGTH) r = 1 - fminl(1, fmaxl(0, (s->original * inv / turn - s->low) / ((long double)s->high - s->low)));
    const long double turns = s->kind == CEV_ROPE_PLAIN ? inv / turn : inv * (1 - r + r / s->factor) / turn;  // below 0.16
    steps[i] = (uint64_t)roundl(ldexpl(turns, 64));
  }
  *factor = s->attention_factor > 0.0 ? (float)s->attention_factor
                                      : s->kind == CEV_ROPE_YARN ? (float)(0.1L * logl(s->factor) + 1) : 1.0f;
  return CEV_OK;
}

extern "C" int32_t cev_rope_desc_init(cev_rope_desc* d, int32_t dtype, int32_t hq, int32_t hkv, int32_t hd, int32_t t, int32_t rotary_dim,
                                      int32_t page_size, int32_t n_slots) {
  CEV_CHECK_ARG(d != nullptr, "cev_rope_desc_init: null descriptor");
  memset(d, 0, sizeof *d);
  d->dtype = dtype;
  d->n_q_heads = hq;
  d->n_kv_heads = hkv;
  d->head_dim = hd;
  d->t = t;
  d->rotary_dim = rotary_dim;
  d->factor = 1.0f;
  d->page_size = page_size;
  d->n_slots = n_slots;
  d->qi_stride_h = d->qo_stride_h = d->ki_stride_h = d->vi_stride_h = d->ko_stride_h = d->vo_stride_h = hd;
  d->qi_stride_t = d->qo_stride_t = (int64_t)hq * hd;
  d->ki_stride_t = d->vi_stride_t = d->ko_stride_t = d->vo_stride_t = (int64_t)hkv * hd;
  d->ko_stride_p = d->vo_stride_p = (int64_t)page_size * hkv * hd;
  return CEV_OK;
}
