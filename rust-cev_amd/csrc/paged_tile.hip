// Attention over a paged K/V cache for requests with many new rows (prompts,
// chunks of prompts): bf16, d = 128 or 256.
//
// A workgroup's 8 waves x 32 query slots hold 256 / g rows of one request times
// the g query heads of one KV head, and share the chunks that it walks (64 keys, at
// d = 256 32):
// a chunk is read once for 256 slots, where the kernel of few rows
// (paged_attn.hip) reads it for every 32 and is bound by L2 there.  The loop of
// d = 128 is packed_attn.hip's: S^T = K . Q^T of one 32-key sub-tile runs beside the
// softmax of the one before, then O^T += V^T . P^T, with waves 4-7 one region
// ahead of waves 0-3; it differs in
//   - the fetch: a wave's 8 rows of a chunk lie in one page, whose 64-bit base
//     is scalar, so the cache may have any size;
//   - the softmax argument: scale * log2 e times the f32 score less the row's
//     maximum in one FMA.  (Q scaled and rounded to bf16 beforehand would save
//     the FMA, and adds as much error as the probabilities' own rounding.)
//   - the masks: by position, from the row's last key, the window and the first
//     tokens that stay visible;
//   - infinities and NaN of V that only some of a chunk's rows see.
// d = 256 scores a chunk, makes its probabilities and multiplies, one after the
// other: O and Q take 192 of a lane's 256 registers.
// Pieces of a split tile are joined as in paged_attn.hip.
//
// Bound by the matrix cores and the softmax beside them: a chunk of 64 keys takes
// 4100 cycles of a workgroup (2048 of MFMAs a SIMD).  4 chunks of 450 rows after 12000
// to 32000 keys (32 over 8 heads) 556 to 576 us by card, 990 to 950 TFLOP/s; 7600 rows that see 1024
// keys and the first four 185 to 191 us, 710 to 690 TFLOP/s: a tile of 19 chunks has 15000 cycles of its
// own (first scores and their maximum 5000, a chunk's masks, the rows' stores).
// Without the fetch the chunks' call took 478 of 569 us, without the exponentials 536.
// d = 256: 64 requests of 256 rows in 2048 keys (16 over 4 heads) 592 to 670 us by card,
// 870 to 770 TFLOP/s; 32 slots a workgroup took 2800.  What lies in scratch counts by
// how it is used: two values that a chunk reloads are in this form (592 us); with
// parts of Q reloaded it took 790 where this one took 623, with K reads three units
// ahead 718, and with so few addresses kept that nothing of the loop was in scratch 676.
#include "attn_pipe.h"
#include "paged_device.h"

namespace {

using namespace pipe;

constexpr int kWaves = 8;
constexpr int kThreads = kWaves * 64;
constexpr int kSlots = paged_slots(kPagedMany);
static_assert(kSlots == kWaves * 32, "tile layout");

// This lane's half of the wave, computed afresh (opaque to hoisting).
__device__ __forceinline__ int fresh_half() { return fresh_lane_id() >> 5; }

// LDS reads of d = 256's chunk body: 16 K reads kKPF ahead of their MFMA, then 16
// V fragments of two reads kVPF ahead, beside whose last units the next body's
// first K reads go out.  What a unit waits for: the reads issued after its own.
constexpr int kKPF = 2, kVPF = 3;
constexpr int wait_k256(int st) { return 15 - st < kKPF - 1 ? 15 - st : kKPF - 1; }
constexpr int wait_v256(int unit) {
  int at[16] = {}, n = 0, wait = 0;
  for (int j = 0; j < kVPF; ++j) at[j] = n += 2;
  for (int j = 0; j <= unit; ++j) {
    wait = n - at[j];
    if (j + kVPF < 16) at[j + kVPF] = n += 2;
    if (j >= 16 - kKPF) ++n;
  }
  return wait;
}
static_assert(wait_k256(0) == 1 && wait_k256(15) == 0 && wait_v256(0) == 4 && wait_v256(13) == 4 && wait_v256(14) == 2 && wait_v256(15) == 1,
              "two K and three V fragments ahead");

template <int D>
__global__ __launch_bounds__(kThreads) __attribute__((amdgpu_waves_per_eu(2, 2))) void paged_tile_kernel(PagedArgs a) {
  using F = Frag<__bf16, D>;
  using P = typename F::P;
  using Sched = Schedule<true>;
  constexpr int NDT = D / 32, kKeys = paged_keys(kPagedMany, D), kRowBytes = 2 * D;
  constexpr int kRows = kKeys / kWaves, kLoadRows = 1024 / kRowBytes, kBlk = kRowBytes / 16;  // a wave's rows of a chunk, an instruction's, blocks of a row
  static_assert(kTileBytes == kKeys * kRowBytes && kRows == 2 * kLoadRows, "two loads of K and two of V a wave and chunk");
  __shared__ __align__(1024) char lds[2 * kBuf * kTileBytes];
  __shared__ int32_t odd_s, bad_s, last_s;

  const int run = blockIdx.x / (uint32_t)a.hkv, kvh = blockIdx.x - run * a.hkv;
  PagedWalk walk(a, run);
  int n_parts;
  if (!paged_plan_ok(a, kPagedMany, n_parts)) return;  // the other kernel writes NaN
  if (run >= n_parts) return;
  const int tid = threadIdx.x, lane = tid & 63, wave = uniform_i32(tid >> 6);
  const int n = lane & 31, u = lane >> 5;
  const int gs = __builtin_ctz(a.g);

  // Per-lane LDS addresses of the operand reads; the sub-tile and half are
  // immediates.  They move on by one buffer a chunk (12 adds beside 32 MFMAs; a
  // body for each of the four buffers, with the buffer as an immediate, leaves
  // the loop in four places, and O and the scores were copied between them:
  // 1.7 KB a lane of spills).
  const int lds_base = (int)(size_t)(const __attribute__((address_space(3))) char*)lds;
  // (bit 4 of a block's place is its own: the upper 128 columns of d = 256 are 256
  // bytes further)
  // d = 256 keeps the first of each, and makes the others of their places' bits
  // (with all kept nine values of the loop lay in scratch, now two).
  constexpr int kKoff = D == 128 ? 8 : 1, kVoff = D == 128 ? 4 : 1;
  int koff[kKoff], voff[kVoff];
#pragma unroll
  for (int st = 0; st < kKoff; ++st) koff[st] = lds_base + n * kRowBytes + (k_slot(2 * st + u, n) << 4);
  {
    const int i = lane & 15, g16 = (lane >> 4) & 1, rr = i >> 2;
    const int blk = 2 * g16 + ((i & 3) >> 1);  // 16-byte block of the read, within a 64-byte slice
#pragma unroll
    for (int dt = 0; dt < kVoff; ++dt)
      voff[dt] = lds_base + kVBase + (4 * u + rr) * kRowBytes + (v_slot(4 * dt + blk, rr) << 4) + 8 * (i & 1);
  }
  struct VFrag {
    i32x2 lo, hi;
  };
  auto v_issue = [&](auto kt_c, auto j_c) {
    constexpr int KT = decltype(kt_c)::value, J = decltype(j_c)::value;
    constexpr int OFF = (KT * 32 + 16 * (J / NDT)) * kRowBytes + 256 * (J % NDT / 4);
    const int at = D == 128 ? voff[J % kVoff] : voff[0] ^ (J % 4 << 6);
    return VFrag{read_tr<OFF>(at), read_tr<OFF + 8 * kRowBytes>(at)};
  };
  auto v_ready = [](VFrag& f, auto j_c) {
    constexpr int J = decltype(j_c)::value;
    if constexpr (D == 128)
      wait_tr<Sched::wait_b(J)>(f.lo, f.hi);
    else
      wait_tr<wait_v256(J)>(f.lo, f.hi);
    const bf16x4 lo = __builtin_bit_cast(bf16x4, f.lo), hi = __builtin_bit_cast(bf16x4, f.hi);
    return bf16x8{lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
  };
  auto k_issue = [&](auto kt_c, auto st_c) {
    constexpr int ST = decltype(st_c)::value;
    return read_b128<decltype(kt_c)::value * 32 * kRowBytes + 256 * (ST / 8)>(D == 128 ? koff[ST % kKoff] : koff[0] ^ (ST % 8 << 5));
  };
  auto k_ready = [](KFrag& r, auto st_c) {
    constexpr int ST = decltype(st_c)::value;
    if constexpr (D == 128)
      wait_b128<Sched::wait_a(ST)>(r);
    else
      wait_b128<wait_k256(ST)>(r);
    return __builtin_bit_cast(bf16x8, r);
  };

  // Cache rows of this KV head.  A wave fetches kRows rows of K and of V of a chunk,
  // 1 KB an instruction.
  const uint64_t kbase = (uint64_t)((const __bf16*)a.kc + kvh * a.kc_sh), vbase = (uint64_t)((const __bf16*)a.vc + kvh * a.vc_sh);
  const int kr = uniform_i32((int)(2 * a.kc_st)), vr = uniform_i32((int)(2 * a.vc_st));
  int kat[2], vat[2];
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    const int of = kLoadRows * r + lane / kBlk, row = kRows * wave + of, blk = lane % kBlk;
    kat[r] = of * kr + (k_slot(blk, row) << 4);
    vat[r] = of * vr + (v_slot(blk, row) << 4);
  }

  // The current item's state, of this wave where it says so.
  PagedItem it;
  PagedSpan span;
  int pos, w_pos0, w_pos1, w_lo, w_hi, t_lo, t_hi, nc;  // last position that the lane's row sees; unmasked() below
  bool row_ok, wave_active;
  const int32_t* bt;
  F fr;
  // chunks [it.c_begin, it.c_begin + nc) of the tile's stream
  auto first_key = [&](int i) {
    const int c = it.c_begin + i;
    return kKeys * (c < span.sinks ? c : c - span.sinks + span.first);
  };
  // Chunks of the part before lo and from hi on hold keys that not all rows
  // at positions [p0, p1] see (those before lo may also be seen by all).
  auto unmasked = [&](int p0, int p1, int& lo, int& hi) {
    // the chunks of the window start at stream place span.sinks; the last key
    // of the one at place c is first_key + kKeys - 1
    hi = span.sinks + (p0 + 1) / kKeys - span.first - it.c_begin;
    lo = 0;
    if (a.window > 0 && p1 >= a.window) lo = span.sinks + (p1 - a.window) / kKeys + 1 - span.first - it.c_begin;
  };
  // Lane l keeps the addresses of this wave's rows of K and of V of chunk 64 b +
  // l of the current batch b, and whether they are fetched at all.
  int batch_first = 0, k_lo = 0, k_hi = 0, v_lo = 0, v_hi = 0, fetched = 0;
  bool bad_page = false;
  auto load_pages = [&](int i) {
    batch_first = i;
    const int key0 = first_key(min(i + fresh_lane_id(), nc - 1)) + kRows * wave;
    // (the last chunk may reach beyond the block table's last page)
    int page = bt[min(key0 >> a.page_shift, a.max_pages - 1)];
    // rows that some row of the tile sees
    const bool seen = key0 < span.end && !(key0 >= span.skip_lo && key0 + kRows <= span.skip_hi);
    const bool in = (uint32_t)page < (uint32_t)a.n_pages;
    bad_page |= __any(seen && !in);
    fetched = seen && in ? kRows : 0;
    page = in ? page : 0;
    const int64_t off = key0 & ((1 << a.page_shift) - 1);
    const uint64_t kp = kbase + 2 * (uint64_t)(page * a.kc_sp + off * a.kc_st), vp = vbase + 2 * (uint64_t)(page * a.vc_sp + off * a.vc_st);
    k_lo = (int)(uint32_t)kp, k_hi = (int)(uint32_t)(kp >> 32);
    v_lo = (int)(uint32_t)vp, v_hi = (int)(uint32_t)(vp >> 32);
  };
  // Chunk i into its buffer, i mod kBuf; past the end: zeros.
  auto fetch = [&](int i) {
    const bool real = i < nc;
    if (real && i >= batch_first + 64) load_pages(i);
    const int l = real ? i - batch_first : 0;
    const int rows = real ? __builtin_amdgcn_readlane(fetched, l) : 0;
    const uint64_t kp = (uint32_t)__builtin_amdgcn_readlane(k_lo, l) | (uint64_t)(uint32_t)__builtin_amdgcn_readlane(k_hi, l) << 32;
    const uint64_t vp = (uint32_t)__builtin_amdgcn_readlane(v_lo, l) | (uint64_t)(uint32_t)__builtin_amdgcn_readlane(v_hi, l) << 32;
    const __amdgpu_buffer_rsrc_t rk = __builtin_amdgcn_make_buffer_rsrc((void*)kp, (short)0, rows * kr, kBufferWord3);
    const __amdgpu_buffer_rsrc_t rv = __builtin_amdgcn_make_buffer_rsrc((void*)vp, (short)0, rows * vr, kBufferWord3);
    int ka[2] = {kat[0], kat[1]}, va[2] = {vat[0], vat[1]};
    if (i >= t_hi || i < t_lo) {  // it may hold keys that no row sees
      const int key0 = (real ? first_key(i) : 0) + kRows * wave + fresh_lane_id() / kBlk;
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        const int key = key0 + kLoadRows * r;
        const bool load = key < span.end && !(key >= span.skip_lo && key < span.skip_hi);
        ka[r] = load ? ka[r] : INT32_MAX;
        va[r] = load ? va[r] : INT32_MAX;
      }
    }
    char* const dst = lds + i % kBuf * kTileBytes + kRows * wave * kRowBytes;
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      __builtin_amdgcn_raw_ptr_buffer_load_lds(rk, (__attribute__((address_space(3))) void*)(dst + 1024 * r), 16, ka[r], 0, 0, 0);
      __builtin_amdgcn_raw_ptr_buffer_load_lds(rv, (__attribute__((address_space(3))) void*)(dst + kVBase + 1024 * r), 16, va[r], 0, 0, 0);
    }
  };
  constexpr int kLoadsPerChunk = 4;

  // 0 times an infinity or NaN is NaN: a key that only some of the rows see
  // must not reach the others.  Where the rows differ in what they see of chunk
  // i, such values among the V rows that this wave fetched (landed by now)
  // become zeros; after the loop the rows that see them get them.
  auto clean = [&](int i) {
    if (i >= nc || (i >= t_lo && i < t_hi)) return;
    const int lane = fresh_lane_id(), at = kVBase + i % kBuf * kTileBytes + kRows * wave * kRowBytes + lane * 16;
    i32x4* const v = (i32x4*)(lds + at);
    KFrag vr[2] = {read_b128<0>(lds_base + at), read_b128<1024>(lds_base + at)};
    wait_b128<1>(vr[0]);
    wait_b128<0>(vr[1]);
    bool odd = false;
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      i32x4 x = __builtin_bit_cast(i32x4, vr[r]);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const bool hi = (x[e] & 0x7f800000) == 0x7f800000, lo = (x[e] & 0x7f80) == 0x7f80;
        odd |= hi | lo;
        x[e] &= (hi ? 0 : (int)0xffff0000) | (lo ? 0 : 0xffff);
      }
      if (odd) v[64 * r] = x;
    }
    if (__ballot(odd) && lane == 0) *(volatile int32_t*)&odd_s = 1;
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  };
  auto mask_sub = [&](f32x16& s, int key0) {
    // bounds of the register's place, 8 (i / 4) + i % 4 (constants to compare
    // with, where the keys themselves would be 16 values to hold)
    const int k0 = key0 + 4 * fresh_half(), hi = pos - k0;
    const int lo = a.window == 0 || pos < a.window ? INT32_MIN : pos - a.window - k0, first = a.sinks - k0;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const int at = 8 * (i >> 2) + (i & 3);
      s[i] = (at <= hi) & ((at > lo) | (at < first)) ? s[i] : -INFINITY;
    }
  };

  // Takes the run's next item and asks for its Q, its pages and its first chunks.
  auto begin = [&] {
    const int lane = fresh_lane_id(), n = lane & 31, u = lane >> 5;
    it = walk.item();
    const int pos1 = it.pos0 + it.n_rows - 1;
    span = paged_span(kKeys, it.pos0, pos1, a.window, a.sinks);
    nc = it.c_end - it.c_begin;
    // Query slot (wave, n) holds row slot / g of the tile and query head slot % g:
    // the rows of a short tile fill the first waves.
    const int rit = (wave * 32 + n) >> gs;
    row_ok = rit < it.n_rows;
    pos = row_ok ? it.pos0 + rit : -1;
    const int w_row0 = (wave * 32) >> gs, w_row1 = min((wave * 32 + 31) >> gs, it.n_rows - 1);
    wave_active = w_row0 < it.n_rows;
    w_pos0 = it.pos0 + w_row0, w_pos1 = it.pos0 + w_row1;
    unmasked(w_pos0, w_pos1, w_lo, w_hi);    // of this wave's rows
    unmasked(it.pos0, pos1, t_lo, t_hi);     // of all of the tile's
    bt = a.bt + it.req * a.bt_stride;
    bad_page = false;
    load_pages(0);
    const int row = it.row0 + (row_ok ? rit : 0), head = kvh * a.g + (n & (a.g - 1));
    fr.load_q((const __bf16*)a.q + (int64_t)row * a.q_st + (int64_t)head * a.q_sh, row_ok, u);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int k = 0; k < kAhead; ++k) fetch(k);
    __builtin_amdgcn_sched_barrier(0);
    // Q is waited for here, where only the chunks are behind it.
#pragma unroll
    for (int st = 0; st < F::NQK; ++st) {
      i32x4 x = __builtin_bit_cast(i32x4, fr.q[st]);
      asm volatile("" : "+v"(x));
      fr.q[st] = __builtin_bit_cast(bf16x8, x);
    }
  };
  if (tid == 0) odd_s = bad_s = 0;
  begin();
  for (;;) {
    f32x16 o[NDT];
#pragma unroll
    for (int dt = 0; dt < NDT; ++dt) o[dt] = f32x16{};
    // m_run: a maximum that the row reached, in base-2 softmax units (0 until
    // it has seen a key, m_set); rows that never see one keep l = 0.
    float m_run = 0.0f, l_run = 0.0f;
    bool m_set = false;
    const float c = a.scale_log2;

    wait_vmcnt<kLoadsPerChunk * (kAhead - 2)>();  // chunks 0 and 1 landed
    lds_barrier();                                // (the flags are clear)
    clean(0);
    clean(1);
    lds_barrier();

    using I0 = std::integral_constant<int, 0>;
    using I1 = std::integral_constant<int, 1>;
    if constexpr (D == 128) {
      f32x16 sa, sb;
      constexpr int KPF = Sched::KPF, VPF = Sched::VPF;
      KFrag kf[KPF];
      if (wave_active) {
        // Sub-tile 0: its row maximum (over both lane halves) is the first m_run.
        sa = f32x16{};
        KFrag k0[F::NQK];
        static_for<F::NQK>([&](auto st_c) { k0[decltype(st_c)::value] = k_issue(I0{}, st_c); });
        static_for<F::NQK>([&](auto st_c) {
          constexpr int st = decltype(st_c)::value;
          wait_b128<F::NQK - 1 - st>(k0[st]);
          fr.qk_mfma(__builtin_bit_cast(bf16x8, k0[st]), st, sa);
        });
        if (0 >= w_hi || 0 < w_lo) mask_sub(sa, first_key(0));
        float mx = -INFINITY;
#pragma unroll
        for (int i = 0; i < 16; ++i) mx = fmaxf(mx, sa[i]);
        const float m0 = pair_max(mx) * c;
        m_set = m0 > -INFINITY;
        m_run = m_set ? m0 : 0.0f;
        // The first body's K reads (sub-tile 1 of chunk 0), waited for in full, so
        // that its counted waits see no fewer reads than a steady-state body's.
        static_for<KPF>([&](auto f_c) { kf[decltype(f_c)::value] = k_issue(I1{}, f_c); });
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      }
      VFrag vf[VPF];
      P p;
      const bf16x2 one = {(__bf16)1.0f, (__bf16)1.0f};
      // Region A of sub-tile KT of this chunk: the next sub-tile's scores on the
      // MFMA unit beside this one's probabilities, then the check of the row's
      // maximum.  (The last sub-tile also scores one past the end, never used.)
      auto region_a = [&](auto kt_c) {
        constexpr int kt = decltype(kt_c)::value;
        using KTN_c = std::integral_constant<int, 1 - kt>;
        f32x16& s = kt == 0 ? sa : sb;
        f32x16& sn = kt == 0 ? sb : sa;
        float rs = 0.0f;
        static_for<F::NQK>([&](auto st_c) {
          constexpr int st = decltype(st_c)::value;
          if constexpr (st == 0)
            sn = __builtin_amdgcn_mfma_f32_32x32x16_bf16(k_ready(kf[0], st_c), fr.q[0], f32x16{}, 0, 0, 0);
          else
            fr.qk_mfma(k_ready(kf[st % KPF], st_c), st, sn);
          if constexpr (st + KPF < F::NQK) kf[st % KPF] = k_issue(KTN_c{}, std::integral_constant<int, st + KPF>{});
          if constexpr (st >= F::NQK - VPF)
            vf[st - (F::NQK - VPF)] = v_issue(kt_c, std::integral_constant<int, st - (F::NQK - VPF)>{});
          const float e0 = fast_exp2(__builtin_fmaf(s[2 * st], c, -m_run));
          const float e1 = fast_exp2(__builtin_fmaf(s[2 * st + 1], c, -m_run));
          const bf16x2 pr = {(__bf16)e0, (__bf16)e1};
          p.h[st / 4][2 * (st % 4)] = pr[0];
          p.h[st / 4][2 * (st % 4) + 1] = pr[1];
          rs = __builtin_amdgcn_fdot2_f32_bf16(pr, one, rs, false);
          pin(rs);
          __builtin_amdgcn_sched_barrier(0);
        });
        // The probabilities stand as long as their sum stays within kMaxP.
        // Otherwise, or for a row with no maximum yet, the row moves its maximum
        // (a set one only when it grew by more than kRescale).  No LDS operation,
        // so the counted waits of region B still hold.
        if (__ballot((rs > kMaxP) | !m_set)) {
          float ml = -INFINITY;
#pragma unroll
          for (int i = 0; i < 16; ++i) ml = fmaxf(ml, s[i]);
          const float cand = pair_max(ml) * c, delta = cand - m_run;
          const bool move = m_set ? delta > kRescale : cand > -INFINITY;
          const float alpha = m_set && move ? fast_exp2(-delta) : 1.0f;
          m_set = m_set | move;
          m_run = move ? cand : m_run;
          l_run *= alpha;
#pragma unroll
          for (int dt = 0; dt < NDT; ++dt) o[dt] *= alpha;
          rs = 0.0f;
#pragma unroll
          for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int j = 0; j < 8; j += 2) {
              const bf16x2 pr = {(__bf16)fast_exp2(__builtin_fmaf(s[8 * h + j], c, -m_run)),
                                 (__bf16)fast_exp2(__builtin_fmaf(s[8 * h + j + 1], c, -m_run))};
              p.h[h][j] = pr[0];
              p.h[h][j + 1] = pr[1];
              rs = __builtin_amdgcn_fdot2_f32_bf16(pr, one, rs, false);
            }
        }
        l_run += rs;
      };
      // Region B of sub-tile KT of chunk i: P.V, the next region's first K reads
      // (it scores sub-tile KT of the next chunk), then the mask of the next scores.
      auto region_b = [&](auto kt_c, int i) {
        constexpr int kt = decltype(kt_c)::value;
        f32x16& sn = kt == 0 ? sb : sa;
        static_for<F::NPV>([&](auto j_c) {
          constexpr int j = decltype(j_c)::value;
          F::pv_mfma(v_ready(vf[j % VPF], j_c), j, p, o);
          if constexpr (j + VPF < F::NPV) vf[j % VPF] = v_issue(kt_c, std::integral_constant<int, j + VPF>{});
          if constexpr (j >= F::NPV - KPF) kf[j - (F::NPV - KPF)] = k_issue(kt_c, std::integral_constant<int, j - (F::NPV - KPF)>{});
          __builtin_amdgcn_sched_barrier(0);
        });
        const int in = i + kt;  // chunk of the next scores
        if (in < w_lo || in >= w_hi) mask_sub(sn, first_key(in) + 32 * (1 - kt));
      };
      const bool lead = wave >= kWaves / 2;
      if (wave_active && lead) region_a(I0{});
#pragma unroll 1
      for (int i = 0; i < nc; ++i) {
        const int next = i % kBuf == kBuf - 1 ? -kAhead * kTileBytes : kTileBytes;  // to the next chunk's buffer
        if (wave_active && !lead) region_a(I0{});
        fetch(i + kAhead);
        if (wave_active) {
#pragma unroll
          for (int st = 0; st < kKoff; ++st) koff[st] += next;
          region_b(I0{}, i);
          region_a(I1{});
          region_b(I1{}, i);
#pragma unroll
          for (int dt = 0; dt < kVoff; ++dt) voff[dt] += next;
          if (lead && i + 1 < nc) region_a(I0{});
        }
        // Chunk i + 2 must have landed before the barrier; chunk i + kAhead may
        // stay in flight.
        wait_vmcnt<kLoadsPerChunk * (kAhead - 2)>();
        clean(i + 2);
        __builtin_amdgcn_s_barrier();
      }
    } else {
      // Scores, softmax, then products of one 32-key chunk after the other (the
      // registers of O and Q leave none for a second one's scores).
      KFrag kf[kKPF];
      if (wave_active) {
        static_for<kKPF>([&](auto f_c) { kf[decltype(f_c)::value] = k_issue(I0{}, f_c); });
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      }
#pragma unroll 1
      for (int i = 0; i < nc; ++i) {
        const int next = i % kBuf == kBuf - 1 ? -kAhead * kTileBytes : kTileBytes;  // to the next chunk's buffer
        fetch(i + kAhead);
        if (wave_active) {
          f32x16 s = f32x16{};
          static_for<F::NQK>([&](auto st_c) {
            constexpr int st = decltype(st_c)::value;
            fr.qk_mfma(k_ready(kf[st % kKPF], st_c), st, s);
            if constexpr (st + kKPF < F::NQK) kf[st % kKPF] = k_issue(I0{}, std::integral_constant<int, st + kKPF>{});
          });
          // the first V fragments load under the softmax
          VFrag vf[kVPF];
          static_for<kVPF>([&](auto j_c) { vf[decltype(j_c)::value] = v_issue(I0{}, j_c); });
          if (i < w_lo || i >= w_hi) mask_sub(s, first_key(i));
          // The maximum moves when a probability would pass kMaxP, or for a row
          // that has none yet.
          float ml = -INFINITY;
#pragma unroll
          for (int e = 0; e < 16; ++e) ml = fmaxf(ml, s[e]);
          if (__ballot((__builtin_fmaf(ml, c, -m_run) > kLog2MaxP) | !m_set)) {
            const float cand = pair_max(ml) * c, delta = cand - m_run;
            const bool move = m_set ? delta > kRescale : cand > -INFINITY;
            const float alpha = m_set && move ? fast_exp2(-delta) : 1.0f;
            m_set = m_set | move;
            m_run = move ? cand : m_run;
            l_run *= alpha;
#pragma unroll
            for (int dt = 0; dt < NDT; ++dt) o[dt] *= alpha;
          }
#pragma unroll
          for (int e = 0; e < 16; ++e) s[e] = fast_exp2(__builtin_fmaf(s[e], c, -m_run));
          P p;
          F::make_p(s, p, l_run);
#pragma unroll
          for (int st = 0; st < kKoff; ++st) koff[st] += next;
          static_for<F::NPV>([&](auto j_c) {
            constexpr int j = decltype(j_c)::value;
            F::pv_mfma(v_ready(vf[j % kVPF], j_c), j, p, o);
            if constexpr (j + kVPF < F::NPV) vf[j % kVPF] = v_issue(I0{}, std::integral_constant<int, j + kVPF>{});
            // the next chunk's first K reads (past the end of a buffer never used)
            if constexpr (j >= F::NPV - kKPF) kf[j - (F::NPV - kKPF)] = k_issue(I0{}, std::integral_constant<int, j - (F::NPV - kKPF)>{});
          });
#pragma unroll
          for (int dt = 0; dt < kVoff; ++dt) voff[dt] += next;
        }
        // Chunk i + 2 must have landed before the barrier; chunk i + kAhead may
        // stay in flight.
        wait_vmcnt<kLoadsPerChunk * (kAhead - 2)>();
        clean(i + 2);
        __builtin_amdgcn_s_barrier();
      }
    }
    // Fetches past the end still write zeros into LDS: drain them, and the last
    // body's K reads of a sub-tile past the end, before LDS is used again.
    wait_vmcnt<0>();
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    if (wave_active) {
      // back to the first buffer
#pragma unroll
      for (int st = 0; st < kKoff; ++st) koff[st] -= nc % kBuf * kTileBytes;
#pragma unroll
      for (int dt = 0; dt < kVoff; ++dt) voff[dt] -= nc % kBuf * kTileBytes;
    }

    // (computed again here, and held in no register through the loop)
    const int lane = fresh_lane_id(), n = lane & 31, u = lane >> 5;
    const bool one = wave == 0 && lane == 0;
    if (bad_page && lane == 0) *(volatile int32_t*)&bad_s = 1;  // one wave's finding
    __syncthreads();
    float l = pair_sum(l_run);
    // Infinities and NaN of V (see note_odd): the tile's chunks whose rows differ in
    // what they see held some, or a row has come out so.
    bool odd_masked = uniform_i32(*(volatile int32_t*)&odd_s);
    auto odd_rows = [&] {
      float t[4] = {};
#pragma unroll
      for (int dt = 0; dt < NDT; ++dt)
#pragma unroll
        for (int e = 0; e < 16; ++e) t[e % 4] = __builtin_fmaf(o[dt][e], 0.0f, t[e % 4]);
      return __any(row_ok & (l == l) & !((t[0] + t[1]) + (t[2] + t[3]) == 0.0f));
    };
    if (*(volatile int32_t*)&bad_s && wave_active) {
      // a page outside the cache makes the rows NaN that see it
#pragma unroll 1
      for (int i = 0; i < nc; ++i)
#pragma unroll 1
        for (int key = first_key(i), k = 0; k < kKeys / 16; ++k, key += 16) {
          if (key >= span.end || (key >= span.skip_lo && key + 16 <= span.skip_hi)) continue;
          const bool bad = (uint32_t)bt[key >> a.page_shift] >= (uint32_t)a.n_pages;
          const bool vis = (key <= pos) & ((a.window == 0) | (key + 15 > pos - a.window) | (key < a.sinks));
          l += (bad & vis) ? __builtin_nanf("") : 0.0f;
        }
    }

    bool write = row_ok;
    const bool split = it.n_pieces > 1;
    // Partial results: [wave][D / 8 vectors of 4 columns][lane], then (m, l) of
    // each slot.
    constexpr int kRec = kSlots * (D + 2);
    float* const rec0 = (float*)(a.work + a.records_off) + ((int64_t)it.rec * a.hkv + kvh) * kRec;
    const int64_t rec_step = (int64_t)a.hkv * kRec;
    auto record = [&](int piece) {
      return __builtin_amdgcn_make_buffer_rsrc((void*)uniform_u64((uint64_t)(rec0 + piece * rec_step)), (short)0, kRec * 4, kBufferWord3);
    };
    const int vec0 = wave * (D / 8) * 1024 + lane * 16, ml0 = kSlots * D * 4 + (wave * 32 + n) * 8;
    if (split) {
      const __amdgpu_buffer_rsrc_t rs = record(it.piece);
      if (wave_active) {
#pragma unroll
        for (int v = 0; v < D / 8; ++v)
          put_past_l2(rs, vec0, f32x4{o[v / 4][4 * (v % 4)], o[v / 4][4 * (v % 4) + 1], o[v / 4][4 * (v % 4) + 2], o[v / 4][4 * (v % 4) + 3]}, 1024 * v);
        if (u == 0) put_past_l2(rs, ml0, make_float2(m_set ? m_run : -1e30f, l));
      }
      // The stores have reached memory before the workgroup counts itself.
      __builtin_amdgcn_s_waitcnt(0);
      __syncthreads();
      int32_t* const counter = (int32_t*)(a.work + a.counters_off) + (int64_t)it.split * a.hkv + kvh;
      if (one) {
        // (pieces with odd_masked count in the upper half too)
        const int before = __hip_atomic_fetch_add(counter, odd_masked ? 0x10001 : 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        const bool all = (before & 0xffff) == it.n_pieces - 1;
        if (all) *counter = 0;  // for the next call with this plan
        last_s = all ? 1 + (before >> 16) : 0;
      }
      __syncthreads();
      const int last = uniform_i32(last_s);
      odd_masked |= last > 1;
      __syncthreads();
      write = write && last;
      // The last one: 64 columns at a time; the next piece is on its way while one is
      // added (a trip past the L2 takes longer than the adding).
      if (last && wave_active) {
#pragma unroll
        for (int half = 0; half < NDT / 2; ++half) {
          f32x4 x[2][8];
          float2 w[2];
          auto get = [&](int q, f32x4* to, float2& to_w) {
            const __amdgpu_buffer_rsrc_t rq = record(min(q, it.n_pieces - 1));
            to_w = get2_past_l2(rq, ml0);
#pragma unroll
            for (int v = 0; v < 8; ++v) to[v] = get4_past_l2(rq, vec0, 1024 * (8 * half + v));
          };
          float M = -1e30f;
          l = 0.0f;
          o[2 * half] = o[2 * half + 1] = f32x16{};
          auto add = [&](const f32x4* from, const float2& from_w) {
            const float m = fmaxf(M, from_w.x), f0 = fast_exp2(M - m), f = fast_exp2(from_w.x - m);
            M = m;
            l = l * f0 + f * from_w.y;
#pragma unroll
            for (int v = 0; v < 8; ++v)
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                const int dt = 2 * half + v / 4, at = 4 * (v % 4) + e;
                o[dt][at] = o[dt][at] * f0 + f * from[v][e];
              }
          };
          get(0, x[0], w[0]);
          for (int q = 0;;) {
            get(q + 1, x[1], w[1]);
            add(x[0], w[0]);
            if (++q == it.n_pieces) break;
            get(q + 1, x[0], w[0]);
            add(x[1], w[1]);
            if (++q == it.n_pieces) break;
          }
        }
      }
    }
    const bool odd_row = odd_rows();
    // The row's 16-byte vectors: a half wave holds four columns of each eight, and
    // the halves exchange theirs of two vectors.
    i32x4 res[D / 16];
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
#pragma unroll
    for (int w = 0; w < D / 16; ++w) {
      int x[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float x0 = o[w / 2][8 * (w % 2) + 2 * e], x1 = o[w / 2][8 * (w % 2) + 2 * e + 1];
        const bf16x2 y = {(__bf16)(l == 0.0f ? 0.0f : x0 * inv), (__bf16)(l == 0.0f ? 0.0f : x1 * inv)};
        x[e] = __builtin_bit_cast(int, y);
      }
      const auto r0 = __builtin_amdgcn_permlane32_swap(x[0], x[2], false, false), r1 = __builtin_amdgcn_permlane32_swap(x[1], x[3], false, false);
      res[w] = i32x4{(int)r0[0], (int)r1[0], (int)r0[1], (int)r1[1]};
    }
    __bf16* const op = (__bf16*)a.out + (int64_t)(it.row0 + ((wave * 32 + n) >> gs)) * a.o_st + (int64_t)(kvh * a.g + (n & (a.g - 1))) * a.o_sh + 8 * u;
    auto store = [&] {
#pragma unroll
      for (int w = 0; w < D / 16; ++w) *(i32x4*)(op + 32 * (w / 2) + 16 * (w % 2)) = res[w];
    };
    if (__any(write) && (odd_masked || odd_row)) {
      // They go over the rows in memory, where O no longer takes registers (changed in
      // place it cost the loop 100 bytes a lane of scratch).
      if (write) store();
      __builtin_amdgcn_s_waitcnt(0);
#pragma unroll 1
      for (int w = 0; w < D; w += 64) {
        uint32_t up = 0, down = 0;  // bit 4 j + e: column w + 8 j + 4 u + e
#pragma unroll 1
        for (int i = -it.c_begin; i < span.total - it.c_begin; ++i) {
          if (!odd_row && i >= t_lo && i < t_hi) continue;
#pragma unroll 1
          for (int first = first_key(i), left = kKeys; left > 0; left -= 16, first += 16) {
            if (first >= span.end || (first >= span.skip_lo && first + 16 <= span.skip_hi)) continue;
            const int page = bt[first >> a.page_shift];
            if ((uint32_t)page >= (uint32_t)a.n_pages || !__any(write & ((up & down) != ~0u))) continue;
            const __bf16* const v = (const __bf16*)(vbase + 2 * (uint64_t)(page * a.vc_sp + (first & ((1 << a.page_shift) - 1)) * a.vc_st)) + w;
            // sixteen rows' bytes, 32 of a lane; most hold none
            const bf16x8 x0 = *(const bf16x8*)(v + lane / 8 * a.vc_st + lane % 8 * 8), x1 = *(const bf16x8*)(v + (8 + lane / 8) * a.vc_st + lane % 8 * 8);
            bool any = false;
#pragma unroll
            for (int e = 0; e < 8; ++e) any |= !__builtin_isfinite((float)x0[e]) | !__builtin_isfinite((float)x1[e]);
            if (!__any(any)) continue;
#pragma unroll 1
            for (int at = 0; at < 16 * 8; ++at) {
              const int key = first + at / 8;
              const bool vis = (key <= pos) & ((a.window == 0) | (key > pos - a.window) | (key < a.sinks));
              const bf16x4 x = *(const bf16x4*)(v + at / 8 * a.vc_st + at % 8 * 8 + 4 * u);
#pragma unroll
              for (int e = 0; e < 4; ++e) note_odd((float)x[e], vis, 1u << (4 * (at % 8) + e), up, down);
            }
          }
        }
#pragma unroll 1
        for (int i = 0; i < 32; ++i, up >>= 1, down >>= 1)
          if (write & (l == l) & ((up | down) & 1)) (op - 4 * u)[w + 8 * (i / 4) + i % 4] = (__bf16)odd_or(0.0f, 1, up, down);
      }
      write = false;
    }
    // The next item's first chunks come while this one's rows are written.
    lds_barrier();  // every wave has read the flags
    if (one) odd_s = bad_s = 0;
    const bool more = it.next >= 0;
    if (more) begin();
    if (write) store();
    if (!more) break;
  }
}

}  // namespace

int32_t cev_paged_tile_launch(const PagedArgs& a, int32_t d, int32_t target, void* stream) {
  if (d == 128)
    hipLaunchKernelGGL(paged_tile_kernel<128>, dim3((unsigned)(target * a.hkv)), dim3(kThreads), 0, (hipStream_t)stream, a);
  else
    hipLaunchKernelGGL(paged_tile_kernel<256>, dim3((unsigned)(target * a.hkv)), dim3(kThreads), 0, (hipStream_t)stream, a);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return cev_fail(CEV_ERR_HIP, "paged attention launch: %s", hipGetErrorString(e));
  return CEV_OK;
}
