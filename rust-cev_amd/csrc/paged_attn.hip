// Attention of each request's new tokens over a paged K/V cache.
//
// This file: requests with few new rows (one token to a short question).
// A work item (cev_paged_plan) is up to 32 query slots (rows x the g query
// heads of one KV head: slot -> row slot / g, head slot % g) and a run of the
// 32-key sub-tiles that they see.  Its workgroup's four waves take the
// sub-tiles in turn, each on its own: no barrier until their partial results
// are joined.  Scores are computed transposed, S^T = K . Q^T, on 32x32 MFMA
// tiles, so a lane holds 16 keys of one query row and the softmax's running
// max and sum stay in its registers; O^T = V^T . P^T follows with P as the B
// operand.
//
// K and V go from HBM straight into this wave's own LDS (buffer_load ... lds,
// 1 KB an instruction), one sub-tile ahead: K of the next one is asked for when
// its scores are made, V when its products are.  A page's base is a scalar
// 64-bit address (page ids are wave-uniform), so the cache may have any size;
// keys past the end, in pages behind the window or not visible to any row of
// the item get an offset out of the resource's range and read as zero.
//
// Rounding: scores, sums, the running maximum and O are f32; bf16 probabilities
// are rounded to bf16 for the product (at most 2^-8 of each weight, no more than
// the output's own rounding is off by), and their sum is that of the rounded
// ones, so that a row's weights add up to one.
//
// What bounds it, alone on the card, us:
//   bf16 d = 128  64 requests of one token, 64 to 8192 keys, 8 KV heads: 186 to
//                 189, for 1077 MB 5.7 TB/s: HBM
//   bf16 d = 128  one token after 300 keys: 9.0, a chain of trips: the list's item,
//                 page ids, K, scores, V, the pieces' join; a launch is 3.5
//   bf16 d = 256  28 requests of 1 to 8 rows and 4 of 64, 100 to 4096 keys: 92 to
//                 104, for 560 MB 6.1 to 5.4 TB/s of HBM and MALL.  276 MB would do: the tiles of
//                 one request read its keys each for themselves.  Of a round's 7000
//                 cycles 4000 are spent handing out loads that wait for room
//   f32           12 chunks of 17 to 41 rows, 256 to 2048 keys: 59, of which a
//                 quarter are the items' starts and joins; a round of 9100 cycles has 3000
//                 of MFMAs, the rest makes bf16 parts of K and V beside them and
//                 hands over the loads
//
// Pieces of a tile whose keys lie in several workgroups' runs write partial
// results (f32); the last of them to arrive (a counter per tile and KV head)
// joins all in their order, so the result does not depend on who is last.
#include "attn_pipe.h"
#include "paged_device.h"

namespace {

constexpr int kWaves = 4;
constexpr int kThreads = kWaves * 64;
constexpr int kKeys = 32, kSlots = paged_slots(kPagedFew);  // keys of a sub-tile
static_assert(paged_keys(kPagedFew, 128) == kKeys && paged_keys(kPagedFew, 256) == kKeys, "the work list's sub-tiles");

// Workgroup b writes NaN over its share of out's rows.
template <typename T, int D>
__device__ void paged_poison(const PagedArgs& a) {
  const int64_t G = gridDim.x;
  const int64_t r0 = (int64_t)blockIdx.x * a.t / G, r1 = (int64_t)(blockIdx.x + 1) * a.t / G;
  const int64_t per_row = (int64_t)a.hkv * a.g * D;
  for (int64_t i = threadIdx.x; i < (r1 - r0) * per_row; i += blockDim.x) {
    const int64_t r = r0 + i / per_row, h = (i % per_row) / D, e = i % D;
    ((T*)a.out)[r * a.o_st + h * a.o_sh + e] = (T)__builtin_nanf("");
  }
}

// f32 values as sums of three bf16 parts and the six large part products
// (see fan_attn.hip).
typedef float f32x2 __attribute__((ext_vector_type(2)));
__device__ __forceinline__ void bf16_parts(const float* x, bf16x8* p) {
#pragma unroll
  for (int e = 0; e < 8; e += 2) {
    f32x2 r = {x[e], x[e + 1]};
#pragma unroll
    for (int i = 0; i < 3; ++i) {
      const bf16x2 b = __builtin_convertvector(r, bf16x2);
      p[i][e] = b[0];
      p[i][e + 1] = b[1];
      r = r - __builtin_convertvector(b, f32x2);
    }
  }
}
__device__ __forceinline__ f32x16 parts_mma(const bf16x8* a, const bf16x8* b, f32x16 c) {
#pragma unroll
  for (int o = 2; o >= 0; --o)
#pragma unroll
    for (int i = 0; i <= o; ++i) c = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a[i], b[o - i], c, 0, 0, 0);
  return c;
}

// 16-byte block of row `row` that block blk of K is stored at: a row's blocks
// are permuted so that the operand reads (16 rows at once) meet every bank.
__device__ __forceinline__ int k_place(int blk, int row) { return blk ^ (row & 15); }
// of V: bf16 is read transposed, four rows x four blocks at once; f32 by two
// half waves whose rows differ in bit 2.
template <typename T>
__device__ __forceinline__ int v_place(int blk, int row) {
  return sizeof(T) == 2 ? blk ^ ((row & 3) << 2) : blk ^ (((row >> 2) & 1) << 3);
}

// Operand reads through asm: the compiler places a wait for every load in
// flight before each LDS read that it emits itself (it cannot tell the
// buffers apart), which would drain the fetches ahead.
using pipe::i32x4;
using pipe::read_b128;
template <int OFF>
__device__ __forceinline__ float read_b32(int vaddr) {
  static_assert(OFF >= 0 && OFF < 65536, "ds offset field");
  float r;
  asm volatile("ds_read_b32 %0, %1 offset:%2" : "=v"(r) : "v"(vaddr), "i"(OFF) : "memory");
  return r;
}
template <int N, typename R>
__device__ __forceinline__ void pass_through(R& r) {
  asm volatile("s_waitcnt lgkmcnt(%1)" : "+v"(r) : "i"(N));
}
// All LDS reads but the last N have returned, and the values given are there.
template <int N, typename... R>
__device__ __forceinline__ void wait_reads(R&... r) {
  static_assert(N >= 0 && N < 16, "lgkmcnt range");
  (void)std::initializer_list<int>{(pass_through<N>(r), 0)...};
}
// Six MFMAs with the vector instructions of the region spread between them.
__device__ __forceinline__ void beside_mfmas() {
#pragma unroll
  for (int i = 0; i < 6; ++i) {
    __builtin_amdgcn_sched_group_barrier(0x8, 1, 0);  // one MFMA
    __builtin_amdgcn_sched_group_barrier(0x2, 8, 0);  // eight VALU instructions
  }
}
// Every LDS read has returned, and r holds its value.
template <typename R>
__device__ __forceinline__ void wait_read(R& r) {
  asm volatile("s_waitcnt lgkmcnt(0)" : "+v"(r));
}

// Waves a SIMD that registers are left for: two workgroups of bf16 d = 128 share
// a CU, the others' LDS holds one.
template <typename T, int D>
constexpr int kMinWaves = sizeof(T) == 2 && D == 128 ? 2 : 1;
template <typename T, int D>
__global__ __launch_bounds__(kThreads) __attribute__((amdgpu_waves_per_eu(kMinWaves<T, D>))) void paged_attn_kernel(PagedArgs a) {
  using F = Frag<T, D>;
  constexpr bool BF = sizeof(T) == 2;
  constexpr int NDT = D / 32;
  constexpr int kRB = D * (int)sizeof(T);        // bytes of one key row
  constexpr int kTile = kKeys * kRB;        // K or V of a sub-tile
  constexpr int kLoads = kTile / 1024;           // 1 KB loads of it
  constexpr int kRows = 1024 / kRB, kBlk = kRB / 16;  // rows of one load, 16-byte blocks of a row
  constexpr int RS = D + 4;                      // row stride (floats) of a partial result in LDS
  constexpr int kRing = kWaves * 2 * kTile, kOut = kWaves * 32 * RS * 4, kBody = kRing > kOut ? kRing : kOut;
  // Q of d = 256 lies in LDS, shared by the waves (with it in registers O is
  // moved to and from the accumulation registers, and some of it spilled).
  constexpr bool kQInLds = BF && D == 256;
  __shared__ __align__(16) char lds[kBody + (kQInLds ? D / 16 * 1024 : 0)];
  __shared__ float2 ml[kWaves * 32];  // of a slot: maximum, sum; below zero (or -0) with odd_v
  __shared__ int32_t last_s;

  const int run = blockIdx.x / (uint32_t)a.hkv, kvh = blockIdx.x - run * a.hkv;
  PagedWalk walk(a, run);
  int n_parts;
  if (!paged_plan_ok(a, kPagedFew, n_parts)) {
    paged_poison<T, D>(a);
    return;
  }
  if (run >= n_parts) return;
  for (bool more = true; more;) {
    const PagedItem it = walk.item();
    more = it.next >= 0;
    const int tid = threadIdx.x, lane = tid & 63, wave = uniform_i32(tid >> 6);
    const int n = lane & 31, u = lane >> 5;
    const int gs = __builtin_ctz(a.g);
    const bool ok = (n >> gs) < it.n_rows;
    const int row = it.row0 + (ok ? n >> gs : 0), head = kvh * a.g + (n & (a.g - 1));
    const int pos = ok ? it.pos0 + (n >> gs) : -1;
    const int pos1 = it.pos0 + it.n_rows - 1;
    const PagedSpan span = paged_span(kKeys, it.pos0, pos1, a.window, a.sinks);

    // ---- Q, as the B operand; zeros in slots without a row
    const T* const qrow = (const T*)a.q + (int64_t)row * a.q_st + (int64_t)head * a.q_sh;
    F fr;
    auto load_q8 = [&](int st, f32x4* x) {
      x[0] = ok ? *(const f32x4*)(qrow + 16 * st + 8 * u) : f32x4{};
      x[1] = ok ? *(const f32x4*)(qrow + 16 * st + 8 * u + 4) : f32x4{};
    };
    bf16x8 qp[BF ? 1 : D / 16][3];  // f32: the parts of q[16 st + 8 u ..]
    if constexpr (!BF) {
#pragma unroll
      for (int st = 0; st < D / 16; ++st) {
        f32x4 q[2];
        float x[8];
        load_q8(st, q);
        __builtin_memcpy(x, q, 32);
        bf16_parts(x, qp[st]);
      }
    } else if constexpr (kQInLds) {
#pragma unroll
      for (int i = 0; i < D / 16 / kWaves; ++i) {
        const int st = wave * (D / 16 / kWaves) + i;
        const bf16x8 z = {};
        *(bf16x8*)(lds + kBody + st * 1024 + lane * 16) = ok ? *(const bf16x8*)(qrow + 16 * st + 8 * u) : z;
      }
    } else {
      fr.load_q(qrow, ok, u);
    }

    // ---- this wave's sub-tiles: c_begin + wave, + kWaves, ...
    const int c_end = it.c_end;
    auto first_key = [&](int c) { return kKeys * (c < span.sinks ? c : c - span.sinks + span.first); };
    const int32_t* const bt = a.bt + it.req * a.bt_stride;
    const uint64_t kbase = (uint64_t)((const T*)a.kc + kvh * a.kc_sh), vbase = (uint64_t)((const T*)a.vc + kvh * a.vc_sh);
    const int kr = uniform_i32((int)(a.kc_st * (int64_t)sizeof(T))), vr = uniform_i32((int)(a.vc_st * (int64_t)sizeof(T)));
    // Lane l keeps the two page ids of this wave's sub-tile 64 b + l of the
    // current batch b (a page of 16 keys holds half a sub-tile).
    int batch_first = 0, page_a = 0, page_b = 0;
    auto load_pages = [&](int c0) {
      batch_first = c0;
      const int c = min(c0 + kWaves * lane, c_end - 1);
      const int j = first_key(max(c, 0));
      // (the last sub-tile may reach beyond the block table's last page)
      page_a = bt[min(j >> a.page_shift, a.max_pages - 1)];
      page_b = bt[min((j + 16) >> a.page_shift, a.max_pages - 1)];
    };
    bool sees_bad = false;  // this lane's row sees a key of a page outside the cache
    char* const ring = lds + wave * 2 * kTile;
    const int lds_ring = (int)(size_t)(const __attribute__((address_space(3))) char*)ring;
    // Row (of load 0 of a half) and block there of this lane's 16 bytes.
    const int ld_row = lane / kBlk, ld_blk = lane % kBlk;
    // K (which = 0) or V (1) of sub-tile c into its buffer; past the end: zeros.
    auto fetch = [&](int c, auto which_c) {
      constexpr int which = decltype(which_c)::value;
      const bool real = c < c_end;
      if (real && which == 0 && c >= batch_first + kWaves * 64) load_pages(c);
      const int key0 = real ? first_key(c) : 0;
      const int l = real ? (c - batch_first) / kWaves : 0;
      const int stride = which ? vr : kr;
      const int64_t page_bytes = (which ? a.vc_sp : a.kc_sp) * (int64_t)sizeof(T);
      // every key of it is seen by some row of the item
      const bool full = key0 + kKeys <= span.end && !(key0 < span.skip_hi && key0 + kKeys > span.skip_lo);
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const int first = key0 + 16 * half;
        const bool seen = real && first < span.end && !(first >= span.skip_lo && first + 16 <= span.skip_hi);
        int page = half ? __builtin_amdgcn_readlane(page_b, l) : __builtin_amdgcn_readlane(page_a, l);
        const bool in = (uint32_t)page < (uint32_t)a.n_pages;
        if (which == 0 && seen && !in) sees_bad |= (first <= pos) & ((a.window == 0) | (first + 15 > pos - a.window) | (first < a.sinks));
        page = in ? page : 0;
        const uint64_t base = (which ? vbase : kbase) + (uint64_t)(page * page_bytes) + (uint64_t)((first & ((1 << a.page_shift) - 1)) * (int64_t)stride);
        const __amdgpu_buffer_rsrc_t rs = __builtin_amdgcn_make_buffer_rsrc((void*)uniform_u64(base), (short)0, uniform_i32(seen && in ? 16 * stride : 0), kBufferWord3);
        char* const to = ring + which * kTile + half * (kTile / 2);
        // (the two cases apart, or every load is a branch of its own)
        auto loads = [&](auto full_c) {
#pragma unroll
          for (int i = 0; i < kLoads / 2; ++i) {
            const int r = kRows * i + ld_row;
            int off = r * stride + ((which ? v_place<T>(ld_blk, r) : k_place(ld_blk, r)) << 4);
            if (!decltype(full_c)::value) {
              const int key = first + r;
              off = ((key < span.end) & !((key >= span.skip_lo) & (key < span.skip_hi))) ? off : INT32_MAX;
            }
            __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, (__attribute__((address_space(3))) void*)(to + 1024 * i), 16, off, 0, 0, 0);
          }
        };
        if (full)
          loads(std::true_type{});
        else
          loads(std::false_type{});
      }
    };
    using K_c = std::integral_constant<int, 0>;
    using V_c = std::integral_constant<int, 1>;

    f32x16 o[NDT];
    float m_run, l_run;
    auto reset = [&] {
#pragma unroll
      for (int dt = 0; dt < NDT; ++dt) o[dt] = f32x16{};
      m_run = -1e30f;
      l_run = 0.0f;
    };
    reset();
    const int lds_q = (int)(size_t)(const __attribute__((address_space(3))) char*)lds + kBody + lane * 16;
    // Byte offsets of the operand reads within a sub-tile of K and of V.
    int koff[8], voff[NDT];
#pragma unroll
    for (int j = 0; j < 8; ++j) koff[j] = n * kRB + (k_place(BF ? 2 * j + u : 4 * (j >> 1) + 2 * u + (j & 1), n) << 4);
    {
      const int i = lane & 15, rr = i >> 2, blk = 2 * ((lane >> 4) & 1) + ((i & 3) >> 1);
#pragma unroll
      for (int dt = 0; dt < NDT; ++dt)
        voff[dt] = BF ? (4 * u + rr) * kRB + (v_place<T>(4 * dt + blk, rr) << 4) + 8 * (i & 1)
                      : 4 * u * kRB + (v_place<T>(8 * dt + n / 4, 4 * u) << 4) + 4 * (n & 3);
    }
    // Whether the rows differ in what they see of the sub-tile at key0.
    auto is_masked = [&](int key0) {
      return key0 + kKeys - 1 > it.pos0 || (a.window > 0 && key0 <= pos1 - a.window && key0 + kKeys > a.sinks);
    };
    bool odd_v = false;  // such a sub-tile's V held infinities or NaN

    // This wave's sub-tiles.  f32: an infinite value (or one above bf16's range)
    // has no parts; a wave that ends with anything non-finite walks its keys again
    // on the f32 unit (exact).
    auto pass = [&](auto exact_c) {
      constexpr bool kExact = decltype(exact_c)::value;
      int c = it.c_begin + wave;
      if (c < c_end) load_pages(c);
      if constexpr (kQInLds) __syncthreads();  // Q is in LDS
      if (c >= c_end) return;
      fetch(c, K_c{});
      fetch(c, V_c{});
      auto step = [&] {
        const int key0 = first_key(c);
        // K of this sub-tile has landed once only later loads are in flight
        pipe::wait_vmcnt<kLoads>();
        asm volatile("" ::: "memory");
        f32x16 s = f32x16{};
        const int ka = lds_ring;
        if constexpr (BF) {
          // K operands (and Q's of d = 256) in groups, one group ahead of the MFMAs
          constexpr int kSteps = kQInLds ? 2 : 4, kQReads = kQInLds ? 1 : 0;
          i32x4 kf[2][kSteps], qf[2][kSteps * kQReads + 1];
          auto k_issue = [&](auto g_c) {
            constexpr int G = decltype(g_c)::value;
            static_for<kSteps>([&](auto e_c) {
              // read J is block 2 J + u; bit 4 of a block's place is its own
              constexpr int E = decltype(e_c)::value, J = G * kSteps + E;
              kf[G & 1][E] = read_b128<(J / 8) * 256>(ka + koff[J % 8]);
            });
            static_for<kSteps * kQReads>([&](auto e_c) {
              constexpr int E = decltype(e_c)::value;
              qf[G & 1][E] = read_b128<(G * kSteps + E) * 1024>(lds_q);
            });
          };
          k_issue(std::integral_constant<int, 0>{});
          static_for<D / 16 / kSteps>([&](auto g_c) {
            constexpr int G = decltype(g_c)::value;
            static_for<kSteps>([&](auto e_c) { wait_read(kf[G & 1][decltype(e_c)::value]); });
            static_for<kSteps * kQReads>([&](auto e_c) { wait_read(qf[G & 1][decltype(e_c)::value]); });
            if constexpr (G + 1 < D / 16 / kSteps) k_issue(std::integral_constant<int, G + 1>{});
            static_for<kSteps>([&](auto e_c) {
              constexpr int E = decltype(e_c)::value, st = G * kSteps + E;
              const bf16x8 k = __builtin_bit_cast(bf16x8, kf[G & 1][E]);
              if constexpr (kQInLds)
                s = __builtin_amdgcn_mfma_f32_32x32x16_bf16(k, __builtin_bit_cast(bf16x8, qf[G & 1][E]), s, 0, 0, 0);
              else
                fr.qk_mfma(k, st, s);
            });
          });
        } else {
          // Step st: two reads (blocks 4 st + 2 u and the next), the parts of their
          // values, six MFMAs.  A step's parts are made beside the MFMAs of the one
          // before; its reads are two steps ahead.
          i32x4 kf[3][2];
          bf16x8 kp[2][3];
          auto k_issue = [&](auto st_c) {
            constexpr int ST = decltype(st_c)::value;
            static_for<2>([&](auto e_c) {
              constexpr int E = decltype(e_c)::value, J = 2 * ST + E;
              kf[ST % 3][E] = read_b128<(J / 8) * 256>(ka + koff[J % 8]);
            });
          };
          auto values = [&](auto st_c, float* x) {
            constexpr int ST = decltype(st_c)::value;
            __builtin_memcpy(x, &kf[ST % 3][0], 16);
            __builtin_memcpy(x + 4, &kf[ST % 3][1], 16);
          };
          k_issue(std::integral_constant<int, 0>{});
          k_issue(std::integral_constant<int, 1>{});
          wait_reads<2>(kf[0][0], kf[0][1]);
          if constexpr (!kExact) {
            float x[8];
            values(std::integral_constant<int, 0>{}, x);
            bf16_parts(x, kp[0]);
          }
          static_for<D / 16>([&](auto st_c) {
            constexpr int ST = decltype(st_c)::value;
            if constexpr (ST + 2 < D / 16) k_issue(std::integral_constant<int, ST + 2>{});
            if constexpr (ST + 1 < D / 16) wait_reads<(ST + 2 < D / 16 ? 2 : 0)>(kf[(ST + 1) % 3][0], kf[(ST + 1) % 3][1]);
            float x[8];
            if constexpr (kExact) {
              float q[8];
              f32x4 q4[2];
              values(st_c, x);
              load_q8(ST, q4);
              __builtin_memcpy(q, q4, 32);
#pragma unroll
              for (int e = 0; e < 8; ++e) s = __builtin_amdgcn_mfma_f32_32x32x2f32(x[e], q[e], s, 0, 0, 0);
            } else {
              if constexpr (ST + 1 < D / 16) {
                values(std::integral_constant<int, ST + 1>{}, x);
                bf16_parts(x, kp[(ST + 1) & 1]);
              }
              s = parts_mma(kp[ST & 1], qp[ST], s);
              beside_mfmas();
            }
          });
        }
        asm volatile("" ::: "memory");
        const bool masked = is_masked(key0);
        if (masked) {
          // bounds of the register's place, 8 (i / 4) + i % 4
          const int k0 = key0 + 4 * (fresh_lane_id() >> 5), hi = pos - k0;
          const int lo = a.window == 0 || pos < a.window ? INT32_MIN : pos - a.window - k0, first = a.sinks - k0;
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            const int at = 8 * (i >> 2) + (i & 3);
            s[i] = (at <= hi) & ((at > lo) | (at < first)) ? s[i] : -INFINITY;
          }
        }
        // (s is made: K's buffer is free for the next sub-tile)
        __builtin_amdgcn_sched_barrier(0);
        fetch(c + kWaves, K_c{});
        __builtin_amdgcn_sched_barrier(0);
        float mx = -INFINITY;
#pragma unroll
        for (int i = 0; i < 16; ++i) mx = fmaxf(mx, s[i]);
        const float m_cand = pair_max(mx) * a.scale_log2;
        const bool grow = m_cand > m_run + kRescale;
        if (__ballot(grow)) {
          const float m_new = grow ? m_cand : m_run;
          const float alpha = fast_exp2(m_run - m_new);
          m_run = m_new;
          l_run *= alpha;
#pragma unroll
          for (int dt = 0; dt < NDT; ++dt) o[dt] *= alpha;
        }
#pragma unroll
        for (int i = 0; i < 16; ++i) s[i] = fast_exp2(__builtin_fmaf(s[i], a.scale_log2, -m_run));
        typename F::P p;
        F::make_p(s, p, l_run);
        pipe::wait_vmcnt<kLoads>();
        asm volatile("" ::: "memory");
        if (masked) {
          // 0 times an infinity or NaN is NaN: a key that only some of the rows
          // see must not reach the others.  Such values are zeros for the products;
          // the rows that see them get them when the waves' results are joined.
          const f32x4* const vt = (const f32x4*)(ring + kTile);
          uint32_t odd = 0;
#pragma unroll
          for (int i = 0; i < kTile / 1024; ++i) {
            const f32x4 w = vt[64 * i + lane];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const uint32_t x = __float_as_uint(w[e]);
              odd |= (uint32_t)((x & 0x7f800000u) == 0x7f800000u);
              if (BF) odd |= (uint32_t)((x & 0x7f80u) == 0x7f80u);
            }
          }
          if (__ballot(odd != 0)) {
            odd_v = true;
            wave_lds_sync();
            for (int i = lane; i < kKeys * D; i += 64) {
              T* const x = (T*)(ring + kTile) + i;
              const float v = (float)*x;
              if ((__float_as_uint(v) & 0x7f800000u) == 0x7f800000u) *x = (T)0.0f;
            }
            wave_lds_sync();
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
          }
        }
        if constexpr (BF) {
          const int va = lds_ring + kTile;
          constexpr int kGrp = 4;
          pipe::i32x2 f[2][kGrp][2];
          auto issue = [&](auto g_c) {
            constexpr int G = decltype(g_c)::value;
            static_for<kGrp>([&](auto e_c) {
              constexpr int E = decltype(e_c)::value, J = G * kGrp + E;
              constexpr int OFF = 16 * (J / NDT) * kRB;
              f[G & 1][E][0] = pipe::read_tr<OFF>(va + voff[J % NDT]);
              f[G & 1][E][1] = pipe::read_tr<OFF + 8 * kRB>(va + voff[J % NDT]);
            });
          };
          issue(std::integral_constant<int, 0>{});
          static_for<F::NPV / kGrp>([&](auto g_c) {
            constexpr int G = decltype(g_c)::value;
            static_for<kGrp>([&](auto e_c) {
              constexpr int E = decltype(e_c)::value;
              pipe::wait_tr<0>(f[G & 1][E][0], f[G & 1][E][1]);
            });
            if constexpr (G + 1 < F::NPV / kGrp) issue(std::integral_constant<int, G + 1>{});
            static_for<kGrp>([&](auto e_c) {
              constexpr int E = decltype(e_c)::value;
              const bf16x4 lo = __builtin_bit_cast(bf16x4, f[G & 1][E][0]), hi = __builtin_bit_cast(bf16x4, f[G & 1][E][1]);
              F::pv_mfma(bf16x8{lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]}, G * kGrp + E, p, o);
            });
          });
        } else {
          // V values of step j = 4 h + dt, keys 16 h + 8 (e / 4) + 4 u + e % 4 of
          // column 32 dt + n: as above
          float vf[3][8];
          const int va = lds_ring + kTile;
          auto v_issue = [&](auto j_c) {
            constexpr int J = decltype(j_c)::value, H = J / NDT, DT = J % NDT;
            static_for<8>([&](auto e_c) {
              constexpr int E = decltype(e_c)::value;
              vf[J % 3][E] = read_b32<(16 * H + 8 * (E >> 2) + (E & 3)) * kRB>(va + voff[DT]);
            });
          };
          constexpr int kSteps = 2 * NDT;
          bf16x8 pp[2][3], vp[2][3];
          v_issue(std::integral_constant<int, 0>{});
          v_issue(std::integral_constant<int, 1>{});
          if constexpr (!kExact) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              float x[8];
#pragma unroll
              for (int e = 0; e < 8; ++e) x[e] = p.v[8 * h + e];
              bf16_parts(x, pp[h]);
            }
          }
          wait_reads<8>(vf[0][0], vf[0][1], vf[0][2], vf[0][3], vf[0][4], vf[0][5], vf[0][6], vf[0][7]);
          if constexpr (!kExact) bf16_parts(vf[0], vp[0]);
          static_for<kSteps>([&](auto j_c) {
            constexpr int J = decltype(j_c)::value, H = J / NDT, DT = J % NDT, N = (J + 1) % 3;
            if constexpr (J + 2 < kSteps) v_issue(std::integral_constant<int, J + 2>{});
            if constexpr (J + 1 < kSteps)
              wait_reads<(J + 2 < kSteps ? 8 : 0)>(vf[N][0], vf[N][1], vf[N][2], vf[N][3], vf[N][4], vf[N][5], vf[N][6], vf[N][7]);
            if constexpr (kExact) {
#pragma unroll
              for (int e = 0; e < 8; ++e) o[DT] = __builtin_amdgcn_mfma_f32_32x32x2f32(vf[J % 3][e], p.v[8 * H + e], o[DT], 0, 0, 0);
            } else {
              if constexpr (J + 1 < kSteps) bf16_parts(vf[N], vp[(J + 1) & 1]);
              o[DT] = parts_mma(vp[J & 1], pp[H], o[DT]);
              beside_mfmas();
            }
          });
        }
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        __builtin_amdgcn_sched_barrier(0);
        fetch(c + kWaves, V_c{});
        __builtin_amdgcn_sched_barrier(0);
        c += kWaves;
      };
      while (c < c_end) step();
      // loads past the end still write zeros into LDS
      pipe::wait_vmcnt<0>();
      asm volatile("" ::: "memory");
    };
    pass(std::false_type{});
    if constexpr (!BF) {
      float t = l_run * 0.0f + m_run * 0.0f;
#pragma unroll
      for (int dt = 0; dt < NDT; ++dt)
#pragma unroll
        for (int i = 0; i < 16; ++i) t += o[dt][i] * 0.0f;
      if (__any(!(t == 0.0f))) {
        reset();
        pass(std::true_type{});
      }
    }

    // ---- join the waves' partial results through LDS
    const float l = pair_sum(l_run) + (sees_bad ? __builtin_nanf("") : 0.0f);
    __syncthreads();  // every wave is done with its part of the ring
    float* const ob = (float*)lds;
#pragma unroll
    for (int dt = 0; dt < NDT; ++dt)
#pragma unroll
      for (int q4 = 0; q4 < 4; ++q4)
        *(f32x4*)(ob + (wave * 32 + n) * RS + dt * 32 + 8 * q4 + 4 * u) = f32x4{o[dt][4 * q4], o[dt][4 * q4 + 1], o[dt][4 * q4 + 2], o[dt][4 * q4 + 3]};
    if (u == 0) ml[wave * 32 + n] = make_float2(m_run, odd_v ? -l : l);
    __syncthreads();
    const int slots = it.n_rows << gs;
    constexpr int kCols = D / 4;  // 4-column units of a slot
    const bool split = it.n_pieces > 1;
    // partial results of the tile's pieces, [slot][D] then [slot] (m, l)
    constexpr int kRec = kSlots * (D + 2);
    float* const rec0 = (float*)(a.work + a.records_off) + ((int64_t)it.rec * a.hkv + kvh) * kRec;
    auto record = [&](int piece) {
      return __builtin_amdgcn_make_buffer_rsrc((void*)uniform_u64((uint64_t)(rec0 + (int64_t)piece * a.hkv * kRec)), (short)0, kRec * 4, kBufferWord3);
    };
    auto put = [&](int slot, int col, const f32x4& x, float L) {
      T* const op = (T*)a.out + (int64_t)(it.row0 + (slot >> gs)) * a.o_st + (int64_t)(kvh * a.g + (slot & (a.g - 1))) * a.o_sh + col;
      // a row that sees no key is 0; a sum that is NaN makes its row NaN
      float v[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] = L == 0.0f ? 0.0f : x[e] / L;
      store_vec4<T>(op, v);
    };
    auto put_odd = [&](int slot, int col, uint32_t up, uint32_t down) {
      T* const op = (T*)a.out + (int64_t)(it.row0 + (slot >> gs)) * a.o_st + (int64_t)(kvh * a.g + (slot & (a.g - 1))) * a.o_sh + col;
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if ((up | down) >> e & 1) op[e] = (T)odd_or(0.0f, 1u << e, up, down);
    };
    const __amdgpu_buffer_rsrc_t mine = record(it.piece);
    const __amdgpu_buffer_rsrc_t all = __builtin_amdgcn_make_buffer_rsrc((void*)uniform_u64((uint64_t)rec0), (short)0, uniform_i32(it.n_pieces * a.hkv * kRec * 4), kBufferWord3);
    bool odd = false, odd_masked = false;
    for (int i = tid; i < slots * kCols; i += kThreads) {
      const int slot = i / kCols, col = 4 * (i % kCols);
      float M = -INFINITY, L = 0.0f;
      f32x4 x = f32x4{};
#pragma unroll
      for (int w = 0; w < kWaves; ++w) M = fmaxf(M, ml[w * 32 + slot].x);
#pragma unroll
      for (int w = 0; w < kWaves; ++w) {
        const float2 v = ml[w * 32 + slot];
        const float f = fast_exp2(v.x - M);
        L += f * __builtin_fabsf(v.y);
        odd_masked |= __builtin_signbitf(v.y) != 0;
        x += f * *(const f32x4*)(ob + (w * 32 + slot) * RS + col);
      }
      odd |= (L == L) & !finite4(x);
      if (!split) {
        put(slot, col, x, L);
      } else {
        put_past_l2(mine, (slot * D + col) * 4, x);
        if (col == 0) put_past_l2(mine, (kSlots * D + 2 * slot) * 4, make_float2(M, L));
      }
    }
    // Infinities and NaN of V (see note_odd): the sub-tiles whose rows differ in what
    // they see held some, or a row has come out so.  They go over what was written
    // (in the loop above they took it 0.4 us).
    if (__any(odd | odd_masked)) {
      const bool every = __any(odd);
      __builtin_amdgcn_s_waitcnt(0);
#pragma unroll 1
      for (int i = tid; i < slots * kCols; i += kThreads) {
        const int slot = i / kCols, col = 4 * (i % kCols), row_pos = it.pos0 + (slot >> gs);
        uint32_t up = 0, down = 0;
#pragma unroll 1
        for (int c = it.c_begin; c < c_end; ++c) {
          if (!every && !is_masked(first_key(c))) continue;
#pragma unroll 1
          for (int first = first_key(c), half = 0; half < 2; ++half, first += 16) {
            if (first >= span.end || (first >= span.skip_lo && first + 16 <= span.skip_hi)) continue;
            const int page = bt[first >> a.page_shift];
            if ((uint32_t)page >= (uint32_t)a.n_pages) continue;
            const T* const v = (const T*)(vbase + sizeof(T) * (uint64_t)(page * a.vc_sp + (first & ((1 << a.page_shift) - 1)) * a.vc_st)) + col;
#pragma unroll 4
            for (int k = 0; k < 16; ++k) {
              const int key = first + k;
              const bool vis = (key <= row_pos) & ((a.window == 0) | (key > row_pos - a.window) | (key < a.sinks));
              typedef T vec4 __attribute__((ext_vector_type(4)));
              const vec4 y = *(const vec4*)(v + k * a.vc_st);
#pragma unroll
              for (int e = 0; e < 4; ++e) note_odd((float)y[e], vis, 1u << e, up, down);
            }
          }
        }
        bool nan_row = false;
        for (int w = 0; w < kWaves; ++w) nan_row |= ml[w * 32 + slot].y != ml[w * 32 + slot].y;
        if (nan_row) continue;
        if (!split) put_odd(slot, col, up, down);
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (split && ((up | down) >> e & 1)) put_past_l2(mine, (slot * D + col + e) * 4, odd_or(0.0f, 1u << e, up, down));
      }
    }
    // A split tile's stores have reached memory before the workgroup counts
    // itself; and the ring is the next item's.
    __builtin_amdgcn_s_waitcnt(0);
    __syncthreads();
    if (!split) continue;
    int32_t* const counter = (int32_t*)(a.work + a.counters_off) + (int64_t)it.split * a.hkv + kvh;
    if (tid == 0) last_s = __hip_atomic_fetch_add(counter, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == it.n_pieces - 1;
    __syncthreads();
    const bool last = last_s;
    __syncthreads();
    if (!last) continue;
    // Threads -> (group of pieces, 4-column units kThreads apart): with few rows
    // several groups walk the pieces and meet in LDS.  All loads of kUnits x
    // kBatch partial results are in flight at once: a trip past the L2 takes
    // 1.5 us (with one unit at a time the joining of three pieces of 32 slots took
    // 6 us at d = 128, 12 us at d = 256).  Two units of bf16 d = 128, whose registers
    // two workgroups share: with four, 16 requests of 32 rows in 1024 keys took 26.5 us,
    // 24.9 with two.
    constexpr int kUnits = BF && D == 128 ? 2 : 4, kBatch = 4;
    const int units = slots * kCols;
    int groups = 1;
    while (groups < 8 && 2 * groups * units <= kThreads && 2 * groups < it.n_pieces) groups *= 2;
    odd = false;
    const int group = groups > 1 ? tid / units : 0, unit0 = groups > 1 ? tid % units : tid;
    for (int i0 = 0; i0 < units; i0 += kUnits * kThreads) {
      float M[kUnits], L[kUnits];
      f32x4 x[kUnits];
#pragma unroll
      for (int k = 0; k < kUnits; ++k) {
        M[k] = -INFINITY;
        L[k] = 0.0f;
        x[k] = f32x4{};
      }
      if (group < groups) {
        for (int p0 = group; p0 < it.n_pieces; p0 += kBatch * groups) {
          f32x4 y[kUnits][kBatch];
          float2 w[kUnits][kBatch];
#pragma unroll
          for (int k = 0; k < kUnits; ++k) {
            // (units beyond the last, and pieces beyond theirs, read the last again)
            const int unit = min(i0 + unit0 + k * kThreads, units - 1), slot = unit / kCols, col = 4 * (unit % kCols);
            if (k > 0 && i0 + k * kThreads >= units) break;
#pragma unroll
            for (int b = 0; b < kBatch; ++b) {
              const int at = min(p0 + b * groups, it.n_pieces - 1) * (int)(a.hkv * kRec * 4);
              y[k][b] = get4_past_l2(all, at + (slot * D + col) * 4);
              w[k][b] = get2_past_l2(all, at + (kSlots * D + 2 * slot) * 4);
            }
          }
#pragma unroll
          for (int k = 0; k < kUnits; ++k) {
            if (k > 0 && i0 + k * kThreads >= units) break;
            float m = M[k];
#pragma unroll
            for (int b = 0; b < kBatch; ++b) m = fmaxf(m, w[k][b].x);
            const float f0 = fast_exp2(M[k] - m);
            M[k] = m;
            L[k] *= f0;
            x[k] *= f0;
#pragma unroll
            for (int b = 0; b < kBatch; ++b) {
              const float f = p0 + b * groups < it.n_pieces ? fast_exp2(w[k][b].x - m) : 0.0f;
              L[k] += f * w[k][b].y;
              x[k] += f * y[k][b];
            }
          }
        }
        if (groups > 1) {
          *(f32x4*)(ob + (group * units + unit0) * 8) = x[0];
          *(float2*)(ob + (group * units + unit0) * 8 + 4) = make_float2(M[0], L[0]);
        }
      }
      if (groups > 1) {
        __syncthreads();
        if (group == 0) {
          for (int k = 1; k < groups; ++k) {
            const float2 w = *(const float2*)(ob + (k * units + unit0) * 8 + 4);
            const f32x4 y = *(const f32x4*)(ob + (k * units + unit0) * 8);
            const float m = fmaxf(M[0], w.x), f0 = fast_exp2(M[0] - m), f = fast_exp2(w.x - m);
            M[0] = m;
            L[0] = L[0] * f0 + f * w.y;
            x[0] = x[0] * f0 + f * y;
          }
        }
      }
#pragma unroll
      for (int k = 0; k < kUnits; ++k) {
        const int unit = i0 + unit0 + k * kThreads, slot = unit / kCols, col = 4 * (unit % kCols);
        if (group == 0 && unit < units) {
          odd |= (L[k] == L[k]) & !finite4(x[k]);
          put(slot, col, x[k], L[k]);
        }
      }
    }
    if (__any(odd)) {  // (the weight of a piece that has such a sum may be 0)
      __builtin_amdgcn_s_waitcnt(0);
#pragma unroll 1
      for (int unit = unit0; group == 0 && unit < units; unit += kThreads) {
        const int slot = unit / kCols, col = 4 * (unit % kCols);
        uint32_t up = 0, down = 0;
        bool nan_row = false;
#pragma unroll 1
        for (int p = 0; p < it.n_pieces; ++p) {
          const int at = p * (int)(a.hkv * kRec * 4);
          const f32x4 y = get4_past_l2(all, at + (slot * D + col) * 4);
          const float l_piece = get2_past_l2(all, at + (kSlots * D + 2 * slot) * 4).y;
          nan_row |= l_piece != l_piece;
#pragma unroll
          for (int e = 0; e < 4; ++e) note_odd(y[e], true, 1u << e, up, down);
        }
        if (!nan_row) put_odd(slot, col, up, down);
      }
    }
    __syncthreads();
    if (tid == 0) *counter = 0;  // for the next call with this plan
  }
}

template <typename T, int D>
int32_t launch(const PagedArgs& a, int32_t target, hipStream_t stream) {
  hipLaunchKernelGGL((paged_attn_kernel<T, D>), dim3((unsigned)(target * a.hkv)), dim3(kThreads), 0, stream, a);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return cev_fail(CEV_ERR_HIP, "paged attention launch: %s", hipGetErrorString(e));
  return CEV_OK;
}

}  // namespace

extern "C" int32_t cev_paged_attention(const cev_paged_desc* d, const void* q, const void* k_cache, const void* v_cache,
                                       const int32_t* block_table, void* out, void* work, size_t work_bytes, cev_stream stream) {
  PagedBounds b;
  const int32_t rc = cev_paged_bounds(d, &b);
  if (rc) return rc;
  CEV_CHECK_ARG(q && k_cache && v_cache && block_table && out && work, "cev_paged_attention: null argument");
  CEV_CHECK_ARG((((uintptr_t)q | (uintptr_t)k_cache | (uintptr_t)v_cache | (uintptr_t)out | (uintptr_t)work) & 15) == 0 &&
                    ((uintptr_t)block_table & 3) == 0,
                "cev_paged_attention: device buffers must be 16-byte aligned");
  if (work_bytes < b.bytes) return cev_fail(CEV_ERR_SPACE, "cev_paged_attention: work buffer of %zu bytes, %zu needed", work_bytes, b.bytes);
  PagedArgs a;
  a.q = q;
  a.kc = k_cache;
  a.vc = v_cache;
  a.bt = block_table;
  a.out = out;
  a.work = (char*)work;
  a.q_st = d->q_stride_t;
  a.q_sh = d->q_stride_h;
  a.kc_sp = d->kc_stride_p;
  a.kc_st = d->kc_stride_t;
  a.kc_sh = d->kc_stride_h;
  a.vc_sp = d->vc_stride_p;
  a.vc_st = d->vc_stride_t;
  a.vc_sh = d->vc_stride_h;
  a.o_st = d->o_stride_t;
  a.o_sh = d->o_stride_h;
  a.bt_stride = d->bt_stride;
  a.hkv = d->n_kv_heads;
  a.g = d->n_q_heads / d->n_kv_heads;
  a.t = d->t;
  a.page_shift = __builtin_ctz((unsigned)d->page_size);
  a.n_pages = d->n_pages;
  a.max_pages = d->max_pages;
  a.window = d->window;
  a.sinks = d->sinks;
  a.scale_log2 = d->scale * 1.4426950408889634f;
  a.sig = b.sig;
  auto list = [&](int i) {
    a.first_off = b.list[i].first_off;
    a.items_off = b.list[i].items_off;
    a.counters_off = b.list[i].counters_off;
    a.records_off = b.list[i].records_off;
    return b.list[i].target;
  };
  const hipStream_t s = (hipStream_t)stream;
  if (const int32_t target = list(kPagedMany)) {
    const int32_t rc = cev_paged_tile_launch(a, d->head_dim, target, s);
    if (rc) return rc;
  }
  const int32_t target = list(kPagedFew);
  if (d->dtype == CEV_F32) return launch<float, 128>(a, target, s);
  return d->head_dim == 128 ? launch<__bf16, 128>(a, target, s) : launch<__bf16, 256>(a, target, s);
}
