// Products of many rows in e4m3 (see fp8_linear.hip for the mathematics).
//
// A workgroup's 4 waves compute 16 TT rows x 256 weight rows, each wave 64 of
// them, by v_mfma_scale_f32_16x16x128_f8f6f4: a block of columns an
// instruction, and 8 % more of them under the card's power limit than of the
// 32 x 32 x 64 form (4.35 against 4.03 PFLOP/s with nothing else to do).  Up
// to 128 rows two workgroups a CU: they share no barrier, so one's reads,
// scalings and waits lie under the other's matrix products.  Where there are
// no more workgroups than CUs, two teams of 4 waves stand in for the second one:
// each takes half of the column blocks, in LDS of its own, and their sums meet
// there at the end (1021 x 4096 x 12288, 256 workgroups: 52.3 us against 56.1,
// with f32 scales 58.1 against 68.4).  Column blocks:
//   rows     into LDS straight from memory (buffer_load ... lds), four blocks
//            deep, the 16-byte pieces c of row r at place c ^ (r / 2 + 2 & 7):
//            the lanes that LDS serves together (0-3, 12-15 and 20-27 of 32,
//            and the others) fall on all 64 banks;
//   weights  from the packed layout into registers, two blocks deep: no other
//            wave of the workgroup reads them;
//   scales   the rows' through LDS, four blocks at a time; the weights' in
//            registers, four blocks of bytes or one of f32.
// The tiles of the workgroups that run on one XCD together are neighbours,
// kPanel tiles of rows by as many as there are of weight rows, so its L2
// serves most reads.
#include "fp8.h"

namespace {

constexpr int kStages = 4;
constexpr int kPanel = 8;  // row tiles of a panel

constexpr int kBufferWord3 = 0x00020000;  // raw buffer, no format

__device__ __forceinline__ int uniform(int x) { return __builtin_amdgcn_readfirstlane(x); }

// A buffer of `bytes` from p on (counted to 2 GB; a 64-bit comparison would
// take it out of the scalar registers).
__device__ __forceinline__ __amdgpu_buffer_rsrc_t buffer(const void* p, int64_t bytes) {
  return __builtin_amdgcn_make_buffer_rsrc((void*)p, (short)0, (uint32_t)(bytes >> 31) ? INT32_MAX : (int)bytes, kBufferWord3);
}

// LDS reads through asm: the compiler would wait for every load in flight
// before each, as it cannot tell the buffers in LDS apart.
template <int OFF>
__device__ __forceinline__ u32x4_t read_b128(int vaddr) {
  static_assert(OFF >= 0 && OFF < 65536, "ds offset field");
  u32x4_t r;
  asm volatile("ds_read_b128 %0, %1 offset:%2" : "=v"(r) : "v"(vaddr), "i"(OFF) : "memory");
  return r;
}
template <int OFF>
__device__ __forceinline__ int read_u8(int vaddr) {
  static_assert(OFF >= 0 && OFF < 65536, "ds offset field");
  int r;
  asm volatile("ds_read_u8 %0, %1 offset:%2" : "=v"(r) : "v"(vaddr), "i"(OFF) : "memory");
  return r;
}

// A row tile's operand of one block: 16 rows, and their scales.
struct Unit {
  u32x4_t v[2];
  int s;
};
// All but the N last LDS reads have come, this one among them.
template <int N>
__device__ __forceinline__ void wait_unit(Unit& u) {
  asm volatile("s_waitcnt lgkmcnt(%3)" : "+v"(u.v[0]), "+v"(u.v[1]), "+v"(u.s) : "i"(N));
}

template <bool E8M0, bool GATE_UP, bool EXACT, int TT, int TEAMS>
__device__ __forceinline__ void tile(const Fp8Args& a, int row_tiles, int col_tiles) {
  constexpr int ROWS = 16 * TT;
    constexpr int STAGE = ROWS * kFp8Block;
  constexpr int XQ = TT / 2;  // 1 KB pieces of a block's rows that a wave fetches
  constexpr int PITCH = 144;  // of the rows that the results pass through LDS in: 128 bytes, moved on by four banks each
  constexpr int OUT = GATE_UP ? ROWS * (PITCH + 16) : 4 * ROWS * PITCH;
  constexpr int SCALES = kStages * STAGE;  // of the rows, four blocks each: of three groups of four blocks
  constexpr int LDS = SCALES + 3 * ROWS * 4 > OUT ? SCALES + 3 * ROWS * 4 : OUT;
  __shared__ __align__(1024) char all_lds[TEAMS * LDS];
  const int team = TEAMS > 1 ? uniform(threadIdx.x >> 8) : 0, tid = threadIdx.x & 255;
  const int wave = uniform(tid >> 6), lane = tid & 63, quad = lane >> 4, l16 = lane & 15;
  char* const lds = all_lds + team * LDS;

  // which tile: XCD b % 8 gets a run of tiles, in panels of kPanel row tiles
  int64_t row0;
  int col_tile, part;
  {
    const int tiles = row_tiles * col_tiles, per = gridDim.x / 8, more = gridDim.x % 8, x = blockIdx.x % 8;
    const int at = x * per + min(x, more) + blockIdx.x / 8;
    part = at / tiles;
    const int l = at - part * tiles, panel = l / (kPanel * col_tiles), r = l - panel * kPanel * col_tiles;
    const int high = min(kPanel, row_tiles - panel * kPanel);  // row tiles of this panel
    col_tile = r / high;
    row0 = (int64_t)(panel * kPanel + r - col_tile * high) * ROWS;
  }
  // the team's column blocks, whole groups of four in the first team
  const int part0 = part * a.blocks_part, part1 = min(a.kb, part0 + a.blocks_part);
  const int share = TEAMS > 1 ? (part1 - part0 + 7) / 8 * 4 : part1 - part0;
  const int kb0 = part0 + team * share, kb1 = min(part1, kb0 + share);
  const int pitch = a.kb * kFp8Block;  // bytes of a row
  const int group0 = col_tile * 8 + wave * 2;
  const int rows_left = (int)min<int64_t>(ROWS, a.t - row0);

  // rows, 8 an instruction
  const __amdgpu_buffer_rsrc_t rx = buffer((const uint8_t*)a.x + row0 * pitch, (a.t - row0) * pitch);
  int xat[XQ];
#pragma unroll
  for (int q = 0; q < XQ; ++q)
    xat[q] = min((wave * XQ + q) * 8 + (lane >> 3), rows_left - 1) * pitch + (((lane & 7) ^ (((wave * XQ + q) * 4 + quad + 2) & 7)) << 4);
  auto fetch_x = [&](int q, int kb, int stage) {
    const int at = min(kb, part1 - 1) * kFp8Block;
    __builtin_amdgcn_raw_ptr_buffer_load_lds(rx, (__attribute__((address_space(3))) void*)(lds + stage + (wave * XQ + q) * 1024), 16, xat[q], at, 0, 0);
  };

  // weights: lane l takes row l % 16 of each half of a group of 32, columns 32 (l / 16) .. + 31
  const int group_bytes = a.kb * kFp8GroupBytes;
  const __amdgpu_buffer_rsrc_t rw = buffer(a.w + (int64_t)group0 * group_bytes, (int64_t)2 * group_bytes);
  const int wat = (quad >> 1) * 2048 + (quad & 1) * 512 + l16 * 16;
  u32x4_t w[2][4][2];
  uint32_t sw[2][2];  // f32 scales
  uint32_t sw4[2], sw4_next[2];  // e8m0, of four blocks
  const __amdgpu_buffer_rsrc_t rws =
      buffer(a.ws + (int64_t)group0 * a.ws_pitch * (E8M0 ? 1 : 4), (int64_t)2 * a.ws_pitch * (E8M0 ? 1 : 4));
  int nil = 0;  // (scalar loads of the scales would be waited for with the LDS reads)
  asm volatile("" : "+v"(nil));
  auto fetch_w = [&](auto b_c, auto p_c, int kb) {  // an eighth of them
    constexpr int B = decltype(b_c)::value, P = decltype(p_c)::value, J = P / 2, H = P % 2;
    const int at = min(kb, part1 - 1);
    w[B][J][H] = __builtin_bit_cast(u32x4_t, __builtin_amdgcn_raw_buffer_load_b128(
                                                 rw, wat, at * kFp8GroupBytes + (J >> 1) * group_bytes + (J & 1) * 256 + H * 1024, 0));
    if constexpr (!E8M0 && P < 2) sw[B][P] = (uint32_t)__builtin_amdgcn_raw_buffer_load_b32(rws, nil, (P * a.ws_pitch + at) * 4, 0);
  };
  auto fetch_sw4 = [&](uint32_t* s, int kb) {
#pragma unroll
    for (int j = 0; j < 2; ++j) s[j] = (uint32_t)__builtin_amdgcn_raw_buffer_load_b32(rws, nil, j * a.ws_pitch + min(kb, a.ws_pitch - 4), 0);
  };

  // The rows' scales: thread r brings row r's of four blocks at a time.  (The
  // last row's last blocks: the four bytes before the end, moved down; a later
  // tile's buffer starts four bytes early for that.)  0 behind the last block.
  const int early = row0 > 0 ? 4 : 0;
  const int64_t s_bytes = (a.t - row0) * a.kb + early;
  const __amdgpu_buffer_rsrc_t rs = buffer(a.xs + row0 * a.kb - early, s_bytes);
  const int s_last = ((uint32_t)(s_bytes >> 31) ? INT32_MAX : (int)s_bytes) - 4;
  const int sat = min(tid, rows_left - 1) * a.kb + early;
  auto fetch_xs = [&](int kb) {
    const int from = sat + min(kb, part1 - 1), at = min(from, s_last), n = kb1 - kb;
    const uint32_t v = (uint32_t)__builtin_amdgcn_raw_buffer_load_b32(rs, at, 0, 0) >> (8 * (from - at) & 31);
    return v & (n >= 4 ? 0xffffffffu : n <= 0 ? 0u : (1u << 8 * n) - 1);
  };
  auto put_xs = [&](uint32_t v, int slot) {
    // (tid from the lane again: kept over the loop, it went to memory, and its reload waited for all loads in flight)
    int from = 0;
    asm volatile("" : "+s"(from));
    const int t = wave * 64 + (int)__builtin_amdgcn_mbcnt_hi(~0u, __builtin_amdgcn_mbcnt_lo(~0u, (uint32_t)from));
    if (ROWS == 256 || t < ROWS) *(uint32_t*)(lds + SCALES + (slot * ROWS + t) * 4) = v;
  };

  // Reads of the rows, AHEAD tiles of 16 ahead of the one that is computed.
  constexpr int AHEAD = TT > 8 ? 2 : 1, RING = 2 * AHEAD;
  static_assert(TT % RING == 0 && AHEAD <= TT / 2, "a tile's registers are the same ones in every block");
  const int base = (int)(uint32_t)(uintptr_t)(__attribute__((address_space(3))) char*)lds;
  int rat[2];
#pragma unroll
  for (int h = 0; h < 2; ++h) rat[h] = base + l16 * kFp8Block + (((quad * 2 + h) ^ ((lane >> 1) + 2 & 7)) << 4);
  const int rs_at = base + SCALES + l16 * 4;
  Unit xr[RING];
  auto read_part = [&](auto u_c, auto p_c, int stage, int scale) {  // the two halves of the operand, and the scale
    constexpr int U = decltype(u_c)::value, P = decltype(p_c)::value;
    if constexpr (P < 2)
      xr[U % RING].v[P] = read_b128<U * 16 * kFp8Block>(rat[P] + stage);
    else
      xr[U % RING].s = read_u8<U * 64>(rs_at + scale);
  };
  auto read_unit = [&](auto u_c, int stage, int scale) { static_for<3>([&](auto p_c) { read_part(u_c, p_c, stage, scale); }); };

  f32x4 acc[TT][4];
#pragma unroll
  for (int i = 0; i < TT; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) acc[i][j] = f32x4{};

  constexpr std::integral_constant<int, 0> even{};
  constexpr std::integral_constant<int, 1> odd{};
  int stage = 0;  // LDS of block kb; the next blocks' follow
  auto after = [&](int st, int n) { return (st + n * STAGE) & (kStages * STAGE - 1); };
  static_assert((kStages * STAGE & (kStages * STAGE - 1)) == 0, "stages wrap by a mask");
#pragma unroll
  for (int i = 0; i < kStages - 1; ++i)
#pragma unroll
    for (int q = 0; q < XQ; ++q) fetch_x(q, kb0 + i, i * STAGE);
  static_for<8>([&](auto p_c) { fetch_w(even, p_c, kb0); });
  if constexpr (E8M0) fetch_sw4(sw4, kb0);
  put_xs(fetch_xs(kb0), 0);
  uint32_t xs_next = fetch_xs(kb0 + 4);
  asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
  static_for<AHEAD>([&](auto u_c) { read_unit(u_c, 0, 0); });
  static_for<AHEAD>([&](auto u_c) { wait_unit<0>(xr[decltype(u_c)::value]); });

  // Block kb, whose scales are at `scale` (the next block's at scale_next).
  // Its weights are in the registers of b_c; those of block kb + 1 go to the others.
  auto block = [&](auto b_c, int kb, int b4, int scale, int scale_next) {
    constexpr int B = decltype(b_c)::value;
    uint32_t s2[2] = {};
    if constexpr (E8M0)
#pragma unroll
      for (int j = 0; j < 2; ++j) s2[j] = sw4[j] >> (8 * b4);
    Fp8Scale s[2];
    if constexpr (!E8M0 || EXACT)
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        s[j] = fp8_scale<E8M0>(E8M0 ? s2[j] & 255 : (uint32_t)uniform((int)sw[B][j]));
        // (in scalar registers: two vector ones more and the loop reloads one, behind all loads in flight)
        if constexpr (!E8M0 && !EXACT) s[j].rest = __uint_as_float((uint32_t)uniform((int)__float_as_uint(s[j].rest)));
      }
    f32x4 p[2];
    auto scale_in = [&](auto u_c, auto j_c) {
      constexpr int U = decltype(u_c)::value, J = decltype(j_c)::value;
#pragma unroll
      for (int r = 0; r < 4; ++r) acc[U][J][r] = __builtin_fmaf(p[J % 2][r], s[J >> 1].rest, acc[U][J][r]);
    };
    static_for<TT>([&](auto u_c) {
      constexpr int U = decltype(u_c)::value;
      if constexpr (U == TT / 2) {
        // Block kb + 1 is in LDS when every wave has seen its part arrive, and
        // block kb - 1 has been read by all: its place is for block kb + 3.
        // Fetched after the part of block kb + 1: at least that of block kb + 2
        // and the weights of block kb + 1.
        asm volatile("s_waitcnt vmcnt(%0)\n\ts_barrier" ::"i"(XQ + 8) : "memory");
      }
      // Read since: the tiles up to U + AHEAD - 1; for the last one the next block's first tiles, one read alternating with its own where AHEAD is 1.
      wait_unit<(U < AHEAD ? 15 : U == TT - 1 ? (AHEAD == 1 ? 1 : 3 * AHEAD) : 3 * AHEAD - 3)>(xr[U % RING]);
      const i32x8 x = fp8_join(xr[U % RING].v[0], xr[U % RING].v[1]);
      const int sx = xr[U % RING].s;
      bf16x8 wide[4];
      float by[2] = {};
      if constexpr (EXACT) {
        const Fp8RowScale row = fp8_row_scale(sx);
#pragma unroll
        for (int c = 0; c < 4; ++c) wide[c] = fp8_widen(x[2 * c], x[2 * c + 1], row.values);
#pragma unroll
        for (int j = 0; j < 2; ++j) by[j] = fp8_factor(row, s[j]);
      }
      // Four matrix products, and between them what is read for later ones: a
      // product takes 32 cycles, in which seven other instructions can start.
      static_for<4>([&](auto j_c) {
        constexpr int J = decltype(j_c)::value;
        const i32x8 wv = fp8_join(w[B][J][0], w[B][J][1]);
        if constexpr (EXACT) {
          f32x4 q = {};
#pragma unroll
          for (int c = 0; c < 4; ++c) q = __builtin_amdgcn_mfma_f32_16x16x32_bf16(fp8_widen(wv[2 * c], wv[2 * c + 1]), wide[c], q, 0, 0, 0);
#pragma unroll
          for (int r = 0; r < 4; ++r) acc[U][J][r] = __builtin_fmaf(q[r], by[J >> 1], acc[U][J][r]);
        } else if constexpr (E8M0) {
          acc[U][J] = fp8_mfma(wv, x, acc[U][J], (int)s2[J >> 1], sx);
        } else {
          // (ahead of the other wave's scalings, which fill its time: gate and up of
          // 2048 x 12288 x 4096 192.1 us without, 188.4 with; e8m0 and f32 outputs the same)
          __builtin_amdgcn_s_setprio(1);
          p[J % 2] = fp8_mfma(wv, x, f32x4{}, s[J >> 1].code, sx);
          __builtin_amdgcn_s_setprio(0);
        }
        __builtin_amdgcn_sched_barrier(0);
        if constexpr (J < 3) {
          // (the next block's first tiles come a tile early: they are waited for at this block's end)
          if constexpr (U + AHEAD < TT) read_part(std::integral_constant<int, U + AHEAD>{}, j_c, stage, scale);
          if constexpr (U == TT - 2) static_for<AHEAD>([&](auto n_c) { read_part(n_c, j_c, after(stage, 1), scale_next); });
        } else {
          // (a load or two a tile: more in a row wait for the address unit, and the products behind them with it)
          if constexpr (U >= TT / 2) fetch_x(U - TT / 2, kb + kStages - 1, after(stage, kStages - 1));
          if constexpr (U < TT / 2)
            static_for<16 / TT>([&](auto n_c) { fetch_w(std::integral_constant<int, 1 - B>{}, std::integral_constant<int, U * (16 / TT) + decltype(n_c)::value>{}, kb + 1); });
        }
        // (f32 scales: of the product before, so that none is waited for)
        if constexpr (!E8M0 && !EXACT && (U > 0 || J > 0)) scale_in(std::integral_constant<int, (4 * U + J - 1) / 4>{}, std::integral_constant<int, (J + 3) % 4>{});
        __builtin_amdgcn_sched_barrier(0);
      });
    });
    if constexpr (!E8M0 && !EXACT) scale_in(std::integral_constant<int, TT - 1>{}, std::integral_constant<int, 3>{});
    stage = after(stage, 1);
    // (a register that a read is still to fill is carried into no other iteration: it might be moved on the way)
    static_for<AHEAD>([&](auto u_c) { wait_unit<0>(xr[decltype(u_c)::value]); });
  };
  // (no branch within the inner loop: the compiler would take the matrix
  // products behind it)
  int slot = 0;  // of this group of four blocks' scales
  for (int kb4 = kb0; kb4 < kb1; kb4 += 4) {
    const int slot_next = slot == 2 ? 0 : slot + 1;
    put_xs(xs_next, slot_next);  // (read from the next block on, two barriers from here; the slot's last readers were two groups back)
    xs_next = fetch_xs(kb4 + 8);
    if constexpr (E8M0) {
      fetch_sw4(sw4_next, kb4 + 4);
      if (kb1 - kb4 < 4) sw4[0] &= 0x00ffffffu >> (8 * (3 - (kb1 - kb4))), sw4[1] &= 0x00ffffffu >> (8 * (3 - (kb1 - kb4)));
    }
    // an odd number of blocks: behind the last one it comes once more, under scales of 2^-254 or 0
    const int end = min(kb4 + 4, kb1), at = slot * ROWS * 4, at_next = slot_next * ROWS * 4;
    for (int kb = kb4; kb < end; kb += 2) {
      const int b4 = kb - kb4;
      block(even, kb, b4, at + b4, at + b4 + 1);
      if constexpr (!E8M0)
#pragma unroll
        for (int j = 0; j < 2; ++j) sw[1][j] = kb + 1 < kb1 ? sw[1][j] : 0;
      block(odd, kb + 1, b4 + 1, at + b4 + 1, b4 == 2 ? at_next : at + b4 + 2);
    }
    if constexpr (E8M0) sw4[0] = sw4_next[0], sw4[1] = sw4_next[1];
    slot = slot_next;
  }
  if constexpr (TEAMS > 1)  // a barrier a block, also for blocks that the second team has not got
    for (int kb = 2 * ((max(kb1 - kb0, 0) + 1) / 2); kb < 2 * ((share + 1) / 2); ++kb) asm volatile("s_barrier" ::: "memory");
  asm volatile("s_waitcnt vmcnt(0)\n\ts_barrier" ::: "memory");
  if constexpr (TEAMS > 1) {  // the teams' sums
    f32x4* const sums = (f32x4*)all_lds + tid;
    if (team == 1) {
#pragma unroll
      for (int i = 0; i < TT; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) sums[(i * 4 + j) * 256] = acc[i][j];
    }
    __syncthreads();
    if (team == 1) return;  // (later barriers do not wait for waves that have ended)
#pragma unroll
    for (int i = 0; i < TT; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) acc[i][j] += sums[(i * 4 + j) * 256];
    __syncthreads();
  }

  // Results.  Lane l holds row l % 16 of each row tile, columns 16 j + 4 (l /
  // 16) .. + 3 of the wave's 64.
  if constexpr (!GATE_UP) {
    if (a.part) {
      const int64_t width = (int64_t)a.groups * kFp8Group;
#pragma unroll
      for (int i = 0; i < TT; ++i) {
        const int64_t row = row0 + i * 16 + l16;
        if (row >= a.t) continue;
        float* const p = a.part + ((int64_t)part * a.t + row) * width + (int64_t)group0 * kFp8Group + 4 * quad;
#pragma unroll
        for (int j = 0; j < 4; ++j) *(f32x4*)(p + 16 * j) = acc[i][j];
      }
      return;
    }
    if constexpr (EXACT) {
#pragma unroll
      for (int i = 0; i < TT; ++i) {
        const int64_t row = row0 + i * 16 + l16;
        if (row >= a.t) continue;
#pragma unroll
        for (int j = 0; j < 4; ++j) fp8_store4((float*)a.out + row * a.out_st, a.n, (int64_t)group0 * kFp8Group + 16 * j + 4 * quad, acc[i][j]);
      }
      return;
    }
    // through LDS, the wave's rows of 64 columns side by side
    char* const mine = lds + wave * ROWS * PITCH;
#pragma unroll
    for (int i = 0; i < TT; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const f32x4& v = acc[i][j];
        *(u32x2_t*)(mine + (i * 16 + l16) * PITCH + j * 32 + quad * 8) =
            u32x2_t{(uint32_t)bf16_bits(v[0]) | (uint32_t)bf16_bits(v[1]) << 16, (uint32_t)bf16_bits(v[2]) | (uint32_t)bf16_bits(v[3]) << 16};
      }
    wave_lds_sync();
    const int64_t col = (int64_t)group0 * kFp8Group + (lane & 7) * 8;
    const bool wide = a.n % 8 == 0 && a.out_st % 8 == 0 && ((uintptr_t)a.out & 15) == 0;
#pragma unroll
    for (int i = 0; i < 2 * TT; ++i) {
      const int r = i * 8 + (lane >> 3);
      const int64_t row = row0 + r;
      const u32x4_t v = *(const u32x4_t*)(mine + r * PITCH + (lane & 7) * 16);
      uint16_t* const o = (uint16_t*)a.out + row * a.out_st + col;
      if (row < a.t) {
        if (wide) {
          if (col < a.n) *(u32x4_t*)o = v;
        } else {
#pragma unroll
          for (int e = 0; e < 8; ++e)
            if (col + e < a.n) o[e] = (uint16_t)(v[e >> 1] >> (16 * (e & 1)));
        }
      }
    }
  } else {
    // group 0 is gate's 32 columns, group 1 up's: the tile's 128 columns are one block of the rows
    float* const tops = (float*)(lds + ROWS * PITCH);  // (ROWS, 4)
    const int col0 = col_tile * 128 + wave * 32 + 4 * quad;
#pragma unroll
    for (int i = 0; i < TT; ++i) {
      uint32_t top = 0;
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const float v = fp8_swiglu(acc[i][j][r], acc[i][2 + j][r]);
          acc[i][j][r] = col0 + 16 * j + r < a.n ? v : 0.0f;
          top = max(top, fp8_size(acc[i][j][r]));
        }
      top = max(top, (uint32_t)__shfl_xor((int)top, 16, 64));
      top = max(top, (uint32_t)__shfl_xor((int)top, 32, 64));
      if (quad == 0) tops[(i * 16 + l16) * 4 + wave] = __uint_as_float(top);
    }
    __syncthreads();
    const int64_t blocks = (a.n + 127) / 128;
#pragma unroll
    for (int i = 0; i < TT; ++i) {
      const int r = i * 16 + l16;
      const u32x4_t o = *(const u32x4_t*)(tops + r * 4);
      const uint32_t code = fp8_code(max(max(o[0], o[1]), max(o[2], o[3])));
      const float f = fp8_inverse(code);
      if (wave == 0 && quad == 0 && row0 + r < a.t) a.out_s[(row0 + r) * blocks + col_tile] = (uint8_t)code;
#pragma unroll
      for (int j = 0; j < 2; ++j)
        *(uint32_t*)(lds + r * PITCH + wave * 32 + 16 * j + 4 * quad) = fp8_pack4(acc[i][j][0] * f, acc[i][j][1] * f, acc[i][j][2] * f, acc[i][j][3] * f);
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < TT / 2; ++i) {
      const int r = i * 32 + (tid >> 3);
      const u32x4_t v = *(const u32x4_t*)(lds + r * PITCH + (tid & 7) * 16);
      if (row0 + r < a.t) *(u32x4_t*)((uint8_t*)a.out + ((row0 + r) * blocks + col_tile) * 128 + (tid & 7) * 16) = v;
    }
  }
}

template <bool E8M0, bool GATE_UP, bool EXACT, int TT, int TEAMS>
__global__ __launch_bounds__(256 * TEAMS, TT > 8 ? 1 : 2) void fp8_tile_kernel(Fp8Args a, int row_tiles, int col_tiles) {
  tile<E8M0, GATE_UP, EXACT, TT, TEAMS>(a, row_tiles, col_tiles);
}

template <bool E8M0, bool GATE_UP, bool EXACT, int TT, int TEAMS>
int32_t launch(const Fp8Args& a, hipStream_t s) {
  const int64_t row_tiles = (a.t + 16 * TT - 1) / (16 * TT), col_tiles = a.groups / kFp8TileGroups, grid = row_tiles * col_tiles * a.parts;
  hipLaunchKernelGGL((fp8_tile_kernel<E8M0, GATE_UP, EXACT, TT, TEAMS>), dim3((unsigned)grid), dim3(256 * TEAMS), 0, s, a, (int)row_tiles, (int)col_tiles);
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? CEV_OK : cev_fail(CEV_ERR_HIP, "cev_fp8_product launch: %s", hipGetErrorString(e));
}

template <bool E8M0, bool EXACT, int TT, int TEAMS>
int32_t launch(const Fp8Args& a, bool gate_up, hipStream_t s) {
  if constexpr (!EXACT)
    if (gate_up) return launch<E8M0, true, false, TT, TEAMS>(a, s);
  return launch<E8M0, false, EXACT, TT, TEAMS>(a, s);
}

template <bool EXACT, int TEAMS>
int32_t launch4(const Fp8Args& a, bool e8m0, bool gate_up, hipStream_t s) {
  return e8m0 ? launch<true, EXACT, 4, TEAMS>(a, gate_up, s) : launch<false, EXACT, 4, TEAMS>(a, gate_up, s);
}

}  // namespace

int32_t fp8_launch_tile(const Fp8Args& a, int tt, int teams, bool exact, bool e8m0, bool gate_up, hipStream_t s) {
  if (a.part) gate_up = false;  // (sums of parts are joined elsewhere)
  if (exact) return teams > 1 ? launch4<true, 2>(a, e8m0, false, s) : launch4<true, 1>(a, e8m0, false, s);
  if (tt == 4) return teams > 1 ? launch4<false, 2>(a, e8m0, gate_up, s) : launch4<false, 1>(a, e8m0, gate_up, s);
  if (tt == 16) return launch<true, false, 16, 1>(a, gate_up, s);
  if (e8m0) return launch<true, false, 8, 1>(a, gate_up, s);
  return teams > 1 ? launch<false, false, 8, 2>(a, gate_up, s) : launch<false, false, 8, 1>(a, gate_up, s);
}
