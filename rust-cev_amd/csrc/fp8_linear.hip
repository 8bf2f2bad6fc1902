// Products of rows and weights in e4m3 (see fp8_device.h for the scales):
//
//   y[t, n] = sum over blocks b of 128 columns:  2^e[t, b] s[n / 128, b] (q[t, b] . w[n, b])
//
// Two kinds of matrix product:
//
//   bf16 outputs, and gate and up of many rows
//       v_mfma_scale_f32_16x16x128_f8f6f4, which takes 2^e as an operand, and s
//       where it is a power of two (of an f32 s its power of two; the rest of it,
//       1 to 2, multiplies the block's 16 x 16 results).  It adds eight
//       neighbouring columns' products after cutting each towards zero to a
//       multiple of 2^(E - 13), 2^E the largest one's power of two (measured bit
//       by bit); what follows is f32.  A sum is therefore up to 7 * 2^-13 of its
//       largest products off; on normal data it is 4.5e-5 of the result, a
//       fortieth of bf16's rounding.  Of gate and up's e4m3 values, whose steps
//       are 2^-3 to 2^-4 apart, one in a thousand becomes the nearest but one:
//       which ones depends on the form, and with it on how many rows a call has.
//       (By f32 sums 8192 x 4096 x 12288 takes 745 us instead of 278.)
//   f32 outputs, and gate and up of few rows
//       v_mfma_f32_16x16x32_bf16 on the same values in bf16, which holds them
//       exactly: products and sums in f32, at half the rate.  Where the weight's
//       bytes are what counts that is nearly free (gate and up of 16 x 6144 x
//       2048: 9.2 us against 8.8).
#include <algorithm>
#include <cmath>

#include "fp8.h"

namespace {

constexpr int kWaves = 8;  // waves of a workgroup of the kernel for few rows, each with its share of the column blocks

// Where 16 bytes of a staged block of 16 rows x 128 columns stand: rows of 128
// bytes, their pieces in an order of their own, so that neither a store nor an
// operand's read meets a bank twice.
__device__ __forceinline__ int staged(int r, int piece) { return r * 128 + ((piece ^ ((r >> 1) + 2)) & 7) * 16; }

// 16 MT rows times 16 weight rows (GATE_UP: times 16 of gate and of up; MT = 4:
// times 32, so that the rows are read half as often).  The
// weight streams through once, so what counts is how much of it is on the way:
// a workgroup holds few weight rows and its waves share the column blocks, each
// with DEEP of them under way; their sums are joined in LDS, in the waves'
// order.  (Parts of the columns in other workgroups would cost a second launch.)
// An operand's lanes hold 16 rows, and a load by that pattern costs the L1 16
// lines; so a wave loads its rows in memory's order and turns them in LDS (16
// rows x 12288 x 4096 12.3 us before, 10.0 after, 5.1 TB/s; 64 x 4096 x 4096 14.2
// and 8.1).  Rows in the model's type go into e4m3 on the way.  Eight waves, as
// with sixteen a CU holds one workgroup and waits for its slowest wave (14.1 us
// instead of 12.3).
template <typename T, typename O, bool E8M0, bool GATE_UP, int MT>
__global__ __launch_bounds__(kWaves * 64, 4) void fp8_small_kernel(Fp8Args a, unsigned col_tiles) {
  constexpr bool PACK = sizeof(T) > 1;
  constexpr bool WIDE = MT == 4;  // both halves of a group of 32 weight rows
  constexpr int NH = GATE_UP || WIDE ? 2 : 1, DEEP = WIDE ? 1 : (PACK ? 2 : 4 / MT) / NH;
  constexpr bool EXACT = sizeof(O) == 4;
  constexpr int QUAD = 80;  // floats of a quad's 16 rows x 4 columns, and 16 more: the sums' reads fall on different banks
  constexpr int STAGE = DEEP * MT * 2048, SUMS = NH * MT * 4 * QUAD * 4;
  __shared__ __align__(16) uint8_t space[kWaves][STAGE > SUMS ? STAGE : SUMS];  // a wave's rows, then its sums
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, quad = lane >> 4, l16 = lane & 15;
  // 16 MT rows, 16 columns.  Workgroups b and b + 8 run on one XCD: those of the
  // same columns follow each other there, so that its L2 serves all but the
  // first (192 x 1000 x 2056: 4.9 us, 6.3 with all columns of a row tile first).
  const unsigned row_tile = blockIdx.x / 8, c16 = blockIdx.y * 8 + blockIdx.x % 8;
  if (c16 >= col_tiles) return;
  const int64_t row0 = (int64_t)row_tile * (16 * MT);
  uint8_t* const own = space[wave];
  // what the lane loads: PACK, 8 values of rows 4 j + lane / 16, else 16 bytes of rows 8 j + lane / 8
  constexpr int LOADS = PACK ? 4 : 2 * MT, LANES = PACK ? 16 : 8;
  const uint8_t* xp[LOADS];
#pragma unroll
  for (int j = 0; j < LOADS; ++j) {
    const int64_t row = min(row0 + j * (64 / LANES) + lane / LANES, a.t - 1);
    xp[j] = (const uint8_t*)a.x + (PACK ? row * a.x_st * (int64_t)sizeof(T) : row * a.kb * kFp8Block);
  }
  const uint8_t* const sp = PACK ? nullptr : a.xs + min(row0 + lane / DEEP, a.t - 1) * a.kb;
  // the group of 32 weight rows (gate's; up's follows), and the lane's place in its half
  const int64_t group = WIDE ? c16 : (int64_t)(c16 >> 1) * NH;
  const uint8_t* const wp = a.w + group * a.kb * kFp8GroupBytes + (quad >> 1) * 2048 + (quad & 1) * 512 + (WIDE ? 0 : (c16 & 1) * 256) + l16 * 16;
  f32x4 acc[NH][MT];
#pragma unroll
  for (int h = 0; h < NH; ++h)
#pragma unroll
    for (int i = 0; i < MT; ++i) acc[h][i] = f32x4{};
  const int share = (a.kb + kWaves - 1) / kWaves, end = min(a.kb, (wave + 1) * share);
  for (int kb0 = wave * share; kb0 < end; kb0 += DEEP) {
    u32x4_t w[DEEP][NH][2];
    uint32_t sw[DEEP][NH];
    u32x4_t x[DEEP][LOADS];
    float v[DEEP][LOADS][8];
    int codes = 127;
    if constexpr (!PACK) codes = sp[min(kb0 + lane % DEEP, a.kb - 1)];
#pragma unroll
    for (int d = 0; d < DEEP; ++d) {
      const int kb = kb0 + d;
      if (kb >= end) break;
#pragma unroll
      for (int j = 0; j < LOADS; ++j) {
        if constexpr (PACK) {
          const int col = kb * kFp8Block + l16 * 8;
          load8((const T*)xp[j] + (col < a.k ? col : 0), a.k - col, v[d][j]);
        } else {
          x[d][j] = *(const u32x4_t*)(xp[j] + (int64_t)kb * kFp8Block + lane % LANES * 16);
        }
      }
#pragma unroll
      for (int h = 0; h < NH; ++h) {
        const uint8_t* const p = wp + (WIDE ? (int64_t)kb * kFp8GroupBytes + h * 256 : ((int64_t)h * a.kb + kb) * kFp8GroupBytes);
        w[d][h][0] = *(const u32x4_t*)p;
        w[d][h][1] = *(const u32x4_t*)(p + 1024);
        const int64_t at = (group + (WIDE ? 0 : h)) * a.ws_pitch + kb;
        sw[d][h] = E8M0 ? a.ws[at] : ((const uint32_t*)a.ws)[at];
      }
    }
    int sx[DEEP][MT];
#pragma unroll
    for (int d = 0; d < DEEP; ++d) {
      if (kb0 + d >= end) break;
      uint8_t* const at = own + d * MT * 2048;
      if constexpr (PACK) {
        uint32_t code[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int r = 4 * j + quad;
          *(u32x2_t*)(at + staged(r, l16 >> 1) + (l16 & 1) * 8) = fp8_block16(v[d][j], code[j]);
        }
        // row r's scale is in the lanes 16 (r % 4) .. + 15, as their code[r / 4]
        const uint32_t c = (l16 & 2) ? (l16 & 1) ? code[3] : code[2] : (l16 & 1) ? code[1] : code[0];
        sx[d][0] = __shfl((int)c, (l16 & 3) * 16 + (l16 >> 2), 64);
      } else {
#pragma unroll
        for (int j = 0; j < LOADS; ++j) *(u32x4_t*)(at + (j >> 1) * 2048 + staged((j & 1) * 8 + (lane >> 3), lane & 7)) = x[d][j];
#pragma unroll
        for (int i = 0; i < MT; ++i) sx[d][i] = __shfl(codes, (i * 16 + l16) * DEEP + d, 64);
      }
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");  // (the wave's own stores: LDS takes them in order)
#pragma unroll
    for (int d = 0; d < DEEP; ++d) {
      if (kb0 + d >= end) break;
      i32x8 xv[MT];
#pragma unroll
      for (int i = 0; i < MT; ++i) {
        const uint8_t* const at = own + (d * MT + i) * 2048;
        xv[i] = fp8_join(*(const u32x4_t*)(at + staged(l16, 2 * quad)), *(const u32x4_t*)(at + staged(l16, 2 * quad + 1)));
      }
#pragma unroll
      for (int h = 0; h < NH; ++h) {
        const i32x8 wv = fp8_join(w[d][h][0], w[d][h][1]);
        const Fp8Scale f = fp8_scale<E8M0>(sw[d][h]);
#pragma unroll
        for (int i = 0; i < MT; ++i) {
          if constexpr (EXACT) {
            const Fp8RowScale row = fp8_row_scale(sx[d][i]);
            f32x4 p = {};
#pragma unroll
            for (int c = 0; c < 4; ++c)
              p = __builtin_amdgcn_mfma_f32_16x16x32_bf16(fp8_widen(wv[2 * c], wv[2 * c + 1]), fp8_widen(xv[i][2 * c], xv[i][2 * c + 1], row.values), p, 0, 0, 0);
            const float by = fp8_factor(row, f);
#pragma unroll
            for (int r = 0; r < 4; ++r) acc[h][i][r] = __builtin_fmaf(p[r], by, acc[h][i][r]);
          } else if constexpr (E8M0) {
            acc[h][i] = fp8_mfma(wv, xv[i], acc[h][i], (int)sw[d][h], sx[d][i]);
          } else {
            const f32x4 p = fp8_mfma(wv, xv[i], f32x4{}, f.code, sx[d][i]);
#pragma unroll
            for (int r = 0; r < 4; ++r) acc[h][i][r] = __builtin_fmaf(p[r], f.rest, acc[h][i][r]);
          }
        }
      }
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  }
  // lane l holds row l % 16, columns 4 (l / 16) .. + 3
#pragma unroll
  for (int h = 0; h < NH; ++h)
#pragma unroll
    for (int i = 0; i < MT; ++i) *(f32x4*)((float*)own + (h * MT + i) * 4 * QUAD + quad * QUAD + l16 * 4) = acc[h][i];
  __syncthreads();
  for (int e = threadIdx.x; e < MT * 256; e += kWaves * 64) {
    const int i = e >> 8, r = (e >> 4) & 15, n = e & 15, at = i * 4 * QUAD + (n >> 2) * QUAD + r * 4 + (n & 3);
    float v[NH];
#pragma unroll
    for (int h = 0; h < NH; ++h) {
      v[h] = ((const float*)space[0])[h * MT * 4 * QUAD + at];
#pragma unroll
      for (int w = 1; w < kWaves; ++w) v[h] += ((const float*)space[w])[h * MT * 4 * QUAD + at];
    }
    const int64_t out_row = row0 + i * 16 + r, col = (int64_t)c16 * (WIDE ? 32 : 16) + n;
    if (out_row >= a.t) continue;
    if constexpr (GATE_UP) {
      if (col < a.n) a.part[out_row * a.out_st + col] = fp8_swiglu(v[0], v[1]);
    } else {
#pragma unroll
      for (int h = 0; h < NH; ++h)
        if (col + h * 16 < a.n) ((O*)a.out)[out_row * a.out_st + col + h * 16] = (O)v[h];
    }
  }
}

// The sums of the parts of the columns, into the output's type: four columns a thread.
struct JoinArgs {
  const float* part;
  void* out;
  uint8_t* out_s;
  int64_t t, n, out_st, width;  // width: padded columns of a row of sums
  int32_t parts, quads;         // quads (gate and up: chunks of 8 columns) of a row
};

template <typename O>
__global__ __launch_bounds__(256) void fp8_join_kernel(JoinArgs a) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int64_t row = i / a.quads;
  if (row >= a.t) return;
  const int64_t col = (i - row * a.quads) * 4;
  const float* p = a.part + row * a.width + col;
  f32x4 v = *(const f32x4*)p;
#pragma unroll 4
  for (int s = 1; s < a.parts; ++s) v += *(const f32x4*)(p + (int64_t)s * a.t * a.width);
  fp8_store4((O*)a.out + row * a.out_st, a.n, col, v);
}

// Sums of gate and up (groups of 32 columns in turn) into rows in e4m3: 8
// columns a thread, 16 threads a block.
__global__ __launch_bounds__(256) void fp8_join_gate_up_kernel(JoinArgs a) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int64_t row = i / a.quads;
  if (row >= a.t) return;  // (16 threads of a block leave together)
  const int col = (int)(i - row * a.quads) * 8;
  const float* p = a.part + row * a.width + col / kFp8Group * 2 * kFp8Group + col % kFp8Group;
  f32x4 g[2] = {}, u[2] = {};
#pragma unroll 4
  for (int s = 0; s < a.parts; ++s, p += a.t * a.width)
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      g[j] += *(const f32x4*)(p + 4 * j);
      u[j] += *(const f32x4*)(p + kFp8Group + 4 * j);
    }
  float v[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) v[j] = col + j < a.n ? fp8_swiglu(g[j >> 2][j & 3], u[j >> 2][j & 3]) : 0.0f;
  uint32_t code;
  const u32x2_t q = fp8_block16(v, code);
  *(u32x2_t*)((uint8_t*)a.out + (row * a.quads + col / 8) * 8) = q;
  if ((col & 127) == 0) a.out_s[row * (a.quads >> 4) + (col >> 7)] = (uint8_t)code;
}

int32_t launched(const char* what) {
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? CEV_OK : cev_fail(CEV_ERR_HIP, "%s launch: %s", what, hipGetErrorString(e));
}

constexpr int kTileBlocks = 32768;  // column blocks that the offsets of the kernel for many rows reach

// How a product runs.
struct Form {
  int32_t tt;   // the kernel for many rows, 16 tt of them a workgroup; 0: the one for few
  bool pack_x;  // rows of the model's type go into e4m3 in a launch of their own
  int32_t mt;     // of the kernel for few, 16 mt of them a workgroup
  int32_t teams;  // of the kernel for many rows
  int32_t groups, kb, parts, blocks_part;
  size_t rows_bytes, scales_bytes, part_bytes;
};

size_t up256(size_t n) { return (n + 255) & ~(size_t)255; }

// Times of the kernel for many rows in us, measured at 64 to 4096 rows, 2048
// to 12288 weight rows, 2048 to 12288 columns: a launch, and a block of columns
// (with two teams: two blocks) alone on the card, with a workgroup on every CU,
// and with two.
struct TileTimes {
  float fixed, one, all, two;
};
constexpr TileTimes kE8m0Times[] = {{4.2f, 0.455f, 0.54f, 0.95f}, {5.6f, 0.57f, 0.745f, 1.5f}, {4.0f, 0.9f, 1.36f, 0.0f}};
constexpr TileTimes kF32Times[] = {{4.8f, 0.545f, 0.665f, 1.1f}, {5.8f, 0.87f, 1.02f, 1.85f}};
constexpr TileTimes kExactTimes[] = {{4.7f, 1.3f, 1.33f, 1.9f}};
constexpr TileTimes kE8m0Teams[] = {{6.0f, 0.77f, 0.95f, 0.0f}};
constexpr TileTimes kF32Teams[] = {{5.6f, 0.87f, 1.1f, 0.0f}, {8.0f, 1.3f, 1.8f, 0.0f}};
constexpr TileTimes kExactTeams[] = {{7.7f, 1.7f, 1.92f, 0.0f}};

// Blocks of columns that all workgroups of the kernel for few rows go through,
// where each holds `rows` rows and `columns` weight rows.
double units_of(const cev_fp8_desc& d, int32_t kb, int rows, int columns) {
  return (double)((d.t + rows - 1) / rows) * ((d.n + columns - 1) / columns) * kb;
}

// Which kernel, with which tile, by the time that each would take.  The one for
// few rows streams the weight at the card's rate (16 rows x 12288 x 4096: 10 us
// against 14), and is ahead as long as its repeated reads of the rows cost less
// than the other's slow start (12288 x 4096: 32 rows 10.6 us against 15.4, 64
// rows 14.7 against 17.1, 128 rows 21.2 against 18.7; 4096 x 4096: 128 rows 8.7
// against 15.3).  Of the other's tiles, fewer and larger ones read less and
// compute at a higher rate; more of them, and parts of the columns, fill the
// card.  A part's sums cost a round trip through memory (7 TB/s, most of it in
// the card's cache) and another launch.  Two teams go where a CU has one
// workgroup; with e8m0 scales and 128 rows they gain nothing (1536 x 4096 x 4096:
// 27.6 us against 26.9).
void plan(const cev_fp8_desc& d, Form& f) {
  const bool exact = !d.gate_up && d.out_dtype == CEV_F32, e8m0 = d.scales == CEV_FP8_SCALES_E8M0;
  double best = 1e-3 * units_of(d, f.kb, 32, 16) * (d.gate_up ? 0.57 : exact ? 0.33 : 0.30) + (d.gate_up ? 6.8 : exact ? 3.0 : 2.6);
  if (!exact && !d.gate_up && d.t > 32) {
    // 64 rows and 32 weight rows a workgroup, whose waves take at least 1.3 us
    // for a block (128 rows x 4096 x 4096: 8.7 us against 12.3, 64 rows 8.5 against
    // 7.9, 64 rows x 12288 x 4096 14.7 against 17.6).  In f32 sums the registers
    // do not hold it.
    const double wide = 3.5 + std::max(0.74e-3 * units_of(d, f.kb, 64, 32), 1.3 / kWaves * f.kb);
    if (wide < best) best = wide, f.mt = 4;
  }
  const TileTimes* const times = exact ? kExactTimes : e8m0 ? kE8m0Times : kF32Times;
  // (it reads the rows' scales four at a time, so that there have to be four;
  // up to 16 rows it is never the faster one by more than the model's error)
  const TileTimes* const teams = exact ? kExactTeams : e8m0 ? kE8m0Teams : kF32Teams;
  const int teamed = exact || e8m0 ? 1 : 2;  // kinds with two teams
  const int kinds = d.t <= 16 || f.kb > kTileBlocks ? 0 : exact ? 1 : e8m0 ? 3 : 2;
  const double sums = (double)d.t * f.groups * kFp8Group * 4;  // bytes of one part's
  for (int i = 0; i < kinds; ++i) {
    const int tt = 4 << i;
    const double tiles = (double)((d.t + 16 * tt - 1) / (16 * tt)) * (f.groups / kFp8TileGroups);
    for (int p = 1; p <= 8; p *= 2) {  // (16 parts cost more to join than they save)
      const int blocks = ((f.kb + p - 1) / p + 3) & ~3, parts = (f.kb + blocks - 1) / blocks;
      if (p > 1 && blocks < 8) break;
      const double wgs = tiles * parts, room = tt == 16 ? 256 : 512;  // workgroups that run together
      const double join = parts > 1 ? 3.0 + 2 * parts * sums / 7e6 : 0.0;
      auto take = [&](int teams_n, double us) {
        if (us >= best) return;
        best = us;
        f.tt = tt, f.teams = teams_n, f.parts = parts, f.blocks_part = blocks;
      };
      // up to a full card the others' reads slow a block down by and by; beyond, CUs take turns
      double block = times[i].one + (times[i].all - times[i].one) * wgs / 256;
      if (wgs > room)
        block = (tt == 16 ? times[i].all : times[i].two) * std::ceil(wgs / 256) * 256 / room;
      else if (wgs > 256)
        block = times[i].one + (times[i].two - times[i].one) * wgs / 512;
      // (a tile's start and end: under the other workgroup's blocks, where a CU has one)
      const double turns = std::ceil(wgs / room);
      const double starts = tt == 16 ? (d.gate_up ? 9.0 : 5.5) * turns : times[i].fixed * (0.5 * turns - 0.5);
      take(1, times[i].fixed + starts + blocks * block + join);
      if (i < teamed && wgs <= 256 && blocks >= 8)
        take(2, teams[i].fixed + (blocks + 7) / 8 * 4 * (teams[i].one + (teams[i].all - teams[i].one) * wgs / 256) + join);
    }
  }
}

Form form_of(const cev_fp8_desc& d) {
  Form f{};
  f.kb = (int32_t)((d.k + 127) / 128);
  f.groups = (int32_t)(d.gate_up ? (d.n + 127) / 128 * 8 : (d.n + 255) / 256 * 8);
  f.teams = f.parts = 1;
  f.mt = d.t <= 16 ? 1 : 2;
  f.blocks_part = f.kb;
  // The kernel for few rows can bring its 16 rows into e4m3 by itself, over and
  // over in each workgroup: for small weights that costs less than a launch (16
  // rows x 4096 x 2048: 5.9 us against 6.9; x 12288 x 4096: 22 against 14).
  f.pack_x = d.x_dtype != CEV_E4M3 && (d.t > 16 || units_of(d, f.kb, 16, 16) > 4096);
  if (d.x_dtype == CEV_E4M3 || f.pack_x) plan(d, f);
  if (f.pack_x) {
    f.rows_bytes = up256((size_t)d.t * f.kb * kFp8Block);
    f.scales_bytes = up256((size_t)d.t * f.kb);
  }
  if (f.parts > 1)
    f.part_bytes = (size_t)f.parts * d.t * f.groups * kFp8Group * 4;
  else if (d.gate_up && f.tt == 0)
    f.part_bytes = (size_t)d.t * ((d.n + 127) / 128) * 128 * 4;
  return f;
}

// Whether a form's launches count their threads in 32 bits.
bool grids_fit(const cev_fp8_desc& d, const Form& f) {
  if (f.tt == 0) {
    const int columns = f.mt == 4 ? 32 : 16;
    const int64_t col_tiles = (d.n + columns - 1) / columns, row_tiles = (d.t + 16 * f.mt - 1) / (16 * f.mt);
    return col_tiles <= 8 * 65535 && fp8_grid_fits(row_tiles * ((col_tiles + 7) / 8 * 8), kWaves * 64);
  }
  const int64_t row_tiles = (d.t + 16 * f.tt - 1) / (16 * f.tt);
  if (!fp8_grid_fits(row_tiles * (f.groups / kFp8TileGroups) * f.parts, 256 * f.teams)) return false;
  const int64_t quads = d.gate_up ? (d.n + 127) / 128 * 16 : (d.n + 3) / 4;
  return f.parts == 1 || fp8_grid_fits((d.t * quads + 255) / 256, 256);
}

int32_t check_desc(const char* what, const cev_fp8_desc* d) {
  CEV_CHECK_ARG(d != nullptr, "%s: null descriptor", what);
  if (d->x_dtype != CEV_F32 && d->x_dtype != CEV_BF16 && d->x_dtype != CEV_E4M3) return cev_fail(CEV_ERR_UNSUPPORTED, "%s: x dtype %d", what, d->x_dtype);
  if (d->gate_up ? d->out_dtype != CEV_E4M3 : d->out_dtype != CEV_F32 && d->out_dtype != CEV_BF16)
    return cev_fail(CEV_ERR_UNSUPPORTED, "%s: out dtype %d", what, d->out_dtype);
  if (d->scales != CEV_FP8_SCALES_E8M0 && d->scales != CEV_FP8_SCALES_F32) return cev_fail(CEV_ERR_UNSUPPORTED, "%s: scale kind %d", what, d->scales);
  CEV_CHECK_ARG(d->t >= 0 && d->t <= INT32_MAX && d->n >= 1 && d->n <= INT32_MAX - 256 && d->k >= 1 && d->k <= INT32_MAX - 128,
                "%s: %lld rows, %lld x %lld weight", what, (long long)d->t, (long long)d->n, (long long)d->k);
  // (the workspace's bytes stay within 64 bits)
  CEV_CHECK_ARG(d->t <= ((int64_t)1 << 46) / std::max(d->n, d->k), "%s: %lld rows are too large", what, (long long)d->t);
  return CEV_OK;
}

template <typename T, typename O, bool GATE_UP, int MT>
int32_t launch_small(const Fp8Args& a, bool e8m0, hipStream_t s) {
  const int columns = MT == 4 ? 32 : 16;
  const int64_t col_tiles = (a.n + columns - 1) / columns, row_tiles = (a.t + 16 * MT - 1) / (16 * MT);
  if (e8m0)
    hipLaunchKernelGGL((fp8_small_kernel<T, O, true, GATE_UP, MT>), dim3((unsigned)row_tiles * 8, (unsigned)((col_tiles + 7) / 8)), dim3(kWaves * 64), 0, s, a, (unsigned)col_tiles);
  else
    hipLaunchKernelGGL((fp8_small_kernel<T, O, false, GATE_UP, MT>), dim3((unsigned)row_tiles * 8, (unsigned)((col_tiles + 7) / 8)), dim3(kWaves * 64), 0, s, a, (unsigned)col_tiles);
  return launched("cev_fp8_product");
}

template <typename O, bool GATE_UP>
int32_t launch_small(const Fp8Args& a, int x_dtype, int mt, bool e8m0, hipStream_t s) {
  if (x_dtype == CEV_BF16) return launch_small<__bf16, O, GATE_UP, 1>(a, e8m0, s);
  if (x_dtype == CEV_F32) return launch_small<float, O, GATE_UP, 1>(a, e8m0, s);
  if constexpr (sizeof(O) == 2)
    if (mt == 4) return launch_small<uint8_t, O, GATE_UP, 4>(a, e8m0, s);
  return mt == 1 ? launch_small<uint8_t, O, GATE_UP, 1>(a, e8m0, s) : launch_small<uint8_t, O, GATE_UP, 2>(a, e8m0, s);
}

}  // namespace

extern "C" int32_t cev_fp8_work_size(const cev_fp8_desc* d, size_t* bytes) {
  if (const int32_t rc = check_desc("cev_fp8_work_size", d)) return rc;
  CEV_CHECK_ARG(bytes != nullptr, "cev_fp8_work_size: null output");
  const Form f = form_of(*d);
  *bytes = f.rows_bytes + f.scales_bytes + f.part_bytes;
  return CEV_OK;
}

extern "C" int32_t cev_fp8_form(const cev_fp8_desc* d, int32_t* rows, int32_t* parts, int32_t* teams) {
  if (const int32_t rc = check_desc("cev_fp8_form", d)) return rc;
  CEV_CHECK_ARG(rows && parts && teams, "cev_fp8_form: null output");
  const Form f = form_of(*d);
  *rows = 16 * (f.tt ? f.tt : f.mt);
  *parts = f.parts;
  *teams = f.tt ? f.teams : 0;
  return CEV_OK;
}

extern "C" int32_t cev_fp8_product(const cev_fp8_desc* d, const void* x, const void* x_scales, const void* weight, size_t weight_bytes,
                                   void* out, void* out_scales, void* work, size_t work_bytes, cev_stream stream) {
  const char* const me = "cev_fp8_product";
  if (const int32_t rc = check_desc(me, d)) return rc;
  size_t need = 0;
  if (const int32_t rc = cev_fp8_weight_size(d->n, d->k, d->gate_up, &need)) return rc;
  if (weight_bytes < need) return cev_fail(CEV_ERR_SPACE, "%s: a weight of %zu bytes, %zu needed", me, weight_bytes, need);
  if (d->t == 0) return CEV_OK;
  CEV_CHECK_ARG(x && weight && out, "%s: null buffer", me);
  CEV_CHECK_ARG((((uintptr_t)x | (uintptr_t)weight) & 15) == 0, "%s: x and the weight must be 16-byte aligned", me);
  CEV_CHECK_ARG((d->x_dtype == CEV_E4M3) == (x_scales != nullptr) && (d->gate_up != 0) == (out_scales != nullptr), "%s: rows in e4m3 come with their scales", me);
  if (d->x_dtype != CEV_E4M3 && d->t > 1) {
    const int vec = d->x_dtype == CEV_BF16 ? 8 : 4;
    CEV_CHECK_ARG(d->x_stride >= d->k && d->x_stride % vec == 0 && cev_stride_fits(d->x_stride, d->t),
                  "%s: the row stride of x must cover a row and be a multiple of %d elements", me, vec);
  }
  if (!d->gate_up) {
    CEV_CHECK_ARG(d->t <= 1 || (d->out_stride >= d->n && cev_stride_fits(d->out_stride, d->t)), "%s: the row stride of out must cover a row", me);
    CEV_CHECK_ARG(((uintptr_t)out & (d->out_dtype == CEV_BF16 ? 1 : 3)) == 0, "%s: misaligned out", me);
  } else {
    CEV_CHECK_ARG(((uintptr_t)out & 15) == 0, "%s: rows in e4m3 must be 16-byte aligned", me);
  }
  const Form f = form_of(*d);
  const size_t space_bytes = f.rows_bytes + f.scales_bytes + f.part_bytes;
  if (work_bytes < space_bytes) return cev_fail(CEV_ERR_SPACE, "%s: a workspace of %zu bytes, %zu needed", me, work_bytes, space_bytes);
  CEV_CHECK_ARG(space_bytes == 0 || (work && ((uintptr_t)work & 255) == 0), "%s: the workspace must be 256-byte aligned", me);
  if (!grids_fit(*d, f)) return cev_fail(CEV_ERR_UNSUPPORTED, "%s: grid too large", me);
  {
    const int64_t e = d->x_dtype == CEV_E4M3 ? 1 : d->x_dtype == CEV_BF16 ? 2 : 4, kb = f.kb, nb = (d->n + 127) / 128;
    const CevRows o = d->gate_up ? CevRows{out, 1, 0, d->t * nb * 128} : cev_rows(out, d->t, d->out_stride, d->n, d->out_dtype == CEV_BF16 ? 2 : 4);
    CEV_CHECK_ARG(fp8_apart({o, cev_rows(out_scales, 1, 0, d->t * nb, 1), cev_rows(space_bytes ? work : nullptr, 1, 0, (int64_t)space_bytes, 1)},
                            {d->x_dtype == CEV_E4M3 ? CevRows{x, 1, 0, d->t * kb * 128} : cev_rows(x, d->t, d->x_stride, d->k, e),
                             cev_rows(x_scales, 1, 0, d->t * kb, 1), cev_rows(weight, 1, 0, (int64_t)need, 1)}),
                  "%s: the output, and the workspace, must have memory of its own", me);
  }
  const hipStream_t s = (hipStream_t)stream;
  uint8_t* const space = (uint8_t*)work;
  int x_dtype = d->x_dtype;
  Fp8Args a{};
  a.x = x, a.xs = (const uint8_t*)x_scales;
  a.x_st = d->t > 1 ? d->x_stride : 0;
  if (f.pack_x) {
    if (const int32_t rc = cev_fp8_rows(d->x_dtype, d->t, d->k, x, d->x_stride, space, space + f.rows_bytes, stream)) return rc;
    a.x = space, a.xs = space + f.rows_bytes;
    x_dtype = CEV_E4M3;
  }
  a.w = (const uint8_t*)weight;
  a.ws = a.w + (int64_t)f.groups * f.kb * kFp8GroupBytes;
  a.ws_pitch = d->scales == CEV_FP8_SCALES_E8M0 ? (f.kb + 3) & ~3 : f.kb;
  a.out = out, a.out_st = d->t > 1 ? d->out_stride : 0;
  a.t = d->t, a.n = d->n, a.k = (int32_t)d->k, a.kb = f.kb, a.groups = f.groups, a.parts = f.parts, a.blocks_part = f.blocks_part;
  if (f.part_bytes) a.part = (float*)(space + f.rows_bytes + f.scales_bytes);
  const bool e8m0 = d->scales == CEV_FP8_SCALES_E8M0;
  a.out_s = (uint8_t*)out_scales;
  if (d->gate_up && f.tt == 0) {
    a.out_st = (d->n + 127) / 128 * 128;
    if (const int32_t rc = launch_small<float, true>(a, x_dtype, f.mt, e8m0, s)) return rc;
    return cev_fp8_rows(CEV_F32, d->t, d->n, a.part, a.out_st, out, out_scales, stream);
  }
  const int32_t rc = f.tt > 0 ? fp8_launch_tile(a, f.tt, f.teams, !d->gate_up && d->out_dtype == CEV_F32, e8m0, d->gate_up != 0, s)
                     : d->out_dtype == CEV_F32 ? launch_small<float, false>(a, x_dtype, f.mt, e8m0, s)
                                               : launch_small<__bf16, false>(a, x_dtype, f.mt, e8m0, s);
  if (rc || !a.part) return rc;
  JoinArgs j{a.part, out, (uint8_t*)out_scales, d->t, d->n, a.out_st, (int64_t)f.groups * kFp8Group, f.parts, 0};
  j.quads = (int32_t)(d->gate_up ? (d->n + 127) / 128 * 16 : (d->n + 3) / 4);
  const int64_t grid = (d->t * j.quads + 255) / 256;
  if (d->gate_up)
    hipLaunchKernelGGL(fp8_join_gate_up_kernel, dim3((unsigned)grid), dim3(256), 0, s, j);
  else if (d->out_dtype == CEV_BF16)
    hipLaunchKernelGGL(fp8_join_kernel<__bf16>, dim3((unsigned)grid), dim3(256), 0, s, j);
  else
    hipLaunchKernelGGL(fp8_join_kernel<float>, dim3((unsigned)grid), dim3(256), 0, s, j);
  return launched(me);
}
