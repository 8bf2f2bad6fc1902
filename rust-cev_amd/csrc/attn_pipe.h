// The bf16 d = 128 loop's LDS layout and read schedule, shared by the kernels
// over packed (packed_attn.hip) and paged keys (paged_tile.hip).
#pragma once
#include "attn_device.h"

namespace {

// K/V chunks go from HBM straight into LDS (buffer_load ... lds), kBuf chunk
// buffers deep.  Tiles are unpadded, 256 bytes a key row, with the 16-byte
// column blocks of a row permuted so the operand reads are free of bank
// conflicts:
//   K: block c of row r at slot c ^ (r & 15)   (ds_read_b128, one key row
//      per lane, 16 rows per 256 bytes read)
//   V: block c of row r at slot c ^ 4(r & 3)   (ds_read_b64_tr_b16, four
//      rows x four blocks per 16 lanes)
namespace pipe {
constexpr int kBuf = 4;             // chunk buffers
constexpr int kAhead = kBuf - 1;    // chunk i + kAhead is fetched in iteration i
constexpr int kRowBytes = 256;      // one bf16 key row of d = 128
constexpr int kTileBytes = 64 * kRowBytes;
constexpr int kVBase = kBuf * kTileBytes;  // K tiles first, then V tiles

__device__ __forceinline__ int k_slot(int blk, int row) { return blk ^ (row & 15); }

// Workgroup barrier after this wave's LDS operations have completed; global
// loads may still be in flight.  The asm is a compiler memory barrier too.
__device__ __forceinline__ void lds_barrier() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

typedef int i32x4 __attribute__((ext_vector_type(4)));

// The K operand reads go through asm as well, so that every LDS read in the
// loop body is one whose position the waits below can count.
template <int OFF>
__device__ __forceinline__ i32x4 read_b128(int vaddr) {
  static_assert(OFF >= 0 && OFF < 65536, "ds offset field");
  i32x4 r;
  asm volatile("ds_read_b128 %0, %1 offset:%2" : "=v"(r) : "v"(vaddr), "i"(OFF) : "memory");
  return r;
}
// One K operand fragment: a 16-byte read per lane.  Two 8-byte reads of
// the same bytes measured no faster; the reads are bound by LDS bytes.
typedef i32x4 KFrag;
template <int N>
__device__ __forceinline__ void wait_b128(i32x4& r) {
  static_assert(N >= 0 && N < 16, "lgkmcnt range");
  asm volatile("s_waitcnt lgkmcnt(%1)" : "+v"(r) : "i"(N));
}

// Issue order of the LDS reads of one sub-tile body (NQK = 8 QK units, then
// NPV = 8 PV units), K reads KPF and V fragments VPF ahead of their MFMA.
// QK unit u waits for K read u, then issues K read u + KPF (if any) and, in
// its last VPF units, the two reads of V fragment u - (8 - VPF).  PV unit j
// waits for V fragment j, then issues V fragment j + VPF (if any) and, in
// its last KPF units, K read j - (8 - KPF) of the next body.  The wait of
// each unit is the number of LDS reads issued after the one it needs; the
// count below replays one steady-state body.
struct ReadSchedule {
  int wait_a[8], wait_b[8];
};
constexpr ReadSchedule read_schedule(int kpf, int vpf) {
  ReadSchedule r{};
  int kpos[8] = {}, vhi[8] = {};
  int pos = 0;
  // the previous body's PV units: V reads of that body, then this body's
  // first kpf K reads
  for (int j = 0; j < 8; ++j) {
    if (j + vpf < 8) pos += 2;
    if (j >= 8 - kpf) kpos[j - (8 - kpf)] = pos++;
  }
  for (int u = 0; u < 8; ++u) {
    r.wait_a[u] = pos - kpos[u] - 1;
    if (u + kpf < 8) kpos[u + kpf] = pos++;
    if (u >= 8 - vpf) {
      vhi[u - (8 - vpf)] = pos + 1;
      pos += 2;
    }
  }
  for (int j = 0; j < 8; ++j) {
    r.wait_b[j] = pos - vhi[j] - 1;
    if (j + vpf < 8) {
      vhi[j + vpf] = pos + 1;
      pos += 2;
    }
    if (j >= 8 - kpf) ++pos;
  }
  return r;
}
constexpr bool waits_in_range(const ReadSchedule& r) {
  for (int i = 0; i < 8; ++i)
    if (r.wait_a[i] < 0 || r.wait_a[i] > 15 || r.wait_b[i] < 0 || r.wait_b[i] > 15) return false;
  return true;
}
// The loop's two forms.  Staggered (STAG): waves 4-7 run one region ahead of
// waves 0-3; on the 32k-key prefill with all 8 waves busy it ran 1.4 %
// faster than in step, and four K and two V fragments ahead ran 0.5 %
// faster there than three and three.  In step, three and three: a tile with
// at most 4 busy waves (a short block, the KV-streaming shape) has nothing
// to stagger, and there the staggered form's code ran 3 % slower.
template <bool STAG>
struct Schedule {
  static constexpr int KPF = STAG ? 4 : 3;  // K fragments in flight ahead of their MFMA
  static constexpr int VPF = STAG ? 2 : 3;  // V fragments in flight ahead of their MFMA
  static_assert(KPF >= 1 && KPF <= 8 && VPF >= 1 && VPF <= 8, "prefetch depths");
  static constexpr ReadSchedule reads = read_schedule(KPF, VPF);
  static_assert(waits_in_range(reads), "lgkmcnt range");
  static constexpr int wait_a(int st) { return reads.wait_a[st]; }
  static constexpr int wait_b(int j) { return reads.wait_b[j]; }
};
static_assert(Schedule<false>::wait_a(0) == 2 && Schedule<false>::wait_a(5) == 2 && Schedule<false>::wait_a(6) == 3 &&
                  Schedule<false>::wait_a(7) == 4 && Schedule<false>::wait_b(0) == 4 && Schedule<false>::wait_b(4) == 4 &&
                  Schedule<false>::wait_b(5) == 4 && Schedule<false>::wait_b(6) == 3 && Schedule<false>::wait_b(7) == 2,
              "wait counts at three fragments ahead");
static_assert(Schedule<true>::wait_a(0) == 5 && Schedule<true>::wait_a(1) == 3 && Schedule<true>::wait_a(5) == 2 &&
                  Schedule<true>::wait_a(6) == 1 && Schedule<true>::wait_a(7) == 2 && Schedule<true>::wait_b(0) == 2 &&
                  Schedule<true>::wait_b(5) == 3 && Schedule<true>::wait_b(6) == 4 && Schedule<true>::wait_b(7) == 2,
              "wait counts at four K and two V fragments ahead");
}  // namespace pipe

}  // namespace
