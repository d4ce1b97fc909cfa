// fgg_f16.cu - products grouped by expert in bf16 / fp16, over contiguous token
// rows with the group offsets on the device: the forward product and its two
// gradients.
//
//   forward  y[r, n]    = sum_k x[r, k]  W_g[n, k]     r in group g
//   dgrad    dx[r, k]   = sum_n dy[r, n] W_g[n, k]
//   wgrad    dW_g[n, k] = sum_{r in g} dy[r, n] x[r, k]
//
// All three run one persistent kernel of CTA pairs (tcgen05 .cta_group::2,
// .kind::f16, fp32 accumulators in TMEM).  The tensor core's M axis is the
// weights' output axis (n forward, k dgrad, n wgrad), 256 per pair; its N axis
// is the group's tokens (forward, dgrad: up to 256, in steps of 32, so that a
// ragged group costs what its rows cost) or k (wgrad, 256).  No operand is
// transposed in memory: where the contraction is not the contiguous axis
// (W in dgrad, both operands in wgrad) the tiles are read MN-major, boxes of
// 64 x 64 whose descriptor names the major axis.
//
// Ragged edges cost no branches in the main loop:
//   * tokens behind a group's end (forward, dgrad) are the next group's: they
//     only reach accumulator columns that are not stored;
//   * in wgrad they would enter the sum (and an infinity there spoil it, even
//     against a zero), so a group's last rows % 16 rows are read from a copy with
//     zeros behind them, which the prepare kernel makes (16 rows per group and
//     operand); the step before it multiplies only its whole sixteens of rows;
//   * n and k need not be multiples of the tile: TMA fills zeros, and the
//     epilogues clip.
//
// The tensor core adds each instruction's sixteen products to its fp32
// accumulator with truncation, so a long sum drifts towards zero: by 5e-6 of its
// value on average over groups of 4000 rows, ten times what fp32 additions in
// order lose.  Against a gradient's fp32 that is visible, so wgrad sums 512 rows
// at a time in TMEM and the epilogue adds those sums in registers, rounding to
// nearest; a 16-bit result hides it (forward, dgrad).
//
// A few tiles, or a few long ones (a small expert's gradient over all its rows, one
// expert's tokens), leave pairs idle: the prepare kernel cuts such a tile along the
// contraction into up to 16 slices, units of work like the other tiles.  Their fp32
// sums are joined two by two: of two neighbours the warp that is done first leaves its
// sums in the workspace and goes on, the other adds them to its own and stands for
// both.  Nothing waits, and as a + b = b + a the results do not depend on timing.  They
// may depend, in the last fp32 bits before the rounding, on the call's other tiles.
//
// What bounds it: the tensor pipe for groups of about 250 tokens and more (forward,
// dgrad) or some thousand rows (wgrad), the weights' HBM stream below that in forward
// and dgrad.  In wgrad with short groups no unit is full: at 256 rows each the SMs' L1,
// through which the operands come and the gradient leaves, is busiest with 74 %, then
// DRAM 58 %, L2 52 %, tensor pipe 29 % (groups of 4096 rows: 47, 17, 38 and 73 %).  In
// seconds-long runs of any of them but the decode shapes it is the 1000 W cap (clocks
// of 1.0 to 1.5 GHz), under which what counts is energy: the bytes moved as much as
// the products.  Measured, bf16, short bursts / under the cap (3 to 6 % more on some
// machines):
//   forward 8192^3                             1.53 / 1.34 PFLOP/s, tensor pipe 95 %
//                                              active (the library's product 1.56 / 1.40)
//   forward 8 groups, 4352 rows, 4096 x 7168   200 / 238 us, tensor pipe 88 % active,
//                                              582 MB of DRAM reads (541 MB needed)
//   forward 64 groups, 544 rows, 7168 x 2048   280 us, 6.7 TB/s
//   dgrad 64 skewed groups, 16384 rows         0.90 / 1.10 ms
//   wgrad 64 skewed groups, 32768 rows, fp32   1.10 / 1.32 ms
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>
#include <atomic>
#include <cstring>

#include "fgg_engine.cuh"
#include "fgg_host.cuh"

namespace fgg {
namespace {

constexpr int kFwd = 0, kDgrad = 1, kWgrad = 2;
constexpr int kF16BadOffsets = 0x203;  // offsets decreasing, negative or past max_rows

// Token boxes of 16, 32, ..., 128 rows: a CTA loads half of its tile's tokens.
constexpr int kTokenMaps = 8;

struct F16Slot {
  int32_t g;       // group, -1 = no more tiles
  int32_t mt;      // tile of the M axis
  int32_t row0;    // first token row of the tile (wgrad: of the group)
  int32_t rows;    // tokens of the tile (forward, dgrad) / of the group (wgrad)
  int32_t ct;      // tile of the N axis (wgrad)
  int32_t k0, k1;  // its steps of the contraction
  uint32_t split;  // 0 = all of them, else the unit's word (see split_word)
};
static_assert(sizeof(F16Slot) == 32, "slot is 8 words");

// A tile is split if a pair's share of the call's steps (over all pairs of the GPU, so
// that neither spare rows nor empty groups count) is at most half of the tile's own, and
// for a tile of fewer than 4 kMinSlice steps at most a fifth; into slices of about that
// share, of at least kMinSlice steps: the units of split tiles are at most as many as
// pairs.  A join costs 4 to 5 us, up to 9 where all pairs join at once after few steps,
// and a step about 0.26 us of a pair.  Unsplit -> split, cold L2, a host call's time with
// it: one tile of 64 steps in two (a gradient of 64 x 64 over 4096 rows) 31.7 -> 27.6 us,
// 8 of them (one token, 2048 x 4096) 25.6 -> 23.4, 16 of them 25.9 -> 27.0, 24 of them
// (256 tokens) 36.3 -> 39.0; one of 128 in four (one token, K 8192) 34.1 -> 23.5; of 470
// in 14 (30000 rows) 144 -> 37; 32 tiles of 128 in two (one token, 8192 x 8192) 50.1 ->
// 47.9.  With slices of at least 16 steps the 24 tiles of 256 tokens take 43.4 us (36.7),
// 8 tiles of 94 steps 39.9 (37.8), one tile of 64 steps 25.6 (27.6); of at least 64 the
// 30000 rows take 43.8 (37.0), one token of 4096 x 14336 60.4 (43.8).
constexpr int kMaxSplitUnits = 96;
constexpr int kMaxSlices = 16;
constexpr int kMinSlice = 32;
// 128 fp32 sums per lane and epilogue warp of a pair
constexpr int kWarpSums = 2 * 8;
constexpr int kUnitFloats = kWarpSums * 128 * 32;
// Unit of a split tile: tile, slice, slices, the tile's first unit.
__host__ __device__ constexpr uint32_t split_word(int tile, int slice, int slices, int first) {
  return uint32_t(tile) | uint32_t(slice) << 8 | uint32_t(slices) << 16 | uint32_t(first) << 24;
}

struct F16Params {
  CUtensorMap tmap_w;                // forward, dgrad: [G, N, K] weights
  CUtensorMap tmap_tok[kTokenMaps];  // forward, dgrad: [rows, contraction] tokens
  CUtensorMap tmap_a, tmap_b;        // wgrad: dy [rows, N], x [rows, K]
  CUtensorMap tmap_ta, tmap_tb;      // wgrad: the groups' last rows, [16 G, N], [16 G, K]
  const uint64_t* tiles;             // forward, dgrad: group << 48 | mt << 32 | first row
  const int32_t* tile_rows;          // forward, dgrad: tokens of each tile
  const int32_t* offsets;
  const int32_t* order;  // wgrad: groups, the largest first
  void* out;
  const uint32_t* units;  // of the split tiles, which are the list's first
  int32_t* arrived;       // per unit and epilogue warp: sides that came to that join
  float* partial;         // per unit: the epilogue warps' sums
  int* status;  // [0] status [1] unit counter [3] tiles [4] split tiles [5] their units
  int32_t num_groups;
  int32_t m_ext;   // extent of the M axis (the output's columns; wgrad: its rows n)
  int32_t c_ext;   // wgrad: extent of the N axis (k)
  int32_t ksteps;  // forward, dgrad: 64-element steps of the contraction
  int32_t mts, cts;
  int32_t max_rows;
  int32_t grid_units;  // host bound on the tiles and slices
  int32_t bf16;        // operands bf16 (1) or fp16 (0)
  int32_t out_fp32;    // wgrad: fp32 gradient
  int32_t accumulate;  // wgrad, fp32: add to the gradient
  int32_t debug_flags;
};

__device__ __forceinline__ uint32_t pack_16(float lo, float hi, bool bf16) {
  if (bf16) return pack_bf16x2(lo, hi);
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}

template <int MODE_, bool SPLIT_>
struct F16Cfg {
  static constexpr int MODE = MODE_;
  // Tiles may be split.  A build of its own, for problems whose sizes allow it: with the
  // joins' registers the unsplit gradient of 64 skewed experts, 32768 rows, 7168 x 2048
  // took 1368 us in place of 1319.  Whole tiles of a
  // problem that may have split ones pay up to 1 us (16 skewed groups, 4096 rows,
  // 1024 x 512: 26.7 -> 27.8 us).
  static constexpr bool SPLIT = SPLIT_;
  static constexpr bool A_MN = MODE_ != kFwd;
  static constexpr bool B_MN = MODE_ == kWgrad;
  static constexpr int BN = 256;   // N axis of a pair tile
  static constexpr int KS = 64;    // contraction per stage: one 128-byte swizzle row
  static constexpr uint32_t A_BYTES = 128 * 128;
  static constexpr uint32_t B_BYTES = 128 * 128;  // half of 256 columns
  static constexpr uint32_t STAGE_BYTES = A_BYTES + B_BYTES;
  static constexpr int STAGES = 7;
  static constexpr uint32_t TMEM_COLS = 512;  // two accumulators of 256 columns
  static constexpr int SCHED = 8;
  // Epilogue warps of a CTA: two per TMEM quadrant.  In wgrad each holds 128
  // columns in registers over the chunks of a long group.
  static constexpr int EPI_WARPS = 8;
  static constexpr int THREADS = 128 + 32 * EPI_WARPS;
  // wgrad's registers: launched with 168 per thread (384 threads), of which the
  // four other warps give most to the epilogue's 128 sums
  static constexpr int REGS_OTHER = 64, REGS_EPI = 216;
  static constexpr int REGS_TOTAL = 128 * REGS_OTHER + 32 * EPI_WARPS * REGS_EPI;
  // steps of the contraction that one TMEM accumulator sums
  static constexpr int CHUNK = MODE_ == kWgrad ? 8 : 1 << 30;
  // arrivals that free a slot: on the leader its producer, MMA warp and epilogue warps
  // and the follower's forwarding warp; on the follower its producer and epilogue warps
  static constexpr uint32_t READERS_LEADER = 3 + EPI_WARPS;
  static constexpr uint32_t READERS_FOLLOWER = 1 + EPI_WARPS;
  static constexpr uint32_t NBARS = 2 * STAGES + 4 + 2 * SCHED + 4;
  static constexpr uint32_t BAR_REGION = STAGES * STAGE_BYTES;
  static constexpr uint32_t SMEM_BYTES = 1024 + BAR_REGION + 8 * NBARS + 32 * SCHED + 16;
  static_assert(SMEM_BYTES <= 232448, "shared memory budget exceeded");
};

// ------------------------------------------------------------- epilogues
// Forward, dgrad.  The warp's 32 TMEM lanes are the output columns m0 + lane, its
// TMEM columns the tile's tokens.  A word of two tokens' results per column goes
// through three rounds of swaps between lanes 1, 2 and 4 apart, after which lane l
// holds columns (l & ~7) .. + 7 of tokens 2 (l & 7), 2 (l & 7) + 1 and those 16
// further on: 16 contiguous bytes to store, 64 of each token per instruction.
// Columns past the output's edge are not stored.
struct F16Rows {
  uint16_t* out;  // at column m0 + (lane & ~7)
  size_t row0, ldn;
  int rows;
  bool col_ok, bf16;
};
__device__ __forceinline__ void f16_pack_block(const uint32_t (&r)[32], bool bf16,
                                               uint32_t (&w)[16]) {
#pragma unroll
  for (int i = 0; i < 16; ++i)  // tokens 2 i, 2 i + 1 of column l
    w[i] = pack_16(__uint_as_float(r[2 * i]), __uint_as_float(r[2 * i + 1]), bf16);
}
__device__ __forceinline__ void f16_turn_block(const F16Rows& d, int c0, const uint32_t (&w)[16]) {
  const int lane = threadIdx.x & 31;
  const bool b0 = lane & 1, b1 = lane & 2, b2 = lane & 4;
  uint32_t x[8][2];  // token pair 2 i + b0 of columns (l & ~1) + 0, 1
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const uint32_t got = __shfl_xor_sync(kFullMask, b0 ? w[2 * i] : w[2 * i + 1], 1);
    x[i][0] = b0 ? got : w[2 * i];
    x[i][1] = b0 ? w[2 * i + 1] : got;
  }
  uint32_t y[4][4];  // token pair 4 i + 2 b1 + b0 of columns (l & ~3) + 0 .. 3
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const uint32_t got = __shfl_xor_sync(kFullMask, b1 ? x[2 * i][j] : x[2 * i + 1][j], 2);
      y[i][j] = b1 ? got : x[2 * i][j];
      y[i][2 + j] = b1 ? x[2 * i + 1][j] : got;
    }
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    uint32_t z[8];  // token pair 8 i + (l & 7) of columns (l & ~7) + 0 .. 7
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint32_t got = __shfl_xor_sync(kFullMask, b2 ? y[2 * i][j] : y[2 * i + 1][j], 4);
      z[j] = b2 ? got : y[2 * i][j];
      z[4 + j] = b2 ? y[2 * i + 1][j] : got;
    }
    const int t = c0 + 16 * i + 2 * (lane & 7);
    uint16_t* const at = d.out + (d.row0 + size_t(t)) * d.ldn;
    if (t < d.rows && d.col_ok)
      *reinterpret_cast<uint4*>(at) =
          make_uint4(__byte_perm(z[0], z[1], 0x5410), __byte_perm(z[2], z[3], 0x5410),
                     __byte_perm(z[4], z[5], 0x5410), __byte_perm(z[6], z[7], 0x5410));
    if (t + 1 < d.rows && d.col_ok)
      *reinterpret_cast<uint4*>(at + d.ldn) =
          make_uint4(__byte_perm(z[0], z[1], 0x7632), __byte_perm(z[2], z[3], 0x7632),
                     __byte_perm(z[4], z[5], 0x7632), __byte_perm(z[6], z[7], 0x7632));
  }
}

// A whole tile: the quadrant's two warps by turns, 32 tokens each; the next ones are
// read while these are turned and stored.
__device__ __forceinline__ void f16_epilogue_rows(const F16Rows& d, int ncols, int part,
                                                  uint32_t taddr) {
  uint32_t r[32];
  int c0 = 32 * part;
  if (c0 < ncols) tmem_ld32(taddr + c0, r);
  for (; c0 < ncols; c0 += 64) {
    tmem_wait_ld();
    uint32_t w[16];
    f16_pack_block(r, d.bf16, w);
    if (c0 + 64 < ncols) tmem_ld32(taddr + c0 + 64, r);
    f16_turn_block(d, c0, w);
  }
}

// ----------------------------------------------------------- split tiles
// The tree over a split tile's slices, walked by one warp.  At height h it stands for
// the slices first .. first + 2^h - 1, as far as there are so many; its neighbour's
// begin where bit h of `first` is the other way.  A join is known by the first slice
// of its right side.
struct F16Tree {
  float* sums;       // this warp's and lane's, of the tile's slice 0
  int32_t* arrived;  // this warp's, of the tile's slice 0
  int first, slices, h;
  __device__ __forceinline__ float* mine() const { return sums + size_t(first) * kUnitFloats; }
  __device__ __forceinline__ float* other() const {
    return sums + size_t(first ^ (1 << h)) * kUnitFloats;
  }
  // Up to the next join; false at the top.
  __device__ __forceinline__ bool next() {
    while ((1 << h) < slices && (first ^ (1 << h)) >= slices) ++h;
    return (1 << h) < slices;
  }
  // This side's sums are in mine().  True if the other's are in other(): go on for both.
  __device__ __forceinline__ bool arrive() {
    __threadfence();
    __syncwarp();
    int before = 0;
    if ((threadIdx.x & 31) == 0) before = atomicAdd(arrived + (first | 1 << h) * kWarpSums, 1);
    before = __shfl_sync(kFullMask, before, 0);
    __threadfence();
    return before != 0;
  }
  __device__ __forceinline__ void joined() { first &= ~(1 << h++); }
};
// Of epilogue warp `ewarp` (0 .. 15 over both CTAs) of the unit.
__device__ __forceinline__ F16Tree f16_tree(const F16Params& p, uint32_t unit, int ewarp) {
  F16Tree t;
  const size_t unit0 = unit >> 24;
  t.sums = p.partial + unit0 * kUnitFloats + ewarp * 4096 + (threadIdx.x & 31);
  t.arrived = p.arrived + unit0 * kWarpSums + ewarp;
  t.first = int(unit >> 8 & 0xFFu);
  t.slices = int(unit >> 16 & 0xFFu);
  t.h = 0;
  return t;
}

// 32 bytes of one lane to a 16-byte aligned address (one store where it is
// 32-byte aligned), of which the first `bytes` (32 or 16) are the tensor's.
template <bool kFp32>
__device__ __forceinline__ void store_sector(uint8_t* at, uint32_t (&v)[8], int bytes,
                                             bool accumulate) {
  if (kFp32 && accumulate) {  // whole sectors
    const float4 lo = *reinterpret_cast<const float4*>(at);
    const float4 hi = *reinterpret_cast<const float4*>(at + 16);
    const float old[8] = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = __float_as_uint(old[j] + __uint_as_float(v[j]));
  }
  if (bytes == 32 && (reinterpret_cast<uintptr_t>(at) & 31u) == 0) {
    asm volatile("st.global.cs.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(at), "r"(v[0]),
                 "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7])
                 : "memory");
  } else {
    __stcs(reinterpret_cast<uint4*>(at), make_uint4(v[0], v[1], v[2], v[3]));
    if (bytes == 32) __stcs(reinterpret_cast<uint4*>(at) + 1, make_uint4(v[4], v[5], v[6], v[7]));
  }
}

// Wgrad.  The warp's lanes hold gradient rows n0 + lane, `acc` 128 columns from
// k0 of each.  Neighbouring lanes swap halves of 64 bytes, so that the two of them
// store 64 contiguous bytes of one row and then of the other: 6.7 TB/s of L2 writes
// over all SMs (32-byte pieces of 32 rows: 4.6; whole 128-byte lines: 7.5).  Lines
// would take a turn through shared memory, which made the 64 skewed groups slower
// (1193 against 1089 us): more traffic of the unit that short groups keep busiest.
// With accumulate the lane that stores reads what is there and adds: one addition
// per element.
template <bool kFp32>
__device__ __forceinline__ void f16_store_wgrad(const F16Params& p, int g, int n0, int k0,
                                                const float (&acc)[128]) {
  const int lane = threadIdx.x & 31;
  const bool odd = lane & 1;
  const int kcols = min(128, p.c_ext - k0);
  if (n0 >= p.m_ext || kcols <= 0) return;
  constexpr int eb = kFp32 ? 4 : 2;
  const size_t pitch = size_t(p.c_ext) * eb;
  const int row = n0 + (lane & ~1);
  uint8_t* const out = static_cast<uint8_t*>(p.out) +
                       (size_t(g) * size_t(p.m_ext) + size_t(row)) * pitch + size_t(k0) * eb +
                       (odd ? 32 : 0);
#pragma unroll
  for (int c = 0; c < 2 * eb; ++c) {  // 64 bytes of each row
    if (c * (64 / eb) >= kcols) break;
    uint32_t first[8], second[8];  // the even lane's row, the odd lane's
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      uint32_t lo, hi;
      if constexpr (kFp32) {
        lo = __float_as_uint(acc[16 * c + j]);
        hi = __float_as_uint(acc[16 * c + 8 + j]);
      } else {
        const bool b = p.bf16 != 0;
        lo = pack_16(acc[32 * c + 2 * j], acc[32 * c + 2 * j + 1], b);
        hi = pack_16(acc[32 * c + 16 + 2 * j], acc[32 * c + 17 + 2 * j], b);
      }
      const uint32_t got = __shfl_xor_sync(kFullMask, odd ? lo : hi, 1);
      first[j] = odd ? got : lo;
      second[j] = odd ? hi : got;
    }
    // columns are a multiple of 8: a 16-bit sector may be half the tensor's
    const int bytes = min(32, (kcols - c * (64 / eb)) * eb - (odd ? 32 : 0));
    if (bytes > 0) {
      if (row < p.m_ext) store_sector<kFp32>(out + c * 64, first, bytes, p.accumulate != 0);
      if (row + 1 < p.m_ext)
        store_sector<kFp32>(out + pitch + c * 64, second, bytes, p.accumulate != 0);
    }
  }
}

// Steps of the contraction over a group of m rows (wgrad): 64 rows each, then
// the whole sixteens of what is left, then the last m % 16 rows' copy.
__device__ __forceinline__ int wgrad_flat_steps(int m) { return (m / 16 + 3) / 4; }
__device__ __forceinline__ int wgrad_steps(int m) {
  return wgrad_flat_steps(m) + ((m & 15) != 0 ? 1 : 0);
}

// ------------------------------------------------------------ the kernel
// The words from k0 on are published where tiles may be split.
__device__ __forceinline__ F16Slot f16_read_slot(const volatile F16Slot* ring, int slot) {
  F16Slot s;
  s.g = ring[slot].g;
  s.mt = ring[slot].mt;
  s.row0 = ring[slot].row0;
  s.rows = ring[slot].rows;
  s.ct = ring[slot].ct;
  s.k0 = ring[slot].k0;
  s.k1 = ring[slot].k1;
  s.split = ring[slot].split;
  return s;
}

// Tile `local` of a group's rows x cols tiles: strips of eight columns, row by row.
// The 74 pairs then work on about nine rows and eight columns at a time, whose
// operands they share in L2, whatever the grid's shape.
constexpr int kStrip = 8;
__device__ __forceinline__ void f16_place(int local, int rows, int cols, int* row, int* col) {
  const int strip = local / (kStrip * rows);
  const int rest = local - strip * kStrip * rows;
  const int width = min(kStrip, cols - strip * kStrip);
  *row = rest / width;
  *col = strip * kStrip + rest - *row * width;
}

template <class C>
__device__ __forceinline__ F16Slot f16_make_slot(const F16Params& p, int unit, int num_tiles,
                                                 int split_tiles, int split_units) {
  F16Slot s;
  s.g = -1;
  s.mt = s.row0 = s.rows = s.ct = s.k0 = s.k1 = 0;
  s.split = 0;
  int t = unit;
  if constexpr (C::SPLIT) {
    t += split_tiles - split_units;
    if (unit < split_units) {
      s.split = p.units[unit];
      t = int(s.split & 0xFFu);
    }
  }
  if (t >= num_tiles) return s;
  if constexpr (C::MODE == kWgrad) {
    const int per = p.mts * p.cts;
    const int pos = t / per;
    const int local = t - pos * per;
    s.g = p.order[pos];
    f16_place(local, p.mts, p.cts, &s.mt, &s.ct);
    s.row0 = p.offsets[s.g];
    s.rows = p.offsets[s.g + 1] - s.row0;
  } else {
    const uint64_t tile = p.tiles[t];
    s.g = int(tile >> 48);
    s.mt = int((tile >> 32) & 0xFFFFu);
    s.row0 = int(uint32_t(tile));
    s.rows = p.tile_rows[t];
  }
  s.k1 = C::MODE == kWgrad ? wgrad_steps(s.rows) : p.ksteps;
  if (C::SPLIT && s.split != 0) {
    const int64_t steps = s.k1, slice = s.split >> 8 & 0xFFu, slices = s.split >> 16 & 0xFFu;
    s.k0 = int(steps * slice / slices);
    s.k1 = int(steps * (slice + 1) / slices);
  }
  return s;
}

// What forms addresses is checked before it does: a tile that is not one of the
// problem's ends the kernel with a status.
template <class C>
__device__ __forceinline__ bool f16_slot_in_range(const F16Params& p, const F16Slot& s) {
  const bool rows = C::MODE == kWgrad ? s.rows >= 0 : s.rows > 0 && s.rows <= C::BN;
  return rows && unsigned(s.g) < unsigned(p.num_groups) && unsigned(s.mt) < unsigned(p.mts) &&
         unsigned(s.ct) < unsigned(p.cts) && s.row0 >= 0 && s.row0 <= p.max_rows - s.rows &&
         (s.split >> 24) + (s.split >> 8 & 0xFFu) < unsigned(kMaxSplitUnits);
}

// Roles as in the block-scaled pair kernel (fgg_engine.cuh): warp 0 producer in
// both CTAs, warp 1 MMA issuer in the leader and forwarder of releases in the
// follower, warp 2 TMEM, warp 3 scheduler in the leader, the others epilogue.
template <class C>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(C::THREADS, 1)
    f16_pair_kernel(const __grid_constant__ F16Params p) {
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw = smem_u32(smem_raw);
  const uint32_t base = (raw + 1023u) & ~1023u;
  uint8_t* const gbase = smem_raw + (base - raw);

  const uint32_t bars = base + C::BAR_REGION;
  auto full_bar = [&](int s) { return bars + 8u * s; };
  auto empty_bar = [&](int s) { return bars + 8u * (C::STAGES + s); };
  auto accf_bar = [&](int b) { return bars + 8u * (2 * C::STAGES + b); };
  auto acce_bar = [&](int b) { return bars + 8u * (2 * C::STAGES + 2 + b); };
  auto schedf_bar = [&](int i) { return bars + 8u * (2 * C::STAGES + 4 + i); };
  auto schede_bar = [&](int i) { return bars + 8u * (2 * C::STAGES + 4 + C::SCHED + i); };
  const uint32_t tmem_ready_bar = bars + 8u * (2 * C::STAGES + 4 + 2 * C::SCHED);
  const uint32_t drain_bar = tmem_ready_bar + 8u;
  auto taken_bar = [&](uint32_t n) { return tmem_ready_bar + 16u + 8u * (n & 1u); };
  uint8_t* const misc = gbase + C::BAR_REGION + 8 * C::NBARS;
  volatile F16Slot* const ring = reinterpret_cast<volatile F16Slot*>(misc);
  volatile uint32_t* const tmem_holder =
      reinterpret_cast<volatile uint32_t*>(misc + 32 * C::SCHED);
  volatile int* const abort_flag = reinterpret_cast<volatile int*>(misc + 32 * C::SCHED + 4);

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const uint32_t rank = cluster_ctarank();
  const bool leader = (rank == 0);
  const uint32_t peer = rank ^ 1u;

  auto sA = [&](int s) { return base + s * C::STAGE_BYTES; };
  auto sB = [&](int s) { return base + s * C::STAGE_BYTES + C::A_BYTES; };
  // MMA N of a tile: multiples of 32, so that each CTA holds a multiple of 16 rows
  auto tile_ncols = [&](int rows) -> int {
    return C::MODE == kWgrad ? C::BN : min(C::BN, (rows + 31) & ~31);
  };

  // steps of a unit
  auto unit_k0 = [&](int slot) -> int {
    return C::SPLIT ? __shfl_sync(kFullMask, ring[slot].k0, 0) : 0;
  };
  auto unit_k1 = [&](int slot, int rows) -> int {
    if constexpr (C::SPLIT) return __shfl_sync(kFullMask, ring[slot].k1, 0);
    return C::MODE == kWgrad ? wgrad_steps(rows) : p.ksteps;
  };

  if (threadIdx.x == 0) {
    for (int s = 0; s < C::STAGES; ++s) {
      mbar_init(full_bar(s), 1);
      mbar_init(empty_bar(s), 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(accf_bar(b), 1);
      mbar_init(acce_bar(b), C::EPI_WARPS + (leader ? 1 : 0));  // and the forwarder
    }
    for (int i = 0; i < C::SCHED; ++i) {
      mbar_init(schedf_bar(i), 1);
      mbar_init(schede_bar(i), leader ? C::READERS_LEADER : C::READERS_FOLLOWER);
    }
    mbar_init(tmem_ready_bar, 1);
    mbar_init(drain_bar, 1);
    mbar_init(taken_bar(0), 1);
    mbar_init(taken_bar(1), 1);
    *abort_flag = 0;
    fence_mbar_init();
  }
  cluster_sync();

  if (warp == 2) {
    tmem_alloc_pair(smem_u32(const_cast<uint32_t*>(tmem_holder)), C::TMEM_COLS);
    tmem_relinquish_pair();
    tc_fence_before();
    __syncwarp();
    if (lane == 0) mbar_arrive(tmem_ready_bar);
  }

  // the tile list, the copies of last rows and the status words come from the
  // prepare kernel just before this launch, which it may overlap until here
  griddep_wait();
  const uint32_t leader_schede0 = mapa_shared(schede_bar(0), 0);
  const uint32_t leader_acce0 = mapa_shared(acce_bar(0), 0);
  const uint32_t leader_full0 = mapa_shared(full_bar(0), 0);

  // the register split comes first in each branch: the compiler allots by branch
  if (warp < 4) {
    if constexpr (C::MODE == kWgrad) regs_dec<C::REGS_OTHER>();
    if (warp == 3) {
      // ---------------------------------------------- scheduler (leader only)
      if (lane == 0 && leader) {
        int slot = 0;
        uint32_t sphase = 0;
        const int num_tiles = p.status[3];
        const int split_tiles = C::SPLIT ? p.status[4] : 0;
        const int split_units = C::SPLIT ? p.status[5] : 0;
        const int num_units = num_tiles - split_tiles + split_units;
        const bool few = C::SPLIT && num_units <= int(gridDim.x >> 1);
        const uint32_t remote_ring0 = mapa_shared(smem_u32(const_cast<F16Slot*>(ring)), peer);
        const uint32_t remote_schedf0 = mapa_shared(schedf_bar(0), peer);
        for (uint32_t n = 0;; ++n) {
          // Claim tile n once the producer has taken tile n - 2 (even and odd tiles
          // on a barrier each): claiming and publishing take about 3 us (an atomic's
          // way to L2, the peer's ring), longer than a short tile.  A pair then holds
          // at most two tiles that it has not started.
          // A tile of wgrad is as long as its group: this wait alone may take a minute.
          bool taken = n < 2;
          for (int tries = 0; !taken && tries < 60 && *abort_flag == 0; ++tries)
            taken = mbar_wait_one(taken_bar(n), ((n >> 1) - 1u) & 1u, kWaitLimitNs);
          if (!taken) {
            atomicCAS(p.status, 0, kStatusTimeoutProducer);
            *abort_flag = 1;
            break;
          }
          // few units: one for each pair, none claimed ahead of a pair that has none
          const int unit = few ? (n == 0 ? int(blockIdx.x >> 1) : num_units)
                               : atomicAdd(p.status + 1, 1);
          F16Slot s = f16_make_slot<C>(p, unit, num_tiles, split_tiles, split_units);
          if (s.g != -1 && !f16_slot_in_range<C>(p, s)) {
            atomicCAS(p.status, 0, kStatusBadTile);
            s.g = -1;
          }
          if (!mbar_wait1<true>(schede_bar(slot), sphase ^ 1, abort_flag, p.status,
                                kStatusTimeoutProducer))
            break;
          const uint32_t words[8] = {uint32_t(s.g),    uint32_t(s.mt), uint32_t(s.row0),
                                     uint32_t(s.rows), uint32_t(s.ct), uint32_t(s.k0),
                                     uint32_t(s.k1),   s.split};
#pragma unroll
          for (int i = 0; i < (C::SPLIT ? 8 : 5); ++i) {
            reinterpret_cast<volatile uint32_t*>(ring + slot)[i] = words[i];
            st_shared_remote_u32(remote_ring0 + 32u * slot + 4u * i, words[i]);
          }
          mbar_arrive(schedf_bar(slot));
          mbar_arrive_remote(remote_schedf0 + 8u * slot);
          if (++slot == C::SCHED) {
            slot = 0;
            sphase ^= 1;
          }
          if (s.g < 0) break;
        }
      }
      __syncwarp();
    } else if (warp == 0) {
      // ------------------------------------------------- producer (both CTAs)
      int stage = 0;
      uint32_t phase = 0;
      int slot = 0;
      uint32_t sphase = 0;
      uint32_t arms = 0;
      uint32_t tiles_taken = 0;
      if (lane == 0) {
        if constexpr (C::MODE == kWgrad) {
          prefetch_tensormap(&p.tmap_a);
          prefetch_tensormap(&p.tmap_b);
        } else {
          prefetch_tensormap(&p.tmap_w);
          prefetch_tensormap(&p.tmap_tok[kTokenMaps - 1]);
        }
      }
      while (true) {
        if (!mbar_wait<true>(schedf_bar(slot), sphase, abort_flag, p.status,
                             kStatusTimeoutProducer))
          break;
        const int g = __shfl_sync(kFullMask, ring[slot].g, 0);
        const int mt = __shfl_sync(kFullMask, ring[slot].mt, 0);
        const int row0 = __shfl_sync(kFullMask, ring[slot].row0, 0);
        const int rows = __shfl_sync(kFullMask, ring[slot].rows, 0);
        const int ct = __shfl_sync(kFullMask, ring[slot].ct, 0);
        const int k0 = unit_k0(slot);
        const int k1 = unit_k1(slot, rows);
        if (lane == 0) {
          mbar_arrive(schede_bar(slot));
          if (leader) mbar_arrive(taken_bar(tiles_taken));
        }
        ++tiles_taken;
        if (++slot == C::SCHED) {
          slot = 0;
          sphase ^= 1;
        }
        if (g < 0) {
          if (lane == 0) griddep_launch_dependents();  // no new tiles for this CTA
          break;
        }
        const int half = tile_ncols(rows) >> 1;
        // bytes that both CTAs' loads of one step deliver to the leader's barrier
        const uint32_t tx_step = 2u * (C::A_BYTES + uint32_t(half) * 128u);
        const int flat_steps = C::MODE == kWgrad ? wgrad_flat_steps(rows) : k1;
        const int m0 = mt * 256 + int(rank) * 128;     // this CTA's rows of the M axis
        const int tok = row0 + int(rank) * half;       // forward, dgrad: its tokens
        const int c0 = ct * 256 + int(rank) * 128;     // wgrad: its columns k
        const CUtensorMap* const tb =
            C::MODE == kWgrad ? &p.tmap_b : &p.tmap_tok[half / 16 - 1];
        bool ok = true;
        for (int ks = k0; ks < k1; ++ks) {
          if (!mbar_wait(empty_bar(stage), phase ^ 1, abort_flag, p.status,
                         kStatusTimeoutProducer)) {
            ok = false;
            break;
          }
          const uint32_t fb = leader_full0 + 8u * stage;
          const int x = ks * C::KS;
          const bool arm = (p.debug_flags & kDebugNoLoads) == 0;
          if (arm && elect_one()) {
            // the copy of a group's last rows comes in boxes of 16 rows
            const bool tail = C::MODE == kWgrad && ks >= flat_steps;
            if (leader) mbar_arrive_expect_tx(full_bar(stage), tail ? tx_step / 4 : tx_step);
            if constexpr (C::MODE == kFwd) {
              tma_load_3d_pair(sA(stage), &p.tmap_w, fb, x, m0, g);
              tma_load_2d_pair(sB(stage), tb, fb, x, tok);
            } else if constexpr (C::MODE == kDgrad) {
              tma_load_3d_pair(sA(stage), &p.tmap_w, fb, m0, x, g);
              tma_load_3d_pair(sA(stage) + 8192u, &p.tmap_w, fb, m0 + 64, x, g);
              tma_load_2d_pair(sB(stage), tb, fb, x, tok);
            } else {
              const CUtensorMap* const ma = tail ? &p.tmap_ta : &p.tmap_a;
              const CUtensorMap* const mb = tail ? &p.tmap_tb : tb;
              const int y = tail ? 16 * g : row0 + x;
              tma_load_2d_pair(sA(stage), ma, fb, m0, y);
              tma_load_2d_pair(sA(stage) + 8192u, ma, fb, m0 + 64, y);
              tma_load_2d_pair(sB(stage), mb, fb, c0, y);
              tma_load_2d_pair(sB(stage) + 8192u, mb, fb, c0 + 64, y);
            }
          }
          __syncwarp();
          if (arm) ++arms;
          if (++stage == C::STAGES) {
            stage = 0;
            phase ^= 1;
          }
        }
        if (!ok) break;
      }
      // the leader's full barriers cover both CTAs' bytes: they land before exit
      if (leader && lane == 0) {
        const uint32_t first = arms > uint32_t(C::STAGES) ? arms - C::STAGES : 0u;
        for (uint32_t a = first; a < arms; ++a)
          mbar_wait_one(full_bar(int(a % C::STAGES)), (a / C::STAGES) & 1u, 200000000ull);
      }
      __syncwarp();
    } else if (warp == 1 && leader) {
      // ------------------------------------------------------- MMA issuer
      bool ok = mbar_wait(tmem_ready_bar, 0, abort_flag, p.status, kStatusTimeoutMma);
      tc_fence_after();
      const uint32_t tmem = __shfl_sync(kFullMask, *tmem_holder, 0);
      if (ok && !tmem_in_range(tmem, C::TMEM_COLS)) {
        give_up(p.status, abort_flag, kStatusBadTmem);
        ok = false;
      }
      int stage = 0;
      uint32_t phase = 0;
      int slot = 0;
      uint32_t sphase = 0;
      uint32_t lt = 0;
      bool issued_any = false;
      while (ok) {
        if (!mbar_wait<true>(schedf_bar(slot), sphase, abort_flag, p.status, kStatusTimeoutMma))
          break;
        const int g = __shfl_sync(kFullMask, ring[slot].g, 0);
        const int rows = __shfl_sync(kFullMask, ring[slot].rows, 0);
        const int k0 = unit_k0(slot);
        const int k1 = unit_k1(slot, rows);
        if (lane == 0) mbar_arrive(schede_bar(slot));
        if (++slot == C::SCHED) {
          slot = 0;
          sphase ^= 1;
        }
        if (g < 0) break;
        const int ncols = tile_ncols(rows);
        const uint32_t idesc =
            idesc_f16(p.bf16 ? 1u : 0u, C::A_MN ? 1u : 0u, C::B_MN ? 1u : 0u, 256, ncols);
        // an empty group's gradient (wgrad) is a chunk without steps
        int ks = k0;
        do {
          const int chunk0 = ks;
          const int chunk1 = min(k1 - chunk0, C::CHUNK) + chunk0;
          const uint32_t b = lt & 1u;
          if (!mbar_wait<true>(acce_bar(b), ((lt >> 1) & 1u) ^ 1u, abort_flag, p.status,
                               kStatusTimeoutMma)) {
            ok = false;
            break;
          }
          tc_fence_after();
          const uint32_t d_tmem = tmem + b * C::BN;
          for (; ks < chunk1; ++ks) {
            if (!mbar_wait(full_bar(stage), phase, abort_flag, p.status, kStatusTimeoutMma)) {
              ok = false;
              break;
            }
            tc_fence_after();
            const uint64_t adesc =
                C::A_MN ? desc_mn_sw128(sA(stage), 8192u) : desc_k_sw128(sA(stage));
            const uint64_t bdesc =
                C::B_MN ? desc_mn_sw128(sB(stage), 8192u) : desc_k_sw128(sB(stage));
            // 16 of the contraction: 32 bytes of a K-major row, 16 rows of an MN-major tile
            constexpr uint32_t kStepA = C::A_MN ? 2048u >> 4 : 32u >> 4;
            constexpr uint32_t kStepB = C::B_MN ? 2048u >> 4 : 32u >> 4;
            // wgrad: the whole sixteens of rows that this step holds; its last, the copy
            const int nj = C::MODE == kWgrad
                               ? (ks < wgrad_flat_steps(rows) ? min(4, rows / 16 - 4 * ks) : 1)
                               : 4;
            if (elect_one()) {
#pragma unroll
              for (int j = 0; j < 4; ++j)
                if (j < nj)
                  tc_mma_f16_pair(d_tmem, adesc + kStepA * j, bdesc + kStepB * j, idesc,
                                  ((ks - chunk0) | j) != 0 ? 1u : 0u);
              tc_commit_pair(empty_bar(stage), 0x3);
            }
            __syncwarp();
            issued_any = true;
            if (++stage == C::STAGES) {
              stage = 0;
              phase ^= 1;
            }
          }
          if (!ok) break;
          if (elect_one()) tc_commit_pair(accf_bar(b), 0x3);
          __syncwarp();
          issued_any = true;
          ++lt;
        } while (ks < k1);
      }
      if (issued_any) {
        if (elect_one()) {
          tc_commit_pair(drain_bar, 0x1);
          if (!mbar_wait_one(drain_bar, 0, 200000000ull))
            atomicCAS(p.status, 0, kStatusTimeoutDrain);
        }
      }
      __syncwarp();
    } else if (warp == 1) {
      // --------------------------------------- forwarder (follower only)
      // The leader writes this CTA's slots and its MMAs this CTA's accumulators, so
      // what frees them for it is released at cluster scope.  That waits for the
      // warp's global stores, so it is done by a warp that has none, once the
      // readers have arrived here: a tile's slot with its first accumulator.  The
      // last accumulator of the last tile nobody waits for; the slot after a tile's
      // is published once the producer has the tile.
      int slot = 0;
      uint32_t sphase = 0;
      uint32_t lt = 0;
      bool ok = mbar_wait<true>(schedf_bar(0), 0, abort_flag, p.status, kStatusTimeoutEpilogue);
      bool more = ok && __shfl_sync(kFullMask, ring[0].g, 0) >= 0;
      while (more) {
        const int rows = __shfl_sync(kFullMask, ring[slot].rows, 0);
        const int k0 = unit_k0(slot);
        const int k1 = unit_k1(slot, rows);
        const int next = slot + 1 == C::SCHED ? 0 : slot + 1;
        const uint32_t nphase = next == 0 ? sphase ^ 1u : sphase;
        ok = mbar_wait(schede_bar(slot), sphase, abort_flag, p.status, kStatusTimeoutEpilogue);
        for (int ks = k0; ok && more; ks += C::CHUNK) {  // the accumulators of the tile
          const uint32_t b = lt & 1u;
          ok = mbar_wait(acce_bar(b), (lt >> 1) & 1u, abort_flag, p.status, kStatusTimeoutEpilogue);
          const bool last = ks + C::CHUNK >= k1;
          if (ok && last) {
            ok = mbar_wait<true>(schedf_bar(next), nphase, abort_flag, p.status,
                                 kStatusTimeoutEpilogue);
            more = ok && __shfl_sync(kFullMask, ring[next].g, 0) >= 0;
          }
          if (!ok || !more) break;
          tc_fence_after();
          tc_fence_before();
          if (lane < (ks == k0 ? 2 : 1))
            mbar_arrive_remote(lane == 0 ? leader_acce0 + 8u * b : leader_schede0 + 8u * slot);
          ++lt;
          if (last) break;
        }
        more = more && ok;
        slot = next;
        sphase = nphase;
      }
      __syncwarp();
    }
  } else {
    // --------------------------------------------------------- epilogue
    if constexpr (C::MODE == kWgrad) regs_inc<C::REGS_EPI>();
    const int q = warp & 3, part = (warp - 4) >> 2;
    bool ok = mbar_wait(tmem_ready_bar, 0, abort_flag, p.status, kStatusTimeoutEpilogue);
    tc_fence_after();
    const uint32_t tmem = *tmem_holder;
    if (ok && !tmem_in_range(tmem, C::TMEM_COLS)) {
      give_up(p.status, abort_flag, kStatusBadTmem);
      ok = false;
    }
    int slot = 0;
    uint32_t sphase = 0;
    uint32_t lt = 0;
    // The next tile's slot (g < 0: none).  A tile takes it before it stores, as
    // the arrival that frees the slot would otherwise wait behind the stores.
    auto take = [&]() -> F16Slot {
      F16Slot t;
      t.g = -1;
      if (!mbar_wait<true>(schedf_bar(slot), sphase, abort_flag, p.status,
                           kStatusTimeoutEpilogue))
        return t;
      t = f16_read_slot(ring, slot);
      __syncwarp();
      if (lane == 0) mbar_arrive(schede_bar(slot));
      if (++slot == C::SCHED) {
        slot = 0;
        sphase ^= 1;
      }
      return t;
    };
    F16Slot next;
    next.g = -1;
    if (ok) next = take();
    while (ok && next.g >= 0) {
      const F16Slot s = next;
      const int m0 = s.mt * 256 + int(rank) * 128 + q * 32;
      auto release_acc = [&](uint32_t b) {  // this warp has read accumulator b
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(acce_bar(b));
      };
      if constexpr (C::MODE == kWgrad) {
        float acc[128];
#pragma unroll
        for (int j = 0; j < 128; ++j) acc[j] = 0.0f;
        const int k0 = C::SPLIT ? s.k0 : 0;
        const int k1 = C::SPLIT ? s.k1 : wgrad_steps(s.rows);
        int ks = k0;
        do {
          const uint32_t b = lt & 1u;
          if (!mbar_wait(accf_bar(b), (lt >> 1) & 1u, abort_flag, p.status,
                         kStatusTimeoutEpilogue)) {
            ok = false;
            break;
          }
          tc_fence_after();
          const uint32_t taddr = tmem + (uint32_t(q * 32) << 16) + b * C::BN + 128u * part;
          if (k1 > 0) {
#pragma unroll
            for (int c = 0; c < 8; ++c) {
              uint32_t r[16];
              tmem_ld16(taddr + 16 * c, r);
              tmem_wait_ld();
#pragma unroll
              for (int j = 0; j < 16; ++j) acc[16 * c + j] += __uint_as_float(r[j]);
            }
          }
          release_acc(b);
          ++lt;
          ks += C::CHUNK;
        } while (ks < k1);
        next = take();
        bool store = s.rows > 0 || !p.accumulate;
        if (C::SPLIT && (m0 >= p.m_ext || s.ct * 256 + 128 * part >= p.c_ext)) store = false;
        if (C::SPLIT && ok && s.split != 0) {
          F16Tree tree = f16_tree(p, s.split, int(rank) * C::EPI_WARPS + warp - 4);
          while (store && tree.next()) {
#pragma unroll
            for (int j = 0; j < 128; ++j) __stcg(tree.mine() + 32 * j, acc[j]);
            store = tree.arrive();
            if (store) {
#pragma unroll
              for (int j = 0; j < 128; j += 32) {
                float o[32];
#pragma unroll
                for (int i = 0; i < 32; ++i) o[i] = __ldcg(tree.other() + 32 * (j + i));
#pragma unroll
                for (int i = 0; i < 32; ++i) acc[j + i] += o[i];
              }
              tree.joined();
            }
          }
        }
        if (ok && store) {
          if (p.out_fp32)
            f16_store_wgrad<true>(p, s.g, m0, s.ct * 256 + 128 * part, acc);
          else
            f16_store_wgrad<false>(p, s.g, m0, s.ct * 256 + 128 * part, acc);
        }
      } else {
        const uint32_t b = lt & 1u;
        if (!mbar_wait(accf_bar(b), (lt >> 1) & 1u, abort_flag, p.status, kStatusTimeoutEpilogue))
          break;
        tc_fence_after();
        next = take();
        const uint32_t taddr = tmem + (uint32_t(q * 32) << 16) + b * C::BN;
        const int ncols = tile_ncols(s.rows);
        const int col = m0 + (lane & ~7);
        const F16Rows d = {static_cast<uint16_t*>(p.out) + col, size_t(s.row0), size_t(p.m_ext),
                           s.rows, col < p.m_ext, p.bf16 != 0};
        if (C::SPLIT && s.split != 0) {
          // blocks of 32 tokens as in f16_epilogue_rows, 1024 sums each
          F16Tree tree = f16_tree(p, s.split, int(rank) * C::EPI_WARPS + warp - 4);
          bool more = m0 < p.m_ext;
          if (more)
            for (int c0 = 32 * part, at = 0; c0 < ncols; c0 += 64, at += 1024) {
              uint32_t r[32];
              tmem_ld32(taddr + c0, r);
              tmem_wait_ld();
#pragma unroll
              for (int j = 0; j < 32; ++j)
                __stcg(tree.mine() + at + 32 * j, __uint_as_float(r[j]));
            }
          release_acc(b);
          while (more && tree.next() && (more = tree.arrive())) {
            const float* const lo = tree.mine();
            const float* const hi = tree.other();
            tree.joined();
            const bool top = !tree.next();
            for (int c0 = 32 * part, at = 0; c0 < ncols; c0 += 64, at += 1024) {
              uint32_t r[32], w[16];
              float o[32];
#pragma unroll
              for (int j = 0; j < 32; ++j) r[j] = __float_as_uint(__ldcg(lo + at + 32 * j));
#pragma unroll
              for (int j = 0; j < 32; ++j) o[j] = __ldcg(hi + at + 32 * j);
#pragma unroll
              for (int j = 0; j < 32; ++j)
                r[j] = __float_as_uint(__uint_as_float(r[j]) + o[j]);
              if (top) {
                f16_pack_block(r, d.bf16, w);
                f16_turn_block(d, c0, w);
              } else {
#pragma unroll
                for (int j = 0; j < 32; ++j)
                  __stcg(tree.mine() + at + 32 * j, __uint_as_float(r[j]));
              }
            }
          }
        } else {
          if (m0 < p.m_ext) f16_epilogue_rows(d, ncols, part, taddr);
          release_acc(b);
        }
        ++lt;
      }
    }
  }

  __syncthreads();
  // the leader's MMAs write the follower's TMEM and read its shared memory
  cluster_sync();
  if (warp == 2) {
    tc_fence_after();
    tmem_dealloc_pair(*tmem_holder, C::TMEM_COLS);
  }
}

// ---------------------------------------------------------------- prepare
struct F16PrepParams {
  const int32_t* offsets;
  const uint4* a;  // wgrad: dy, x in 16-byte vectors
  const uint4* b;
  uint4* tail_a;   // wgrad: the groups' last rows, 16 rows each
  uint4* tail_b;
  uint64_t* tiles;
  int32_t* tile_rows;
  int* status;
  int32_t vec_a, vec_b;  // wgrad: vectors per row
  int32_t num_groups, max_rows, mts, tile_cap;
  int32_t wgrad_tiles;  // wgrad: every group's tiles; 0 = forward, dgrad
  int32_t* order;       // wgrad: groups, the largest first
  uint32_t* units;      // split tiles'
  int32_t* arrived;
  int32_t split_pairs;  // the GPU's pairs; 0 = no tile of this problem is split
  int32_t ksteps;       // forward, dgrad: steps of the contraction
};

// Slices of a tile of `steps` steps whose call has a share of `total` / pairs for each
// pair.  At most 2^31 rows in steps of 64 (wgrad), 2^31 / 64 steps of a row (the
// others), 48 tiles and 96 pairs: products stay below 2^32.
__device__ __forceinline__ int f16_slices(uint32_t steps, uint32_t total, uint32_t pairs) {
  const uint32_t share = steps * pairs / max(total, 1u);
  if (share < 5 && steps < 4 * kMinSlice) return 1;
  return int(min(min(share, steps / kMinSlice), uint32_t(kMaxSlices)));
}

// Token tiles of a group of m rows: the fewest of at most 256 rows, of equal
// size up to a multiple of 32 (two of 160 and 140 for 300 rows, not 256 and 44:
// an MMA of 44 columns takes the time of 64).
__device__ __forceinline__ int f16_tile_count(int m) { return (m + 255) / 256; }
__device__ __forceinline__ int f16_tile_height(int m, int count) {
  return ((m + count - 1) / count + 31) & ~31;
}

// Every block ranks the groups by size (at most 512 of them; the largest go first,
// so that no long tile starts last) and scans their tile counts in shared memory,
// and writes its share of the tile list, group by group; or copies its share of
// the groups' last rows % 16 rows, with zeros up to 16 (wgrad).  Running the tiles of
// small groups, bound by their weights' stream, between those of large ones, bound
// by the tensor pipe, gained 2 % in dgrad (64 skewed groups) and is left out there:
// under the power cap their costs add up.  It was not tried in wgrad, where the cap
// binds less.
__global__ void __launch_bounds__(256) f16_prepare_kernel(const __grid_constant__ F16PrepParams p) {
  griddep_launch_dependents();
  griddep_wait();
  __shared__ int32_t soff[FGG_MAX_GROUPS + 1];
  __shared__ int32_t srows[FGG_MAX_GROUPS];
  __shared__ int32_t sorder[FGG_MAX_GROUPS];      // groups, the largest first
  __shared__ int32_t sbegin[FGG_MAX_GROUPS + 1];  // first tile (per M tile) in that order
  __shared__ int32_t swarp[8];
  __shared__ int s_bad;
  __shared__ int s_steps;  // wgrad: of all groups
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int G = p.num_groups;
  if (threadIdx.x == 0) s_bad = s_steps = 0;
  for (int i = threadIdx.x; i <= G; i += 256) soff[i] = p.offsets[i];
  if (p.split_pairs > 0 && blockIdx.x == 0)
    for (int i = threadIdx.x; i < kMaxSplitUnits * kWarpSums / 4; i += 256)
      reinterpret_cast<int4*>(p.arrived)[i] = make_int4(0, 0, 0, 0);
  __syncthreads();
  for (int g = threadIdx.x; g < G; g += 256) {
    const int lo = soff[g], hi = soff[g + 1];
    const bool bad = lo < 0 || hi < lo || hi > p.max_rows;
    srows[g] = bad ? 0 : hi - lo;
    if (bad) s_bad = 1;
    if (p.wgrad_tiles > 0 && p.split_pairs > 0 && !bad) atomicAdd(&s_steps, wgrad_steps(hi - lo));
  }
  __syncthreads();
  for (int g = threadIdx.x; g < G; g += 256) {
    const int m = srows[g];
    int rank = 0;
    for (int i = 0; i < G; ++i) {
      const int o = srows[i];
      rank += o > m || (o == m && i < g) ? 1 : 0;
    }
    sorder[rank] = g;
  }
  __syncthreads();
  // two positions per thread cover FGG_MAX_GROUPS
  static_assert(FGG_MAX_GROUPS <= 512, "two groups per thread");
  int cnt[2], run = 0;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int r = 2 * threadIdx.x + i;
    cnt[i] = r < G ? f16_tile_count(srows[sorder[r]]) : 0;
    run += cnt[i];
  }
  int incl = run;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int y = __shfl_up_sync(kFullMask, incl, o);
    if (lane >= o) incl += y;
  }
  if (lane == 31) swarp[warp] = incl;
  __syncthreads();
  int acc = incl - run;
  for (int w = 0; w < warp; ++w) acc += swarp[w];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int r = 2 * threadIdx.x + i;
    if (r <= G) sbegin[r] = acc;
    acc += cnt[i];
  }
  if (threadIdx.x == 255 && G == 512) sbegin[512] = acc;
  __syncthreads();
  int num_tiles = p.wgrad_tiles > 0 ? p.wgrad_tiles : sbegin[G] * p.mts;
  if (s_bad || num_tiles > p.tile_cap) num_tiles = 0;
  if (blockIdx.x == 0) {
    if (threadIdx.x == 0) {
      p.status[0] = s_bad ? kF16BadOffsets : 0;
      p.status[1] = 0;
      p.status[2] = 0;
      p.status[3] = num_tiles;
      // the longest tiles come first in the list, so that those to split lead it
      int tiles = 0, units = 0;
      const bool wgrad = p.wgrad_tiles > 0;
      const int per = wgrad ? p.wgrad_tiles / G : num_tiles;
      while (tiles < num_tiles && per <= p.split_pairs / 2) {
        const uint32_t steps = wgrad ? wgrad_steps(srows[sorder[tiles / per]]) : p.ksteps;
        const int slices =
            f16_slices(steps, (wgrad ? uint32_t(s_steps) : steps) * per, p.split_pairs);
        if (slices < 2) break;
        for (int t = 0; t < per; ++t) {
          for (int i = 0; i < slices; ++i) p.units[units + i] = split_word(tiles, i, slices, units);
          ++tiles;
          units += slices;
        }
      }
      p.status[4] = tiles;
      p.status[5] = units;
    }
    if (p.wgrad_tiles > 0)
      for (int r = threadIdx.x; r < G; r += 256) p.order[r] = sorder[r];
  }
  if (num_tiles == 0) return;
  if (p.wgrad_tiles > 0) {
    const int vecs = p.vec_a + p.vec_b;
    const int64_t total = int64_t(G) * 16 * vecs;
    for (int64_t i = int64_t(blockIdx.x) * 256 + threadIdx.x; i < total;
         i += int64_t(gridDim.x) * 256) {
      const int64_t r = i / vecs;
      const int c = int(i - r * vecs);
      const int g = int(r >> 4), row = int(r & 15);
      const int rest = (soff[g + 1] - soff[g]) & 15;
      if (rest == 0) continue;  // never read
      const bool is_a = c < p.vec_a;
      const int col = is_a ? c : c - p.vec_a;
      const int64_t pitch = is_a ? p.vec_a : p.vec_b;
      const int64_t src = int64_t(soff[g + 1] - rest + row);
      uint4 v = make_uint4(0u, 0u, 0u, 0u);
      if (row < rest) v = (is_a ? p.a : p.b)[src * pitch + col];
      (is_a ? p.tail_a : p.tail_b)[r * pitch + col] = v;
    }
    return;
  }
  for (int t = blockIdx.x * 256 + threadIdx.x; t < num_tiles; t += gridDim.x * 256) {
    // the group whose tiles (token tiles x mts) hold t
    int lo = 0, hi = G;
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (sbegin[mid] * p.mts <= t)
        lo = mid;
      else
        hi = mid;
    }
    const int g = sorder[lo];
    const int m = srows[g];
    const int count = sbegin[lo + 1] - sbegin[lo];
    const int height = f16_tile_height(m, count);
    const int local = t - sbegin[lo] * p.mts;
    int mt, xt;
    f16_place(local, p.mts, count, &mt, &xt);
    p.tiles[t] = (uint64_t(g) << 48) | (uint64_t(mt) << 32) | uint32_t(soff[g] + xt * height);
    p.tile_rows[t] = min(height, m - xt * height);
  }
}

// ------------------------------------------------------------------- host
struct F16Layout {
  int mts = 0, cts = 0, tile_cap = 0;
  size_t status = 0, order = 0, tiles = 0, tile_rows = 0, tail_a = 0, tail_b = 0, total = 0;
  size_t units = 0, arrived = 0, partial = 0;
  int max_slices = 1;  // of a tile
};

int plan_f16(const FggF16RowsProblem* p, int direction, F16Layout* L) {
  if (p == nullptr) return set_error(FGG_EINVAL, "problem is null");
  if (direction < kFwd || direction > kWgrad)
    return set_error(FGG_EINVAL, "direction=%d must be 0 (forward), 1 (dgrad) or 2 (wgrad)",
                     direction);
  const int G = p->num_groups;
  if (G < 1 || G > FGG_MAX_GROUPS)
    return set_error(FGG_EINVAL, "num_groups=%d outside [1, %d]", G, FGG_MAX_GROUPS);
  if (p->n < 8 || p->n % 8 != 0 || p->k < 8 || p->k % 8 != 0)
    return set_error(FGG_EBADSHAPE, "N=%d and K=%d must be positive multiples of 8", p->n, p->k);
  if (p->max_rows < 0) return set_error(FGG_EINVAL, "max_rows=%d is negative", p->max_rows);
  if (p->dtype != 1 && p->dtype != 2)
    return set_error(FGG_EINVAL, "dtype=%d must be 1 (bf16) or 2 (fp16)", p->dtype);
  if (p->out_dtype != p->dtype && !(direction == kWgrad && p->out_dtype == 0))
    return set_error(FGG_EINVAL, "out_dtype=%d must be the operands' type%s", p->out_dtype,
                     direction == kWgrad ? " or 0 (fp32)" : "");
  if (p->accumulate != 0 && (direction != kWgrad || p->out_dtype != 0))
    return set_error(FGG_EINVAL, "accumulate needs a weight gradient in fp32");
  const int m_ext = direction == kDgrad ? p->k : p->n;
  L->mts = (m_ext + 255) / 256;
  L->cts = (p->k + 255) / 256;
  if (L->mts > 0xFFFF) return set_error(FGG_EBADSHAPE, "N=%d or K=%d too large", p->n, p->k);
  Carver cv;
  L->status = cv.take(kStatusBytes, 256);
  int64_t cap;
  if (direction == kWgrad) {
    cap = int64_t(G) * L->mts * L->cts;
    L->order = cv.take(size_t(G) * 4, 256);
    L->tail_a = cv.take(size_t(G) * 16 * size_t(p->n) * 2, 256);
    L->tail_b = cv.take(size_t(G) * 16 * size_t(p->k) * 2, 256);
  } else {
    // sum over groups of ceil(m / 256) <= rows / 256 + groups (and <= rows)
    cap = std::min<int64_t>(int64_t(p->max_rows) / 256 + G, p->max_rows) * L->mts;
    L->tiles = cv.take(size_t(std::max<int64_t>(cap, 1)) * 8, 256);
    L->tile_rows = cv.take(size_t(std::max<int64_t>(cap, 1)) * 4, 256);
  }
  // the tile counter runs past the last tile by one claim per pair
  if (cap > INT32_MAX - 4096) return set_error(FGG_EBADSHAPE, "problem too large");
  L->tile_cap = int(cap);
  // The fewest tiles of a call are those of one group, in wgrad with all the rows; more
  // than half as many as pairs, or short ones, are never split.
  const int least = direction == kWgrad ? L->mts * L->cts : L->mts;
  const int64_t steps = direction == kWgrad ? int64_t(p->max_rows) / 64 + 2
                                            : ((direction == kFwd ? p->k : p->n) + 63) / 64;
  if (least * 2 <= kMaxSplitUnits)
    L->max_slices = int(std::max<int64_t>(1, std::min<int64_t>(steps / kMinSlice, kMaxSlices)));
  if (L->max_slices > 1) {
    L->units = cv.take(kMaxSplitUnits * 4, 256);
    L->arrived = cv.take(kMaxSplitUnits * kWarpSums * 4, 256);
    const int64_t units = std::min<int64_t>(cap * L->max_slices, kMaxSplitUnits);
    L->partial = cv.take(size_t(units) * kUnitFloats * 4, 256);
  }
  L->total = cv.off;
  return FGG_OK;
}

constexpr CUtensorMapDataType kMap16 = CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;  // moved as bits

template <int MODE, bool SPLIT>
int launch_f16(const F16Params& gp, const DeviceInfo& dev, cudaStream_t s) {
  using C = F16Cfg<MODE, SPLIT>;
  if (int rc = ensure_max_dynamic_smem(reinterpret_cast<const void*>(f16_pair_kernel<C>),
                                       int(C::SMEM_BYTES)))
    return rc;
  if constexpr (MODE == kWgrad) {
    // a split of more registers than the block starts with would never be granted
    static std::atomic<int> known{0};
    int regs = known.load(std::memory_order_relaxed);
    if (regs == 0) {
      cudaFuncAttributes a = {};
      FGG_CUDA_CHECK(cudaFuncGetAttributes(&a, f16_pair_kernel<C>));
      regs = a.numRegs;
      known.store(regs, std::memory_order_relaxed);
    }
    if (regs * C::THREADS < C::REGS_TOTAL)
      return set_error(FGG_ECUDA, "the kernel was built with %d registers per thread, needs %d",
                       regs, (C::REGS_TOTAL + C::THREADS - 1) / C::THREADS);
  }
  const int pairs = std::max(1, std::min(gp.grid_units, dev.sm_count / 2));
  const cudaError_t e = launch_pdl(f16_pair_kernel<C>, dim3(2 * pairs), dim3(C::THREADS),
                                   C::SMEM_BYTES, s, gp);
  if (e != cudaSuccess) return set_error(FGG_ECUDA, "GEMM launch failed: %s", cudaGetErrorString(e));
  return FGG_OK;
}

}  // namespace
}  // namespace fgg

using namespace fgg;

extern "C" {

size_t fgg_f16_rows_workspace_bytes(const FggF16RowsProblem* p, int32_t direction) {
  F16Layout L;
  if (plan_f16(p, direction, &L) != FGG_OK) return 0;
  return L.total;
}

int fgg_f16_grouped_gemm_rows(const FggF16RowsProblem* p, int32_t direction, void* workspace,
                              size_t ws_bytes, void* stream) {
  F16Layout L;
  if (int rc = plan_f16(p, direction, &L)) return rc;
  if (workspace == nullptr) return set_error(FGG_EINVAL, "workspace is null");
  if ((reinterpret_cast<uintptr_t>(workspace) & 127u) != 0)
    return set_error(FGG_EALIGN, "workspace must be 128-byte aligned");
  if (ws_bytes < L.total)
    return set_error(FGG_EWORKSPACE, "workspace has %zu bytes, needs %zu", ws_bytes, L.total);
  if (p->offsets == nullptr || p->out == nullptr) {
    // without rows the token tensors may be null, and so may an empty output
    if (p->offsets == nullptr || direction == kWgrad || p->max_rows > 0)
      return set_error(FGG_EINVAL, "offsets / out is null");
  }
  if (p->max_rows > 0 && (p->a == nullptr || p->b == nullptr))
    return set_error(FGG_EINVAL, "a / b is null");
  if (!aligned16(p->a) || !aligned16(p->b) || !aligned16(p->out))
    return set_error(FGG_EALIGN, "a, b and out must be 16-byte aligned");
  if (!aligned4(p->offsets)) return set_error(FGG_EALIGN, "offsets must be 4-byte aligned");
  DeviceInfo dev;
  if (int rc = current_device(&dev)) return rc;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  const uint64_t G = uint64_t(p->num_groups), N = uint64_t(p->n), K = uint64_t(p->k);
  const uint64_t R = uint64_t(p->max_rows);

  F16PrepParams pp;
  memset(&pp, 0, sizeof(pp));
  F16Params gp;
  memset(&gp, 0, sizeof(gp));
  pp.offsets = gp.offsets = p->offsets;
  pp.status = gp.status = reinterpret_cast<int*>(ws + L.status);
  pp.num_groups = gp.num_groups = p->num_groups;
  pp.max_rows = p->max_rows;
  pp.mts = gp.mts = L.mts;
  gp.max_rows = p->max_rows;
  gp.cts = L.cts;
  pp.tile_cap = L.tile_cap;
  gp.grid_units = int(std::min<int64_t>(int64_t(L.tile_cap) * L.max_slices, INT32_MAX));
  gp.bf16 = p->dtype == 1 ? 1 : 0;
  gp.out = p->out;
  gp.debug_flags = debug_flags();
  if (L.max_slices > 1) {
    pp.units = reinterpret_cast<uint32_t*>(ws + L.units);
    pp.arrived = reinterpret_cast<int32_t*>(ws + L.arrived);
    // all of the GPU's pairs: a tile's slices are at most max_slices whatever its share, so
    // that the units stay within grid_units and `partial`
    pp.split_pairs = std::min(dev.sm_count / 2, kMaxSplitUnits);
    gp.units = pp.units;
    gp.arrived = pp.arrived;
    gp.partial = reinterpret_cast<float*>(ws + L.partial);
  }
  int blocks;
  if (direction == kWgrad) {
    pp.a = static_cast<const uint4*>(p->a);
    pp.b = static_cast<const uint4*>(p->b);
    pp.tail_a = reinterpret_cast<uint4*>(ws + L.tail_a);
    pp.tail_b = reinterpret_cast<uint4*>(ws + L.tail_b);
    pp.vec_a = p->n / 8;
    pp.vec_b = p->k / 8;
    // (without rows the token tensors may be null, and no step reads them)
    const void* const a = R > 0 ? p->a : pp.tail_a;
    const void* const b = R > 0 ? p->b : pp.tail_b;
    const uint64_t rows = R > 0 ? R : 16 * G;
    if (int rc = encode_2d(&gp.tmap_a, kMap16, a, N, rows, N * 2, 64, 64)) return rc;
    if (int rc = encode_2d(&gp.tmap_b, kMap16, b, K, rows, K * 2, 64, 64)) return rc;
    if (int rc = encode_2d(&gp.tmap_ta, kMap16, pp.tail_a, N, 16 * G, N * 2, 64, 16)) return rc;
    if (int rc = encode_2d(&gp.tmap_tb, kMap16, pp.tail_b, K, 16 * G, K * 2, 64, 16)) return rc;
    pp.wgrad_tiles = L.tile_cap;
    pp.order = reinterpret_cast<int32_t*>(ws + L.order);
    gp.order = pp.order;
    gp.m_ext = p->n;
    gp.c_ext = p->k;
    gp.out_fp32 = p->out_dtype == 0 ? 1 : 0;
    gp.accumulate = p->accumulate != 0 ? 1 : 0;
    const int64_t vecs = int64_t(p->num_groups) * 16 * (pp.vec_a + pp.vec_b);
    blocks = int(std::min<int64_t>((vecs + 255) / 256, 8 * dev.sm_count));
  } else {
    const uint64_t ck = direction == kFwd ? K : N;  // contraction: the tokens' row length
    pp.tiles = reinterpret_cast<uint64_t*>(ws + L.tiles);
    pp.tile_rows = reinterpret_cast<int32_t*>(ws + L.tile_rows);
    pp.ksteps = int((ck + 63) / 64);
    if (R == 0) {  // no tile, but the offsets are looked at
      FGG_CUDA_CHECK(launch_dependent(f16_prepare_kernel, 1, 0, s, pp));
      return FGG_OK;
    }
    if (int rc = encode_3d(&gp.tmap_w, kMap16, p->b, K, N, G, K * 2, N * K * 2, 64,
                           direction == kFwd ? 128 : 64, 1))
      return rc;
    for (int i = 0; i < kTokenMaps; ++i)
      if (int rc = encode_2d(&gp.tmap_tok[i], kMap16, p->a, ck, R, ck * 2, 64,
                             uint32_t(16 * (i + 1))))
        return rc;
    gp.tiles = pp.tiles;
    gp.tile_rows = pp.tile_rows;
    gp.m_ext = direction == kFwd ? p->n : p->k;
    gp.ksteps = pp.ksteps;
    blocks = std::min((L.tile_cap + 255) / 256, dev.sm_count);
  }
  FGG_CUDA_CHECK(launch_dependent(f16_prepare_kernel, std::max(blocks, 1), 0, s, pp));
  const bool split = L.max_slices > 1;
  if (direction == kFwd)
    return split ? launch_f16<kFwd, true>(gp, dev, s) : launch_f16<kFwd, false>(gp, dev, s);
  if (direction == kDgrad)
    return split ? launch_f16<kDgrad, true>(gp, dev, s) : launch_f16<kDgrad, false>(gp, dev, s);
  return split ? launch_f16<kWgrad, true>(gp, dev, s) : launch_f16<kWgrad, false>(gp, dev, s);
}

}  // extern "C"
