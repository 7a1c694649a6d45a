// Products of rows grouped by expert in 8-bit floating point, with a scale for each 128 values of a row and
// each 128 x 128 of the weights, on CTA pairs (tcgen05 cta_group::2, kind::f8f6f4).
//
//   product  y[r, c] = sum over blocks b of 128 k's of  sx[r, b] sw_e[c / 128, b] sum_{k in b} xq[r, k] wq_e[c, k]
//            (+ bias[e, c])                                            for the rows r of group e
//   gated    h[r, f] = act(y[r, f]) y[r, hidden + f], which leaves as 8-bit values with scales of their own
//
// A block of K is a stage: its products go to a fresh accumulator, and the epilogue adds that, times its scale, to
// sums in registers while the tensor core fills the other.  Tensor memory holds two accumulators of 256 columns.  What
// bounds a long product is the way round: the products of a stage take 512 cycles, their end is known 180 cycles
// later, an epilogue warp takes 400 to 500 to add 128 columns up (two warps share a scheduler, and 256 of them are
// multiply-adds), and it is another 200 until the leader knows that both CTAs have, the one's word to the other going
// through the cluster.  So with two accumulators a stage takes 855 to 880 cycles.  That is not all of it: with 128 columns,
// whose products take half as long and whose four accumulators leave time for the way round, a stage still takes 700 to 720,
// on half of the pairs as on all of them, so some 550 cycles depend on neither width nor accumulators.  Which role's chain they
// are has not been measured.  8192^3 takes 474 to 530 us over a few dozen calls (2.1 to 2.3 PFLOP/s) and 548 (2.0) where they
// go on for half a second and the power cap leaves 1.25 GHz.  (As two accumulators of 128 columns each, with products and
// barriers of their own, it took 579 instead of 485.)  Behind the last
// stage of a tile come 2500 cycles, gated 5000 (of which 2700 for the activation: two special-function instructions for
// each of 64 values), in which the tensor core does the next tile's first two stages.
//
// Which side is which.  Rows of x are the lanes of tensor memory and output features its columns, the other way
// round than in grouped_gemm.cu.  So a thread has a row, and a stage has one scale for it, its own times the one of
// the 128 features that its warp holds: a register, where scales that differ from column to column would have
// to come from shared memory, whose port the operands need.  What it costs: a group's last 256 lanes are not all
// rows.  Where groups have few rows the weights' way from memory is the longer one anyway (a stage of 256 features
// is 32 KB, which memory gives a pair in 700 cycles).  Warps without rows read nothing, nor are rows loaded that
// no lane needs.
//
// Gated: a CTA loads rows of the gate and the same ones of the projection it gates, so that the columns of an
// epilogue warp are half the one and half the other, and a thread has both for its features; two warps
// share the largest magnitude of 128 features.
//
// Tiles take equal time, so they are dealt to the pairs in turn.  A launch with few tiles cuts them into slices of
// K, whose sums are parked and added in order by the warp that is the last to come.
//
// Barriers ("leader" = cluster rank 0):
//   full[s]       leader's only: 2 arrivals, one from each CTA's producer, and the bytes of both CTAs' loads
//   empty[s]      in both CTAs: commit multicast from the leader
//   acc_full[b]   in both CTAs: commit multicast
//   acc_empty[b]  leader's only: one arrival from each epilogue warp of both CTAs
//   tile_full[i]  own: 1 arrival, from the warp that works out the tiles
//   tile_empty[i] own: 1 arrival from each role that took the tile
//   sc_full[b]    own: 32 arrivals, of the copies of each lane of the warp that fetches scales
//   sc_empty[b]   own: one arrival from each epilogue warp
//   pair[q]       own, gated: 2 arrivals, one from each epilogue warp that has quarter q of the lanes
// Every wait is bounded; no TMA multicast is used.
#include "activation.cuh"
#include "block_scale.cuh"
#include "f8_common.cuh"
#include "gemm_common.cuh"
#include "grouped.hpp"
#include "ptx.cuh"

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <mutex>
#include <type_traits>

namespace cumpsgemm_b200 {
namespace {

constexpr uint32_t ROWS_CTA = 128, ROWS = 2 * ROWS_CTA; // lanes of a CTA and of a pair
constexpr uint32_t COLS = 256;                          // most columns of a tile
constexpr uint32_t WIDTHS = 2;                          // that a launch chooses from: 256, 128
constexpr uint32_t BLOCK = 128;                         // of K, in values and in bytes
constexpr uint32_t BOX_ROWS = 32;                       // of the smaller boxes
constexpr uint32_t TILE_BYTES = ROWS_CTA * BLOCK;       // an operand's part of a stage in one CTA
constexpr uint32_t STAGE_BYTES = 2 * TILE_BYTES;
constexpr uint32_t TMEM_COLS = 512;
constexpr uint32_t MOST_SLOTS = 4;      // accumulators, of TMEM_COLS / slots columns
__device__ __forceinline__ uint32_t slots_of(uint32_t width) { return width > 128 ? 2u : MOST_SLOTS; }
constexpr uint32_t BAND = 8;        // row tiles that are walked together
constexpr uint32_t MAX_SLICES = 16;
constexpr uint32_t MIN_SLICE = 4;   // least blocks of K in a slice
constexpr uint32_t PART = COLS * ROWS_CTA; // elements of a parked sum of one CTA
constexpr uint32_t JOIN_AHEAD = 8;  // slices whose sums are fetched together
constexpr uint32_t AT_ONCE = 4;     // blocks of K whose scales are copied together, into two buffers in turn
constexpr uint32_t SCALE_WORDS = ROWS_CTA + 4; // of a block: the rows', then two of the weights'
constexpr uint32_t AHEAD = 3;       // tiles that the roles may be apart
// Two epilogue warps share the 256 columns of 32 lanes.  (With four of 64 columns 8192 x 8192 x 8192 took 598 us where
// these took 565, and the gated product of 32764 rows x 2048 x 2 x 4096 takes 726 where these take 643: a stage costs a
// warp what it costs with half as many columns, and twice as many warps want to issue.)  The four warps that
// issue give back registers that the epilogue's take.
constexpr uint32_t PARTS = 2, MOST = COLS / PARTS; // most columns of a warp
constexpr uint32_t READ = 16;                      // that it reads at a time
constexpr int EPI_WARPS = 4 * PARTS, THREADS = 128 + 32 * EPI_WARPS;
constexpr int REGS_LAUNCH = 168, REGS_REST = 64, REGS_EPI = 216;
static_assert(128 * REGS_REST + 32 * EPI_WARPS * REGS_EPI <= THREADS * REGS_LAUNCH, "setmaxnreg draws on the launch's registers");

constexpr uint32_t MOST_STAGES = 6, FULL = 0, EMPTY = FULL + 8 * MOST_STAGES, ACC_FULL = EMPTY + 8 * MOST_STAGES,
                   ACC_EMPTY = ACC_FULL + 8 * MOST_SLOTS, TILE_FULL = ACC_EMPTY + 8 * MOST_SLOTS, TILE_EMPTY = TILE_FULL + 8 * AHEAD,
                   SC_FULL = TILE_EMPTY + 8 * AHEAD, SC_EMPTY = SC_FULL + 16,
                   PAIR = SC_EMPTY + 16, // gated, for each quarter of the lanes
                   LAST = PAIR + 8 * 4, TMEM_PTR = LAST + 4 * 4, ABORT = TMEM_PTR + 4, WIDTH = ABORT + 4,
                   TILE = 320,                       // the tiles of the roles
                   TOPS = TILE + AHEAD * 48,         // gated: largest magnitudes, [tile's parity][part][lane]
                   START = TOPS + 2 * PARTS * ROWS_CTA * 4, FIRST_TILE = START + 4 * (kMaxGroups + 2),
                   SCALE = (FIRST_TILE + 4 * (kMaxGroups + 2) + 127) / 128 * 128,
                   OUT = (SCALE + 2 * AT_ONCE * SCALE_WORDS * 4 + 1023) / 1024 * 1024;
static_assert(PAIR % 8 == 0 && WIDTH + 4 <= TILE && TILE % 16 == 0 && OUT % 16 == 0, "barriers and flags");
// What a warp's results take on their way out, 64 bytes of each of its rows (gated) or 256; the stages take the rest.
constexpr uint32_t OUT_ROW = 256, OUT_BOX = 128, OUT_PITCH = OUT_ROW + 16; // of a row; of it in a box; of rows that leave one by one
template <bool GATED> struct Shared {
  static constexpr uint32_t STAGES = GATED ? 6 : 4, OUT_BYTES = GATED ? 32 * 64 : (32 * OUT_PITCH + 1023) / 1024 * 1024,
                            FIRST = OUT + EPI_WARPS * OUT_BYTES,
                            BYTES = FIRST + STAGES * STAGE_BYTES + 1024; // and what the alignment takes
  static_assert(STAGES <= MOST_STAGES && FIRST % 1024 == 0 && BYTES <= 232448, "shared memory of a CTA");
};

struct F8Params {
  const int32_t *ends;
  void *out; // gated: the 8-bit values
  uint64_t ldo;
  const float *x_scale;
  uint64_t x_scale_row, x_scale_block;
  const float *w_scale; // [groups][blocks of w's rows][blocks of K]
  const float *bias;    // nullable; gated: none
  float *out_scale;     // gated
  uint64_t out_scale_row, out_scale_block;
  float *parts; // nullable: sums of slices, [slot][CTA rank][COLS][ROWS_CTA]
  unsigned *counters;
  int *status;
  uint32_t rows, groups, n, blocks; // n: features of the result
  uint32_t idesc;
  uint16_t out_type; // gated: F8Type
  uint8_t activation;
  uint8_t vector_out; // rows of the result allow 16-byte accesses
};

// A tile, or a slice of one: `rows` rows from row0 on, features from col0 on, blocks [k0, k0 + blocks) of K.
struct alignas(16) Tile {
  uint32_t group, row0, rows, col0; // rows == 0: there are no more tiles
  uint32_t k0, blocks, slices, slice;
  uint32_t slot, number, pad0, pad1;
};
static_assert(sizeof(Tile) == 48, "three times 16 bytes");

// What a launch is expected to take, in cycles: a stage of a tile `width` columns wide (38 or 72 tiles, operands in L2, by
// the slope over K: 855 to 880 with 256 columns, 700 to 720 with 128; the line is some 4 % below both, and only which of two
// launches is the shorter counts), and the join of slices, which passes over the columns of a warp.
__device__ __forceinline__ float stage_cycles(uint32_t width) { return 560.f + width; }
__device__ __forceinline__ float join_cycles(uint32_t width, uint32_t slices) {
  return slices > 1 ? 4000.f + width * (30.f + 4.f * slices) : 0.f;
}
// Slices of K that tiles are cut into, where there are at most half as many as pairs: as many as make the sum of both
// least, if that is less than a whole tile.
__device__ __forceinline__ uint32_t slices_of(const F8Params &p, uint32_t tiles, uint32_t clusters, uint32_t width) {
  if (p.parts == nullptr || tiles == 0 || tiles > clusters / 2) return 1;
  const uint32_t most = min(min(clusters / tiles, p.blocks / MIN_SLICE), MAX_SLICES);
  const uint32_t cut = max(1u, min(most, static_cast<uint32_t>(sqrtf(p.blocks * stage_cycles(width) / (4.f * width)))));
  return (p.blocks - (p.blocks + cut - 1) / cut) * stage_cycles(width) > join_cycles(width, cut) ? cut : 1u;
}

// The items of a launch, which are tiles or slices of tiles, by their numbers: groups in turn; within one, bands
// of row tiles that all column tiles pass over, so that what runs at the same time shares operands in L2.
template <bool GATED> struct Items {
  uint32_t sbase, group, total, slices, cols;
  __device__ __forceinline__ Items(uint32_t sbase_, const F8Params &p, uint32_t clusters) : sbase(sbase_), group(0) {
    cols = ld_shared_one<uint32_t>(sbase + WIDTH);
    const uint32_t tiles = first_tile(p.groups + 1);
    slices = slices_of(p, tiles, clusters, cols);
    total = tiles * slices;
  }
  __device__ __forceinline__ uint32_t start(uint32_t g) const { return ld_shared_one<uint32_t>(sbase + START + 4 * g); }
  __device__ __forceinline__ uint32_t first_tile(uint32_t g) const { return ld_shared_one<uint32_t>(sbase + FIRST_TILE + 4 * g); }
  // item < total, and not below that of an earlier call; false: it is none (a tile of zeros has one slice)
  __device__ __forceinline__ bool get(const F8Params &p, uint32_t item, Tile &x) {
    x.number = slices > 1 ? item / slices : item;
    x.slot = item;
    while (x.number >= first_tile(group + 1)) ++group;
    const uint32_t features = GATED ? cols / 2 : cols; // of the result, in a tile
    const uint32_t r0 = start(group), r = start(group + 1) - r0;
    const uint32_t row_tiles = (r + ROWS - 1) / ROWS, col_tiles = (p.n + features - 1) / features;
    const uint32_t local = x.number - first_tile(group);
    const uint32_t band = local / (BAND * col_tiles), in_band = local - band * BAND * col_tiles;
    const uint32_t height = min(BAND, row_tiles - band * BAND);
    const uint32_t ct = in_band / height, rt = band * BAND + (in_band - ct * height);
    x.group = group;
    x.row0 = r0 + rt * ROWS;
    x.rows = min(ROWS, r - rt * ROWS);
    x.col0 = ct * features;
    x.slices = group < p.groups ? slices : 1u;
    x.slice = slices > 1 ? item - x.number * slices : 0u;
    if (x.slice >= x.slices) return false;
    const uint32_t all = group < p.groups ? p.blocks : 0u;
    x.k0 = all * x.slice / x.slices;
    x.blocks = all * (x.slice + 1) / x.slices - x.k0;
    return true;
  }
};

// The tiles a role takes, as a warp of its CTA works them out: a handful of divisions, 500 cycles.
template <bool WARP> struct Tiles { // taken by a warp, or by one thread
  uint32_t sbase, turn, phase;
  __device__ __forceinline__ explicit Tiles(uint32_t sbase_) : sbase(sbase_), turn(0), phase(0) {}
  // the next tile is there; false: the wait gave up
  __device__ __forceinline__ bool wait(int *status) const {
    const bool ok = ptx::mbar_wait_s(sbase + TILE_FULL + 8 * turn, phase, sbase + ABORT, status, ptx::kErrWaitTile);
    return WARP ? ptx::warp_agrees(ok) : ok;
  }
  __device__ __forceinline__ uint32_t advance() { // returns the turn it was
    const uint32_t was = turn;
    if (++turn == AHEAD) {
      turn = 0;
      phase ^= 1u;
    }
    return was;
  }
  __device__ __forceinline__ void read(uint32_t at, Tile &x) const {
    const uint4 a = ld_shared(sbase + TILE + 48 * at), b = ld_shared(sbase + TILE + 48 * at + 16),
                c = ld_shared(sbase + TILE + 48 * at + 32);
    x.group = a.x, x.row0 = a.y, x.rows = a.z, x.col0 = a.w;
    x.k0 = b.x, x.blocks = b.y, x.slices = b.z, x.slice = b.w;
    x.slot = c.x, x.number = c.y;
  }
  // by all of the warp, or the thread, when what was read has come (its words have been used)
  __device__ __forceinline__ void give_back(uint32_t at) const {
    if (WARP) __syncwarp();
    if (!WARP || (threadIdx.x & 31u) == 0) ptx::mbar_arrive(sbase + TILE_EMPTY + 8 * at);
  }
  // one thread: the next tile; false at the end, or where the wait gave up
  __device__ __forceinline__ bool next(int *status, Tile &x) {
    if (!wait(status)) return false;
    const uint32_t at = advance();
    read(at, x);
    give_back(at); // (a release: the reads are in front of it)
    return x.rows != 0;
  }
};

// First row and first tile of each group, and the width of the tiles, by one warp.  What `ends` holds is never
// trusted: a total that falls back or passes the number of rows is taken as the one in front of it, or as
// that number.  The rows behind the last group are a group of their own, whose tiles have no blocks.
template <bool GATED>
__device__ __forceinline__ void find_groups(uint8_t *smem, const F8Params &p, uint32_t clusters) {
  uint32_t *start = reinterpret_cast<uint32_t *>(smem + START);
  uint32_t *first_tile = reinterpret_cast<uint32_t *>(smem + FIRST_TILE);
  const uint32_t lane = threadIdx.x & 31u;
  uint32_t end_before = 0, row_tiles = 0; // row tiles in front
  for (uint32_t g0 = 0; g0 < p.groups + 1; g0 += 32) {
    const uint32_t g = g0 + lane;
    uint32_t end = 0;
    if (g < p.groups)
      end = p.ends == nullptr ? p.rows
                              : static_cast<uint32_t>(min(max(__ldg(p.ends + g), 0), static_cast<int32_t>(p.rows)));
    else if (g == p.groups) end = p.rows;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const uint32_t o = __shfl_up_sync(0xffffffffu, end, d);
      if (static_cast<int>(lane) >= d) end = max(end, o);
    }
    end = max(end, end_before);
    uint32_t begin = __shfl_up_sync(0xffffffffu, end, 1);
    if (lane == 0) begin = end_before;
    uint32_t upto = g <= p.groups ? (end - begin + ROWS - 1) / ROWS : 0u;
    const uint32_t mine = upto;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const uint32_t o = __shfl_up_sync(0xffffffffu, upto, d);
      if (static_cast<int>(lane) >= d) upto += o;
    }
    if (g <= p.groups) {
      start[g] = begin;
      first_tile[g] = row_tiles + upto - mine;
    }
    if (g == p.groups) start[g + 1] = end;
    end_before = __shfl_sync(0xffffffffu, end, 31);
    row_tiles += __shfl_sync(0xffffffffu, upto, 31);
  }
  // The width.  With many tiles, the widest.  Else the one with the earliest end: waves of tiles (or slices), with 6000
  // cycles for what a tile takes besides its stages (3000 and 4500 chose the same for eleven shapes of 1000 to 8000 rows).
  uint32_t cols = COLS;
  if constexpr (!GATED) { // (a gated tile has a whole block of 128 features)
    if (row_tiles * ((p.n + COLS - 1) / COLS) < 4 * clusters) {
      float best = 0.f;
#pragma unroll
      for (uint32_t i = 0; i < WIDTHS; ++i) {
        const uint32_t w = COLS >> i, tiles = row_tiles * ((p.n + w - 1) / w), cut = slices_of(p, tiles, clusters, w),
                       waves = (tiles * cut + clusters - 1) / clusters, blocks = (p.blocks + cut - 1) / cut;
        const float ends_at = waves * (blocks * stage_cycles(w) + 6000.f) + join_cycles(w, cut);
        if (i == 0 || ends_at < 0.95f * best) {
          best = ends_at;
          cols = w;
        }
      }
    }
  }
  const uint32_t features = GATED ? cols / 2 : cols, col_tiles = (p.n + features - 1) / features;
  for (uint32_t g = lane; g <= p.groups; g += 32) first_tile[g] *= col_tiles;
  if (lane == 0) {
    first_tile[p.groups + 1] = row_tiles * col_tiles;
    *reinterpret_cast<uint32_t *>(smem + WIDTH) = cols;
  }
}

__device__ __forceinline__ void read_columns(uint32_t taddr, uint32_t (&v)[16]) { ptx::tmem_ld_32x32b_x16(taddr, v); }
__device__ __forceinline__ void read_columns(uint32_t taddr, uint32_t (&v)[32]) { ptx::tmem_ld_32x32b_x32(taddr, v); }

// sums += scale * COLUMNS columns from taddr on; the next are on their way while these are added.  Gated: the second
// half of the columns has a scale of its own.
template <bool GATED, uint32_t COLUMNS>
__device__ __forceinline__ void drain(uint32_t taddr, float (&sums)[MOST], float s0, float s1) {
  uint32_t x[2][READ];
  read_columns(taddr, x[0]);
#pragma unroll
  for (uint32_t c = 0; c < COLUMNS; c += READ) {
    ptx::tmem_ld_wait();
    if (c + READ < COLUMNS) read_columns(taddr + c + READ, x[(c / READ + 1) & 1]);
    const float s = GATED && c >= COLUMNS / 2 ? s1 : s0;
#pragma unroll
    for (uint32_t i = 0; i < READ; ++i) sums[c + i] = fmaf(__uint_as_float(x[(c / READ) & 1][i]), s, sums[c + i]);
  }
}

__device__ __forceinline__ void arrive_cluster_relaxed_if(bool yes, uint32_t cluster_addr) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %1, 0;\n\t"
      "@p mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];\n\t}\n" ::"r"(cluster_addr),
      "r"(static_cast<uint32_t>(yes))
      : "memory");
}

// the way back
__device__ __forceinline__ void put_back(uint32_t taddr, const float (&sums)[MOST], uint32_t cols) {
#pragma unroll
  for (uint32_t c = 0; c < MOST; c += 16) {
    if (c >= cols) break;
    uint32_t v[16];
#pragma unroll
    for (uint32_t i = 0; i < 16; ++i) v[i] = __float_as_uint(sums[c + i]);
    ptx::tmem_st_32x32b_x16(taddr + c, v);
  }
  ptx::tmem_st_wait();
}

// `cols` columns of a slice's sums (a multiple of 16) are parked, column c of the warp at c * ROWS_CTA, for whoever
// is the last of the tile's slices to do so and counts up to their number.  Nothing waits.
__device__ __forceinline__ float *part_of(const F8Params &p, uint32_t slot, uint32_t rank, uint32_t quarter, uint32_t col) {
  return p.parts + (static_cast<uint64_t>(slot) * 2 + rank) * PART + static_cast<uint64_t>(col) * ROWS_CTA +
         quarter * 32u + (threadIdx.x & 31u);
}
__device__ __forceinline__ void park(float *mine, uint32_t cols, uint32_t taddr) {
#pragma unroll 1
  for (uint32_t c = 0; c < cols; c += 16) {
    uint32_t v[16];
    ptx::tmem_ld_32x32b_x16(taddr + c, v);
    ptx::tmem_ld_wait();
#pragma unroll
    for (uint32_t j = 0; j < 16; ++j) __stcg(mine + (c + j) * ROWS_CTA, __uint_as_float(v[j]));
  }
  __syncwarp();
}
// by one lane: whether all other slices' sums of these lanes (and columns) have been parked.  It counts for what other lanes
// and, gated, another warp have parked as well, of which it has been told inside the CTA: so the fences are its own, in front
// of its count and behind it, and not those of each lane.
__device__ __forceinline__ bool is_last(const F8Params &p, const Tile &x, uint32_t rank, uint32_t which) {
  __threadfence();
  const bool last = atomicInc(p.counters + 2 + (x.number * 2 + rank) * 16 + which, x.slices - 1) == x.slices - 1;
  __threadfence();
  return last;
}
// the sums of all slices, the first of which is at `first`, added in their order, back to tensor memory
__device__ __forceinline__ void join(const float *first, uint32_t slices, uint32_t cols, uint32_t taddr) {
  __syncwarp(); // (the lane that counted has been told first)
#pragma unroll 1
  for (uint32_t c = 0; c < cols; c += 16) {
    float v[16];
#pragma unroll
    for (uint32_t j = 0; j < 16; ++j) v[j] = 0.f;
#pragma unroll 1
    for (uint32_t s = 0; s < slices; s += JOIN_AHEAD) {
      float y[JOIN_AHEAD][16]; // several slices' values are on their way at once
#pragma unroll
      for (uint32_t i = 0; i < JOIN_AHEAD; ++i)
#pragma unroll
        for (uint32_t j = 0; j < 16; ++j)
          y[i][j] = s + i < slices ? __ldcg(first + static_cast<uint64_t>(s + i) * 2 * PART + (c + j) * ROWS_CTA) : 0.f;
#pragma unroll
      for (uint32_t i = 0; i < JOIN_AHEAD; ++i)
#pragma unroll
        for (uint32_t j = 0; j < 16; ++j) v[j] += y[i][j];
    }
    uint32_t w[16];
#pragma unroll
    for (uint32_t j = 0; j < 16; ++j) w[j] = __float_as_uint(v[j]);
    ptx::tmem_st_32x32b_x16(taddr + c, w);
  }
  ptx::tmem_st_wait();
}

// Results leave the warp's buffer by asynchronous copies, and the next tile's stages go on meanwhile: boxes of 32 rows, or
// where a group ends in between the rows one by one (gated ones from the lanes).  (All pairs come to the end of a tile
// together.  Stored by the lanes, their results had to wait for the way to memory, 64 KB from each SM at 3.8 TB/s: 4000
// cycles a tile.  With all rows one by one 8192 x 8192 x 8192 took 490 us where boxes took 484, and gated ones, of 64
// bytes, 712 instead of 675.)
__device__ __forceinline__ void wait_copied() { asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory"); }
__device__ __forceinline__ void wait_written() { asm volatile("cp.async.bulk.wait_group 0;" ::: "memory"); }
__device__ __forceinline__ void fence_to_copy() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }
__device__ __forceinline__ void commit_copies() { asm volatile("cp.async.bulk.commit_group;" ::: "memory"); }
__device__ __forceinline__ void copy_row(void *to, uint32_t from, uint32_t bytes) {
  asm volatile("cp.async.bulk.global.shared::cta.bulk_group [%0], [%1], %2;" ::"l"(to), "r"(from), "r"(bytes) : "memory");
}
__device__ __forceinline__ void copy_box(const CUtensorMap *map, uint32_t from, uint32_t byte, uint32_t row) {
  asm volatile("cp.async.bulk.tensor.3d.global.shared::cta.tile.bulk_group [%0, {%1, %2, %3}], [%4];" ::"l"(map), "r"(byte),
               "r"(row), "r"(0), "r"(from)
               : "memory");
}

// 64 bytes of each of a warp's rows, which its lanes have in w, to the warp's buffer: a lane stores its own as 16-byte
// chunks (those of two rows side by side XORed, so that neither side meets a bank twice).
__device__ __forceinline__ void to_buffer(uint32_t buf, const uint32_t (&w)[16]) {
  const uint32_t lane = threadIdx.x & 31u;
  wait_copied();
  __syncwarp(); // the buffer has been read
#pragma unroll
  for (uint32_t i = 0; i < 4; ++i)
    st_shared(buf + lane * 64u + ((i ^ ((lane >> 1) & 3u)) << 4), w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]);
  __syncwarp();
}
// `elems` elements of each of `rows` rows, at any address: element by element, neighbours by neighbouring lanes
template <class E>
__device__ __forceinline__ void store_elements(uint32_t buf, const uint32_t (&w)[16], E *out, uint64_t ldo, uint32_t rows,
                                               uint32_t elems) {
  constexpr uint32_t PER = 16 / sizeof(E), ALL = 4 * PER;
  to_buffer(buf, w);
  const uint32_t lane = threadIdx.x & 31u, e = lane % ALL, first = lane / ALL; // (its rows are a step of 32 / ALL apart)
  out += first * ldo + e;
#pragma unroll 8
  for (uint32_t i = 0; i < ALL; ++i) {
    const uint32_t row = first + i * (32 / ALL);
    const E v = ld_shared_one<E>(buf + row * 64u + (((e / PER) ^ ((row >> 1) & 3u)) << 4) + (e % PER) * sizeof(E));
    if (row < rows && e < elems) *out = v;
    out += (32 / ALL) * ldo;
  }
}

// N columns of a warp's sums; where there are none (zero) the product is 0
template <uint32_t N> __device__ __forceinline__ void fetch(uint32_t taddr, bool zero, uint32_t (&v)[N]) {
  if (zero) {
#pragma unroll
    for (uint32_t j = 0; j < N; ++j) v[j] = 0;
  } else {
    read_columns(taddr, v);
    ptx::tmem_ld_wait();
  }
}

// 64 bytes of a lane's row of sums, with the bias added and rounded: the one rounding.  E: an element of the result
template <class E>
__device__ __forceinline__ void results(uint32_t taddr, bool zero, const float *bias, uint32_t cols, bool bf16, uint32_t (&w)[16]) {
  constexpr uint32_t PER = 64 / sizeof(E);
  uint32_t v[PER];
  fetch(taddr, zero, v);
  if (bias != nullptr) {
#pragma unroll
    for (uint32_t j = 0; j < PER; ++j) v[j] = __float_as_uint(__uint_as_float(v[j]) + (j < cols ? __ldg(bias + j) : 0.f));
  }
  if constexpr (sizeof(E) == 4) {
#pragma unroll
    for (uint32_t i = 0; i < 16; ++i) w[i] = v[i];
  } else {
#pragma unroll
    for (uint32_t i = 0; i < 16; ++i) {
      const float x = __uint_as_float(v[2 * i]), y = __uint_as_float(v[2 * i + 1]);
      w[i] = bf16 ? pack_bf16(x, y) : pack_f16(x, y);
    }
  }
}
// The same for 32 rows of 128 columns of 16 bits from the registers, in two boxes.  (No branches in between: with a test for
// the bias at every pair the stores took 2200 cycles.)
template <bool BF16>
__device__ __forceinline__ void store_whole(const CUtensorMap *map, uint32_t buf, float (&sums)[MOST], uint32_t row, uint32_t col,
                                            const float *bias) {
  static_assert(MOST * 2 == OUT_ROW, "a row of the buffer");
  const uint32_t lane = threadIdx.x & 31u, mine = buf + lane * OUT_BOX;
  if (bias != nullptr) {
#pragma unroll
    for (uint32_t c = 0; c < MOST; ++c) sums[c] += __ldg(bias + c);
  }
  wait_copied();
  __syncwarp();
#pragma unroll
  for (uint32_t c = 0; c < MOST; c += 8) {
    uint32_t w[4];
#pragma unroll
    for (uint32_t i = 0; i < 4; ++i)
      w[i] = BF16 ? pack_bf16(sums[c + 2 * i], sums[c + 2 * i + 1]) : pack_f16(sums[c + 2 * i], sums[c + 2 * i + 1]);
    constexpr uint32_t CHUNKS = OUT_BOX / 16;
    st_shared(mine + c / 8 / CHUNKS * (32 * OUT_BOX) + (((c / 8 % CHUNKS) ^ (lane & 7u)) << 4), w[0], w[1], w[2], w[3]);
  }
  fence_to_copy();
  __syncwarp();
  if (lane == 0) {
    copy_box(map, buf, 2 * col, row);
    copy_box(map, buf + 32 * OUT_BOX, 2 * col + OUT_BOX, row);
  }
  commit_copies();
}

// `cols` columns of a warp's sums to the result, from `row` and `col` on.
template <class E>
__device__ __forceinline__ void store_sums(const F8Params &p, const CUtensorMap *map, uint32_t buf, uint32_t taddr, bool zero,
                                           uint32_t row, uint32_t col, uint32_t rows, uint32_t cols, const float *bias) {
  constexpr uint32_t PER = 64 / sizeof(E), ROW = OUT_ROW / sizeof(E);
  const uint32_t lane = threadIdx.x & 31u;
  const bool bf16 = static_cast<GroupedOut>(p.out_type) == GroupedOut::bf16;
  E *out = static_cast<E *>(p.out) + static_cast<uint64_t>(row) * p.ldo + col;
  if (p.vector_out != 0 && cols * sizeof(E) % 16 == 0) {
    const bool boxes = rows == 32;
#pragma unroll 1
    for (uint32_t c0 = 0; c0 < cols; c0 += ROW) {
      const uint32_t here = min(cols - c0, ROW);
      wait_copied();
      __syncwarp();
#pragma unroll 1
      for (uint32_t c = 0; c < here; c += PER) {
        uint32_t w[16];
        results<E>(taddr + c0 + c, zero, bias == nullptr ? nullptr : bias + c0 + c, here - c, bf16, w);
        // a box has its 16-byte chunks XORed with the row (modulo 8), as its map says
        const uint32_t b = c * sizeof(E), to = boxes ? buf + b / OUT_BOX * (32 * OUT_BOX) + lane * OUT_BOX : buf + lane * OUT_PITCH + b,
                       first = boxes ? b % OUT_BOX / 16 : 0u, flip = boxes ? lane & 7u : 0u;
#pragma unroll
        for (uint32_t i = 0; i < 4; ++i)
          st_shared(to + (((first + i) ^ flip) << 4), w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]);
      }
      fence_to_copy();
      if (boxes) {
        __syncwarp();
        if (lane == 0)
          for (uint32_t b = 0; b < here * sizeof(E); b += OUT_BOX)
            copy_box(map, buf + 32 * b, (col + c0) * sizeof(E) + b, row);
      } else if (lane < rows) {
        copy_row(out + lane * p.ldo + c0, buf + lane * OUT_PITCH, here * sizeof(E));
      }
      commit_copies();
    }
  } else {
#pragma unroll 1
    for (uint32_t c = 0; c < cols; c += PER) {
      uint32_t w[16];
      results<E>(taddr + c, zero, bias == nullptr ? nullptr : bias + c, cols - c, bf16, w);
      store_elements(buf, w, out + c, p.ldo, rows, cols - c);
    }
  }
}

// The warp asks once whether all of its rows can be brought to 8 bits by one factor.
template <F8Type TYPE>
__device__ __forceinline__ void quantise(const BlockScale &s, bool real, const float (&h)[MOST / 2], uint32_t (&w)[MOST / 8]) {
  float f;
  const bool one = s.plain(f) && !s.zero;
  if (__all_sync(0xffffffffu, one || !real)) {
#pragma unroll
    for (uint32_t i = 0; i < MOST / 8; ++i)
      w[i] = BlockScale::four_by<TYPE>(f, h[4 * i], h[4 * i + 1], h[4 * i + 2], h[4 * i + 3]);
  } else {
#pragma unroll
    for (uint32_t i = 0; i < MOST / 8; ++i)
      w[i] = one ? BlockScale::four_by<TYPE>(f, h[4 * i], h[4 * i + 1], h[4 * i + 2], h[4 * i + 3])
                 : s.four<TYPE>(h[4 * i], h[4 * i + 1], h[4 * i + 2], h[4 * i + 3]);
  }
}

template <bool GATED>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(THREADS, 1)
    f8_gemm_kernel(const __grid_constant__ CUtensorMap map_x, const __grid_constant__ CUtensorMap map_x_few,
                   const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_w_few,
                   const __grid_constant__ CUtensorMap map_out, const __grid_constant__ F8Params p) {
  using S = Shared<GATED>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t *const smem =
      reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  const uint32_t sbase = ptx::smem_u32(smem);
  volatile int *const abort_flag = reinterpret_cast<volatile int *>(smem + ABORT);
  const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31u;
  const uint32_t rank = ptx::cluster_ctarank();
  const bool leader = rank == 0;
  const uint32_t cluster_id = blockIdx.x >> 1, clusters = gridDim.x >> 1;

  if (threadIdx.x == 0) {
    for (uint32_t s = 0; s < S::STAGES; ++s) {
      ptx::mbar_init(sbase + FULL + 8 * s, 2);
      ptx::mbar_init(sbase + EMPTY + 8 * s, 1);
    }
    for (uint32_t b = 0; b < MOST_SLOTS; ++b) {
      ptx::mbar_init(sbase + ACC_FULL + 8 * b, 1);
      ptx::mbar_init(sbase + ACC_EMPTY + 8 * b, 2 * EPI_WARPS);
    }
    for (uint32_t q = 0; q < 4; ++q) ptx::mbar_init(sbase + PAIR + 8 * q, PARTS);
    for (uint32_t i = 0; i < AHEAD; ++i) {
      ptx::mbar_init(sbase + TILE_FULL + 8 * i, 1);
      ptx::mbar_init(sbase + TILE_EMPTY + 8 * i, EPI_WARPS + (leader ? 3 : 2)); // and who loads, copies, issues
    }
    for (uint32_t i = 0; i < 2; ++i) {
      ptx::mbar_init(sbase + SC_FULL + 8 * i, 32);
      ptx::mbar_init(sbase + SC_EMPTY + 8 * i, EPI_WARPS);
    }
    *abort_flag = 0;
    ptx::mbar_init_fence();
    ptx::prefetch_tensormap(&map_x);
    ptx::prefetch_tensormap(&map_x_few);
    ptx::prefetch_tensormap(&map_w);
    ptx::prefetch_tensormap(&map_w_few);
    ptx::prefetch_tensormap(&map_out);
  }
  if (warp == 1) {
    ptx::tmem_alloc_pair(sbase + TMEM_PTR, TMEM_COLS);
    ptx::tmem_relinquish_pair();
  }
  // Everything above needs nothing of the kernel in front, everything below may.
  ptx::griddep_wait();
  if (warp == 2) find_groups<GATED>(smem, p, clusters);
  ptx::tc_fence_before();
  __syncthreads();
  // both CTAs' barriers must exist before any remote arrive / remote TMA completion
  ptx::cluster_arrive();
  ptx::cluster_wait();
  ptx::tc_fence_after();
  const uint32_t tmem_base = *reinterpret_cast<const uint32_t *>(smem + TMEM_PTR);

  if (warp < 4) {
    ptx::setmaxnreg_dec<REGS_REST>();
    const uint32_t width = ld_shared_one<uint32_t>(sbase + WIDTH);
    Tile x;
    if (warp == 0) {
      // ============================================================== TMA producer (both CTAs)
      if (ptx::elect_one()) {
        uint32_t s = 0, ph = 1;
        bool ok = true;
        const uint32_t half = width / 2; // columns that this CTA loads
        Tiles<false> tiles(sbase);
        while (ok && tiles.next(p.status, x)) {
          // boxes of rows: one of 128, or as many of 32 as it takes; none where this CTA has no rows
          const uint32_t rows = x.rows > rank * ROWS_CTA ? min(x.rows - rank * ROWS_CTA, ROWS_CTA) : 0u;
          const uint32_t x_boxes = (rows + BOX_ROWS - 1) / BOX_ROWS;
          const bool x_whole = x_boxes == ROWS_CTA / BOX_ROWS;
          const uint32_t bytes = (x_boxes * BOX_ROWS + half) * BLOCK;
          const int row = static_cast<int>(x.row0 + rank * ROWS_CTA);
          const int e = static_cast<int>(x.group);
          for (uint32_t kb = 0; kb < x.blocks; ++kb) {
            ok = ptx::mbar_wait(sbase + EMPTY + 8 * s, ph, abort_flag, p.status, ptx::kErrWaitEmpty);
            if (!ok) break;
            const uint32_t x_dst = sbase + S::FIRST + s * STAGE_BYTES, w_dst = x_dst + TILE_BYTES;
            const uint32_t full = ptx::map_to_cta(sbase + FULL + 8 * s, 0); // the leader's barrier
            if (leader) ptx::mbar_arrive_expect_tx(sbase + FULL + 8 * s, bytes);
            else ptx::mbar_arrive_expect_tx_cluster(full, bytes);
            const int k = static_cast<int>((x.k0 + kb) * BLOCK);
            if (x_whole) {
              ptx::tma_load_3d_pair(x_dst, &map_x, full, k, row, 0);
            } else {
              for (uint32_t b = 0; b < x_boxes; ++b)
                ptx::tma_load_3d_pair(x_dst + b * BOX_ROWS * BLOCK, &map_x_few, full, k,
                                      row + static_cast<int>(b * BOX_ROWS), 0);
            }
            if constexpr (GATED) { // for each warp's columns rows of the gate, then the same of the projection
#pragma unroll
              for (uint32_t b = 0; b < COLS / 2 / BOX_ROWS; ++b) {
                const uint32_t local = b * BOX_ROWS % MOST, f = x.col0 + (rank * (COLS / 2) + b * BOX_ROWS) / MOST * (MOST / 2);
                ptx::tma_load_3d_pair(w_dst + b * BOX_ROWS * BLOCK, &map_w_few, full, k,
                                      static_cast<int>(local < MOST / 2 ? f + local : p.n + f + local - MOST / 2), e);
              }
            } else {
              const int c = static_cast<int>(x.col0 + rank * half);
              if (half == COLS / 2) {
                ptx::tma_load_3d_pair(w_dst, &map_w, full, k, c, e);
              } else {
                for (uint32_t b = 0; b < half / BOX_ROWS; ++b)
                  ptx::tma_load_3d_pair(w_dst + b * BOX_ROWS * BLOCK, &map_w_few, full, k,
                                        c + static_cast<int>(b * BOX_ROWS), e);
              }
            }
            if (++s == S::STAGES) {
              s = 0;
              ph ^= 1u;
            }
          }
        }
      }
    } else if (warp == 1) {
      // ============================================================== MMA issuer (leader only)
      if (leader && ptx::elect_one()) {
        constexpr uint16_t BOTH = 0x3;
        constexpr uint64_t kStage = STAGE_BYTES >> 4;
        const uint64_t a0 = ptx::make_kmajor_desc<BLOCK>(sbase + S::FIRST), b0 = ptx::make_kmajor_desc<BLOCK>(sbase + S::FIRST + TILE_BYTES);
        const uint32_t idesc = p.idesc | ((width >> 3) << 17);
        const uint32_t slots = slots_of(width), slot_cols = TMEM_COLS / slots;
        uint32_t s = 0, ph = 0, acc = 0, e_ph = 1;
        bool ok = true;
        Tiles<false> tiles(sbase);
        while (ok && tiles.next(p.status, x)) {
          for (uint32_t kb = 0; kb < x.blocks; ++kb) {
            // (the accumulator last: what follows its wait lengthens the way round)
            ok = ptx::mbar_wait(sbase + FULL + 8 * s, ph, abort_flag, p.status, ptx::kErrWaitFull) &&
                 ptx::mbar_wait(sbase + ACC_EMPTY + 8 * acc, e_ph, abort_flag, p.status, ptx::kErrWaitD0Empty);
            if (!ok) break;
            ptx::tc_fence_after();
            const uint32_t d = tmem_base + acc * slot_cols;
#pragma unroll
            for (uint32_t ks = 0; ks < 4; ++ks)
              ptx::mma_f8_ss_pair(d, a0 + s * kStage + 2 * ks, b0 + s * kStage + 2 * ks, idesc, ks != 0);
            ptx::tc_commit_pair(sbase + ACC_FULL + 8 * acc, BOTH);
            ptx::tc_commit_pair(sbase + EMPTY + 8 * s, BOTH);
            if (++acc == slots) {
              acc = 0;
              e_ph ^= 1u;
            }
            if (++s == S::STAGES) {
              s = 0;
              ph ^= 1u;
            }
          }
        }
      }
    } else if (warp == 2) {
      // ============================================================== the next tiles (both CTAs, each its own)
      if (ptx::elect_one()) {
        Items<GATED> items(sbase, p, clusters);
        uint32_t turn = 0, ph = 1;
        for (uint32_t item = cluster_id;; item += clusters) {
          const bool more = item < items.total;
          if (more && !items.get(p, item, x)) continue;
          if (!more) x = Tile{};
          if (!ptx::mbar_wait_backoff(sbase + TILE_EMPTY + 8 * turn, ph, abort_flag, p.status, ptx::kErrWaitTile, 64)) break;
          const uint32_t to = sbase + TILE + 48 * turn;
          st_shared(to, x.group, x.row0, x.rows, x.col0);
          st_shared(to + 16, x.k0, x.blocks, x.slices, x.slice);
          st_shared(to + 32, x.slot, x.number, 0, 0);
          ptx::mbar_arrive(sbase + TILE_FULL + 8 * turn);
          if (!more) break;
          if (++turn == AHEAD) {
            turn = 0;
            ph ^= 1u;
          }
        }
      }
    } else {
      // ============================================================== scales (both CTAs)
      // Asynchronous copies that announce themselves: nothing waits for memory.  (An epilogue warp with loads of its own
      // on their way waits for them at every read of tensor memory: its stages took 600 cycles instead of 370.)
      const uint32_t w_blocks = ((GATED ? 2 * p.n : p.n) + BLOCK - 1) / BLOCK;
      uint32_t b = 0, ph = 1;
      bool ok = true;
      Tiles<true> tiles(sbase);
      while (ok) {
        ok = tiles.wait(p.status);
        if (!ok) break;
        const uint32_t turn = tiles.advance();
        tiles.read(turn, x);
        tiles.give_back(turn);
        if (x.rows == 0) break;
        const uint32_t row0 = rank * ROWS_CTA, rows = x.rows > row0 ? min(x.rows - row0, ROWS_CTA) : 0u;
        const float *xs = p.x_scale + (static_cast<uint64_t>(x.row0) + row0 + lane) * p.x_scale_row + x.k0 * p.x_scale_block;
        const uint32_t block = GATED ? (x.col0 + lane * p.n) / BLOCK : x.col0 / BLOCK + lane;
        // (columns behind the last block have any)
        const float *ws = p.w_scale + (static_cast<uint64_t>(x.group) * w_blocks + min(block, w_blocks - 1)) * p.blocks + x.k0;
        for (uint32_t kb = 0; kb < x.blocks; kb += AT_ONCE) {
          ok = ptx::warp_agrees(ptx::mbar_wait_backoff(sbase + SC_EMPTY + 8 * b, ph, abort_flag, p.status, ptx::kErrWaitTile, 64));
          if (!ok) break;
          for (uint32_t i = 0; i < AT_ONCE && kb + i < x.blocks; ++i) {
            const uint32_t to = sbase + SCALE + (b * AT_ONCE + i) * (SCALE_WORDS * 4) + lane * 4u;
#pragma unroll
            for (uint32_t j = 0; j < 4; ++j)
              if (lane + 32 * j < rows) copy_word(to + 128u * j, xs + 32 * j * p.x_scale_row);
            if (lane < 2) copy_word(to + ROWS_CTA * 4, ws);
            xs += p.x_scale_block;
            ++ws;
          }
          copies_arrive(sbase + SC_FULL + 8 * b);
          b ^= 1u;
          if (b == 0) ph ^= 1u;
        }
      }
      wait_copies();
    }
  } else {
    // ================================================================ epilogue (both CTAs)
    ptx::setmaxnreg_inc<REGS_EPI>();
    Tile x;
    const uint32_t epi = warp - 4, quarter = warp & 3u, part = epi >> 2;
    const uint32_t width = ld_shared_one<uint32_t>(sbase + WIDTH), slots = slots_of(width), slot_cols = TMEM_COLS / slots;
    const uint32_t mine = width / PARTS; // columns of the warp, from part * mine on
    const uint32_t t_lanes = tmem_base + ((quarter * 32u) << 16) + part * mine;
    const uint32_t acc_empty = ptx::map_to_cta(sbase + ACC_EMPTY, 0);
    const uint32_t buf = sbase + OUT + epi * S::OUT_BYTES;
    const uint32_t lane0 = rank * ROWS_CTA + quarter * 32u; // the warp's first row in a tile
    uint32_t turn = 0, group = 0, pair_ph = 0, parity = 0; // accumulators and groups of scales that are behind
    bool ok = true;
    const uint32_t slots_log2 = slots == 2 ? 1u : 2u;
    auto slot_now = [&]() { return turn & (slots - 1u); };
    // An accumulator is given back when its reads are complete (wait::ld): that is all there is to order.
    auto give_back = [&](bool yes) {
      ptx::tc_fence_before();
      __syncwarp();
      arrive_cluster_relaxed_if(yes && lane == 0, acc_empty + 8 * slot_now());
      turn += yes;
    };
    // The stages of a tile; the last accumulator is not given back.
    auto all_stages = [&](uint32_t blocks, auto &&add) {
      const uint32_t scales = sbase + SCALE + (quarter * 32u + lane) * 4u;
      const uint32_t weights = sbase + SCALE + (ROWS_CTA + (GATED ? 0u : part * mine / BLOCK)) * 4u;
#pragma unroll 1
      for (uint32_t kb = 0; kb < blocks; ++kb) {
        const uint32_t b = group & 1u, sc_full = sbase + SC_FULL + 8 * b, full = sbase + ACC_FULL + 8 * slot_now();
        const uint32_t sc_ph = (group >> 1) & 1u, ph = (turn >> slots_log2) & 1u;
        if (!ptx::warp_agrees(both_over(sc_full, sc_ph, full, ph))) {
          ok = ptx::warp_agrees(ptx::mbar_wait_s(sc_full, sc_ph, sbase + ABORT, p.status, ptx::kErrWaitTile) &&
                                ptx::mbar_wait_s(full, ph, sbase + ABORT, p.status, ptx::kErrWaitD0Full));
          if (!ok) break;
        }
        ptx::tc_fence_after();
        const uint32_t offset = (b * AT_ONCE + kb % AT_ONCE) * (SCALE_WORDS * 4);
        const float own = __uint_as_float(ld_shared_one<uint32_t>(scales + offset));
        const float t0 = own * __uint_as_float(ld_shared_one<uint32_t>(weights + offset)),
                    t1 = GATED ? own * __uint_as_float(ld_shared_one<uint32_t>(weights + offset + 4)) : 0.f;
        add(t_lanes + slot_now() * slot_cols, t0, t1);
        give_back(kb + 1 < blocks);
        const bool last = kb % AT_ONCE == AT_ONCE - 1 || kb + 1 == blocks; // of the scales that were copied together
        arrive_if(last && lane == 0, sbase + SC_EMPTY + 8 * b);
        group += last;
      }
    };
    Tiles<true> tiles(sbase);
    ok = tiles.wait(p.status);
    uint32_t slot = tiles.advance();
    if (ok) tiles.read(slot, x);
    while (ok && x.rows > 0) {
      float sums[MOST];
#pragma unroll
      for (uint32_t i = 0; i < MOST; ++i) sums[i] = 0.f;
      const bool zero = x.blocks == 0;
      if (!zero) {
        if (x.rows <= lane0) {
          all_stages(x.blocks, [](uint32_t, float, float) {});
        } else if (GATED || mine == MOST) {
          all_stages(x.blocks, [&](uint32_t from, float t0, float t1) { drain<GATED, MOST>(from, sums, t0, t1); });
        } else {
          all_stages(x.blocks, [&](uint32_t from, float t0, float t1) { drain<GATED, MOST / 2>(from, sums, t0, t1); });
        }
        if (!ok) break;
      }
      // The tile again: kept over the loop it took registers from the sums.
      tiles.read(slot, x);
      const uint32_t rows = x.rows > lane0 ? min(x.rows - lane0, 32u) : 0u;
      // Whole tiles leave from the registers, and the last accumulator is free at once.  Otherwise the sums take its place:
      // what follows has few registers then, and little code.
      const bool whole = x.slices == 1 &&
                         (GATED || (p.vector_out != 0 && rows == 32 && x.col0 + (part + 1) * MOST <= p.n && mine == MOST &&
                                    static_cast<GroupedOut>(p.out_type) != GroupedOut::f32));
      if (!zero) {
        if (whole) give_back(true);
        else if (rows > 0) put_back(t_lanes + slot_now() * slot_cols, sums, mine);
      }
      const bool real = lane < rows;
      const uint32_t t_sums = t_lanes + slot_now() * slot_cols;
      bool done = rows == 0;
      if constexpr (GATED) {
        // (all warps that have these lanes have rows, or none)
        auto meet = [&]() { // the other warps; false: the wait gave up
          __syncwarp();
          if (lane == 0) ptx::mbar_arrive(sbase + PAIR + 8 * quarter);
          const bool met = ptx::warp_agrees(
              ptx::mbar_wait_s(sbase + PAIR + 8 * quarter, pair_ph, sbase + ABORT, p.status, ptx::kErrWaitD1Full));
          pair_ph ^= 1u;
          return met;
        };
        if (!done && x.slices > 1) { // all are last, or none
          park(part_of(p, x.slot, rank, quarter, part * mine), mine, t_sums);
          ok = meet();
          if (!ok) break;
          volatile uint32_t *last = reinterpret_cast<volatile uint32_t *>(smem + LAST) + quarter;
          if (part == 0 && lane == 0) *last = is_last(p, x, rank, quarter);
          ok = meet();
          if (!ok) break;
          done = *last == 0;
          if (!done) join(part_of(p, x.slot - x.slice, rank, quarter, part * mine), x.slices, mine, t_sums);
        }
        if (!done) {
          if (!whole) {
#pragma unroll
            for (uint32_t c = 0; c < MOST; c += 16) {
              uint32_t v[16];
              fetch(t_sums + c, zero, v);
#pragma unroll
              for (uint32_t i = 0; i < 16; ++i) sums[c + i] = __uint_as_float(v[i]);
            }
          }
          float h[MOST / 2];
          uint32_t top = 0;
#pragma unroll
          for (uint32_t c = 0; c < MOST / 2; c += 16) { // (the four activations of all of them at once spilled)
            with_activation(p.activation, [&](auto act) {
#pragma unroll
              for (uint32_t i = 0; i < 16; ++i) h[c + i] = activate<act.value, true>(sums[c + i]).value * sums[MOST / 2 + c + i];
            });
#pragma unroll
            for (uint32_t i = 0; i < 16; ++i) top = max(top, __float_as_uint(h[c + i]) & 0x7fffffffu);
          }
          // (written again two tiles on, when the other warps have long read them: they have been met since)
          uint32_t *tops = reinterpret_cast<uint32_t *>(smem + TOPS) + parity * PARTS * ROWS_CTA + quarter * 32u + lane;
          parity ^= 1u;
          tops[part * ROWS_CTA] = top;
          ok = meet();
          if (!ok) break;
#pragma unroll
          for (uint32_t i = 0; i < PARTS; ++i) top = max(top, tops[i * ROWS_CTA]);
          const auto type = static_cast<F8Type>(p.out_type);
          const BlockScale s(__uint_as_float(top), type);
          uint32_t w[MOST / 8];
          if (type == F8Type::e4m3) quantise<F8Type::e4m3>(s, real, h, w);
          else quantise<F8Type::e5m2>(s, real, h, w);
          const uint64_t row = x.row0 + lane0;
          uint8_t *out = static_cast<uint8_t *>(p.out) + (row + lane) * p.ldo + x.col0 + part * (MOST / 2);
          if (p.vector_out != 0 && rows == 32) {
            wait_copied();
            __syncwarp();
#pragma unroll
            for (uint32_t i = 0; i < MOST / 32; ++i)
              st_shared(buf + lane * 64u + 16 * i, w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]);
            fence_to_copy();
            __syncwarp();
            if (lane == 0) copy_box(&map_out, buf, x.col0 + part * (MOST / 2), static_cast<uint32_t>(row));
            commit_copies();
          } else if (real && p.vector_out != 0) {
#pragma unroll
            for (uint32_t i = 0; i < MOST / 32; ++i)
              reinterpret_cast<uint4 *>(out)[i] = make_uint4(w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]);
          } else if (real) {
#pragma unroll
            for (uint32_t i = 0; i < MOST / 2; ++i) out[i] = static_cast<uint8_t>(w[i / 4] >> (8 * (i & 3u)));
          }
          if (part == 0 && real) p.out_scale[(row + lane) * p.out_scale_row + x.col0 / BLOCK * p.out_scale_block] = s.scale;
        }
      } else {
        const uint32_t col = x.col0 + part * mine;
        const uint32_t cols = p.n > col ? min(mine, p.n - col) : 0u;
        done |= cols == 0;
        if (!done && x.slices > 1) {
          park(part_of(p, x.slot, rank, quarter, part * mine), mine, t_sums);
          const bool last = lane == 0 && is_last(p, x, rank, epi);
          done = !__any_sync(0xffffffffu, last);
          if (!done) join(part_of(p, x.slot - x.slice, rank, quarter, part * mine), x.slices, mine, t_sums);
        }
        if (!done) {
          const float *bias = p.bias != nullptr && x.group < p.groups ? p.bias + static_cast<uint64_t>(x.group) * p.n + col : nullptr;
          if (whole && static_cast<GroupedOut>(p.out_type) == GroupedOut::bf16)
            store_whole<true>(&map_out, buf, sums, x.row0 + lane0, col, bias);
          else if (whole) store_whole<false>(&map_out, buf, sums, x.row0 + lane0, col, bias);
          else if (static_cast<GroupedOut>(p.out_type) == GroupedOut::f32)
            store_sums<uint32_t>(p, &map_out, buf, t_sums, zero, x.row0 + lane0, col, rows, cols, bias);
          else store_sums<uint16_t>(p, &map_out, buf, t_sums, zero, x.row0 + lane0, col, rows, cols, bias);
        }
      }
      if (!zero && !whole) give_back(true);
      tiles.give_back(slot);
      ok = tiles.wait(p.status);
      if (!ok) break;
      slot = tiles.advance();
      tiles.read(slot, x);
    }
    wait_written();
  }

  // ---------------------------------------------------------------- teardown
  // The peer's shared memory and TMEM are in use by the leader's MMAs until the last accumulator has
  // been announced in both CTAs; neither CTA leaves before the other has finished its epilogue.
  ptx::tc_fence_before();
  __syncthreads();
  ptx::cluster_arrive();
  ptx::cluster_wait();
  if (*abort_flag) {
    const uint64_t t0 = ptx::globaltimer_ns();
    while (ptx::globaltimer_ns() - t0 < 2000000ull) __nanosleep(1000);
    __syncthreads();
  }
  if (warp == 1) {
    ptx::tc_fence_after();
    ptx::tmem_dealloc_pair(tmem_base, TMEM_COLS);
  }
}

// Per device and kernel, once (any thread): shared-memory attribute and the pairs the device keeps resident.
template <bool GATED> cudaError_t set_up(int *clusters_out) {
  static std::once_flag once[64];
  static cudaError_t setup_error[64];
  static int max_clusters[64];
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev < 0 || dev >= 64) return cudaErrorInvalidDevice;
  std::call_once(once[dev], [&]() {
    const auto kernel = f8_gemm_kernel<GATED>;
    setup_error[dev] = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, Shared<GATED>::BYTES);
    int sms = 0;
    cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
    int clusters = sms / 2;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(static_cast<unsigned>(2 * clusters));
    cfg.blockDim = dim3(THREADS);
    cfg.dynamicSmemBytes = Shared<GATED>::BYTES;
    int active = 0;
    if (setup_error[dev] == cudaSuccess && cudaOccupancyMaxActiveClusters(&active, kernel, &cfg) == cudaSuccess) {
      if (active > 0 && active < clusters) clusters = active;
    } else {
      cudaGetLastError();
    }
    max_clusters[dev] = clusters > 0 ? clusters : 1;
  });
  *clusters_out = max_clusters[dev];
  return setup_error[dev];
}

bool operand_map(CUtensorMap *map, const GroupedOperand &o, uint32_t box_rows) {
  return make_byte_map(map, 1, o.ptr, {o.inner, o.outer, o.batch}, {o.ld, o.batch > 1 ? o.stride : o.ld},
                       {BLOCK, box_rows, 1}, true);
}

template <bool GATED> cudaError_t launch(const GroupedArgs &a, const F8Args &f, cudaStream_t stream) {
  int clusters = 1;
  const cudaError_t se = set_up<GATED>(&clusters);
  if (se != cudaSuccess) return se;
  CUtensorMap map_x, map_x_few, map_w, map_w_few, map_out;
  if (!operand_map(&map_x_few, a.b, BOX_ROWS) || !operand_map(&map_w_few, a.a, BOX_ROWS))
    return cudaErrorInvalidValue;
  // boxes of 128 rows are for tiles that have as many, and not for gated ones' weights
  map_x = map_x_few;
  map_w = map_w_few;
  if (a.rows > ROWS_CTA - BOX_ROWS && !operand_map(&map_x, a.b, ROWS_CTA)) return cudaErrorInvalidValue;
  if (!GATED && !operand_map(&map_w, a.a, COLS / 2)) return cudaErrorInvalidValue;
  F8Params p = {};
  p.ends = a.ends;
  p.out = a.out;
  p.ldo = a.ldo;
  p.x_scale = a.col_scale;
  p.x_scale_row = f.x_scale_row;
  p.x_scale_block = f.x_scale_block;
  p.w_scale = a.lane_scale;
  p.bias = a.bias;
  p.out_scale = f.out_scale;
  p.out_scale_row = f.out_scale_row;
  p.out_scale_block = f.out_scale_block;
  p.parts = a.parts;
  p.counters = a.counters;
  p.status = a.dev_status;
  p.rows = a.rows;
  p.groups = a.groups;
  p.n = a.lane_dim;
  p.blocks = (a.k + BLOCK - 1) / BLOCK;
  // FP32 sums; the formats of A (x) and B (w), e4m3 (0) or e5m2 (1)
  p.idesc = (1u << 4) | (static_cast<uint32_t>(f.x_type) << 7) | (static_cast<uint32_t>(f.w_type) << 10) | ((ROWS >> 4) << 24);
  p.out_type = static_cast<uint16_t>(GATED ? f.out_type : static_cast<int>(a.out_type));
  p.activation = static_cast<uint8_t>(f.activation);
  const uint64_t out_bytes = GATED ? 1 : a.out_type == GroupedOut::f32 ? 4 : 2;
  p.vector_out = (reinterpret_cast<uintptr_t>(a.out) & 15u) == 0 && a.ldo * out_bytes % 16 == 0;
  // in bytes; used only where rows of the result are whole 16 bytes (and no larger than a map's)
  const uint64_t row_bytes = p.n * out_bytes, pitch = a.ldo * out_bytes;
  if (row_bytes >= 1ull << 31 || pitch >= 1ull << 40) p.vector_out = 0;
  map_out = map_x_few;
  if (p.vector_out && !make_byte_map(&map_out, 1, a.out, {row_bytes, p.rows, 1}, {pitch, pitch}, {GATED ? MOST / 2 : OUT_BOX, 32, 1}, !GATED))
    return cudaErrorInvalidValue;
  return launch_chained(f8_gemm_kernel<GATED>, static_cast<unsigned>(2 * clusters), THREADS, Shared<GATED>::BYTES, stream, map_x,
                        map_x_few, map_w, map_w_few, map_out, p);
}

} // namespace

std::size_t f8_parts_bytes(const GroupedArgs &a, unsigned num_sms) {
  if (a.f8->few_rows) return f8_few_rows_parts_bytes(a, num_sms);
  const uint64_t pairs = num_sms / 2, features = a.f8->gated ? COLS / 2 : COLS;
  // tiles there are at least: groups may leave some unfilled
  const uint64_t least = ((a.rows + ROWS - 1) / ROWS) * ((a.lane_dim + features - 1) / features);
  return least <= pairs / 2 ? pairs * 2 * PART * sizeof(float) : 0;
}

cudaError_t launch_f8_gemm(const GroupedArgs &a, cudaStream_t stream) {
  if (a.f8->few_rows) return launch_f8_few_rows(a, stream);
  return a.f8->gated ? launch<true>(a, *a.f8, stream) : launch<false>(a, *a.f8, stream);
}

} // namespace cumpsgemm_b200
