// Products of rows grouped by expert, on CTA pairs (tcgen05 cta_group::2).
//
//   product  y[r, :] = alpha * x[r, :] op(w_e) + beta * y[r, :]     for the rows r of group e
//   wgrad    dw_e    = alpha * x_e^T dy_e + beta * dw_e             over the rows of group e
//   8 bits   y[r, c] = sx[r] * sw[e][c] * sum_k xq[r, k] wq_e[c, k] (+ bias[e][c])
//
// The sizes of the groups are known on the device only (`ends`, the running total of rows), so the
// grid is one persistent CTA pair per SM pair, and every pair walks the tiles of all groups, which it
// finds from the running totals in shared memory.
//
// Which side is which.  The weights' output features are the M side of the tensor core's product
// (lanes of tensor memory, 256 per pair) and the rows of a group its N side (columns): N goes by
// steps of 32 to 256, so a group whose rows fill no tile costs what its rows cost, and a step of
// decoding with four rows per expert multiplies 32 columns, not 256.  It also lets a warp's lanes
// hold neighbouring features, which are neighbours in the row-major output.  For wgrad both
// sides are weight dimensions, and lanes are the one that is contiguous in the output.
//
// Operands come by TMA as they lie in memory.  A 16-bit operand whose lanes (or columns) are the
// contiguous dimension is read as such (make_mnmajor_desc): no transposed copies.  FP32
// operands have been split into hi and lo FP16 planes of the same layout (row_kernels.cu), hi*hi is
// drained from tensor memory every two stages and added in registers and the corrections have an
// accumulator of their own, as in tcec_gemm_pair.cu.
//
// wgrad reduces over a group's rows, which end inside a 64-row block.  The next group's rows must not
// count, not even multiplied by zero, since they may be NaN: a warp of its own waits for such a last
// block, zeroes the rows up to the next multiple of 16 in both operands, and the tensor core gets only
// as many steps of 16.  (With the warp that issues the loads doing it the next tile's loads waited too:
// 32768 rows x 4096 x 4096 over 16 experts in bfloat16 took 984 us instead of 895.)
//
// Barriers ("leader" = cluster rank 0):
//   full[s]       leader's only: 2 arrivals, one from each CTA's producer (the leader's with the
//                 bytes of both CTAs' loads), or for a last block from the warps that zero its rows
//   empty[s]      in both CTAs: commit multicast from the leader
//   acc_full[b]   in both CTAs: commit multicast.  b: one of two accumulators (f16, i8), or hi*hi (0)
//                 and the corrections (1)
//   acc_empty[b]  leader's only: 16 arrivals, one from each epilogue warp of both CTAs
//   tail[s]       own: a last block's loads
//   next_full[i]  in both CTAs: 1 arrival, from the leader's warp that fetches the tiles, and their bytes
//   next_empty[i] leader's only: one arrival from each role that took the tile
//   want          leader's only: 1 arrival, from its producer towards the end of each tile
// Every wait is bounded; no TMA multicast is used.
#include "epilogue.cuh"
#include "gemm_common.cuh"
#include "grouped.hpp"
#include "ptx.cuh"
#include "split_math.cuh"

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <mutex>
#include <type_traits>

namespace cumpsgemm_b200 {
namespace {

constexpr int BM_CTA = 128;            // lanes per CTA
constexpr uint32_t LANES = 2 * BM_CTA; // per pair
constexpr uint32_t COLS = 256;         // most columns of a tile
constexpr uint32_t WIDTHS = 3;         // that a launch chooses from: 256, 128, 64
constexpr uint32_t ROW_BYTES = kGemmRowBytes;
constexpr uint32_t TILE_BYTES = 128 * ROW_BYTES; // an operand's part of a stage in one CTA
constexpr uint32_t ATOM_BYTES = 64 * ROW_BYTES;  // lanes (columns) contiguous: 64 of them by 64 of K
constexpr uint32_t FEW_ROWS = 32;                // rows of the smaller box
constexpr int NUM_THREADS = 384;
constexpr int NUM_EPI_WARPS = 8;
constexpr uint32_t TMEM_COLS = 512;
constexpr uint32_t DRAIN_STAGES = 2; // tcec: 128 k values per drain (tcec_gemm_pair.cu has the figures)
constexpr uint32_t BAND = 8;         // column tiles that are walked together
constexpr uint32_t AHEAD = 3;        // tiles that the roles may be apart
constexpr uint32_t WANT_BLOCKS = 4;  // blocks of a tile that are left to load when the next one is fetched
constexpr uint32_t TILE_WORDS = 12;  // of a Tile
constexpr uint32_t MIN_SLICED = 32;  // least blocks of K in a tile that is sliced, and in a slice of it
constexpr uint32_t MIN_SLICE = 8;
constexpr uint32_t MAX_SLICES = 16;
constexpr uint32_t JOIN_AHEAD = 4;   // slices whose sums are fetched together
constexpr uint32_t PART = COLS * BM_CTA; // elements of a parked sum of one CTA
constexpr uint32_t OUT_COLS = 32;    // columns that a warp stores at a time
constexpr uint32_t OUT_BYTES = OUT_COLS * 32 * 2; // 32 lanes of 16-bit elements

constexpr int kF16 = static_cast<int>(GroupedKind::f16), kTcec = static_cast<int>(GroupedKind::tcec),
              kI8 = static_cast<int>(GroupedKind::i8);

template <int KIND> struct Cfg {
  static constexpr uint32_t PLANES = KIND == kTcec ? 2 : 1;
  static constexpr uint32_t STAGE_BYTES = 2 * PLANES * TILE_BYTES;
  static constexpr uint32_t STAGES = KIND == kTcec ? 3 : 6;
  static constexpr uint32_t K_ELEMS = KIND == kI8 ? 128 : 64; // of K in a stage
  // What a step of K takes, in columns of products, and what a tile takes besides (about 3 us): a step is
  // as long as its products or its loads, 128 lanes and half the columns in each CTA.
  static __device__ __forceinline__ float step_cost(uint32_t cols) {
    return fmaxf(static_cast<float>(cols), LOADS * static_cast<float>(256u + cols));
  }
  static constexpr float LOADS = KIND == kTcec ? 0.4f : KIND == kF16 ? 0.5f : 0.8f;
  static constexpr float TILE_COST = KIND == kTcec ? 700.f : KIND == kF16 ? 2500.f : 5000.f;
  static constexpr uint32_t BARS = STAGES * STAGE_BYTES;      // offsets in shared memory
  static constexpr uint32_t FULL = BARS, EMPTY = FULL + 8 * STAGES, ACC_FULL = EMPTY + 8 * STAGES,
                            ACC_EMPTY = ACC_FULL + 16, TAIL = ACC_EMPTY + 16, NEXT_FULL = TAIL + 8 * STAGES,
                            NEXT_EMPTY = NEXT_FULL + 8 * AHEAD, WANT = NEXT_EMPTY + 8 * AHEAD, TMEM_PTR = WANT + 8,
                            ABORT = TMEM_PTR + 4, WIDTH = ABORT + 4, NEXT = BARS + 256, START = NEXT + AHEAD * TILE_WORDS * 4,
                            FIRST_TILE = START + 4 * (kMaxGroups + 2),
                            OUT = (FIRST_TILE + 4 * (kMaxGroups + 2) + 127) / 128 * 128,
                            BYTES = OUT + (KIND == kTcec ? 0 : NUM_EPI_WARPS * OUT_BYTES);
  static_assert(WIDTH + 4 <= NEXT && STAGES <= 32, "barriers and flags; phases are bits");
  static constexpr uint32_t SMEM = BYTES + 1024; // and what the alignment of the stages takes
};

struct GroupedParams {
  const int32_t *ends;
  void *out;
  uint64_t ldo, stride_o;
  const float *lane_scale; // i8; tcec: the two factors of `unscale`, or null
  const float *col_scale, *bias;
  float *parts;       // nullable: sums of slices, [slot][CTA rank][COLS][BM_CTA]
  unsigned *counters; // next tile, pairs that are through, then arrivals for each sliced tile, CTA and warp
  int *status;
  uint32_t rows, groups, lane_dim;
  uint32_t col_dim; // wgrad; product: steps of K
  uint32_t idesc;
  float alpha, beta;
  uint16_t out_type;
  uint16_t vector_out; // 16-bit results in rows that allow 16-byte accesses, and beta is 0
};
static_assert(sizeof(GroupedParams) <= 128, "read from the constant bank (gemm_common.cuh)");

// A tile, or a slice of one: `cols` columns from col0 on (of the rows of x, or wgrad: of a weight
// dimension), 256 lanes from lane0 on, steps [k0, k0 + blocks) of K.  Without any, its product is zero.
struct alignas(16) Tile {
  uint32_t group, lane0, col0, cols; // cols == 0: there are no more tiles
  uint32_t k0, blocks;
  uint32_t row0, rows;          // wgrad: the group's
  uint32_t slices, slice, slot; // slot: of the slice's sum; the tile's others follow or precede it
  uint32_t sliced;              // the tile's number
  __device__ __forceinline__ uint32_t width() const { return (cols + 31u) & ~31u; } // N of the product
  // wgrad: rows of the group in step kb of the slice
  __device__ __forceinline__ uint32_t rows_at(uint32_t kb) const { return min(64u, rows - (k0 + kb) * 64u); }
};
static_assert(sizeof(Tile) == TILE_WORDS * 4, "three times 16 bytes");

// The items of a launch, which are tiles or slices of tiles, by their numbers: groups in turn; within one,
// bands of column tiles that all lane tiles pass over, so that what runs at the same time shares
// operands in L2.
// Tiles that are at most half as many as pairs are cut into slices of K, whose sums are parked and added in
// the order of the slices by the warp that comes last.  A block of K takes 0.3 us (256 columns), and a
// slice adds 1.6 us for the SM that fetches its sums, so the sum of both is least with the square root
// of 50 * blocks / columns slices, and below 32 blocks with one (256 rows of 4096, one expert of 1024: 25 us
// whole, 21 so; 54 with 16 slices).  Slicing the last tiles of longer launches was no gain.
template <int KIND, bool WGRAD> struct Items {
  const uint32_t *start, *first_tile;
  uint32_t group, total, slices; // slices: item numbers of a tile
  uint32_t cols;                 // of a tile that is not a group's last
  __device__ __forceinline__ Items(const uint8_t *smem, const GroupedParams &p, uint32_t clusters) {
    start = reinterpret_cast<const uint32_t *>(smem + Cfg<KIND>::START);
    first_tile = reinterpret_cast<const uint32_t *>(smem + Cfg<KIND>::FIRST_TILE);
    group = 0;
    cols = *reinterpret_cast<const uint32_t *>(smem + Cfg<KIND>::WIDTH);
    const uint32_t tiles = first_tile[p.groups + 1];
    slices = p.parts != nullptr && tiles > 0 && tiles <= clusters / 2 ? min(clusters / tiles, MAX_SLICES) : 1u;
    total = tiles * slices;
  }
  // item < total, and not below that of an earlier call; false: it is none (a tile of few blocks has
  // fewer slices than others)
  __device__ __forceinline__ bool get(const GroupedParams &p, uint32_t item, Tile &x) {
    const uint32_t tile = slices > 1 ? item / slices : item;
    x.slices = 1;
    x.slice = 0;
    x.slot = item;
    x.sliced = tile;
    while (tile >= first_tile[group + 1]) ++group;
    const uint32_t r0 = start[group], r = start[group + 1] - r0;
    const uint32_t lane_tiles = (p.lane_dim + LANES - 1) / LANES;
    const uint32_t col_dim = WGRAD ? p.col_dim : r;
    const uint32_t col_tiles = (col_dim + cols - 1) / cols;
    const uint32_t local = tile - first_tile[group];
    const uint32_t band = local / (BAND * lane_tiles), in_band = local - band * BAND * lane_tiles;
    const uint32_t width = min(BAND, col_tiles - band * BAND);
    const uint32_t lt = in_band / width, ct = band * BAND + (in_band - lt * width);
    x.group = group;
    x.lane0 = lt * LANES;
    x.cols = min(cols, col_dim - ct * cols);
    x.col0 = ct * cols + (WGRAD ? 0u : r0);
    x.row0 = r0;
    x.rows = r;
    x.k0 = 0;
    x.blocks = WGRAD ? (r + 63u) / 64u : (group < p.groups ? p.col_dim : 0u);
    if (slices > 1) {
      const uint32_t all = x.blocks;
      if (all >= MIN_SLICED)
        x.slices = max(1u, min(min(slices, all / MIN_SLICE), static_cast<uint32_t>(sqrtf(50.f * all / x.cols))));
      x.slice = item - tile * slices;
      if (x.slice >= x.slices) return false;
      x.k0 = all * x.slice / x.slices;
      x.blocks = all * (x.slice + 1) / x.slices - x.k0;
    }
    return true;
  }
};

__device__ __forceinline__ void ld_shared_v4(uint32_t addr, uint32_t &x, uint32_t &y, uint32_t &z, uint32_t &w) {
  asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(x), "=r"(y), "=r"(z), "=r"(w) : "r"(addr));
}

// The tiles a role takes.  Their numbers come from a counter that all pairs share, as they get through:
// tiles differ in width (product) and depth (wgrad), and dealt in turn the slowest pair of the cases
// measured was up to a quarter behind the mean.  A warp of the leader fetches one when the producer has
// WANT_BLOCKS blocks of the last to load (a tile that is taken earlier waits where another pair may be
// idle), works it out, a handful of divisions, and sends it to both CTAs.
template <int KIND, bool WARP> struct Tiles { // taken by a warp, or by one thread
  uint32_t sbase, turn, phase;
  __device__ __forceinline__ explicit Tiles(uint32_t sbase_) : sbase(sbase_), turn(0), phase(0) {}
  // false at the end, or where the wait gave up
  __device__ __forceinline__ bool next(const GroupedParams &p, volatile int *abort_flag, Tile &x) {
    if (!look(p, abort_flag, x)) return false;
    take(x);
    return x.cols != 0;
  }
  // The same in two steps: the tile can be read again until it is taken.
  __device__ __forceinline__ bool look(const GroupedParams &p, volatile int *abort_flag, Tile &x) {
    bool ok = ptx::mbar_wait(sbase + Cfg<KIND>::NEXT_FULL + 8 * turn, phase, abort_flag, p.status,
                             ptx::kErrWaitTile);
    if (WARP) ok = ptx::warp_agrees(ok);
    if (ok) read(x);
    return ok;
  }
  __device__ __forceinline__ void read(Tile &x) const {
    const uint32_t at = sbase + Cfg<KIND>::NEXT + turn * sizeof(Tile);
    ld_shared_v4(at, x.group, x.lane0, x.col0, x.cols);
    ld_shared_v4(at + 16, x.k0, x.blocks, x.row0, x.rows);
    ld_shared_v4(at + 32, x.slices, x.slice, x.slot, x.sliced);
  }
  __device__ __forceinline__ void take(const Tile &x) {
    using C = Cfg<KIND>;
    // The slot is given back relaxed, so its three reads have to have come in: a word of each is compared (none
    // of these is ever ~0), by every lane that read.
    bool has_come = max(max(x.group, x.k0), x.slices) != ~0u;
    if (WARP) has_come = __all_sync(0xffffffffu, has_come) != 0 && (threadIdx.x & 31) == 0;
    if (has_come) ptx::mbar_arrive_cluster_relaxed(ptx::map_to_cta(sbase + C::NEXT_EMPTY + 8 * turn, 0));
    if (++turn == AHEAD) {
      turn = 0;
      phase ^= 1u;
    }
  }
};

// First row and first tile of each group, and the width of the tiles, by one warp.  What `ends` holds is
// never trusted: a total that falls back or passes the number of rows is taken as the one in front of it,
// or as that number.  The rows behind the last group are a group of their own (product: its tiles have no
// blocks; wgrad: it has no tiles).
template <int KIND, bool WGRAD>
__device__ __forceinline__ void find_groups(uint8_t *smem, const GroupedParams &p, uint32_t clusters) {
  uint32_t *start = reinterpret_cast<uint32_t *>(smem + Cfg<KIND>::START);
  uint32_t *first_tile = reinterpret_cast<uint32_t *>(smem + Cfg<KIND>::FIRST_TILE);
  const uint32_t lane = threadIdx.x & 31u;
  const uint32_t lane_tiles = (p.lane_dim + LANES - 1) / LANES;
  uint32_t end_before = 0, most = 0; // most rows of a group, of this lane's
  for (uint32_t g0 = 0; g0 < p.groups + 1; g0 += 32) {
    const uint32_t g = g0 + lane;
    uint32_t end = 0;
    if (g < p.groups)
      end = p.ends == nullptr ? p.rows
                              : static_cast<uint32_t>(min(max(__ldg(p.ends + g), 0),
                                                          static_cast<int32_t>(p.rows)));
    else if (g == p.groups) end = p.rows;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const uint32_t o = __shfl_up_sync(0xffffffffu, end, d);
      if (static_cast<int>(lane) >= d) end = max(end, o);
    }
    end = max(end, end_before);
    uint32_t begin = __shfl_up_sync(0xffffffffu, end, 1);
    if (lane == 0) begin = end_before;
    if (g <= p.groups) start[g] = begin;
    if (g == p.groups) start[g + 1] = end;
    most = max(most, end - begin);
    end_before = __shfl_sync(0xffffffffu, end, 31);
  }
  __syncwarp();
  // tiles of group g (for g == groups, the rows behind the last) that are `cols` wide
  auto tiles_of = [&](uint32_t g, uint32_t cols) {
    if (WGRAD) return g < p.groups ? lane_tiles * ((p.col_dim + cols - 1) / cols) : 0u;
    return lane_tiles * ((start[g + 1] - start[g] + cols - 1) / cols);
  };
  // The width.  With many tiles, the widest.  Else the one with the earliest end by this estimate: the
  // work shared by all pairs and half a tile, or the longest tile where there are no more tiles than
  // pairs.  (us with tiles of 256 / so: bfloat16 256 x 4096 x 1024 21.6 / 13.9, 1024^3 11.3 / 9.6, 1024 rows
  // over 4 experts of 2048 x 2048 23.4 / 15.9, over 4 of 1024 x 1024 in FP32 34.6 / 23.4; 16 rows over 8
  // experts, where there is nothing to choose, 8.6 / 8.8.)
  uint32_t cols = COLS;
  if (__any_sync(0xffffffffu, WGRAD ? p.col_dim > COLS >> (WIDTHS - 1) : most > COLS >> (WIDTHS - 1))) {
    uint32_t tiles[WIDTHS];
    float work[WIDTHS], longest[WIDTHS];
#pragma unroll
    for (uint32_t i = 0; i < WIDTHS; ++i) tiles[i] = 0, work[i] = longest[i] = 0.f;
    for (uint32_t g = lane; g <= p.groups; g += 32) {
      const uint32_t rows = start[g + 1] - start[g], col_dim = WGRAD ? p.col_dim : rows;
      if (col_dim == 0 || (WGRAD && g == p.groups)) continue;
      const float steps = static_cast<float>(WGRAD ? (rows + 63u) / 64u : g < p.groups ? p.col_dim : 0u);
#pragma unroll
      for (uint32_t i = 0; i < WIDTHS; ++i) {
        const uint32_t w = COLS >> i, whole = col_dim / w, rest = (col_dim - whole * w + 31u) & ~31u;
        const float wide = steps * Cfg<KIND>::step_cost(w) + Cfg<KIND>::TILE_COST,
                    narrow = steps * Cfg<KIND>::step_cost(rest) + Cfg<KIND>::TILE_COST;
        tiles[i] += lane_tiles * (whole + (rest > 0));
        work[i] += lane_tiles * (whole * wide + (rest > 0 ? narrow : 0.f));
        longest[i] = fmaxf(longest[i], whole > 0 ? wide : narrow);
      }
    }
    float best = 0.f;
#pragma unroll
    for (uint32_t i = 0; i < WIDTHS; ++i) {
      const uint32_t n = __reduce_add_sync(0xffffffffu, tiles[i]);
      if (i == 0 && n >= 4 * clusters) break;
      float sum = work[i];
#pragma unroll
      for (int d = 16; d > 0; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
      // (non-negative floats are ordered as their bits)
      const float most_of_one = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(longest[i])));
      const float ends_at = n <= clusters ? most_of_one : fmaxf(most_of_one, sum / clusters + 0.5f * most_of_one);
      if (i == 0 || ends_at < 0.95f * best) {
        best = ends_at;
        cols = COLS >> i;
      }
    }
  }
  uint32_t tiles_before = 0;
  for (uint32_t g0 = 0; g0 < p.groups + 1; g0 += 32) {
    const uint32_t g = g0 + lane;
    const uint32_t tiles = g <= p.groups ? tiles_of(g, cols) : 0u;
    uint32_t upto = tiles;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const uint32_t o = __shfl_up_sync(0xffffffffu, upto, d);
      if (static_cast<int>(lane) >= d) upto += o;
    }
    if (g <= p.groups) first_tile[g] = tiles_before + upto - tiles;
    if (g == p.groups) first_tile[g + 1] = tiles_before + upto;
    tiles_before += __shfl_sync(0xffffffffu, upto, 31);
  }
  if (lane == 0) *reinterpret_cast<uint32_t *>(smem + Cfg<KIND>::WIDTH) = cols;
}

template <int KIND>
__device__ __forceinline__ void mma(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
  if constexpr (KIND == kI8) ptx::mma_i8_ss_pair(d, a, b, idesc, acc);
  else ptx::mma_f16_ss_pair(d, a, b, idesc, acc);
}

__device__ __forceinline__ float load_as_float(const __half *p) { return __half2float(*p); }
__device__ __forceinline__ float load_as_float(const __nv_bfloat16 *p) { return __bfloat162float(*p); }
__device__ __forceinline__ float load_as_float(const float *p) { return *p; }
// the one rounding of a result to its type
__device__ __forceinline__ void store_from_float(__half *p, float v) { *p = __float2half_rn(v); }
__device__ __forceinline__ void store_from_float(__nv_bfloat16 *p, float v) { *p = __float2bfloat16_rn(v); }
__device__ __forceinline__ void store_from_float(float *p, float v) { *p = v; }

// drain_sums and add_corrections_in_tmem (epilogue.cuh) for the first `cols` columns, a multiple of 16.
// A warp's columns end where its neighbour's begin, and in a narrow tile that is short of COLS / 2.
__device__ __forceinline__ void drain_columns(uint32_t taddr, float (&sums)[COLS / 2], uint32_t cols) {
#pragma unroll
  for (uint32_t c = 0; c < COLS / 2; c += 16) {
    if (c >= cols) break;
    uint32_t v[16];
    ptx::tmem_ld_32x32b_x16(taddr + c, v);
    ptx::tmem_ld_wait();
#pragma unroll
    for (uint32_t i = 0; i < 16; ++i) {
      sums[c + i] += __uint_as_float(v[i]);
      asm volatile("" : "+f"(sums[c + i])); // added here and now, not where the sum is next used
    }
  }
}
__device__ __forceinline__ void add_corrections(uint32_t taddr, const float (&sums)[COLS / 2],
                                                uint32_t cols) {
#pragma unroll
  for (uint32_t c = 0; c < COLS / 2; c += 16) {
    if (c >= cols) break;
    uint32_t v[16];
    ptx::tmem_ld_32x32b_x16(taddr + c, v);
    ptx::tmem_ld_wait();
#pragma unroll
    for (uint32_t i = 0; i < 16; ++i)
      v[i] = __float_as_uint(fmaf(__uint_as_float(v[i]), 1.f / 2048.f, sums[c + i]));
    ptx::tmem_st_32x32b_x16(taddr + c, v);
  }
  ptx::tmem_st_wait();
}

// What turns a sum into a result, for one lane.
struct Finish {
  float f0, f1, add; // sum * f0 * f1 + add  (i8: f0 the lane's scale, f1 the column's)
  float beta;
};

template <int KIND>
__device__ __forceinline__ float result(uint32_t sum, float col_scale, const Finish &f) {
  if constexpr (KIND == kI8) return fmaf(__int2float_rn(static_cast<int>(sum)) * f.f0, col_scale, f.add);
  else return __uint_as_float(sum) * f.f0 * f.f1;
}
// two results to 16 bits, x in the low half
template <class T> __device__ __forceinline__ uint32_t pack_results(float x, float y) {
  uint32_t w;
  if constexpr (std::is_same_v<T, __nv_bfloat16>)
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(w) : "f"(y), "f"(x));
  else asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(w) : "f"(y), "f"(x));
  return w;
}

// A slice of a tile: its sums are parked, and the warp that is the last of the tile's slices to park the
// same lanes and columns adds them all, in the order of the slices, and leaves the total in tensor
// memory in place of its own.  Returns whether it was that warp.  Nothing waits.
template <int KIND>
__device__ __forceinline__ bool join_slices(const GroupedParams &p, const Tile &x, uint32_t rank,
                                            uint32_t warp, uint32_t col, uint32_t quarter,
                                            uint32_t taddr, uint32_t cols) {
  const uint32_t lane = threadIdx.x & 31u;
  const uint64_t at = static_cast<uint64_t>(col) * BM_CTA + quarter * 32u + lane;
  uint32_t *parts = reinterpret_cast<uint32_t *>(p.parts) + rank * static_cast<uint64_t>(PART) + at;
  uint32_t *mine = parts + static_cast<uint64_t>(x.slot) * 2 * PART;
#pragma unroll 1
  for (uint32_t c = 0; c < cols; c += 16) {
    uint32_t v[16];
    ptx::tmem_ld_32x32b_x16(taddr + c, v);
    ptx::tmem_ld_wait();
#pragma unroll
    for (uint32_t j = 0; j < 16; ++j) __stcg(mine + (c + j) * BM_CTA, v[j]);
  }
  __threadfence();
  __syncwarp();
  uint32_t before = 0;
  if (lane == 0)
    before = atomicInc(p.counters + 2 + (x.sliced * 2 + rank) * NUM_EPI_WARPS + warp, x.slices - 1);
  if (__shfl_sync(0xffffffffu, before, 0) != x.slices - 1) return false;
  __threadfence();
  const uint32_t *first = parts + static_cast<uint64_t>(x.slot - x.slice) * 2 * PART;
#pragma unroll 1
  for (uint32_t c = 0; c < cols; c += 16) {
    uint32_t v[16];
#pragma unroll
    for (uint32_t j = 0; j < 16; ++j) v[j] = 0;
    // several slices' values are on their way at once: one slice after the other took 2.8 us each for
    // 256 columns
#pragma unroll 1
    for (uint32_t s = 0; s < x.slices; s += JOIN_AHEAD) {
      uint32_t y[JOIN_AHEAD][16];
#pragma unroll
      for (uint32_t i = 0; i < JOIN_AHEAD; ++i)
#pragma unroll
        for (uint32_t j = 0; j < 16; ++j)
          y[i][j] = s + i < x.slices ? __ldcg(first + static_cast<uint64_t>(s + i) * 2 * PART + (c + j) * BM_CTA) : 0u;
#pragma unroll
      for (uint32_t i = 0; i < JOIN_AHEAD; ++i)
#pragma unroll
        for (uint32_t j = 0; j < 16; ++j)
          v[j] = KIND == kI8 ? v[j] + y[i][j] : __float_as_uint(__uint_as_float(v[j]) + __uint_as_float(y[i][j]));
    }
    ptx::tmem_st_32x32b_x16(taddr + c, v);
  }
  ptx::tmem_st_wait();
  return true;
}

// `cols` columns of one lane from tensor memory (zero: there is no sum, the product is 0) to global
// memory, column c at out + c * ldo.  A warp's lanes hold neighbouring elements.  The loop body has no
// branches but the one for its own group: with one for each element's bounds and beta 16 columns took
// 1500 cycles.
template <int KIND, class T, bool BETA>
__device__ __forceinline__ void store_columns(uint32_t taddr, bool zero, T *out, uint64_t ldo,
                                              uint32_t cols, bool lane_ok, const Finish &f,
                                              const float *col_scale) {
  constexpr uint32_t G = kEpiGroup;
  const uint32_t lane = threadIdx.x & 31u;
#pragma unroll 1
  for (uint32_t c = 0; c < cols; c += G) {
    float cs = 1.f;
    if constexpr (KIND == kI8) {
      if (lane < G && c + lane < cols) cs = __ldg(col_scale + c + lane);
    }
    uint32_t v[G];
    float old[G], x[G];
    const uint32_t here = lane_ok ? cols - c : 0u; // columns that this lane stores
    T *at = out;
    if constexpr (BETA) {
#pragma unroll
      for (uint32_t j = 0; j < G; ++j, at += ldo) old[j] = j < here ? load_as_float(at) : 0.f;
      at = out;
    }
    if (!zero) {
      ptx::tmem_ld_32x32b_x16(taddr + c, v);
      ptx::tmem_ld_wait();
    }
#pragma unroll
    for (uint32_t j = 0; j < G; ++j) {
      x[j] = result<KIND>(v[j], KIND == kI8 ? __shfl_sync(0xffffffffu, cs, j) : 1.f, f);
      if (zero) x[j] = 0.f;
      if constexpr (BETA) x[j] = fmaf(f.beta, old[j], x[j]);
    }
#pragma unroll
    for (uint32_t j = 0; j < G; ++j, at += ldo)
      if (j < here) store_from_float(at, x[j]);
    out = at;
  }
}
template <int KIND, class T>
__device__ __forceinline__ void store_columns(uint32_t taddr, bool zero, T *out, uint64_t ldo,
                                              uint32_t cols, bool lane_ok, const Finish &f,
                                              const float *col_scale) {
  if (KIND != kI8 && f.beta != 0.f)
    store_columns<KIND, T, true>(taddr, zero, out, ldo, cols, lane_ok, f, col_scale);
  else store_columns<KIND, T, false>(taddr, zero, out, ldo, cols, lane_ok, f, col_scale);
}

// The same for 16-bit results in rows that allow 16-byte accesses, 32 columns at a time: read as fragments,
// stored transposed to the warp's own buffer in shared memory (64 bytes for each column, the 16-byte
// chunks of two columns side by side XORed so that neither side meets a bank twice), and from there 16 bytes
// a lane.  Stored from the registers, 2 bytes a lane, a 256 x 256 tile took 7 to 11 us; 2 bytes a lane
// into shared memory the gradient of 64 experts of 2000 x 1000 took 98 us, and this way 93.
template <int KIND, class T>
__device__ __forceinline__ void store_by_rows(uint32_t taddr, bool zero, T *out, uint64_t ldo,
                                              uint32_t buf, uint32_t cols, uint32_t lanes,
                                              const Finish (&f)[4], const float *col_scale) {
  const uint32_t lane = threadIdx.x & 31u;
  const uint32_t chunk = lane & 3u; // of 8 elements
  const uint32_t elems = lanes > 8 * chunk ? min(lanes - 8 * chunk, 8u) : 0u; // of it, that there are
  // this thread's matrix row on the way in, and its 16 bytes of every 8 columns on the way out
  const uint32_t in = buf + (lane & 7u) * 64u + (((lane >> 3) ^ ((lane >> 1) & 3u)) << 4);
  const uint32_t back = buf + (lane >> 2) * 64u + ((chunk ^ ((lane >> 3) & 3u)) << 4);
  const uint64_t step = 8 * ldo;
  T *at = out + (lane >> 2) * ldo + 8 * chunk;
#pragma unroll 1
  for (uint32_t c = 0; c < cols; c += OUT_COLS) {
    uint32_t w[4][4];
    if (!zero) {
      uint32_t lo[16], hi[16];
      float cs[8];
      ptx::tmem_ld_16x256b_x4(taddr + c, lo);
      ptx::tmem_ld_16x256b_x4(taddr + c + (16u << 16), hi);
      if constexpr (KIND == kI8) {
#pragma unroll
        for (uint32_t i = 0; i < 8; ++i) {
          const uint32_t col = c + (i >> 1) * 8 + 2 * chunk + (i & 1);
          cs[i] = col < cols ? __ldg(col_scale + col) : 0.f;
        }
      }
      ptx::tmem_ld_wait();
#pragma unroll
      for (uint32_t g = 0; g < 4; ++g) {
        const float s0 = KIND == kI8 ? cs[2 * g] : 1.f, s1 = KIND == kI8 ? cs[2 * g + 1] : 1.f;
#pragma unroll
        for (uint32_t i = 0; i < 4; ++i) {
          const uint32_t x = i < 2 ? lo[4 * g + 2 * i] : hi[4 * g + 2 * i - 4],
                         y = i < 2 ? lo[4 * g + 2 * i + 1] : hi[4 * g + 2 * i - 3];
          w[g][i] = pack_results<T>(result<KIND>(x, s0, f[i]), result<KIND>(y, s1, f[i]));
        }
      }
    } else {
#pragma unroll
      for (uint32_t g = 0; g < 4; ++g) w[g][0] = w[g][1] = w[g][2] = w[g][3] = 0;
    }
    __syncwarp(); // the buffer has been read
#pragma unroll
    for (uint32_t g = 0; g < 4; ++g)
      ptx::stmatrix_x4_trans(in + g * 512u, w[g][0], w[g][1], w[g][2], w[g][3]);
    __syncwarp();
    const uint32_t first = c + (lane >> 2);
#pragma unroll
    for (uint32_t g = 0; g < 4; ++g)
      ld_shared_v4(back + g * 512u, w[g][0], w[g][1], w[g][2], w[g][3]);
#pragma unroll
    for (uint32_t g = 0; g < 4; ++g)
      if (first + 8 * g < cols && elems == 8)
        *reinterpret_cast<uint4 *>(at + g * step) = make_uint4(w[g][0], w[g][1], w[g][2], w[g][3]);
    if (elems > 0 && elems < 8) { // the last lanes of a width that is no multiple of 8
#pragma unroll
      for (uint32_t g = 0; g < 4; ++g)
        if (first + 8 * g < cols)
          for (uint32_t i = 0; i < elems; ++i) {
            const uint32_t e = i < 4 ? (i < 2 ? w[g][0] : w[g][1]) : (i < 6 ? w[g][2] : w[g][3]);
            reinterpret_cast<uint16_t *>(at + g * step)[i] = static_cast<uint16_t>(e >> (16 * (i & 1)));
          }
    }
    at += 4 * step;
  }
}

template <int KIND, bool A_LANES, bool WGRAD>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(NUM_THREADS, 1)
    grouped_gemm_kernel(const __grid_constant__ CUtensorMap map_a,
                        const __grid_constant__ CUtensorMap map_b,
                        const __grid_constant__ CUtensorMap map_b_few,
                        const GroupedParams p) {
  using C = Cfg<KIND>;
  constexpr uint32_t PLANES = C::PLANES, STAGES = C::STAGES, STAGE_BYTES = C::STAGE_BYTES;
  extern __shared__ uint8_t smem_raw[];
  uint8_t *const smem = reinterpret_cast<uint8_t *>(
      (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  const uint32_t sbase = ptx::smem_u32(smem);
  volatile int *const abort_flag = reinterpret_cast<volatile int *>(smem + C::ABORT);

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const uint32_t rank = ptx::cluster_ctarank();
  const bool leader = rank == 0;
  const uint32_t cluster_id = blockIdx.x >> 1;
  const uint32_t clusters = gridDim.x >> 1;

  if (threadIdx.x == 0) {
    for (uint32_t s = 0; s < STAGES; ++s) {
      ptx::mbar_init(sbase + C::FULL + 8 * s, 2);
      ptx::mbar_init(sbase + C::EMPTY + 8 * s, 1);
      ptx::mbar_init(sbase + C::TAIL + 8 * s, 1);
    }
    for (uint32_t b = 0; b < 2; ++b) {
      ptx::mbar_init(sbase + C::ACC_FULL + 8 * b, 1);
      ptx::mbar_init(sbase + C::ACC_EMPTY + 8 * b, 2 * NUM_EPI_WARPS);
    }
    *abort_flag = 0;
    for (uint32_t i = 0; i < AHEAD; ++i) {
      ptx::mbar_init(sbase + C::NEXT_FULL + 8 * i, 1);
      // taken by the issuer, and in both CTAs by producer, epilogue warps and (wgrad) the warp for last blocks
      ptx::mbar_init(sbase + C::NEXT_EMPTY + 8 * i, 1 + 2 * (1 + NUM_EPI_WARPS + (WGRAD ? 1 : 0)));
    }
    ptx::mbar_init(sbase + C::WANT, 1);
    ptx::mbar_init_fence();
    ptx::prefetch_tensormap(&map_a);
    ptx::prefetch_tensormap(&map_b);
    if (!WGRAD) ptx::prefetch_tensormap(&map_b_few);
  }
  if (warp == 1) {
    ptx::tmem_alloc_pair(sbase + C::TMEM_PTR, TMEM_COLS);
    ptx::tmem_relinquish_pair();
  }
  // Everything above needs nothing of the kernel in front, everything below may.  The kernel behind is
  // not let in early: pairs end one by one, and the blocks of a pass over rows would crowd on the SMs that
  // are free first (FP32, 192 rows over 7 experts of 6469 x 2804, calls back to back: 513 us instead of 407).
  ptx::griddep_wait();
  if (warp == 2) find_groups<KIND, WGRAD>(smem, p, clusters);
  ptx::tc_fence_before();
  __syncthreads();
  // both CTAs' barriers must exist before any remote arrive / remote TMA completion
  ptx::cluster_arrive();
  ptx::cluster_wait();
  ptx::tc_fence_after();
  const uint32_t tmem_base = *reinterpret_cast<const uint32_t *>(smem + C::TMEM_PTR);

  if (warp == 0) {
    // ================================================================ TMA producer (both CTAs)
    if (ptx::elect_one()) {
      uint32_t s = 0, ph = 1;
      bool ok = true;
      Tiles<KIND, false> tiles(sbase);
      Tile x;
      while (ok && tiles.next(p, abort_flag, x)) {
        const int a_lane = static_cast<int>(x.lane0 + rank * BM_CTA);
        const uint32_t half = x.width() / 2;
        const int b_col = static_cast<int>(x.col0 + rank * half);
        // boxes of the column operand: of 64 columns (wgrad), one of 128 rows, or as many of 32 as it takes
        const bool whole_box = !WGRAD && half > 128 - FEW_ROWS;
        const uint32_t boxes = WGRAD ? (half + 63u) / 64u
                                     : (whole_box ? 1u : (half + FEW_ROWS - 1u) / FEW_ROWS);
        const uint32_t bytes =
            PLANES * (TILE_BYTES + boxes * (WGRAD ? ATOM_BYTES : whole_box ? TILE_BYTES : FEW_ROWS * ROW_BYTES));
        const uint32_t want = x.blocks > WANT_BLOCKS ? x.blocks - WANT_BLOCKS : 0u;
        if (leader && x.blocks == 0) ptx::mbar_arrive(sbase + C::WANT);
        for (uint32_t kb = 0; kb < x.blocks; ++kb) {
          if (leader && kb == want) ptx::mbar_arrive(sbase + C::WANT);
          ok = ptx::mbar_wait(sbase + C::EMPTY + 8 * s, ph, abort_flag, p.status, ptx::kErrWaitEmpty);
          if (!ok) break;
          const uint32_t st = sbase + s * STAGE_BYTES;
          const uint32_t full = ptx::map_to_cta(sbase + C::FULL + 8 * s, 0); // the leader's barrier
          const bool tail = WGRAD && x.rows_at(kb) < 64u;
          if (tail) ptx::mbar_arrive_expect_tx(sbase + C::TAIL + 8 * s, bytes);
          else if (leader) ptx::mbar_arrive_expect_tx(sbase + C::FULL + 8 * s, 2 * bytes);
          else ptx::mbar_arrive_cluster(full);
          auto load = [&](uint32_t dst, const CUtensorMap *m, int c0, int c1, int c2) {
            if (tail) ptx::tma_load_3d(dst, m, sbase + C::TAIL + 8 * s, c0, c1, c2);
            else ptx::tma_load_3d_pair(dst, m, full, c0, c1, c2);
          };
          const int red = static_cast<int>(WGRAD ? x.row0 + (x.k0 + kb) * 64u : (x.k0 + kb) * C::K_ELEMS);
#pragma unroll
          for (uint32_t pl = 0; pl < PLANES; ++pl) {
            const uint32_t a_dst = st + pl * TILE_BYTES, b_dst = st + (PLANES + pl) * TILE_BYTES;
            const int za = static_cast<int>(WGRAD ? pl : pl * p.groups + x.group);
            if constexpr (A_LANES) {
              load(a_dst, &map_a, a_lane, red, za);
              load(a_dst + ATOM_BYTES, &map_a, a_lane + 64, red, za);
            } else {
              load(a_dst, &map_a, red, a_lane, za);
            }
            if constexpr (WGRAD) {
              for (uint32_t b = 0; b < boxes; ++b)
                load(b_dst + b * ATOM_BYTES, &map_b, b_col + static_cast<int>(64 * b), red,
                     static_cast<int>(pl));
            } else if (whole_box) {
              load(b_dst, &map_b, red, b_col, static_cast<int>(pl));
            } else {
              for (uint32_t b = 0; b < boxes; ++b)
                load(b_dst + b * FEW_ROWS * ROW_BYTES, &map_b_few, red,
                     b_col + static_cast<int>(FEW_ROWS * b), static_cast<int>(pl));
            }
          }
          if (++s == STAGES) {
            s = 0;
            ph ^= 1u;
          }
        }
      }
    }
  } else if (WGRAD && warp == 2) {
    // ================================================================ last blocks of groups (both CTAs)
    uint32_t at = 0;    // stage uses in front of this tile's
    uint32_t phases = 0; // bit s: the phase of TAIL[s]
    bool ok = true;
    Tiles<KIND, true> tiles(sbase);
    Tile x;
    while (ok && tiles.next(p, abort_flag, x)) {
      at += x.blocks;
      if (x.blocks == 0 || x.rows_at(x.blocks - 1) == 64u) continue;
      const uint32_t s = (at - 1) % STAGES, st = sbase + s * STAGE_BYTES;
      ok = ptx::warp_agrees(ptx::mbar_wait_backoff(sbase + C::TAIL + 8 * s, (phases >> s) & 1u, abort_flag,
                                                   p.status, ptx::kErrWaitFull, 32));
      if (!ok) break;
      phases ^= 1u << s;
      // (a row of 128 bytes is a row of 128 bytes under the swizzle too)
      const uint32_t rows_here = x.rows_at(x.blocks - 1), upto = (rows_here + 15u) & ~15u;
      const uint32_t boxes = (x.width() / 2 + 63u) / 64u;
      for (uint32_t pl = 0; pl < PLANES; ++pl)
        for (uint32_t i = 0; i < 2 + boxes; ++i) {
          const uint32_t atom = st + (i < 2 ? pl : PLANES + pl) * TILE_BYTES + (i < 2 ? i : i - 2) * ATOM_BYTES;
          for (uint32_t b = rows_here * ROW_BYTES + 16u * lane; b < upto * ROW_BYTES; b += 512u)
            st_shared_v4(atom + b, 0u, 0u, 0u, 0u);
        }
      fence_proxy_async_shared();
      __syncwarp();
      if (lane == 0) ptx::mbar_arrive_cluster(ptx::map_to_cta(sbase + C::FULL + 8 * s, 0));
    }
  } else if (warp == 1) {
    // ================================================================ MMA issuer (leader only)
    if (leader && ptx::elect_one()) {
      constexpr uint16_t BOTH = 0x3;
      constexpr uint64_t kStage = STAGE_BYTES >> 4, kTile = TILE_BYTES >> 4;
      constexpr uint32_t A_STEP = A_LANES ? 2048 >> 4 : 2, B_STEP = WGRAD ? 2048 >> 4 : 2;
      const uint64_t a0 = A_LANES ? ptx::make_mnmajor_desc(sbase, ATOM_BYTES)
                                  : ptx::make_kmajor_desc<ROW_BYTES>(sbase);
      const uint32_t b_addr = sbase + PLANES * TILE_BYTES;
      const uint64_t b0 = WGRAD ? ptx::make_mnmajor_desc(b_addr, ATOM_BYTES)
                                : ptx::make_kmajor_desc<ROW_BYTES>(b_addr);
      uint32_t s = 0, ph = 0;
      uint32_t acc = 0, e_ph = 1;          // accumulator in turn (f16, i8) and the phase of its barrier
      uint32_t d0_ph = 1, d1_ph = 1;       // tcec
      bool ok = true;
      Tiles<KIND, false> tiles(sbase);
      Tile x;
      while (ok && tiles.next(p, abort_flag, x)) {
        if (x.blocks == 0) continue;
        const uint32_t idesc = p.idesc | ((x.width() >> 3) << 17);
        if constexpr (KIND != kTcec) {
          ok = ptx::mbar_wait(sbase + C::ACC_EMPTY + 8 * acc, e_ph, abort_flag, p.status,
                              ptx::kErrWaitD0Empty);
          if (!ok) break;
          ptx::tc_fence_after();
        }
        const uint32_t d = tmem_base + acc * COLS;
        for (uint32_t kb = 0; kb < x.blocks; ++kb) {
          ok = ptx::mbar_wait(sbase + C::FULL + 8 * s, ph, abort_flag, p.status, ptx::kErrWaitFull);
          if (!ok) break;
          ptx::tc_fence_after();
          const uint64_t a = a0 + s * kStage, b = b0 + s * kStage;
          const uint32_t steps = WGRAD ? (x.rows_at(kb) + 15u) / 16u : 4u;
          if constexpr (KIND != kTcec) {
#pragma unroll
            for (uint32_t ks = 0; ks < 4; ++ks)
              if (!WGRAD || ks < steps)
                mma<KIND>(d, a + A_STEP * ks, b + B_STEP * ks, idesc, (kb | ks) != 0);
          } else {
            const bool first = kb % DRAIN_STAGES == 0;
            auto corrections = [&](uint32_t acc_first) {
#pragma unroll
              for (uint32_t ks = 0; ks < 4; ++ks)
                if (!WGRAD || ks < steps)
                  mma<KIND>(tmem_base + COLS, a + kTile + A_STEP * ks, b + B_STEP * ks, idesc,
                            ks > 0 ? 1u : acc_first);
#pragma unroll
              for (uint32_t ks = 0; ks < 4; ++ks)
                if (!WGRAD || ks < steps)
                  mma<KIND>(tmem_base + COLS, a + A_STEP * ks, b + kTile + B_STEP * ks, idesc, 1u);
            };
            // The corrections of a chunk's first stage come before its hi*hi products: the drain of
            // the previous chunk hides behind them.  In a tile's first stage they wait for the
            // epilogue to give their accumulator back, so they come last.
            if (first && kb > 0) corrections(1u);
            if (first) {
              ok = ptx::mbar_wait(sbase + C::ACC_EMPTY, d0_ph, abort_flag, p.status,
                                  ptx::kErrWaitD0Empty);
              if (!ok) break;
              d0_ph ^= 1u;
              ptx::tc_fence_after();
            }
#pragma unroll
            for (uint32_t ks = 0; ks < 4; ++ks)
              if (!WGRAD || ks < steps)
                mma<KIND>(tmem_base, a + A_STEP * ks, b + B_STEP * ks, idesc, !first || ks > 0);
            if (kb % DRAIN_STAGES == DRAIN_STAGES - 1 || kb + 1 == x.blocks)
              ptx::tc_commit_pair(sbase + C::ACC_FULL, BOTH);
            if (!(first && kb > 0)) {
              if (kb == 0) {
                ok = ptx::mbar_wait(sbase + C::ACC_EMPTY + 8, d1_ph, abort_flag, p.status,
                                    ptx::kErrWaitD1Empty);
                if (!ok) break;
                d1_ph ^= 1u;
                ptx::tc_fence_after();
              }
              corrections(kb > 0 ? 1u : 0u);
            }
          }
          ptx::tc_commit_pair(sbase + C::EMPTY + 8 * s, BOTH);
          if (++s == STAGES) {
            s = 0;
            ph ^= 1u;
          }
        }
        if (!ok) break;
        if constexpr (KIND == kTcec) {
          ptx::tc_commit_pair(sbase + C::ACC_FULL + 8, BOTH);
        } else {
          ptx::tc_commit_pair(sbase + C::ACC_FULL + 8 * acc, BOTH);
          acc ^= 1u;
          if (acc == 0) e_ph ^= 1u;
        }
      }
    }
  } else if (warp == 3) {
    // ================================================================ the next tiles (leader only)
    if (leader && ptx::elect_one()) {
      Items<KIND, WGRAD> items(smem, p, clusters);
      Tile x;
      uint32_t turn = 0, ph = 1, want = 0, item = cluster_id; // the first is the pair's own
      bool more = true;
      while (more) {
        while (item < items.total && !items.get(p, item, x)) item = clusters + atomicAdd(p.counters, 1u);
        more = item < items.total;
        if (!more) x = Tile{};
        if (!ptx::mbar_wait(sbase + C::NEXT_EMPTY + 8 * turn, ph, abort_flag, p.status, ptx::kErrWaitTile))
          break;
#pragma unroll
        for (uint32_t r = 0; r < 2; ++r) {
          const uint32_t to = ptx::map_to_cta(sbase + C::NEXT + turn * sizeof(Tile), r),
                         bar = ptx::map_to_cta(sbase + C::NEXT_FULL + 8 * turn, r);
          ptx::mbar_arrive_expect_tx_cluster(bar, sizeof(Tile));
          ptx::send_words(to, make_uint4(x.group, x.lane0, x.col0, x.cols), bar);
          ptx::send_words(to + 16, make_uint4(x.k0, x.blocks, x.row0, x.rows), bar);
          ptx::send_words(to + 32, make_uint4(x.slices, x.slice, x.slot, x.sliced), bar);
        }
        if (++turn == AHEAD) {
          turn = 0;
          ph ^= 1u;
        }
        if (more) {
          if (!ptx::mbar_wait(sbase + C::WANT, want, abort_flag, p.status, ptx::kErrWaitTile)) break;
          want ^= 1u;
          item = clusters + atomicAdd(p.counters, 1u);
        }
      }
      // the last pair to get here leaves the counter as it was found; the other wraps by itself
      if (atomicInc(p.counters + 1, clusters - 1) == clusters - 1) atomicExch(p.counters, 0u);
    }
  } else if (warp >= 4) {
    // ================================================================ epilogue (both CTAs)
    const uint32_t quarter = static_cast<uint32_t>(warp & 3), second = static_cast<uint32_t>(warp - 4) >> 2;
    const uint32_t t_lanes = tmem_base + ((quarter * 32u) << 16);
    const uint32_t acc_empty = ptx::map_to_cta(sbase + C::ACC_EMPTY, 0);
    const uint32_t buf = sbase + C::OUT + static_cast<uint32_t>(warp - 4) * OUT_BYTES;
    uint32_t acc = 0, f_ph = 0, d0_ph = 0, d1_ph = 0;
    bool ok = true;
    Tiles<KIND, true> tiles(sbase);
    Tile x;
    // The reads of tensor memory are complete (wait::ld): that is all there is to order.  (As a release
    // it also waited for the results to be written, 1 to 2 us a tile.)
    auto release = [&](uint32_t b) {
      ptx::tc_fence_before();
      __syncwarp();
      if (lane == 0) ptx::mbar_arrive_cluster_relaxed(acc_empty + 8 * b);
    };
    auto give_back = [&]() { // the accumulator that held the sums
      if constexpr (KIND == kTcec) {
        release(1);
      } else {
        release(acc);
        acc ^= 1u;
        if (acc == 0) f_ph ^= 1u;
      }
    };
    while (true) {
      if constexpr (KIND == kTcec) ok = tiles.look(p, abort_flag, x) && x.cols != 0;
      else ok = tiles.next(p, abort_flag, x);
      if (!ok) break;
      uint32_t t_sums = t_lanes + second * (x.width() / 2);
      if constexpr (KIND == kTcec) {
        // (the sums take the registers that the tile was in: it is read again behind them)
        const uint32_t half = x.width() / 2;
        const bool zero = x.blocks == 0;
        if (!zero) {
          float sums[COLS / 2];
#pragma unroll
          for (uint32_t i = 0; i < COLS / 2; ++i) sums[i] = 0.f;
          const uint32_t chunks = (x.blocks + DRAIN_STAGES - 1) / DRAIN_STAGES;
#pragma unroll 1
          for (uint32_t c = 0; c < chunks; ++c) {
            ok = ptx::warp_agrees(ptx::mbar_wait(sbase + C::ACC_FULL, d0_ph, abort_flag, p.status,
                                                 ptx::kErrWaitD0Full));
            if (!ok) break;
            d0_ph ^= 1u;
            ptx::tc_fence_after();
            drain_columns(t_sums, sums, half);
            release(0);
          }
          if (!ok) break;
          ok = ptx::warp_agrees(ptx::mbar_wait(sbase + C::ACC_FULL + 8, d1_ph, abort_flag, p.status,
                                               ptx::kErrWaitD1Full));
          if (!ok) break;
          d1_ph ^= 1u;
          ptx::tc_fence_after();
          add_corrections(t_sums + COLS, sums, half);
        }
        tiles.read(x);
        tiles.take(x);
        t_sums = t_lanes + second * (x.width() / 2) + COLS;
      } else if (x.blocks != 0) {
        ok = ptx::warp_agrees(ptx::mbar_wait(sbase + C::ACC_FULL + 8 * acc, f_ph, abort_flag, p.status,
                                             ptx::kErrWaitD0Full));
        if (!ok) break;
        ptx::tc_fence_after();
        t_sums += acc * COLS;
      }
      const uint32_t half = x.width() / 2;
      const bool zero = x.blocks == 0;
      if (x.slices > 1 && !join_slices<KIND>(p, x, rank, static_cast<uint32_t>(warp - 4), second * half,
                                             quarter, t_sums, min(half, x.width() - second * half))) {
        give_back();
        continue;
      }
      const uint32_t lane0 = x.lane0 + rank * BM_CTA + quarter * 32u; // the warp's first
      const uint32_t col = second * half;
      const uint32_t cols = x.cols > col && lane0 < p.lane_dim ? min(half, x.cols - col) : 0u;
      const uint64_t at = (WGRAD ? x.group * p.stride_o : 0ull) +
                          static_cast<uint64_t>(x.col0 + col) * p.ldo + lane0;
      const float *col_scale = KIND == kI8 ? p.col_scale + x.col0 + col : nullptr;
      auto finish_of = [&](uint32_t l) { // of lane lane0 + l
        Finish f = {p.alpha, 1.f, 0.f, p.beta};
        if constexpr (KIND == kI8) {
          f.f0 = 0.f;
          if (!zero && lane0 + l < p.lane_dim) {
            const uint64_t feature = static_cast<uint64_t>(x.group) * p.lane_dim + lane0 + l;
            f.f0 = __ldg(p.lane_scale + feature);
            if (p.bias != nullptr) f.add = __ldg(p.bias + feature);
          }
        } else if (KIND == kTcec && p.lane_scale != nullptr) {
          f.f0 = p.alpha * __ldg(p.lane_scale);
          f.f1 = __ldg(p.lane_scale + 1);
        }
        return f;
      };
      const auto type = static_cast<GroupedOut>(p.out_type);
      if (KIND != kTcec && p.vector_out != 0) {
        const uint32_t l = static_cast<uint32_t>(lane) >> 2;
        const Finish f[4] = {finish_of(l), finish_of(l + 8), finish_of(l + 16), finish_of(l + 24)};
        const uint32_t lanes = p.lane_dim > lane0 ? p.lane_dim - lane0 : 0u;
        if (type == GroupedOut::bf16)
          store_by_rows<KIND>(t_sums, zero, static_cast<__nv_bfloat16 *>(p.out) + at, p.ldo, buf, cols, lanes, f, col_scale);
        else
          store_by_rows<KIND>(t_sums, zero, static_cast<__half *>(p.out) + at, p.ldo, buf, cols, lanes, f, col_scale);
      } else {
        const Finish f = finish_of(static_cast<uint32_t>(lane));
        const bool lane_ok = lane0 + static_cast<uint32_t>(lane) < p.lane_dim;
        const uint64_t mine = at + static_cast<uint32_t>(lane);
        if (KIND != kF16 && type == GroupedOut::f32)
          store_columns<KIND>(t_sums, zero, static_cast<float *>(p.out) + mine, p.ldo, cols, lane_ok, f, col_scale);
        else if (KIND != kTcec && type == GroupedOut::bf16)
          store_columns<KIND>(t_sums, zero, static_cast<__nv_bfloat16 *>(p.out) + mine, p.ldo, cols, lane_ok, f, col_scale);
        else if (KIND != kTcec)
          store_columns<KIND>(t_sums, zero, static_cast<__half *>(p.out) + mine, p.ldo, cols, lane_ok, f, col_scale);
      }
      if (!zero) give_back();
    }
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

// Per device and kernel, once (any thread): shared-memory attribute and the pairs the device keeps
// resident.  (A kernel of each instance has a type of its own here: its statics are its own.)
template <int KIND, bool A_LANES, bool WGRAD> cudaError_t set_up(int *clusters_out) {
  static std::once_flag once[64];
  static cudaError_t setup_error[64];
  static int max_clusters[64];
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev < 0 || dev >= 64) return cudaErrorInvalidDevice;
  std::call_once(once[dev], [&]() {
    const auto kernel = grouped_gemm_kernel<KIND, A_LANES, WGRAD>;
    setup_error[dev] = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                            Cfg<KIND>::SMEM);
    int sms = 0;
    cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
    int clusters = sms / 2;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(static_cast<unsigned>(2 * clusters));
    cfg.blockDim = dim3(NUM_THREADS);
    cfg.dynamicSmemBytes = Cfg<KIND>::SMEM;
    int active = 0;
    if (setup_error[dev] == cudaSuccess &&
        cudaOccupancyMaxActiveClusters(&active, kernel, &cfg) == cudaSuccess) {
      if (active > 0 && active < clusters) clusters = active;
    } else {
      cudaGetLastError();
    }
    max_clusters[dev] = clusters > 0 ? clusters : 1;
  });
  *clusters_out = max_clusters[dev];
  return setup_error[dev];
}

// `inner_box` by `outer_box` elements; with nothing in it (no rows at all) the map is of one row, which
// no load asks for.
bool operand_map(CUtensorMap *map, const GroupedOperand &o, int elem_bytes, const void *fallback,
                 uint32_t inner_box, uint32_t outer_box) {
  const uint64_t es = static_cast<uint64_t>(elem_bytes), planes = static_cast<uint64_t>(o.batch) * o.planes;
  const uint64_t matrix = o.batch > 1 ? o.stride : (o.planes > 1 ? o.plane_stride : o.ld);
  return make_byte_map(map, elem_bytes, o.outer > 0 ? o.ptr : fallback,
                       {o.inner, o.outer > 0 ? o.outer : 1, planes}, {o.ld * es, matrix * es},
                       {inner_box, outer_box, 1}, true);
}

template <int KIND, bool A_LANES, bool WGRAD>
cudaError_t launch(const GroupedArgs &a, cudaStream_t stream) {
  int clusters = 1;
  const cudaError_t se = set_up<KIND, A_LANES, WGRAD>(&clusters);
  if (se != cudaSuccess) return se;
  constexpr int ES = KIND == kI8 ? 1 : 2;
  CUtensorMap map_a, map_b, map_b_few;
  // (any address does for an operand without rows; this one is 16-byte aligned)
  const void *fallback = a.dev_status;
  if (!operand_map(&map_a, a.a, ES, fallback, Cfg<KIND>::K_ELEMS, A_LANES ? 64 : BM_CTA) ||
      !operand_map(&map_b_few, a.b, ES, fallback, Cfg<KIND>::K_ELEMS, WGRAD ? 64 : FEW_ROWS))
    return cudaErrorInvalidValue;
  // boxes of 128 rows are for tiles of more than 192
  map_b = map_b_few;
  if (!WGRAD && a.rows > 2 * (128 - FEW_ROWS) &&
      !operand_map(&map_b, a.b, ES, fallback, Cfg<KIND>::K_ELEMS, BM_CTA))
    return cudaErrorInvalidValue;
  GroupedParams p = {};
  p.ends = a.ends;
  p.out = a.out;
  p.ldo = a.ldo;
  p.stride_o = a.stride_o;
  p.lane_scale = KIND == kTcec ? a.unscale : a.lane_scale;
  p.col_scale = a.col_scale;
  p.bias = a.bias;
  p.parts = a.parts;
  p.counters = a.counters;
  p.status = a.dev_status;
  p.rows = a.rows;
  p.groups = a.groups;
  p.lane_dim = a.lane_dim;
  p.col_dim = WGRAD ? a.col_dim : (a.k + Cfg<KIND>::K_ELEMS - 1) / Cfg<KIND>::K_ELEMS;
  // formats: F32 sums of F16 (0) or BF16 (1), or S32 sums of S8 (1); bits 15 and 16: A, B with their
  // lanes, columns contiguous
  const uint32_t sum_format = KIND == kI8 ? 2u : 1u, format = KIND == kI8 ? 1u : (a.bf16 ? 1u : 0u);
  p.idesc = (sum_format << 4) | (format << 7) | (format << 10) | (A_LANES ? 1u << 15 : 0u) |
            (WGRAD ? 1u << 16 : 0u) | ((LANES >> 4) << 24);
  p.alpha = a.alpha;
  p.beta = a.beta;
  p.out_type = static_cast<uint16_t>(a.out_type);
  p.vector_out = a.out_type != GroupedOut::f32 && a.beta == 0.f &&
                 (reinterpret_cast<uintptr_t>(a.out) & 15u) == 0 && a.ldo % 8 == 0 &&
                 (!a.wgrad || a.groups == 1 || a.stride_o % 8 == 0);
  return launch_chained(grouped_gemm_kernel<KIND, A_LANES, WGRAD>, static_cast<unsigned>(2 * clusters),
                        NUM_THREADS, Cfg<KIND>::SMEM, stream, map_a, map_b, map_b_few, p);
}

} // namespace

std::size_t grouped_parts_bytes(const GroupedArgs &a, unsigned num_sms) {
  const uint64_t pairs = num_sms / 2, lane_tiles = (a.lane_dim + LANES - 1) / LANES;
  // tiles there are at least: the groups of a product may leave some unfilled
  const uint64_t least = lane_tiles * (a.wgrad ? a.groups * static_cast<uint64_t>((a.col_dim + COLS - 1) / COLS)
                                               : (a.rows + COLS - 1) / COLS);
  return least <= pairs / 2 ? pairs * 2 * PART * sizeof(float) : 0;
}

cudaError_t launch_grouped_gemm(const GroupedArgs &a, cudaStream_t stream) {
  if (a.kind == GroupedKind::i8) {
    if (a.wgrad || a.a_lane_contig) return cudaErrorInvalidValue;
    return launch<kI8, false, false>(a, stream);
  }
  if (a.kind == GroupedKind::tcec)
    return a.wgrad            ? launch<kTcec, true, true>(a, stream)
           : a.a_lane_contig  ? launch<kTcec, true, false>(a, stream)
                              : launch<kTcec, false, false>(a, stream);
  return a.wgrad           ? launch<kF16, true, true>(a, stream)
         : a.a_lane_contig ? launch<kF16, true, false>(a, stream)
                           : launch<kF16, false, false>(a, stream);
}

} // namespace cumpsgemm_b200
