// The product of f8_gemm.cu for groups of few rows, on single CTAs (tcgen05 cta_group::1, kind::f8f6f4).
//
//   y[r, c] = sum over blocks b of 128 k's of  sx[r, b] sw_e[c / 128, b] sum_{k in b} xq[r, k] wq_e[c, k]  (+ bias[e, c])
//
// Bound by memory: the weights of each group with rows pass once.  Here features are the lanes of tensor memory, 128
// for a CTA, whose weights have one scale for each block of K, and up to 64 rows of a group its columns.  A block's
// products take 64 to 128 cycles instead of 512, eight accumulators of 64 columns are under way, and a CTA needs no
// word from another: f8_gemm.cu, where a stage of 256 features takes more than 800 cycles however few the rows
// are, read the weights of 32 experts of 4096 x 4096 for 8 rows each at 4.1 TB/s; this one takes 83 us, 6.5 TB/s, and
// 89 with 64 rows each.  One row of 4096 x 4096 takes 8.9 us, most of it in front of the first product and behind the last.
//
// Tiles are dealt to the CTAs in turn, the tiles of a group's rows with the same weights one behind the other.  A
// launch with few tiles cuts them into slices of K, whose sums are parked and added in order by the warp that is
// the last to come.
//
// Barriers, all of the CTA's own:
//   full[s], empty[s]         operands: bytes of the loads; commit
//   acc_full[a], acc_empty[a] accumulators: commit; one arrival from each epilogue warp
//   tile_full[i], tile_empty[i]  the warp that works out the tiles; one arrival from each role that took the tile
//   sc_full[b], sc_empty[b]   scales: the copies of each lane of a warp; one arrival from each epilogue warp
// Every wait is bounded.
#include "f8_common.cuh"
#include "gemm_common.cuh"
#include "grouped.hpp"

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <mutex>

namespace cumpsgemm_b200 {
namespace {

constexpr uint32_t LANES = 128;                 // features of a tile
constexpr uint32_t COLS = 64, BOX_ROWS = 32;    // most rows of a tile, and those of a load
constexpr uint32_t BLOCK = 128;                 // of K, in values and in bytes
constexpr uint32_t W_BYTES = LANES * BLOCK, STAGE_BYTES = W_BYTES + COLS * BLOCK, STAGES = 8;
constexpr uint32_t TMEM_COLS = 512, SLOTS = TMEM_COLS / COLS; // accumulators
constexpr uint32_t PARTS = 2, MOST = COLS / PARTS;            // epilogue warps of the same lanes, and columns of each
constexpr int EPI_WARPS = 4 * PARTS, THREADS = 128 + 32 * EPI_WARPS;
constexpr uint32_t AT_ONCE = 4;                // blocks of K whose scales are copied together, into two buffers in turn
constexpr uint32_t SCALE_WORDS = COLS + 4;     // of a block: the rows', then the weights'
constexpr uint32_t AHEAD = 3;                  // tiles that the roles may be apart
constexpr uint32_t MAX_SLICES = 16, MIN_SLICE = 2;
constexpr uint32_t PART = COLS * LANES;        // elements of a parked sum

constexpr uint32_t BARS = STAGES * STAGE_BYTES, FULL = BARS, EMPTY = FULL + 8 * STAGES, ACC_FULL = EMPTY + 8 * STAGES,
                   ACC_EMPTY = ACC_FULL + 8 * SLOTS, TILE_FULL = ACC_EMPTY + 8 * SLOTS, TILE_EMPTY = TILE_FULL + 8 * AHEAD,
                   SC_FULL = TILE_EMPTY + 8 * AHEAD, SC_EMPTY = SC_FULL + 16, TMEM_PTR = SC_EMPTY + 16, ABORT = TMEM_PTR + 4,
                   TILE = BARS + 384, START = TILE + AHEAD * 48, FIRST_TILE = START + 4 * (kMaxGroups + 2),
                   SCALE = (FIRST_TILE + 4 * (kMaxGroups + 2) + 127) / 128 * 128,
                   BYTES = SCALE + 2 * AT_ONCE * SCALE_WORDS * 4;
static_assert(ABORT + 4 <= TILE && TILE % 16 == 0, "barriers and flags");
constexpr uint32_t SMEM = BYTES + 1024; // and what the alignment of the stages takes
static_assert(SMEM <= 232448, "shared memory of a CTA");

struct FewParams {
  const int32_t *ends;
  void *out;
  uint64_t ldo;
  const float *x_scale;
  uint64_t x_scale_row, x_scale_block;
  const float *w_scale; // [groups][blocks of n][blocks of K]
  const float *bias;    // nullable
  float *parts;         // nullable: sums of slices, [slot][COLS][LANES]
  unsigned *counters;
  int *status;
  uint32_t rows, groups, n, blocks;
  uint32_t idesc;
  uint32_t out_type; // GroupedOut
};

// A tile, or a slice of one: `rows` rows from row0 on, features from col0 on, blocks [k0, k0 + blocks) of K.
struct alignas(16) Tile {
  uint32_t group, row0, rows, col0; // rows == 0: there are no more tiles
  uint32_t k0, blocks, slices, slice;
  uint32_t slot, number, pad0, pad1;
};
static_assert(sizeof(Tile) == 48, "three times 16 bytes");

// Slices of K that tiles are cut into, where there are at most half as many as CTAs.  A block takes some 700 cycles from
// memory, the join some 3000 and 700 for each slice: their sum is least with the square root of the blocks.
__device__ __forceinline__ uint32_t slices_of(const FewParams &p, uint32_t tiles) {
  if (p.parts == nullptr || tiles == 0 || tiles > gridDim.x / 2) return 1;
  const uint32_t most = min(min(gridDim.x / tiles, p.blocks / MIN_SLICE), MAX_SLICES);
  const uint32_t cut = max(1u, min(most, static_cast<uint32_t>(sqrtf(static_cast<float>(p.blocks)))));
  return (p.blocks - (p.blocks + cut - 1) / cut) * 700u > 3000u + 700u * cut ? cut : 1u;
}

// The items of a launch, which are tiles or slices of tiles, by their numbers.
struct Items {
  uint32_t sbase, group, total, slices;
  __device__ __forceinline__ Items(uint32_t sbase_, const FewParams &p) : sbase(sbase_), group(0) {
    const uint32_t tiles = first_tile(p.groups + 1);
    slices = slices_of(p, tiles);
    total = tiles * slices;
  }
  __device__ __forceinline__ uint32_t start(uint32_t g) const { return ld_shared_one<uint32_t>(sbase + START + 4 * g); }
  __device__ __forceinline__ uint32_t first_tile(uint32_t g) const { return ld_shared_one<uint32_t>(sbase + FIRST_TILE + 4 * g); }
  // item < total, and not below that of an earlier call; false: it is none (a tile of zeros has one slice)
  __device__ __forceinline__ bool get(const FewParams &p, uint32_t item, Tile &x) {
    x.number = item / slices;
    x.slice = item - x.number * slices;
    x.slot = item;
    while (x.number >= first_tile(group + 1)) ++group;
    const uint32_t r0 = start(group), r = start(group + 1) - r0, row_tiles = (r + COLS - 1) / COLS;
    const uint32_t local = x.number - first_tile(group), ct = local / row_tiles, rt = local - ct * row_tiles;
    x.group = group;
    x.row0 = r0 + rt * COLS;
    x.rows = min(COLS, r - rt * COLS);
    x.col0 = ct * LANES;
    x.slices = group < p.groups ? slices : 1u;
    if (x.slice >= x.slices) return false;
    const uint32_t all = group < p.groups ? p.blocks : 0u;
    x.k0 = all * x.slice / x.slices;
    x.blocks = all * (x.slice + 1) / x.slices - x.k0;
    return true;
  }
};

// The tiles a role takes, as a warp of the CTA works them out.
struct Tiles {
  uint32_t sbase, turn, phase;
  __device__ __forceinline__ explicit Tiles(uint32_t sbase_) : sbase(sbase_), turn(0), phase(0) {}
  __device__ __forceinline__ bool wait(int *status) const { // false: the wait gave up
    return ptx::mbar_wait_s(sbase + TILE_FULL + 8 * turn, phase, sbase + ABORT, status, ptx::kErrWaitTile);
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
  // one thread: the next tile; false at the end, or where the wait gave up
  __device__ __forceinline__ bool next(int *status, Tile &x) {
    if (!wait(status)) return false;
    const uint32_t at = advance();
    read(at, x);
    ptx::mbar_arrive(sbase + TILE_EMPTY + 8 * at); // (a release: the reads are in front of it)
    return x.rows != 0;
  }
};

// First row and first tile of each group, by one warp.  What `ends` holds is never trusted: a total that falls back
// or passes the number of rows is taken as the one in front of it, or as that number.  The rows behind the last
// group are a group of their own, whose tiles have no blocks.
__device__ __forceinline__ void find_groups(uint8_t *smem, const FewParams &p) {
  uint32_t *start = reinterpret_cast<uint32_t *>(smem + START);
  uint32_t *first_tile = reinterpret_cast<uint32_t *>(smem + FIRST_TILE);
  const uint32_t lane = threadIdx.x & 31u, col_tiles = (p.n + LANES - 1) / LANES;
  uint32_t end_before = 0, tiles = 0; // tiles in front
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
    const uint32_t mine = g <= p.groups ? (end - begin + COLS - 1) / COLS * col_tiles : 0u;
    uint32_t upto = mine;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const uint32_t o = __shfl_up_sync(0xffffffffu, upto, d);
      if (static_cast<int>(lane) >= d) upto += o;
    }
    if (g <= p.groups) {
      start[g] = begin;
      first_tile[g] = tiles + upto - mine;
    }
    if (g == p.groups) {
      start[g + 1] = end;
      first_tile[g + 1] = tiles + upto;
    }
    end_before = __shfl_sync(0xffffffffu, end, 31);
    tiles += __shfl_sync(0xffffffffu, upto, 31);
  }
}

template <class E> __device__ __forceinline__ E rounded(float v, bool bf16) {
  if constexpr (sizeof(E) == 4) return __float_as_uint(v);
  else return static_cast<E>(bf16 ? pack_bf16(v, 0.f) : pack_f16(v, 0.f));
}
// One feature of `rows` rows: a warp's lanes hold neighbours.  The one rounding.
template <class E>
__device__ __forceinline__ void store_sums(E *out, uint64_t ldo, const float (&sums)[MOST], uint32_t rows, float add, bool bf16) {
#pragma unroll
  for (uint32_t c = 0; c < MOST; ++c) {
    if (c >= rows) break;
    *out = rounded<E>(sums[c] + add, bf16);
    out += ldo;
  }
}

__global__ void __launch_bounds__(THREADS, 1)
    f8_few_rows_kernel(const __grid_constant__ CUtensorMap map_x, const __grid_constant__ CUtensorMap map_w,
                       const __grid_constant__ FewParams p) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t *const smem =
      reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  const uint32_t sbase = ptx::smem_u32(smem);
  volatile int *const abort_flag = reinterpret_cast<volatile int *>(smem + ABORT);
  const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31u;

  if (threadIdx.x == 0) {
    for (uint32_t s = 0; s < STAGES; ++s) {
      ptx::mbar_init(sbase + FULL + 8 * s, 1);
      ptx::mbar_init(sbase + EMPTY + 8 * s, 1);
    }
    for (uint32_t a = 0; a < SLOTS; ++a) {
      ptx::mbar_init(sbase + ACC_FULL + 8 * a, 1);
      ptx::mbar_init(sbase + ACC_EMPTY + 8 * a, EPI_WARPS);
    }
    for (uint32_t i = 0; i < AHEAD; ++i) {
      ptx::mbar_init(sbase + TILE_FULL + 8 * i, 1);
      ptx::mbar_init(sbase + TILE_EMPTY + 8 * i, EPI_WARPS + 3); // and who loads, copies, issues
    }
    for (uint32_t i = 0; i < 2; ++i) {
      ptx::mbar_init(sbase + SC_FULL + 8 * i, 32);
      ptx::mbar_init(sbase + SC_EMPTY + 8 * i, EPI_WARPS);
    }
    *abort_flag = 0;
    ptx::mbar_init_fence();
    ptx::prefetch_tensormap(&map_x);
    ptx::prefetch_tensormap(&map_w);
  }
  if (warp == 1) {
    ptx::tmem_alloc(sbase + TMEM_PTR, TMEM_COLS);
    ptx::tmem_relinquish();
  }
  // Everything above needs nothing of the kernel in front, everything below may.
  ptx::griddep_wait();
  if (warp == 2) find_groups(smem, p);
  ptx::tc_fence_before();
  __syncthreads();
  ptx::tc_fence_after();
  const uint32_t tmem_base = *reinterpret_cast<const uint32_t *>(smem + TMEM_PTR);
  Tile x;

  if (warp == 0) {
    // ================================================================ TMA producer
    if (ptx::elect_one()) {
      uint32_t s = 0, ph = 1;
      bool ok = true;
      Tiles tiles(sbase);
      while (ok && tiles.next(p.status, x)) {
        const uint32_t boxes = x.rows > BOX_ROWS ? 2u : 1u;
        for (uint32_t kb = 0; kb < x.blocks; ++kb) {
          ok = ptx::mbar_wait(sbase + EMPTY + 8 * s, ph, abort_flag, p.status, ptx::kErrWaitEmpty);
          if (!ok) break;
          const uint32_t dst = sbase + s * STAGE_BYTES, full = sbase + FULL + 8 * s;
          ptx::mbar_arrive_expect_tx(full, W_BYTES + boxes * BOX_ROWS * BLOCK);
          const int k = static_cast<int>((x.k0 + kb) * BLOCK);
          ptx::tma_load_3d(dst, &map_w, full, k, static_cast<int>(x.col0), static_cast<int>(x.group));
          for (uint32_t b = 0; b < boxes; ++b)
            ptx::tma_load_3d(dst + W_BYTES + b * BOX_ROWS * BLOCK, &map_x, full, k, static_cast<int>(x.row0 + b * BOX_ROWS), 0);
          if (++s == STAGES) {
            s = 0;
            ph ^= 1u;
          }
        }
      }
    }
  } else if (warp == 1) {
    // ================================================================ MMA issuer
    if (ptx::elect_one()) {
      constexpr uint64_t kStage = STAGE_BYTES >> 4;
      const uint64_t a0 = ptx::make_kmajor_desc<BLOCK>(sbase), b0 = ptx::make_kmajor_desc<BLOCK>(sbase + W_BYTES);
      uint32_t s = 0, ph = 0, slot = 0, e_ph = 1;
      bool ok = true;
      Tiles tiles(sbase);
      while (ok && tiles.next(p.status, x)) {
        const uint32_t idesc = p.idesc | ((x.rows > BOX_ROWS ? COLS : BOX_ROWS) >> 3 << 17);
        for (uint32_t kb = 0; kb < x.blocks; ++kb) {
          ok = ptx::mbar_wait(sbase + FULL + 8 * s, ph, abort_flag, p.status, ptx::kErrWaitFull) &&
               ptx::mbar_wait(sbase + ACC_EMPTY + 8 * slot, e_ph, abort_flag, p.status, ptx::kErrWaitD0Empty);
          if (!ok) break;
          ptx::tc_fence_after();
          const uint32_t d = tmem_base + slot * COLS;
#pragma unroll
          for (uint32_t ks = 0; ks < 4; ++ks)
            ptx::mma_f8_ss(d, a0 + s * kStage + 2 * ks, b0 + s * kStage + 2 * ks, idesc, ks != 0);
          ptx::tc_commit(sbase + ACC_FULL + 8 * slot);
          ptx::tc_commit(sbase + EMPTY + 8 * s);
          if (++slot == SLOTS) {
            slot = 0;
            e_ph ^= 1u;
          }
          if (++s == STAGES) {
            s = 0;
            ph ^= 1u;
          }
        }
      }
    }
  } else if (warp == 2) {
    // ================================================================ the next tiles
    if (ptx::elect_one()) {
      Items items(sbase, p);
      uint32_t turn = 0, ph = 1;
      for (uint32_t item = blockIdx.x;; item += gridDim.x) {
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
  } else if (warp == 3) {
    // ================================================================ scales: asynchronous copies that announce themselves
    const uint32_t w_blocks = (p.n + BLOCK - 1) / BLOCK;
    uint32_t b = 0, ph = 1;
    bool ok = true;
    Tiles tiles(sbase);
    while (ok) {
      ok = ptx::warp_agrees(tiles.wait(p.status));
      if (!ok) break;
      const uint32_t turn = tiles.advance();
      tiles.read(turn, x);
      __syncwarp();
      if (lane == 0) ptx::mbar_arrive(sbase + TILE_EMPTY + 8 * turn);
      if (x.rows == 0) break;
      const float *xs = p.x_scale + (static_cast<uint64_t>(x.row0) + lane) * p.x_scale_row + x.k0 * p.x_scale_block;
      const float *ws = p.w_scale + (static_cast<uint64_t>(x.group) * w_blocks + x.col0 / BLOCK) * p.blocks + x.k0;
      for (uint32_t kb = 0; kb < x.blocks; kb += AT_ONCE) {
        ok = ptx::warp_agrees(ptx::mbar_wait_backoff(sbase + SC_EMPTY + 8 * b, ph, abort_flag, p.status, ptx::kErrWaitTile, 64));
        if (!ok) break;
        for (uint32_t i = 0; i < AT_ONCE && kb + i < x.blocks; ++i) {
          const uint32_t to = sbase + SCALE + (b * AT_ONCE + i) * (SCALE_WORDS * 4) + lane * 4u;
#pragma unroll
          for (uint32_t j = 0; j < COLS / 32; ++j)
            if (lane + 32 * j < x.rows) copy_word(to + 128u * j, xs + 32 * j * p.x_scale_row);
          if (lane == 0) copy_word(to + COLS * 4, ws);
          xs += p.x_scale_block;
          ++ws;
        }
        copies_arrive(sbase + SC_FULL + 8 * b);
        b ^= 1u;
        if (b == 0) ph ^= 1u;
      }
    }
    wait_copies();
  } else {
    // ================================================================ epilogue
    const uint32_t epi = warp - 4, quarter = warp & 3u, part = epi >> 2;
    const uint32_t t_lanes = tmem_base + ((quarter * 32u) << 16) + part * MOST;
    uint32_t turn = 0, group = 0; // accumulators and groups of scales that are behind
    bool ok = true;
    Tiles tiles(sbase);
    while (true) {
      ok = ptx::warp_agrees(tiles.wait(p.status));
      if (!ok) break;
      const uint32_t at = tiles.advance();
      tiles.read(at, x);
      if (x.rows == 0) break;
      const uint32_t rows = x.rows > part * MOST ? min(x.rows - part * MOST, MOST) : 0u; // of the warp's columns
      float sums[MOST];
#pragma unroll
      for (uint32_t i = 0; i < MOST; ++i) sums[i] = 0.f;
#pragma unroll 1
      for (uint32_t kb = 0; kb < x.blocks; ++kb) {
        const uint32_t b = group & 1u, slot = turn % SLOTS, sc_full = sbase + SC_FULL + 8 * b, full = sbase + ACC_FULL + 8 * slot;
        const uint32_t sc_ph = (group >> 1) & 1u, ph = (turn / SLOTS) & 1u;
        if (!ptx::warp_agrees(both_over(sc_full, sc_ph, full, ph))) {
          ok = ptx::warp_agrees(ptx::mbar_wait_s(sc_full, sc_ph, sbase + ABORT, p.status, ptx::kErrWaitTile) &&
                                ptx::mbar_wait_s(full, ph, sbase + ABORT, p.status, ptx::kErrWaitD0Full));
          if (!ok) break;
        }
        ptx::tc_fence_after();
        if (rows > 0) {
          const uint32_t scales = sbase + SCALE + (b * AT_ONCE + kb % AT_ONCE) * (SCALE_WORDS * 4);
          uint32_t v[MOST];
          ptx::tmem_ld_32x32b_x32(t_lanes + slot * COLS, v);
          const float w = __uint_as_float(ld_shared_one<uint32_t>(scales + COLS * 4));
          uint4 s[MOST / 4]; // (columns without a row have any)
#pragma unroll
          for (uint32_t i = 0; i < MOST / 4; ++i) s[i] = ld_shared(scales + part * (MOST * 4) + 16 * i);
          ptx::tmem_ld_wait();
#pragma unroll
          for (uint32_t i = 0; i < MOST / 4; ++i) {
            sums[4 * i] = fmaf(__uint_as_float(v[4 * i]), __uint_as_float(s[i].x) * w, sums[4 * i]);
            sums[4 * i + 1] = fmaf(__uint_as_float(v[4 * i + 1]), __uint_as_float(s[i].y) * w, sums[4 * i + 1]);
            sums[4 * i + 2] = fmaf(__uint_as_float(v[4 * i + 2]), __uint_as_float(s[i].z) * w, sums[4 * i + 2]);
            sums[4 * i + 3] = fmaf(__uint_as_float(v[4 * i + 3]), __uint_as_float(s[i].w) * w, sums[4 * i + 3]);
          }
        }
        ptx::tc_fence_before();
        __syncwarp();
        arrive_if(lane == 0, sbase + ACC_EMPTY + 8 * slot);
        ++turn;
        const bool last = kb % AT_ONCE == AT_ONCE - 1 || kb + 1 == x.blocks; // of the scales that were copied together
        arrive_if(last && lane == 0, sbase + SC_EMPTY + 8 * b);
        group += last;
      }
      if (!ok) break;
      bool done = rows == 0;
      if (!done && x.slices > 1) { // the last of the tile's slices to park these lanes and columns adds them all, in order
        float *parts = p.parts + static_cast<uint64_t>(x.slot) * PART + part * MOST * LANES + quarter * 32u + lane;
#pragma unroll
        for (uint32_t c = 0; c < MOST; ++c)
          if (c < rows) __stcg(parts + c * LANES, sums[c]);
        __threadfence();
        __syncwarp();
        uint32_t before = 0;
        if (lane == 0) before = atomicInc(p.counters + 2 + x.number * EPI_WARPS + epi, x.slices - 1);
        done = __shfl_sync(0xffffffffu, before, 0) != x.slices - 1;
        if (!done) {
          __threadfence();
          const float *first = parts - static_cast<uint64_t>(x.slice) * PART;
#pragma unroll
          for (uint32_t c = 0; c < MOST; ++c) sums[c] = 0.f;
#pragma unroll 1
          for (uint32_t i = 0; i < x.slices; ++i, first += PART)
#pragma unroll
            for (uint32_t c = 0; c < MOST; ++c) sums[c] += c < rows ? __ldcg(first + c * LANES) : 0.f;
        }
      }
      const uint32_t feature = x.col0 + quarter * 32u + lane;
      if (!done && feature < p.n) {
        const float add = p.bias != nullptr && x.group < p.groups ? __ldg(p.bias + static_cast<uint64_t>(x.group) * p.n + feature) : 0.f;
        const uint64_t to = (static_cast<uint64_t>(x.row0) + part * MOST) * p.ldo + feature;
        const auto type = static_cast<GroupedOut>(p.out_type);
        if (type == GroupedOut::f32) store_sums(static_cast<uint32_t *>(p.out) + to, p.ldo, sums, rows, add, false);
        else store_sums(static_cast<uint16_t *>(p.out) + to, p.ldo, sums, rows, add, type == GroupedOut::bf16);
      }
      __syncwarp();
      if (lane == 0) ptx::mbar_arrive(sbase + TILE_EMPTY + 8 * at);
    }
  }

  // ---------------------------------------------------------------- teardown
  ptx::tc_fence_before();
  __syncthreads();
  if (*abort_flag) { // (loads and products may be under way)
    const uint64_t t0 = ptx::globaltimer_ns();
    while (ptx::globaltimer_ns() - t0 < 2000000ull) __nanosleep(1000);
    __syncthreads();
  }
  if (warp == 1) {
    ptx::tc_fence_after();
    ptx::tmem_dealloc(tmem_base, TMEM_COLS);
  }
}

// Per device, once (any thread): shared-memory attribute and the number of SMs, each of which has a CTA.
cudaError_t set_up(int *sms_out) {
  static std::once_flag once[64];
  static cudaError_t setup_error[64];
  static int sms[64];
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev < 0 || dev >= 64) return cudaErrorInvalidDevice;
  std::call_once(once[dev], [&]() {
    setup_error[dev] = cudaFuncSetAttribute(f8_few_rows_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM);
    sms[dev] = 1;
    cudaDeviceGetAttribute(&sms[dev], cudaDevAttrMultiProcessorCount, dev);
  });
  *sms_out = sms[dev];
  return setup_error[dev];
}

bool operand_map(CUtensorMap *map, const GroupedOperand &o, uint32_t box_rows) {
  return make_byte_map(map, 1, o.ptr, {o.inner, o.outer, o.batch}, {o.ld, o.batch > 1 ? o.stride : o.ld},
                       {BLOCK, box_rows, 1}, true);
}

} // namespace

std::size_t f8_few_rows_parts_bytes(const GroupedArgs &a, unsigned num_sms) {
  // tiles there are at least: groups may leave some unfilled
  const uint64_t least = ((a.rows + COLS - 1) / COLS) * static_cast<uint64_t>((a.lane_dim + LANES - 1) / LANES);
  return least <= num_sms / 2 ? static_cast<uint64_t>(num_sms) * PART * sizeof(float) : 0;
}

cudaError_t launch_f8_few_rows(const GroupedArgs &a, cudaStream_t stream) {
  int sms = 1;
  const cudaError_t se = set_up(&sms);
  if (se != cudaSuccess) return se;
  CUtensorMap map_x, map_w;
  if (!operand_map(&map_x, a.b, BOX_ROWS) || !operand_map(&map_w, a.a, LANES)) return cudaErrorInvalidValue;
  FewParams p = {};
  p.ends = a.ends;
  p.out = a.out;
  p.ldo = a.ldo;
  p.x_scale = a.col_scale;
  p.x_scale_row = a.f8->x_scale_row;
  p.x_scale_block = a.f8->x_scale_block;
  p.w_scale = a.lane_scale;
  p.bias = a.bias;
  p.parts = a.parts;
  p.counters = a.counters;
  p.status = a.dev_status;
  p.rows = a.rows;
  p.groups = a.groups;
  p.n = a.lane_dim;
  p.blocks = (a.k + BLOCK - 1) / BLOCK;
  // FP32 sums; the formats of A (w) and B (x), e4m3 (0) or e5m2 (1)
  p.idesc = (1u << 4) | (static_cast<uint32_t>(a.f8->w_type) << 7) | (static_cast<uint32_t>(a.f8->x_type) << 10) | ((LANES >> 4) << 24);
  p.out_type = static_cast<uint32_t>(a.out_type);
  return launch_chained(f8_few_rows_kernel, static_cast<unsigned>(sms), THREADS, SMEM, stream, map_x, map_w, p);
}

} // namespace cumpsgemm_b200
