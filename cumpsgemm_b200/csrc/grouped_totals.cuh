// The running totals of rows after each group as a block of kTotalsThreads threads reads them.
#pragma once
#include "grouped.hpp"

namespace cumpsgemm_b200 {

constexpr uint32_t kTotalsThreads = 256;

// What `ends` holds is never trusted, as find_groups does it (grouped_gemm.cu): a total that falls back or
// passes the number of rows is taken as the one in front of it, or as that number.  A thread has `each`
// neighbouring groups from `first` on, of which i ends at end[i]; the first begins at `begin`.  Group number
// `groups` are the rows behind the last; groups behind it, and i >= each, are empty.
struct GroupTotals {
  static constexpr uint32_t MOST = (kMaxGroups + kTotalsThreads) / kTotalsThreads;
  uint32_t first, each, begin, end[MOST];

  // by all threads
  __device__ __forceinline__ GroupTotals(const int32_t *ends, uint32_t groups, uint32_t rows) {
    auto total = [&](uint32_t g) { // as it stands there
      return g >= groups || ends == nullptr
                 ? rows
                 : static_cast<uint32_t>(min(max(__ldg(ends + g), 0), static_cast<int32_t>(rows)));
    };
    each = groups / kTotalsThreads + 1;
    first = threadIdx.x * each;
    begin = first == 0 ? 0u : total(first - 1);
    uint32_t last = begin;
    bool falls = false;
#pragma unroll
    for (uint32_t i = 0; i < MOST; ++i) {
      end[i] = i < each ? total(first + i) : last;
      falls |= end[i] < last;
      last = end[i];
    }
    if (!__syncthreads_or(falls)) return;
    for (uint32_t g = 0; g < first && g < groups; ++g) begin = max(begin, total(g));
#pragma unroll
    for (uint32_t i = 0; i < MOST; ++i) end[i] = max(end[i], begin_of(i));
  }
  __device__ __forceinline__ uint32_t begin_of(uint32_t i) const { return i == 0 ? begin : end[i - 1]; }
};

// The rows of one group, at most MOST_ROWS of them, that a block multiplies.
struct Chunk {
  uint32_t group, row0, rows; // rows == 0: there is none
};
// Chunk `number` (all threads give the same), and how many there are, by all threads.
template <uint32_t MOST_ROWS>
__device__ __forceinline__ Chunk find_chunk(const int32_t *ends, uint32_t groups, uint32_t rows, uint32_t number, uint32_t &all) {
  constexpr uint32_t WARPS = kTotalsThreads / 32;
  __shared__ uint32_t chunks[WARPS];
  __shared__ Chunk found;
  const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31u;
  const GroupTotals t(ends, groups, rows);
  auto chunks_of = [&](uint32_t i) { return (t.end[i] - t.begin_of(i) + MOST_ROWS - 1) / MOST_ROWS; };
  uint32_t mine = 0;
#pragma unroll
  for (uint32_t i = 0; i < GroupTotals::MOST; ++i) mine += chunks_of(i);
  uint32_t at = mine; // chunks in front of the thread's
#pragma unroll
  for (uint32_t d = 1; d < 32; d <<= 1) {
    const uint32_t o = __shfl_up_sync(0xffffffffu, at, d);
    if (lane >= d) at += o;
  }
  if (lane == 31) chunks[warp] = at;
  if (threadIdx.x == 0) found.rows = 0;
  at -= mine;
  __syncthreads();
  all = 0;
#pragma unroll
  for (uint32_t w = 0; w < WARPS; ++w) {
    if (w == warp) at += all;
    all += chunks[w];
  }
  if (number >= at && number < at + mine) {
#pragma unroll
    for (uint32_t i = 0; i < GroupTotals::MOST; ++i) {
      const uint32_t n = chunks_of(i);
      if (number >= at && number < at + n) {
        const uint32_t row0 = t.begin_of(i) + (number - at) * MOST_ROWS;
        found = {t.first + i, row0, min(t.end[i] - row0, MOST_ROWS)};
      }
      at += n;
    }
  }
  __syncthreads();
  return found;
}

} // namespace cumpsgemm_b200
