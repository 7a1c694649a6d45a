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

} // namespace cumpsgemm_b200
