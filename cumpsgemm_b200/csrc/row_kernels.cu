// Passes over rows in front of the grouped products (grouped_gemm.cu): operands brought into a form
// that TMA and the tensor core read, and rows quantised to 8 bits.  All of them move bytes and
// little else; a warp takes a row at a time, in 16-byte accesses where the row's address allows.
#include "grouped_totals.cuh"
#include "row_access.cuh"

namespace cumpsgemm_b200 {
namespace {

constexpr int kThreads = kTotalsThreads;
constexpr int kWarps = kThreads / 32;

// Which rows of an operand are of use: rows in front of the last group's end; weights of groups with
// rows.  By all threads of the block.
struct Used {
  uint32_t rows;
  const uint32_t *groups; // a bit for each, in shared memory
  __device__ __forceinline__ explicit Used(const StageArgs &a) {
    __shared__ uint32_t most, bits[kMaxGroups / 32];
    if (threadIdx.x < kMaxGroups / 32) bits[threadIdx.x] = 0;
    if (threadIdx.x == 0) most = 0;
    const GroupTotals t(a.ends, a.groups, a.rows); // (passes a barrier)
    uint32_t upto = 0;
    auto take = [&](uint32_t i) { // whether group i of the thread's is used
      const bool some = i < t.each && t.first + i < a.groups && t.end[i] > t.begin_of(i);
      if (some) upto = t.end[i];
      return some;
    };
    if (t.each == 1) { // a warp has 32 groups side by side
      const uint32_t word = __ballot_sync(0xffffffffu, take(0));
      if ((threadIdx.x & 31) == 0) bits[threadIdx.x >> 5] = word;
    } else {
#pragma unroll
      for (uint32_t i = 0; i < GroupTotals::MOST; ++i)
        if (take(i)) atomicOr(&bits[(t.first + i) / 32], 1u << ((t.first + i) % 32));
    }
    upto = __reduce_max_sync(0xffffffffu, upto);
    if ((threadIdx.x & 31) == 0 && upto != 0) atomicMax(&most, upto);
    __syncthreads();
    rows = most;
    groups = bits;
  }
  __device__ __forceinline__ bool has(uint32_t group) const { return (groups[group / 32] >> (group % 32)) & 1u; }
};

constexpr uint32_t kBatch = 4; // 16-byte loads that a lane has on its way at once

// The segments of all operands' rows, one after the other, dealt to the warps of the grid.  2^lanes_log2
// lanes take one, so a warp takes several short rows together; a row is one segment, unless there are
// too few of them to occupy all warps.  (With a row to a warp 110,000 rows of 183 bytes took 49 us, and
// take 14, and 480 of 29 KB took 17 and take 8.)
struct Segments {
  Used used;
  uint32_t units[2];  // segments of each operand
  uint64_t first[3];  // turns of a warp: first of each operand, and their end
  __device__ __forceinline__ explicit Segments(const StageArgs &a) : used(a) {
    first[0] = 0;
    for (int i = 0; i < 2; ++i) {
      const StageOperand &op = a.op[i];
      units[i] = i >= a.count ? 0u
                              : (op.rows_are_grouped ? used.rows : static_cast<uint32_t>(op.batch * op.outer)) *
                                    op.segments;
      first[i + 1] = first[i] + ((units[i] + (32u >> op.lanes_log2) - 1u) >> (5u - op.lanes_log2));
    }
  }
};
// One lane's part of a turn.
struct Segment {
  int o; // operand
  uint32_t row, lanes, lane, first, steps; // first: of its pieces of 16 bytes; the next are `lanes` further on
  bool ends;                               // the row's ends are this segment's too
  uint64_t src_at;                         // of the row's first element
  // false: there is none, or of weights that no row uses
  __device__ __forceinline__ bool get(const StageArgs &a, const Segments &s, uint64_t turn) {
    o = turn >= s.first[1];
    const StageOperand &op = o ? a.op[1] : a.op[0];
    const uint32_t all = threadIdx.x & 31u, log2 = op.lanes_log2, segments = op.segments;
    lanes = 1u << log2;
    lane = all & (lanes - 1u);
    const uint32_t unit = (static_cast<uint32_t>(turn - s.first[o]) << (5u - log2)) + (all >> log2);
    if (unit >= s.units[o]) return false;
    row = unit / segments;
    const uint32_t segment = unit - row * segments, outer = static_cast<uint32_t>(op.outer);
    const uint32_t b = row / outer;
    steps = op.steps;
    first = segment * steps * kBatch * lanes + lane;
    ends = segment == 0;
    src_at = b * op.stride + (row - b * outer) * op.ld;
    return op.rows_are_grouped || op.batch == 1 || s.used.has(b);
  }
};
// The pieces of a row that aligned accesses inside it give: [from, to) in units of 16 bytes (RowReader::inside).
struct Inside {
  const uint4 *aligned; // the row's first byte and what lies in front of it in its 16 bytes
  uint32_t shift, from, to;
  __device__ __forceinline__ explicit Inside(const RowReader &row)
      : aligned(reinterpret_cast<const uint4 *>(row.p - row.shift)), shift(row.shift), from(row.shift != 0) {
    const uint64_t need = shift == 0 ? 16 : 32;
    to = row.bytes + shift < need ? 0u : static_cast<uint32_t>((row.bytes + shift - need) / 16 + 1);
  }
  __device__ __forceinline__ bool has(uint32_t piece) const { return piece >= from && piece < to; }
  template <int ES> // pieces at, at + lanes, ...; all loads are on their way before the first is looked at
  __device__ __forceinline__ void load(uint32_t at, uint32_t lanes, uint4 (&x)[kBatch]) const {
    uint4 next[kBatch];
#pragma unroll
    for (uint32_t j = 0; j < kBatch; ++j) {
      const uint32_t piece = at + j * lanes;
      x[j] = next[j] = make_uint4(0, 0, 0, 0);
      if (has(piece)) {
        x[j] = __ldg(aligned + piece);
        if (shift != 0) next[j] = __ldg(aligned + piece + 1);
      }
    }
    if (shift == 0) return;
#pragma unroll
    for (uint32_t j = 0; j < kBatch; ++j) x[j] = shifted<ES>(x[j], next[j], shift);
  }
};

// ---------------------------------------------------------------- scales of FP32 operands
// records[op * kScaleRecords + block] = largest finite magnitude that block met.  Infinities and NaN
// say nothing of the range of the others, and rows of no group may hold anything.
// (Without the bound on blocks ptxas takes 32 registers and has a lane's loads wait for one another: 71 us
// for 55 million values instead of 45.)
__global__ void __launch_bounds__(kThreads, 4) largest_magnitude_kernel(const StageArgs a) {
  // (the pass behind comes when this one is through: see grouped_few_rows.cu)
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const Segments all(a);
  const uint32_t lane = threadIdx.x & 31u;
  const uint64_t step = static_cast<uint64_t>(gridDim.x) * kWarps;
  float most[2] = {0.f, 0.f};
  for (uint64_t turn = blockIdx.x * kWarps + (threadIdx.x >> 5); turn < all.first[2]; turn += step) {
    Segment seg;
    if (!seg.get(a, all, turn)) continue;
    const StageOperand &op = seg.o ? a.op[1] : a.op[0];
    const float *src = static_cast<const float *>(op.src) + seg.src_at;
    // in front of the first 16-byte boundary and behind the last one by one, 16 bytes at a time between
    const uint32_t inner = static_cast<uint32_t>(op.inner);
    const uint32_t head = min(inner, static_cast<uint32_t>(0u - (reinterpret_cast<uintptr_t>(src) >> 2)) & 3u);
    const uint32_t vectors = (inner - head) / 4, rest = head + 4 * vectors;
    const float4 *body = reinterpret_cast<const float4 *>(src + head);
    float4 ends = make_float4(0.f, 0.f, 0.f, 0.f);
    if (seg.ends) { // (at least four lanes, and at most three values at either end)
      if (seg.lane < head) ends.x = src[seg.lane];
      if (rest + seg.lane < inner) ends.y = src[rest + seg.lane];
    }
    float m = 0.f;
    auto take = [&](float v) { m = fmaxf(m, finite(v) ? fabsf(v) : 0.f); };
    uint32_t at = seg.first;
    for (uint32_t t = 0; t < seg.steps; ++t, at += kBatch * seg.lanes) {
      float4 x[kBatch];
#pragma unroll
      for (uint32_t j = 0; j < kBatch; ++j) {
        const uint32_t i = at + j * seg.lanes;
        x[j] = i < vectors ? __ldg(body + i) : make_float4(0.f, 0.f, 0.f, 0.f);
      }
#pragma unroll
      for (uint32_t j = 0; j < kBatch; ++j) take(x[j].x), take(x[j].y), take(x[j].z), take(x[j].w);
    }
    take(ends.x), take(ends.y);
    most[seg.o] = fmaxf(most[seg.o], m);
  }
  __shared__ uint32_t found[2];
  if (threadIdx.x < 2) found[threadIdx.x] = 0;
  __syncthreads();
  for (int o = 0; o < 2; ++o) {
    const uint32_t m = __reduce_max_sync(0xffffffffu, __float_as_uint(most[o])); // ordered as the values
    if (lane == 0) atomicMax(&found[o], m);
  }
  __syncthreads();
  if (threadIdx.x < 2)
    a.records[threadIdx.x * kScaleRecords + blockIdx.x] = __uint_as_float(found[threadIdx.x]);
}

// Exponent of the power of two that brings the largest magnitude to [2^14, 2^15), the scaling target
// of the other FP16TCEC_SCALING calls; at most 2^126, so operands below 2^-112 are brought up less.
__device__ __forceinline__ int scale_exponent(float largest) {
  if (largest == 0.f) return 0;
  int e;
  frexpf(largest, &e); // largest in [2^(e-1), 2^e)
  return min(15 - e, 126);
}
__device__ __forceinline__ float power_of_two(int e) { return ldexpf(1.f, e); }

// ---------------------------------------------------------------- operands into TMA's form
// BYTES 4: hi = RN_fp16(v), lo = RN_fp16((v - hi) * 2^11) for v = scale * x (split_math.cuh), in planes
// of outer * ld_dst elements for each matrix of the batch.  BYTES 1, 2: copied.
template <int BYTES>
__global__ void __launch_bounds__(kThreads) stage_kernel(const StageArgs a) {
  CUMPSGEMM_CHAINED_KERNEL_ENTRY();
  const Segments all(a);
  const uint32_t lane = threadIdx.x & 31u;
  float scale[2] = {1.f, 1.f};
  if (BYTES == 4 && a.scale) {
    __shared__ uint32_t found[2];
    if (threadIdx.x < 2) found[threadIdx.x] = 0;
    __syncthreads();
    for (int o = 0; o < 2; ++o) {
      float m = 0.f;
      for (uint32_t i = threadIdx.x; i < kScaleRecords; i += kThreads)
        m = fmaxf(m, a.records[o * kScaleRecords + i]);
      const uint32_t w = __reduce_max_sync(0xffffffffu, __float_as_uint(m));
      if (lane == 0) atomicMax(&found[o], w);
    }
    __syncthreads();
    const int e0 = scale_exponent(__uint_as_float(found[0])), e1 = scale_exponent(__uint_as_float(found[1]));
    scale[0] = power_of_two(e0);
    scale[1] = power_of_two(e1);
    if (blockIdx.x == 0 && threadIdx.x == 0) {
      // 2^-(e0 + e1) in two factors of about the same size, neither of which leaves the range
      const int e = -(e0 + e1), h = e / 2;
      a.unscale[0] = power_of_two(max(min(h, 126), -126));
      a.unscale[1] = power_of_two(max(min(e - h, 126), -126));
    }
  }
  const uint64_t step = static_cast<uint64_t>(gridDim.x) * kWarps;
  for (uint64_t turn = blockIdx.x * kWarps + (threadIdx.x >> 5); turn < all.first[2]; turn += step) {
    Segment seg;
    if (!seg.get(a, all, turn)) continue;
    const StageOperand &op = seg.o ? a.op[1] : a.op[0];
    const RowReader row(static_cast<const uint8_t *>(op.src) + seg.src_at * BYTES, op.inner * BYTES);
    const Inside in(row);
    const uint64_t dst_at = seg.row * op.ld_dst;
    // what is not inside, at most four pieces of a row, by the first lanes of its first segment
    const uint64_t end = seg.ends && seg.lane < 4 ? row.end_piece(seg.lane) : row.bytes;
    const bool has_end = end < row.bytes;
    uint4 end_x = make_uint4(0, 0, 0, 0);
    if (has_end) end_x = row.load_end<BYTES>(end);
    auto all_pieces = [&](auto &&put) {
      uint32_t at = seg.first;
      for (uint32_t t = 0; t < seg.steps; ++t, at += kBatch * seg.lanes) {
        uint4 x[kBatch];
        in.load<BYTES>(at, seg.lanes, x);
#pragma unroll
        for (uint32_t j = 0; j < kBatch; ++j)
          if (in.has(at + j * seg.lanes)) put(at + j * seg.lanes, x[j]);
      }
      if (has_end) put(static_cast<uint32_t>(end / 16), end_x);
    };
    if constexpr (BYTES == 4) {
      const float s = seg.o ? scale[1] : scale[0];
      uint2 *hi = reinterpret_cast<uint2 *>(static_cast<__half *>(op.dst) + dst_at);
      uint2 *lo = hi + static_cast<uint64_t>(op.batch) * op.outer * op.ld_dst / 4;
      all_pieces([&](uint32_t piece, const uint4 &v) { // of four values
        const uint32_t b[4] = {v.x, v.y, v.z, v.w};
        uint32_t h[2], l[2];
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          const float v0 = __uint_as_float(b[2 * t]) * s, v1 = __uint_as_float(b[2 * t + 1]) * s;
          const __half2 hh = __floats2half2_rn(v0, v1);
          const float2 hf = __half22float2(hh);
          const __half2 ll = __floats2half2_rn((v0 - hf.x) * 2048.f, (v1 - hf.y) * 2048.f);
          h[t] = *reinterpret_cast<const uint32_t *>(&hh);
          l[t] = *reinterpret_cast<const uint32_t *>(&ll);
        }
        hi[piece] = make_uint2(h[0], h[1]);
        lo[piece] = make_uint2(l[0], l[1]);
      });
    } else {
      uint4 *dst = reinterpret_cast<uint4 *>(static_cast<uint8_t *>(op.dst) + dst_at * BYTES);
      all_pieces([&](uint32_t piece, const uint4 &v) { dst[piece] = v; });
    }
  }
}

// ---------------------------------------------------------------- rows to 8 bits
// top = max_i |x_i|, scale = top / 127, q_i = rint(x_i * (127 / top)), where 127 / top and the product are
// rounded to FP32 first: |x_i| / top <= 1, so q_i stays within +-127, and an element is off by at most
// half a step of top / 127 (and 2^-16 of one, by those roundings).  The product is not fused with the
// addition that rounds it to an integer: halves are common (x_i = top / 2 in 16 bits), and unrounded such a
// product goes the way of the error of 127 / top instead of to the even neighbour.  A row of zeros has scale
// 0.  A row with an infinity or NaN has no scale: its scale is NaN, its q_i are 0, and so every product with
// it is NaN.  Rows too small for 127 / top (below 2^-100) are multiplied by 2^100 first.  Below 127 * 2^-126
// the scale is subnormal, a multiple of 2^-149, and an element is off by up to another 127 * 2^-150; a row
// whose scale comes to 0 so is one of zeros.  A row whose index lies outside x reads as zeros.
struct RowScale {
  float up, inverse, scale;
  bool none; // no scale
  __device__ __forceinline__ explicit RowScale(float top) {
    up = 1.f;
    inverse = 0.f;
    scale = 0.f;
    none = !finite(top);
    if (none) {
      scale = __uint_as_float(0x7fffffffu);
    } else if (top > 0.f) {
      scale = __fdiv_rn(top, 127.f);
      if (top < 0x1p-100f) up = 0x1p100f;
      if (scale > 0.f) inverse = __fdiv_rn(127.f, top * up);
    }
  }
  // Added to 1.5 * 2^23 the product is rounded to an integer, ties to even, whose low byte is the sum's.
  __device__ __forceinline__ uint32_t four(float x, float y, float z, float w) const {
    if (up != 1.f) x *= up, y *= up, z *= up, w *= up;
    const float m = 12582912.f;
    auto rounded = [&](float v) { return __float_as_uint(__fadd_rn(__fmul_rn(v, inverse), m)); };
    const uint32_t a = rounded(x), b = rounded(y), c = rounded(z), d = rounded(w);
    const uint32_t q = __byte_perm(__byte_perm(a, b, 0x0040), __byte_perm(c, d, 0x0040), 0x5410);
    return none ? 0u : q;
  }
  template <class Values> __device__ __forceinline__ uint2 eight(const Values &x) const {
    float v[8];
    x.values(v);
    return make_uint2(four(v[0], v[1], v[2], v[3]), four(v[4], v[5], v[6], v[7]));
  }
};

// row r of the result's source
template <class T> __device__ __forceinline__ RowReader source_row(const QuantizeArgs &a, uint64_t r) {
  const int64_t from = a.row_index != nullptr ? __ldg(a.row_index + r) : static_cast<int64_t>(r);
  const bool real = from >= 0 && from < static_cast<int64_t>(a.src_rows);
  return RowReader(static_cast<const T *>(a.x) + (real ? from : 0) * a.ldx,
                   real ? a.k * static_cast<uint64_t>(sizeof(T)) : 0);
}

// TPR threads to a row (a warp or the block), which they keep in registers: VEC groups of 8 values each.
// Bound by memory.  Where a block shares a row, the next one is on its way while this one's largest
// magnitude is found and its values leave: without, and with a conversion instruction for each value,
// 8192 rows of 8192 bfloat16 values took 92 us (2.2 TB/s) instead of 35.  Warps with rows of their own
// cover for one another.
template <class T, bool WHOLE, int TPR, int VEC>
__global__ void __launch_bounds__(kThreads) quantize_rows_kernel(const QuantizeArgs a) {
  CUMPSGEMM_CHAINED_KERNEL_ENTRY();
  constexpr int kRowsPerBlock = kThreads / TPR;
  const uint32_t t = threadIdx.x % TPR;
  __shared__ uint32_t tops[2][kWarps];
  uint32_t turn = 0;
  const uint64_t step = static_cast<uint64_t>(gridDim.x) * kRowsPerBlock;
  uint64_t r = static_cast<uint64_t>(blockIdx.x) * kRowsPerBlock + threadIdx.x / TPR;
  constexpr bool kAhead = TPR > 32;
  Eight<T, WHOLE> v[VEC];
  auto fetch = [&](uint64_t row) { Eight<T, WHOLE>::load(source_row<T>(a, row), t, TPR, v); };
  if (kAhead && r < a.rows) fetch(r);
  for (; r < a.rows; r += step, turn ^= 1u) {
    if (!kAhead) fetch(r);
    uint32_t top = 0;
#pragma unroll
    for (int j = 0; j < VEC; ++j) top = v[j].largest(top);
    Eight<T, WHOLE> mine[VEC];
#pragma unroll
    for (int j = 0; j < VEC; ++j) mine[j] = v[j];
    if (kAhead && r + step < a.rows) fetch(r + step);
    top = warp_largest<T>(top);
    if constexpr (TPR > 32) {
      if ((threadIdx.x & 31) == 0) tops[turn][threadIdx.x >> 5] = top;
      __syncthreads(); // (the other turn's slots are free: everybody has passed this barrier since)
#pragma unroll
      for (int w = 0; w < kWarps; ++w) top = max(top, tops[turn][w]);
    }
    const RowScale s(value_of<T>(top));
    int8_t *dst = a.q + r * a.ldq;
#pragma unroll
    for (int j = 0; j < VEC; ++j) {
      const uint64_t i = 8ull * (t + j * TPR);
      if (i < a.k) store_eight(dst, i, a.k, s.eight(mine[j]));
    }
    if (t == 0) a.scale[r] = s.scale;
  }
}

// Rows that no block can hold: read twice.
template <class T, bool WHOLE>
__global__ void __launch_bounds__(kThreads) quantize_long_rows_kernel(const QuantizeArgs a) {
  CUMPSGEMM_CHAINED_KERNEL_ENTRY();
  __shared__ uint32_t tops[2][kWarps];
  uint32_t turn = 0;
  const uint64_t chunks = (static_cast<uint64_t>(a.k) + 7) / 8;
  for (uint64_t r = blockIdx.x; r < a.rows; r += gridDim.x, turn ^= 1u) {
    const RowReader src = source_row<T>(a, r);
    uint32_t top = 0;
    for (uint64_t i = threadIdx.x; i < chunks; i += kThreads) {
      Eight<T, WHOLE> v[1];
      Eight<T, WHOLE>::load(src, i, 0, v);
      top = v[0].largest(top);
    }
    top = warp_largest<T>(top);
    if ((threadIdx.x & 31) == 0) tops[turn][threadIdx.x >> 5] = top;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kWarps; ++w) top = max(top, tops[turn][w]);
    const RowScale s(value_of<T>(top));
    for (uint64_t i = threadIdx.x; i < chunks; i += kThreads) {
      Eight<T, WHOLE> v[1];
      Eight<T, WHOLE>::load(src, i, 0, v);
      store_eight(a.q + r * a.ldq, 8 * i, a.k, s.eight(v[0]));
    }
    if (threadIdx.x == 0) a.scale[r] = s.scale;
  }
}

template <class T, bool WHOLE>
cudaError_t quantize(const QuantizeArgs &a, unsigned num_sms, cudaStream_t stream) {
  const uint64_t resident = static_cast<uint64_t>(num_sms) * 8;
  auto go = [&](auto kernel, uint32_t rows_per_block) {
    const uint64_t want = (static_cast<uint64_t>(a.rows) + rows_per_block - 1) / rows_per_block;
    return launch_chained(kernel, static_cast<unsigned>(want < resident ? want : resident), kThreads, 0,
                          stream, a);
  };
  // A warp holds a row of up to 1024 values, or 2048 of 16 bits, a block one of up to 8192.  (With few rows
  // a block each is faster: a warp alone takes longer over its row than 8.)
  const bool few = a.rows < num_sms * 4;
  if (!few && a.k <= 1024) return go(quantize_rows_kernel<T, WHOLE, 32, 4>, kWarps);
  if constexpr (sizeof(T) == 2)
    if (!few && a.k <= 2048) return go(quantize_rows_kernel<T, WHOLE, 32, 8>, kWarps);
  if (a.k <= 2048) return go(quantize_rows_kernel<T, WHOLE, kThreads, 1>, 1);
  if (a.k <= 4096) return go(quantize_rows_kernel<T, WHOLE, kThreads, 2>, 1);
  if (a.k <= 8192) return go(quantize_rows_kernel<T, WHOLE, kThreads, 4>, 1);
  return go(quantize_long_rows_kernel<T, WHOLE>, 1);
}
template <class T> cudaError_t quantize(const QuantizeArgs &a, unsigned num_sms, cudaStream_t stream) {
  // rows of whole aligned 16 bytes, the usual case: no code for ends
  const bool whole = (reinterpret_cast<uintptr_t>(a.x) & 15u) == 0 && a.ldx * sizeof(T) % 16 == 0 &&
                     a.k * sizeof(T) % 16 == 0;
  return whole ? quantize<T, true>(a, num_sms, stream) : quantize<T, false>(a, num_sms, stream);
}

} // namespace

cudaError_t launch_stage(const StageArgs &args, unsigned num_sms, cudaStream_t stream) {
  if (args.count == 0) return cudaSuccess;
  StageArgs a = args;
  uint64_t turns = 0;
  for (int i = 0; i < 2; ++i) {
    StageOperand &op = a.op[i];
    const uint64_t pieces = (op.inner * static_cast<uint64_t>(a.elem_bytes) + 15) / 16;
    op.lanes_log2 = 2;
    while (op.lanes_log2 < 5 && (static_cast<uint64_t>(kBatch) << op.lanes_log2) < pieces) ++op.lanes_log2;
    const uint64_t at_once = static_cast<uint64_t>(kBatch) << op.lanes_log2, steps = (pieces + at_once - 1) / at_once;
    // two turns for each of 32 warps an SM, if the rows go so far
    const uint64_t rows = op.outer * op.batch, wanted = (static_cast<uint64_t>(num_sms) * 64) << (5 - op.lanes_log2);
    uint64_t segments = rows >= wanted || rows == 0 ? 1 : (wanted + rows - 1) / rows;
    if (segments > steps) segments = steps;
    op.steps = static_cast<uint32_t>(segments > 0 ? (steps + segments - 1) / segments : 1);
    op.segments = static_cast<uint32_t>((steps + op.steps - 1) / op.steps);
    if (i >= a.count) continue;
    // (numbers of segments are 32-bit)
    if (op.segments * op.outer >= (1ull << 32) / op.batch) return cudaErrorInvalidValue;
    turns += ((op.segments * rows) >> (5 - op.lanes_log2)) + 1;
  }
  const uint64_t want = (turns + kWarps - 1) / kWarps, resident = static_cast<uint64_t>(num_sms) * 8;
  const unsigned grid = static_cast<unsigned>(want < resident ? want : resident);
  if (a.elem_bytes == 4 && a.scale) {
    const cudaError_t e = launch_chained(largest_magnitude_kernel, kScaleRecords, kThreads, 0, stream, a);
    if (e != cudaSuccess) return e;
  }
  switch (a.elem_bytes) {
  case 1:
    return launch_chained(stage_kernel<1>, grid, kThreads, 0, stream, a);
  case 2:
    return launch_chained(stage_kernel<2>, grid, kThreads, 0, stream, a);
  default:
    return launch_chained(stage_kernel<4>, grid, kThreads, 0, stream, a);
  }
}

cudaError_t launch_quantize_rows(const QuantizeArgs &a, unsigned num_sms, cudaStream_t stream) {
  switch (static_cast<GroupedOut>(a.type)) {
  case GroupedOut::f32:
    return quantize<float>(a, num_sms, stream);
  case GroupedOut::bf16:
    return quantize<__nv_bfloat16>(a, num_sms, stream);
  default:
    return quantize<__half>(a, num_sms, stream);
  }
}

} // namespace cumpsgemm_b200
