// Gradient of a pooled lookup (include/fwd_eb_train.h).
//
// grad_table[r] is the sum of the grad_out rows of all lookups of r: a reduction by key whose keys
// are the indices.  Adding with atomics would take them in any order, so the lookups are
// sorted by row first: a stable radix sort of (row, payload) pairs, digits of 8 bits, two kernels
// a digit (histogram of every tile, then scatter; up to 4096 lookups: one kernel in one CTA).  The
// sort is bound by latency and leaves the memory idle, so the same launches carry CTAs that fill
// the dense gradient with zeros.
//
// A warp then takes a run of 32 sorted lookups, keeps its columns' running sum in registers,
// and stores a row's sum where the row's lookups end.  The weights' gradient falls out of the same
// pass: the table row is read once for all its lookups.  A row whose lookups cross from one run into
// the next leaves partial sums, which a last kernel adds in run order; a popular row's thousands
// of runs are first added 32 at a time.  Every sum has one order, whatever the schedule.
#include <climits>

#include "eb_train.cuh"

namespace fwd_eb {
namespace {

constexpr int kSortThreads = 512;
constexpr int kSortWarps = kSortThreads / 32;
constexpr int kItems = 5;                          // pairs a thread ranks at a time
constexpr int kSubTile = kSortThreads * kItems;
constexpr int kSmallItems = 7;                     // ... in the kernel that sorts all of a small call
constexpr int kSmall = kSortThreads * kSmallItems;
constexpr int kDigits = 256;
constexpr int kStarts = 2048;                      // bag starts a tile keeps in shared memory
constexpr int kRun = 32;                           // sorted lookups of a run, runs of a block of runs
constexpr unsigned kNone = 0xffffffffu;

struct ZeroSpan {          // words of grad_table that a launch fills with zeros
  char* base;
  long long stride;        // bytes between rows
  long long per_row;       // words a row
  long long begin, end;
  int word;                // bytes: 16, 4 or 2
};

struct BackArgs {
  // the lookups
  const void* indices;
  const void* offsets;
  const float* psw;
  long long row_lo;
  long long padding_idx;
  unsigned num_rows;      // also the key of a lookup that contributes nothing
  int n;                  // lookups
  int num_bags;
  int fixed_len;          // 1 for GATHER: every lookup is a bag
  int idx64, include_last;
  int mean, mean_raw;
  // the gradients
  const char* grad_out;
  long long go_stride;    // bytes
  const char* table;
  long long table_stride;
  char* grad_table;
  long long gt_stride;
  const int2* winners;
  long long win_stride;   // pairs
  unsigned char* won;     // [num_bags][pstride]: the low byte of each winner's position
  float* grad_weights;
  int dim;
  int table_f16, gt_f16, square, accumulate;
  // scratch
  int* bag_of;            // [n]
  int* counted;           // [num_bags]: non-padding lookups (mean with a padding index)
  uint2* pairs[2];        // [n] {row, payload}
  int by_bag;             // the payload is the bag (-1 with a row of num_rows), else the lookup
  unsigned* hist;         // [tiles][kDigits]
  float* partial;         // [runs][2][pstride]: sums of a run's first row, when it began before the run,
                          // and of its last, when it began in the run and goes on
  float* super;           // [runs / 32][pstride]
  int pstride;
  int tiles, tile;        // sort tiles and lookups a tile
  int runs;
};

__device__ __forceinline__ long long index_at(const void* p, int idx64, long long i) {
  return idx64 ? __ldg(static_cast<const long long*>(p) + i) : (long long)__ldg(static_cast<const int*>(p) + i);
}

// Row of lookup j in the table window, or num_rows where it contributes nothing.
__device__ __forceinline__ unsigned row_of(const BackArgs& a, int j, int bag) {
  const long long idx = index_at(a.indices, a.idx64, j);
  const unsigned long long r = (unsigned long long)idx - (unsigned long long)a.row_lo;
  const bool ok = bag >= 0 && !(a.padding_idx >= 0 && idx == a.padding_idx) && r < a.num_rows;
  return ok ? (unsigned)r : a.num_rows;
}

// First lookup and length of a bag, as the forward kernels clamp them.
__device__ __forceinline__ void bag_range(const BackArgs& a, int bag, long long& start, long long& end) {
  if (a.fixed_len > 0) {
    start = (long long)bag * a.fixed_len;
    end = start + a.fixed_len;
  } else {
    start = index_at(a.offsets, a.idx64, bag);
    end = (a.include_last || bag + 1 < a.num_bags) ? index_at(a.offsets, a.idx64, bag + 1) : a.n;
  }
  if (start < 0) start = 0;
  if (end > a.n) end = a.n;
  if (end < start) end = start;
}

// The number of starts (ascending) in [lo, hi) that are <= j, plus lo.
template <typename Start>
__device__ __forceinline__ int upper_bound(Start start, long long j, int lo, int hi) {
  while (lo < hi) {
    const int mid = lo + (hi - lo) / 2;
    if (start(mid) <= j) lo = mid + 1; else hi = mid;
  }
  return lo;
}
// The same over all starts by a whole CTA: every thread tests one start a round.
template <int THREADS>
__device__ __forceinline__ int upper_bound_cta(const BackArgs& a, long long j, int n) {
  int lo = 0, len = n;
  while (len > 0) {
    const int step = (len + THREADS - 1) / THREADS;
    const long long at = lo + (long long)(threadIdx.x + 1) * step - 1;
    const int c = __syncthreads_count(at < lo + len && index_at(a.offsets, a.idx64, at) <= j);
    const int next = lo + c * step;
    len = min(step - 1, lo + len - next);
    lo = next;
  }
  return lo;
}

__device__ __forceinline__ void zero_span(const ZeroSpan& z, int part, int parts) {
  const long long total = z.end - z.begin;
  const bool dense = z.per_row * z.word == z.stride;
  for (long long k = (long long)part * blockDim.x + threadIdx.x; k < total; k += (long long)parts * blockDim.x) {
    const long long i = z.begin + k;
    char* q = dense ? z.base + i * z.word : z.base + (i / z.per_row) * z.stride + (i % z.per_row) * z.word;
    if (z.word == 16) *reinterpret_cast<uint4*>(q) = make_uint4(0, 0, 0, 0);
    else if (z.word == 4) *reinterpret_cast<unsigned*>(q) = 0;
    else *reinterpret_cast<unsigned short*>(q) = 0;
  }
}

__global__ void __launch_bounds__(kSortThreads) zero_kernel(const ZeroSpan z) {
  pdl_enter();
  zero_span(z, blockIdx.x, gridDim.x);
}

// counted[b] = length of bag b; the histogram kernel takes the padding off.
__global__ void __launch_bounds__(256) bag_length_kernel(const BackArgs a) {
  pdl_enter();
  const int b = blockIdx.x * 256 + threadIdx.x;
  if (b >= a.num_bags) return;
  long long s, e;
  bag_range(a, b, s, e);
  a.counted[b] = (int)(e - s);
}

// The bag starts that the lookups [begin, end) of a tile can lie behind.
struct TileStarts {
  int lo, hi;        // the number of starts <= a lookup lies in [lo, hi]
  bool in_shared;    // starts [lo, hi) are in shared memory
};
__device__ __forceinline__ TileStarts find_starts(const BackArgs& a, int begin, int end, long long* shared) {
  TileStarts t = {0, 0, false};
  if (a.fixed_len > 0 || begin >= end) return t;
  const int n = a.num_bags > 0 ? a.num_bags + (a.include_last ? 1 : 0) : 0;
  t.lo = upper_bound_cta<kSortThreads>(a, begin, n);
  t.hi = max(t.lo, upper_bound_cta<kSortThreads>(a, end - 1, n));
  t.in_shared = t.hi - t.lo <= kStarts;
  if (t.in_shared) {
    for (int i = t.lo + threadIdx.x; i < t.hi; i += kSortThreads) shared[i - t.lo] = index_at(a.offsets, a.idx64, i);
    __syncthreads();
  }
  return t;
}
// The bag that holds lookup j: the last one that starts at or before it; -1 where there is none.
__device__ __forceinline__ int bag_of(const BackArgs& a, int j, const TileStarts& t, const long long* shared) {
  if (a.fixed_len > 0) {
    const int bag = j / a.fixed_len;
    return bag < a.num_bags ? bag : -1;
  }
  const int bag = (t.in_shared ? upper_bound([&](int i) { return shared[i - t.lo]; }, j, t.lo, t.hi)
                               : upper_bound([&](int i) { return index_at(a.offsets, a.idx64, i); }, j, t.lo, t.hi)) - 1;
  return bag < a.num_bags ? bag : -1;     // behind the last offset of include_last_offset
}
// Padding is not counted for a mean: one subtraction a warp and bag.  All lanes of the warp call it.
__device__ __forceinline__ void uncount_padding(const BackArgs& a, int j, bool in, int bag) {
  const bool pad = in && bag >= 0 && index_at(a.indices, a.idx64, j) == a.padding_idx;
  const unsigned same = __match_any_sync(0xffffffffu, pad ? bag : -1);
  if (pad && (threadIdx.x & 31) == __ffs(same) - 1) atomicSub(a.counted + bag, __popc(same));
}

// hist[tile][d] = keys of the tile whose digit is d.  FIRST: the keys are made from the indices, and
// bag_of is written.  CTAs from `tiles` on fill their span with zeros.
template <bool FIRST>
__global__ void __launch_bounds__(kSortThreads) sort_histogram_kernel(const BackArgs a, const uint2* from, int shift,
                                                                      const ZeroSpan z) {
  pdl_enter();
  if ((int)blockIdx.x >= a.tiles) {
    zero_span(z, blockIdx.x - a.tiles, gridDim.x - a.tiles);
    return;
  }
  __shared__ unsigned count[kDigits];
  __shared__ long long starts[FIRST ? kStarts : 1];
  for (int d = threadIdx.x; d < kDigits; d += kSortThreads) count[d] = 0;
  const int begin = blockIdx.x * a.tile;
  const int end = min(a.n, begin + a.tile);
  TileStarts t = {};
  if (FIRST) t = find_starts(a, begin, end, starts);
  __syncthreads();
  for (int base = begin; base < end; base += kSubTile) {
    unsigned key[kItems];
#pragma unroll
    for (int i = 0; i < kItems; ++i) {
      const int j = base + i * kSortThreads + threadIdx.x;
      key[i] = 0;
      if (FIRST) {
        int bag = -1;
        if (j < end) {
          bag = bag_of(a, j, t, starts);
          a.bag_of[j] = bag;
          key[i] = row_of(a, j, bag);
        }
        if (a.counted) uncount_padding(a, j, j < end, bag);
      } else if (j < end) {
        key[i] = from[j].x;
      }
    }
#pragma unroll
    for (int i = 0; i < kItems; ++i) {
      if (base + i * kSortThreads + (int)threadIdx.x < end) atomicAdd(&count[(key[i] >> shift) & (kDigits - 1)], 1u);
    }
  }
  __syncthreads();
  for (int d = threadIdx.x; d < kDigits; d += kSortThreads) a.hist[blockIdx.x * kDigits + d] = count[d];
}

// Ranks of a CTA's items among those of the same digit, in the order of (warp, item, lane): in the warp here, and
// in_warp[w][d] becomes the number of warp w's items with digit d.  kNone is no digit.
template <int ITEMS>
__device__ __forceinline__ void rank_items(const unsigned (&digit)[ITEMS], unsigned (&rank)[ITEMS],
                                           unsigned (*in_warp)[kDigits]) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  for (int i = threadIdx.x; i < kSortWarps * kDigits; i += kSortThreads) (&in_warp[0][0])[i] = 0;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < ITEMS; ++i) {
    const unsigned same = __match_any_sync(0xffffffffu, digit[i]);
    const bool in = digit[i] != kNone;
    rank[i] = in ? in_warp[warp][digit[i]] + __popc(same & ((1u << lane) - 1u)) : 0;
    __syncwarp();
    if (in && lane == __ffs(same) - 1) in_warp[warp][digit[i]] += __popc(same);
    __syncwarp();
  }
  __syncthreads();
}
// in_warp[w][d] becomes the place of warp w's first item with digit d; place[d] moves behind all of them.
__device__ __forceinline__ void place_warps(unsigned (*in_warp)[kDigits], unsigned* place) {
  if (threadIdx.x < kDigits) {
    unsigned count[kSortWarps];
#pragma unroll
    for (int w = 0; w < kSortWarps; ++w) count[w] = in_warp[w][threadIdx.x];
    unsigned at = place[threadIdx.x];
#pragma unroll
    for (int w = 0; w < kSortWarps; ++w) {
      in_warp[w][threadIdx.x] = at;
      at += count[w];
    }
    place[threadIdx.x] = at;
  }
  __syncthreads();
}
// Exclusive sums over the digits of `mine` (threads below kDigits); `total` is scratch.  All threads call it.
__device__ __forceinline__ unsigned digits_below(unsigned mine, unsigned* total) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  unsigned sum = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const unsigned x = __shfl_up_sync(0xffffffffu, sum, o);
    if (lane >= o) sum += x;
  }
  if (lane == 31 && warp < kDigits / 32) total[warp] = sum;
  __syncthreads();
  for (int w = 0; w < warp && w < kDigits / 32; ++w) sum += total[w];
  __syncthreads();
  return sum - mine;
}

// Moves a tile's pairs to their place in the order of the digit, ties in the order they came.
template <bool FIRST>
__global__ void __launch_bounds__(kSortThreads) sort_scatter_kernel(const BackArgs a, const uint2* from, uint2* to,
                                                                    int shift, const ZeroSpan z) {
  pdl_enter();
  if ((int)blockIdx.x >= a.tiles) {
    zero_span(z, blockIdx.x - a.tiles, gridDim.x - a.tiles);
    return;
  }
  __shared__ unsigned place[kDigits];                    // next free place of a digit
  __shared__ unsigned in_warp[kSortWarps][kDigits];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int begin = blockIdx.x * a.tile;
  const int end = min(a.n, begin + a.tile);
  uint2 pair[kItems];
  auto fetch = [&](int base) {
#pragma unroll
    for (int i = 0; i < kItems; ++i) {
      const int j = base + (warp * kItems + i) * 32 + lane;
      pair[i] = make_uint2(0, 0);
      if (j >= end) continue;
      if (FIRST) {
        const int bag = a.bag_of[j];
        pair[i] = make_uint2(row_of(a, j, bag), a.by_bag ? (unsigned)bag : (unsigned)j);
      } else {
        pair[i] = from[j];
      }
    }
  };
  fetch(begin);
  // place[d] = keys with a lower digit + keys with digit d in earlier tiles: 4 digits a thread, every 8th tile
  {
    constexpr int kColumns = kDigits / 4, kGroups = kSortThreads / kColumns;
    const int column = threadIdx.x % kColumns, group = threadIdx.x / kColumns;
    uint4 all = make_uint4(0, 0, 0, 0), before = all;
#pragma unroll 8
    for (int t = group; t < a.tiles; t += kGroups) {
      const uint4 c = reinterpret_cast<const uint4*>(a.hist + t * kDigits)[column];
      const unsigned m = t < (int)blockIdx.x ? 0xffffffffu : 0u;
      all.x += c.x, all.y += c.y, all.z += c.z, all.w += c.w;
      before.x += c.x & m, before.y += c.y & m, before.z += c.z & m, before.w += c.w & m;
    }
    reinterpret_cast<uint4*>(in_warp[group])[column] = all;
    reinterpret_cast<uint4*>(in_warp[kGroups + group])[column] = before;
    static_assert(2 * kGroups <= kSortWarps, "both sums' groups fit in_warp");
    __syncthreads();
    unsigned sum = 0, earlier = 0;
    if (threadIdx.x < kDigits) {
#pragma unroll
      for (int g = 0; g < kGroups; ++g) {
        sum += in_warp[g][threadIdx.x];
        earlier += in_warp[kGroups + g][threadIdx.x];
      }
    }
    const unsigned lower = digits_below(sum, place);
    if (threadIdx.x < kDigits) place[threadIdx.x] = lower + earlier;
    __syncthreads();
  }
  for (int base = begin; base < end; base += kSubTile) {
    if (base != begin) {
      __syncthreads();
      fetch(base);
    }
    unsigned digit[kItems], rank[kItems];
#pragma unroll
    for (int i = 0; i < kItems; ++i) {
      const int j = base + (warp * kItems + i) * 32 + lane;
      digit[i] = j < end ? (pair[i].x >> shift) & (kDigits - 1) : kNone;
    }
    rank_items<kItems>(digit, rank, in_warp);
    place_warps(in_warp, place);
#pragma unroll
    for (int i = 0; i < kItems; ++i) {
      if (digit[i] != kNone) to[in_warp[warp][digit[i]] + rank[i]] = pair[i];
    }
  }
}

// Up to kSmall lookups: CTA 0 finds the bags and does all digits in shared memory, the others fill with zeros.
__global__ void __launch_bounds__(kSortThreads) sort_small_kernel(const BackArgs a, uint2* to, int passes, const ZeroSpan z) {
  pdl_enter();
  if (blockIdx.x > 0) {
    zero_span(z, blockIdx.x - 1, gridDim.x - 1);
    return;
  }
  __shared__ unsigned place[kDigits];
  __shared__ unsigned in_warp[kSortWarps][kDigits];
  __shared__ __align__(16) char buffer[kSmall * sizeof(uint2)];   // the starts, then the pairs between digits
  static_assert(kSmall >= kStarts, "the starts fit");
  long long* starts = reinterpret_cast<long long*>(buffer);
  uint2* pairs = reinterpret_cast<uint2*>(buffer);
  __shared__ unsigned total[kDigits / 32];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const TileStarts t = find_starts(a, 0, a.n, starts);
  uint2 pair[kSmallItems];
#pragma unroll
  for (int i = 0; i < kSmallItems; ++i) {
    const int j = (warp * kSmallItems + i) * 32 + lane;
    int bag = -1;
    pair[i] = make_uint2(0, 0);
    if (j < a.n) {
      bag = bag_of(a, j, t, starts);
      a.bag_of[j] = bag;
      pair[i] = make_uint2(row_of(a, j, bag), a.by_bag ? (unsigned)bag : (unsigned)j);
    }
    if (a.counted) uncount_padding(a, j, j < a.n, bag);
  }
  for (int pass = 0; pass < passes; ++pass) {
    unsigned digit[kSmallItems], rank[kSmallItems];
#pragma unroll
    for (int i = 0; i < kSmallItems; ++i) {
      const int j = (warp * kSmallItems + i) * 32 + lane;
      digit[i] = j < a.n ? (pair[i].x >> (8 * pass)) & (kDigits - 1) : kNone;
    }
    rank_items<kSmallItems>(digit, rank, in_warp);
    unsigned sum = 0;
    if (threadIdx.x < kDigits) {
#pragma unroll
      for (int w = 0; w < kSortWarps; ++w) sum += in_warp[w][threadIdx.x];
    }
    const unsigned lower = digits_below(sum, total);
    if (threadIdx.x < kDigits) place[threadIdx.x] = lower;
    __syncthreads();
    place_warps(in_warp, place);
    const bool last = pass + 1 == passes;
#pragma unroll
    for (int i = 0; i < kSmallItems; ++i) {
      if (digit[i] == kNone) continue;
      const unsigned at = in_warp[warp][digit[i]] + rank[i];
      if (last) to[at] = pair[i]; else pairs[at] = pair[i];
    }
    if (last) break;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kSmallItems; ++i) {
      const int j = (warp * kSmallItems + i) * 32 + lane;
      if (j < a.n) pair[i] = pairs[j];
    }
    __syncthreads();
  }
}

// won[b][c] = the low byte of the position that won column c of bag b: what the sum below compares in bags of
// fewer than 256 lookups, an eighth of the pairs' bytes.
__global__ void __launch_bounds__(256) winner_bytes_kernel(const BackArgs a) {
  pdl_enter();
  const long long total = (long long)a.num_bags * a.dim;
  for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < total; i += (long long)gridDim.x * 256) {
    const long long bag = i / a.dim;
    const int col = (int)(i - bag * a.dim);
    a.won[bag * a.pstride + col] = (unsigned char)__ldg(&a.winners[bag * a.win_stride + col].y);
  }
}

// Store the finished sum of a row.
template <int VE>
__device__ __forceinline__ void store_row(const BackArgs& a, unsigned row, int col, float (&acc)[VE]) {
  if (a.square) {
    float x[VE];
    const char* q = a.table + (long long)row * a.table_stride;
    if (a.table_f16) {
      Pack<__half, VE> r;
      r.load_ro(reinterpret_cast<const __half*>(q) + col);
      r.get(x);
    } else {
      Pack<float, VE> r;
      r.load_ro(reinterpret_cast<const float*>(q) + col);
      r.get(x);
    }
#pragma unroll
    for (int i = 0; i < VE; ++i) acc[i] *= 2.0f * x[i];
  }
  char* q = a.grad_table + (long long)row * a.gt_stride;
  if (a.gt_f16) {
    Pack<__half, VE> r;
    __half* to = reinterpret_cast<__half*>(q) + col;
    if (a.accumulate) {
      float old[VE];
      r.load(to);
      r.get(old);
#pragma unroll
      for (int i = 0; i < VE; ++i) acc[i] += old[i];
    }
    r.set(acc);
    r.store(to);
  } else {
    Pack<float, VE> r;
    float* to = reinterpret_cast<float*>(q) + col;
    if (a.accumulate) {
      float old[VE];
      r.load(to);
      r.get(old);
#pragma unroll
      for (int i = 0; i < VE; ++i) acc[i] += old[i];
    }
    r.set(acc);
    r.store(to);
  }
}

template <int VE>
__device__ __forceinline__ void load_table(const BackArgs& a, unsigned row, int col, float (&x)[VE]) {
  const char* q = a.table + (long long)row * a.table_stride;
  if (a.table_f16) {
    Pack<__half, VE> r;
    r.load_ro(reinterpret_cast<const __half*>(q) + col);
    r.get(x);
  } else {
    Pack<float, VE> r;
    r.load_ro(reinterpret_cast<const float*>(q) + col);
    r.get(x);
  }
}

// kPlain adds rows, kScaled takes a factor a lookup, kWeights does so and writes grad_weights, kMax masks columns.
enum Kind { kPlain = 0, kScaled = 1, kWeights = 2, kMax = 3 };

// A warp per run of 32 sorted lookups; blockIdx.y is a tile of 32 * VE columns.
template <typename TG, int VE, int KIND>
__global__ void __launch_bounds__(256) segment_sum_kernel(const BackArgs a, const uint2* pairs) {
  pdl_enter();
  constexpr int U = VE == 8 && KIND != kPlain && KIND != kScaled ? 4 : 8;   // lookups whose loads are issued together
  constexpr unsigned kAll = 0xffffffffu;
  const int lane = threadIdx.x & 31;
  const int run = blockIdx.x * 8 + (threadIdx.x >> 5);
  if (run >= a.runs) return;
  const int base = run * kRun;
  const int col = (blockIdx.y * 32 + lane) * VE;
  const bool col_ok = col < a.dim;
  uint2 pair = make_uint2(a.num_rows, 0);
  if (base + lane < a.n) pair = pairs[base + lane];
  const unsigned prev = base > 0 ? pairs[base - 1].x : kNone;
  const unsigned next = base + kRun < a.n ? pairs[base + kRun].x : kNone;
  const int valid = __popc(__ballot_sync(kAll, pair.x < a.num_rows));   // the rest sorts behind
  if (KIND == kWeights && lane >= valid && base + lane < a.n) a.grad_weights[pair.y] = 0.0f;
  if (valid == 0) return;
  int bag = 0, pos = 0;
  float coef = 1.0f;
  if (lane < valid) {
    bag = a.by_bag ? (int)pair.y : a.bag_of[pair.y];
    if (KIND == kScaled || KIND == kWeights) {
      if (a.psw) {
        coef = a.psw[pair.y];
      } else if (a.counted) {
        coef = 1.0f / (float)a.counted[bag];
      } else if (a.mean) {
        long long s, e;
        bag_range(a, bag, s, e);
        coef = 1.0f / (float)(e - s);
      }
    } else if (KIND == kMax) {
      long long s, e;
      bag_range(a, bag, s, e);
      pos = (int)pair.y - (int)s;
      if (e - s >= 256) pos |= INT_MIN;      // compare whole positions
    }
  }
  float acc[VE];
#pragma unroll
  for (int i = 0; i < VE; ++i) acc[i] = 0.0f;
  unsigned row = __shfl_sync(kAll, pair.x, 0);
  bool began_before = row == prev;

  auto put = [&](bool goes_on) {
    if (!col_ok) return;
    if (!began_before && !goes_on) {
      store_row<VE>(a, row, col, acc);
    } else {
      Pack<float, VE> r;
      r.set(acc);
      r.store(a.partial + ((long long)run * 2 + (began_before ? 0 : 1)) * a.pstride + col);
    }
  };
  float x[KIND == kWeights ? VE : 1];     // the table row of the running segment
  for (int e0 = 0; e0 < valid; e0 += U) {
    Pack<TG, VE> g[U];
    Pack<unsigned char, VE> won[KIND == kMax ? U : 1];
    float xs[KIND == kWeights ? U : 1][KIND == kWeights ? VE : 1];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int b = __shfl_sync(kAll, bag, e0 + u);
      const unsigned r = __shfl_sync(kAll, pair.x, e0 + u);
      const unsigned before = __shfl_sync(kAll, pair.x, (e0 + u - 1) & 31);
      g[u].zero();
      if (e0 + u < valid && col_ok) {
        g[u].load_ro(reinterpret_cast<const TG*>(a.grad_out + (long long)b * a.go_stride) + col);
        if constexpr (KIND == kMax) won[u].load_ro(a.won + (long long)b * a.pstride + col);
        if constexpr (KIND == kWeights) {   // a segment's first lookup in the run brings the row
          if (e0 + u == 0 || r != before) load_table<VE>(a, r, col, xs[u]);
        }
      }
    }
    float dot[KIND == kWeights ? U : 1];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const unsigned r = __shfl_sync(kAll, pair.x, e0 + u);
      const float c = __shfl_sync(kAll, coef, e0 + u);
      const int at = __shfl_sync(kAll, pos, e0 + u);
      if constexpr (KIND == kWeights) dot[u] = 0.0f;
      if (e0 + u >= valid) continue;
      const bool starts = e0 + u == 0 || r != row;
      if (r != row) {
        put(false);
        row = r;
        began_before = false;
#pragma unroll
        for (int i = 0; i < VE; ++i) acc[i] = 0.0f;
      }
      float f[VE];
      g[u].get(f);
      if constexpr (KIND == kWeights) {
        if (starts) {
#pragma unroll
          for (int i = 0; i < VE; ++i) x[i] = xs[u][i];
        }
        if (col_ok) {
#pragma unroll
          for (int i = 0; i < VE; ++i) dot[u] = fmaf(f[i], x[i], dot[u]);
        }
      }
      if constexpr (KIND == kMax) {
        unsigned char w[VE];
        memcpy(w, won[u].w, sizeof(w));
        const int b = __shfl_sync(kAll, bag, e0 + u);
#pragma unroll
        for (int i = 0; i < VE; ++i) {
          bool mine = w[i] == (unsigned char)at;
          if (at < 0 && mine && col_ok)
            mine = __ldg(&a.winners[(long long)b * a.win_stride + col + i].y) == (at & 0x7fffffff);
          acc[i] += mine ? f[i] : 0.0f;
        }
      } else {
#pragma unroll
        for (int i = 0; i < VE; ++i) acc[i] = KIND == kPlain ? acc[i] + f[i] : fmaf(c, f[i], acc[i]);
      }
    }
    if constexpr (KIND == kWeights) {
      // sums over the lanes of U values at once: a step halves the values a lane carries or the lanes of one
      int n = U;
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) {
        const bool upper = (lane & o) != 0;
        if (n > 1) {
          n /= 2;
#pragma unroll
          for (int k = 0; k < U / 2; ++k) {
            if (k >= n) break;
            const float give = upper ? dot[k] : dot[k + n];
            const float keep = upper ? dot[k + n] : dot[k];
            dot[k] = keep + __shfl_xor_sync(kAll, give, o);
          }
        } else {
          dot[0] += __shfl_xor_sync(kAll, dot[0], o);
        }
      }
      constexpr int kShift = U == 8 ? 2 : 3;      // lanes that share a value: 2^kShift
      const int u = lane >> kShift;
      const unsigned j = __shfl_sync(kAll, pair.y, e0 + u);
      if ((lane & ((1 << kShift) - 1)) == 0 && e0 + u < valid) a.grad_weights[j] = dot[0];
    }
  }
  put(row == next);
}

__device__ __forceinline__ unsigned first_row(const uint2* pairs, int run) { return pairs[run * kRun].x; }

// super[s] = sum of the 32 runs of block s, where one row's lookups fill all the block's run starts.
template <int VE>
__global__ void __launch_bounds__(256) segment_block_kernel(const BackArgs a, const uint2* pairs) {
  pdl_enter();
  const int block = blockIdx.x * 8 + (threadIdx.x >> 5);
  const int col = (blockIdx.y * 32 + (threadIdx.x & 31)) * VE;
  const int run0 = block * kRun;
  if (run0 + kRun > a.runs || block == 0 || col >= a.dim) return;
  const unsigned row = first_row(pairs, run0);
  if (row >= a.num_rows || pairs[run0 * kRun - 1].x != row || first_row(pairs, run0 + kRun - 1) != row) return;
  float acc[4][VE];
#pragma unroll
  for (int k = 0; k < 4; ++k) {
#pragma unroll
    for (int i = 0; i < VE; ++i) acc[k][i] = 0.0f;
  }
#pragma unroll
  for (int r = 0; r < kRun; r += 8) {
    Pack<float, VE> p[8];
#pragma unroll
    for (int u = 0; u < 8; ++u) p[u].load(a.partial + (long long)(run0 + r + u) * 2 * a.pstride + col);
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      float f[VE];
      p[u].get(f);
#pragma unroll
      for (int i = 0; i < VE; ++i) acc[u & 3][i] += f[i];
    }
  }
#pragma unroll
  for (int i = 0; i < VE; ++i) acc[0][i] = (acc[0][i] + acc[1][i]) + (acc[2][i] + acc[3][i]);
  Pack<float, VE> r;
  r.set(acc[0]);
  r.store(a.super + (long long)block * a.pstride + col);
}

// Rows that cross runs.  A warp looks at one run: where a row starts in it and goes on, the warp adds the row's
// pieces itself if they are few, else the CTA's 8 warps share them.
constexpr int kFewPieces = 24;
template <int VE>
__global__ void __launch_bounds__(256) segment_join_kernel(const BackArgs a, const uint2* pairs) {
  pdl_enter();
  __shared__ int last_run[8];
  __shared__ float part[8][32 * VE];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int col = (blockIdx.y * 32 + lane) * VE;
  const bool col_ok = col < a.dim;
  const int run = blockIdx.x * 8 + warp;
  int last = -1;          // the row's last run, -1: nothing to join here
  if (run + 1 < a.runs) {
    const unsigned row = pairs[run * kRun + kRun - 1].x;
    const unsigned before = run > 0 ? pairs[run * kRun - 1].x : kNone;
    // the next 32 runs at once; rows of more are searched for
    const unsigned ahead = run + 1 + lane < a.runs ? first_row(pairs, run + 1 + lane) : kNone;
    const unsigned same = __ballot_sync(0xffffffffu, ahead == row);
    if (row < a.num_rows && before != row && (same & 1u)) {
      if (same != 0xffffffffu) {
        last = run + __ffs(~same) - 1;
      } else {
        int lo = run + 32, hi = a.runs - 1;    // the last run that starts with the row
        while (lo < hi) {
          const int mid = hi - (hi - lo) / 2;
          if (first_row(pairs, mid) == row) lo = mid; else hi = mid - 1;
        }
        last = lo;
      }
    }
  }
  float acc[4][VE];
  // the row's pieces [begin, end) into acc[0]: its tail in `from`, single runs up to a block border, whole
  // blocks, single runs
  auto add_pieces = [&](int from, int to, int begin, int end) {
    const int first = from + 1;
    int b0 = (first + kRun - 1) / kRun, b1 = (to + 1) / kRun;     // whole blocks [b0, b1)
    if (!a.super || b1 < b0) b0 = b1 = 0;
    const int head = b1 > b0 ? b0 * kRun - first : to - first + 1;
    auto piece = [&](int i) -> const float* {
      if (i == 0) return a.partial + ((long long)from * 2 + 1) * a.pstride;
      i -= 1;
      if (i < head) return a.partial + (long long)(first + i) * 2 * a.pstride;
      i -= head;
      if (i < b1 - b0) return a.super + (long long)(b0 + i) * a.pstride;
      return a.partial + (long long)(b1 * kRun + (i - (b1 - b0))) * 2 * a.pstride;
    };
#pragma unroll
    for (int k = 0; k < 4; ++k) {
#pragma unroll
      for (int i = 0; i < VE; ++i) acc[k][i] = 0.0f;
    }
    if (!col_ok) return;
    for (int i0 = begin; i0 < end; i0 += 4) {
      Pack<float, VE> p[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        p[u].zero();
        if (i0 + u < end) p[u].load(piece(i0 + u) + col);
      }
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        float f[VE];
        p[u].get(f);
#pragma unroll
        for (int i = 0; i < VE; ++i) acc[u][i] += f[i];
      }
    }
#pragma unroll
    for (int i = 0; i < VE; ++i) acc[0][i] = (acc[0][i] + acc[1][i]) + (acc[2][i] + acc[3][i]);
  };
  auto count_pieces = [&](int from, int to) {
    const int first = from + 1;
    const int b0 = (first + kRun - 1) / kRun, b1 = (to + 1) / kRun;
    if (!a.super || b1 <= b0) return 1 + to - first + 1;
    return 1 + (b0 * kRun - first) + (b1 - b0) + (to + 1 - b1 * kRun);
  };
  if (last >= 0) {
    const int pieces = count_pieces(run, last);
    if (pieces <= kFewPieces) {
      add_pieces(run, last, 0, pieces);
      if (col_ok) store_row<VE>(a, pairs[run * kRun + kRun - 1].x, col, acc[0]);
      last = -1;
    }
  }
  if (lane == 0) last_run[warp] = last;
  if (__syncthreads_or(last >= 0) == 0) return;
  for (int w = 0; w < 8; ++w) {
    const int to = last_run[w];
    if (to < 0) continue;              // the same for the whole CTA
    const int from = blockIdx.x * 8 + w;
    const int pieces = count_pieces(from, to);
    const int share = (pieces + 7) / 8;
    add_pieces(from, to, min(pieces, warp * share), min(pieces, (warp + 1) * share));
#pragma unroll
    for (int i = 0; i < VE; ++i) part[warp][lane * VE + i] = acc[0][i];
    __syncthreads();
    if (warp == 0 && col_ok) {
      float sum[VE];
#pragma unroll
      for (int i = 0; i < VE; ++i) {
        sum[i] = 0.0f;
#pragma unroll
        for (int k = 0; k < 8; ++k) sum[i] += part[k][lane * VE + i];
      }
      store_row<VE>(a, pairs[from * kRun + kRun - 1].x, col, sum);
    }
    __syncthreads();
  }
}

// grad_weights[j] = <table[row j], grad_out[bag j]>, a warp per lookup.
template <typename TG, typename TT, int VE>
__global__ void __launch_bounds__(256) weight_gradient_kernel(const BackArgs a) {
  pdl_enter();
  const int lane = threadIdx.x & 31;
  const long long step = (long long)gridDim.x * 8;
  for (long long j = (long long)blockIdx.x * 8 + (threadIdx.x >> 5); j < a.n; j += step) {
    const int bag = a.bag_of[j];
    const unsigned row = row_of(a, (int)j, bag);
    float s = 0.0f;
    if (row < a.num_rows) {
      const TG* g = reinterpret_cast<const TG*>(a.grad_out + (long long)bag * a.go_stride);
      const TT* x = reinterpret_cast<const TT*>(a.table + (long long)row * a.table_stride);
      for (int col = lane * VE; col < a.dim; col += 32 * VE) {
        Pack<TG, VE> pg;
        Pack<TT, VE> px;
        float fg[VE], fx[VE];
        pg.load_ro(g + col);
        px.load_ro(x + col);
        pg.get(fg);
        px.get(fx);
#pragma unroll
        for (int i = 0; i < VE; ++i) s = fmaf(fg[i], fx[i], s);
      }
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    if (lane == 0) a.grad_weights[j] = s;
  }
}

// ---- host -----------------------------------------------------------------------------

struct BackPlan {
  BackArgs a;
  int passes;                // of the sort, a digit each
  int ve;                    // columns a lane
  bool want_table;
  bool fused_weights;        // grad_weights comes out of the segment sum
  size_t bytes;              // workspace
};

int64_t stride_or(int64_t s, int64_t dim) { return s ? s : dim; }

int make_back_plan(const fwd_eb_backward_params* p, BackPlan* pl) {
  if (!p) return fail(FWD_EB_EINVAL, "params is null");
  const fwd_eb_params& f = p->fwd;
  int rc = check_lookup(&f);
  if (rc) return rc;
  if (f.flags & FWD_EB_FLAG_OFFSET_PAIRS)
    return fail(FWD_EB_EUNSUPPORTED, "the gradient of a call with offset pairs is not implemented");
  if (p->flags & ~(uint32_t)FWD_EB_BACKWARD_ACCUMULATE) return fail(FWD_EB_EINVAL, "unknown flags %u", p->flags);
  if (f.num_indices > INT_MAX - 65536 || f.num_bags > INT_MAX - 65536)
    return fail(FWD_EB_ETOOBIG, "the gradient takes fewer than 2^31 - 65536 indices and bags");
  const bool gather = f.mode == FWD_EB_MODE_GATHER;
  if (p->grad_out_dtype != FWD_EB_F32 && p->grad_out_dtype != FWD_EB_F16)
    return fail(FWD_EB_EINVAL, "unknown grad_out_dtype %d", p->grad_out_dtype);
  if (p->grad_table_dtype != FWD_EB_F32 && p->grad_table_dtype != FWD_EB_F16)
    return fail(FWD_EB_EINVAL, "unknown grad_table_dtype %d", p->grad_table_dtype);
  const int64_t bags = gather ? f.num_indices : f.num_bags;
  if (bags > 0 && !p->grad_out) return fail(FWD_EB_EINVAL, "grad_out is null");
  if (!p->grad_table && !p->grad_weights) return fail(FWD_EB_EINVAL, "neither grad_table nor grad_weights is wanted");
  if (p->grad_weights && f.mode != FWD_EB_MODE_SUM) return fail(FWD_EB_EINVAL, "grad_weights need mode SUM");
  if (p->grad_weights && f.num_rows > 0 && !f.table) return fail(FWD_EB_EINVAL, "grad_weights need the table");
  if (f.mode == FWD_EB_MODE_SQUARE_SUM && f.num_rows > 0 && !f.table)
    return fail(FWD_EB_EINVAL, "mode SQUARE_SUM needs the table");
  if (f.mode == FWD_EB_MODE_MAX && bags > 0 && p->grad_table && !p->winners)
    return fail(FWD_EB_EINVAL, "mode MAX needs the winners of the forward call (out_dtype FWD_EB_F32_POS)");
  if (p->grad_out_stride != 0 && p->grad_out_stride < f.dim) return fail(FWD_EB_EINVAL, "grad_out_stride smaller than dim");
  if (p->grad_table_stride != 0 && p->grad_table_stride < f.dim)
    return fail(FWD_EB_EINVAL, "grad_table_stride smaller than dim");
  if (p->winners_stride != 0 && p->winners_stride < f.dim) return fail(FWD_EB_EINVAL, "winners_stride smaller than dim");
  const size_t ge = dtype_size(p->grad_out_dtype), te = dtype_size(p->grad_table_dtype);
  const size_t fe = dtype_size(f.table_dtype), ie = f.index_dtype == FWD_EB_I64 ? 8 : 4;
  if (!aligned_to(p->grad_out, ge) || !aligned_to(p->grad_table, te) || !aligned_to(p->grad_weights, 4) ||
      (f.mode == FWD_EB_MODE_MAX && !aligned_to(p->winners, 8)) || !aligned_to(f.table, fe) || !aligned_to(f.indices, ie) ||
      !aligned_to(f.offsets, ie) || !aligned_to(f.per_sample_weights, 4))
    return fail(FWD_EB_EALIGN, "a pointer is not aligned to its type");

  *pl = BackPlan{};
  BackArgs& a = pl->a;
  a.indices = f.indices;
  a.offsets = f.offsets;
  a.psw = f.per_sample_weights;
  a.row_lo = f.row_lo;
  a.padding_idx = f.padding_idx;
  a.num_rows = (unsigned)f.num_rows;
  a.n = (int)f.num_indices;
  a.num_bags = (int)bags;
  a.fixed_len = gather ? 1 : f.fixed_len;
  a.idx64 = f.index_dtype == FWD_EB_I64;
  a.include_last = a.fixed_len == 0 && f.include_last_offset != 0;
  a.mean = f.mode == FWD_EB_MODE_MEAN;
  a.mean_raw = (f.flags & FWD_EB_FLAG_MEAN_RAW_LENGTH) != 0;
  a.grad_out = static_cast<const char*>(p->grad_out);
  a.go_stride = stride_or(p->grad_out_stride, f.dim) * (int64_t)ge;
  a.table = static_cast<const char*>(f.table);
  a.table_stride = stride_or(f.table_stride, f.dim) * (int64_t)fe;
  a.grad_table = static_cast<char*>(p->grad_table);
  a.gt_stride = stride_or(p->grad_table_stride, f.dim) * (int64_t)te;
  a.winners = f.mode == FWD_EB_MODE_MAX ? static_cast<const int2*>(p->winners) : nullptr;
  a.win_stride = stride_or(p->winners_stride, f.dim);
  a.grad_weights = p->grad_weights;
  a.dim = f.dim;
  a.table_f16 = f.table_dtype == FWD_EB_F16;
  a.gt_f16 = p->grad_table_dtype == FWD_EB_F16;
  a.square = f.mode == FWD_EB_MODE_SQUARE_SUM;
  a.accumulate = (p->flags & FWD_EB_BACKWARD_ACCUMULATE) != 0;
  pl->want_table = p->grad_table != nullptr && f.num_rows > 0;

  // columns a lane: the fewest that let a warp cover the row, as far as all addresses allow
  auto fits = [&](int ve) {
    auto ok = [&](const void* q, int64_t stride, size_t e) {
      const size_t bytes = ve * e < 16 ? ve * e : 16;
      return !q || (aligned_to(q, bytes) && stride % (int64_t)bytes == 0);
    };
    return f.dim % ve == 0 && ok(a.grad_out, a.go_stride, ge) && ok(a.grad_table, a.gt_stride, te) &&
           ((!a.square && !a.grad_weights) || ok(a.table, a.table_stride, fe));
  };
  pl->ve = 1;
  for (int ve = 2; ve <= (ge == 2 ? 8 : 4) && pl->ve * 32 < f.dim && fits(ve); ve *= 2) pl->ve = ve;

  pl->passes = 1;
  while (pl->passes < 4 && (a.num_rows >> (8 * pl->passes)) != 0) ++pl->passes;   // num_rows itself is a key
  const long long per = ((long long)a.n + sm_count() - 1) / sm_count();
  a.tile = (int)(per < 1024 ? 1024 : (per + 31) / 32 * 32);
  a.tiles = (int)(((long long)a.n + a.tile - 1) / a.tile);
  a.runs = (int)(((long long)a.n + kRun - 1) / kRun);
  a.pstride = (f.dim + 7) / 8 * 8;
  pl->fused_weights = pl->want_table && a.grad_weights && f.dim <= 32 * pl->ve;
  a.by_bag = !a.winners && !a.psw && !pl->fused_weights;

  // scratch, each part on a 256-byte border
  size_t at = 0;
  auto take = [&](size_t bytes) {
    const size_t here = at;
    at += (bytes + 255) & ~(size_t)255;
    return here;
  };
  char* ws = static_cast<char*>(p->workspace);
  const size_t n = (size_t)a.n;
  a.bag_of = reinterpret_cast<int*>(ws + take(n * 4));
  const bool count = a.mean && !a.mean_raw && a.padding_idx >= 0;
  const size_t counted = take(count ? (size_t)a.num_bags * 4 : 0);
  a.counted = count ? reinterpret_cast<int*>(ws + counted) : nullptr;
  if (pl->want_table) {
    a.pairs[0] = reinterpret_cast<uint2*>(ws + take(n * 8));
    a.pairs[1] = reinterpret_cast<uint2*>(ws + take(pl->passes > 1 ? n * 8 : 0));
    a.hist = reinterpret_cast<unsigned*>(ws + take((size_t)a.tiles * kDigits * 4));
    a.partial = reinterpret_cast<float*>(ws + take((size_t)a.runs * 2 * a.pstride * 4));
    const int blocks = a.runs / kRun;
    const size_t super = take((size_t)blocks * a.pstride * 4);
    a.super = blocks > 1 ? reinterpret_cast<float*>(ws + super) : nullptr;
    a.won = reinterpret_cast<unsigned char*>(ws + take(a.winners ? (size_t)a.num_bags * a.pstride : 0));
  } else {
    a.hist = reinterpret_cast<unsigned*>(ws + take((size_t)a.tiles * kDigits * 4));
  }
  pl->bytes = a.n > 0 ? at : 0;
  return 0;
}

#define FWD_EB_TRY(call)                 \
  do {                                   \
    cudaError_t e_ = (call);             \
    if (e_ != cudaSuccess) return e_;    \
  } while (0)

template <typename TG, int VE>
cudaError_t launch_segments(const BackPlan& pl, const uint2* sorted, cudaStream_t st) {
  const BackArgs& a = pl.a;
  const unsigned tiles = (unsigned)((a.dim + 32 * VE - 1) / (32 * VE));
  const dim3 grid((unsigned)((a.runs + 7) / 8), tiles);
  if (a.winners) FWD_EB_TRY(launch_pdl(segment_sum_kernel<TG, VE, kMax>, grid, 256, 0, st, a, sorted));
  else if (pl.fused_weights) FWD_EB_TRY(launch_pdl(segment_sum_kernel<TG, VE, kWeights>, grid, 256, 0, st, a, sorted));
  else if (a.psw || a.mean) FWD_EB_TRY(launch_pdl(segment_sum_kernel<TG, VE, kScaled>, grid, 256, 0, st, a, sorted));
  else FWD_EB_TRY(launch_pdl(segment_sum_kernel<TG, VE, kPlain>, grid, 256, 0, st, a, sorted));
  if (a.super) {
    const dim3 blocks((unsigned)((a.runs / kRun + 7) / 8), tiles);
    FWD_EB_TRY(launch_pdl(segment_block_kernel<VE>, blocks, 256, 0, st, a, sorted));
  }
  if (a.runs > 1) FWD_EB_TRY(launch_pdl(segment_join_kernel<VE>, grid, 256, 0, st, a, sorted));
  return cudaSuccess;
}

template <typename TG>
cudaError_t launch_segments_ve(const BackPlan& pl, const uint2* sorted, cudaStream_t st) {
  switch (pl.ve) {
    case 8:
      if constexpr (sizeof(TG) == 2) return launch_segments<TG, 8>(pl, sorted, st);
      return cudaErrorInvalidValue;
    case 4: return launch_segments<TG, 4>(pl, sorted, st);
    case 2: return launch_segments<TG, 2>(pl, sorted, st);
    default: return launch_segments<TG, 1>(pl, sorted, st);
  }
}

template <typename TG, typename TT>
cudaError_t launch_weights(const BackPlan& pl, cudaStream_t st) {
  const BackArgs& a = pl.a;
  const long long blocks = ((long long)a.n + 7) / 8, most = 32LL * sm_count();
  const dim3 grid((unsigned)(blocks < most ? blocks : most));
  switch (pl.ve) {
    case 8: return launch_pdl(weight_gradient_kernel<TG, TT, 8>, grid, 256, 0, st, a);
    case 4: return launch_pdl(weight_gradient_kernel<TG, TT, 4>, grid, 256, 0, st, a);
    case 2: return launch_pdl(weight_gradient_kernel<TG, TT, 2>, grid, 256, 0, st, a);
    default: return launch_pdl(weight_gradient_kernel<TG, TT, 1>, grid, 256, 0, st, a);
  }
}

// The zeros of a dense gradient, in as many equal spans as there are launches to carry them.
struct Zeros {
  ZeroSpan z;
  long long words;
  int spans, done;
  Zeros(const BackPlan& pl, int spans_) : z(), words(0), spans(spans_), done(0) {
    const BackArgs& a = pl.a;
    if (!pl.want_table || a.accumulate) return;
    const long long row_bytes = (long long)a.dim * (a.gt_f16 ? 2 : 4);
    const bool wide = aligned_to(a.grad_table, 16) && a.gt_stride % 16 == 0 && row_bytes % 16 == 0;
    z.word = wide ? 16 : (a.gt_f16 ? 2 : 4);
    z.base = a.grad_table;
    z.stride = a.gt_stride;
    z.per_row = row_bytes / z.word;
    words = z.per_row * a.num_rows;
  }
  ZeroSpan next() {
    z.begin = words * done / spans;
    ++done;
    z.end = words * done / spans;
    return z;
  }
  // CTAs that fill a span beside a sort's: two an SM, fewer for little
  unsigned ctas() const {
    const long long most = 2LL * sm_count(), want = (words / spans + 4 * kSortThreads) / (4 * kSortThreads);
    return words == 0 ? 0u : (unsigned)(want < most ? want : most);
  }
};

cudaError_t launch_backward(const BackPlan& pl, const fwd_eb_backward_params* p, cudaStream_t st) {
  const BackArgs& a = pl.a;
  const bool small = a.n <= kSmall;
  Zeros zeros(pl, a.n == 0 || small || !pl.want_table ? 1 : 2 * pl.passes);
  const unsigned zc = zeros.ctas();
  if (a.n == 0) return zc == 0 ? cudaSuccess : launch_pdl(zero_kernel, dim3(zc), kSortThreads, 0, st, zeros.next());
  if (a.counted && a.num_bags > 0)
    FWD_EB_TRY(launch_pdl(bag_length_kernel, dim3((unsigned)((a.num_bags + 255) / 256)), 256, 0, st, a));
  if (pl.want_table && a.winners) {
    const long long blocks = ((long long)a.num_bags * a.dim + 255) / 256, most = 16LL * sm_count();
    if (blocks > 0)
      FWD_EB_TRY(launch_pdl(winner_bytes_kernel, dim3((unsigned)(blocks < most ? blocks : most)), 256, 0, st, a));
  }
  const dim3 tiles((unsigned)a.tiles + zc);
  const uint2* none = nullptr;
  int now = 0;
  if (small && pl.want_table) {
    FWD_EB_TRY(launch_pdl(sort_small_kernel, dim3(1 + zc), kSortThreads, 0, st, a, a.pairs[0], pl.passes, zeros.next()));
  } else {
    FWD_EB_TRY(launch_pdl(sort_histogram_kernel<true>, tiles, kSortThreads, 0, st, a, none, 0, zeros.next()));
    if (pl.want_table)
      FWD_EB_TRY(launch_pdl(sort_scatter_kernel<true>, tiles, kSortThreads, 0, st, a, none, a.pairs[0], 0, zeros.next()));
    for (int pass = 1; pass < pl.passes && pl.want_table; ++pass, now ^= 1) {
      const uint2* from = a.pairs[now];
      FWD_EB_TRY(launch_pdl(sort_histogram_kernel<false>, tiles, kSortThreads, 0, st, a, from, pass * 8, zeros.next()));
      FWD_EB_TRY(launch_pdl(sort_scatter_kernel<false>, tiles, kSortThreads, 0, st, a, from, a.pairs[now ^ 1], pass * 8,
                            zeros.next()));
    }
  }
  if (a.grad_weights && !pl.fused_weights) {
    const bool g16 = p->grad_out_dtype == FWD_EB_F16;
    FWD_EB_TRY(g16 ? (a.table_f16 ? launch_weights<__half, __half>(pl, st) : launch_weights<__half, float>(pl, st))
                   : (a.table_f16 ? launch_weights<float, __half>(pl, st) : launch_weights<float, float>(pl, st)));
  }
  if (!pl.want_table) return cudaSuccess;
  return p->grad_out_dtype == FWD_EB_F16 ? launch_segments_ve<__half>(pl, a.pairs[now], st)
                                         : launch_segments_ve<float>(pl, a.pairs[now], st);
}

}  // namespace
}  // namespace fwd_eb

using namespace fwd_eb;

extern "C" size_t fwd_eb_backward_params_size(void) { return sizeof(fwd_eb_backward_params); }

extern "C" size_t fwd_eb_backward_workspace_size(const fwd_eb_backward_params* p) {
  BackPlan pl;
  return make_back_plan(p, &pl) == 0 ? pl.bytes : 0;
}

extern "C" int fwd_eb_backward(const fwd_eb_backward_params* p, void* stream) {
  NvtxRange range("fwd_eb_backward");
  BackPlan pl;
  int rc = make_back_plan(p, &pl);
  if (rc) return rc;
  if (pl.bytes > 0 && (!p->workspace || p->workspace_bytes < pl.bytes))
    return fail(FWD_EB_EWORKSPACE, "the gradient needs %zu bytes of workspace, got %zu", pl.bytes,
                p->workspace ? p->workspace_bytes : (size_t)0);
  if (pl.bytes > 0 && !aligned_to(p->workspace, 256)) return fail(FWD_EB_EALIGN, "workspace must be 256-byte aligned");
  clear_error();
  cudaError_t e = launch_backward(pl, p, static_cast<cudaStream_t>(stream));
  return e == cudaSuccess ? 0 : cuda_fail(e, "kernel launch");
}
