// Gradient of a pooled lookup (include/fwd_eb_train.h).
//
// grad_table[r] is the sum of the grad_out rows of all lookups of r: a reduction by key whose keys
// are the indices.  Adding with atomics would take them in any order, so the lookups are
// sorted by row first: a stable radix sort of (row, payload) pairs by digits of up to 8 bits.  Two kernels
// a digit: one counts it in every tile (the first also makes the pairs), one moves the pairs, brought
// into the digit's order in shared memory first so that neighbours are stored together.  Up to kSmall
// lookups are sorted in one CTA.
//
// A warp then takes a run of 32 sorted lookups, keeps its columns' running sum in registers,
// and stores a row's sum where the row's lookups end.  The weights' gradient falls out of the same
// pass: the table row is read once for all its lookups.  A row whose lookups cross from one run into
// the next leaves partial sums, which a last kernel adds in a fixed order; a popular row's thousands
// of runs are first added 32 at a time.  Every sum has one order, whatever the schedule.
//
// Measured on B200 (a call, of the copy rate measured there): 655 k Zipf lookups of a 1 M x 128 fp16 table, mean, dense gradient
// 113 us, 0.36: sort 38, sums beside zeros 66, joins 14; 262 k of a 1 M x 256 fp16 table, max 144 us, 0.57; 1.3 M weighted
// lookups of a 4 M x 128 fp32 table, both gradients, accumulated 203 us, 0.37: sort 48, sums 136, bound by the latency of rows
// from DRAM and by issue slots in like parts; 655 k uniform lookups of a 1 M x 128 fp16 table, square sum 144 us, 0.46 (65 % of
// the issue slots in the sums), gather 115.
//
// The rows of a dense gradient that no lookup names are filled with zeros by other CTAs of the same launch, which
// find the named ones in the sorted pairs: every row is written once, and the sums, bound by
// instructions and the L2, run beside the zeros, bound by DRAM.
#include <climits>

#include "eb_train.cuh"

namespace fwd_eb {
namespace {

constexpr int kSortThreads = 512;
constexpr int kSortWarps = kSortThreads / 32;
// Pairs a thread of the sort ranks at a time: 5 where they cover a tile (2560 pairs), else 9.
constexpr int kItemsFew = 5, kItemsMany = 9;
constexpr int kSmallItems = 7;                     // ... in the kernel that sorts all of a small call
constexpr int kSmall = kSortThreads * kSmallItems;
constexpr int kTiny = 2 * kSortThreads;            // lookups of a call that one launch does
constexpr int kDigits = 256;                       // at most
constexpr int kStarts = 2048;                      // bag starts a tile keeps in shared memory
constexpr int kRun = 32;                           // sorted lookups of a run, runs of a block of runs
constexpr unsigned kNone = 0xffffffffu;
constexpr int kMostColumns = 1 << 20;

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
  unsigned fixed_magic;   // j / fixed_len = j * fixed_magic >> 31 + fixed_shift for j below 2^31
  int fixed_shift;
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
  unsigned* hist;         // [tiles][kDigits]: pairs of a tile by digit
  unsigned* hist16;       // [passes][(tiles + 15) / 16][kDigits]: of 16 tiles
  float* partial;         // [runs][2][pstride]: sums of a run's first row, when it began before the run,
                          // and of its last, when it began in the run and goes on
  float* super;           // [runs / 32][pstride]
  int pstride;
  int tiles, tile;        // sort tiles and lookups a tile
  int passes, bits;       // digits of the sort and bits of a digit
  int runs;
  // zeros
  int zero_rows, zero_blocks;   // table rows a CTA fills, and such CTAs (0: none)
  int word;                     // bytes of a store: 16, 4 or 2
};

// All loads are plain ones, not through the read-only path: this kernel's CTAs may be resident before what an earlier kernel of
// the chain has written is there, or a call ahead of it whose kernels let their successors in at their start (the
// forward call's winners, the indices that a window's compaction keeps).
__device__ __forceinline__ long long index_at(const void* p, int idx64, long long i) {
  return idx64 ? static_cast<const long long*>(p)[i] : (long long)static_cast<const int*>(p)[i];
}

// Row of a lookup's index in the table window, or num_rows where it contributes nothing.
__device__ __forceinline__ unsigned row_of(const BackArgs& a, long long idx, int bag) {
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
  // what malformed offsets name stays within the lookups: both ends index shared memory in the tiny kernel
  if (start < 0) start = 0;
  if (start > a.n) start = a.n;
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
// The same for two values over all starts by a whole CTA: every thread tests one start a round.
template <int THREADS>
__device__ __forceinline__ int2 upper_bound_cta(const BackArgs& a, long long j0, long long j1, int n) {
  int lo0 = 0, len0 = n, lo1 = 0, len1 = n;
  while (len0 > 0 || len1 > 0) {
    const int step0 = (len0 + THREADS - 1) / THREADS, step1 = (len1 + THREADS - 1) / THREADS;
    const long long at0 = lo0 + (long long)(threadIdx.x + 1) * step0 - 1;
    const long long at1 = lo1 + (long long)(threadIdx.x + 1) * step1 - 1;
    const bool in0 = step0 > 0 && at0 < lo0 + len0, in1 = step1 > 0 && at1 < lo1 + len1;
    const long long v0 = in0 ? index_at(a.offsets, a.idx64, at0) : 0;
    const long long v1 = in1 ? index_at(a.offsets, a.idx64, at1) : 0;
    const int c0 = __syncthreads_count(in0 && v0 <= j0), c1 = __syncthreads_count(in1 && v1 <= j1);
    const int next0 = lo0 + c0 * step0, next1 = lo1 + c1 * step1;
    len0 = step0 > 0 ? min(step0 - 1, lo0 + len0 - next0) : 0;
    len1 = step1 > 0 ? min(step1 - 1, lo1 + len1 - next1) : 0;
    lo0 = next0;
    lo1 = next1;
  }
  return make_int2(lo0, lo1);
}

// counted[b] = length of bag b; the kernel that makes the pairs takes the padding off.
__global__ void __launch_bounds__(256) bag_length_kernel(const BackArgs a) {
  pdl_enter(true);
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
__device__ __forceinline__ int clamp_start(long long s) { return s < 0 ? -1 : (s > INT_MAX ? INT_MAX : (int)s); }
template <int MOST>   // starts that fit `shared`
__device__ __forceinline__ TileStarts find_starts(const BackArgs& a, int begin, int end, int* shared) {
  TileStarts t = {0, 0, false};
  if (a.fixed_len > 0 || begin >= end) return t;
  const int n = a.num_bags > 0 ? a.num_bags + (a.include_last ? 1 : 0) : 0;
  const int2 found = upper_bound_cta<kSortThreads>(a, begin, end - 1, n);
  t.lo = found.x;
  t.hi = max(found.x, found.y);
  t.in_shared = t.hi - t.lo <= MOST;
  if (t.in_shared) {
    for (int i = t.lo + threadIdx.x; i < t.hi; i += kSortThreads)
      shared[i - t.lo] = clamp_start(index_at(a.offsets, a.idx64, i));
    __syncthreads();
  }
  return t;
}
// The bags of consecutive lookups, 32 at a time: a lane's bag is the last one that starts at or before its lookup, -1 where
// there is none.  The warp keeps the number of starts before its lookups and looks at the next 32.
struct BagWalk {
  int known;         // starts <= the last lookup walked
  template <typename Start>
  __device__ __forceinline__ int step(const BackArgs& a, int j, const TileStarts& t, Start start) {
    constexpr unsigned kAll = 0xffffffffu;
    const int lane = threadIdx.x & 31;
    const int s = known + lane < t.hi ? start(known + lane) : INT_MAX;
    const int last = __shfl_sync(kAll, j, 31);
    int count;
    if (__shfl_sync(kAll, s, 31) <= last) {          // more starts than lanes (empty bags): search all of them
      count = upper_bound(start, j, known, t.hi);
    } else {
      int at = 0;
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) {
        const int v = __shfl_sync(kAll, s, at + o - 1);
        at += v <= j ? o : 0;
      }
      count = known + at;
    }
    known = __shfl_sync(kAll, count, 31);
    const int bag = count - 1;
    return bag < a.num_bags ? bag : -1;              // behind the last offset of include_last_offset
  }
};
// Calls visit(i, bag) for a warp's lookups begin + 32 i + lane, ITEMS of them a lane, those at `end` and behind with -1.
template <int ITEMS, typename Visit>
__device__ __forceinline__ void walk_bags(const BackArgs& a, int begin, int end, const TileStarts& t, const int* shared,
                                          BagWalk& walk, Visit visit) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int i = 0; i < ITEMS; ++i) {
    const int j = begin + i * 32 + lane;
    int bag;
    if (a.fixed_len > 0) {
      bag = (int)(((unsigned long long)(unsigned)j * a.fixed_magic) >> (31 + a.fixed_shift));
      if (bag >= a.num_bags) bag = -1;
    } else if (t.in_shared) {
      bag = walk.step(a, j, t, [&](int k) { return shared[k - t.lo]; });
    } else {
      bag = walk.step(a, j, t, [&](int k) { return clamp_start(index_at(a.offsets, a.idx64, k)); });
    }
    visit(i, j < end ? bag : -1);
  }
}
__device__ __forceinline__ BagWalk walk_from(const BackArgs& a, int begin, const TileStarts& t, const int* shared) {
  BagWalk w = {t.lo};
  if (a.fixed_len == 0)
    w.known = t.in_shared ? upper_bound([&](int k) { return shared[k - t.lo]; }, begin - 1, t.lo, t.hi)
                          : upper_bound([&](int k) { return clamp_start(index_at(a.offsets, a.idx64, k)); }, begin - 1, t.lo, t.hi);
  return w;
}

// Padding is not counted for a mean: one subtraction a warp and bag.  All lanes of the warp call it.
__device__ __forceinline__ void uncount_padding(const BackArgs& a, long long idx, bool in, int bag) {
  const bool pad = in && bag >= 0 && idx == a.padding_idx;
  const unsigned same = __match_any_sync(0xffffffffu, pad ? bag : -1);
  if (pad && (threadIdx.x & 31) == __ffs(same) - 1) atomicSub(a.counted + bag, __popc(same));
}

// Zeros where the sums of 16 tiles will be counted.
__global__ void __launch_bounds__(kSortThreads) clear_sums_kernel(unsigned* hist16, int words) {
  pdl_enter(true);
  const int i = blockIdx.x * kSortThreads + threadIdx.x;
  if (i < words) hist16[i] = 0;
}

// A tile's histogram, and its share of the sums of 16 tiles.
__device__ __forceinline__ void put_counts(const BackArgs& a, const unsigned* count, int pass) {
  unsigned* sums = a.hist16 + (pass * ((a.tiles + 15) / 16) + blockIdx.x / 16) * kDigits;
  for (int d = threadIdx.x; d < kDigits; d += kSortThreads) {
    a.hist[blockIdx.x * kDigits + d] = count[d];
    if (count[d]) atomicAdd(sums + d, count[d]);
  }
}

// Every lookup's pair (and bag, where it is wanted apart), and the histogram of the first digit.  A warp takes consecutive
// lookups; all its indices are asked for at once (they may come from DRAM, a microsecond and a half a round).
template <int ITEMS>
__global__ void __launch_bounds__(kSortThreads) make_pairs_kernel(const BackArgs a, uint2* to) {
  pdl_enter(true);
  __shared__ unsigned count[kDigits];
  __shared__ int starts[kStarts];
  for (int d = threadIdx.x; d < kDigits; d += kSortThreads) count[d] = 0;
  const int begin = blockIdx.x * a.tile;
  const int end = min(a.n, begin + a.tile);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int share = (a.tile / 32 + kSortWarps - 1) / kSortWarps * 32;
  const int first = begin + warp * share, last = min(end, first + share);
  long long index[ITEMS];
  auto fetch = [&](int base) {
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) {
      const int j = base + i * 32 + lane;
      index[i] = j < last ? index_at(a.indices, a.idx64, j) : 0;
    }
  };
  fetch(first);
  const TileStarts t = find_starts<kStarts>(a, begin, end, starts);
  __syncthreads();
  BagWalk walk = walk_from(a, first, t, starts);
  const unsigned mask = (1u << a.bits) - 1u;
  for (int base = first; base < last; base += ITEMS * 32) {
    if (base != first) fetch(base);
    walk_bags<ITEMS>(a, base, last, t, starts, walk, [&](int i, int bag) {
      const int j = base + i * 32 + lane;
      if (j < last) {
        if (a.bag_of) a.bag_of[j] = bag;
        if (to) {
          const unsigned row = row_of(a, index[i], bag);
          to[j] = make_uint2(row, a.by_bag ? (unsigned)bag : (unsigned)j);
          atomicAdd(&count[row & mask], 1u);
        }
      }
      if (a.counted) uncount_padding(a, index[i], j < last, bag);
    });
  }
  __syncthreads();
  if (to) put_counts(a, count, 0);
}

// The histogram of a later digit.
template <int ITEMS>
__global__ void __launch_bounds__(kSortThreads) sort_histogram_kernel(const BackArgs a, const uint2* from, int pass) {
  pdl_enter(true);
  __shared__ unsigned count[kDigits];
  for (int d = threadIdx.x; d < kDigits; d += kSortThreads) count[d] = 0;
  __syncthreads();
  const int begin = blockIdx.x * a.tile;
  const int end = min(a.n, begin + a.tile);
  const unsigned mask = (1u << a.bits) - 1u;
  for (int base = begin; base < end; base += ITEMS * kSortThreads) {
    unsigned key[ITEMS];
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) {
      const int j = base + i * kSortThreads + threadIdx.x;
      key[i] = j < end ? from[j].x : 0;
    }
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) {
      if (base + i * kSortThreads + (int)threadIdx.x < end) atomicAdd(&count[(key[i] >> (pass * a.bits)) & mask], 1u);
    }
  }
  __syncthreads();
  put_counts(a, count, pass);
}

// Ranks of a CTA's items among those of the same digit, in the order of (warp, item, lane): in the warp here, and
// in_warp[w][d] becomes the number of warp w's items with digit d.  kNone is no digit.
template <int ITEMS>
__device__ __forceinline__ void rank_items(const unsigned (&digit)[ITEMS], unsigned (&rank)[ITEMS],
                                           unsigned (*in_warp)[kDigits], int bits) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  for (int i = threadIdx.x; i < kSortWarps * kDigits; i += kSortThreads) (&in_warp[0][0])[i] = 0;
  __syncthreads();
  const unsigned below = (1u << lane) - 1u;
  unsigned same[ITEMS];      // lanes with the same digit, by a vote a bit
#pragma unroll
  for (int i = 0; i < ITEMS; ++i) same[i] = __ballot_sync(0xffffffffu, digit[i] != kNone);
  for (int bit = 0; bit < bits; ++bit) {
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) {
      const bool set = (digit[i] >> bit) & 1u;
      const unsigned vote = __ballot_sync(0xffffffffu, set);
      same[i] &= set ? vote : ~vote;
    }
  }
#pragma unroll
  for (int i = 0; i < ITEMS; ++i) {
    const bool in = digit[i] != kNone;
    rank[i] = in ? in_warp[warp][digit[i]] + __popc(same[i] & below) : 0;
    __syncwarp();
    if (in && (same[i] & below) == 0) in_warp[warp][digit[i]] += __popc(same[i]);
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

// Moves a tile's pairs to their place in the order of digit `pass`, ties in the order they came.
template <int ITEMS>
struct DigitShared {
  uint2 pairs[ITEMS * kSortThreads];                   // in the digit's order
  unsigned in_warp[kSortWarps][kDigits];
  unsigned place[kDigits];                 // next free place of a digit
  unsigned local[kDigits];                 // first place of a digit in `pairs`
  unsigned total[kDigits / 32];
};
template <int ITEMS>
__global__ void __launch_bounds__(kSortThreads) sort_digit_kernel(const BackArgs a, const uint2* from, uint2* to, int pass) {
  pdl_enter(true);
  extern __shared__ uint4 dynamic[];
  DigitShared<ITEMS>& s = *reinterpret_cast<DigitShared<ITEMS>*>(dynamic);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int begin = blockIdx.x * a.tile;
  const int end = min(a.n, begin + a.tile);
  const int shift = pass * a.bits;
  const unsigned mask = (1u << a.bits) - 1u;
  uint2 pair[ITEMS];
  auto fetch = [&](int base) {
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) {
      const int j = base + (warp * ITEMS + i) * 32 + lane;
      pair[i] = j < end ? from[j] : make_uint2(0, 0);
    }
  };
  fetch(begin);
  // place[d] = keys with a lower digit + keys with digit d in earlier tiles: 4 digits a thread, and the tiles
  // shared among the threads of a digit, so that a thread's loads are few and all under way together.  Sums of 16
  // tiles stand for all tiles but the 16 around this one (293 tiles: 3 us less a digit)
  {
    const int digits = (int)mask + 1, columns = digits < 4 ? 1 : digits / 4, groups = min(kSortThreads / columns, 32);
    const int column = threadIdx.x % columns, group = threadIdx.x / columns;
    uint4 all = make_uint4(0, 0, 0, 0), before = all;
    if (group < groups) {
      const int sums = (a.tiles + 15) / 16, mine = (int)blockIdx.x / 16;
      const unsigned* hist16 = a.hist16 + pass * sums * kDigits;
      const unsigned* near = a.hist + mine * 16 * kDigits;           // the tiles that are looked at one by one
      const int rows = sums + (int)blockIdx.x - mine * 16;
#pragma unroll 6
      for (int r = group; r < rows; r += groups) {
        const uint4 c = reinterpret_cast<const uint4*>(r < sums ? hist16 + r * kDigits : near + (r - sums) * kDigits)[column];
        const unsigned w = r < sums ? 0xffffffffu : 0u;                       // of the whole count
        const unsigned m = r < mine || r >= sums ? 0xffffffffu : 0u;          // in earlier tiles
        all.x += c.x & w, all.y += c.y & w, all.z += c.z & w, all.w += c.w & w;
        before.x += c.x & m, before.y += c.y & m, before.z += c.z & m, before.w += c.w & m;
      }
    }
    // scratch: `pairs`, for 2 * groups * max(digits, 4) words
    uint4* scratch = reinterpret_cast<uint4*>(s.pairs);
    static_assert(sizeof(s.pairs) >= 2 * 4 * kSortThreads * 4, "a uint4 a thread, twice");
    if (group < groups) {
      scratch[group * columns + column] = all;
      scratch[(groups + group) * columns + column] = before;
    }
    __syncthreads();
    unsigned sum = 0, earlier = 0;
    if ((int)threadIdx.x < digits) {
      const unsigned* words = reinterpret_cast<const unsigned*>(s.pairs);
      for (int g = 0; g < groups; ++g) {
        sum += words[g * columns * 4 + threadIdx.x];
        earlier += words[(groups + g) * columns * 4 + threadIdx.x];
      }
    }
    const unsigned lower = digits_below(sum, s.total);
    if (threadIdx.x < kDigits) s.place[threadIdx.x] = lower + earlier;
    __syncthreads();
  }
  for (int base = begin; base < end; base += (ITEMS * kSortThreads)) {
    if (base != begin) {
      __syncthreads();
      fetch(base);
    }
    unsigned digit[ITEMS], rank[ITEMS];
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) {
      const int j = base + (warp * ITEMS + i) * 32 + lane;
      digit[i] = j < end ? (pair[i].x >> shift) & mask : kNone;
    }
    rank_items<ITEMS>(digit, rank, s.in_warp, a.bits);
    unsigned sum = 0;
    if (threadIdx.x < kDigits) {
#pragma unroll
      for (int w = 0; w < kSortWarps; ++w) sum += s.in_warp[w][threadIdx.x];
    }
    const unsigned local = digits_below(sum, s.total);
    if (threadIdx.x < kDigits) s.local[threadIdx.x] = local;
    __syncthreads();
    unsigned moved = local;
    if (threadIdx.x < kDigits) {     // in_warp: where a warp's first item of the digit goes in `pairs`
#pragma unroll
      for (int w = 0; w < kSortWarps; ++w) {
        const unsigned c = s.in_warp[w][threadIdx.x];
        s.in_warp[w][threadIdx.x] = moved;
        moved += c;
      }
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) {
      if (digit[i] != kNone) s.pairs[s.in_warp[warp][digit[i]] + rank[i]] = pair[i];
    }
    __syncthreads();
    const int count = min((ITEMS * kSortThreads), end - base);
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) {
      const int k = i * kSortThreads + threadIdx.x;
      if (k >= count) continue;
      const uint2 p = s.pairs[k];
      const unsigned d = (p.x >> shift) & mask;
      to[s.place[d] + (k - s.local[d])] = p;
    }
    __syncthreads();
    if (threadIdx.x < kDigits) s.place[threadIdx.x] += sum;
  }
}

// What a CTA needs to sort up to ITEMS * kSortThreads lookups by itself.
template <int ITEMS>
struct SmallSort {
  uint2 pairs[ITEMS * kSortThreads];     // the bag starts before the first digit, then the pairs between digits
  unsigned place[kDigits];
  unsigned in_warp[kSortWarps][kDigits];
  unsigned total[kDigits / 32];
};
// Finds the bags of all lookups and sorts them by row into `to` (shared or global memory).
template <int ITEMS>
__device__ __forceinline__ void sort_all(const BackArgs& a, SmallSort<ITEMS>& s, uint2* to, bool keep_bags) {
  int* starts = reinterpret_cast<int*>(s.pairs);
  constexpr int kFit = ITEMS * kSortThreads * 2;        // starts that fit there
  const unsigned mask = (1u << a.bits) - 1u;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int first = warp * ITEMS * 32;
  long long index[ITEMS];
#pragma unroll
  for (int i = 0; i < ITEMS; ++i) {
    const int j = first + i * 32 + lane;
    index[i] = j < a.n ? index_at(a.indices, a.idx64, j) : 0;
  }
  const TileStarts t = find_starts<(kFit < kStarts ? kFit : kStarts)>(a, 0, a.n, starts);
  uint2 pair[ITEMS];
  BagWalk walk = walk_from(a, first, t, starts);
  walk_bags<ITEMS>(a, first, a.n, t, starts, walk, [&](int i, int bag) {
    const int j = first + i * 32 + lane;
    pair[i] = make_uint2(0, 0);
    if (j < a.n) {
      if (keep_bags && a.bag_of) a.bag_of[j] = bag;
      pair[i] = make_uint2(row_of(a, index[i], bag), a.by_bag ? (unsigned)bag : (unsigned)j);
    }
    if (a.counted && keep_bags) uncount_padding(a, index[i], j < a.n, bag);
  });
  for (int pass = 0; pass < a.passes; ++pass) {
    unsigned digit[ITEMS], rank[ITEMS];
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) {
      const int j = first + i * 32 + lane;
      digit[i] = j < a.n ? (pair[i].x >> (a.bits * pass)) & mask : kNone;
    }
    rank_items<ITEMS>(digit, rank, s.in_warp, a.bits);
    unsigned sum = 0;
    if (threadIdx.x < kDigits) {
#pragma unroll
      for (int w = 0; w < kSortWarps; ++w) sum += s.in_warp[w][threadIdx.x];
    }
    const unsigned lower = digits_below(sum, s.total);
    if (threadIdx.x < kDigits) s.place[threadIdx.x] = lower;
    __syncthreads();
    place_warps(s.in_warp, s.place);
    const bool last = pass + 1 == a.passes;
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) {
      if (digit[i] == kNone) continue;
      const unsigned at = s.in_warp[warp][digit[i]] + rank[i];
      if (last) to[at] = pair[i]; else s.pairs[at] = pair[i];
    }
    __syncthreads();
    if (last) break;
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) {
      const int j = first + i * 32 + lane;
      if (j < a.n) pair[i] = s.pairs[j];
    }
    __syncthreads();
  }
}

// Up to kSmall lookups: one CTA sorts them.
__global__ void __launch_bounds__(kSortThreads) sort_small_kernel(const BackArgs a, uint2* to) {
  pdl_enter(true);
  __shared__ SmallSort<kSmallItems> s;
  sort_all<kSmallItems>(a, s, to, a.bag_of != nullptr || a.counted != nullptr);
}

// won[b][c] = the low byte of the position that won column c of bag b: what the sum below compares in bags of
// fewer than 256 lookups, an eighth of the pairs' bytes.
__global__ void __launch_bounds__(256) winner_bytes_kernel(const BackArgs a) {
  pdl_enter(true);
  const long long total = (long long)a.num_bags * a.dim;
  for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < total; i += (long long)gridDim.x * 256) {
    const long long bag = i / a.dim;
    const int col = (int)(i - bag * a.dim);
    a.won[bag * a.pstride + col] = (unsigned char)a.winners[bag * a.win_stride + col].y;
  }
}

template <int VE>
__device__ __forceinline__ void load_either(const char* row, int f16, int col, float (&x)[VE]) {
  if (f16) {
    Pack<__half, VE> r;
    r.load(reinterpret_cast<const __half*>(row) + col);
    r.get(x);
  } else {
    Pack<float, VE> r;
    r.load(reinterpret_cast<const float*>(row) + col);
    r.get(x);
  }
}
template <int VE>
__device__ __forceinline__ void store_either(char* row, int f16, int col, const float (&x)[VE]) {
  if (f16) {
    Pack<__half, VE> r;
    r.set(x);
    r.store(reinterpret_cast<__half*>(row) + col);
  } else {
    Pack<float, VE> r;
    r.set(x);
    r.store(reinterpret_cast<float*>(row) + col);
  }
}
// row += x.  fp32 adds where the row lies, in the L2: one addition an element and call, so its order does not
// matter, and the warp waits for nothing.  fp16 adds in fp32 and rounds once.
template <int VE>
__device__ __forceinline__ void add_either(char* row, int f16, int col, const float (&x)[VE]) {
  if (f16) {
    float old[VE];
    load_either<VE>(row, 1, col, old);
#pragma unroll
    for (int i = 0; i < VE; ++i) old[i] += x[i];
    store_either<VE>(row, 1, col, old);
    return;
  }
  float* to = reinterpret_cast<float*>(row) + col;
  if constexpr (VE % 4 == 0) {
#pragma unroll
    for (int i = 0; i < VE; i += 4)
      asm volatile("red.global.add.v4.f32 [%0], {%1, %2, %3, %4};"
                   :: "l"(to + i), "f"(x[i]), "f"(x[i + 1]), "f"(x[i + 2]), "f"(x[i + 3]) : "memory");
  } else {
#pragma unroll
    for (int i = 0; i < VE; ++i) asm volatile("red.global.add.f32 [%0], %1;" :: "l"(to + i), "f"(x[i]) : "memory");
  }
}

// Each nibble 8 + k of `which` makes a byte of copies of byte k's top bit.
__device__ __forceinline__ unsigned spread_top(unsigned x, unsigned which) {
  unsigned y;
  asm("prmt.b32 %0, %1, 0, %2;" : "=r"(y) : "r"(x), "r"(which));
  return y;
}

// acc[i] += g[i] in the columns whose byte of `won` is `at` (below 255).
template <typename TG, int VE>
__device__ __forceinline__ void add_won(float (&acc)[VE], const Pack<TG, VE>& g, const Pack<unsigned char, VE>& won, unsigned at) {
  if constexpr (VE % 4 == 0) {
    unsigned w[VE / 4], v[VE * sizeof(TG) / 4];
    memcpy(w, won.w, sizeof(w));
    memcpy(v, g.w, sizeof(v));
#pragma unroll
    for (int k = 0; k < VE / 4; ++k) {
      const unsigned d = w[k] ^ (at * 0x01010101u);
      const unsigned hit = ~(((d & 0x7f7f7f7fu) + 0x7f7f7f7fu) | d) & 0x80808080u;   // the top bit of each zero byte
      if constexpr (sizeof(TG) == 2) {
        // a byte's top bit spread over a half, and over the next
        const unsigned lo = v[2 * k] & spread_top(hit, 0x9988), hi = v[2 * k + 1] & spread_top(hit, 0xbbaa);
        asm("add.rn.f32.f16 %0, %1, %0;" : "+f"(acc[4 * k]) : "h"((unsigned short)lo));
        asm("add.rn.f32.f16 %0, %1, %0;" : "+f"(acc[4 * k + 1]) : "h"((unsigned short)(lo >> 16)));
        asm("add.rn.f32.f16 %0, %1, %0;" : "+f"(acc[4 * k + 2]) : "h"((unsigned short)hi));
        asm("add.rn.f32.f16 %0, %1, %0;" : "+f"(acc[4 * k + 3]) : "h"((unsigned short)(hi >> 16)));
      } else {
        acc[4 * k] += __uint_as_float(v[4 * k] & spread_top(hit, 0x8888));
        acc[4 * k + 1] += __uint_as_float(v[4 * k + 1] & spread_top(hit, 0x9999));
        acc[4 * k + 2] += __uint_as_float(v[4 * k + 2] & spread_top(hit, 0xaaaa));
        acc[4 * k + 3] += __uint_as_float(v[4 * k + 3] & spread_top(hit, 0xbbbb));
      }
    }
  } else {
    unsigned char w[VE];
    float f[VE];
    memcpy(w, won.w, sizeof(w));
    g.get(f);
#pragma unroll
    for (int i = 0; i < VE; ++i) acc[i] += w[i] == at ? f[i] : 0.0f;
  }
}

// Store the finished sum of a row.
template <int VE>
__device__ __forceinline__ void store_row(const BackArgs& a, unsigned row, int col, float (&acc)[VE]) {
  char* to = a.grad_table + (long long)row * a.gt_stride;
  if (a.square) {
    float x[VE];
    load_either<VE>(a.table + (long long)row * a.table_stride, a.table_f16, col, x);
#pragma unroll
    for (int i = 0; i < VE; ++i) acc[i] *= 2.0f * x[i];
  }
  if (a.accumulate) add_either<VE>(to, a.gt_f16, col, acc);
  else store_either<VE>(to, a.gt_f16, col, acc);
}

// kPlain adds rows, kScaled takes a factor a lookup, kWeights does so and writes grad_weights, kMax masks columns,
// kSquare multiplies the sum by twice the table row.
enum Kind { kPlain = 0, kScaled = 1, kWeights = 2, kMax = 3, kSquare = 4 };

// The first pair whose row is >= each of two rows, by a warp: 32 probes a round.
__device__ __forceinline__ int2 find_rows(const uint2* pairs, int n, unsigned row0, unsigned row1) {
  constexpr unsigned kAll = 0xffffffffu;
  const int lane = threadIdx.x & 31;
  int lo0 = 0, len0 = n, lo1 = 0, len1 = n;
  while (len0 > 0 || len1 > 0) {
    const int step0 = (len0 + 31) / 32, step1 = (len1 + 31) / 32;
    const long long at0 = lo0 + (lane + 1LL) * step0 - 1, at1 = lo1 + (lane + 1LL) * step1 - 1;
    const bool in0 = step0 > 0 && at0 < lo0 + len0, in1 = step1 > 0 && at1 < lo1 + len1;
    const unsigned v0 = in0 ? pairs[at0].x : kNone, v1 = in1 ? pairs[at1].x : kNone;
    const int c0 = __popc(__ballot_sync(kAll, in0 && v0 < row0)), c1 = __popc(__ballot_sync(kAll, in1 && v1 < row1));
    const int next0 = lo0 + c0 * step0, next1 = lo1 + c1 * step1;
    len0 = step0 > 0 ? min(step0 - 1, lo0 + len0 - next0) : 0;
    len1 = step1 > 0 ? min(step1 - 1, lo1 + len1 - next1) : 0;
    lo0 = next0;
    lo1 = next1;
  }
  return make_int2(lo0, lo1);
}

constexpr int kZeroRows = 1024;      // at most, of a block
// Zeros in the rows [first, first + rows) of the table that are not marked in `named`, by a CTA.
__device__ __forceinline__ void fill_zeros(const BackArgs& a, const unsigned* named, long long first, int rows) {
  const int lane = threadIdx.x & 31, warps = blockDim.x >> 5;
  const int per_row = a.dim * (a.gt_f16 ? 2 : 4) / a.word;      // stores a row
  int shift = 5;                                                // a warp's lanes share 1, 2, 4, ... rows
  while (shift > 0 && (1 << (shift - 1)) >= per_row) --shift;
  const int at = lane & ((1 << shift) - 1), sub = lane >> shift, together = 32 >> shift;
  char* base = a.grad_table + first * a.gt_stride;
  if (a.word == 16 && per_row <= 1 << shift && at < per_row) {
    // a store a lane and row: 32 rows of one mark word at a time
    for (int g = threadIdx.x >> 5; g * 32 < rows; g += warps) {
      const unsigned word = named[g];
      const int most = min(32, rows - g * 32);
      char* to = base + (long long)(g * 32 + sub) * a.gt_stride + at * 16;
#pragma unroll 4
      for (int r = sub; r < most; r += together, to += together * a.gt_stride) {
        if (!(word >> r & 1u)) *reinterpret_cast<uint4*>(to) = make_uint4(0, 0, 0, 0);
      }
    }
    return;
  }
  for (int r = (threadIdx.x >> 5) * together + sub; r < rows; r += warps * together) {
    if (named[r >> 5] >> (r & 31) & 1u) continue;
    char* to = base + r * a.gt_stride;
    for (int w = at; w < per_row; w += 1 << shift) {
      if (a.word == 16) reinterpret_cast<uint4*>(to)[w] = make_uint4(0, 0, 0, 0);
      else if (a.word == 4) reinterpret_cast<unsigned*>(to)[w] = 0;
      else reinterpret_cast<unsigned short*>(to)[w] = 0;
    }
  }
}
// Fills the rows of a block of the table that no lookup names with zeros.
__device__ __forceinline__ void zero_block(const BackArgs& a, const uint2* pairs, int block) {
  __shared__ unsigned named[kZeroRows / 32];
  __shared__ int2 span;
  const long long first = (long long)block * a.zero_rows;
  const int rows = (int)min((long long)a.zero_rows, a.num_rows - first);
  for (int i = threadIdx.x; i < kZeroRows / 32; i += blockDim.x) named[i] = 0;
  if (threadIdx.x < 32) {
    const int2 found = find_rows(pairs, a.n, (unsigned)first, (unsigned)(first + rows));
    if (threadIdx.x == 0) span = found;
  }
  __syncthreads();
  // A lane looks at 32 pairs by their ends: one row's lookups (a popular row has thousands of such) need one mark; the
  // warp goes through the others together.
  const int lane = threadIdx.x & 31, warps = blockDim.x >> 5;
  auto mark = [&](unsigned row) {
    const unsigned k = row - (unsigned)first;
    atomicOr(&named[k >> 5], 1u << (k & 31));
  };
  for (int base = span.x + (threadIdx.x >> 5) * 1024; base < span.y; base += warps * 1024) {
    const int from = base + lane * 32, to = min(from + 32, span.y);
    unsigned row = kNone;
    bool mixed = false;
    if (from < to) {
      row = pairs[from].x;
      mixed = pairs[to - 1].x != row;
      if (!mixed) mark(row);
    }
    for (unsigned left = __ballot_sync(0xffffffffu, mixed); left != 0;) {
      unsigned rows4[4];
      bool in[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        in[u] = false;
        if (left == 0) continue;
        const int i = base + (__ffs(left) - 1) * 32 + lane;
        left &= left - 1;
        in[u] = i < span.y;
        if (in[u]) rows4[u] = pairs[i].x;
      }
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        if (in[u]) mark(rows4[u]);
      }
    }
  }
  __syncthreads();
  fill_zeros(a, named, first, rows);
}
__global__ void __launch_bounds__(256) zero_kernel(const BackArgs a) {     // no lookups at all
  pdl_enter(false);
  zero_block(a, nullptr, blockIdx.x);
}

// A warp per run of 32 sorted lookups and tile of 32 * VE columns.  The CTAs that fill with zeros are spread evenly
// among those that add.  ACC: what grad_table holds is added.
// A table row that is wanted is read with the loads of the row's first lookup, so that no load is waited for alone.
// SAME: the table and grad_table have grad_out's type; branches on their types in every unrolled step would not fit the
// instruction cache (4 M x 128 fp32, weighted and accumulated: 219 us a call against 232).  kWeights is held to
// 64 registers, four CTAs an SM: 205 us against 210.
template <typename TG, int VE, int KIND, bool ACC, bool SAME>
__global__ void __launch_bounds__(256, KIND == kWeights ? 4 : 0) segment_sum_kernel(const BackArgs a, const uint2* pairs) {
  pdl_enter(a.runs > 1);
  int cta = blockIdx.x;
  if (!ACC && a.zero_blocks > 0) {
    const int before = (int)((long long)cta * a.zero_blocks / gridDim.x);        // zero CTAs among the earlier ones
    if ((int)((long long)(cta + 1) * a.zero_blocks / gridDim.x) != before) {
      zero_block(a, pairs, before);
      return;
    }
    cta -= before;
  }
  const int of_run = (a.runs + 7) / 8;          // CTAs a tile of columns
  const int tile = cta / of_run;
  cta -= tile * of_run;
  constexpr bool kTable = KIND == kWeights || KIND == kSquare;
  const int gt_f16 = SAME ? sizeof(TG) == 2 : a.gt_f16, table_f16 = SAME ? sizeof(TG) == 2 : a.table_f16;
  constexpr int U = kTable || VE == 8 ? 4 : 8;   // lookups whose loads are issued together
  constexpr unsigned kAll = 0xffffffffu;
  const int lane = threadIdx.x & 31;
  const int run = cta * 8 + (threadIdx.x >> 5);
  if (run >= a.runs) return;
  const int base = run * kRun;
  const int col = (tile * 32 + lane) * VE;
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
  const unsigned left_row = __shfl_up_sync(kAll, pair.x, 1);
  // lookups at which a row begins (the run's first always counts)
  const unsigned heads = __ballot_sync(kAll, lane == 0 || (lane < valid && pair.x != left_row));
  if constexpr (kTable) {
    // the table rows of the run are asked for together: they come from DRAM, most of grad_out from the L2
    if (heads >> lane & 1u) {
      const char* row = a.table + (long long)pair.x * a.table_stride + (long long)tile * 32 * VE * (table_f16 ? 2 : 4);
      const int bytes = min(32 * VE, a.dim - tile * 32 * VE) * (table_f16 ? 2 : 4);
      for (int b = 0; b < bytes; b += 128) asm volatile("prefetch.global.L2 [%0];" :: "l"(row + b));
    }
  }
  float acc[VE];
  float x[kTable ? VE : 1];     // the running row of the table
#pragma unroll
  for (int i = 0; i < VE; ++i) acc[i] = 0.0f;
  bool began_before = __shfl_sync(kAll, pair.x, 0) == prev;

  auto put = [&](int last, bool goes_on) {         // the row whose last lookup here is `last` is done
    const unsigned row = __shfl_sync(kAll, pair.x, last);
    if (col_ok) {
      if (!began_before && !goes_on) {
        if constexpr (KIND == kSquare) {
#pragma unroll
          for (int i = 0; i < VE; ++i) acc[i] *= 2.0f * x[i];
        }
        char* to = a.grad_table + (long long)row * a.gt_stride;
        if constexpr (ACC) add_either<VE>(to, gt_f16, col, acc);
        else store_either<VE>(to, gt_f16, col, acc);
      } else {
        Pack<float, VE> r;
        r.set(acc);
        r.store(a.partial + ((long long)run * 2 + (began_before ? 0 : 1)) * a.pstride + col);
      }
    }
    began_before = false;
#pragma unroll
    for (int i = 0; i < VE; ++i) acc[i] = 0.0f;
  };
  for (int e0 = 0; e0 < valid; e0 += U) {
    Pack<TG, VE> g[U];
    [[maybe_unused]] Pack<unsigned char, VE> won[KIND == kMax ? U : 1];
    [[maybe_unused]] float xs[kTable ? U : 1][kTable ? VE : 1];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int b = __shfl_sync(kAll, bag, e0 + u);
      const bool in = e0 + u < valid && col_ok;
      g[u].zero();
      if (in) g[u].load(reinterpret_cast<const TG*>(a.grad_out + (long long)b * a.go_stride) + col);
      if constexpr (KIND == kMax) {
        won[u].zero();
        if (in) won[u].load(a.won + (long long)b * a.pstride + col);
      }
      if constexpr (kTable) {
        const unsigned r = __shfl_sync(kAll, pair.x, e0 + u);
        if (in && (heads >> (e0 + u) & 1u)) load_either<VE>(a.table + (long long)r * a.table_stride, table_f16, col, xs[u]);
      }
    }
    [[maybe_unused]] float dot[KIND == kWeights ? U : 1];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if constexpr (KIND == kWeights) dot[u] = 0.0f;
      if (e0 + u >= valid) continue;
      if (heads >> (e0 + u) & 1u) {
        if (e0 + u > 0) put(e0 + u - 1, false);
        if constexpr (kTable) {
#pragma unroll
          for (int i = 0; i < VE; ++i) x[i] = xs[u][i];
        }
      }
      if constexpr (KIND == kMax) {
        const int at = __shfl_sync(kAll, pos, e0 + u);
        if (at >= 0) {
          add_won<TG, VE>(acc, g[u], won[u], (unsigned)at);
        } else {
          const int b = __shfl_sync(kAll, bag, e0 + u);
          float f[VE];
          g[u].get(f);
          if (col_ok) {
            for (int i = 0; i < VE; ++i) {
              if (a.winners[(long long)b * a.win_stride + col + i].y == (at & INT_MAX)) acc[i] += f[i];
            }
          }
        }
        continue;
      }
      float f[VE];
      g[u].get(f);
      if constexpr (KIND == kWeights) {
        if (col_ok) {
#pragma unroll
          for (int i = 0; i < VE; ++i) dot[u] = fmaf(f[i], x[i], dot[u]);
        }
      }
      if constexpr (KIND == kScaled || KIND == kWeights) {
        const float c = __shfl_sync(kAll, coef, e0 + u);
#pragma unroll
        for (int i = 0; i + 1 < VE; i += 2) {
          const float2 t = fma2(both(c), make_float2(f[i], f[i + 1]), make_float2(acc[i], acc[i + 1]));
          acc[i] = t.x, acc[i + 1] = t.y;
        }
        if (VE == 1) acc[0] = fmaf(c, f[0], acc[0]);
      } else {
#pragma unroll
        for (int i = 0; i + 1 < VE; i += 2) {
          const float2 t = add2(make_float2(f[i], f[i + 1]), make_float2(acc[i], acc[i + 1]));
          acc[i] = t.x, acc[i + 1] = t.y;
        }
        if (VE == 1) acc[0] += f[0];
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
      static_assert(U == 4, "8 lanes share a value");
      const int u = lane >> 3;
      const unsigned j = __shfl_sync(kAll, pair.y, e0 + u);
      if ((lane & 7) == 0 && e0 + u < valid) a.grad_weights[j] = dot[0];
    }
  }
  put(valid - 1, __shfl_sync(kAll, pair.x, valid - 1) == next);
}

__device__ __forceinline__ unsigned first_row(const uint2* pairs, int run) { return pairs[run * kRun].x; }

// super[s] = sum of the 32 runs of block s, where one row's lookups fill all the block's run starts.  A CTA a block.
template <int VE>
__global__ void __launch_bounds__(256) segment_block_kernel(const BackArgs a, const uint2* pairs) {
  pdl_enter(true);
  __shared__ float part[8][32 * VE];
  const int run0 = blockIdx.x * kRun;
  if (run0 + kRun > a.runs || blockIdx.x == 0) return;
  const unsigned row = first_row(pairs, run0), before = pairs[run0 * kRun - 1].x, last = first_row(pairs, run0 + kRun - 1);
  if (row >= a.num_rows || before != row || last != row) return;       // the same for the CTA
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int col = (blockIdx.y * 32 + lane) * VE;
  Pack<float, VE> p[kRun / 8];
  float sum[VE];
#pragma unroll
  for (int u = 0; u < kRun / 8; ++u) {
    p[u].zero();
    if (col < a.dim) p[u].load(a.partial + (long long)(run0 + warp * (kRun / 8) + u) * 2 * a.pstride + col);
  }
#pragma unroll
  for (int i = 0; i < VE; ++i) sum[i] = 0.0f;
#pragma unroll
  for (int u = 0; u < kRun / 8; ++u) {
    float f[VE];
    p[u].get(f);
#pragma unroll
    for (int i = 0; i < VE; ++i) sum[i] += f[i];
  }
#pragma unroll
  for (int i = 0; i < VE; ++i) part[warp][lane * VE + i] = sum[i];
  __syncthreads();
  if (warp != 0 || col >= a.dim) return;
#pragma unroll
  for (int i = 0; i < VE; ++i) {
    sum[i] = 0.0f;
#pragma unroll
    for (int w = 0; w < 8; ++w) sum[i] += part[w][lane * VE + i];
  }
  Pack<float, VE> r;
  r.set(sum);
  r.store(a.super + (long long)blockIdx.x * a.pstride + col);
}

// Rows that cross runs.  A warp looks at 8 runs at once.  Most rows that start in one of them and go on end in the next:
// two pieces, added for four rows at a time.  Of the others the warp adds the pieces itself if they are few;
// else the CTA's 8 warps share them.
constexpr int kFewPieces = 24;
constexpr int kJoinRuns = 8;       // of a warp
template <int VE>
__global__ void __launch_bounds__(256) segment_join_kernel(const BackArgs a, const uint2* pairs) {
  pdl_enter(false);
  constexpr unsigned kAll = 0xffffffffu;
  __shared__ int long_from[8 * kJoinRuns], long_to[8 * kJoinRuns];
  __shared__ int longs;
  __shared__ float part[8][32 * VE];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int col = (blockIdx.y * 32 + lane) * VE;
  const bool col_ok = col < a.dim;
  if (threadIdx.x == 0) longs = 0;
  __syncthreads();
  const int run0 = (blockIdx.x * 8 + warp) * kJoinRuns;
  unsigned row = kNone;
  bool crosses = false, two = false;
  if (lane < kJoinRuns && run0 + lane + 1 < a.runs) {
    const int run = run0 + lane;
    row = pairs[run * kRun + kRun - 1].x;
    const unsigned before = run > 0 ? pairs[run * kRun - 1].x : kNone;
    const unsigned next = first_row(pairs, run + 1);
    const unsigned next2 = run + 2 < a.runs ? first_row(pairs, run + 2) : kNone;
    crosses = row < a.num_rows && before != row && next == row;
    two = crosses && next2 != row;
  }
  float acc[4][VE];
  for (unsigned left = __ballot_sync(kAll, two); left != 0;) {
    Pack<float, VE> tail[4], head[4];
    int at[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      at[u] = left != 0 ? __ffs(left) - 1 : -1;
      if (left != 0) left &= left - 1;
      if (at[u] >= 0 && col_ok) {
        const float* p = a.partial + (long long)(run0 + at[u]) * 2 * a.pstride + col;
        tail[u].load(p + a.pstride);
        head[u].load(p + 2 * a.pstride);
      }
    }
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      if (at[u] < 0) continue;
      const unsigned r = __shfl_sync(kAll, row, at[u]);
      if (!col_ok) continue;
      float t[VE], h[VE];
      tail[u].get(t);
      head[u].get(h);
#pragma unroll
      for (int i = 0; i < VE; ++i) t[i] += h[i];
      store_row<VE>(a, r, col, t);
    }
  }
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
    constexpr int kTogether = VE == 8 ? 4 : 8;
    for (int i0 = begin; i0 < end; i0 += kTogether) {
      Pack<float, VE> p[kTogether];
#pragma unroll
      for (int u = 0; u < kTogether; ++u) {
        p[u].zero();
        if (i0 + u < end) p[u].load(piece(i0 + u) + col);
      }
#pragma unroll
      for (int u = 0; u < kTogether; ++u) {
        float f[VE];
        p[u].get(f);
#pragma unroll
        for (int i = 0; i < VE; ++i) acc[u & 3][i] += f[i];
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
  for (unsigned left = __ballot_sync(kAll, crosses && !two); left != 0; left &= left - 1) {
    const int from = run0 + __ffs(left) - 1;
    const unsigned r = __shfl_sync(kAll, row, from - run0);
    // the last run that starts with the row: the next 32 at once, then 32 probes a round
    const unsigned ahead = from + 1 + lane < a.runs ? first_row(pairs, from + 1 + lane) : kNone;
    const unsigned same = __ballot_sync(kAll, ahead == r);
    int to = from + __ffs(~same) - 1;
    if (same == kAll) {
      to = from + 32;
      int len = a.runs - 1 - to;
      while (len > 0) {
        const int step = (len + 31) / 32;
        const long long at = to + (lane + 1LL) * step;
        const bool mine = at <= (long long)to + len && first_row(pairs, (int)at) == r;
        const int c = __popc(__ballot_sync(kAll, mine));
        len = min(step - 1, len - c * step);
        to += c * step;
      }
    }
    const int pieces = count_pieces(from, to);
    if (pieces > kFewPieces) {
      if (lane == 0) {
        const int k = atomicAdd(&longs, 1);
        long_from[k] = from;
        long_to[k] = to;
      }
      continue;
    }
    add_pieces(from, to, 0, pieces);
    if (col_ok) store_row<VE>(a, r, col, acc[0]);
  }
  __syncthreads();
  for (int k = 0; k < longs; ++k) {          // in any order: each is a row of its own
    const int from = long_from[k], to = long_to[k];
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
        for (int w = 0; w < 8; ++w) sum[i] += part[w][lane * VE + i];
      }
      store_row<VE>(a, pairs[from * kRun + kRun - 1].x, col, sum);
    }
    __syncthreads();
  }
}

// Up to kTiny lookups in one launch: every CTA sorts all of them for itself, a few microseconds that no other CTA has
// to be waited for, and takes its share of the rows.  A warp sums a row of up to 32 lookups, the CTA's
// warps together one of more; the rows that no lookup names are filled with zeros.  The kind of the call is
// a branch here: instructions do not count at this size, launches do.
template <int ITEMS>                // lookups a thread sorts
struct TinyShared {
  static constexpr int kMost = ITEMS * kSortThreads;
  SmallSort<ITEMS> sort;
  uint2 pairs[kMost];               // sorted
  int begins[kMost + 1];            // of each row's lookups
  int padding[kMost + 1];           // among the lookups before each
  int count;                        // rows
  int total;
  int warps[kSortWarps];
  unsigned named[kZeroRows / 32];
};
template <typename TG, int VE, int ITEMS>
__global__ void __launch_bounds__(kSortThreads) tiny_kernel(const BackArgs a, int kind) {
  pdl_enter(false);
  extern __shared__ uint4 dynamic[];
  TinyShared<ITEMS>& s = *reinterpret_cast<TinyShared<ITEMS>*>(dynamic);
  constexpr unsigned kAll = 0xffffffffu;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  sort_all<ITEMS>(a, s.sort, s.pairs, false);
  // sums over the threads before this one; s.total: over all
  auto scan = [&](int mine) {
    int sum = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int v = __shfl_up_sync(kAll, sum, o);
      if (lane >= o) sum += v;
    }
    if (lane == 31) s.warps[warp] = sum;
    __syncthreads();
    int all = 0;
    for (int w = 0; w < kSortWarps; ++w) {
      if (w < warp) sum += s.warps[w];
      all += s.warps[w];
    }
    __syncthreads();
    if (threadIdx.x == 0) s.total = all;
    return sum - mine;
  };
  const int k0 = threadIdx.x * ITEMS;
  const bool count_padding = a.mean && !a.mean_raw && a.padding_idx >= 0;
  if (count_padding) {     // padding[j]: of the lookups before j
    int mine = 0, is[ITEMS];
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) mine += is[i] = k0 + i < a.n && index_at(a.indices, a.idx64, k0 + i) == a.padding_idx;
    int at = scan(mine);
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) {
      if (k0 + i <= a.n) s.padding[k0 + i] = at;
      at += is[i];
    }
    if (threadIdx.x == kSortThreads - 1) s.padding[ITEMS * kSortThreads] = at;
    __syncthreads();
  }
  // the rows' first lookups, in order; those of no row (num_rows) sort last
  {
    int mine = 0, is[ITEMS], in = 0;
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) {
      const int k = k0 + i;
      const bool row = k < a.n && s.pairs[k].x < a.num_rows;
      in += row;
      mine += is[i] = row && (k == 0 || s.pairs[k - 1].x != s.pairs[k].x);
    }
    scan(in);
    __syncthreads();
    const int behind = s.total;
    __syncthreads();
    int at = scan(mine);
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) {
      if (is[i]) s.begins[at++] = k0 + i;
    }
    __syncthreads();
    if (threadIdx.x == 0) {
      s.count = s.total;
      s.begins[s.count] = behind;
    }
    __syncthreads();
  }
  const int rows = s.count, valid = s.begins[rows];
  auto bag_of_lookup = [&](unsigned payload) {
    if (a.by_bag) return (int)payload;
    const int j = (int)payload;
    if (a.fixed_len > 0) return j / a.fixed_len;
    return max(0, upper_bound([&](int i) { return index_at(a.offsets, a.idx64, i); }, j, 0, a.num_bags) - 1);
  };
  const int column_tiles = (a.dim + 32 * VE - 1) / (32 * VE);
  // the lookups [from, to) of one row into acc, columns `col` on
  auto add = [&](int from, int to, int col, float (&acc)[VE]) {
#pragma unroll
    for (int i = 0; i < VE; ++i) acc[i] = 0.0f;
    for (int base = from; base < to; base += 32) {
      const int most = min(32, to - base);
      int bag = 0, pos = 0;      // a lane finds one lookup's bag, position in it and factor
      float c = 1.0f;
      if (lane < most) {
        const unsigned payload = s.pairs[base + lane].y;
        bag = bag_of_lookup(payload);
        if (a.psw) c = a.psw[payload];
        if (a.mean || kind == kMax) {
          long long b, e;
          bag_range(a, bag, b, e);
          pos = (int)payload - (int)b;
          if (a.mean) c = 1.0f / (float)((int)(e - b) - (count_padding ? s.padding[e] - s.padding[b] : 0));
        }
      }
      constexpr int U = 4;
      for (int e0 = 0; e0 < most; e0 += U) {
        Pack<TG, VE> g[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const int b = __shfl_sync(kAll, bag, e0 + u);
          g[u].zero();
          if (e0 + u < most && col < a.dim)
            g[u].load(reinterpret_cast<const TG*>(a.grad_out + (long long)b * a.go_stride) + col);
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const int b = __shfl_sync(kAll, bag, e0 + u), p = __shfl_sync(kAll, pos, e0 + u);
          const float f = __shfl_sync(kAll, c, e0 + u);
          if (e0 + u >= most || col >= a.dim) continue;
          float x[VE];
          g[u].get(x);
#pragma unroll
          for (int i = 0; i < VE; ++i) {
            if (kind == kMax) acc[i] += a.winners[(long long)b * a.win_stride + col + i].y == p ? x[i] : 0.0f;
            else acc[i] = fmaf(f, x[i], acc[i]);
          }
        }
      }
    }
  };
  // rows of up to 32 lookups, a warp each
  for (int r = blockIdx.x * kSortWarps + warp; r < rows; r += gridDim.x * kSortWarps) {
    const int from = s.begins[r], to = s.begins[r + 1];
    if (to - from > kRun) continue;
    for (int tile = 0; tile < column_tiles; ++tile) {
      const int col = (tile * 32 + lane) * VE;
      float acc[VE];
      add(from, to, col, acc);
      if (col < a.dim) store_row<VE>(a, s.pairs[from].x, col, acc);
    }
  }
  // rows of more, a CTA each: a warp takes consecutive shares, which are added in order
  float* part = reinterpret_cast<float*>(s.sort.in_warp);       // [16 warps][32 * VE]
  static_assert(sizeof(s.sort.in_warp) >= kSortWarps * 32 * VE * sizeof(float), "the warps' sums fit");
  for (int r = blockIdx.x; r < rows; r += gridDim.x) {
    const int from = s.begins[r], to = s.begins[r + 1];
    if (to - from <= kRun) continue;
    const int share = (to - from + kSortWarps - 1) / kSortWarps;
    for (int tile = 0; tile < column_tiles; ++tile) {
      const int col = (tile * 32 + lane) * VE;
      float acc[VE];
      add(min(to, from + warp * share), min(to, from + (warp + 1) * share), col, acc);
#pragma unroll
      for (int i = 0; i < VE; ++i) part[warp * 32 * VE + lane * VE + i] = acc[i];
      __syncthreads();
      if (warp == 0 && col < a.dim) {
#pragma unroll
        for (int i = 0; i < VE; ++i) {
          acc[i] = 0.0f;
#pragma unroll
          for (int w = 0; w < kSortWarps; ++w) acc[i] += part[w * 32 * VE + lane * VE + i];
        }
        store_row<VE>(a, s.pairs[from].x, col, acc);
      }
      __syncthreads();
    }
  }
  if (a.grad_weights) {      // a warp a lookup; the payload is the lookup
    for (int k = blockIdx.x * kSortWarps + warp; k < a.n; k += gridDim.x * kSortWarps) {
      const uint2 p = s.pairs[k];
      float dot = 0.0f;
      if (k < valid) {
        const char* g = a.grad_out + (long long)bag_of_lookup(p.y) * a.go_stride;
        for (int col = lane * VE; col < a.dim; col += 32 * VE) {
          Pack<TG, VE> r;
          float fg[VE], fx[VE];
          r.load(reinterpret_cast<const TG*>(g) + col);
          r.get(fg);
          load_either<VE>(a.table + (long long)p.x * a.table_stride, a.table_f16, col, fx);
#pragma unroll
          for (int i = 0; i < VE; ++i) dot = fmaf(fg[i], fx[i], dot);
        }
      }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) dot += __shfl_xor_sync(kAll, dot, o);
      if (lane == 0) a.grad_weights[p.y] = dot;
    }
  }
  for (int block = blockIdx.x; block < a.zero_blocks; block += gridDim.x) {
    const long long first = (long long)block * a.zero_rows;
    const int most = (int)min((long long)a.zero_rows, a.num_rows - first);
    __syncthreads();
    for (int i = threadIdx.x; i < kZeroRows / 32; i += kSortThreads) s.named[i] = 0;
    __syncthreads();
    for (int k = threadIdx.x; k < valid; k += kSortThreads) {
      const long long r = (long long)s.pairs[k].x - first;
      if (r >= 0 && r < most) atomicOr(&s.named[r >> 5], 1u << (r & 31));
    }
    __syncthreads();
    fill_zeros(a, s.named, first, most);
  }
}

// grad_weights[j] = <table[row j], grad_out[bag j]>.  A warp takes up to 32 lookups at a time: a lane finds one's bag and row,
// and the rows of U lookups are under way together, four where one load a lane covers a row, else two.  With the lookups
// behind one another, each after the last one's store, 655 k of a 1 M x 128 fp32 table took 172 us a call (now 73),
// 300 k of a 1 M x 256 fp32 table 110 (now 66).
template <typename TG, typename TT, int VE, int U>
__global__ void __launch_bounds__(256) weight_gradient_kernel(const BackArgs a, int share) {
  pdl_enter(a.pairs[0] != nullptr);     // the sums follow where the table's gradient is wanted too
  constexpr unsigned kAll = 0xffffffffu;
  const int lane = threadIdx.x & 31;
  const long long step = (long long)gridDim.x * 8 * share;      // share: a multiple of U
  for (long long base = ((long long)blockIdx.x * 8 + (threadIdx.x >> 5)) * share; base < a.n; base += step) {
    const int most = (int)min((long long)share, a.n - base);
    int bag = 0;
    unsigned row = a.num_rows;
    if (lane < most) {
      bag = a.bag_of[base + lane];
      row = row_of(a, index_at(a.indices, a.idx64, base + lane), bag);
    }
    float mine = 0.0f;
    for (int e0 = 0; e0 < most; e0 += U) {
      float s[U];
      const TG* g[U];
      const TT* x[U];
      bool in[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        s[u] = 0.0f;
        const unsigned r = __shfl_sync(kAll, row, e0 + u);
        const int b = __shfl_sync(kAll, bag, e0 + u);
        in[u] = r < a.num_rows;         // not so behind the last lookup
        g[u] = reinterpret_cast<const TG*>(a.grad_out + (in[u] ? (long long)b * a.go_stride : 0));
        x[u] = reinterpret_cast<const TT*>(a.table + (in[u] ? (long long)r * a.table_stride : 0));
      }
      auto columns = [&](int col) {
        Pack<TG, VE> pg[U];
        Pack<TT, VE> px[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
          pg[u].zero();
          px[u].zero();
          if (in[u]) {
            pg[u].load(g[u] + col);
            px[u].load(x[u] + col);
          }
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
          float fg[VE], fx[VE];
          pg[u].get(fg);
          px[u].get(fx);
#pragma unroll
          for (int i = 0; i < VE; ++i) s[u] = fmaf(fg[i], fx[i], s[u]);
        }
      };
      if constexpr (U == 4) {
        if (lane * VE < a.dim) columns(lane * VE);
      } else {
#pragma unroll 2
        for (int col = lane * VE; col < a.dim; col += 32 * VE) columns(col);
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) s[u] += __shfl_xor_sync(kAll, s[u], o);
        if (lane == e0 + u) mine = s[u];
      }
    }
    if (lane < most) a.grad_weights[base + lane] = mine;
  }
}

// ---- host -----------------------------------------------------------------------------

struct BackPlan {
  BackArgs a;
  int ve;                    // columns a lane
  bool want_table;
  bool fused_weights;        // grad_weights comes out of the segment sum
  bool tiny;                 // one launch does everything
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
  if (f.dim > kMostColumns) return fail(FWD_EB_ETOOBIG, "the gradient takes rows of up to 2^20 columns");
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

  int bits = 1;
  while (bits < 32 && (a.num_rows >> bits) != 0) ++bits;     // num_rows itself is a key
  a.passes = (bits + 7) / 8;
  a.bits = (bits + a.passes - 1) / a.passes;
  // two sort CTAs an SM: 1.3 M lookups 232 us a call against 264 with one of twice the lookups
  const long long per = ((long long)a.n + 2 * sm_count() - 1) / (2 * sm_count());
  a.tile = (int)(per < 1024 ? 1024 : (per + 31) / 32 * 32);
  a.tiles = (int)(((long long)a.n + a.tile - 1) / a.tile);
  a.runs = (int)(((long long)a.n + kRun - 1) / kRun);
  a.pstride = (f.dim + 7) / 8 * 8;
  pl->fused_weights = pl->want_table && a.grad_weights && f.dim <= 32 * pl->ve;
  if (a.fixed_len > 0) {
    while ((1LL << a.fixed_shift) < a.fixed_len) ++a.fixed_shift;
    a.fixed_magic = (unsigned)(((1ull << (31 + a.fixed_shift)) + a.fixed_len - 1) / a.fixed_len);
  }
  if (pl->want_table && !a.accumulate) {   // about 128 KB a CTA
    const long long row_bytes = (long long)f.dim * (int64_t)te;
    a.word = aligned_to(a.grad_table, 16) && a.gt_stride % 16 == 0 && row_bytes % 16 == 0 ? 16 : (int)te;
    const long long rows = (128 * 1024 + row_bytes - 1) / row_bytes;
    a.zero_rows = (int)(rows > kZeroRows ? kZeroRows : rows);
    const long long blocks = (f.num_rows + a.zero_rows - 1) / a.zero_rows;
    a.zero_blocks = (int)blocks;
  }
  a.by_bag = !a.winners && !a.psw && !pl->fused_weights;
  // One launch for few lookups, although every CTA sorts them all and a popular row is the work of one CTA: 320 lookups
  // of a 10000 x 64 fp32 table 7.2 us against 17.0 in three launches, 1024 lookups 9.3 against 18.8, all 1024 of one
  // row of it 17.2 against 18.5 (of a table of that row alone 16.8 against 14.2).  The zeros of large tables are faster from
  // the CTAs of the other form: 32 and 1024 lookups of 1 M x 128 fp16 (256 MB) 47 and 52 us against 51 and 56, of
  // 1 M x 128 fp32 (512 MB) 89 and 93 against 85 and 90, of 4 M x 128 fp32 328 and 330 against 289 and 294.
  const bool many_zeros = a.zero_blocks > 0 && f.num_rows * f.dim * (int64_t)te > 384LL << 20;
  pl->tiny = a.n <= kTiny && pl->want_table && !many_zeros;
  if (pl->tiny) {
    a.by_bag = !a.winners && !a.psw && !a.grad_weights;
    if (a.zero_blocks > 0) {      // a share of the zeros for every CTA
      const long long rows = (f.num_rows + sm_count() - 1) / sm_count();
      a.zero_rows = (int)(rows < 32 ? 32 : (rows < kZeroRows ? rows : kZeroRows));
      a.zero_blocks = (int)((f.num_rows + a.zero_rows - 1) / a.zero_rows);
    }
  }
  const bool bags_apart = !a.by_bag || (a.grad_weights && !pl->fused_weights);

  if (pl->tiny) return 0;     // no scratch

  // scratch, each part on a 256-byte border
  size_t at = 0;
  auto take = [&](size_t bytes) {
    const size_t here = at;
    at += (bytes + 255) & ~(size_t)255;
    return here;
  };
  char* ws = static_cast<char*>(p->workspace);
  const size_t n = (size_t)a.n;
  const size_t bag = take(bags_apart ? n * 4 : 0);
  a.bag_of = bags_apart ? reinterpret_cast<int*>(ws + bag) : nullptr;
  const bool count = a.mean && !a.mean_raw && a.padding_idx >= 0;
  const size_t counted = take(count ? (size_t)a.num_bags * 4 : 0);
  a.counted = count ? reinterpret_cast<int*>(ws + counted) : nullptr;
  if (pl->want_table) {
    a.pairs[0] = reinterpret_cast<uint2*>(ws + take(n * 8));
    a.pairs[1] = reinterpret_cast<uint2*>(ws + take(n * 8));
    a.hist = reinterpret_cast<unsigned*>(ws + take((size_t)a.tiles * kDigits * 4));
    a.hist16 = reinterpret_cast<unsigned*>(ws + take((size_t)a.passes * ((a.tiles + 15) / 16) * kDigits * 4));
    a.partial = reinterpret_cast<float*>(ws + take((size_t)a.runs * 2 * a.pstride * 4));
    const int blocks = a.runs / kRun;
    const size_t super = take((size_t)blocks * a.pstride * 4);
    // below that the rows' pieces are few enough to be added in one step (a launch less)
    a.super = blocks >= kRun ? reinterpret_cast<float*>(ws + super) : nullptr;
    a.won = reinterpret_cast<unsigned char*>(ws + take(a.winners ? (size_t)a.num_bags * a.pstride : 0));
  } else {
    a.passes = 0;
  }
  pl->bytes = a.n > 0 ? at : 0;
  return 0;
}

#define FWD_EB_TRY(...)                  \
  do {                                   \
    cudaError_t e_ = (__VA_ARGS__);      \
    if (e_ != cudaSuccess) return e_;    \
  } while (0)

template <typename TG, int VE, bool ACC, bool SAME>
cudaError_t launch_sums(const BackPlan& pl, dim3 grid, const uint2* sorted, cudaStream_t st) {
  const BackArgs& a = pl.a;
  if (a.winners) return launch_pdl(segment_sum_kernel<TG, VE, kMax, ACC, SAME>, grid, 256, 0, st, a, sorted);
  if (a.square) return launch_pdl(segment_sum_kernel<TG, VE, kSquare, ACC, SAME>, grid, 256, 0, st, a, sorted);
  if (pl.fused_weights) return launch_pdl(segment_sum_kernel<TG, VE, kWeights, ACC, SAME>, grid, 256, 0, st, a, sorted);
  if (a.psw || a.mean) return launch_pdl(segment_sum_kernel<TG, VE, kScaled, ACC, SAME>, grid, 256, 0, st, a, sorted);
  return launch_pdl(segment_sum_kernel<TG, VE, kPlain, ACC, SAME>, grid, 256, 0, st, a, sorted);
}

template <typename TG, int VE>
cudaError_t launch_segments(const BackPlan& pl, const uint2* sorted, cudaStream_t st) {
  const BackArgs& a = pl.a;
  const unsigned tiles = (unsigned)((a.dim + 32 * VE - 1) / (32 * VE));
  const dim3 grid((unsigned)((a.runs + 7) / 8), tiles);
  const long long ctas = (long long)grid.x * tiles + a.zero_blocks;
  if (ctas > INT_MAX) return cudaErrorInvalidConfiguration;
  const dim3 sums((unsigned)ctas);
  const bool f16 = sizeof(TG) == 2, same = (a.gt_f16 != 0) == f16 && (a.table_f16 != 0) == f16;
  if (a.accumulate) FWD_EB_TRY(same ? launch_sums<TG, VE, true, true>(pl, sums, sorted, st) : launch_sums<TG, VE, true, false>(pl, sums, sorted, st));
  else FWD_EB_TRY(same ? launch_sums<TG, VE, false, true>(pl, sums, sorted, st) : launch_sums<TG, VE, false, false>(pl, sums, sorted, st));
  if (a.super) {
    const dim3 blocks((unsigned)(a.runs / kRun), tiles);
    FWD_EB_TRY(launch_pdl(segment_block_kernel<VE>, blocks, 256, 0, st, a, sorted));
  }
  if (a.runs > 1) {
    const dim3 joins((unsigned)((a.runs + 8 * kJoinRuns - 1) / (8 * kJoinRuns)), tiles);
    FWD_EB_TRY(launch_pdl(segment_join_kernel<VE>, joins, 256, 0, st, a, sorted));
  }
  return cudaSuccess;
}

template <typename TG, int VE, int ITEMS>
cudaError_t launch_tiny_items(const BackArgs& a, unsigned ctas, cudaStream_t st) {
  constexpr int bytes = (int)sizeof(TinyShared<ITEMS>);
  FWD_EB_TRY(allow_shared<tiny_kernel<TG, VE, ITEMS>, bytes>());
  return launch_pdl(tiny_kernel<TG, VE, ITEMS>, dim3(ctas), kSortThreads, bytes, st, a, a.winners ? kMax : kPlain);
}
template <typename TG, int VE>
cudaError_t launch_tiny(const BackPlan& pl, cudaStream_t st) {
  const BackArgs& a = pl.a;
  // a warp a row, and CTAs for the zeros, up to one an SM
  const int want = (a.n + kSortWarps - 1) / kSortWarps, most = sm_count();
  int ctas = want > a.zero_blocks ? want : a.zero_blocks;
  if (ctas > most) ctas = most;
  return a.n <= kSortThreads ? launch_tiny_items<TG, VE, 1>(a, (unsigned)ctas, st) : launch_tiny_items<TG, VE, 2>(a, (unsigned)ctas, st);
}

template <typename TG>
cudaError_t launch_tiny_ve(const BackPlan& pl, cudaStream_t st) {
  switch (pl.ve) {
    case 8:
      if constexpr (sizeof(TG) == 2) return launch_tiny<TG, 8>(pl, st);
      return cudaErrorInvalidValue;
    case 4: return launch_tiny<TG, 4>(pl, st);
    case 2: return launch_tiny<TG, 2>(pl, st);
    default: return launch_tiny<TG, 1>(pl, st);
  }
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

template <typename TG, typename TT, int VE>
cudaError_t launch_weights_ve(const BackPlan& pl, cudaStream_t st) {
  const BackArgs& a = pl.a;
  // lookups a warp: up to 32 of narrow rows where 16 warps an SM are busy even so, up to 8 of wide ones where 64 are
  const bool narrow = a.dim <= 32 * VE;
  const int want = (narrow ? 16 : 64) * sm_count(), top = narrow ? 32 : 8, together = narrow ? 4 : 2;
  const long long per = ((long long)a.n + want - 1) / want;
  const int share = per < top ? (int)(per + together - 1) / together * together : top;
  const long long blocks = ((long long)a.n + 8 * share - 1) / (8 * share), most = 32LL * sm_count();
  const dim3 grid((unsigned)(blocks < most ? blocks : most));
  return narrow ? launch_pdl(weight_gradient_kernel<TG, TT, VE, 4>, grid, 256, 0, st, a, share)
                : launch_pdl(weight_gradient_kernel<TG, TT, VE, 2>, grid, 256, 0, st, a, share);
}
template <typename TG, typename TT>
cudaError_t launch_weights(const BackPlan& pl, cudaStream_t st) {
  switch (pl.ve) {
    case 8: return launch_weights_ve<TG, TT, 8>(pl, st);
    case 4: return launch_weights_ve<TG, TT, 4>(pl, st);
    case 2: return launch_weights_ve<TG, TT, 2>(pl, st);
    default: return launch_weights_ve<TG, TT, 1>(pl, st);
  }
}

// Pairs into pairs[1], then from one buffer to the other a digit at a time.
template <int ITEMS>
cudaError_t launch_sort(const BackPlan& pl, cudaStream_t st) {
  const BackArgs& a = pl.a;
  const dim3 tiles((unsigned)a.tiles);
  uint2* first = pl.want_table ? a.pairs[1] : nullptr;
  if (first) {
    const int words = a.passes * ((a.tiles + 15) / 16) * kDigits;
    FWD_EB_TRY(launch_pdl(clear_sums_kernel, dim3((unsigned)((words + kSortThreads - 1) / kSortThreads)), kSortThreads, 0, st,
                          a.hist16, words));
  }
  FWD_EB_TRY(launch_pdl(make_pairs_kernel<ITEMS>, tiles, kSortThreads, 0, st, a, first));
  int now = 1;
  for (int pass = 0; pass < a.passes; ++pass, now ^= 1) {
    const uint2* from = a.pairs[now];
    if (pass > 0) FWD_EB_TRY(launch_pdl(sort_histogram_kernel<ITEMS>, tiles, kSortThreads, 0, st, a, from, pass));
    constexpr int bytes = (int)sizeof(DigitShared<ITEMS>);
    FWD_EB_TRY(allow_shared<sort_digit_kernel<ITEMS>, bytes>());
    FWD_EB_TRY(launch_pdl(sort_digit_kernel<ITEMS>, tiles, kSortThreads, bytes, st, a, from, a.pairs[now ^ 1], pass));
  }
  return cudaSuccess;
}

cudaError_t launch_backward(const BackPlan& pl, const fwd_eb_backward_params* p, cudaStream_t st) {
  const BackArgs& a = pl.a;
  if (a.n == 0) return a.zero_blocks > 0 ? launch_pdl(zero_kernel, dim3((unsigned)a.zero_blocks), 256, 0, st, a) : cudaSuccess;
  if (pl.tiny) return p->grad_out_dtype == FWD_EB_F16 ? launch_tiny_ve<__half>(pl, st) : launch_tiny_ve<float>(pl, st);
  if (a.counted && a.num_bags > 0)
    FWD_EB_TRY(launch_pdl(bag_length_kernel, dim3((unsigned)((a.num_bags + 255) / 256)), 256, 0, st, a));
  if (pl.want_table && a.winners) {
    const long long blocks = ((long long)a.num_bags * a.dim + 255) / 256, most = 16LL * sm_count();
    if (blocks > 0)
      FWD_EB_TRY(launch_pdl(winner_bytes_kernel, dim3((unsigned)(blocks < most ? blocks : most)), 256, 0, st, a));
  }
  int now = 0;
  if (a.n <= kSmall && pl.want_table) {
    FWD_EB_TRY(launch_pdl(sort_small_kernel, dim3(1), kSortThreads, 0, st, a, a.pairs[0]));
  } else {
    FWD_EB_TRY(a.tile <= kItemsFew * kSortThreads ? launch_sort<kItemsFew>(pl, st) : launch_sort<kItemsMany>(pl, st));
    now = (1 + a.passes) & 1;
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
