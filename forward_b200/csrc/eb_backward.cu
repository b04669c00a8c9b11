// Gradient of a pooled lookup (include/fwd_eb_train.h).
//
// grad_table[r] is the sum of the grad_out rows of all lookups of r: a reduction by key whose keys
// are the indices.  Adding with atomics would take them in any order, so the lookups are
// sorted by row first: a stable radix sort of (row, lookup) pairs, digits of up to 8 bits, two
// kernels a digit (histogram of every tile, then scatter).  A warp then takes 32 sorted lookups, keeps
// its columns' running sum in registers, and stores a row's sum where the row's lookups end.  A row
// whose lookups cross from one run of 32 into the next leaves partial sums, which a last kernel adds in
// run order; a popular row's thousands of runs are first added 32 at a time.  Every sum has
// one order, whatever the schedule.
#include <climits>

#include "eb_train.cuh"

namespace fwd_eb {
namespace {

constexpr int kSortThreads = 512;
constexpr int kSortWarps = kSortThreads / 32;
constexpr int kItems = 4;                          // keys a thread handles at a time
constexpr int kSubTile = kSortThreads * kItems;
constexpr int kDigits = 256;
constexpr int kRun = 32;                           // sorted lookups of a run, runs of a block of runs
constexpr unsigned kNone = 0xffffffffu;

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
  float* grad_weights;
  int dim;
  int table_f16, gt_f16, square, accumulate;
  // scratch
  int* bag_of;            // [n]
  int* counted;           // [num_bags]: non-padding lookups (mean with a padding index)
  uint2* pairs[2];        // [n] {row, lookup}
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

// The bag that holds lookup j: the last one that starts at or before it; -1 where there is none.
__device__ __forceinline__ int find_bag(const BackArgs& a, int j, int lo, int hi) {
  // the number of starts <= j lies in [lo, hi]
  while (lo < hi) {
    const int mid = lo + (hi - lo) / 2;
    if (index_at(a.offsets, a.idx64, mid) <= j) lo = mid + 1; else hi = mid;
  }
  return lo - 1;
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

__global__ void __launch_bounds__(256) zero_rows_kernel(char* p, long long row_bytes, long long stride, long long rows,
                                                        int word) {
  pdl_enter();
  const long long per_row = row_bytes / word;
  const long long total = per_row * rows;
  for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < total; i += (long long)gridDim.x * 256) {
    char* q = per_row * word == stride ? p + i * word : p + (i / per_row) * stride + (i % per_row) * word;
    if (word == 16) *reinterpret_cast<uint4*>(q) = make_uint4(0, 0, 0, 0);
    else if (word == 4) *reinterpret_cast<unsigned*>(q) = 0;
    else *reinterpret_cast<unsigned short*>(q) = 0;
  }
}

// hist[tile][d] = keys of the tile whose digit is d.  FIRST: the keys are made from the indices, and
// bag_of is written.
template <bool FIRST>
__global__ void __launch_bounds__(kSortThreads) sort_histogram_kernel(const BackArgs a, const uint2* from, int shift) {
  pdl_enter();
  __shared__ unsigned count[kDigits];
  for (int d = threadIdx.x; d < kDigits; d += kSortThreads) count[d] = 0;
  __syncthreads();
  const int begin = blockIdx.x * a.tile;
  const int end = min(a.n, begin + a.tile);
  const int starts = a.num_bags > 0 ? a.num_bags + (a.include_last ? 1 : 0) : 0;
  int lo = 0, hi = starts;
  if (FIRST && a.fixed_len == 0) {   // the starts that this tile's lookups can lie behind
    lo = find_bag(a, begin, 0, starts) + 1;
    hi = find_bag(a, end - 1, lo, starts) + 1;
  }
  for (int base = begin; base < end; base += kSortThreads) {
    const int j = base + threadIdx.x;
    const bool in = j < end;
    unsigned key = 0;
    if (FIRST) {
      int bag = -1;
      if (in) {
        bag = a.fixed_len > 0 ? j / a.fixed_len : find_bag(a, j, lo, hi);
        if (bag >= a.num_bags) bag = -1;      // behind the last offset of include_last_offset
        a.bag_of[j] = bag;
        key = row_of(a, j, bag);
      }
      if (a.counted) {   // padding is not counted: one subtraction a warp and bag
        const bool pad = in && bag >= 0 && index_at(a.indices, a.idx64, j) == a.padding_idx;
        const unsigned same = __match_any_sync(0xffffffffu, pad ? bag : -1);
        if (pad && (threadIdx.x & 31) == __ffs(same) - 1) atomicSub(a.counted + bag, __popc(same));
      }
    } else if (in) {
      key = from[j].x;
    }
    if (in) atomicAdd(&count[(key >> shift) & (kDigits - 1)], 1u);
  }
  __syncthreads();
  for (int d = threadIdx.x; d < kDigits; d += kSortThreads) a.hist[blockIdx.x * kDigits + d] = count[d];
}

// Moves a tile's pairs to their place in the order of the digit, ties in the order they came.
template <bool FIRST>
__global__ void __launch_bounds__(kSortThreads) sort_scatter_kernel(const BackArgs a, const uint2* from, uint2* to,
                                                                    int shift) {
  pdl_enter();
  __shared__ unsigned place[kDigits];                    // next free place of a digit
  __shared__ unsigned in_warp[kSortWarps][kDigits];
  __shared__ unsigned scan[kSortThreads];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  // place[d] = keys with a lower digit + keys with digit d in earlier tiles
  {
    const int d = threadIdx.x & (kDigits - 1), half = threadIdx.x / kDigits;
    unsigned before = 0, all = 0;
    for (int t = half; t < a.tiles; t += kSortThreads / kDigits) {
      const unsigned c = a.hist[t * kDigits + d];
      all += c;
      before += t < (int)blockIdx.x ? c : 0;
    }
    in_warp[half][d] = before;
    scan[threadIdx.x] = all;
    __syncthreads();
    unsigned mine = 0;
    if (threadIdx.x < kDigits) {
      before = in_warp[0][d] + in_warp[1][d];
      all = scan[d] + scan[d + kDigits];
      mine = all;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const unsigned x = __shfl_up_sync(0xffffffffu, mine, o);
        if (lane >= o) mine += x;
      }
      if (lane == 31) place[warp] = mine;    // 8 warps' totals, for a moment
    }
    __syncthreads();
    unsigned lower = 0;
    if (threadIdx.x < kDigits) {
      for (int w = 0; w < warp; ++w) lower += place[w];
    }
    __syncthreads();
    if (threadIdx.x < kDigits) place[d] = lower + mine - all + before;
  }
  static_assert(kSortThreads == 2 * kDigits, "two threads a digit above");

  const int begin = blockIdx.x * a.tile;
  const int end = min(a.n, begin + a.tile);
  for (int base = begin; base < end; base += kSubTile) {
    __syncthreads();
    for (int i = threadIdx.x; i < kSortWarps * kDigits; i += kSortThreads) (&in_warp[0][0])[i] = 0;
    __syncthreads();
    uint2 pair[kItems];
    unsigned rank[kItems];
#pragma unroll
    for (int i = 0; i < kItems; ++i) {
      const int j = base + (warp * kItems + i) * 32 + lane;
      const bool in = j < end;
      pair[i] = make_uint2(0, 0);
      if (in) pair[i] = FIRST ? make_uint2(row_of(a, j, a.bag_of[j]), (unsigned)j) : from[j];
      const unsigned d = in ? (pair[i].x >> shift) & (kDigits - 1) : kNone;
      const unsigned same = __match_any_sync(0xffffffffu, d);
      rank[i] = in ? in_warp[warp][d] + __popc(same & ((1u << lane) - 1u)) : 0;
      __syncwarp();
      if (in && lane == __ffs(same) - 1) in_warp[warp][d] += __popc(same);
      __syncwarp();
    }
    __syncthreads();
    if (threadIdx.x < kDigits) {
      unsigned at = place[threadIdx.x];
      for (int w = 0; w < kSortWarps; ++w) {
        const unsigned c = in_warp[w][threadIdx.x];
        in_warp[w][threadIdx.x] = at;
        at += c;
      }
      place[threadIdx.x] = at;
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kItems; ++i) {
      const int j = base + (warp * kItems + i) * 32 + lane;
      if (j < end) to[in_warp[warp][(pair[i].x >> shift) & (kDigits - 1)] + rank[i]] = pair[i];
    }
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

enum Kind { kPlain = 0, kScaled = 1, kMax = 2 };

// A warp per run of 32 sorted lookups; blockIdx.y is a tile of 32 * VE columns.
template <typename TG, int VE, int KIND>
__global__ void __launch_bounds__(256) segment_sum_kernel(const BackArgs a, const uint2* pairs) {
  pdl_enter();
  const int lane = threadIdx.x & 31;
  const int run = blockIdx.x * 8 + (threadIdx.x >> 5);
  if (run >= a.runs) return;
  const int base = run * kRun;
  const int col = (blockIdx.y * 32 + lane) * VE;
  const bool col_ok = col < a.dim;
  uint2 pair = make_uint2(a.num_rows, 0);
  if (base + lane < a.n) pair = pairs[base + lane];
  const int valid = __popc(__ballot_sync(0xffffffffu, pair.x < a.num_rows));   // the rest sorts behind
  if (valid == 0) return;
  const unsigned prev = base > 0 ? pairs[base - 1].x : kNone;
  const unsigned next = base + kRun < a.n ? pairs[base + kRun].x : kNone;
  int bag = 0, pos = 0;
  float coef = 1.0f;
  if (lane < valid) {
    const int j = (int)pair.y;
    bag = a.bag_of[j];
    if (KIND == kScaled) {
      if (a.psw) {
        coef = a.psw[j];
      } else if (a.counted) {
        coef = 1.0f / (float)a.counted[bag];
      } else {
        long long s, e;
        bag_range(a, bag, s, e);
        coef = 1.0f / (float)(e - s);
      }
    } else if (KIND == kMax) {
      long long s, e;
      bag_range(a, bag, s, e);
      pos = j - (int)s;
    }
  }
  float acc[VE];
#pragma unroll
  for (int i = 0; i < VE; ++i) acc[i] = 0.0f;
  unsigned row = __shfl_sync(0xffffffffu, pair.x, 0);
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
  constexpr int U = 8;
  for (int e0 = 0; e0 < valid; e0 += U) {
    Pack<TG, VE> g[U];
    int2 win[KIND == kMax ? U : 1][KIND == kMax ? VE : 1];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int b = __shfl_sync(0xffffffffu, bag, e0 + u);
      g[u].zero();
      if (e0 + u < valid && col_ok) {
        g[u].load_ro(reinterpret_cast<const TG*>(a.grad_out + (long long)b * a.go_stride) + col);
        if (KIND == kMax) {
#pragma unroll
          for (int i = 0; i < VE; ++i) win[u][i] = __ldg(a.winners + (long long)b * a.win_stride + col + i);
        }
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const unsigned r = __shfl_sync(0xffffffffu, pair.x, e0 + u);
      const float c = __shfl_sync(0xffffffffu, coef, e0 + u);
      const int at = __shfl_sync(0xffffffffu, pos, e0 + u);
      if (e0 + u >= valid) continue;
      if (r != row) {
        put(false);
        row = r;
        began_before = false;
#pragma unroll
        for (int i = 0; i < VE; ++i) acc[i] = 0.0f;
      }
      float f[VE];
      g[u].get(f);
#pragma unroll
      for (int i = 0; i < VE; ++i) {
        if (KIND == kPlain) acc[i] += f[i];
        else if (KIND == kScaled) acc[i] = fmaf(c, f[i], acc[i]);
        else acc[i] += col_ok && win[u][i].y == at ? f[i] : 0.0f;
      }
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

// Rows that cross runs: a CTA looks at 8 runs and joins, one after the other, the rows that start in one of
// them and go on.  Its 8 warps take consecutive shares of the row's partial sums.
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
    const bool from_before = run > 0 && pairs[run * kRun - 1].x == row;
    if (row < a.num_rows && first_row(pairs, run + 1) == row && !from_before) {
      int lo = run + 1, hi = a.runs - 1;    // the last run that starts with the row
      while (lo < hi) {
        const int mid = hi - (hi - lo) / 2;
        if (first_row(pairs, mid) == row) lo = mid; else hi = mid - 1;
      }
      last = lo;
    }
  }
  if (lane == 0) last_run[warp] = last;
  __syncthreads();
  for (int w = 0; w < 8; ++w) {
    const int to = last_run[w];
    if (to < 0) continue;              // the same for the whole CTA
    const int from = blockIdx.x * 8 + w;
    // the row's pieces: its tail in `from`, single runs up to a block border, whole blocks, single runs
    const int first = from + 1;
    int b0 = (first + kRun - 1) / kRun, b1 = (to + 1) / kRun;     // whole blocks [b0, b1)
    if (!a.super || b1 < b0) b0 = b1 = 0;
    const bool blocks = b1 > b0;
    const int head = blocks ? b0 * kRun - first : to - first + 1;
    const int pieces = 1 + head + (blocks ? (b1 - b0) + (to + 1 - b1 * kRun) : 0);
    auto piece = [&](int i) -> const float* {
      if (i == 0) return a.partial + ((long long)from * 2 + 1) * a.pstride;
      i -= 1;
      if (i < head) return a.partial + (long long)(first + i) * 2 * a.pstride;
      i -= head;
      if (i < b1 - b0) return a.super + (long long)(b0 + i) * a.pstride;
      return a.partial + (long long)(b1 * kRun + (i - (b1 - b0))) * 2 * a.pstride;
    };
    const int share = (pieces + 7) / 8;
    const int begin = warp * share, end = min(pieces, begin + share);
    float acc[4][VE];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
#pragma unroll
      for (int i = 0; i < VE; ++i) acc[k][i] = 0.0f;
    }
    if (col_ok) {
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
    }
#pragma unroll
    for (int i = 0; i < VE; ++i) part[warp][lane * VE + i] = (acc[0][i] + acc[1][i]) + (acc[2][i] + acc[3][i]);
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
  const int most_tiles = sm_count();
  const long long per = ((long long)a.n + most_tiles - 1) / most_tiles;
  a.tile = (int)((per + kSortThreads - 1) / kSortThreads * kSortThreads);
  if (a.tile < kSortThreads) a.tile = kSortThreads;
  a.tiles = (int)(((long long)a.n + a.tile - 1) / a.tile);
  a.runs = (int)(((long long)a.n + kRun - 1) / kRun);
  a.pstride = (f.dim + 7) / 8 * 8;

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

cudaError_t launch_backward(const BackPlan& pl, const fwd_eb_backward_params* p, cudaStream_t st) {
  const BackArgs& a = pl.a;
  if (pl.want_table && !a.accumulate) {
    const long long row_bytes = (long long)a.dim * (a.gt_f16 ? 2 : 4);
    const bool wide = aligned_to(a.grad_table, 16) && a.gt_stride % 16 == 0 && row_bytes % 16 == 0;
    const int word = wide ? 16 : (a.gt_f16 ? 2 : 4);
    const long long words = row_bytes / word * a.num_rows, most = 8LL * sm_count();
    const long long blocks = (words + 255) / 256;
    FWD_EB_TRY(launch_pdl(zero_rows_kernel, dim3((unsigned)(blocks < most ? blocks : most)), 256, 0, st, a.grad_table,
                          row_bytes, a.gt_stride, (long long)a.num_rows, word));
  }
  if (a.n == 0) return cudaSuccess;
  if (a.counted && a.num_bags > 0)
    FWD_EB_TRY(launch_pdl(bag_length_kernel, dim3((unsigned)((a.num_bags + 255) / 256)), 256, 0, st, a));
  const dim3 tiles((unsigned)a.tiles);
  const uint2* none = nullptr;
  FWD_EB_TRY(launch_pdl(sort_histogram_kernel<true>, tiles, kSortThreads, 0, st, a, none, 0));
  if (a.grad_weights) {
    const bool g16 = p->grad_out_dtype == FWD_EB_F16;
    FWD_EB_TRY(g16 ? (a.table_f16 ? launch_weights<__half, __half>(pl, st) : launch_weights<__half, float>(pl, st))
                   : (a.table_f16 ? launch_weights<float, __half>(pl, st) : launch_weights<float, float>(pl, st)));
  }
  if (!pl.want_table) return cudaSuccess;
  FWD_EB_TRY(launch_pdl(sort_scatter_kernel<true>, tiles, kSortThreads, 0, st, a, none, a.pairs[0], 0));
  int now = 0;
  for (int pass = 1; pass < pl.passes; ++pass, now ^= 1) {
    const uint2* from = a.pairs[now];
    FWD_EB_TRY(launch_pdl(sort_histogram_kernel<false>, tiles, kSortThreads, 0, st, a, from, pass * 8));
    FWD_EB_TRY(launch_pdl(sort_scatter_kernel<false>, tiles, kSortThreads, 0, st, a, from, a.pairs[now ^ 1], pass * 8));
  }
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
