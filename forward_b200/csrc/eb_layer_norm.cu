// Layer norm of pooled rows and its gradients (include/fwd_eb_train.h).
//
// Both directions are bound by memory as long as few instructions are spent on an element.  TPR threads
// share a row, up to 16 elements each, and a CTA walks rows with a fixed grid: the next rows are
// under way to shared memory while this one is worked on (each thread copies what it will read itself, so
// no barrier stands between), the weights stay in registers, and so do a column's shares of
// grad_weight and grad_bias, which a second kernel adds in CTA order.  A row's values are converted
// once and stay in registers as fp32; the mean is taken first, then the squared distances from it (no
// cancellation).  Arithmetic is done on pairs (sm_100's packed fp32).
//
// Measured on B200 (a call, of the copy rate measured there): forward of 32768 x 4096 bf16 94-96 us, 0.86-0.87;
// backward of 16383 x 2000 bf16 50.5 us, 0.59: a row's chain of loads, two sums and one barrier, with 125 registers
// a thread leaving 16 warps an SM to hide it (8 elements a thread and twice the warps measured 59).
//
// Rows that do not fit the registers of a CTA take the *_loop kernels, which read them again for
// each pass.
#include <climits>
#include <cmath>

#include "eb_train.cuh"

namespace fwd_eb {
namespace {

struct NormArgs {
  const char* x;
  const char* gy;
  char* out;                 // y, or grad_x (may be null)
  const void* weight;
  const void* bias;
  float* mean;
  float* rstd;
  float* partial;            // [gridDim.x][2][cols] or null
  long long x_stride, gy_stride, out_stride;   // elements
  long long rows;
  int cols;
  int wtype;
  float eps;
};

// Sums over the TPR threads of a row, the same values in each.  `red` belongs to this call alone until every
// thread of the CTA has passed one more synchronisation: callers alternate between two.
template <int TPR, int K>
__device__ __forceinline__ void row_sum(float (&v)[K], float (*red)[K]) {
  constexpr int kWidth = TPR < 32 ? TPR : 32;
#pragma unroll
  for (int o = kWidth / 2; o > 0; o >>= 1) {
#pragma unroll
    for (int k = 0; k < K; ++k) v[k] += __shfl_xor_sync(0xffffffffu, v[k], o);
  }
  if constexpr (TPR > 32) {
    constexpr int kWarps = TPR / 32;
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int k = 0; k < K; ++k) {
      if (lane == k) red[threadIdx.x >> 5][k] = v[k];
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < K; ++k) v[k] = lane < kWarps ? red[lane][k] : 0.0f;
#pragma unroll
    for (int o = kWarps / 2; o > 0; o >>= 1) {
#pragma unroll
      for (int k = 0; k < K; ++k) v[k] += __shfl_xor_sync(0xffffffffu, v[k], o);
    }
#pragma unroll
    for (int k = 0; k < K; ++k) v[k] = __shfl_sync(0xffffffffu, v[k], 0);
  }
}
template <int TPR>
__device__ __forceinline__ float row_sum(float v, float (*red)[1]) {
  float one[1] = {v};
  row_sum<TPR, 1>(one, red);
  return one[0];
}

// sum / cols where a value is taken off that may be the mean itself (a row of one value): the product with 1 / cols, and what
// it leaves of the sum shared out once more.  Two fused operations; a division in their place cost the
// gradient of 32768 x 1000 bf16 5 % (50.6 us against 48.0).
__device__ __forceinline__ float mean_of(float sum, float cols, float inv_cols) {
  const float mean = sum * inv_cols, rest = fmaf(-mean, cols, sum);
  return rest == rest ? fmaf(rest, inv_cols, mean) : mean;     // an infinite sum stays
}

template <int VEC>
__device__ __forceinline__ void load_weight(const void* w, int dtype, int col, float unset, float (&f)[VEC]) {
  if (w) {
    load_any<VEC>(w, dtype, col, f);
  } else {
#pragma unroll
    for (int i = 0; i < VEC; ++i) f[i] = unset;
  }
}

// Threads of a CTA: one row above a warp (row_sum synchronises the CTA), else as many rows as fit 256 threads.
template <int TPR>
constexpr int kThreads = TPR <= 32 ? 256 : TPR;
inline int cta_threads(int tpr) { return tpr <= 32 ? 256 : tpr; }
// Threads an SM holds: the registers a thread may take (85 and 128).
constexpr int kForwardThreads = 768, kBackwardThreads = 512;
// Rows under way for each that is worked on.
constexpr int kForwardDepth = 2;
template <typename T>
constexpr int kBackwardDepth = sizeof(T) == 2 ? 3 : 2;
constexpr int resident_ctas(int threads, int cta) { return threads / cta < 1 ? 1 : threads / cta; }

// Elementwise on V fp32 values, in pairs where there are any.
template <int V, typename F2, typename F1>
__device__ __forceinline__ void each(F2 two, F1 one) {
#pragma unroll
  for (int i = 0; i + 1 < V; i += 2) two(i);
  if (V % 2) one(V - 1);
}
__device__ __forceinline__ float2 at2(const float* f, int i) { return make_float2(f[i], f[i + 1]); }
__device__ __forceinline__ void put2(float* f, int i, float2 v) {
  f[i] = v.x;
  f[i + 1] = v.y;
}

// The rows a thread is about to read, ARRAYS arrays of them: DEPTH rows ahead in shared memory where an
// access is 16 bytes, else one row ahead in registers.
template <typename T, int VEC, int NV, int TPR, int ARRAYS, int DEPTH>
struct Ahead {
  static constexpr bool kAsync = VEC * sizeof(T) == 16;
  static constexpr int kDepth = kAsync ? DEPTH : 1;
  static constexpr int kBytes = kAsync ? DEPTH * ARRAYS * NV * kThreads<TPR> * 16 : 0;   // of shared memory
  uint4* mine;                                  // [DEPTH][ARRAYS][NV][threads], this thread's
  Pack<T, VEC> reg[kAsync ? 1 : ARRAYS][kAsync ? 1 : NV];
  int slot;                                     // of the oldest row
  int cols, lane;
  __device__ __forceinline__ void init(void* shared, int cols_) {
    mine = static_cast<uint4*>(shared) + threadIdx.x;
    slot = 0;
    cols = cols_;
    lane = threadIdx.x % TPR;
  }
  __device__ __forceinline__ uint4* at(int s, int array, int k) {
    return mine + ((s * ARRAYS + array) * NV + k) * kThreads<TPR>;
  }
  // `from`: the row in each array; `live`: there is such a row.  s: 0 is behind the oldest row, kDepth - 1 the newest.
  __device__ __forceinline__ void fetch(const T* const (&from)[ARRAYS], bool live, int s) {
    int to = slot + s;
    if (to >= kDepth) to -= kDepth;
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const int col = (k * TPR + lane) * VEC;
#pragma unroll
      for (int q = 0; q < ARRAYS; ++q) {
        if constexpr (kAsync) {
          if (live && col < cols) copy16_async(at(to, q, k), from[q] + col);
        } else {
          reg[q][k].zero();
          if (live && col < cols) reg[q][k].load(from[q] + col);
        }
      }
    }
    if constexpr (kAsync) copy_commit();
  }
  // The oldest row's values (zeros behind its end) and its slot freed.
  __device__ __forceinline__ void take(float (&f)[ARRAYS][NV][VEC]) {
    if constexpr (kAsync) copy_wait<kDepth - 1>();
#pragma unroll
    for (int q = 0; q < ARRAYS; ++q) {
#pragma unroll
      for (int k = 0; k < NV; ++k) {
        Pack<T, VEC> r;
        if constexpr (kAsync) {
          r.zero();
          if ((k * TPR + lane) * VEC < cols) r.load(at(slot, q, k));
        } else {
          r = reg[q][k];
        }
        r.get(f[q][k]);
      }
    }
    if (++slot == kDepth) slot = 0;
  }
};

template <typename T, int VEC, int NV, int TPR>
__global__ void __launch_bounds__(kThreads<TPR>, kForwardThreads / kThreads<TPR> < 1 ? 1 : kForwardThreads / kThreads<TPR>)
layer_norm_forward_kernel(const NormArgs a) {
  pdl_enter(false);
  constexpr int kRows = kThreads<TPR> / TPR;
  __shared__ float red[2][32][1];
  const int lane = threadIdx.x % TPR;
  const float inv_cols = 1.0f / (float)a.cols;
  float w[NV][VEC], b[NV][VEC];
  extern __shared__ uint4 ring[];
  using Rows = Ahead<T, VEC, NV, TPR, 1, kForwardDepth>;
  Rows ahead;
  ahead.init(ring, a.cols);
  const long long step = (long long)gridDim.x * kRows;
  auto fetch = [&](long long row, int s) {
    const T* from[1] = {reinterpret_cast<const T*>(a.x) + row * a.x_stride};
    ahead.fetch(from, row < a.rows, s);
  };
  for (int s = 0; s < Rows::kDepth; ++s) fetch((long long)blockIdx.x * kRows + threadIdx.x / TPR + s * step, s);
#pragma unroll
  for (int k = 0; k < NV; ++k) {
    const int col = (k * TPR + lane) * VEC;
    const bool in = col < a.cols;
    load_weight<VEC>(in ? a.weight : nullptr, a.wtype, col, 1.0f, w[k]);
    load_weight<VEC>(in ? a.bias : nullptr, a.wtype, col, 0.0f, b[k]);
  }
  // every thread of the CTA makes the same number of turns
  for (long long base = (long long)blockIdx.x * kRows; base < a.rows; base += step) {
    const long long row = base + threadIdx.x / TPR;
    float taken[1][NV][VEC];
    ahead.take(taken);
    fetch(row + Rows::kDepth * step, Rows::kDepth - 1);
    float (&f)[NV][VEC] = taken[0];
    float2 sum = both(0.0f);
#pragma unroll
    for (int k = 0; k < NV; ++k)
      each<VEC>([&](int i) { sum = add2(sum, at2(f[k], i)); }, [&](int i) { sum.x += f[k][i]; });
    const float mean = mean_of(row_sum<TPR>(sum.x + sum.y, red[0]), (float)a.cols, inv_cols);
    float2 square = both(0.0f);
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      if ((k * TPR + lane) * VEC >= a.cols) continue;
      each<VEC>(
          [&](int i) {
            const float2 d = add2(at2(f[k], i), both(-mean));
            put2(f[k], i, d);
            square = fma2(d, d, square);
          },
          [&](int i) {
            f[k][i] -= mean;
            square.x = fmaf(f[k][i], f[k][i], square.x);
          });
    }
    const float rstd = 1.0f / sqrtf(fmaf(row_sum<TPR>(square.x + square.y, red[1]), inv_cols, a.eps));
    if (row >= a.rows) continue;
    if (lane == 0) {
      if (a.mean) a.mean[row] = mean;
      if (a.rstd) a.rstd[row] = rstd;
    }
    T* y = reinterpret_cast<T*>(a.out) + row * a.out_stride;
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const int col = (k * TPR + lane) * VEC;
      if (col >= a.cols) continue;
      each<VEC>([&](int i) { put2(f[k], i, fma2(mul2(at2(f[k], i), both(rstd)), at2(w[k], i), at2(b[k], i))); },
                [&](int i) { f[k][i] = fmaf(f[k][i] * rstd, w[k][i], b[k][i]); });
      Pack<T, VEC> out;
      out.set(f[k]);
      out.store(y + col);
    }
  }
}

// Rows of any width: three passes over the row, the last two mostly from L2.
template <typename T, int VEC>
__global__ void __launch_bounds__(1024)
layer_norm_forward_loop_kernel(const NormArgs a) {
  pdl_enter(false);
  __shared__ float red[2][32][1];
  const int step = blockDim.x * VEC;
  for (long long row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const T* x = reinterpret_cast<const T*>(a.x) + row * a.x_stride;
    T* y = reinterpret_cast<T*>(a.out) + row * a.out_stride;
    float sum = 0.0f, square = 0.0f;
    for (int col = threadIdx.x * VEC; col < a.cols; col += step) {
      Pack<T, VEC> r;
      float f[VEC];
      r.load(x + col);
      r.get(f);
#pragma unroll
      for (int i = 0; i < VEC; ++i) sum += f[i];
    }
    const float mean = row_sum<1024>(sum, red[0]) / (float)a.cols;
    for (int col = threadIdx.x * VEC; col < a.cols; col += step) {
      Pack<T, VEC> r;
      float f[VEC];
      r.load(x + col);
      r.get(f);
#pragma unroll
      for (int i = 0; i < VEC; ++i) square = fmaf(f[i] - mean, f[i] - mean, square);
    }
    const float rstd = 1.0f / sqrtf(row_sum<1024>(square, red[1]) / (float)a.cols + a.eps);
    if (threadIdx.x == 0) {
      if (a.mean) a.mean[row] = mean;
      if (a.rstd) a.rstd[row] = rstd;
    }
    for (int col = threadIdx.x * VEC; col < a.cols; col += step) {
      Pack<T, VEC> r;
      float f[VEC], w[VEC], b[VEC];
      load_weight<VEC>(a.weight, a.wtype, col, 1.0f, w);
      load_weight<VEC>(a.bias, a.wtype, col, 0.0f, b);
      r.load(x + col);
      r.get(f);
#pragma unroll
      for (int i = 0; i < VEC; ++i) f[i] = fmaf((f[i] - mean) * rstd, w[i], b[i]);
      r.set(f);
      r.store(y + col);
    }
  }
}

// grad_x of the rows this CTA walks, and its share of grad_weight and grad_bias.
template <typename T, int VEC, int NV, int TPR>
__global__ void __launch_bounds__(kThreads<TPR>, kBackwardThreads / kThreads<TPR> < 1 ? 1 : kBackwardThreads / kThreads<TPR>)
layer_norm_backward_kernel(const NormArgs a) {
  pdl_enter(a.partial != nullptr);
  constexpr int kRows = kThreads<TPR> / TPR;
  __shared__ float red[2][32][2];
  // the rows under way; at the end, with more than one row a CTA, [8 warps][2][cols] sums
  extern __shared__ uint4 ring[];
  const int lane = threadIdx.x % TPR;
  const float inv_cols = 1.0f / (float)a.cols;
  float w[NV][VEC], dw[NV][VEC], db[NV][VEC];
  using Rows = Ahead<T, VEC, NV, TPR, 2, kBackwardDepth<T>>;
  Rows ahead;
  ahead.init(ring, a.cols);
  const long long step = (long long)gridDim.x * kRows;
  float mean_next = 0.0f, rstd_next = 0.0f;
  auto fetch = [&](long long row, int s) {
    const T* from[2] = {reinterpret_cast<const T*>(a.x) + row * a.x_stride,
                        reinterpret_cast<const T*>(a.gy) + row * a.gy_stride};
    ahead.fetch(from, row < a.rows, s);
  };
  auto fetch_stats = [&](long long row) {
    if (row < a.rows) {
      mean_next = a.mean[row];
      rstd_next = a.rstd[row];
    }
  };
  {
    const long long row = (long long)blockIdx.x * kRows + threadIdx.x / TPR;
    for (int s = 0; s < Rows::kDepth; ++s) fetch(row + s * step, s);
    fetch_stats(row);
  }
#pragma unroll
  for (int k = 0; k < NV; ++k) {
    const int col = (k * TPR + lane) * VEC;
    load_weight<VEC>(col < a.cols ? a.weight : nullptr, a.wtype, col, 1.0f, w[k]);
#pragma unroll
    for (int i = 0; i < VEC; ++i) dw[k][i] = db[k][i] = 0.0f;
  }
  int turn = 0;
  for (long long base = (long long)blockIdx.x * kRows; base < a.rows; base += step, turn ^= 1) {
    const long long row = base + threadIdx.x / TPR;
    const bool live = row < a.rows;
    const float mean = mean_next, rstd = rstd_next;
    float taken[2][NV][VEC];
    ahead.take(taken);
    fetch(row + Rows::kDepth * step, Rows::kDepth - 1);
    fetch_stats(row + step);
    float (&h)[NV][VEC] = taken[0];   // x, then (x - mean) * rstd
    float (&g)[NV][VEC] = taken[1];   // grad_y, then grad_y * weight
    float2 s1 = both(0.0f), s2 = both(0.0f);
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      if (!live || (k * TPR + lane) * VEC >= a.cols) continue;
      each<VEC>(
          [&](int i) {
            const float2 hi = mul2(add2(at2(h[k], i), both(-mean)), both(rstd)), gy = at2(g[k], i);
            put2(dw[k], i, fma2(gy, hi, at2(dw[k], i)));
            put2(db[k], i, add2(gy, at2(db[k], i)));
            const float2 gw = mul2(gy, at2(w[k], i));
            s1 = add2(s1, gw);
            s2 = fma2(gw, hi, s2);
            put2(h[k], i, hi);
            put2(g[k], i, gw);
          },
          [&](int i) {
            const float hi = (h[k][i] - mean) * rstd;
            dw[k][i] = fmaf(g[k][i], hi, dw[k][i]);
            db[k][i] += g[k][i];
            const float gw = g[k][i] * w[k][i];
            s1.x += gw;
            s2.x = fmaf(gw, hi, s2.x);
            h[k][i] = hi;
            g[k][i] = gw;
          });
    }
    if (a.out) {
      float s[2] = {s1.x + s1.y, s2.x + s2.y};
      row_sum<TPR, 2>(s, red[turn]);
      const float m1 = mean_of(s[0], (float)a.cols, inv_cols), m2 = s[1] * inv_cols;
      T* gx = reinterpret_cast<T*>(a.out) + row * a.out_stride;
#pragma unroll
      for (int k = 0; k < NV; ++k) {
        const int col = (k * TPR + lane) * VEC;
        if (!live || col >= a.cols) continue;
        each<VEC>(
            [&](int i) {
              const float2 d = fma2(at2(h[k], i), both(-m2), add2(at2(g[k], i), both(-m1)));
              put2(g[k], i, mul2(d, both(rstd)));
            },
            [&](int i) { g[k][i] = rstd * fmaf(h[k][i], -m2, g[k][i] - m1); });
        Pack<T, VEC> out;
        out.set(g[k]);
        out.store(gx + col);
      }
    }
  }
  if (!a.partial) return;
  float* mine = a.partial + (long long)blockIdx.x * 2 * a.cols;
  if constexpr (kRows > 1) {
    // the row groups of a warp by shuffles, then the warps in order: the order of the additions is fixed
    constexpr int kWarps = kThreads<TPR> / 32;
#pragma unroll
    for (int o = TPR; o < 32; o <<= 1) {
#pragma unroll
      for (int k = 0; k < NV; ++k) {
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
          dw[k][i] += __shfl_xor_sync(0xffffffffu, dw[k][i], o);
          db[k][i] += __shfl_xor_sync(0xffffffffu, db[k][i], o);
        }
      }
    }
    float* share = reinterpret_cast<float*>(ring);
    if constexpr (Rows::kAsync) {   // nobody's copies land here any more
      copy_wait<0>();
      __syncthreads();
    }
    if ((threadIdx.x & 31) < TPR) {
      float* to = share + (threadIdx.x >> 5) * 2 * a.cols;
#pragma unroll
      for (int k = 0; k < NV; ++k) {
        const int col = (k * TPR + lane) * VEC;
        if (col >= a.cols) continue;
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
          to[col + i] = dw[k][i];
          to[a.cols + col + i] = db[k][i];
        }
      }
    }
    __syncthreads();
    for (int i = threadIdx.x; i < 2 * a.cols; i += kThreads<TPR>) {
      float sum = share[i];
#pragma unroll
      for (int k = 1; k < kWarps; ++k) sum += share[k * 2 * a.cols + i];
      mine[i] = sum;
    }
  } else {
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const int col = (k * TPR + lane) * VEC;
      if (col >= a.cols) continue;
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        mine[col + i] = dw[k][i];
        mine[a.cols + col + i] = db[k][i];
      }
    }
  }
}

// Rows of any width: grad_x, two passes over a row.
template <typename T, int VEC>
__global__ void __launch_bounds__(1024)
layer_norm_backward_loop_kernel(const NormArgs a) {
  pdl_enter(a.partial != nullptr);
  __shared__ float red[2][32][1];
  const int step = blockDim.x * VEC;
  for (long long row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const T* x = reinterpret_cast<const T*>(a.x) + row * a.x_stride;
    const T* gy = reinterpret_cast<const T*>(a.gy) + row * a.gy_stride;
    T* gx = reinterpret_cast<T*>(a.out) + row * a.out_stride;
    const float mean = a.mean[row], rstd = a.rstd[row];
    float s1 = 0.0f, s2 = 0.0f;
    for (int col = threadIdx.x * VEC; col < a.cols; col += step) {
      Pack<T, VEC> rx, rg;
      float fx[VEC], fg[VEC], w[VEC];
      rx.load(x + col);
      rg.load(gy + col);
      load_weight<VEC>(a.weight, a.wtype, col, 1.0f, w);
      rx.get(fx);
      rg.get(fg);
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        const float g = fg[i] * w[i];
        s1 += g;
        s2 = fmaf(g, (fx[i] - mean) * rstd, s2);
      }
    }
    s1 = row_sum<1024>(s1, red[0]) / (float)a.cols;
    s2 = row_sum<1024>(s2, red[1]) / (float)a.cols;
    for (int col = threadIdx.x * VEC; col < a.cols; col += step) {
      Pack<T, VEC> rx, rg;
      float fx[VEC], fg[VEC], w[VEC];
      rx.load(x + col);
      rg.load(gy + col);
      load_weight<VEC>(a.weight, a.wtype, col, 1.0f, w);
      rx.get(fx);
      rg.get(fg);
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        const float h = (fx[i] - mean) * rstd;
        fg[i] = rstd * (fmaf(fg[i], w[i], -s1) - h * s2);
      }
      rg.set(fg);
      rg.store(gx + col);
    }
  }
}

// Rows of any width: a thread sums one column over the rows of its slice (blockIdx.y).
template <typename T>
__global__ void __launch_bounds__(256)
layer_norm_columns_kernel(const NormArgs a) {
  pdl_enter(true);
  const long long col = (long long)blockIdx.x * blockDim.x + threadIdx.x;
  if (col >= a.cols) return;
  float dw = 0.0f, db = 0.0f;
  for (long long row = blockIdx.y; row < a.rows; row += gridDim.y) {
    const float g = to_float(reinterpret_cast<const T*>(a.gy)[row * a.gy_stride + col]);
    const float h = (to_float(reinterpret_cast<const T*>(a.x)[row * a.x_stride + col]) - a.mean[row]) * a.rstd[row];
    dw = fmaf(g, h, dw);
    db += g;
  }
  float* mine = a.partial + (long long)blockIdx.y * 2 * a.cols;
  mine[col] = dw;
  mine[a.cols + col] = db;
}

// grad_weight and grad_bias: column sums of partial [parts][2 * cols].  32 columns a CTA; 32 rows of threads
// take every 32nd part each, and their sums are added in order.
__global__ void __launch_bounds__(1024)
layer_norm_join_kernel(const float* partial, int parts, int cols, int wtype, void* gw, void* gb) {
  pdl_enter(false);
  __shared__ float part[32][33];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const long long col = (long long)blockIdx.x * 32 + lane;   // over both halves
  float s = 0.0f;
  if (col < 2LL * cols) {
#pragma unroll 8
    for (int p = warp; p < parts; p += 32) s += partial[(long long)p * 2 * cols + col];
  }
  part[warp][lane] = s;
  __syncthreads();
  s = part[lane][warp];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  const long long mine = (long long)blockIdx.x * 32 + warp;
  if (lane == 0 && mine < 2LL * cols) {
    void* to = mine < cols ? gw : gb;
    const float one[1] = {s};
    if (to) store_any<1>(to, wtype, mine < cols ? mine : mine - cols, one);
  }
}

// ---- host -----------------------------------------------------------------------------

constexpr int kLaneElements = 16;   // elements of a row a thread keeps

// How a call runs: elements a load and threads a row; tpr = 0 is the loop kernel.
struct NormPlan {
  int vec, tpr;
  int grid;        // CTAs of the main kernel
  int parts;       // backward: rows of the partial sums
};

bool known(int dtype) { return dtype == FWD_EB_F32 || dtype == FWD_EB_F16 || dtype == FWD_EB_BF16; }

int check_norm(const fwd_eb_layer_norm_params* p, bool backward) {
  if (!p) return fail(FWD_EB_EINVAL, "params is null");
  if (!known(p->dtype)) return fail(FWD_EB_EINVAL, "unknown dtype %d", p->dtype);
  if (!known(p->weight_dtype)) return fail(FWD_EB_EINVAL, "unknown weight_dtype %d", p->weight_dtype);
  if (p->rows < 0) return fail(FWD_EB_EINVAL, "rows is negative");
  if (p->cols < 1) return fail(FWD_EB_EINVAL, "cols must be positive (got %lld)", (long long)p->cols);
  if (p->cols > (1LL << 30)) return fail(FWD_EB_ETOOBIG, "cols is limited to 2^30 (got %lld)", (long long)p->cols);
  const size_t e = dtype_size(p->dtype), we = dtype_size(p->weight_dtype);
  const struct { const char* name; const void* p; int64_t stride; bool need; size_t size; } rows[] = {
      {"x", p->x, p->x_stride, true, e},
      {"y", backward ? nullptr : p->y, backward ? 0 : p->y_stride, !backward, e},
      {"grad_y", backward ? p->grad_y : nullptr, backward ? p->grad_y_stride : 0, backward, e},
      {"grad_x", backward ? p->grad_x : nullptr, backward ? p->grad_x_stride : 0, false, e},
      {"weight", p->weight, 0, false, we},
      {"bias", backward ? nullptr : p->bias, 0, false, we},
      {"grad_weight", backward ? p->grad_weight : nullptr, 0, false, we},
      {"grad_bias", backward ? p->grad_bias : nullptr, 0, false, we},
      {"mean", p->mean, 0, backward, 4},
      {"rstd", p->rstd, 0, backward, 4},
  };
  for (const auto& r : rows) {
    if (r.need && !r.p && p->rows > 0) return fail(FWD_EB_EINVAL, "%s is null", r.name);
    if (r.stride != 0 && r.stride < p->cols) return fail(FWD_EB_EINVAL, "%s_stride smaller than cols", r.name);
    if (!aligned_to(r.p, r.size)) return fail(FWD_EB_EALIGN, "%s is not aligned to its type", r.name);
  }
  if (!backward && !(p->eps >= 0.0 && std::isfinite(p->eps)))
    return fail(FWD_EB_EINVAL, "eps must be finite and not negative");
  return 0;
}

int64_t stride_of(int64_t s, int64_t cols) { return s ? s : cols; }

NormPlan plan_norm(const fwd_eb_layer_norm_params* p, bool backward) {
  NormPlan pl = {};
  const size_t e = dtype_size(p->dtype);
  const int full = (int)(16 / e);
  const void* a = backward ? p->grad_y : p->y;
  const void* b = backward ? p->grad_x : nullptr;
  const int64_t sa = stride_of(backward ? p->grad_y_stride : p->y_stride, p->cols);
  const int64_t sb = backward && b ? stride_of(p->grad_x_stride, p->cols) : 0;
  const size_t wbytes = dtype_size(p->weight_dtype) * full < 16 ? dtype_size(p->weight_dtype) * full : 16;
  const bool vec = p->cols % full == 0 && stride_of(p->x_stride, p->cols) % full == 0 && sa % full == 0 &&
                   sb % full == 0 && aligned_to(p->x, 16) && aligned_to(a, 16) && aligned_to(b, 16) &&
                   aligned_to(p->weight, wbytes) && (backward || aligned_to(p->bias, wbytes));
  pl.vec = vec ? full : 1;
  const int tprs[] = {8, 16, 32, 64, 128, 256, 512};
  for (int t : tprs) {
    if (p->cols > (int64_t)kLaneElements * t) continue;
    pl.tpr = t;
    break;
  }
  if (pl.tpr != 0) {
    // as many CTAs as the SMs hold, or fewer with the same number of turns each
    const int cta = cta_threads(pl.tpr), rows = cta / pl.tpr;
    const int64_t groups = (p->rows + rows - 1) / rows;
    const int64_t resident = (int64_t)sm_count() * resident_ctas(backward ? kBackwardThreads : kForwardThreads, cta);
    const int64_t turns = (groups + resident - 1) / resident;
    pl.grid = (int)(turns > 0 ? (groups + turns - 1) / turns : 0);
    pl.parts = pl.grid;
    return pl;
  }
  const int64_t resident = 2LL * sm_count();
  pl.grid = (int)(p->rows < resident ? p->rows : resident);
  if (backward) {   // row slices of the column kernel: about four CTAs an SM
    const int64_t tiles = (p->cols + 255) / 256;
    int64_t slices = (4LL * sm_count() + tiles - 1) / tiles;
    if (slices > p->rows) slices = p->rows;
    if (slices > 256) slices = 256;
    pl.parts = (int)slices;
  }
  return pl;
}

template <auto KERNEL, int MOST>
cudaError_t launch_ring(dim3 grid, int threads, int bytes, cudaStream_t st, const NormArgs& a) {
  cudaError_t e = allow_shared<KERNEL, MOST>();
  return e == cudaSuccess ? launch_pdl(KERNEL, grid, threads, (size_t)bytes, st, a) : e;
}

template <typename T, int VEC, int TPR>
cudaError_t launch_norm_tpr(const NormPlan& pl, const NormArgs& a, bool backward, cudaStream_t st) {
  constexpr int NV = kLaneElements / VEC;
  const dim3 grid((unsigned)pl.grid);
  if (!backward) {
    constexpr int ring = Ahead<T, VEC, NV, TPR, 1, kForwardDepth>::kBytes;
    return launch_ring<layer_norm_forward_kernel<T, VEC, NV, TPR>, ring>(grid, kThreads<TPR>, ring, st, a);
  }
  constexpr int ring = Ahead<T, VEC, NV, TPR, 2, kBackwardDepth<T>>::kBytes;
  // the sums of 8 warps over rows of up to 512 columns
  constexpr int most = TPR <= 32 && kThreads<TPR> / 32 * 2 * kLaneElements * TPR * 4 > ring
                           ? kThreads<TPR> / 32 * 2 * kLaneElements * TPR * 4 : ring;
  const int share = TPR <= 32 && a.partial ? kThreads<TPR> / 32 * 2 * a.cols * (int)sizeof(float) : 0;
  return launch_ring<layer_norm_backward_kernel<T, VEC, NV, TPR>, most>(grid, kThreads<TPR>, share > ring ? share : ring,
                                                                        st, a);
}

template <typename T, int VEC>
cudaError_t launch_norm_vec(const NormPlan& pl, const NormArgs& a, bool backward, cudaStream_t st) {
  switch (pl.tpr) {
    case 8: return launch_norm_tpr<T, VEC, 8>(pl, a, backward, st);
    case 16: return launch_norm_tpr<T, VEC, 16>(pl, a, backward, st);
    case 32: return launch_norm_tpr<T, VEC, 32>(pl, a, backward, st);
    case 64: return launch_norm_tpr<T, VEC, 64>(pl, a, backward, st);
    case 128: return launch_norm_tpr<T, VEC, 128>(pl, a, backward, st);
    case 256: return launch_norm_tpr<T, VEC, 256>(pl, a, backward, st);
    case 512: return launch_norm_tpr<T, VEC, 512>(pl, a, backward, st);
    default: break;
  }
  if (!backward) return launch_pdl(layer_norm_forward_loop_kernel<T, VEC>, dim3((unsigned)pl.grid), 1024, 0, st, a);
  // the column sums first: grad_x may be written over grad_y or x
  if (a.partial) {
    const dim3 grid((unsigned)((a.cols + 255) / 256), (unsigned)pl.parts);
    cudaError_t e = launch_pdl(layer_norm_columns_kernel<T>, grid, 256, 0, st, a);
    if (e != cudaSuccess) return e;
  }
  if (!a.out) return cudaSuccess;
  return launch_pdl(layer_norm_backward_loop_kernel<T, VEC>, dim3((unsigned)pl.grid), 1024, 0, st, a);
}

cudaError_t launch_norm(const NormPlan& pl, const NormArgs& a, int dtype, bool backward, cudaStream_t st) {
  const bool v = pl.vec > 1;
  if (dtype == FWD_EB_F32)
    return v ? launch_norm_vec<float, 4>(pl, a, backward, st) : launch_norm_vec<float, 1>(pl, a, backward, st);
  if (dtype == FWD_EB_F16)
    return v ? launch_norm_vec<__half, 8>(pl, a, backward, st) : launch_norm_vec<__half, 1>(pl, a, backward, st);
  return v ? launch_norm_vec<__nv_bfloat16, 8>(pl, a, backward, st)
           : launch_norm_vec<__nv_bfloat16, 1>(pl, a, backward, st);
}

NormArgs norm_args(const fwd_eb_layer_norm_params* p) {
  NormArgs a = {};
  a.x = static_cast<const char*>(p->x);
  a.x_stride = stride_of(p->x_stride, p->cols);
  a.weight = p->weight;
  a.mean = p->mean;
  a.rstd = p->rstd;
  a.rows = p->rows;
  a.cols = (int)p->cols;
  a.wtype = p->weight_dtype;
  return a;
}

size_t norm_workspace(const fwd_eb_layer_norm_params* p, const NormPlan& pl) {
  return p->grad_weight || p->grad_bias ? (size_t)pl.parts * 2 * (size_t)p->cols * sizeof(float) : 0;
}

}  // namespace
}  // namespace fwd_eb

using namespace fwd_eb;

extern "C" size_t fwd_eb_layer_norm_params_size(void) { return sizeof(fwd_eb_layer_norm_params); }

extern "C" int fwd_eb_layer_norm_forward(const fwd_eb_layer_norm_params* p, void* stream) {
  NvtxRange range("fwd_eb_layer_norm_forward");
  int rc = check_norm(p, false);
  if (rc) return rc;
  clear_error();
  if (p->rows == 0) return 0;
  const NormPlan pl = plan_norm(p, false);
  NormArgs a = norm_args(p);
  a.out = static_cast<char*>(p->y);
  a.out_stride = stride_of(p->y_stride, p->cols);
  a.bias = p->bias;
  a.eps = (float)p->eps;
  cudaError_t e = launch_norm(pl, a, p->dtype, false, static_cast<cudaStream_t>(stream));
  return e == cudaSuccess ? 0 : cuda_fail(e, "kernel launch");
}

extern "C" size_t fwd_eb_layer_norm_workspace_size(const fwd_eb_layer_norm_params* p) {
  if (check_norm(p, true) != 0) return 0;
  return norm_workspace(p, plan_norm(p, true));
}

extern "C" int fwd_eb_layer_norm_backward(const fwd_eb_layer_norm_params* p, void* stream) {
  NvtxRange range("fwd_eb_layer_norm_backward");
  int rc = check_norm(p, true);
  if (rc) return rc;
  const NormPlan pl = plan_norm(p, true);
  const size_t need = norm_workspace(p, pl);
  if (need > 0 && (!p->workspace || p->workspace_bytes < need))
    return fail(FWD_EB_EWORKSPACE, "layer norm's gradient needs %zu bytes of workspace, got %zu", need,
                p->workspace ? p->workspace_bytes : (size_t)0);
  if (need > 0 && !aligned_to(p->workspace, 256))
    return fail(FWD_EB_EALIGN, "workspace must be 256-byte aligned");
  clear_error();
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  NormArgs a = norm_args(p);
  a.gy = static_cast<const char*>(p->grad_y);
  a.gy_stride = stride_of(p->grad_y_stride, p->cols);
  a.out = static_cast<char*>(p->grad_x);
  a.out_stride = stride_of(p->grad_x_stride, p->cols);
  a.partial = need > 0 ? static_cast<float*>(p->workspace) : nullptr;
  cudaError_t e = cudaSuccess;
  if (p->rows > 0 && (a.out || a.partial)) e = launch_norm(pl, a, p->dtype, true, st);
  if (e == cudaSuccess && (p->grad_weight || p->grad_bias))
    e = launch_pdl(layer_norm_join_kernel, dim3((unsigned)((2 * p->cols + 31) / 32)), 1024, 0, st, a.partial,
                   p->rows > 0 ? pl.parts : 0, (int)p->cols, p->weight_dtype, p->grad_weight, p->grad_bias);
  return e == cudaSuccess ? 0 : cuda_fail(e, "kernel launch");
}
