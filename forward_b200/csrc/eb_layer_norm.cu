// Layer norm of pooled rows and its gradients (include/fwd_eb_train.h).
//
// Both directions are bound by memory: a row is read once into registers, its statistics are
// taken from there (mean first, then the squared distances from it: no cancellation), and the
// result is written once.  TPR threads share a row, NV vectors of VEC elements each; the backward
// pass walks rows with a fixed grid so that a thread keeps its columns' share of grad_weight and
// grad_bias in registers, and a second kernel adds the CTAs' shares in CTA order.
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

// Sum over the TPR threads of a row, the same value in each; `red` is TPR / 32 floats, used by
// one sum at a time (a second call may follow at once: it synchronises before it writes).
template <int TPR>
__device__ __forceinline__ float row_sum(float v, float* red) {
  constexpr int kWidth = TPR < 32 ? TPR : 32;
#pragma unroll
  for (int o = kWidth / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  if constexpr (TPR > 32) {
    constexpr int kWarps = TPR / 32;
    __syncthreads();
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
    __syncthreads();
    v = (threadIdx.x & 31) < kWarps ? red[threadIdx.x & 31] : 0.0f;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  }
  return v;
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

template <typename T, int VEC, int NV, int TPR>
__global__ void __launch_bounds__(kThreads<TPR>)
layer_norm_forward_kernel(const NormArgs a) {
  pdl_enter();
  constexpr int kRows = kThreads<TPR> / TPR;
  __shared__ float red[32];
  const int lane = threadIdx.x % TPR;
  const long long step = (long long)gridDim.x * kRows;
  // every thread of the CTA makes the same number of turns
  for (long long base = (long long)blockIdx.x * kRows; base < a.rows; base += step) {
    const long long row = base + threadIdx.x / TPR;
    const bool live = row < a.rows;
    const T* x = reinterpret_cast<const T*>(a.x) + row * a.x_stride;
    Pack<T, VEC> raw[NV];
    float sum = 0.0f;
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const int col = (k * TPR + lane) * VEC;
      raw[k].zero();
      if (live && col < a.cols) raw[k].load(x + col);
    }
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      float f[VEC];
      raw[k].get(f);
#pragma unroll
      for (int i = 0; i < VEC; ++i) sum += f[i];
    }
    const float mean = row_sum<TPR>(sum, red) / (float)a.cols;
    float square = 0.0f;
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const int col = (k * TPR + lane) * VEC;
      float f[VEC];
      raw[k].get(f);
      if (col < a.cols) {
#pragma unroll
        for (int i = 0; i < VEC; ++i) square = fmaf(f[i] - mean, f[i] - mean, square);
      }
    }
    const float rstd = 1.0f / sqrtf(row_sum<TPR>(square, red) / (float)a.cols + a.eps);
    if (!live) continue;
    if (lane == 0) {
      if (a.mean) a.mean[row] = mean;
      if (a.rstd) a.rstd[row] = rstd;
    }
    T* y = reinterpret_cast<T*>(a.out) + row * a.out_stride;
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const int col = (k * TPR + lane) * VEC;
      if (col >= a.cols) continue;
      float f[VEC], w[VEC], b[VEC];
      load_weight<VEC>(a.weight, a.wtype, col, 1.0f, w);
      load_weight<VEC>(a.bias, a.wtype, col, 0.0f, b);
      raw[k].get(f);
#pragma unroll
      for (int i = 0; i < VEC; ++i) f[i] = fmaf((f[i] - mean) * rstd, w[i], b[i]);
      raw[k].set(f);
      raw[k].store(y + col);
    }
  }
}

// Rows of any width: three passes over the row, the last two mostly from L2.
template <typename T, int VEC>
__global__ void __launch_bounds__(1024)
layer_norm_forward_loop_kernel(const NormArgs a) {
  pdl_enter();
  __shared__ float red[32];
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
    const float mean = row_sum<1024>(sum, red) / (float)a.cols;
    for (int col = threadIdx.x * VEC; col < a.cols; col += step) {
      Pack<T, VEC> r;
      float f[VEC];
      r.load(x + col);
      r.get(f);
#pragma unroll
      for (int i = 0; i < VEC; ++i) square = fmaf(f[i] - mean, f[i] - mean, square);
    }
    const float rstd = 1.0f / sqrtf(row_sum<1024>(square, red) / (float)a.cols + a.eps);
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
    // the next row's first row_sum synchronises before it writes `red`
  }
}

// grad_x of the rows this CTA walks, and its share of grad_weight and grad_bias.
template <typename T, int VEC, int NV, int TPR>
__global__ void __launch_bounds__(kThreads<TPR>)
layer_norm_backward_kernel(const NormArgs a) {
  pdl_enter();
  constexpr int kRows = kThreads<TPR> / TPR;
  __shared__ float red[32];
  extern __shared__ float share[];   // kRows > 1: [2][cols] sums of the CTA's row groups
  const int lane = threadIdx.x % TPR;
  const int group = threadIdx.x / TPR;
  float dw[NV][VEC], db[NV][VEC];
#pragma unroll
  for (int k = 0; k < NV; ++k) {
#pragma unroll
    for (int i = 0; i < VEC; ++i) dw[k][i] = db[k][i] = 0.0f;
  }
  const long long step = (long long)gridDim.x * kRows;
  for (long long base = (long long)blockIdx.x * kRows; base < a.rows; base += step) {
    const long long row = base + group;
    const bool live = row < a.rows;
    const T* x = reinterpret_cast<const T*>(a.x) + row * a.x_stride;
    const T* gy = reinterpret_cast<const T*>(a.gy) + row * a.gy_stride;
    Pack<T, VEC> rx[NV], rg[NV];
    const float mean = live ? a.mean[row] : 0.0f;
    const float rstd = live ? a.rstd[row] : 0.0f;
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const int col = (k * TPR + lane) * VEC;
      rx[k].zero();
      rg[k].zero();
      if (live && col < a.cols) {
        rx[k].load(x + col);
        rg[k].load(gy + col);
      }
    }
    float s1 = 0.0f, s2 = 0.0f;
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const int col = (k * TPR + lane) * VEC;
      if (!live || col >= a.cols) continue;
      float fx[VEC], fg[VEC], w[VEC];
      load_weight<VEC>(a.weight, a.wtype, col, 1.0f, w);
      rx[k].get(fx);
      rg[k].get(fg);
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        const float h = (fx[i] - mean) * rstd;
        const float g = fg[i] * w[i];
        s1 += g;
        s2 = fmaf(g, h, s2);
        dw[k][i] = fmaf(fg[i], h, dw[k][i]);
        db[k][i] += fg[i];
      }
    }
    if (a.out) {
      s1 = row_sum<TPR>(s1, red) / (float)a.cols;
      s2 = row_sum<TPR>(s2, red) / (float)a.cols;
      T* gx = reinterpret_cast<T*>(a.out) + row * a.out_stride;
#pragma unroll
      for (int k = 0; k < NV; ++k) {
        const int col = (k * TPR + lane) * VEC;
        if (!live || col >= a.cols) continue;
        float fx[VEC], fg[VEC], w[VEC];
        load_weight<VEC>(a.weight, a.wtype, col, 1.0f, w);
        rx[k].get(fx);
        rg[k].get(fg);
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
          const float h = (fx[i] - mean) * rstd;
          fg[i] = rstd * (fmaf(fg[i], w[i], -s1) - h * s2);
        }
        rg[k].set(fg);
        rg[k].store(gx + col);
      }
    }
  }
  if (!a.partial) return;
  float* mine = a.partial + (long long)blockIdx.x * 2 * a.cols;
  if constexpr (kRows > 1) {
    // the CTA's row groups take turns, so the order of the additions is fixed
    for (int i = threadIdx.x; i < 2 * a.cols; i += blockDim.x) share[i] = 0.0f;
    for (int g = 0; g < kRows; ++g) {
      __syncthreads();
      if (group != g) continue;
#pragma unroll
      for (int k = 0; k < NV; ++k) {
        const int col = (k * TPR + lane) * VEC;
        if (col >= a.cols) continue;
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
          share[col + i] += dw[k][i];
          share[a.cols + col + i] += db[k][i];
        }
      }
    }
    __syncthreads();
    for (int i = threadIdx.x; i < 2 * a.cols; i += blockDim.x) mine[i] = share[i];
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
  pdl_enter();
  __shared__ float red[32];
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
    s1 = row_sum<1024>(s1, red) / (float)a.cols;
    s2 = row_sum<1024>(s2, red) / (float)a.cols;
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
  pdl_enter();
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
  pdl_enter();
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

// How a call runs: vector width, threads a row and vectors a thread; tpr = 0 is the loop kernel.
struct NormPlan {
  int vec, nv, tpr;
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
  const int64_t n = p->cols / pl.vec;   // vectors a row
  const int most = backward ? 512 : 1024;
  const int tprs[] = {8, 32, 128, 256, 512, 1024};
  for (int t : tprs) {
    if (t > most || n > 4LL * t) continue;
    pl.tpr = t;
    pl.nv = n <= t ? 1 : (n <= 2 * t ? 2 : 4);
    break;
  }
  const int64_t groups = pl.tpr == 0 ? p->rows : (p->rows + cta_threads(pl.tpr) / pl.tpr - 1) / (cta_threads(pl.tpr) / pl.tpr);
  if (!backward) {
    pl.grid = (int)(groups < INT_MAX ? groups : INT_MAX);
    return pl;
  }
  const int64_t resident = (int64_t)sm_count() * (pl.tpr == 0 || pl.tpr > 256 ? 2 : 4);
  pl.grid = (int)(groups < resident ? groups : resident);
  pl.parts = pl.grid;
  if (pl.tpr == 0) {   // row slices of the column kernel: about four CTAs an SM
    const int64_t tiles = (p->cols + 255) / 256;
    int64_t slices = (4LL * sm_count() + tiles - 1) / tiles;
    if (slices > p->rows) slices = p->rows;
    if (slices > 256) slices = 256;
    pl.parts = (int)(slices < 1 ? 1 : slices);
    if (p->rows == 0) pl.parts = 0;
  }
  return pl;
}

template <typename T, int VEC, int NV>
cudaError_t launch_norm_nv(const NormPlan& pl, const NormArgs& a, bool backward, cudaStream_t st) {
  const dim3 grid((unsigned)pl.grid);
  const size_t share = backward && pl.tpr <= 32 && a.partial ? (size_t)2 * a.cols * sizeof(float) : 0;
#define FWD_EB_NORM(TPR)                                                                                     \
  case TPR:                                                                                                  \
    return backward ? launch_pdl(layer_norm_backward_kernel<T, VEC, NV, TPR>, grid, kThreads<TPR>, share, \
                                 st, a)                                                                      \
                    : launch_pdl(layer_norm_forward_kernel<T, VEC, NV, TPR>, grid, kThreads<TPR>, 0, st, a)
  switch (pl.tpr) {
    FWD_EB_NORM(8);
    FWD_EB_NORM(32);
    FWD_EB_NORM(128);
    FWD_EB_NORM(256);
    FWD_EB_NORM(512);
    default:
      return launch_pdl(layer_norm_forward_kernel<T, VEC, NV, 1024>, grid, 1024, 0, st, a);
  }
#undef FWD_EB_NORM
}

template <typename T, int VEC>
cudaError_t launch_norm_vec(const NormPlan& pl, const NormArgs& a, bool backward, cudaStream_t st) {
  if (pl.tpr == 0) {
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
  switch (pl.nv) {
    case 1: return launch_norm_nv<T, VEC, 1>(pl, a, backward, st);
    case 2: return launch_norm_nv<T, VEC, 2>(pl, a, backward, st);
    default: return launch_norm_nv<T, VEC, 4>(pl, a, backward, st);
  }
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
