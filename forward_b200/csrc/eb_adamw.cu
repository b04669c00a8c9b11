// AdamW over many tensors at once (include/fwd_eb_train.h).
//
// One launch covers up to 256 tensors: their pointers travel as kernel parameters (80 bytes each),
// so nothing is staged in device memory and the host array may go when the call returns.  A
// CTA takes one chunk of a tensor, which it finds by bisection of the chunk counts.  A
// lane handles 8 consecutive elements, so a warp's 256 are exactly one block of an 8-bit
// state: the block's largest value is one integer reduction over the warp (positive floats order
// as integers), and no value is read or written twice.
#include <cfloat>
#include <climits>
#include <cmath>
#include <cuda_fp8.h>

#include "eb_train.cuh"

namespace fwd_eb {
namespace {

constexpr int kAdamThreads = 256;
constexpr int kLane = 8;                                // elements a lane handles at a time
constexpr int kTurns = 2;                               // times a CTA goes over its chunk
constexpr int kChunk = kAdamThreads * kLane * kTurns;   // elements of a chunk
constexpr int kMost = 256;                              // tensors of a launch
static_assert(32 * kLane == FWD_EB_ADAMW_BLOCK, "a warp's elements are one block of an 8-bit state");
static_assert(kChunk % FWD_EB_ADAMW_BLOCK == 0, "blocks do not cross chunks");

struct AdamTensor {
  void* param;
  const void* grad;
  float* master;
  void* m;
  void* v;
  float* m_scale;      // null: states of 32 bits
  float* v_scale;
  long long n;
  unsigned first;      // the tensor's first chunk within the launch
  float weight_decay;
  float keep;          // 1 - lr * weight_decay
  short ptype, gtype;
  int aligned;         // vector accesses are possible
};

struct AdamScalars {
  float beta1, rest1, beta2, rest2, eps, grad_scale;
  float lr;            // used where d_lr or d_step make the two below unknown on the host
  float step_size;     // lr / (1 - beta1^t)
  float root_scale;    // 1 / sqrt(1 - beta2^t)
  float log1, log2;    // log(beta), for a step that lies on the device
  long long step;
  const float* d_lr;
  const float* d_grad_scale;
  const long long* d_step;
  const int* d_skip;
};

template <int CAP>
struct AdamArgs {
  AdamScalars s;
  int count;
  AdamTensor t[CAP];
};

template <typename T>
__device__ __forceinline__ void load_some(const T* p, int n, float (&f)[kLane]) {
#pragma unroll
  for (int i = 0; i < kLane; ++i) f[i] = i < n ? to_float(p[i]) : 0.0f;
}
__device__ __forceinline__ void load_lane(const void* p, int dtype, long long at, int n, bool whole, float (&f)[kLane]) {
  if (whole) {
    load_any<kLane>(p, dtype, at, f);
  } else if (dtype == FWD_EB_F32) {
    load_some(static_cast<const float*>(p) + at, n, f);
  } else if (dtype == FWD_EB_F16) {
    load_some(static_cast<const __half*>(p) + at, n, f);
  } else {
    load_some(static_cast<const __nv_bfloat16*>(p) + at, n, f);
  }
}
template <typename T>
__device__ __forceinline__ void store_some(T* p, int n, const float (&f)[kLane]) {
#pragma unroll
  for (int i = 0; i < kLane; ++i) {
    if (i < n) p[i] = from_float<T>(f[i]);
  }
}
__device__ __forceinline__ void store_lane(void* p, int dtype, long long at, int n, bool whole, const float (&f)[kLane]) {
  if (whole) {
    store_any<kLane>(p, dtype, at, f);
  } else if (dtype == FWD_EB_F32) {
    store_some(static_cast<float*>(p) + at, n, f);
  } else if (dtype == FWD_EB_F16) {
    store_some(static_cast<__half*>(p) + at, n, f);
  } else {
    store_some(static_cast<__nv_bfloat16*>(p) + at, n, f);
  }
}

// 8 e4m3 codes.
__device__ __forceinline__ uint2 load_codes(const void* p, long long at, int n, bool whole) {
  const unsigned char* q = static_cast<const unsigned char*>(p) + at;
  if (whole) return *reinterpret_cast<const uint2*>(q);
  unsigned char c[kLane];
#pragma unroll
  for (int i = 0; i < kLane; ++i) c[i] = i < n ? q[i] : 0;
  uint2 r;
  memcpy(&r, c, sizeof(r));
  return r;
}
__device__ __forceinline__ void store_codes(void* p, long long at, int n, bool whole, uint2 r) {
  unsigned char* q = static_cast<unsigned char*>(p) + at;
  if (whole) {
    *reinterpret_cast<uint2*>(q) = r;
    return;
  }
  unsigned char c[kLane];
  memcpy(c, &r, sizeof(r));
#pragma unroll
  for (int i = 0; i < kLane; ++i) {
    if (i < n) q[i] = c[i];
  }
}
__device__ __forceinline__ void decode(uint2 r, float scale, float (&f)[kLane]) {
  const unsigned w[2] = {r.x, r.y};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(w[i / 2] >> (16 * (i & 1))), __NV_E4M3);
    const float2 t = __half22float2(__half2(h));
    f[2 * i] = t.x * scale;
    f[2 * i + 1] = t.y * scale;
  }
}

// Codes of a block's values and its scale, the same in every lane: x ~ scale * e4m3(x / scale) with
// scale = max|x| / 448.  Every lane of the warp calls it; `least` is the smallest code that a
// value above zero may get.  A scale below the normal range counts as zero: its reciprocal
// would not be finite.  A block that holds a NaN or an infinity gets a scale that is neither
// finite nor zero, so the whole block reads back as NaN.
__device__ __forceinline__ uint2 encode(const float (&x)[kLane], float least, float& scale) {
  unsigned top = 0;
#pragma unroll
  for (int i = 0; i < kLane; ++i) {
    const unsigned b = __float_as_uint(x[i]) & 0x7fffffffu;
    top = b > top ? b : top;
  }
  scale = __uint_as_float(__reduce_max_sync(0xffffffffu, top)) * (float)(1.0 / 448.0);
  if (scale < FLT_MIN) scale = 0.0f;
  const float inverse = scale > 0.0f ? __frcp_rn(scale) : 0.0f;
  unsigned w[2] = {0, 0};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float2 t = make_float2(x[2 * i] * inverse, x[2 * i + 1] * inverse);
    if (least > 0.0f) {
      if (x[2 * i] > 0.0f && t.x < least) t.x = least;
      if (x[2 * i + 1] > 0.0f && t.y < least) t.y = least;
    }
    w[i / 2] |= (unsigned)__nv_cvt_float2_to_fp8x2(t, __NV_SATFINITE, __NV_E4M3) << (16 * (i & 1));
  }
  return make_uint2(w[0], w[1]);
}

template <int CAP>
__global__ void __launch_bounds__(kAdamThreads)
adamw_kernel(const __grid_constant__ AdamArgs<CAP> a) {
  pdl_enter();
  if (a.s.d_skip && *a.s.d_skip != 0) return;
  int lo = 0, hi = a.count;   // the last tensor whose first chunk is not behind this one
  while (hi - lo > 1) {
    const int mid = (lo + hi) / 2;
    if (a.t[mid].first <= blockIdx.x) lo = mid; else hi = mid;
  }
  const AdamTensor& t = a.t[lo];
  const long long chunk = (long long)(blockIdx.x - t.first) * kChunk;

  float lr = a.s.lr, step_size = a.s.step_size, root_scale = a.s.root_scale, grad_scale = a.s.grad_scale;
  if (a.s.d_lr) lr = *a.s.d_lr;
  if (a.s.d_grad_scale) grad_scale = *a.s.d_grad_scale;
  if (a.s.d_lr || a.s.d_step) {
    // 1 - beta^t = -expm1(t log beta): no cancellation, in fp32
    const float at = (float)(a.s.d_step ? *a.s.d_step : a.s.step);
    step_size = lr / -expm1f(at * a.s.log1);
    root_scale = 1.0f / sqrtf(-expm1f(at * a.s.log2));
  }
  const float keep = a.s.d_lr ? 1.0f - lr * t.weight_decay : t.keep;
  const bool bits8 = t.m_scale != nullptr;

#pragma unroll
  for (int turn = 0; turn < kTurns; ++turn) {
    const long long at = chunk + (turn * kAdamThreads + (int)threadIdx.x) * kLane;
    if (t.n <= at - (int)(threadIdx.x & 31) * kLane) continue;   // the warp's first element: all its lanes go on together
    const long long left = t.n - at;
    const int n = left < 0 ? 0 : (left < kLane ? (int)left : kLane);
    const bool whole = n == kLane && t.aligned;
    float p[kLane], g[kLane], m[kLane], v[kLane];
    load_lane(t.grad, t.gtype, at, n, whole, g);
    if (t.master) {
      load_lane(t.master, FWD_EB_F32, at, n, whole, p);
    } else {
      load_lane(t.param, t.ptype, at, n, whole, p);
    }
    const long long block = at / FWD_EB_ADAMW_BLOCK;
    const bool has_block = block * FWD_EB_ADAMW_BLOCK < t.n;
    if (bits8) {
      const uint2 cm = load_codes(t.m, at, n, whole), cv = load_codes(t.v, at, n, whole);
      decode(cm, has_block ? t.m_scale[block] : 0.0f, m);
      decode(cv, has_block ? t.v_scale[block] : 0.0f, v);
#pragma unroll
      for (int i = 0; i < kLane; ++i) v[i] = __fmul_rn(v[i], v[i]);
    } else {
      load_lane(t.m, FWD_EB_F32, at, n, whole, m);
      load_lane(t.v, FWD_EB_F32, at, n, whole, v);
    }
    float root[kLane];
#pragma unroll
    for (int i = 0; i < kLane; ++i) {
      // each product and sum rounds by itself: an 8-bit code must not depend on how they are fused
      const float gi = __fmul_rn(g[i], grad_scale);
      m[i] = __fadd_rn(__fmul_rn(m[i], a.s.beta1), __fmul_rn(gi, a.s.rest1));
      v[i] = __fadd_rn(__fmul_rn(v[i], a.s.beta2), __fmul_rn(__fmul_rn(gi, gi), a.s.rest2));
      root[i] = __fsqrt_rn(v[i]);
      p[i] = p[i] * keep - step_size * (m[i] / fmaf(root[i], root_scale, a.s.eps));
    }
    if (t.master) store_lane(t.master, FWD_EB_F32, at, n, whole, p);
    store_lane(t.param, t.ptype, at, n, whole, p);
    if (bits8) {
#pragma unroll
      for (int i = 0; i < kLane; ++i) {   // what lies behind the tensor's end takes no part in its last scale
        if (i >= n) m[i] = root[i] = 0.0f;
      }
      float ms, vs;
      const uint2 cm = encode(m, 0.0f, ms), cv = encode(root, 0.001953125f, vs);   // 2^-9: the smallest code
      store_codes(t.m, at, n, whole, cm);
      store_codes(t.v, at, n, whole, cv);
      if ((threadIdx.x & 31) == 0 && has_block) {
        t.m_scale[block] = ms;
        t.v_scale[block] = vs;
      }
    } else {
      store_lane(t.m, FWD_EB_F32, at, n, whole, m);
      store_lane(t.v, FWD_EB_F32, at, n, whole, v);
    }
  }
}

bool known(int dtype) { return dtype == FWD_EB_F32 || dtype == FWD_EB_F16 || dtype == FWD_EB_BF16; }

int check_adamw(const fwd_eb_adamw_tensor* ts, int32_t count, const fwd_eb_adamw_config* c) {
  if (count < 0 || (count > 0 && !ts)) return fail(FWD_EB_EINVAL, "bad tensor list");
  if (!c) return fail(FWD_EB_EINVAL, "config is null");
  auto good = [](double x) { return std::isfinite(x) && x >= 0.0; };
  if (!c->d_lr && !good(c->lr)) return fail(FWD_EB_EINVAL, "lr must be finite and not negative");
  if (!good(c->eps)) return fail(FWD_EB_EINVAL, "eps must be finite and not negative");
  if (!(c->beta1 >= 0.0 && c->beta1 < 1.0) || !(c->beta2 >= 0.0 && c->beta2 < 1.0))
    return fail(FWD_EB_EINVAL, "beta1 and beta2 lie in [0, 1)");
  if (!c->d_grad_scale && !std::isfinite(c->grad_scale)) return fail(FWD_EB_EINVAL, "grad_scale must be finite");
  if (!c->d_step && c->step < 1) return fail(FWD_EB_EINVAL, "step counts from 1 (got %lld)", (long long)c->step);
  if (!aligned_to(c->d_lr, 4) || !aligned_to(c->d_grad_scale, 4) || !aligned_to(c->d_step, 8) || !aligned_to(c->d_skip, 4))
    return fail(FWD_EB_EALIGN, "a device scalar is not aligned to its type");
  for (int i = 0; i < count; ++i) {
    const fwd_eb_adamw_tensor& t = ts[i];
    if (t.n < 0) return fail(FWD_EB_EINVAL, "tensors[%d]: n is negative", i);
    if (t.n > (1LL << 40)) return fail(FWD_EB_ETOOBIG, "tensors[%d]: n is limited to 2^40", i);
    if (!known(t.param_dtype)) return fail(FWD_EB_EINVAL, "tensors[%d]: unknown param_dtype %d", i, t.param_dtype);
    if (!known(t.grad_dtype)) return fail(FWD_EB_EINVAL, "tensors[%d]: unknown grad_dtype %d", i, t.grad_dtype);
    if (t.state_bits != 32 && t.state_bits != 8)
      return fail(FWD_EB_EINVAL, "tensors[%d]: state_bits is 32 or 8 (got %d)", i, t.state_bits);
    if (!std::isfinite(t.weight_decay)) return fail(FWD_EB_EINVAL, "tensors[%d]: weight_decay must be finite", i);
    if (t.state_bits == 32 && (t.exp_avg_scale || t.exp_avg_sq_scale))
      return fail(FWD_EB_EINVAL, "tensors[%d]: states of 32 bits have no scales", i);
    if (t.n == 0) continue;
    if (!t.param || !t.grad || !t.exp_avg || !t.exp_avg_sq) return fail(FWD_EB_EINVAL, "tensors[%d]: a pointer is null", i);
    if (t.state_bits == 8 && (!t.exp_avg_scale || !t.exp_avg_sq_scale))
      return fail(FWD_EB_EINVAL, "tensors[%d]: states of 8 bits need both scale arrays", i);
    const size_t se = t.state_bits == 32 ? 4 : 1;
    if (!aligned_to(t.param, dtype_size(t.param_dtype)) || !aligned_to(t.grad, dtype_size(t.grad_dtype)) ||
        !aligned_to(t.master, 4) || !aligned_to(t.exp_avg, se) || !aligned_to(t.exp_avg_sq, se) ||
        !aligned_to(t.exp_avg_scale, 4) || !aligned_to(t.exp_avg_sq_scale, 4))
      return fail(FWD_EB_EALIGN, "tensors[%d]: a pointer is not aligned to its type", i);
  }
  return 0;
}

AdamScalars scalars_of(const fwd_eb_adamw_config* c) {
  AdamScalars s = {};
  s.beta1 = (float)c->beta1;
  s.rest1 = (float)(1.0 - c->beta1);
  s.beta2 = (float)c->beta2;
  s.rest2 = (float)(1.0 - c->beta2);
  s.eps = (float)c->eps;
  s.grad_scale = (float)c->grad_scale;
  s.lr = (float)c->lr;
  const double t = (double)c->step;
  s.step_size = (float)(c->lr / -std::expm1(t * std::log(c->beta1)));   // log 0 = -inf: the correction is 1
  s.root_scale = (float)(1.0 / std::sqrt(-std::expm1(t * std::log(c->beta2))));
  s.log1 = (float)std::log(c->beta1);
  s.log2 = (float)std::log(c->beta2);
  s.step = c->step;
  s.d_lr = c->d_lr;
  s.d_grad_scale = c->d_grad_scale;
  s.d_step = reinterpret_cast<const long long*>(c->d_step);
  s.d_skip = reinterpret_cast<const int*>(c->d_skip);
  return s;
}

AdamTensor tensor_of(const fwd_eb_adamw_tensor& t, unsigned first, double lr) {
  AdamTensor r = {};
  r.param = t.param;
  r.grad = t.grad;
  r.master = t.master;
  r.m = t.exp_avg;
  r.v = t.exp_avg_sq;
  r.m_scale = t.exp_avg_scale;
  r.v_scale = t.exp_avg_sq_scale;
  r.n = t.n;
  r.first = first;
  r.weight_decay = t.weight_decay;
  r.keep = (float)(1.0 - lr * (double)t.weight_decay);
  r.ptype = (short)t.param_dtype;
  r.gtype = (short)t.grad_dtype;
  const size_t sa = t.state_bits == 32 ? 16 : kLane;
  r.aligned = aligned_to(t.param, 16) && aligned_to(t.grad, 16) && aligned_to(t.master, 16) &&
              aligned_to(t.exp_avg, sa) && aligned_to(t.exp_avg_sq, sa);
  return r;
}

// Fills one launch from the tensors at *next on, moves *next behind them, launches.
template <int CAP>
cudaError_t launch_some(const fwd_eb_adamw_tensor* ts, int count, int* next, const AdamScalars& s, double lr,
                        cudaStream_t st) {
  AdamArgs<CAP> a = {};
  a.s = s;
  long long chunks = 0;
  while (*next < count && a.count < CAP) {
    const fwd_eb_adamw_tensor& t = ts[*next];
    const long long c = (t.n + kChunk - 1) / kChunk;
    if (chunks + c > INT_MAX) break;
    if (c > 0) a.t[a.count++] = tensor_of(t, (unsigned)chunks, lr);
    chunks += c;
    ++*next;
  }
  if (chunks == 0) return cudaSuccess;
  return launch_pdl(adamw_kernel<CAP>, dim3((unsigned)chunks), kAdamThreads, 0, st, a);
}

}  // namespace
}  // namespace fwd_eb

using namespace fwd_eb;

extern "C" size_t fwd_eb_adamw_tensor_size(void) { return sizeof(fwd_eb_adamw_tensor); }
extern "C" size_t fwd_eb_adamw_config_size(void) { return sizeof(fwd_eb_adamw_config); }

extern "C" int fwd_eb_adamw_step(const fwd_eb_adamw_tensor* tensors, int32_t count, const fwd_eb_adamw_config* cfg,
                                 void* stream) {
  NvtxRange range("fwd_eb_adamw_step");
  int rc = check_adamw(tensors, count, cfg);
  if (rc) return rc;
  clear_error();
  const AdamScalars s = scalars_of(cfg);
  for (int next = 0; next < count;) {
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    const int left = count - next;
    cudaError_t e = left <= 8    ? launch_some<8>(tensors, count, &next, s, cfg->lr, st)
                    : left <= 64 ? launch_some<64>(tensors, count, &next, s, cfg->lr, st)
                                 : launch_some<kMost>(tensors, count, &next, s, cfg->lr, st);
    if (e != cudaSuccess) return cuda_fail(e, "kernel launch");
  }
  return 0;
}
