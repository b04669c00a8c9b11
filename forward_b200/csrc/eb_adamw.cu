// AdamW over many tensors at once (include/fwd_eb_train.h).
//
// One launch covers up to 256 tensors: their pointers travel as kernel parameters (88 bytes each),
// so nothing is staged in device memory and the host array may go when the call returns.  A
// CTA takes one chunk of a tensor, which it finds by bisection of the chunk counts.  A
// lane handles 8 consecutive elements, so a warp's 256 are exactly one block of an 8-bit
// state: the block's largest value is one integer reduction over the warp (positive floats order
// as integers), and no value is read or written twice.
//
// States of 32 bits are bound by memory whatever the code does.  With states of 8 bits the bytes
// shrink to a third and the instructions grow, so both count there: a whole chunk's two turns are loaded
// at once, without bounds checks, and all arithmetic is on pairs (sm_100's packed fp32).
// Measured on B200, of the copy rate measured there: 128 M fp16 parameters with master copies and
// states of 32 bits 531-534 us, 1.03; 100 M in 26 tensors with states of 8 bits 197 us, 0.79 (38 instructions
// an element, 65 % of the issue slots: latency and issue slots bound it together).
#include <cfloat>
#include <climits>
#include <cmath>
#include <cuda_fp8.h>

#include "eb_train.cuh"

namespace fwd_eb {
namespace {

constexpr int kAdamThreads = 256;
constexpr int kLane = 8;                                // elements a lane handles at a time
constexpr int kTurn = kAdamThreads * kLane;              // elements a CTA handles at a time
constexpr int kMostTurns = 2;                           // turns of a chunk, at most
constexpr int kMost = 256;                              // tensors of a launch
static_assert(32 * kLane == FWD_EB_ADAMW_BLOCK, "a warp's elements are one block of an 8-bit state");

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
  float none;          // -0, which the compiler does not know
  int flush;           // a v near 2^-126 and below may count as less than it is (see hides_subnormal)
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
  int turns;           // of a chunk
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
__device__ __forceinline__ void decode(uint2 r, float (&f)[kLane]) {
  const unsigned w[2] = {r.x, r.y};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(w[i / 2] >> (16 * (i & 1))), __NV_E4M3);
    const float2 t = __half22float2(__half2(h));
    f[2 * i] = t.x;
    f[2 * i + 1] = t.y;
  }
}

// Root and reciprocal within an ulp or two, in one or a few instructions where the correctly rounded ones
// take ten: the update is lr times smaller than the parameter it is added to.  The reciprocal's argument
// sqrt(v) + eps is zero or normal: an eps above zero is normal, and the root of a subnormal v is.
__device__ __forceinline__ float quick_root(float x) {
  float y;
  asm("sqrt.approx.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float quick_reciprocal(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// What a code of 8 bits is made from is rounded as the formula is written, an operation at a time, so that the states are those of
// plain fp32, whichever path a chunk takes: an ulp more or less makes another code of a value at a code's border, which is
// a tenth of the state from then on.  Root and reciprocal by one step of Newton's iteration from the hardware's
// approximation, with the residual exact in a fused operation (Markstein, 1990); they are the correctly rounded
// ones but for a few in a million.  Of 200 M codes and 1 M scales none differs from torch's elementary operations (with fused
// sums and the approximations by themselves 167 and a third), for 197 us in place of 178 (100 M elements in 26 tensors).
__device__ __forceinline__ float reciprocal(float x) {      // normal, and so is 1 / x
  const float y = quick_reciprocal(x);
  return fmaf(fmaf(-x, y, 1.0f), y, y);
}
// Roots of two values, all with their signs turned (no negation is left to be done); NaN where a value is 0 (unless FTZ), infinite or
// NaN.  FTZ: one below 2^-126 gives some value up to its root, which eps hides.
template <bool FTZ>
__device__ __forceinline__ float2 turned_roots(float2 x) {      // of -x
  float2 s;
  if (FTZ) {
    const float2 w = fma2(x, both(-1.0f), both(FLT_MIN));     // no infinite reciprocal; far above it no change
    asm("rsqrt.approx.ftz.f32 %0, %1;" : "=f"(s.x) : "f"(w.x));
    asm("rsqrt.approx.ftz.f32 %0, %1;" : "=f"(s.y) : "f"(w.y));
  } else {
    asm("rsqrt.approx.f32 %0, %1;" : "=f"(s.x) : "f"(-x.x));
    asm("rsqrt.approx.f32 %0, %1;" : "=f"(s.y) : "f"(-x.y));
  }
  const float2 y = mul2(x, s), over = fma2(y, y, x);
  return fma2(over, mul2(s, both(0.5f)), y);
}
__device__ __forceinline__ float top_of(const float (&x)[kLane]) {      // the largest magnitude, NaN aside
  float top = 0.0f;
#pragma unroll
  for (int i = 0; i < kLane; ++i) top = fmaxf(top, fabsf(x[i]));
  return top;
}

// Codes of a block's values and its scale, the same in every lane: x ~ scale * e4m3(x / scale) with
// scale = max|x| / 448, `top` being the lane's largest.  Every lane of the warp calls it.  TURNED: x <= 0 stands for -x, and a
// value above zero gets the smallest code at least.  A scale below the normal range counts as zero: its reciprocal
// would not be finite.  A NaN gets the code of a NaN and does not touch the scale; an infinity makes
// the scale infinite, and the whole block reads back as NaN.
template <bool TURNED>
__device__ __forceinline__ uint2 encode(const float (&x)[kLane], float top, float& scale) {
  // floats that are not negative order as integers
  scale = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(top))) * (float)(1.0 / 448.0);
  if (scale < FLT_MIN) scale = 0.0f;
  float inverse = scale > 0.0f ? reciprocal(scale) : 0.0f;
  if (TURNED) inverse = -inverse;
  unsigned w[2] = {0, 0};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 t = mul2(make_float2(x[2 * i], x[2 * i + 1]), both(inverse));
    w[i / 2] |= (unsigned)__nv_cvt_float2_to_fp8x2(t, __NV_SATFINITE, __NV_E4M3) << (16 * (i & 1));
  }
  if (TURNED) {
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      w[k] &= 0x7f7f7f7fu;                                               // a zero has no sign
      if (((w[k] - 0x01010101u) & ~w[k] & 0x80808080u) == 0) continue;   // no byte of it is zero
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if (x[4 * k + i] < 0.0f && (w[k] & (0xffu << (8 * i))) == 0) w[k] |= 1u << (8 * i);
      }
    }
  }
  return make_uint2(w[0], w[1]);
}

// What a step multiplies by, once device scalars are read.
struct Rates {
  float beta1, rest1, beta2, rest2, eps, grad_scale, step_size, root_scale, keep, none;
};

// One lane's 8 elements.  BITS8: the states' roundings are those of the formula (see above); v comes out as -sqrt(v), and root_top is
// the largest of its magnitudes.
template <bool BITS8, bool FTZ>
__device__ __forceinline__ void update(const Rates& r, float (&p)[kLane], const float (&g)[kLane], float (&m)[kLane],
                                       float (&v)[kLane], float& root_top) {
  float root[kLane];
  root_top = 0.0f;
#pragma unroll
  for (int i = 0; i < kLane; i += 2) {
    const float2 gi = mul2(make_float2(g[i], g[i + 1]), both(r.grad_scale)), gg = mul2(gi, gi);
    float2 mi = make_float2(m[i], m[i + 1]), vi = make_float2(v[i], v[i + 1]), ri;
    if constexpr (BITS8) {
      // products with -0 added: a product and a sum by themselves are made one operation by the compiler
      const float2 none = both(r.none);
      mi = add2(fma2(mi, both(r.beta1), none), fma2(gi, both(r.rest1), none));
      vi = add2(fma2(vi, both(-r.beta2), none), fma2(gg, both(-r.rest2), none));
      ri = turned_roots<FTZ>(vi);
      asm("max.NaN.f32 %0, %1, %2;" : "=f"(root_top) : "f"(root_top), "f"(fabsf(ri.x)));
      asm("max.NaN.f32 %0, %1, %2;" : "=f"(root_top) : "f"(root_top), "f"(fabsf(ri.y)));
    } else {
      mi = fma2(mi, both(r.beta1), mul2(gi, both(r.rest1)));
      vi = fma2(vi, both(r.beta2), mul2(gg, both(r.rest2)));
      ri = make_float2(quick_root(vi.x), quick_root(vi.y));
    }
    m[i] = mi.x, m[i + 1] = mi.y;
    v[i] = vi.x, v[i + 1] = vi.y;
    root[i] = ri.x, root[i + 1] = ri.y;
  }
  if (BITS8) {
    if (root_top != root_top) {
#pragma unroll
      for (int i = 0; i < kLane; ++i) root[i] = root[i] == root[i] ? root[i] : v[i];      // 0, infinity and NaN are their own roots
      root_top = top_of(root);
    }
#pragma unroll
    for (int i = 0; i < kLane; ++i) v[i] = root[i];
  }
#pragma unroll
  for (int i = 0; i < kLane; i += 2) {
    const float2 den = fma2(make_float2(root[i], root[i + 1]), both(BITS8 ? -r.root_scale : r.root_scale), both(r.eps));
    const float2 upd = mul2(make_float2(m[i], m[i + 1]), make_float2(quick_reciprocal(den.x), quick_reciprocal(den.y)));
    const float2 pi = fma2(make_float2(p[i], p[i + 1]), both(r.keep), mul2(upd, both(-r.step_size)));
    p[i] = pi.x, p[i + 1] = pi.y;
  }
}
// m and v from their codes, sqrt(v)'s scale before the square: its own leaves the normal range already where v is 2e5 times 2^-126.
__device__ __forceinline__ void scaled(float (&m)[kLane], float m_scale, float (&v)[kLane], float v_scale) {
#pragma unroll
  for (int i = 0; i < kLane; i += 2) {
    const float2 a = mul2(make_float2(m[i], m[i + 1]), both(m_scale)), b = mul2(make_float2(v[i], v[i + 1]), both(v_scale));
    const float2 c = mul2(b, b);
    m[i] = a.x, m[i + 1] = a.y;
    v[i] = c.x, v[i + 1] = c.y;
  }
}

// 8 elements as they lie in memory: WIDE of 32 bits, else of 16.
template <bool WIDE>
struct Raw {
  uint4 w[WIDE ? 2 : 1];
  __device__ __forceinline__ void load(const void* p, int at) {
    const uint4* q = reinterpret_cast<const uint4*>(static_cast<const char*>(p) + at * (WIDE ? 4 : 2));
    w[0] = q[0];
    if constexpr (WIDE) w[1] = q[1];
  }
  __device__ __forceinline__ void get(int dtype, float (&f)[kLane]) const {
    if constexpr (WIDE) {
      memcpy(f, w, sizeof(f));
    } else if (dtype == FWD_EB_F16) {
      Pack<__half, kLane> r;
      r.w[0] = w[0];
      r.get(f);
    } else {
      Pack<__nv_bfloat16, kLane> r;
      r.w[0] = w[0];
      r.get(f);
    }
  }
};

// The tensors of a launch are of one kind: 0 has states of 32 bits; 1 to 4 have states of 8, and values of 16 or 32 bits
// that the step works on and gradients of 16 or 32, so that loads under way hang on no branch.
constexpr int kKinds = 5;
inline int kind_of(const fwd_eb_adamw_tensor& t) {
  if (t.state_bits == 32) return 0;
  return 1 + (t.master || t.param_dtype == FWD_EB_F32 ? 2 : 0) + (t.grad_dtype == FWD_EB_F32 ? 1 : 0);
}

template <int CAP, int KIND>
__global__ void __launch_bounds__(kAdamThreads, KIND < 2 ? 4 : 3)   // the others' loads would spill
adamw_kernel(const __grid_constant__ AdamArgs<CAP> a) {
  constexpr bool BITS8 = KIND != 0, PWIDE = BITS8 && (KIND - 1) / 2 == 1, GWIDE = BITS8 && (KIND - 1) % 2 == 1;
  pdl_enter(false);
  if (a.s.d_skip && *a.s.d_skip != 0) return;
  int lo = 0, hi = a.count;   // the last tensor whose first chunk is not behind this one
  while (hi - lo > 1) {
    const int mid = (lo + hi) / 2;
    if (a.t[mid].first <= blockIdx.x) lo = mid; else hi = mid;
  }
  AdamTensor t = a.t[lo];
  Rates r = {a.s.beta1, a.s.rest1, a.s.beta2, a.s.rest2, a.s.eps, a.s.grad_scale, a.s.step_size, a.s.root_scale, t.keep, a.s.none};
  if (a.s.d_grad_scale) r.grad_scale = *a.s.d_grad_scale;
  if (a.s.d_lr || a.s.d_step) {
    // 1 - beta^t = -expm1(t log beta): no cancellation, in fp32
    const float lr = a.s.d_lr ? *a.s.d_lr : a.s.lr;
    const float at = (float)(a.s.d_step ? *a.s.d_step : a.s.step);
    r.step_size = lr / -expm1f(at * a.s.log1);
    r.root_scale = 1.0f / sqrtf(-expm1f(at * a.s.log2));
    if (a.s.d_lr) r.keep = 1.0f - lr * t.weight_decay;
  }
  // this chunk's part of the tensor
  const int chunk = a.turns * kTurn;
  const long long begin = (long long)(blockIdx.x - t.first) * chunk;
  const int left = t.n - begin < chunk ? (int)(t.n - begin) : chunk;
  const int psize = t.ptype == FWD_EB_F32 ? 4 : 2, gsize = t.gtype == FWD_EB_F32 ? 4 : 2;
  t.param = static_cast<char*>(t.param) + begin * psize;
  t.grad = static_cast<const char*>(t.grad) + begin * gsize;
  if (t.master) t.master += begin;
  t.m = static_cast<char*>(t.m) + begin * (BITS8 ? 1 : 4);
  t.v = static_cast<char*>(t.v) + begin * (BITS8 ? 1 : 4);
  if (BITS8) {
    t.m_scale += begin / FWD_EB_ADAMW_BLOCK;
    t.v_scale += begin / FWD_EB_ADAMW_BLOCK;
  }
  const void* from = t.master ? t.master : t.param;      // what the step works on, and its type
  const int ftype = t.master ? FWD_EB_F32 : t.ptype;

  if (BITS8 && left == chunk && t.aligned && a.s.flush && a.turns == kMostTurns) {
    struct Ahead {       // a turn's loads
      Raw<PWIDE> p;
      Raw<GWIDE> g;
      uint2 m, v;
      float ms, vs;
    } ahead[2];
    auto fetch = [&](Ahead& to, int at) {
      to.p.load(from, at);
      to.g.load(t.grad, at);
      to.m = *reinterpret_cast<const uint2*>(static_cast<const char*>(t.m) + at);
      to.v = *reinterpret_cast<const uint2*>(static_cast<const char*>(t.v) + at);
      to.ms = t.m_scale[at / FWD_EB_ADAMW_BLOCK];
      to.vs = t.v_scale[at / FWD_EB_ADAMW_BLOCK];
    };
    auto turn = [&](const Ahead& now, int at) {
      float p[kLane], g[kLane], m[kLane], v[kLane], root_top;
      now.p.get(ftype, p);
      now.g.get(t.gtype, g);
      decode(now.m, m);
      decode(now.v, v);
      scaled(m, now.ms, v, now.vs);
      update<true, true>(r, p, g, m, v, root_top);
      float ms, vs;
      const uint2 cm = encode<false>(m, top_of(m), ms), cv = encode<true>(v, root_top, vs);
      if (PWIDE && t.master) store_any<kLane>(t.master, FWD_EB_F32, at, p);
      store_any<kLane>(t.param, t.ptype, at, p);
      *reinterpret_cast<uint2*>(static_cast<char*>(t.m) + at) = cm;
      *reinterpret_cast<uint2*>(static_cast<char*>(t.v) + at) = cv;
      if ((threadIdx.x & 31) == 0) {
        t.m_scale[at / FWD_EB_ADAMW_BLOCK] = ms;
        t.v_scale[at / FWD_EB_ADAMW_BLOCK] = vs;
      }
    };
    const int at = threadIdx.x * kLane;
    fetch(ahead[0], at);
    fetch(ahead[1], at + kTurn);
    turn(ahead[0], at);
    turn(ahead[1], at + kTurn);
    return;
  }

  for (int turn = 0; turn < a.turns; ++turn) {
    const int at = (turn * kAdamThreads + (int)threadIdx.x) * kLane;
    if (left <= at - (int)(threadIdx.x & 31) * kLane) return;   // the warp's first element: all its lanes go on together
    const int n = left - at < 0 ? 0 : (left - at < kLane ? left - at : kLane);
    const bool whole = n == kLane && t.aligned;
    float p[kLane], g[kLane], m[kLane], v[kLane], root_top;
    load_lane(t.grad, t.gtype, at, n, whole, g);
    load_lane(from, ftype, at, n, whole, p);
    const int block = at / FWD_EB_ADAMW_BLOCK;
    if (BITS8) {
      const uint2 cm = load_codes(t.m, at, n, whole), cv = load_codes(t.v, at, n, whole);
      decode(cm, m);
      decode(cv, v);
      scaled(m, t.m_scale[block], v, t.v_scale[block]);
    } else {
      load_lane(t.m, FWD_EB_F32, at, n, whole, m);
      load_lane(t.v, FWD_EB_F32, at, n, whole, v);
    }
    update<BITS8, false>(r, p, g, m, v, root_top);
    if (t.master) store_lane(t.master, FWD_EB_F32, at, n, whole, p);
    store_lane(t.param, t.ptype, at, n, whole, p);
    if (BITS8) {
#pragma unroll
      for (int i = 0; i < kLane; ++i) {   // what lies behind the tensor's end takes no part in its last scale
        if (i >= n) m[i] = v[i] = 0.0f;
      }
      root_top = top_of(v);
      float ms, vs;
      const uint2 cm = encode<false>(m, top_of(m), ms), cv = encode<true>(v, root_top, vs);
      store_codes(t.m, at, n, whole, cm);
      store_codes(t.v, at, n, whole, cv);
      if ((threadIdx.x & 31) == 0) {
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
  auto good = [](double x) { return x >= 0.0 && x <= FLT_MAX; };
  if (!c->d_lr && !good(c->lr)) return fail(FWD_EB_EINVAL, "lr must be finite and not negative");
  if (!good(c->eps)) return fail(FWD_EB_EINVAL, "eps must be finite and not negative");
  // the least denominator, whose reciprocal has to be a normal fp32 value
  if (c->eps != 0.0 && !(c->eps >= 0x1p-126 && c->eps <= 0x1p126))
    return fail(FWD_EB_EINVAL, "eps is 0 or between 2^-126 and 2^126 (got %g)", c->eps);
  if (!(c->beta1 >= 0.0 && c->beta1 < 1.0) || !(c->beta2 >= 0.0 && c->beta2 < 1.0))
    return fail(FWD_EB_EINVAL, "beta1 and beta2 lie in [0, 1)");
  if (!c->d_grad_scale && !(std::fabs(c->grad_scale) <= FLT_MAX)) return fail(FWD_EB_EINVAL, "grad_scale must be finite");
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

// Whether eps hides what is lost where a v near 2^-126 and below counts as less than it is.  A step then loses less than
// 2^-126 of v, steps 1 to t together less than 2^-126 (1 - beta2^t) / (1 - beta2), so sqrt(v / (1 - beta2^t)) is off by
// less than 2^-63 / sqrt(1 - beta2).  That is half an ulp of a denominator of at least eps where eps is 2^24 times as
// large, and 2^25 leaves room for what v loses when it is decoded: 1.6e-11 at beta2 = 0.95, 1.2e-10 at 0.999.
bool hides_subnormal(double eps, double beta2) { return eps * std::sqrt(1.0 - beta2) >= 0x1p-38; }

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
  s.none = -0.0f;
  s.flush = hides_subnormal(c->eps, c->beta2);
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

// Fills one launch with the tensors of one kind from *next on, moves *next behind them, launches.
template <int CAP, int KIND>
cudaError_t launch_some(const fwd_eb_adamw_tensor* ts, int count, int* next, const AdamScalars& s, double lr,
                        cudaStream_t st) {
  AdamArgs<CAP> a = {};
  a.s = s;
  int end = *next;
  long long total = 0;     // turns, at one turn a chunk
  for (int found = 0; end < count && found < CAP; ++end) {
    const fwd_eb_adamw_tensor& t = ts[end];
    if (t.n == 0 || kind_of(t) != KIND) continue;
    total += (t.n + kTurn - 1) / kTurn;
    ++found;
  }
  // 8-bit chunks of two turns, whose loads are under way together, where a few waves of CTAs are left even so: 100 M
  // elements 174 us against 293 a turn at a time (202 and 220 with chunks of 4 and 8 turns; before the states' roundings
  // were the formula's, 197 us now)
  const long long wave = 3LL * sm_count();
  a.turns = KIND != 0 && total / kMostTurns >= 4 * wave ? kMostTurns : 1;
  long long chunks = 0;
  for (; *next < end; ++*next) {
    const fwd_eb_adamw_tensor& t = ts[*next];
    if (t.n == 0 || kind_of(t) != KIND) continue;
    const long long c = (t.n + (long long)a.turns * kTurn - 1) / ((long long)a.turns * kTurn);
    if (chunks + c > INT_MAX) break;     // the rest in a launch of its own
    a.t[a.count++] = tensor_of(t, (unsigned)chunks, lr);
    chunks += c;
  }
  if (chunks == 0) return cudaSuccess;
  return launch_pdl(adamw_kernel<CAP, KIND>, dim3((unsigned)chunks), kAdamThreads, 0, st, a);
}

template <int KIND>
cudaError_t launch_all(const fwd_eb_adamw_tensor* ts, int count, const AdamScalars& s, double lr, cudaStream_t st) {
  for (int next = 0; next < count;) {
    const int left = count - next;
    cudaError_t e = left <= 8    ? launch_some<8, KIND>(ts, count, &next, s, lr, st)
                    : left <= 64 ? launch_some<64, KIND>(ts, count, &next, s, lr, st)
                                 : launch_some<kMost, KIND>(ts, count, &next, s, lr, st);
    if (e != cudaSuccess) return e;
  }
  return cudaSuccess;
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
  bool any[kKinds] = {};
  for (int i = 0; i < count; ++i) any[kind_of(tensors[i])] = true;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  cudaError_t e = cudaSuccess;
  if (any[0]) e = launch_all<0>(tensors, count, s, cfg->lr, st);
  if (any[1] && e == cudaSuccess) e = launch_all<1>(tensors, count, s, cfg->lr, st);
  if (any[2] && e == cudaSuccess) e = launch_all<2>(tensors, count, s, cfg->lr, st);
  if (any[3] && e == cudaSuccess) e = launch_all<3>(tensors, count, s, cfg->lr, st);
  if (any[4] && e == cudaSuccess) e = launch_all<4>(tensors, count, s, cfg->lr, st);
  return e == cudaSuccess ? 0 : cuda_fail(e, "kernel launch");
}
