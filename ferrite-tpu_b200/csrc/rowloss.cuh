// Row losses over logits [rows, vocab]: what the post-training losses share.
//
// With z = x / tau, every loss here is a function of one row's softmax:
//   lse = log sum_i exp(z_i),  logp_t = z_t - lse,  H = -sum_i p_i log p_i,
// and its gradient is  dx_i = e_i (A + B y_i)  plus a few single-entry terms (the
// target's, or the teacher's listed tokens), where in units of log 2
//   k = log2(e) / tau,  y_i = k (x_i - m),  e_i = 2^y_i,  s = sum e_i,  u = sum e_i y_i,
//   logp_i = ln2 (y_i - log2 s),   H = ln2 (log2 s - u / s),   p_i = e_i / s.
// A row's state is (m, s, u): it is built in one pass (running maximum, rescaled sums)
// and merged pairwise.  All of it is f32; only the gradient is rounded, once, on store.
//
// y_i is one fma(x_i, k, -c) with c = k m rounded: the same c enters every term of s
// and of logp, so its rounding cancels.  Where k m leaves f32 (a row whose maximum is
// the type's lowest value, or infinite) y_i is k (x_i - m) instead.  A logit of -inf
// has e_i = 0 and contributes nothing; NaN and +inf make the row's results NaN.
#pragma once

#include <cmath>
#include <type_traits>

#include "common.cuh"

namespace ferrite {
namespace rowloss {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
constexpr float kBig = 1e38f;  // |k m| above this: the fma form could overflow

// (m, s, u): the maximum, sum of e and sum of e * y of the elements seen so far.
struct State {
  float m, s, u;
};
__device__ __forceinline__ State empty_state() { return State{-INFINITY, 0.f, 0.f}; }

// Rows whose results are asked for.
struct RowIn {
  const void* logits;
  int64_t rows, vocab, ld;
  float k;        // log2(e) / tau
  float inv_tau;  // 1 / tau
};
struct RowOut {
  void* dlogits;  // null: no gradient
  int64_t ld;
  const float* dloss;  // upstream gradient (device scalar); null: 1
  float scale;
};
struct Targets {
  const void* t;
  int is64;
  int64_t ignore;
  __device__ __forceinline__ int64_t at(int64_t r) const {
    return is64 ? static_cast<const int64_t*>(t)[r] : (int64_t) static_cast<const int32_t*>(t)[r];
  }
};

__device__ __forceinline__ bool is_big(float c) { return !(fabsf(c) <= kBig); }

// y of one element against maximum m (c = k m).
__device__ __forceinline__ float y_of(float x, float k, float m, float c) {
  return is_big(c) ? (x - m) * k : fmaf(x, k, -c);
}

// Distance in y from base m1 to base m2 (<= 0 for m1 <= m2), by the same forms.
__device__ __forceinline__ float base_step(float m1, float m2, float k) {
  const float c1 = m1 * k, c2 = m2 * k;
  return is_big(c1) || is_big(c2) ? (m1 - m2) * k : c1 - c2;
}

template <bool ENT>
__device__ __forceinline__ void merge(State& a, const State& b, float k) {
  const float m = fmaxf(a.m, b.m);
  if (m == -INFINITY) {  // nothing but -inf on both sides (s is 0, or NaN)
    a.s += b.s;
    return;
  }
  const float da = base_step(a.m, m, k), db = base_step(b.m, m, k);
  const float fa = ex2_approx(da), fb = ex2_approx(db);
  if constexpr (ENT)
    a.u = (fa > 0.f ? fa * fmaf(a.s, da, a.u) : 0.f) + (fb > 0.f ? fb * fmaf(b.s, db, b.u) : 0.f);
  a.s = fa * a.s + fb * b.s;
  a.m = m;
}

// Adds N elements to a state.
template <bool ENT, int N>
__device__ __forceinline__ void push(State& st, const float (&x)[N], float k) {
  float cm = x[0];
#pragma unroll
  for (int i = 1; i < N; ++i) cm = fmaxf(cm, x[i]);
  if (cm > st.m) {
    const float d = base_step(st.m, cm, k), f = ex2_approx(d);
    if constexpr (ENT) st.u = f > 0.f ? f * fmaf(st.s, d, st.u) : 0.f;
    st.s *= f;
    st.m = cm;
  }
  const float c = st.m * k;
  if (is_big(c)) {  // rare: see the top of the file
#pragma unroll
    for (int i = 0; i < N; ++i) {
      if (st.m == -INFINITY) {
        if (x[i] != x[i]) st.s = x[i];
      } else {
        const float y = (x[i] - st.m) * k, e = ex2_approx(y);
        st.s += e;
        if constexpr (ENT) st.u += e > 0.f ? e * y : 0.f;
      }
    }
    return;
  }
  float s = 0.f, u = 0.f;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    float y = fmaf(x[i], k, -c);
    const float e = ex2_approx(y);
    s += e;
    if constexpr (ENT) u = fmaf(e, fmaxf(y, -1000.f), u);  // y = -inf has e = 0: keep 0 * y finite
  }
  st.s += s;
  if constexpr (ENT) st.u += u;
}

// 16 bytes of T as floats.
template <typename T>
__device__ __forceinline__ void unpack16(const uint4& v, float (&f)[16 / sizeof(T)]) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (std::is_same_v<T, float>) {
      f[i] = __uint_as_float(w[i]);
    } else if constexpr (std::is_same_v<T, __nv_bfloat16>) {  // exact: the bits move up 16 places
      f[2 * i] = __uint_as_float(w[i] << 16);
      f[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    } else {
      const float2 p = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
      f[2 * i] = p.x;
      f[2 * i + 1] = p.y;
    }
  }
}
template <typename T>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
  if constexpr (std::is_same_v<T, __nv_bfloat16>) return pack_bf16x2(a, b);
  else return pack_f16x2(a, b);
}
// N floats to N consecutive T (the address aligned to N * sizeof(T)).
template <typename T, int N>
__device__ __forceinline__ void store_vec(T* p, const float (&f)[N]) {
  if constexpr (std::is_same_v<T, float>) {
#pragma unroll
    for (int i = 0; i < N; i += 4)
      __stcs(reinterpret_cast<float4*>(p + i), make_float4(f[i], f[i + 1], f[i + 2], f[i + 3]));
  } else if constexpr (N == 8) {
    __stcs(reinterpret_cast<uint4*>(p), make_uint4(pack2<T>(f[0], f[1]), pack2<T>(f[2], f[3]), pack2<T>(f[4], f[5]),
                                                   pack2<T>(f[6], f[7])));
  } else {
    static_assert(N == 4, "vector of 4 or 8");
    __stcs(reinterpret_cast<uint2*>(p), make_uint2(pack2<T>(f[0], f[1]), pack2<T>(f[2], f[3])));
  }
}

// Gradient of one element: e (A + B y).
template <bool ENT>
__device__ __forceinline__ float grad_of(float x, float k, float m, float c, bool big, float A, float B) {
  const float y = big ? (x - m) * k : fmaf(x, k, -c);
  const float e = ex2_approx(y);
  if constexpr (ENT) return e * fmaf(B, fmaxf(y, -1000.f), A);
  return e * A;
}

// What the losses of one row hand to its gradient.
struct Coef {
  float A, B;    // dx_i = e_i (A + B y_i)
  float at_t;    // added at the target
  bool masked;   // the row turned out to be masked: zeros
};

// A, B and at_t for dL/dlogp = a and dL/dH = b: dx = g / tau (a ([i = t] - p_i) - b p_i (log p_i + H)).
__device__ __forceinline__ Coef coef_of(float a, float b, float g, const State& st, float inv_tau) {
  const float f = g * inv_tau;
  Coef c;
  c.at_t = a * f;
  c.B = -b * f * kLn2 / st.s;
  c.A = -a * f / st.s - c.B * (st.u / st.s);
  c.masked = false;
  return c;
}

// --------------------------------------------------------------------------
// host
// --------------------------------------------------------------------------
inline int elem_bytes(int dtype) { return dtype == FERRITE_F32 ? 4 : 2; }

// Sizes and types every entry point takes; `out_dtype` < 0 where there is no gradient.
inline int check_rows(const char* op, int64_t rows, int64_t vocab, int64_t ld, float temperature, int dtype,
                      int64_t ld_out, int out_dtype) {
  if (int rc = injected_fault(op)) return rc;
  if (rows < 0 || vocab <= 0 || ld < vocab)
    return fail(FERRITE_BAD_SHAPE, "%s: bad shape rows=%lld vocab=%lld ld=%lld", op, (long long)rows, (long long)vocab, (long long)ld);
  if (rows > 0x7fffffff || vocab > 0x7fffffff) return fail(FERRITE_BAD_SHAPE, "%s: more than 2^31 - 1 rows or columns", op);
  if (!(temperature > 0.f) || !std::isfinite(temperature) || !std::isfinite(kLog2e / temperature))
    return fail(FERRITE_BAD_SHAPE, "%s: temperature %g (it must be positive)", op, (double)temperature);
  if (dtype != FERRITE_F32 && dtype != FERRITE_BF16 && dtype != FERRITE_F16)
    return fail(FERRITE_UNSUPPORTED_DTYPE, "%s: logits dtype %d", op, dtype);
  if (out_dtype >= 0) {
    if (ld_out < vocab) return fail(FERRITE_BAD_SHAPE, "%s: ld_out %lld < vocab %lld", op, (long long)ld_out, (long long)vocab);
    if (out_dtype != dtype && !(dtype == FERRITE_F32 && (out_dtype == FERRITE_BF16 || out_dtype == FERRITE_F16)))
      return fail(FERRITE_UNSUPPORTED_DTYPE, "%s: gradient dtype %d for logits dtype %d (the logits' own, or 16-bit for f32)", op, out_dtype, dtype);
  }
  return FERRITE_OK;
}
inline int check_targets(const char* op, int target_dtype) {
  if (target_dtype != 0 && target_dtype != 1)
    return fail(FERRITE_UNSUPPORTED_DTYPE, "%s: target dtype %d (0 = int32, 1 = int64)", op, target_dtype);
  return FERRITE_OK;
}
inline bool misaligned(const void* p, int esz) { return (reinterpret_cast<uintptr_t>(p) & (uintptr_t)(esz - 1)) != 0; }

// sum_r terms[r] into *loss, in a fixed order (one CTA; f64 partial sums).
int sum_terms(cudaStream_t s, const float* terms, float* loss, int64_t n, float scale, const char* op);

}  // namespace rowloss
}  // namespace ferrite
