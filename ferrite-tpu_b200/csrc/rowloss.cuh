// Row losses over logits [rows, vocab]: what the post-training losses share.
//
// With z = x / tau, every loss here is a function of one row's softmax:
//   lse = log sum_i exp(z_i),  logp_t = z_t - lse,  H = -sum_i p_i log p_i,
// and its gradient is  dx_i = e_i (A + B y_i)  plus a few single-entry terms (the
// target's, or the teacher's listed tokens), where in units of log 2
//   k = log2(e) / tau,  y_i = k (x_i - m),  e_i = 2^y_i,  s = sum e_i,  u = sum e_i y_i,
//   logp_i = ln2 (y_i - log2 s),   H = ln2 (log2 s - u / s),   p_i = e_i / s.
// A row's state is (m, s, u): it is built in one pass and merged pairwise.  m is a base, not the
// maximum: 2^y keeps its precision over the whole exponent range, so any logit of the row's upper
// part serves, and the sums are checked instead -- one that is too high is redone against the largest
// element.  No maximum is taken per element, and no rescaling runs in the usual case.  Too high is 2^10 where
// log p and the entropy are asked for: log2 s and u / s both grow with the distance of the base from
// the row's upper part, the entropy is their difference, and what it loses is a few roundings of
// that distance.  So that few sums are redone, the base there is the largest of the 32 logits that are fetched with the
// target's.  Elsewhere (distillation) it is 2^80, and the base is the student's logit at a teacher's token.  The base's own
// term is 1 without rounding.  All of it is f32; only the gradient is rounded, once, on store.
//
// y_i is K x_i - c with c = k m rounded -- one number for every term of s and for logp, so that its
// rounding cancels -- and K is carried to more than f32: the rounding of k alone would shift every
// log-probability the same way, and sums over long sequences would show it.  The sums take K as
// k_hi + k_rest, two fma: split after 12 bits, because the rest of a split after 24 is less than half
// a unit of a y of 4 or more and would be rounded away each time; positive, because -inf times a rest
// of 0 or below would be NaN.  Where |c| passes
// 2^16 (logits in the tens of thousands, rows of the type's lowest value, infinities) y_i is
// k (x_i - m) with m the maximum.  At its end a row is normalised: c takes up the power of two of s, so that s lies in
// [1, 2) and its logarithm is small beside y.  A logit of -inf has e_i = 0
// and contributes nothing; NaN and +inf make the row's results NaN.
#pragma once

#include <cmath>
#include <type_traits>

#include "common.cuh"

namespace ferrite {
namespace rowloss {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
constexpr float kBig = 65536.f;   // |k m| above this: y is k (x - m)
constexpr float kHigh = 0x1p10f, kHuge = 0x1p80f;  // sums above this (an Op's) are redone against the maximum

// (m, s, u): the base, sum of e and sum of e * y of the elements seen so far; low: the part of s that is known to
// come from elements at or below the base, or hardly above it.
struct State {
  float m, s, u, low;
};
__device__ __forceinline__ State empty_state(float base = -INFINITY) { return State{base, 0.f, 0.f, 0.f}; }

// The mean error of ex2.approx, relative and measured against f64 over 10^7 values an octave: -5.1e-8 below y = -1,
// 3.4e-8 above y = 1, less between.  It is under half a step of f32, but sums of log-probabilities over long sequences
// show what goes one way.  Of what is known to lie below the base it is taken out (logp_of, rebase).
constexpr float kEx2Low = 5.1e-8f;

// Rows whose results are asked for.
struct RowIn {
  const void* logits;
  int64_t rows, vocab, ld;
  float k, k_lo;      // log2(e) / tau, and what its rounding left
  float k_hi, k_rest;  // the same split after 12 bits, k_rest > 0
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

// A logit as a base; -inf (any first element moves it) where it cannot be one.
__device__ __forceinline__ float base_of(float x, const RowIn& in) { return is_big(x * in.k) ? -INFINITY : x; }

// y of base m1 against base m2 >= m1 (neither -inf): the log2 of the factor that takes sums over
// to the new base.
__device__ __forceinline__ float base_step(float m1, float m2, const RowIn& in) {
  const float c1 = __fmul_rn(m1, in.k), c2 = __fmul_rn(m2, in.k);
  if (!is_big(c1)) return !is_big(c2) ? c1 - c2 : -(fmaf(m2, in.k, -c1) + m2 * in.k_lo);
  return !is_big(c2) ? fmaf(m1, in.k, -c2) + m1 * in.k_lo : (m1 - m2) * in.k;
}

// A state's sums against base m >= st.m.  (A base of -inf means no element, or -inf and NaN only: s is 0 or NaN.)
template <bool ENT>
__device__ __forceinline__ void rebase(State& st, float m, const RowIn& in) {
  if (st.m == m || st.m == -INFINITY) {
    st.m = m;
    return;
  }
  const float d = base_step(st.m, m, in), f = ex2_approx(d);
  if constexpr (ENT) st.u = f > 0.f && st.s != 0.f ? f * fmaf(st.s, d, st.u) : 0.f;
  // s f (1 + kEx2Low), rounded once (and never one fma with what is added to it: a row's s has the same bits in every kernel)
  st.s = fmaf(st.s, f, __fmul_rn(__fmul_rn(st.s, f), kEx2Low));
  st.low = __fmul_rn(st.low, f);
  st.m = m;
}

// The states of a warp's lanes merged, in all lanes: one base (they usually have it), plain sums.
template <bool ENT, bool LOGP>
__device__ __forceinline__ State warp_merge(State st, const RowIn& in) {
  if (!__all_sync(0xffffffffu, st.m == __shfl_sync(0xffffffffu, st.m, 0))) {
    float m = st.m;
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, off));
    rebase<ENT>(st, m, in);
  }
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) {
    st.s += __shfl_xor_sync(0xffffffffu, st.s, off);
    if constexpr (ENT) st.u += __shfl_xor_sync(0xffffffffu, st.u, off);
    if constexpr (LOGP) st.low += __shfl_xor_sync(0xffffffffu, st.low, off);
  }
  return st;
}

// Adds N elements to a state: any values, against their maximum where it is above the base.
template <bool ENT, int N>
__device__ __forceinline__ void push_any(State& st, const float (&x)[N], const RowIn& in) {
  float cm = x[0];
#pragma unroll
  for (int i = 1; i < N; ++i) cm = fmaxf(cm, x[i]);
  if (cm > st.m) rebase<ENT>(st, cm, in);
  const float c = st.m * in.k;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    if (st.m == -INFINITY) {  // nothing but -inf so far
      if (x[i] != x[i]) st.s = x[i];
    } else {
      const float y = is_big(c) ? (x[i] - st.m) * in.k : fmaf(x[i], in.k_rest, fmaf(x[i], in.k_hi, -c));
      const float e = ex2_approx(y);
      st.s += e;
      if constexpr (ENT) st.u += e > 0.f ? e * y : 0.f;
    }
  }
}

// -k m for the usual values' form of y, or NaN where the base is big (every sum then fails its check).
__device__ __forceinline__ float minus_c(float m, const RowIn& in) {
  const float c = __fmul_rn(m, in.k);
  return is_big(c) ? __int_as_float(0x7fc00000) : -c;
}

// k, k_hi and k_rest in both halves of register pairs.
struct Pairs2 {
  uint64_t k, k_hi, k_rest;
  __device__ __forceinline__ explicit Pairs2(const RowIn& in) : k(f2_make(in.k, in.k)), k_hi(f2_make(in.k_hi, in.k_hi)), k_rest(f2_make(in.k_rest, in.k_rest)) {}
};

// Sums of the usual values: per pair of elements two packed fma (y), two ex2 and packed adds.  They
// count only if usual() holds of s; otherwise the elements go through push_any.  u then is right too, or NaN from an
// e of 0 times a y of -inf (masked columns, a row's padding): dot_masked has it without those.
template <bool ENT, int N>
__device__ __forceinline__ void sum_usual(uint64_t& s2, uint64_t& u2, const float (&x)[N], float nc, const Pairs2& kk) {
  const uint64_t c2 = f2_make(nc, nc);
#pragma unroll
  for (int i = 0; i < N; i += 2) {
    const uint64_t x2 = f2_make(x[i], x[i + 1]);
    const uint64_t y2 = f2_fma(x2, kk.k_rest, f2_fma(x2, kk.k_hi, c2));
    const uint64_t e2 = f2_make(ex2_approx(f2_lo(y2)), ex2_approx(f2_hi(y2)));
    s2 = f2_add(s2, e2);
    if constexpr (ENT) u2 = f2_fma(e2, y2, u2);
  }
}
// Whether a sum of usual values counts (false for NaN).  By s alone: how a row's s is put together, and so its
// log-probability to the last bit, must not depend on whether u is asked for.
template <bool LOGP>
__device__ __forceinline__ bool usual(float s) {
  return s < (LOGP ? kHigh : kHuge);
}
// A sum up to 2 has no element more than 1 above the base.
constexpr float kLowSum = 2.f;
template <int N>
__device__ __forceinline__ float dot_masked(const float (&x)[N], float nc, const RowIn& in) {
  float u = 0.f;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const float y = fmaf(x[i], in.k_rest, fmaf(x[i], in.k_hi, nc));
    u = fmaf(ex2_approx(y), fmaxf(y, -1000.f), u);
  }
  return u;
}

// Moves the base up to cm, the maximum of what is added next; nc = minus_c(st.m), kept up to date.  What stands for
// elements past a row's end (down to -1e30) is no base.
template <bool ENT>
__device__ __forceinline__ bool raise(State& st, float& nc, float cm, const RowIn& in) {
  if (!(cm > st.m && cm > -9e29f)) return false;
  rebase<ENT>(st, cm, in);
  nc = minus_c(cm, in);
  return true;
}
// Adds N elements to a state; `dot`: to its u alone.
template <bool ENT, bool LOGP, int N>
__device__ __forceinline__ void push(State& st, float& nc, const float (&x)[N], const RowIn& in, const Pairs2& kk, bool dot = false) {
  if constexpr (N % 2 == 0) {
    for (bool again = true; again;) {
      uint64_t s2 = f2_make(0.f, 0.f), u2 = s2;
      sum_usual<ENT>(s2, u2, x, nc, kk);
      const float s = f2_lo(s2) + f2_hi(s2);
      float u = ENT ? f2_lo(u2) + f2_hi(u2) : 0.f;
      if (usual<LOGP>(s)) {
        if constexpr (ENT) {
          if (u != u) u = dot_masked(x, nc, in);
          st.u += u;
        }
        if (!ENT || !dot) {
          st.s += s;
          if (LOGP && s <= kLowSum) st.low += s;
        }
        return;
      }
      float cm = x[0];
#pragma unroll
      for (int i = 1; i < N; ++i) cm = fmaxf(cm, x[i]);
      again = raise<ENT>(st, nc, cm, in);
    }
  }
  push_any<ENT>(st, x, in);
  nc = minus_c(st.m, in);
}

// A finished row: base (c, or m where big), s, the mean of y, u / s, and the share of s that is known to be low
// (the base's own element aside, whose 1 is exact).
struct Norm {
  float base, s, mean, low;
  int big;
};
// Moves the power of two of s into the base, exactly: c2 = c + j is rounded, and what the rounding
// left goes back into s (2^err by its series: |err| <= 2^-7).
template <bool ENT>
__device__ __forceinline__ Norm normalise(const State& st, const RowIn& in) {
  const float c = __fmul_rn(st.m, in.k);
  if (is_big(c) || !(st.s < INFINITY)) return Norm{is_big(c) ? st.m : c, st.s, ENT ? st.u / st.s : 0.f, 0.f, is_big(c)};
  const uint32_t bits = __float_as_uint(st.s);
  const float l = (float)((int)(bits >> 23) - 127), f = __uint_as_float((bits & 0x7fffffu) | 0x3f800000u);  // s = 2^l f
  const float c2 = c + l, b = c2 - c, err = (c - (c2 - b)) + (l - b);  // c + l = c2 + err
  const float t = err * kLn2, s = fmaf(f, fmaf(0.5f * t, t, t), f);
  const float inv = __fdividef(1.f, st.s), low = fmaxf(st.low - 1.f, 0.f) * inv;
  if constexpr (!ENT) return Norm{c2, s, 0.f, low, 0};
  const float q = st.u * inv, rest = fmaf(-q, st.s, st.u) * inv;  // u / s = q + rest
  return Norm{c2, s, (q - l) + (rest + err), low, 0};
}
// log p of one logit, rounded once: the difference is taken in f64, and what is known of s's mean error (kEx2Low) is
// taken out.  What is left of it is that of the part of s from elements above the base or in sums with such, if any:
// within 5.1e-8 whatever the logits.
__device__ __forceinline__ float logp_of(float xt, const Norm& w, const RowIn& in) {
  const double k = (double)in.k + (double)in.k_lo, l = (double)log2f(w.s);
  const double y = w.big ? fma((double)(xt - w.base), k, -l) : fma((double)xt, k, -(double)w.base) - l;
  return (float)fma(y, 0.6931471805599453, (double)(-kEx2Low * w.low));
}
__device__ __forceinline__ float entropy_of(const Norm& w) {
  const float h = (log2f(w.s) - w.mean) * kLn2;
  return h < 0.f ? 0.f : h;
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
// The maximum of Q times 16 bytes of T (of 16-bit types two elements at a time).
template <typename T, int Q>
__device__ __forceinline__ float max_of(const uint4 (&v)[Q]) {
  if constexpr (std::is_same_v<T, float>) {
    float m = -INFINITY;
#pragma unroll
    for (int q = 0; q < Q; ++q)
      m = fmaxf(fmaxf(m, fmaxf(__uint_as_float(v[q].x), __uint_as_float(v[q].y))), fmaxf(__uint_as_float(v[q].z), __uint_as_float(v[q].w)));
    return m;
  } else {
    using T2 = std::conditional_t<std::is_same_v<T, __half>, __half2, __nv_bfloat162>;
    auto as = [](const uint32_t& w) { return *reinterpret_cast<const T2*>(&w); };
    T2 m = as(v[0].x);
#pragma unroll
    for (int q = 0; q < Q; ++q) m = __hmax2(__hmax2(m, __hmax2(as(v[q].x), as(v[q].y))), __hmax2(as(v[q].z), as(v[q].w)));
    return fmaxf(DT<T>::to_f(m.x), DT<T>::to_f(m.y));
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

// What the losses of one row hand to its gradient: dx_i = e_i (A + B y_i) with y_i = k x_i - base, or
// k (x_i - base) where big, but at_t at i = t.
struct alignas(16) Coef {
  float base, A, B;
  float at_t;
  int t;            // no single entry: negative
  int16_t big;
  int16_t masked;   // the row turned out to be masked: zeros
};

// Gradient of one element without the single entry.
template <bool ENT>
__device__ __forceinline__ float grad_of(float x, float k, const Coef& cf) {
  const float y = cf.big ? (x - cf.base) * k : fmaf(x, k, -cf.base);
  const float e = ex2_approx(y);
  if constexpr (ENT) return e * fmaf(cf.B, fmaxf(y, -1000.f), cf.A);
  return e * cf.A;
}

// Gradients of N (even) elements; BIG as cf.big.
template <bool ENT, bool BIG, int N>
__device__ __forceinline__ void grads_of(const float (&x)[N], float (&d)[N], float k, const Coef& cf, const Pairs2& kk) {
  if constexpr (BIG) {
#pragma unroll
    for (int j = 0; j < N; ++j) d[j] = grad_of<ENT>(x[j], k, cf);
  } else {
    const uint64_t c2 = f2_make(-cf.base, -cf.base), A2 = f2_make(cf.A, cf.A), B2 = f2_make(cf.B, cf.B);
#pragma unroll
    for (int j = 0; j < N; j += 2) {
      const uint64_t y2 = f2_fma(f2_make(x[j], x[j + 1]), kk.k, c2);
      const uint64_t e2 = f2_make(ex2_approx(f2_lo(y2)), ex2_approx(f2_hi(y2)));
      uint64_t g2 = A2;
      if constexpr (ENT) g2 = f2_fma(B2, f2_make(fmaxf(f2_lo(y2), -1000.f), fmaxf(f2_hi(y2), -1000.f)), A2);
      g2 = f2_mul(e2, g2);
      d[j] = f2_lo(g2);
      d[j + 1] = f2_hi(g2);
    }
  }
}

// The base and common factor of the gradient's y, which leaves k_lo out: k_lo x is taken at the
// logit whose y is 0, x = base / k, where p is largest; the factor takes up the base's rounding.
__device__ __forceinline__ float grad_base(const Norm& w, const RowIn& in, Coef& c) {
  c.big = (int16_t)w.big;
  c.base = w.base;
  if (w.big) return 1.f;
  const float shift = w.base / in.k * in.k_lo;
  c.base = w.base - shift;
  return ex2_approx((c.base - w.base) + shift);
}
// The coefficients for dL/dlogp = a and dL/dH = b: dx = g / tau (a ([i = t] - p_i) - b p_i (log p_i + H)).
// ENT: b may differ from 0.  xt: the logit at t.
template <bool ENT>
__device__ __forceinline__ Coef coef_of(float a, float b, float g, int64_t t, float xt, const Norm& w, const RowIn& in) {
  const float f = g * in.inv_tau;
  Coef c;
  const float scale = grad_base(w, in, c) / w.s;
  c.t = t >= 0 && t < in.vocab ? (int)t : -1;
  c.B = ENT ? -b * f * kLn2 * scale : 0.f;
  c.A = -a * f * scale - (ENT ? c.B * w.mean : 0.f);
  c.at_t = grad_of<ENT>(xt, in.k, c) + a * f;
  c.masked = 0;
  return c;
}

// --------------------------------------------------------------------------
// host
// --------------------------------------------------------------------------
inline int elem_bytes(int dtype) { return dtype == FERRITE_F32 ? 4 : 2; }

inline RowIn row_in(const void* logits, int64_t rows, int64_t vocab, int64_t ld, double temperature) {
  const double k = 1.4426950408889634 / temperature;
  int e = 0;
  const double f = std::frexp(k, &e);
  const float k_hi = (float)std::ldexp(std::floor(f * 4096.0) - 1.0, e - 12);  // below k: k_rest > 0
  return RowIn{logits, rows, vocab, ld, (float)k, (float)(k - (double)(float)k), k_hi, (float)(k - (double)k_hi), (float)(1.0 / temperature)};
}

// Sizes and types every entry point takes; `out_dtype` < 0 where there is no gradient.
inline int check_rows(const char* op, int64_t rows, int64_t vocab, int64_t ld, double temperature, int dtype,
                      int64_t ld_out, int out_dtype) {
  if (int rc = injected_fault(op)) return rc;
  if (rows < 0 || vocab <= 0 || ld < vocab)
    return fail(FERRITE_BAD_SHAPE, "%s: bad shape rows=%lld vocab=%lld ld=%lld", op, (long long)rows, (long long)vocab, (long long)ld);
  if (rows > 0x7fffffff || vocab > 0x7fffffff) return fail(FERRITE_BAD_SHAPE, "%s: more than 2^31 - 1 rows or columns", op);
  if (!(temperature > 0.0) || !std::isfinite((float)temperature) || !std::isfinite((float)(1.4426950408889634 / temperature)))
    return fail(FERRITE_BAD_SHAPE, "%s: temperature %g (it must be positive)", op, temperature);
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
