// Log-probabilities (and entropies) of given tokens, the clipped policy loss with its KL
// term and entropy bonus, and the preference loss of paired sequences: row losses whose
// gradient has one single-entry term, the target's.  Formulas: rowloss.cuh.
//
//   policy:      ratio = exp(logp - old), pg = -min(ratio A, clamp(ratio, 1 - lo, 1 + hi) A),
//                kl = exp(ref - logp) - (ref - logp) - 1, loss = sum_r w_r (pg + beta kl - c H)
//                dL/dlogp = w (-A ratio [not clipped] + beta (1 - exp(ref - logp))), dL/dH = -w c
//   preference:  d_j = sum (or mean) over sequence j of logp - ref, h = d_chosen - d_rejected,
//                loss = mean over pairs of a function of h; dL/dlogp = +- dloss/dh / pairs (/ count)
#include "rowkernel.cuh"

namespace ferrite {
namespace rowloss {

// The logit at the target; a target outside [0, vocab) gives NaN (nothing is read out of range).
template <typename TI>
__device__ __forceinline__ float logit_at(const TI* x, int64_t t, int64_t n) {
  return t >= 0 && t < n ? DT<TI>::to_f(x[t]) : __int_as_float(0x7fc00000);
}

// The same by a whole warp, and a base: the largest of the 32 logits around it, which come with it.
template <typename TI>
__device__ __forceinline__ float logit_and_base(const TI* x, int64_t t, const RowIn& in, float& base) {
  const int lane = threadIdx.x & 31;
  const int64_t i = (t & ~(int64_t)31) + lane;
  const float v = t >= 0 && t < in.vocab && i < in.vocab ? DT<TI>::to_f(x[i]) : __int_as_float(0x7fc00000);
  float m = v;
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, off));
  base = base_of(m, in);
  return __shfl_sync(0xffffffffu, v, (int)(t & 31));
}

template <bool ENT>
struct LogprobsFwd {
  static constexpr bool kLogp = true, kEnt = ENT, kGradEnt = false, kHasStats = false, kList = false, kForwardOnly = true;
  Targets t;
  float* logp;
  float* entropy;
  float2* stats;
  struct Pre {
    int64_t t;
  };
  struct Row {
    float xt;
  };
  __host__ __device__ int slot_bytes() const { return sizeof(Row); }
  __device__ Pre pre(int64_t r) const { return Pre{t.at(r)}; }
  __device__ bool live(const Pre& p) const { return p.t != t.ignore; }
  __device__ void dead(int64_t r) const {
    logp[r] = 0.f;
    if constexpr (ENT) entropy[r] = 0.f;
    if (stats) stats[r] = make_float2(0.f, 1.f);
  }
  template <typename TI>
  __device__ float prep(int64_t, const Pre& p, const TI* x, const RowIn& in, char* slot) const {
    float base;
    const float xt = logit_and_base(x, p.t, in, base);
    if ((threadIdx.x & 31) == 0) reinterpret_cast<Row*>(slot)->xt = xt;
    return base;
  }
  __device__ Coef finish(int64_t, const Norm&, const RowIn&, float, char*) const { return Coef{}; }
  __device__ void results(int64_t r, const Norm& w, const RowIn& in, char* slot) const {
    if ((threadIdx.x & 31) == 0) {
      logp[r] = logp_of(reinterpret_cast<Row*>(slot)->xt, w, in);
      if constexpr (ENT) entropy[r] = entropy_of(w);
      if (stats) stats[r] = make_float2(w.base, w.big ? -w.s : w.s);
    }
  }
};

template <bool ENT>
struct LogprobsBwd {
  static constexpr bool kLogp = true, kEnt = false, kGradEnt = ENT, kHasStats = true, kList = false, kForwardOnly = false;
  Targets t;
  const float2* stats;
  const float* entropy;   // ENT: the forward's
  const float* dlogp;     // null: 0
  const float* dentropy;  // ENT
  struct Pre {
    int64_t t;
  };
  struct Row {
    Norm w;
    float a, b, xt;
    int64_t t;
  };
  __host__ __device__ int slot_bytes() const { return sizeof(Row); }
  __device__ Pre pre(int64_t r) const { return Pre{t.at(r)}; }
  __device__ bool live(const Pre& p) const { return p.t != t.ignore; }
  __device__ void dead(int64_t) const {}
  template <typename TI>
  __device__ float prep(int64_t r, const Pre& p, const TI* x, const RowIn& in, char* slot) const {
    if ((threadIdx.x & 31) != 0) return 0.f;
    Row& w = *reinterpret_cast<Row*>(slot);
    const float2 v = stats[r];
    w.w = Norm{v.x, fabsf(v.y), 0.f, 0.f, !(v.y > 0.f)};
    w.a = p.t >= 0 && p.t < in.vocab ? (dlogp ? dlogp[r] : 0.f) : __int_as_float(0x7fc00000);
    w.b = 0.f;
    if constexpr (ENT) {
      w.w.mean = log2f(w.w.s) - entropy[r] * kLog2e;
      w.b = dentropy[r];
    }
    w.t = p.t;
    w.xt = logit_at(x, p.t, in.vocab);
    return 0.f;
  }
  __device__ Norm state(const char* slot) const { return reinterpret_cast<const Row*>(slot)->w; }
  __device__ Coef finish(int64_t, const Norm& w, const RowIn& in, float g, char* slot) const {
    const Row& row = *reinterpret_cast<const Row*>(slot);
    return coef_of<ENT>(row.a, row.b, g, row.t, row.xt, w, in);
  }
  __device__ void results(int64_t, const Norm&, const RowIn&, char*) const {}
};

// ENT: the entropy bonus takes part in the gradient (its value is always written).
template <bool ENT>
struct Policy {
  static constexpr bool kLogp = true, kEnt = true, kGradEnt = ENT, kHasStats = false, kList = false, kForwardOnly = false;
  Targets t;
  const float* old_logp;
  const float* adv;
  const float* weights;  // null: 1 / rows
  const float* ref;      // null: no KL term
  float lo, hi, beta, ent_coef, uniform;
  float* terms;  // [rows] w * loss
  float* logp;
  float* entropy;
  float* kl;
  uint8_t* clipped;
  struct Pre {
    int64_t t;
    float w;
  };
  struct Row {
    int64_t t;
    float w, xt, old_logp, adv, ref;
  };
  __host__ __device__ int slot_bytes() const { return sizeof(Row); }
  __device__ Pre pre(int64_t r) const { return Pre{t.at(r), weights ? weights[r] : uniform}; }
  __device__ bool live(const Pre& p) const { return p.t != t.ignore && p.w != 0.f; }
  __device__ void dead(int64_t r) const {
    terms[r] = logp[r] = entropy[r] = kl[r] = 0.f;
    clipped[r] = 0;
  }
  template <typename TI>
  __device__ float prep(int64_t r, const Pre& p, const TI* x, const RowIn& in, char* slot) const {
    float base;
    const float xt = logit_and_base(x, p.t, in, base);
    if ((threadIdx.x & 31) == 0) *reinterpret_cast<Row*>(slot) = Row{p.t, p.w, xt, old_logp[r], adv[r], ref ? ref[r] : 0.f};
    return base;
  }
  struct Step {
    float logp, ratio, plain, bounded, em;  // em = exp(ref - logp) - 1
    bool cut;
  };
  __device__ Step step(const Row& row, const Norm& w, const RowIn& in) const {
    Step t;
    t.logp = logp_of(row.xt, w, in);
    t.ratio = expf(t.logp - row.old_logp);
    t.plain = t.ratio * row.adv;
    t.bounded = fminf(fmaxf(t.ratio, 1.f - lo), 1.f + hi) * row.adv;
    t.cut = t.bounded < t.plain;
    t.em = ref ? expm1f(row.ref - t.logp) : 0.f;
    return t;
  }
  __device__ Coef finish(int64_t, const Norm& w, const RowIn& in, float g, char* slot) const {
    const Row& row = *reinterpret_cast<const Row*>(slot);
    const Step t = step(row, w, in);
    const float da = fmaf(-beta, t.em, t.cut ? 0.f : -t.plain);
    return coef_of<ENT>(row.w * da, ENT ? -row.w * ent_coef : 0.f, g, row.t, row.xt, w, in);
  }
  __device__ void results(int64_t r, const Norm& w, const RowIn& in, char* slot) const {
    const Row& row = *reinterpret_cast<const Row*>(slot);
    const Step t = step(row, w, in);
    const float h = entropy_of(w), klv = ref ? t.em - (row.ref - t.logp) : 0.f;
    if ((threadIdx.x & 31) == 0) {
      terms[r] = row.w * fmaf(-ent_coef, h, fmaf(beta, klv, t.cut ? -t.bounded : -t.plain));
      logp[r] = t.logp;
      entropy[r] = h;
      kl[r] = klv;
      clipped[r] = t.cut;
    }
  }
};

// ---- sums in a fixed order ---------------------------------------------------

constexpr int kSumThreads = 1024;

template <typename T>
__device__ __forceinline__ T block_sum(T v, T* sh) {
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) v += __shfl_xor_sync(0xffffffffu, v, off);
  __syncthreads();  // sh may still be read from a previous call
  if ((threadIdx.x & 31) == 0) sh[threadIdx.x >> 5] = v;
  __syncthreads();
  v = sh[0];
  for (int w = 1; w < (int)(blockDim.x >> 5); ++w) v += sh[w];
  return v;
}

__global__ void __launch_bounds__(kSumThreads) sum_terms_kernel(const float* __restrict__ terms, float* __restrict__ loss, int64_t n, float scale) {
  __shared__ double sh[32];
  pdl_launch_dependents();
  pdl_wait();
  double v = 0.0;
  for (int64_t i = threadIdx.x; i < n; i += blockDim.x) v += (double)terms[i];
  v = block_sum(v, sh);
  if (threadIdx.x == 0) *loss = (float)(v * (double)scale);
}

int sum_terms(cudaStream_t s, const float* terms, float* loss, int64_t n, float scale, const char* op) {
  const int threads = n <= 256 ? 256 : kSumThreads;
  const cudaError_t e = launch_pdl(sum_terms_kernel, dim3(1), dim3(threads), 0, s, terms, loss, n, scale);
  if (e != cudaSuccess) return fail(FERRITE_LAUNCH_FAILED, "%s: %s", op, cudaGetErrorString(e));
  return check_launch(op);
}

// ---- the pairs of the preference loss -----------------------------------------

struct Pairs {
  const float* logp;
  const float* ref;
  Targets t;
  const int64_t* offsets;  // [2 pairs + 1]
  float* terms;            // [pairs]
  float* margins;          // [pairs] beta h
  float* coef;             // [rows] dL/dlogp, null: forward only
  int64_t rows, pairs;
  float beta, smooth;
  int kind, average;
};

constexpr int kPairThreads = 256;

// One CTA per pair: the two sequences' sums of logp - ref (f64, a fixed order), the loss, and
// dL/dlogp of every row of the two sequences.  The first CTA also zeroes the rows before
// the first sequence and the last one those after the last.
__global__ void __launch_bounds__(kPairThreads) pairs_kernel(Pairs a) {
  __shared__ double sh[kPairThreads / 32];
  pdl_launch_dependents();
  pdl_wait();
  const int64_t p = blockIdx.x;
  double d[2];
  float n[2];
  int64_t lo[2], hi[2];
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    lo[j] = min(max(a.offsets[2 * p + j], (int64_t)0), a.rows);
    hi[j] = min(max(a.offsets[2 * p + j + 1], lo[j]), a.rows);
    double s = 0.0, c = 0.0;
    for (int64_t i = lo[j] + threadIdx.x; i < hi[j]; i += blockDim.x)
      if (a.t.at(i) != a.t.ignore) {
        s += (double)a.logp[i] - (double)a.ref[i];
        c += 1.0;
      }
    d[j] = block_sum(s, sh);
    n[j] = 1.f;
    if (a.average) {
      n[j] = (float)fmax(block_sum(c, sh), 1.0);
      d[j] /= (double)n[j];
    }
  }
  const float h = (float)(d[0] - d[1]), b = a.beta, bh = b * h;
  float loss, dh;
  if (a.kind == 0) {  // sigmoid: softplus(-x) = log1p(exp(-|x|)) + max(-x, 0)
    const float l = log1pf(expf(-fabsf(bh)));
    loss = (1.f - a.smooth) * (l + fmaxf(-bh, 0.f)) + a.smooth * (l + fmaxf(bh, 0.f));
    if (bh != bh) loss = bh;
    // e sigma(bh) - (1 - e) sigma(-bh): of two terms near 1 (sigma(bh) - (1 - e)) the difference loses a settled pair's gradient
    dh = b * (a.smooth / (1.f + expf(-bh)) - (1.f - a.smooth) / (1.f + expf(bh)));
  } else if (a.kind == 1) {  // squared
    const float q = h - 0.5f / b;
    loss = q * q;
    dh = 2.f * q;
  } else {  // hinge
    const float q = 1.f - bh;
    loss = q > 0.f ? q : (q != q ? q : 0.f);
    dh = q > 0.f ? -b : (q != q ? q : 0.f);
  }
  if (threadIdx.x == 0) {
    a.terms[p] = loss;
    a.margins[p] = bh;
  }
  if (!a.coef) return;
  const float g = dh / (float)a.pairs;
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const float gj = (j == 0 ? g : -g) / n[j];
    for (int64_t i = lo[j] + threadIdx.x; i < hi[j]; i += blockDim.x) a.coef[i] = a.t.at(i) != a.t.ignore ? gj : 0.f;
  }
  if (p == 0)
    for (int64_t i = threadIdx.x; i < lo[0]; i += blockDim.x) a.coef[i] = 0.f;
  if (p == a.pairs - 1)
    for (int64_t i = hi[1] + threadIdx.x; i < a.rows; i += blockDim.x) a.coef[i] = 0.f;
}

static int check_pairs(const char* op, const float* logp, const float* ref_logp, const void* targets, const int64_t* offsets, float beta,
                       float label_smoothing, int kind, const float* loss, const float* margins, const float* workspace, size_t workspace_bytes,
                       int64_t rows, int64_t pairs, int target_dtype) {
  if (rows < 0 || pairs < 1 || pairs > 0x3fffffff) return fail(FERRITE_BAD_SHAPE, "%s: rows=%lld pairs=%lld", op, (long long)rows, (long long)pairs);
  if (int rc = check_targets(op, target_dtype)) return rc;
  if (kind < 0 || kind > 2) return fail(FERRITE_BAD_SHAPE, "%s: kind %d (0 sigmoid, 1 squared, 2 hinge)", op, kind);
  if (!(beta > 0.f) || !std::isfinite(beta)) return fail(FERRITE_BAD_SHAPE, "%s: beta %g (it must be positive)", op, (double)beta);
  if (!(label_smoothing >= 0.f && label_smoothing < 0.5f)) return fail(FERRITE_BAD_SHAPE, "%s: label_smoothing %g (0 <= it < 0.5)", op, (double)label_smoothing);
  if (workspace_bytes < (size_t)pairs * sizeof(float)) return fail(FERRITE_WORKSPACE_TOO_SMALL, "%s: workspace of %zu bytes, %lld needed", op, workspace_bytes, (long long)pairs * 4);
  if (!offsets || !loss || !margins || !workspace || (rows > 0 && (!logp || !ref_logp || !targets)))
    return fail(FERRITE_BAD_SHAPE, "%s: null pointer", op);
  return FERRITE_OK;
}

}  // namespace rowloss

FERRITE_DEFINE_STATUS_READER(status_logprobs)

}  // namespace ferrite

using namespace ferrite;
using namespace ferrite::rowloss;

extern "C" {

int ferrite_logprobs_fwd(void* stream, const void* logits, const void* targets, float* logp, float* entropy, float* stats, int64_t rows,
                         int64_t vocab, int64_t ld, int64_t ignore_index, double temperature, int dtype, int target_dtype) {
  const char* op = "logprobs_fwd";
  if (int rc = check_rows(op, rows, vocab, ld, temperature, dtype, 0, -1)) return rc;
  if (int rc = check_targets(op, target_dtype)) return rc;
  if (rows == 0) return FERRITE_OK;
  if (!logits || !targets || !logp) return fail(FERRITE_BAD_SHAPE, "%s: null pointer", op);
  if (misaligned(logits, elem_bytes(dtype)) || misaligned(stats, 8)) return fail(FERRITE_BAD_ALIGNMENT, "%s: misaligned pointer", op);
  const RowIn in = row_in(logits, rows, vocab, ld, temperature);
  const Targets t{targets, target_dtype, ignore_index};
  cudaStream_t s = (cudaStream_t)stream;
  if (entropy) return dispatch_row(s, in, RowOut{}, LogprobsFwd<true>{t, logp, entropy, (float2*)stats}, dtype, -1, op);
  return dispatch_row(s, in, RowOut{}, LogprobsFwd<false>{t, logp, nullptr, (float2*)stats}, dtype, -1, op);
}

int ferrite_logprobs_bwd(void* stream, const void* logits, const void* targets, const float* stats, const float* entropy,
                         const float* dlogp, const float* dentropy, const float* dloss, float scale, void* dlogits, int64_t rows,
                         int64_t vocab, int64_t ld, int64_t ld_out, int64_t ignore_index, double temperature, int dtype, int target_dtype,
                         int out_dtype) {
  const char* op = "logprobs_bwd";
  if (int rc = check_rows(op, rows, vocab, ld, temperature, dtype, ld_out, out_dtype < 0 ? 99 : out_dtype)) return rc;
  if (int rc = check_targets(op, target_dtype)) return rc;
  if (rows == 0) return FERRITE_OK;
  if (!logits || !targets || !stats || !dlogits || (dentropy && !entropy)) return fail(FERRITE_BAD_SHAPE, "%s: null pointer", op);
  if (misaligned(logits, elem_bytes(dtype)) || misaligned(dlogits, elem_bytes(out_dtype)) || misaligned(stats, 8))
    return fail(FERRITE_BAD_ALIGNMENT, "%s: misaligned pointer", op);
  const RowIn in = row_in(logits, rows, vocab, ld, temperature);
  const RowOut out{dlogits, ld_out, dloss, scale};
  const Targets t{targets, target_dtype, ignore_index};
  cudaStream_t s = (cudaStream_t)stream;
  if (dentropy) return dispatch_row(s, in, out, LogprobsBwd<true>{t, (const float2*)stats, entropy, dlogp, dentropy}, dtype, out_dtype, op);
  return dispatch_row(s, in, out, LogprobsBwd<false>{t, (const float2*)stats, nullptr, dlogp, nullptr}, dtype, out_dtype, op);
}

int ferrite_policy_loss(void* stream, const void* logits, const void* targets, const float* old_logp, const float* advantages,
                        const float* weights, const float* ref_logp, float clip_low, float clip_high, float kl_coef, float entropy_coef,
                        double temperature, const float* dloss, float scale, float* loss, float* logp, float* entropy, float* kl,
                        uint8_t* clipped, void* dlogits, float* workspace, size_t workspace_bytes, int64_t rows, int64_t vocab, int64_t ld,
                        int64_t ld_out, int64_t ignore_index, int dtype, int target_dtype, int out_dtype) {
  const char* op = "policy_loss";
  if (int rc = check_rows(op, rows, vocab, ld, temperature, dtype, ld_out, dlogits ? (out_dtype < 0 ? 99 : out_dtype) : -1)) return rc;
  if (int rc = check_targets(op, target_dtype)) return rc;
  if (!(clip_low >= 0.f) || !(clip_high >= 0.f)) return fail(FERRITE_BAD_SHAPE, "%s: clip_low %g, clip_high %g (neither may be negative)", op, (double)clip_low, (double)clip_high);
  if (!loss) return fail(FERRITE_BAD_SHAPE, "%s: null pointer", op);
  if (workspace_bytes < (size_t)rows * sizeof(float)) return fail(FERRITE_WORKSPACE_TOO_SMALL, "%s: workspace of %zu bytes, %lld needed", op, workspace_bytes, (long long)rows * 4);
  cudaStream_t s = (cudaStream_t)stream;
  if (rows > 0) {
    if (!logits || !targets || !old_logp || !advantages || !logp || !entropy || !kl || !clipped || !workspace)
      return fail(FERRITE_BAD_SHAPE, "%s: null pointer", op);
    if (misaligned(logits, elem_bytes(dtype)) || (dlogits && misaligned(dlogits, elem_bytes(out_dtype))))
      return fail(FERRITE_BAD_ALIGNMENT, "%s: misaligned pointer", op);
    const RowIn in = row_in(logits, rows, vocab, ld, temperature);
    const RowOut out{dlogits, ld_out, dloss, scale};
    const Targets t{targets, target_dtype, ignore_index};
    const float uniform = 1.f / (float)rows;
    const int od = dlogits ? out_dtype : -1;
    int rc;
    if (entropy_coef != 0.f && dlogits)
      rc = dispatch_row(s, in, out, Policy<true>{t, old_logp, advantages, weights, ref_logp, clip_low, clip_high, kl_coef, entropy_coef, uniform, workspace, logp, entropy, kl, clipped}, dtype, od, op);
    else
      rc = dispatch_row(s, in, out, Policy<false>{t, old_logp, advantages, weights, ref_logp, clip_low, clip_high, kl_coef, entropy_coef, uniform, workspace, logp, entropy, kl, clipped}, dtype, od, op);
    if (rc) return rc;
  }
  return sum_terms(s, workspace, loss, rows, 1.f, op);
}

int ferrite_preference_pairs(void* stream, const float* logp, const float* ref_logp, const void* targets, const int64_t* offsets,
                             float beta, float label_smoothing, int kind, int average, float* loss, float* margins, float* coef,
                             float* workspace, size_t workspace_bytes, int64_t rows, int64_t pairs, int64_t ignore_index, int target_dtype) {
  const char* op = "preference_pairs";
  if (int rc = injected_fault(op)) return rc;
  if (int rc = check_pairs(op, logp, ref_logp, targets, offsets, beta, label_smoothing, kind, loss, margins, workspace, workspace_bytes, rows, pairs, target_dtype))
    return rc;
  cudaStream_t s = (cudaStream_t)stream;
  const Pairs a{logp, ref_logp, Targets{targets, target_dtype, ignore_index}, offsets, workspace, margins, coef, rows, pairs, beta, label_smoothing, kind, average};
  const cudaError_t e = launch_pdl(pairs_kernel, dim3((unsigned)pairs), dim3(kPairThreads), 0, s, a);
  if (e != cudaSuccess) return fail(FERRITE_LAUNCH_FAILED, "%s: %s", op, cudaGetErrorString(e));
  if (int rc = check_launch(op)) return rc;
  return sum_terms(s, workspace, loss, pairs, 1.f / (float)pairs, op);
}

int ferrite_preference_loss(void* stream, const void* logits, const void* targets, const float* ref_logp, const int64_t* offsets, float beta,
                            float label_smoothing, int kind, int average, double temperature, float scale, float* loss, float* margins,
                            float* logp, float* stats, float* coef, void* dlogits, float* workspace, size_t workspace_bytes, int64_t rows,
                            int64_t pairs, int64_t vocab, int64_t ld, int64_t ld_out, int64_t ignore_index, int dtype, int target_dtype,
                            int out_dtype) {
  const char* op = "preference_loss";
  if (int rc = injected_fault(op)) return rc;
  if (dlogits) {  // before anything is launched
    if (int rc = check_rows(op, rows, vocab, ld, temperature, dtype, ld_out, out_dtype < 0 ? 99 : out_dtype)) return rc;
    if (rows > 0 && (!stats || !coef)) return fail(FERRITE_BAD_SHAPE, "%s: null pointer", op);
    if (misaligned(dlogits, elem_bytes(out_dtype))) return fail(FERRITE_BAD_ALIGNMENT, "%s: misaligned pointer", op);
  }
  if (int rc = check_pairs(op, logp, ref_logp, targets, offsets, beta, label_smoothing, kind, loss, margins, workspace, workspace_bytes, rows, pairs, target_dtype))
    return rc;
  if (int rc = ferrite_logprobs_fwd(stream, logits, targets, logp, nullptr, stats, rows, vocab, ld, ignore_index, temperature, dtype, target_dtype)) return rc;
  if (int rc = ferrite_preference_pairs(stream, logp, ref_logp, targets, offsets, beta, label_smoothing, kind, average, loss, margins, coef, workspace,
                                        workspace_bytes, rows, pairs, ignore_index, target_dtype))
    return rc;
  if (!dlogits) return FERRITE_OK;
  return ferrite_logprobs_bwd(stream, logits, targets, stats, nullptr, coef, nullptr, nullptr, scale, dlogits, rows, vocab, ld, ld_out, ignore_index,
                              temperature, dtype, target_dtype, out_dtype);
}

}  // extern "C"
