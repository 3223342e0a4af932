// Distillation from a teacher's top logits: for each row a list of (token, teacher logit)
//   q = softmax(v / tau) over the listed entries,  KL = sum_j q_j (log q_j - logp_{idx_j}),
//   loss = sum_r w_r tau^2 KL_r,   dx_i = w tau (p_i - sum_{j: idx_j = i} q_j)
// with p the student's softmax at the same temperature (rowloss.cuh).  The dense part of
// the gradient is the common row pass; the listed tokens' entries are written after it.
// An entry is absent when its index is negative or its value -inf; a row without entries is
// masked.  A token listed twice counts with the sum of its two weights.
#include "rowkernel.cuh"

namespace ferrite {
namespace rowloss {

constexpr int kMaxTop = 1024;

struct Distill {
  static constexpr bool kEnt = false, kGradEnt = false, kHasStats = false;
  const void* values;   // [rows, top] teacher logits
  const void* indices;  // [rows, top]
  int64_t ld_list;
  int top, value_dtype, index64;
  const float* weights;  // null: 1 / rows
  float uniform, tau;
  float* terms;      // [rows] w * tau^2 * KL
  float* per_token;  // [rows] tau^2 * KL

  // Shared memory: q, the student's logits at the listed tokens, the tokens, and the row's summary.
  struct Shared {
    float* q;
    float* x;
    int* idx;
    float* info;  // [0] sum_j q_j log2 q_j, [1] entries (0: masked row), [2] NaN if an index is out of range
  };
  __device__ Shared shared(char* sh) const {
    Shared s;
    s.q = reinterpret_cast<float*>(sh);
    s.x = s.q + top;
    s.idx = reinterpret_cast<int*>(s.x + top);
    s.info = reinterpret_cast<float*>(s.idx + top);
    return s;
  }
  static size_t shared_bytes(int top) { return (size_t)top * 12 + 16; }

  __device__ float value(int64_t i) const {
    if (value_dtype == FERRITE_F32) return static_cast<const float*>(values)[i];
    if (value_dtype == FERRITE_BF16) return __bfloat162float(static_cast<const __nv_bfloat16*>(values)[i]);
    return __half2float(static_cast<const __half*>(values)[i]);
  }
  __device__ int64_t index(int64_t i) const {
    return index64 ? static_cast<const int64_t*>(indices)[i] : (int64_t) static_cast<const int32_t*>(indices)[i];
  }
  __device__ float weight(int64_t r) const { return weights ? weights[r] : uniform; }
  __device__ bool live(int64_t r) const { return weight(r) != 0.f; }
  __device__ void dead(int64_t r) const { terms[r] = per_token[r] = 0.f; }

  // Warp 0: the teacher's softmax over the list and the student's logits there.
  template <typename TI>
  __device__ void begin(int64_t r, const TI* x, int n, char* sh) const {
    if (threadIdx.x >= 32) return;
    const Shared s = shared(sh);
    const int lane = threadIdx.x;
    const float k = kLog2e / tau;
    float m = -INFINITY, bad = 0.f;
    int count = 0;
    for (int j = lane; j < top; j += 32) {
      int64_t i = index(r * ld_list + j);
      float v = value(r * ld_list + j);
      if (v == -INFINITY) i = -1;
      if (i >= n) bad = __int_as_float(0x7fc00000), i = -1;
      s.idx[j] = i < 0 ? -1 : (int)i;
      s.x[j] = i < 0 ? 0.f : DT<TI>::to_f(x[i]);
      s.q[j] = v;
      if (i >= 0) {
        ++count;
        m = v != v ? v : fmaxf(m, v);  // a NaN value shows through the sums
      }
    }
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) {
      m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, off));
      count += __shfl_xor_sync(0xffffffffu, count, off);
      bad += __shfl_xor_sync(0xffffffffu, bad, off);
    }
    float sum = 0.f, dot = 0.f;
    for (int j = lane; j < top; j += 32) {
      const float y = (s.q[j] - m) * k;
      const float e = s.idx[j] >= 0 ? ex2_approx(y) : 0.f;
      s.q[j] = e;
      sum += e;
      dot += e > 0.f ? e * y : (e != e ? e : 0.f);
    }
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) {
      sum += __shfl_xor_sync(0xffffffffu, sum, off);
      dot += __shfl_xor_sync(0xffffffffu, dot, off);
    }
    for (int j = lane; j < top; j += 32) s.q[j] /= sum;
    if (lane == 0) {
      s.info[0] = dot / sum - log2f(sum);  // sum_j q_j log2 q_j
      s.info[1] = (float)count;
      s.info[2] = bad;
    }
  }
  template <typename TI>
  __device__ Coef finish(int64_t r, const State& st, const TI*, const RowIn& in, float g, bool writer, char* sh) const {
    const Shared s = shared(sh);
    const float w = weight(r);
    const bool any = s.info[1] > 0.f || s.info[2] != s.info[2];
    const float bad = s.info[2];
    if (writer && threadIdx.x < 32) {
      const float c = st.m * in.k, ls = log2f(st.s);
      float part = 0.f;
      for (int j = threadIdx.x; j < top; j += 32)
        if (s.idx[j] >= 0 && s.q[j] != 0.f) part += s.q[j] * (y_of(s.x[j], in.k, st.m, c) - ls);
#pragma unroll
      for (int off = 16; off > 0; off >>= 1) part += __shfl_xor_sync(0xffffffffu, part, off);
      if (threadIdx.x == 0) {
        const float per = any ? tau * tau * kLn2 * (s.info[0] - part) + bad : 0.f;
        per_token[r] = per;
        terms[r] = any ? w * per : 0.f;
      }
    }
    const float f = w * tau * g + bad;
    Coef cf;
    cf.A = f / st.s;
    cf.B = 0.f;
    cf.at_t = -f;
    cf.masked = !any;
    return cf;
  }
  // The listed tokens' entries in [lo, hi): the thread of entry j sums the weights of every entry
  // with the same token, so that a token listed twice is written the same value twice.
  template <typename TO, typename TI>
  __device__ void fix(int64_t, const State& st, const Coef& cf, TO* dx, int lo, int hi, const TI*, const RowIn& in, float, char* sh) const {
    const Shared s = shared(sh);
    if (!(s.info[1] > 0.f)) return;
    const float c = st.m * in.k;
    for (int j = threadIdx.x; j < top; j += blockDim.x) {
      const int i = s.idx[j];
      if (i < lo || i >= hi) continue;
      float q = 0.f;
      for (int l = 0; l < top; ++l) q += s.idx[l] == i ? s.q[l] : 0.f;
      dx[i] = DT<TO>::from_f(fmaf(cf.at_t, q, grad_of<false>(s.x[j], in.k, st.m, c, is_big(c), cf.A, 0.f)));
    }
  }
};

}  // namespace rowloss
}  // namespace ferrite

using namespace ferrite;
using namespace ferrite::rowloss;

extern "C" {

int ferrite_distill_loss(void* stream, const void* logits, const void* values, const void* indices, const float* weights, float temperature,
                         const float* dloss, float scale, float* loss, float* per_token, void* dlogits, float* workspace,
                         size_t workspace_bytes, int64_t rows, int64_t vocab, int64_t top, int64_t ld, int64_t ld_out, int64_t ld_list,
                         int dtype, int value_dtype, int index_dtype, int out_dtype) {
  const char* op = "distill_loss";
  if (int rc = check_rows(op, rows, vocab, ld, temperature, dtype, ld_out, dlogits ? (out_dtype < 0 ? 99 : out_dtype) : -1)) return rc;
  if (top < 1 || top > kMaxTop || ld_list < top)
    return fail(FERRITE_BAD_SHAPE, "%s: lists of %lld entries (1 to %d) with row stride %lld", op, (long long)top, kMaxTop, (long long)ld_list);
  if (value_dtype != FERRITE_F32 && value_dtype != FERRITE_BF16 && value_dtype != FERRITE_F16)
    return fail(FERRITE_UNSUPPORTED_DTYPE, "%s: teacher dtype %d", op, value_dtype);
  if (index_dtype != 0 && index_dtype != 1)
    return fail(FERRITE_UNSUPPORTED_DTYPE, "%s: index dtype %d (0 = int32, 1 = int64)", op, index_dtype);
  if (!loss) return fail(FERRITE_BAD_SHAPE, "%s: null pointer", op);
  if (workspace_bytes < (size_t)rows * sizeof(float)) return fail(FERRITE_WORKSPACE_TOO_SMALL, "%s: workspace of %zu bytes, %lld needed", op, workspace_bytes, (long long)rows * 4);
  cudaStream_t s = (cudaStream_t)stream;
  if (rows > 0) {
    if (!logits || !values || !indices || !per_token || !workspace) return fail(FERRITE_BAD_SHAPE, "%s: null pointer", op);
    if (misaligned(logits, elem_bytes(dtype)) || (dlogits && misaligned(dlogits, elem_bytes(out_dtype))))
      return fail(FERRITE_BAD_ALIGNMENT, "%s: misaligned pointer", op);
    const RowIn in{logits, rows, vocab, ld, kLog2e / temperature, 1.f / temperature};
    const RowOut out{dlogits, ld_out, dloss, scale};
    const Distill d{values, indices, ld_list, (int)top, value_dtype, index_dtype, weights, 1.f / (float)rows, temperature, workspace, per_token};
    if (int rc = dispatch_row(s, in, out, d, dtype, dlogits ? out_dtype : -1, Distill::shared_bytes((int)top), op)) return rc;
  }
  return sum_terms(s, workspace, loss, rows, 1.f, op);
}

}  // extern "C"
