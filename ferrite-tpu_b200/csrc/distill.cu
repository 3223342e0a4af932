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
constexpr int kSeenWords = 256;

struct Distill {
  static constexpr bool kLogp = false, kEnt = false, kGradEnt = false, kHasStats = false, kList = true, kForwardOnly = false;
  const void* values;   // [rows, top] teacher logits
  const void* indices;  // [rows, top]
  int64_t ld_list;
  int top, value_dtype, index64;
  const float* weights;  // null: 1 / rows
  float uniform, tau;
  float* terms;      // [rows] w * tau^2 * KL
  float* per_token;  // [rows] tau^2 * KL

  struct Pre {
    float w;
  };
  // A row in shared memory: this, then q, the student's logits at the listed tokens, the tokens.
  struct alignas(16) Row {
    uint32_t seen[kSeenWords];  // a bit for each token's hash
    float w;
    float bad;     // NaN if an index is out of range
    int16_t entries;  // 0: a masked row
    int16_t twice;    // a token is listed more than once
  };
  struct List {
    float* q;
    float* x;
    int* idx;
  };
  __host__ __device__ int slot_bytes() const { return (int)sizeof(Row) + top * 12; }
  __device__ List list(char* slot) const {
    List l;
    l.q = reinterpret_cast<float*>(slot + sizeof(Row));
    l.x = l.q + top;
    l.idx = reinterpret_cast<int*>(l.x + top);
    return l;
  }
  // Whether a token is listed more than once.  Each entry sets its token's bit in a table of 2^13
  // hashes; an entry that finds its bit set (a token's second, or a chance hit) is compared with the
  // whole list.  (Comparing every entry with every other took 9 us a row at 128 entries, more than
  // the row itself.)
  __device__ bool any_twice(Row& row, const List& l) const {
    const int lane = threadIdx.x & 31;
    for (int j = lane; j < kSeenWords; j += 32) row.seen[j] = 0;
    __syncwarp();
    bool twice = false;
    for (int j0 = 0; j0 < top; j0 += 32) {
      const int mine = j0 + lane < top ? l.idx[j0 + lane] : -1;
      bool hit = false;
      if (mine >= 0) {
        const uint32_t hash = ((uint32_t)mine * 2654435761u) >> 19, bit = 1u << (hash & 31);
        hit = atomicOr(&row.seen[hash >> 5], bit) & bit;
      }
      for (uint32_t hits = __ballot_sync(0xffffffffu, hit); hits; hits &= hits - 1) {
        const int at = __ffs(hits) - 1, token = __shfl_sync(0xffffffffu, mine, at);
        for (int o = lane; o < top; o += 32) twice |= o != j0 + at && l.idx[o] == token;
      }
    }
    return __any_sync(0xffffffffu, twice);
  }

  __device__ float value(int64_t i) const {
    if (value_dtype == FERRITE_F32) return static_cast<const float*>(values)[i];
    if (value_dtype == FERRITE_BF16) return __bfloat162float(static_cast<const __nv_bfloat16*>(values)[i]);
    return __half2float(static_cast<const __half*>(values)[i]);
  }
  __device__ int64_t index(int64_t i) const {
    return index64 ? static_cast<const int64_t*>(indices)[i] : (int64_t) static_cast<const int32_t*>(indices)[i];
  }
  __device__ Pre pre(int64_t r) const { return Pre{weights ? weights[r] : uniform}; }
  __device__ bool live(const Pre& p) const { return p.w != 0.f; }
  __device__ void dead(int64_t r) const { terms[r] = per_token[r] = 0.f; }

  // The teacher's softmax over the list, and the student's logits there.
  template <typename TI>
  __device__ float prep(int64_t r, const Pre& p, const TI* x, const RowIn& in, char* slot) const {
    const List l = list(slot);
    const int lane = threadIdx.x & 31;
    float m = -INFINITY, bad = 0.f, first = -INFINITY;
    int count = 0;
    // Four entries a lane at a time: their tokens and values are all asked for before the first logit.
    for (int j0 = lane; j0 < top; j0 += 128) {
      int64_t i[4];
      float v[4], xs[4];
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int j = j0 + 32 * q;
        i[q] = j < top ? index(r * ld_list + j) : -1;
        v[q] = j < top ? value(r * ld_list + j) : -INFINITY;
      }
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        if (v[q] == -INFINITY) i[q] = -1;
        if (i[q] >= in.vocab) bad = __int_as_float(0x7fc00000), i[q] = -1;
        xs[q] = i[q] < 0 ? 0.f : DT<TI>::to_f(x[i[q]]);
      }
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int j = j0 + 32 * q;
        if (j >= top) break;
        l.idx[j] = i[q] < 0 ? -1 : (int)i[q];
        l.x[j] = xs[q];
        l.q[j] = v[q];
        if (i[q] >= 0) {
          if (count == 0) first = xs[q];
          ++count;
          m = fmaxf(m, v[q]);  // a NaN value shows through the sums
        }
      }
    }
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) {
      m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, off));
      count += __shfl_xor_sync(0xffffffffu, count, off);
      bad += __shfl_xor_sync(0xffffffffu, bad, off);
      first = fmaxf(first, __shfl_xor_sync(0xffffffffu, first, off));
    }
    float sum = 0.f;
    for (int j = lane; j < top; j += 32) {
      const float y = (l.q[j] - m) * in.k;
      const float e = l.idx[j] >= 0 ? ex2_approx(y) : 0.f;
      l.q[j] = e;
      sum += e;
    }
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, off);
    for (int j = lane; j < top; j += 32) l.q[j] /= sum;
    Row& row = *reinterpret_cast<Row*>(slot);
    __syncwarp();
    const bool twice = any_twice(row, l);
    if (lane == 0) {
      row.w = p.w;
      row.bad = bad;
      row.entries = (int16_t)(bad != bad ? max(count, 1) : count);
      row.twice = twice;
    }
    return base_of(first, in);
  }
  __device__ Coef finish(int64_t, const Norm& w, const RowIn& in, float g, char* slot) const {
    const Row& row = *reinterpret_cast<const Row*>(slot);
    Coef cf;
    const float scale = grad_base(w, in, cf) / w.s;
    const float f = row.w * tau * g + row.bad;
    cf.A = f * scale;
    cf.B = 0.f;
    cf.at_t = -f;  // times a token's weight, added where it is listed
    cf.t = -1;
    cf.masked = row.entries == 0;
    return cf;
  }
  __device__ void results(int64_t r, const Norm& w, const RowIn& in, char* slot) const {
    const List l = list(slot);
    const Row& row = *reinterpret_cast<const Row*>(slot);
    const int lane = threadIdx.x & 31;
    // sum q (log q - log p), each difference taken in f64 before the sum: as the student nears the teacher they are
    // small beside the two logarithms
    const double k = (double)in.k + (double)in.k_lo, ls = (double)log2f(w.s);
    float part = 0.f;
    for (int j = lane; j < top; j += 32)
      if (l.idx[j] >= 0 && l.q[j] != 0.f) {
        const double y = w.big ? (double)(l.x[j] - w.base) * k : fma((double)l.x[j], k, -(double)w.base);
        part = fmaf(l.q[j], (float)((double)log2f(l.q[j]) + (ls - y)), part);
      }
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) part += __shfl_xor_sync(0xffffffffu, part, off);
    if (lane == 0) {
      const float per = row.entries ? tau * tau * kLn2 * part + row.bad : 0.f;
      per_token[r] = per;
      terms[r] = row.entries ? row.w * per : 0.f;
    }
  }
  // The listed tokens' entries, by threads tid < threads.  Where a token is listed twice, the
  // thread of each of its entries sums all their weights, and writes the same value.
  template <typename TO>
  __device__ void fix(const Coef& cf, TO* dx, const RowIn& in, char* slot, int tid, int threads) const {
    const List l = list(slot);
    const bool twice = reinterpret_cast<const Row*>(slot)->twice;
    for (int j = tid; j < top; j += threads) {
      const int i = l.idx[j];
      if (i < 0) continue;  // absent
      float q = l.q[j];
      if (twice) {
        q = 0.f;
        for (int o = 0; o < top; ++o) q += l.idx[o] == i ? l.q[o] : 0.f;
      }
      dx[i] = DT<TO>::from_f(fmaf(cf.at_t, q, grad_of<false>(l.x[j], in.k, cf)));
    }
  }
};

}  // namespace rowloss

FERRITE_DEFINE_STATUS_READER(status_distill)

}  // namespace ferrite

using namespace ferrite;
using namespace ferrite::rowloss;

extern "C" {

int ferrite_distill_loss(void* stream, const void* logits, const void* values, const void* indices, const float* weights, double temperature,
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
    const RowIn in = row_in(logits, rows, vocab, ld, temperature);
    const RowOut out{dlogits, ld_out, dloss, scale};
    const Distill d{values, indices, ld_list, (int)top, value_dtype, index_dtype, weights, 1.f / (float)rows, (float)temperature, workspace, per_token};
    if (int rc = dispatch_row(s, in, out, d, dtype, dlogits ? out_dtype : -1, op)) return rc;
  }
  return sum_terms(s, workspace, loss, rows, 1.f, op);
}

}  // extern "C"
