// The kernel that runs one row loss (an Op, see rowloss.cuh for the mathematics) over
// logits [rows, vocab]: one CTA per row, one pass for (m, s, u), a block merge, and a
// second pass over the same row (by then in L2) that writes the gradient.
//
// An Op provides
//   kEnt        whether the sum of e * y is needed for the gradient or the entropy
//   kHasStats   the row's state is an input (no first pass)
//   live(r)     false: the row is masked -- it is not read, its results are zeros
//   dead(r)     writes a masked row's results (one thread)
//   begin(...)  what can start before the row's state is known (all threads)
//   finish(...) the row's results from its state; returns the gradient's coefficients (all threads)
//   fix(...)    the gradient entries that are not e (A + B y): after the row is written
#pragma once

#include "rowloss.cuh"

namespace ferrite {
namespace rowloss {

// Calls f(i, vals) for every vector of N = 16 / sizeof(T) elements of x[0, n) whose address is
// a multiple of 16, and g(i, x_i) for the elements before and after those, over the CTA's threads.
template <typename T, typename F, typename G>
__device__ __forceinline__ void for_row(const T* x, int n, F&& f, G&& g) {
  constexpr int N = 16 / sizeof(T);
  const int head = min(n, (int)(((16 - (reinterpret_cast<uintptr_t>(x) & 15)) & 15) / sizeof(T)));
  const int nv = (n - head) / N;
  const int tail = head + nv * N;
  const int tid = threadIdx.x;
  for (int v = tid; v < nv; v += blockDim.x) {
    const int i = head + v * N;
    float vals[N];
    unpack16<T>(ld_stream_v4(x + i), vals);
    f(i, vals);
  }
  if (tid < head) g(tid, DT<T>::to_f(x[tid]));
  if (tid < n - tail) g(tail + tid, DT<T>::to_f(x[tail + tid]));
}

template <bool ENT>
__device__ __forceinline__ State block_merge(State st, float k, State* sh) {
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) {
    State o;
    o.m = __shfl_xor_sync(0xffffffffu, st.m, off);
    o.s = __shfl_xor_sync(0xffffffffu, st.s, off);
    o.u = ENT ? __shfl_xor_sync(0xffffffffu, st.u, off) : 0.f;
    merge<ENT>(st, o, k);
  }
  if ((threadIdx.x & 31) == 0) sh[threadIdx.x >> 5] = st;
  __syncthreads();
  st = sh[0];
  for (int w = 1; w < (int)(blockDim.x >> 5); ++w) merge<ENT>(st, sh[w], k);
  return st;
}

template <class Op, typename TI, typename TO, bool GRAD>
__global__ void __launch_bounds__(512) row_kernel(RowIn in, RowOut out, Op op) {
  extern __shared__ __align__(16) char sh_op[];
  __shared__ State sh_state[16];
  pdl_launch_dependents();
  pdl_wait();
  const int64_t r = blockIdx.x;
  const int n = (int)in.vocab;
  const TI* x = static_cast<const TI*>(in.logits) + r * in.ld;
  TO* dx = GRAD ? static_cast<TO*>(out.dlogits) + r * out.ld : nullptr;
  if (!op.live(r)) {
    if (threadIdx.x == 0) op.dead(r);
    if constexpr (GRAD)
      for (int i = threadIdx.x; i < n; i += blockDim.x) dx[i] = DT<TO>::from_f(0.f);
    return;
  }
  op.begin(r, x, n, sh_op);
  State st = empty_state();
  if constexpr (Op::kHasStats) {
    st = op.state(r, in.k);
  } else {
    for_row<TI>(
        x, n, [&](int, const float(&v)[16 / sizeof(TI)]) { push<Op::kEnt>(st, v, in.k); },
        [&](int, float v) {
          const float one[1] = {v};
          push<Op::kEnt>(st, one, in.k);
        });
    st = block_merge<Op::kEnt>(st, in.k, sh_state);
  }
  const float g = GRAD ? (out.dloss ? *out.dloss : 1.f) * out.scale : 0.f;
  const Coef cf = op.finish(r, st, x, in, g, true, sh_op);
  if constexpr (GRAD) {
    if (cf.masked) {
      for (int i = threadIdx.x; i < n; i += blockDim.x) dx[i] = DT<TO>::from_f(0.f);
      return;
    }
    constexpr int N = 16 / sizeof(TI);
    const float c = st.m * in.k;
    const bool big = is_big(c);
    const int head = (int)(((16 - (reinterpret_cast<uintptr_t>(x) & 15)) & 15) / sizeof(TI));
    const bool vec = (reinterpret_cast<uintptr_t>(dx + head) & (N * sizeof(TO) - 1)) == 0;
    for_row<TI>(
        x, n,
        [&](int i, const float(&v)[N]) {
          float d[N];
#pragma unroll
          for (int j = 0; j < N; ++j) d[j] = grad_of<Op::kGradEnt>(v[j], in.k, st.m, c, big, cf.A, cf.B);
          if (vec) {
            store_vec<TO, N>(dx + i, d);
          } else {
#pragma unroll
            for (int j = 0; j < N; ++j) dx[i + j] = DT<TO>::from_f(d[j]);
          }
        },
        [&](int i, float v) { dx[i] = DT<TO>::from_f(grad_of<Op::kGradEnt>(v, in.k, st.m, c, big, cf.A, cf.B)); });
    __syncthreads();  // the entries below overwrite what another thread has stored
    op.template fix<TO>(r, st, cf, dx, 0, n, x, in, g, sh_op);
  }
}

inline int row_threads(int64_t vocab) { return vocab <= 1024 ? 64 : vocab <= 4096 ? 128 : vocab <= 16384 ? 256 : 512; }

template <class Op, typename TI, typename TO, bool GRAD>
static int launch_row(cudaStream_t s, const RowIn& in, const RowOut& out, const Op& op, size_t smem, const char* name) {
  const cudaError_t e = launch_pdl(row_kernel<Op, TI, TO, GRAD>, dim3((unsigned)in.rows), dim3(row_threads(in.vocab)), smem, s, in, out, op);
  if (e != cudaSuccess) return fail(FERRITE_LAUNCH_FAILED, "%s: %s", name, cudaGetErrorString(e));
  return check_launch(name);
}

// Dispatch on the logits' and the gradient's type (out_dtype < 0: forward only).
template <class Op>
static int dispatch_row(cudaStream_t s, const RowIn& in, const RowOut& out, const Op& op, int dtype, int out_dtype, size_t smem,
                        const char* name) {
  if (out_dtype < 0) {
    if (dtype == FERRITE_F32) return launch_row<Op, float, float, false>(s, in, out, op, smem, name);
    if (dtype == FERRITE_BF16) return launch_row<Op, __nv_bfloat16, __nv_bfloat16, false>(s, in, out, op, smem, name);
    return launch_row<Op, __half, __half, false>(s, in, out, op, smem, name);
  }
  if (dtype == FERRITE_BF16) return launch_row<Op, __nv_bfloat16, __nv_bfloat16, true>(s, in, out, op, smem, name);
  if (dtype == FERRITE_F16) return launch_row<Op, __half, __half, true>(s, in, out, op, smem, name);
  if (out_dtype == FERRITE_F32) return launch_row<Op, float, float, true>(s, in, out, op, smem, name);
  if (out_dtype == FERRITE_BF16) return launch_row<Op, float, __nv_bfloat16, true>(s, in, out, op, smem, name);
  return launch_row<Op, float, __half, true>(s, in, out, op, smem, name);
}

}  // namespace rowloss
}  // namespace ferrite
