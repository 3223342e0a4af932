// The kernels that run one row loss (an Op; the mathematics is in rowloss.cuh) over logits
// [rows, vocab].
//
// An Op provides
//   kEnt        the sum of e * y is needed (the entropy's value, or its gradient)
//   kGradEnt    the gradient has the entropy's term
//   kHasStats   the row's state is an input: no first pass
//   kList       the gradient has more single entries than the target's
//   Pre, pre(r), live(pre), dead(r)   masked rows: not read, results and gradient zero
//   slot_bytes()                      shared memory of one row
//   prep(r, pre, x, in, slot)         one warp: what does not need the row's state; returns its base
//   finish(r, norm, in, g, writer, slot)  one warp: the results, written by `writer`; returns the
//                                       gradient's coefficients in every lane
//   state(slot)                       kHasStats: the state that prep loaded
//   fix(...)                          kList: the single entries, after the row is written
#pragma once

#include <atomic>

#include "rowloss.cuh"

namespace ferrite {
namespace rowloss {

// A row of n elements cut into 16-byte vectors: `head` elements up to the first 16-byte boundary, nv
// vectors, and the rest.  It goes by the row's address modulo 16 alone.
template <typename T>
struct RowCut {
  static constexpr int N = 16 / sizeof(T);
  int n, head, nv, tail;
  __device__ __forceinline__ RowCut(const T* x, int n_) : n(n_) {
    head = min(n, (int)(((16 - (reinterpret_cast<uintptr_t>(x) & 15)) & 15) / sizeof(T)));
    nv = (n - head) / N;
    tail = head + nv * N;
  }
};
// Whether N elements of dx starting at column `head` can be stored as one vector.
template <typename TO, int N>
__device__ __forceinline__ bool vector_rows(const TO* dx, int head) {
  return (reinterpret_cast<uintptr_t>(dx + head) & (N * sizeof(TO) - 1)) == 0;
}
template <typename TO, int N>
__device__ __forceinline__ void store_at(TO* p, const float (&d)[N], bool vec) {
  if (vec) {
    store_vec<TO, N>(p, d);
  } else {
#pragma unroll
    for (int j = 0; j < N; ++j) p[j] = DT<TO>::from_f(d[j]);
  }
}

// --------------------------------------------------------------------------
// Any row: one CTA per row, which reads it twice (the second time mostly from L2).  Serves the
// vocabularies whose row does not fit the shared memory of a cluster.
// --------------------------------------------------------------------------

template <class Op, typename TI, typename TO, bool GRAD>
__global__ void __launch_bounds__(512) row_kernel(RowIn in, RowOut out, Op op) {
  extern __shared__ __align__(16) char slot[];
  __shared__ State sh_state[16];
  __shared__ Coef sh_coef;
  constexpr int N = 16 / sizeof(TI);
  pdl_launch_dependents();
  pdl_wait();
  const int64_t r = blockIdx.x;
  const int n = (int)in.vocab, tid = threadIdx.x, nt = blockDim.x, warp = tid >> 5, lane = tid & 31;
  const TI* x = static_cast<const TI*>(in.logits) + r * in.ld;
  TO* dx = GRAD ? static_cast<TO*>(out.dlogits) + r * out.ld : nullptr;
  const auto pre = op.pre(r);
  if (!op.live(pre)) {
    if (tid == 0) op.dead(r);
    if constexpr (GRAD)
      for (int i = tid; i < n; i += nt) dx[i] = DT<TO>::from_f(0.f);
    return;
  }
  __shared__ float sh_base;
  const RowCut<TI> cut(x, n);
  const Pairs2 kk(in);
  if (warp == 0) {
    const float base = op.prep(r, pre, x, in, slot);
    if (lane == 0) sh_base = base;
  }
  __syncthreads();
  State st = empty_state(sh_base);
  if constexpr (!Op::kHasStats) {
    float nc = minus_c(st.m, in);
    for (int v = tid; v < cut.nv; v += nt) {
      float vals[N];
      unpack16<TI>(ld_stream_v4(x + cut.head + v * N), vals);
      push<Op::kEnt>(st, nc, vals, in, kk);
    }
    const int e = tid < cut.head ? tid : tid - cut.head + cut.tail;  // an element before or after the vectors
    if (e < cut.head || (tid >= cut.head && e < n)) {
      const float one[1] = {DT<TI>::to_f(x[e])};
      push<Op::kEnt>(st, nc, one, in, kk);
    }
    st = warp_merge<Op::kEnt>(st, in);
    if (lane == 0) sh_state[warp] = st;
    __syncthreads();
  }
  if (warp == 0) {
    __syncwarp();
    Norm w;
    if constexpr (Op::kHasStats) w = op.state(slot);
    else w = normalise<Op::kEnt>(warp_merge<Op::kEnt>(lane < (nt >> 5) ? sh_state[lane] : empty_state(sh_state[0].m), in), in);
    const float g = GRAD ? (out.dloss ? *out.dloss : 1.f) * out.scale : 0.f;
    const Coef cf = op.finish(r, w, in, g, true, slot);
    if (lane == 0) sh_coef = cf;
  }
  if constexpr (GRAD) {
    __syncthreads();
    const Coef cf = sh_coef;
    if (cf.masked) {
      for (int i = tid; i < n; i += nt) dx[i] = DT<TO>::from_f(0.f);
      return;
    }
    const bool vec = vector_rows<TO, N>(dx, cut.head);
    for (int v = tid; v < cut.nv; v += nt) {
      const int i = cut.head + v * N;
      float vals[N], d[N];
      unpack16<TI>(ld_stream_v4(x + i), vals);
      if (cf.big) grads_of<Op::kGradEnt, true>(vals, d, in.k, cf, kk);
      else grads_of<Op::kGradEnt, false>(vals, d, in.k, cf, kk);
      store_at(dx + i, d, vec);
      if ((unsigned)(cf.t - i) < (unsigned)N) dx[cf.t] = DT<TO>::from_f(cf.at_t);
    }
    const int e = tid < cut.head ? tid : tid - cut.head + cut.tail;
    if (e < cut.head || (tid >= cut.head && e < n))
      dx[e] = DT<TO>::from_f(e == cf.t ? cf.at_t : grad_of<Op::kGradEnt>(DT<TI>::to_f(x[e]), in.k, cf));
    if constexpr (Op::kList) {
      __syncthreads();  // the entries below overwrite what another thread has stored
      op.template fix<TO>(cf, dx, 0, n, in, slot, tid, nt);
    }
  }
}

// --------------------------------------------------------------------------
// Short rows: a warp per row, which reads it twice (the second time from L1).  No barriers; many rows
// in flight hide the latency of each.
// --------------------------------------------------------------------------

constexpr int kShortWarps = 4;                 // rows of a CTA
constexpr int kShortSlots = 48 * 1024;         // shared memory that their ops may take
constexpr int kShortRow = 8192;                // bytes: longer rows go to the kernels for whole CTAs

template <class Op, typename TI, typename TO, bool GRAD>
__global__ void __launch_bounds__(kShortWarps * 32) short_row_kernel(RowIn in, RowOut out, Op op) {
  extern __shared__ __align__(16) char slots[];
  constexpr int N = 16 / sizeof(TI);
  pdl_launch_dependents();
  pdl_wait();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, n = (int)in.vocab;
  char* slot = slots + warp * ((op.slot_bytes() + 15) & ~15);
  const Pairs2 kk(in);
  const float g = GRAD ? (out.dloss ? *out.dloss : 1.f) * out.scale : 0.f;
  for (int64_t r = (int64_t)blockIdx.x * kShortWarps + warp; r < in.rows; r += (int64_t)gridDim.x * kShortWarps) {
    const TI* x = static_cast<const TI*>(in.logits) + r * in.ld;
    TO* dx = GRAD ? static_cast<TO*>(out.dlogits) + r * out.ld : nullptr;
    const RowCut<TI> cut(x, n);
    const bool vec = GRAD && vector_rows<TO, N>(dx, cut.head);
    const int e0 = lane < cut.head ? lane : lane - cut.head + cut.tail;  // an element before or after the vectors
    const int edge = e0 < cut.head || (lane >= cut.head && e0 < n) ? e0 : -1;
    auto zeros = [&]() {
      if constexpr (GRAD) {
        const float zero[N] = {};
        for (int v = lane; v < cut.nv; v += 32) store_at(dx + cut.head + v * N, zero, vec);
        if (edge >= 0) dx[edge] = DT<TO>::from_f(0.f);
      }
    };
    const auto pre = op.pre(r);
    if (!op.live(pre)) {
      if (lane == 0) op.dead(r);
      zeros();
      continue;
    }
    __syncwarp();  // the slot is still being read for the row before
    State st = empty_state(op.prep(r, pre, x, in, slot));
    __syncwarp();
    const float edge_x = edge >= 0 ? DT<TI>::to_f(x[edge]) : 0.f;
    Norm w;
    if constexpr (Op::kHasStats) {
      w = op.state(slot);
    } else {
      float nc = minus_c(st.m, in);
      for (int v = lane; v < cut.nv; v += 32) {
        float vals[N];
        unpack16<TI>(ld_v4(x + cut.head + v * N), vals);
        push<Op::kEnt>(st, nc, vals, in, kk);
      }
      if (edge >= 0) {
        const float one[1] = {edge_x};
        push<Op::kEnt>(st, nc, one, in, kk);
      }
      __syncwarp();
      w = normalise<Op::kEnt>(warp_merge<Op::kEnt>(st, in), in);
    }
    const Coef cf = op.finish(r, w, in, g, true, slot);
    if constexpr (GRAD) {
      if (cf.masked) {
        zeros();
        continue;
      }
      for (int v = lane; v < cut.nv; v += 32) {
        const int i = cut.head + v * N;
        float vals[N], d[N];
        unpack16<TI>(ld_v4(x + i), vals);
        if (cf.big) grads_of<Op::kGradEnt, true>(vals, d, in.k, cf, kk);
        else grads_of<Op::kGradEnt, false>(vals, d, in.k, cf, kk);
        store_at(dx + i, d, vec);
        if ((unsigned)(cf.t - i) < (unsigned)N) dx[cf.t] = DT<TO>::from_f(cf.at_t);
      }
      if (edge >= 0) dx[edge] = DT<TO>::from_f(edge == cf.t ? cf.at_t : grad_of<Op::kGradEnt>(edge_x, in.k, cf));
      if constexpr (Op::kList) {
        __syncwarp();  // the entries below overwrite what another lane has stored
        op.template fix<TO>(cf, dx, 0, n, in, slot, lane, 32);
      }
    }
  }
}

// --------------------------------------------------------------------------
// Rows that fit: one read, one write.
//
// Bound: HBM.  A row is read once into shared memory, and both passes (the sums, then the
// gradient) read it there; so traffic is the logits plus the gradient, and the next bound is the
// ex2 unit (16 a clock and SM: two per element, or one without a gradient).
//
// A persistent cluster of C CTAs, two CTAs to an SM, takes rows cluster, cluster + clusters, ...; each
// CTA holds 1/C of a row.  C is 1 unless a slice does not fit a CTA's shared memory.  In a CTA
//   - kGroups warps, one for each group below, issue untiled bulk copies of 16 KB chunks into a ring
//     (mbarriers full / empty), as far ahead as the ring allows.  The ring is a multiple of kGroups
//     chunks, so that each of its places has one copy warp and one group for good.  (One warp for all
//     of them takes about 600 cycles a copy -- its waits and its issue, one after the other -- and
//     held reads to 3.7 TB/s with 8 KB copies.)
//   - kGroups groups of four warps (one to each of the SM's quarters) run the passes, each on chunks
//     of its own in turn: the sums of a row as its chunks land, then its gradient from the resident
//     chunks, released one by one;
//   - what comes between a row's two passes is the work of kHelpers warps, rows in turn: fetch what
//     the row's loss needs besides the logits (ahead of time), merge the passes' states (and the C
//     CTAs', through distributed shared memory, in rank order), write the row's results, hand back
//     the gradient's coefficients, and at last write the single entries of a list.
// While one CTA of an SM waits for its helper, the other's passes have the SM.  (One CTA of twice the
// warps with the gradient a row behind the sums also hides that wait, but pays the fixed part of a
// row, some 2000 cycles, in twice the warps: 222 us against this form's for 8192 x 32000 bf16.)
// Every wait is bounded; an expired one raises the CTA's abort flag and the status word, after which
// no copy is issued, nobody waits, and the copies in flight are waited for before the CTA exits.
// --------------------------------------------------------------------------

constexpr int kGroups = 2;
constexpr int kGroup = 128;                     // threads of a group
constexpr int kPass = kGroups * kGroup;         // threads of the passes
constexpr int kWarps = kPass / 32;
constexpr int kHelpers = 2;
constexpr int kRingThreads = kPass + kGroups * 32 + kHelpers * 32;
constexpr int kChunk = 16384;                   // bytes
constexpr int kChunkVec = kChunk / 16;
constexpr int kVecPer = kChunkVec / kGroup;     // vectors a thread takes of a chunk
constexpr int kMaxChunks = 6;
static_assert(kMaxChunks % kGroups == 0 && kMaxChunks <= 32, "places of one group each; a bit for each place");
constexpr int kRingCluster = 8;

struct RingShared {
  uint64_t full[kMaxChunks], empty[kMaxChunks];
  // of a helper's row: its base is there; the passes' states are; its coefficients are; its
  // gradient is written; the other CTAs' states are there
  // (two places in turn: a CTA that is a whole turn of the helpers ahead must not reach into a
  // place that another still reads)
  uint64_t ready[kHelpers], states[kHelpers], done[kHelpers], written[kHelpers], peers[kHelpers][2];
  State warp_state[kHelpers][kWarps];
  State peer_state[kHelpers][2][kRingCluster];
  alignas(16) Coef coef[kHelpers];
  float base[kHelpers];
  int abort;
};
constexpr int kRingHeader = (int)((sizeof(RingShared) + 127) / 128 * 128);

__device__ __forceinline__ bool mbar_try_wait_cluster(uint64_t* bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(ok)
      : "r"(smem_u32(bar)), "r"(parity)
      : "memory");
  return ok != 0;
}
// The bounded wait of common.cuh for warps that run ahead of the passes: it sleeps between tries, so
// that it takes no issue slots from them.  CLUSTER: other CTAs of the cluster arrive on the barrier.
template <bool CLUSTER = false>
__device__ __forceinline__ bool wait_idle(uint64_t* bar, uint32_t parity, volatile int* abort, int where) {
  if (CLUSTER ? mbar_try_wait_cluster(bar, parity) : mbar_try_wait(bar, parity)) return true;
  const uint64_t t0 = globaltimer_ns();
  while (!(CLUSTER ? mbar_try_wait_cluster(bar, parity) : mbar_try_wait(bar, parity))) {
    if (*abort) return false;
    if (globaltimer_ns() - t0 > kWaitLimitNs) {
      report_timeout(where);
      *abort = 1;
      return false;
    }
    __nanosleep(40);
  }
  return true;
}
__device__ __forceinline__ void st_cluster(uint32_t addr, float v) {
  asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(addr), "f"(v) : "memory");
}

// A row as one CTA of the cluster sees it: its slice of the vectors, and (first and last CTA) the
// elements before and after them.  Kept from row to row while the rows' addresses agree modulo 16.
template <typename T>
struct Slice {
  int n, rank, lg, phase;
  int head, tail, col0, nv, chunks;
  __device__ __forceinline__ Slice(int n_, int rank_, int lg_) : n(n_), rank(rank_), lg(lg_), phase(-1) {}
  __device__ __forceinline__ void at(const T* x) {
    const int p = (int)(reinterpret_cast<uintptr_t>(x) & 15);
    if (p == phase) return;
    phase = p;
    const RowCut<T> cut(x, n);
    const int per = (cut.nv + (1 << lg) - 1) >> lg, v0 = min(rank * per, cut.nv);
    head = cut.head;
    tail = cut.tail;
    nv = min(per, cut.nv - v0);
    col0 = cut.head + v0 * RowCut<T>::N;
    chunks = (nv + kChunkVec - 1) / kChunkVec;
  }
  __device__ __forceinline__ bool first() const { return rank == 0; }
  __device__ __forceinline__ bool last() const { return rank == (1 << lg) - 1; }
  __device__ __forceinline__ int lo() const { return first() ? 0 : col0; }
  __device__ __forceinline__ int hi() const { return last() ? n : col0 + nv * RowCut<T>::N; }
  // the column of the element outside the vectors that thread tid takes, or -1
  __device__ __forceinline__ int edge(int tid) const {
    if (tid >= 32 || (head == 0 && tail == n)) return -1;
    if (first() && tid < head) return tid;
    const int e = tail + tid - 16;
    return last() && tid >= 16 && e < n ? e : -1;
  }
};

// Which of the rows r, r + step, ... are live, asked row by row by a whole warp: 32 rows' masks are
// fetched at a time, so that a row's own is never waited for.
template <class Op>
struct LiveRows {
  const Op& op;
  int64_t rows, step;
  uint32_t mask = 0;
  int left = 0;
  __device__ __forceinline__ bool next(int64_t r) {
    if (left == 0) {
      const int64_t q = r + (int64_t)(threadIdx.x & 31) * step;
      mask = __ballot_sync(0xffffffffu, q < rows && op.live(op.pre(q)));
      left = 32;
    }
    const bool live = mask & 1u;
    mask >>= 1;
    --left;
    return live;
  }
};

// A place in the ring, and the parity of its current use.
struct Place {
  int at = 0;
  uint32_t parity = 0;
  __device__ __forceinline__ void next(int size, int n = 1) {
    while (n > size) {
      n -= size;
      parity ^= 1;
    }
    at += n;
    if (at >= size) {
      at -= size;
      parity ^= 1;
    }
  }
};

template <class Op, typename TI, typename TO, bool GRAD>
__global__ void __launch_bounds__(kRingThreads, 2) ring_kernel(RowIn in, RowOut out, Op op, int ring_chunks, int lg_cluster, int twice) {
  constexpr int N = 16 / sizeof(TI);
  constexpr bool kSums = !Op::kHasStats;        // a first pass
  constexpr bool kBoth = GRAD && kSums;         // both passes
  constexpr bool kFix = GRAD && Op::kList;
  extern __shared__ __align__(128) char smem[];
  RingShared& sh = *reinterpret_cast<RingShared*>(smem);
  char* ring = smem + kRingHeader;
  const int slot_bytes = (op.slot_bytes() + 15) & ~15;
  char* slots = ring + (size_t)ring_chunks * kChunk;
  volatile int* abort = &sh.abort;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int cluster = 1 << lg_cluster;
  const int rank = cluster > 1 ? (int)cluster_ctarank() : 0;
  const int n = (int)in.vocab;
  const int64_t step = gridDim.x >> lg_cluster, r0 = blockIdx.x >> lg_cluster;
  if (tid == 0) {
    for (int i = 0; i < ring_chunks; ++i) {
      mbar_init(&sh.full[i], 1);
      mbar_init(&sh.empty[i], kGroup / 32);
    }
    for (int i = 0; i < kHelpers; ++i) {
      mbar_init(&sh.ready[i], 1);
      mbar_init(&sh.states[i], kWarps);
      mbar_init(&sh.done[i], 1);
      mbar_init(&sh.written[i], kWarps);
      mbar_init(&sh.peers[i][0], cluster);
      mbar_init(&sh.peers[i][1], cluster);
    }
    sh.abort = 0;
    fence_mbar_init();
  }
  pdl_launch_dependents();
  __syncthreads();
  if (cluster > 1) cluster_sync_all();  // the peers' barriers are ready
  pdl_wait();

  LiveRows<Op> rows{op, in.rows, step};
  Slice<TI> sl(n, rank, lg_cluster);
  // registers go where the passes need them: 256 x 88 + 128 x 64 = 384 x 80 of the launch
  if (warp >= kWarps) {
  setmaxnreg_dec<64>();
  if (warp < kWarps + kGroups) {  // ---- copies of one group's chunks
    const int group = warp - kWarps;
    Place p;
    int k = 0;  // which group has the row's first chunk
    uint32_t used = 0, last_parity = 0;  // bit c: place c has held a copy, and the last one's parity
    bool stop = false;
    for (int64_t r = r0; r < in.rows; r += step) {
      if (!rows.next(r)) continue;
      const TI* x = static_cast<const TI*>(in.logits) + r * in.ld;
      sl.at(x);
      for (int pass = 0; pass <= (kBoth ? twice : 0); ++pass) {
      const int c0 = (group - k + kGroups) % kGroups;
      Place at = p;
      at.next(ring_chunks, c0);
      p.next(ring_chunks, sl.chunks);
      k = (k + sl.chunks) % kGroups;
      if (lane != 0 || stop) continue;
      const char* src = reinterpret_cast<const char*>(x + sl.col0) + c0 * kChunk;
      int left = sl.nv - c0 * kChunkVec;
      for (int c = c0; c < sl.chunks; c += kGroups) {
        // a chunk's first use waits for the barrier's phase before the first: no wait
        if (!wait_idle(&sh.empty[at.at], at.parity ^ 1, abort, 201)) {
          stop = true;
          break;
        }
        const uint32_t bytes = (uint32_t)min(left, kChunkVec) * 16u;
        mbar_arrive_expect_tx(&sh.full[at.at], bytes);
        bulk_load(ring + (size_t)at.at * kChunk, src, bytes, &sh.full[at.at]);
        used |= 1u << at.at;
        last_parity = (last_parity & ~(1u << at.at)) | (at.parity << at.at);
        at.next(ring_chunks, kGroups);
        src += kGroups * kChunk;
        left -= kGroups * kChunkVec;
      }
      }
    }
    // the last copy into each chunk has landed before the CTA gives up its shared memory
    if (lane == 0) {
      for (int j = 0; j < ring_chunks; ++j) {
        if (!(used >> j & 1)) continue;
        const uint64_t t0 = globaltimer_ns();
        while (!mbar_try_wait(&sh.full[j], last_parity >> j & 1))
          if (globaltimer_ns() - t0 > kWaitLimitNs) {
            report_timeout(202);
            *abort = 1;
            break;
          }
      }
    }
  } else {  // ---- what lies between a row's two passes
    const int h = warp - kWarps - kGroups;
    char* slot = slots + h * slot_bytes;
    const float g = GRAD ? (out.dloss ? *out.dloss : 1.f) * out.scale : 0.f;
    int turn = 0;
    uint32_t parity = 0, half = 0, half_parity = 0;  // of this helper's barriers; which of the two peers' places
    for (int64_t r = r0; r < in.rows; r += step) {
      if (!rows.next(r)) continue;
      const bool my_turn = turn == h;
      if (++turn == kHelpers) turn = 0;
      if (!my_turn) continue;
      const TI* x = static_cast<const TI*>(in.logits) + r * in.ld;
      const float base = op.prep(r, op.pre(r), x, in, slot);
      __syncwarp();
      Norm w;
      if constexpr (kSums) {
        if (lane == 0) {
          sh.base[h] = base;
          mbar_arrive(&sh.ready[h]);
        }
        (void)wait_idle(&sh.states[h], parity, abort, 203);
        __syncwarp();
        State st = warp_merge<Op::kEnt>(lane < kWarps ? sh.warp_state[h][lane] : empty_state(sh.warp_state[h][0].m), in);
        if (cluster > 1) {
          if (lane < cluster) {
            const uint32_t to = mapa_shared(&sh.peer_state[h][half][rank], lane);
            st_cluster(to, st.m);
            st_cluster(to + 4, st.s);
            st_cluster(to + 8, st.u);
            mbar_arrive_cluster(mapa_shared(&sh.peers[h][half], lane));
          }
          (void)wait_idle<true>(&sh.peers[h][half], half_parity, abort, 204);
          __syncwarp();
          st = warp_merge<Op::kEnt>(lane < cluster ? sh.peer_state[h][half][lane] : empty_state(sh.peer_state[h][half][0].m), in);
          half_parity ^= half;
          half ^= 1;
        }
        w = normalise<Op::kEnt>(st, in);
      } else {
        w = op.state(slot);
      }
      const Coef cf = op.finish(r, w, in, g, rank == 0, slot);
      if constexpr (!kSums) {
        // the passes have read the coefficients of the row before in this place
        (void)wait_idle(&sh.written[h], parity ^ 1, abort, 205);
        __syncwarp();
      }
      if (lane == 0) {
        sh.coef[h] = cf;
        mbar_arrive(&sh.done[h]);
      }
      if constexpr (kFix) {
        (void)wait_idle(&sh.written[h], parity, abort, 206);
        __syncwarp();
        if (!cf.masked) {
          sl.at(x);
          op.template fix<TO>(cf, static_cast<TO*>(out.dlogits) + r * out.ld, sl.lo(), sl.hi(), in, slot, lane, 32);
        }
        __syncwarp();
      }
      parity ^= 1;
    }
  }
  } else {  // ---- the passes
    setmaxnreg_inc<88>();
    const Pairs2 kk(in);
    const int group = warp / (kGroup / 32), gtid = tid % kGroup;
    Place p1, p2, slot1, slot2;  // chunks and helpers of the first and the second pass
    int k1 = 0, k2 = 0;          // which group has a row's first chunk
    // the second pass of row r: its gradient, from the chunks at p2
    auto second = [&](int64_t r) {
      const TI* x = static_cast<const TI*>(in.logits) + r * in.ld;
      sl.at(x);
      TO* dx = static_cast<TO*>(out.dlogits) + r * out.ld;
      const int col0 = sl.col0, edge = sl.edge(tid);
      const bool vec = vector_rows<TO, N>(dx, sl.head);
      const float edge_x = edge >= 0 ? DT<TI>::to_f(x[edge]) : 0.f;
      (void)mbar_wait(&sh.done[slot2.at], slot2.parity, abort, 207);
      const Coef cf = sh.coef[slot2.at];
      const int k2_row = k2, c0 = (group - k2 + kGroups) % kGroups;  // this group's first chunk of the row
      Place at = p2;
      p2.next(ring_chunks, sl.chunks);
      k2 = (k2 + sl.chunks) % kGroups;
      at.next(ring_chunks, c0);
      // What is the same for a whole row is decided here, not vector by vector.
      auto chunks = [&](auto usual_row) {
        constexpr bool kUsual = decltype(usual_row)::value;
        int left = sl.nv - c0 * kChunkVec - gtid;
        TO* to = dx + col0 + (c0 * kChunkVec + gtid) * N;
        for (int c = c0; c < sl.chunks; c += kGroups) {
          if (!kSums || twice) (void)mbar_wait(&sh.full[at.at], at.parity, abort, 208);
          const uint4* p = reinterpret_cast<const uint4*>(ring + (size_t)at.at * kChunk) + gtid;
          if constexpr (kUsual) {  // all of the thread's vectors, side by side
            uint4 raw[kVecPer];
#pragma unroll
            for (int q = 0; q < kVecPer; ++q) raw[q] = p[q * kGroup];
            __syncwarp();
            if (lane == 0) mbar_arrive(&sh.empty[at.at]);
#pragma unroll
            for (int q = 0; q < kVecPer; ++q) {
              float vals[N], d[N];
              unpack16<TI>(raw[q], vals);
              grads_of<Op::kGradEnt, false>(vals, d, in.k, cf, kk);
              if (q * kGroup < left) store_vec<TO, N>(to + q * kGroup * N, d);
            }
          } else {
#pragma unroll 1
            for (int q = 0; q < kVecPer; ++q)
              if (q * kGroup < left) {
                float vals[N], d[N];
                unpack16<TI>(p[q * kGroup], vals);
                if (cf.masked) {
#pragma unroll
                  for (int j = 0; j < N; ++j) d[j] = 0.f;
                } else if (cf.big) {
                  grads_of<Op::kGradEnt, true>(vals, d, in.k, cf, kk);
                } else {
                  grads_of<Op::kGradEnt, false>(vals, d, in.k, cf, kk);
                }
                store_at(to + q * kGroup * N, d, vec);
              }
            __syncwarp();
            if (lane == 0) mbar_arrive(&sh.empty[at.at]);
          }
          at.next(ring_chunks, kGroups);
          left -= kGroups * kChunkVec;
          to += kGroups * kChunkVec * N;
        }
      };
      if (vec && !cf.big && !cf.masked) chunks(std::true_type());
      else chunks(std::false_type());
      if (edge >= 0) dx[edge] = DT<TO>::from_f(cf.masked ? 0.f : edge == cf.t ? cf.at_t : grad_of<Op::kGradEnt>(edge_x, in.k, cf));
      // the target's entry, by the thread that has stored the vector it lies in
      const int tv = (cf.t - col0) / N;
      if (cf.t >= col0 && tv < sl.nv && tv % kGroup == gtid && (tv / kChunkVec + k2_row) % kGroups == group) dx[cf.t] = DT<TO>::from_f(cf.at_t);
      if constexpr (kFix || !kSums) {
        __syncwarp();
        if (lane == 0) mbar_arrive(&sh.written[slot2.at]);
      }
      slot2.next(kHelpers);
    };
    // the first pass of row r: its sums
    auto first = [&](int64_t r) {
      const TI* x = static_cast<const TI*>(in.logits) + r * in.ld;
      sl.at(x);
      const int edge = sl.edge(tid);
      const float edge_x = edge >= 0 ? DT<TI>::to_f(x[edge]) : 0.f;
      (void)mbar_wait(&sh.ready[slot1.at], slot1.parity, abort, 211);
      State st = empty_state(sh.base[slot1.at]);
      float nc = minus_c(st.m, in);
      // What stands for the elements past the row's end in its last chunk: nothing of the sums.  -inf,
      // but in 0 * y where the entropy is summed -1e30; f16 has none that is small enough for every
      // temperature, and sums such a chunk vector by vector.
      constexpr bool kPad = !Op::kEnt || !std::is_same_v<TI, __half>;
      const uint32_t pad = std::is_same_v<TI, float> ? (Op::kEnt ? 0xf149f2cau : 0xff800000u)
                           : std::is_same_v<TI, __half> ? 0xfc00fc00u : (Op::kEnt ? 0xf149f149u : 0xff80ff80u);
      const int c0 = (group - k1 + kGroups) % kGroups;
      Place at = p1;
      p1.next(ring_chunks, sl.chunks);
      k1 = (k1 + sl.chunks) % kGroups;
      at.next(ring_chunks, c0);
      int left = sl.nv - c0 * kChunkVec - gtid;
      for (int c = c0; c < sl.chunks; c += kGroups) {
        (void)mbar_wait(&sh.full[at.at], at.parity, abort, 209);
        const uint4* p = reinterpret_cast<const uint4*>(ring + (size_t)at.at * kChunk) + gtid;
        bool by_one = true;
        if (kPad || (kVecPer - 1) * kGroup < left) {  // all of the thread's vectors at once, one check for them
          uint4 raw[kVecPer];
#pragma unroll
          for (int q = 0; q < kVecPer; ++q) {
            raw[q] = p[q * kGroup];  // past the row's end: whatever the chunk holds
            if (kPad && q * kGroup >= left) raw[q] = make_uint4(pad, pad, pad, pad);
          }
          uint64_t s2 = f2_make(0.f, 0.f), u2 = s2;
#pragma unroll
          for (int q = 0; q < kVecPer; ++q) {
            float vals[N];
            unpack16<TI>(raw[q], vals);
            sum_usual<Op::kEnt>(s2, u2, vals, nc, kk);
          }
          const float s = f2_lo(s2) + f2_hi(s2), u = Op::kEnt ? f2_lo(u2) + f2_hi(u2) : 0.f;
          if (usual<Op::kEnt>(s, u)) {
            st.s += s;
            if constexpr (Op::kEnt) st.u += u;
            by_one = false;
          }
        }
        if (by_one) {
#pragma unroll 1
          for (int q = 0; q < kVecPer; ++q)
            if (q * kGroup < left) {
              float vals[N];
              unpack16<TI>(p[q * kGroup], vals);
              push<Op::kEnt>(st, nc, vals, in, kk);
            }
        }
        if (!kBoth || twice) {
          __syncwarp();
          if (lane == 0) mbar_arrive(&sh.empty[at.at]);
        }
        at.next(ring_chunks, kGroups);
        left -= kGroups * kChunkVec;
      }
      if (edge >= 0) {
        const float one[1] = {edge_x};
        push<Op::kEnt>(st, nc, one, in, kk);
      }
      __syncwarp();
      st = warp_merge<Op::kEnt>(st, in);
      // without a gradient nothing else holds the passes back until the helper has read the
      // states of the row before in this place
      if constexpr (!kBoth) (void)mbar_wait(&sh.done[slot1.at], slot1.parity ^ 1, abort, 210);
      if (lane == 0) {
        sh.warp_state[slot1.at][warp] = st;
        mbar_arrive(&sh.states[slot1.at]);
      }
      slot1.next(kHelpers);
    };
    for (int64_t r = r0; r < in.rows; r += step) {
      if (!rows.next(r)) {  // masked
        if (tid == 0 && rank == 0) op.dead(r);
        if constexpr (GRAD) {
          TO* dx = static_cast<TO*>(out.dlogits) + r * out.ld;
          sl.at(static_cast<const TI*>(in.logits) + r * in.ld);
          const bool vec = vector_rows<TO, N>(dx, sl.head);
          const float zero[N] = {};
          for (int v = tid; v < sl.nv; v += kPass) store_at(dx + sl.col0 + v * N, zero, vec);
          const int edge = sl.edge(tid);
          if (edge >= 0) dx[edge] = DT<TO>::from_f(0.f);
        }
        continue;
      }
      if constexpr (kSums) first(r);
      if constexpr (GRAD) {
        if (kSums && twice) {
          p2 = p1;
          k2 = k1;
        }
        second(r);
        if (kSums && twice) {
          p1 = p2;
          k1 = k2;
        }
      }
    }
  }
  __syncwarp();
  if (cluster > 1) cluster_sync_all();  // nobody leaves while a peer may still write here
}

// --------------------------------------------------------------------------
// host
// --------------------------------------------------------------------------

constexpr int kRingSmem = (227 - 2) * 1024 / 2 / 128 * 128;  // of each of two CTAs, besides what the system keeps
constexpr int kMaxSlots = kHelpers * (2048 + 12 * 1024);  // the helpers' lists at their longest

// How rows are split: chunks of each CTA's ring, log2 of the CTAs per row (-1: the row does not fit).
// The split goes by the row's length and type alone, not by how many rows there are, with a gradient
// or without: so a row's results have the same bits in every call (log-probabilities taken in one
// batch and compared in another differ by nothing), as long as it starts on a 16-byte boundary.
struct RingPlan {
  int chunks, lg_cluster, twice;
  size_t smem;
};
inline RingPlan plan_ring(int64_t vocab, int elem, int slot_bytes) {
  RingPlan p{};
  const int slots = kHelpers * ((slot_bytes + 15) & ~15);
  p.chunks = (kRingSmem - kRingHeader - slots) / kChunk;
  if (p.chunks > kMaxChunks) p.chunks = kMaxChunks;
  p.chunks -= p.chunks % kGroups;
  p.smem = (size_t)kRingHeader + (size_t)p.chunks * kChunk + slots;
  // a slice is resident, beside lists of up to 1024 entries (short ones leave two more chunks, for the next row)
  const int64_t most = (int64_t)((kRingSmem - kRingHeader - kMaxSlots) / kChunk / kGroups * kGroups) * kChunk;
  const int64_t bytes = vocab * elem;
  int lg = 0;
  while ((1 << lg) < kRingCluster && ((bytes + 15) >> lg) + 16 > most) ++lg;
  p.lg_cluster = ((bytes + 15) >> lg) + 16 > most ? -1 : lg;
  if (lg > 0) p.twice = 1, p.lg_cluster = 0;
  return p;
}

inline int row_threads(int64_t vocab) { return vocab <= 4096 ? 128 : vocab <= 16384 ? 256 : 512; }

template <class Op, typename TI, typename TO, bool GRAD>
static int launch_row(cudaStream_t s, const RowIn& in, const RowOut& out, const Op& op, const char* name) {
  const int dev = current_device();
  if (dev < 0 || dev >= 64) return fail(FERRITE_LAUNCH_FAILED, "%s: device ordinal %d", name, dev);
  cudaError_t e;
  const RingPlan p = plan_ring(in.vocab, sizeof(TI), op.slot_bytes());
  const int64_t bytes = in.vocab * (int64_t)sizeof(TI);
  const int slots = kShortWarps * ((op.slot_bytes() + 15) & ~15);
  if (bytes < kShortRow && slots <= kShortSlots) {
    const int64_t ctas = (in.rows + kShortWarps - 1) / kShortWarps, most = (int64_t)num_sms(dev) * 16;
    e = launch_pdl(short_row_kernel<Op, TI, TO, GRAD>, dim3((unsigned)(ctas < most ? ctas : most)), dim3(kShortWarps * 32), slots, s, in, out, op);
  } else if (bytes >= kShortRow && p.lg_cluster >= 0) {
    auto kern = ring_kernel<Op, TI, TO, GRAD>;
    // clusters of each size that are resident at once, per device (set once; racing first calls
    // store the same values): a persistent grid of more would run its last ones after the others
    static std::atomic<int> resident[64][4];
    int clusters = resident[dev][p.lg_cluster].load(std::memory_order_relaxed);
    if (clusters == 0) {
      e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, kRingSmem);
      if (e != cudaSuccess) return fail(FERRITE_LAUNCH_FAILED, "%s: shared memory attribute: %s", name, cudaGetErrorString(e));
      clusters = max_active_clusters((const void*)kern, dim3(kRingThreads), kRingSmem, 1u << p.lg_cluster);
      if (clusters < 1) clusters = 1;
      resident[dev][p.lg_cluster].store(clusters, std::memory_order_relaxed);
    }
    const int64_t used = in.rows < clusters ? in.rows : clusters;
    e = launch_pdl_cluster(kern, dim3((unsigned)(used << p.lg_cluster)), dim3(kRingThreads), p.smem, s, 1u << p.lg_cluster, in, out, op,
                           p.chunks, p.lg_cluster, p.twice);
  } else {
    e = launch_pdl(row_kernel<Op, TI, TO, GRAD>, dim3((unsigned)in.rows), dim3(row_threads(in.vocab)), op.slot_bytes(), s, in, out, op);
  }
  if (e != cudaSuccess) return fail(FERRITE_LAUNCH_FAILED, "%s: %s", name, cudaGetErrorString(e));
  return check_launch(name);
}

// Dispatch on the logits' and the gradient's type (out_dtype < 0: forward only).
template <class Op>
static int dispatch_row(cudaStream_t s, const RowIn& in, const RowOut& out, const Op& op, int dtype, int out_dtype, const char* name) {
  if (out_dtype < 0) {
    if constexpr (Op::kHasStats) {
      return fail(FERRITE_BAD_SHAPE, "%s: no gradient asked for", name);
    } else {
      if (dtype == FERRITE_F32) return launch_row<Op, float, float, false>(s, in, out, op, name);
      if (dtype == FERRITE_BF16) return launch_row<Op, __nv_bfloat16, __nv_bfloat16, false>(s, in, out, op, name);
      return launch_row<Op, __half, __half, false>(s, in, out, op, name);
    }
  }
  if constexpr (Op::kForwardOnly) {
    return fail(FERRITE_BAD_SHAPE, "%s: no gradient to write", name);
  } else {
    if (dtype == FERRITE_BF16) return launch_row<Op, __nv_bfloat16, __nv_bfloat16, true>(s, in, out, op, name);
    if (dtype == FERRITE_F16) return launch_row<Op, __half, __half, true>(s, in, out, op, name);
    if (out_dtype == FERRITE_F32) return launch_row<Op, float, float, true>(s, in, out, op, name);
    if (out_dtype == FERRITE_BF16) return launch_row<Op, float, __nv_bfloat16, true>(s, in, out, op, name);
    return launch_row<Op, float, __half, true>(s, in, out, op, name);
  }
}

}  // namespace rowloss
}  // namespace ferrite
