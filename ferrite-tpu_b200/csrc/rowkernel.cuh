// The kernels that run one row loss (an Op; the mathematics is in rowloss.cuh) over logits
// [rows, vocab].
//
// An Op provides
//   kEnt        the sum of e * y is needed (the entropy's value, or its gradient)
//   kLogp       log p of single logits and the entropy are asked for: sums against a high base
//   kGradEnt    the gradient has the entropy's term
//   kHasStats   the row's state is an input: no first pass
//   kList       the gradient has more single entries than the target's
//   Pre, pre(r), live(pre), dead(r)   masked rows: not read, results and gradient zero
//   slot_bytes()                      shared memory of one row
//   prep(r, pre, x, in, slot)         one warp: what does not need the row's state; returns its base
//   finish(r, norm, in, g, slot)      one warp: the gradient's coefficients, in every lane
//   results(r, norm, in, slot)        one warp: writes the row's results
//   state(slot)                       kHasStats: the finished row that prep loaded
//   fix(cf, dx, in, slot, tid, n)     kList: the single entries, after the row is written
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

// What stands for the elements of vectors past a row's end: nothing of the sums.  -inf, but in 0 * y
// where the entropy is summed -1e30; f16 has none that is small enough for every temperature, and takes the vectors
// of a piece that is not whole one by one, with the entropy or without (a row's s must not depend on that).
template <typename T, bool ENT>
struct Pad {
  static constexpr bool kThere = !std::is_same_v<T, __half>;
  static constexpr uint32_t kBits = std::is_same_v<T, float> ? (ENT ? 0xf149f2cau : 0xff800000u) : (ENT ? 0xf149f149u : 0xff80ff80u);
  static __device__ __forceinline__ uint4 vector() { return make_uint4(kBits, kBits, kBits, kBits); }
};
// Adds Q vectors to a state by one check of their sums.  BELOW: none of them is above the base.  What is left to do, vector by vector: nothing; their
// part of u; or all of it.
enum class Left { kNothing, kDot, kAll };
template <class Op, bool BELOW, typename T, int Q>
__device__ __forceinline__ Left push_usual(State& st, float nc, const uint4 (&raw)[Q], const Pairs2& kk) {
  uint64_t s2 = f2_make(0.f, 0.f), u2 = s2;
#pragma unroll
  for (int q = 0; q < Q; ++q) {
    float vals[16 / sizeof(T)];
    unpack16<T>(raw[q], vals);
    sum_usual<Op::kEnt>(s2, u2, vals, nc, kk);
  }
  const float s = f2_lo(s2) + f2_hi(s2), u = Op::kEnt ? f2_lo(u2) + f2_hi(u2) : 0.f;
  if (usual<Op::kLogp>(Op::kEnt ? fmaf(u, 0.f, s) : s)) {  // s, or NaN where u is
    st.s += s;
    if constexpr (Op::kEnt) st.u += u;
    if (Op::kLogp && (BELOW || s <= kLowSum)) st.low += s;
    return Left::kNothing;
  }
  if (!Op::kEnt || !usual<Op::kLogp>(s)) return Left::kAll;
  st.s += s;
  if (Op::kLogp && (BELOW || s <= kLowSum)) st.low += s;
  return Left::kDot;
}

// --------------------------------------------------------------------------
// Short rows: a warp per row, which reads it twice (the second time from L1 or L2).  No barriers; many
// rows in flight hide the latency of each.  Where log p is asked for, a lane raises its base to the maximum of the
// vectors that it has just fetched (16384 x 4096 bf16: policy 68 -> 65 us, log-probabilities 34 -> 29).  Bound by that latency and by the work of a row that does
// not grow with it.  The other kernel's copies keep up with longer rows.  Where they meet (us, this kernel and the other;
// policy, log-probabilities, lists of 64): 16384 rows of 16 KB, bf16 125 and 130, 49 and 57, 145 and 186, f32 policy 93 and 131; of 18 KB,
// f16 policy 151 and 162; 8192 rows of 24 KB, bf16 106 and 106, 39 and 48, 126 and 110, f32 with entropy bonus 101 and 89; of 28 KB 124 and 110.
// --------------------------------------------------------------------------

constexpr int kShortWarps = 4;                 // rows of a CTA
constexpr int kShortSlots = 48 * 1024;         // shared memory that their ops may take
constexpr int kShortVecs = 4;                  // vectors a lane asks for at a time
constexpr int kShortRow = 20 * 1024;           // bytes: longer rows go to the kernel for whole CTAs

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
      using P = Pad<TI, Op::kEnt>;
      for (int v = lane; v < cut.nv; v += 32 * kShortVecs) {
        const TI* at = x + cut.head + v * N;
        const int left = cut.nv - v;
        uint4 raw[kShortVecs];
        Left todo = Left::kAll;
        if (P::kThere || (kShortVecs - 1) * 32 < left) {
#pragma unroll
          for (int q = 0; q < kShortVecs; ++q) raw[q] = !P::kThere || q * 32 < left ? ld_v4(at + q * 32 * N) : P::vector();
          if constexpr (Op::kLogp) raise<Op::kEnt>(st, nc, max_of<TI>(raw), in);
          todo = push_usual<Op, Op::kLogp, TI>(st, nc, raw, kk);
        }
        if (todo != Left::kNothing) {
#pragma unroll 1
          for (int q = 0; q < kShortVecs; ++q)
            if (q * 32 < left) {
              float vals[N];
              unpack16<TI>(ld_v4(at + q * 32 * N), vals);
              push<Op::kEnt, Op::kLogp>(st, nc, vals, in, kk, todo == Left::kDot);
            }
        }
      }
      if (edge >= 0) {
        const float one[1] = {edge_x};
        push<Op::kEnt, Op::kLogp>(st, nc, one, in, kk);
      }
      __syncwarp();
      w = normalise<Op::kEnt>(warp_merge<Op::kEnt, Op::kLogp>(st, in), in);
    }
    const Coef cf = op.finish(r, w, in, g, slot);
    op.results(r, w, in, slot);
    if constexpr (GRAD) {
      if (cf.masked) {
        zeros();
        continue;
      }
      if (vec && !cf.big) {
        for (int v = lane; v < cut.nv; v += 32 * kShortVecs) {
          const int i = cut.head + v * N, left = cut.nv - v;
          uint4 raw[kShortVecs];
#pragma unroll
          for (int q = 0; q < kShortVecs; ++q)
            if (q * 32 < left) raw[q] = ld_v4(x + i + q * 32 * N);
#pragma unroll
          for (int q = 0; q < kShortVecs; ++q) {
            float vals[N], d[N];
            unpack16<TI>(raw[q], vals);
            grads_of<Op::kGradEnt, false>(vals, d, in.k, cf, kk);
            if (q * 32 < left) store_vec<TO, N>(dx + i + q * 32 * N, d);
          }
        }
      } else {
        for (int v = lane; v < cut.nv; v += 32) {
          const int i = cut.head + v * N;
          float vals[N], d[N];
          unpack16<TI>(ld_v4(x + i), vals);
          if (cf.big) grads_of<Op::kGradEnt, true>(vals, d, in.k, cf, kk);
          else grads_of<Op::kGradEnt, false>(vals, d, in.k, cf, kk);
          store_at(dx + i, d, vec);
        }
      }
      // the target's entry, by the lane that has stored the vector it lies in
      const uint32_t tv = (uint32_t)(cf.t - cut.head) / N;  // not a vector of the row where t < head
      if (tv < (uint32_t)cut.nv && tv % 32 == lane) dx[cf.t] = DT<TO>::from_f(cf.at_t);
      if (edge >= 0) dx[edge] = DT<TO>::from_f(edge == cf.t ? cf.at_t : grad_of<Op::kGradEnt>(edge_x, in.k, cf));
      if constexpr (Op::kList) {
        __syncwarp();  // the entries below overwrite what another lane has stored
        op.template fix<TO>(cf, dx, in, slot, lane, 32);
      }
    }
  }
}

// --------------------------------------------------------------------------
// Rows over 20 KB: one read from HBM, one write.
//
// Bound: HBM.  Both passes over a row (the sums, then the gradient) stream it through shared memory,
// the second one from L2, where the rows in flight stay (296 CTAs x 125 KB, 592 x 62.5 KB are 37 MB): the first
// pass's copies ask L2 to keep them (evict_last), the second's let them go (evict_first).
// The next bounds are instruction issue and the ex2 unit (16 a clock and SM; two per element, or one
// without a gradient).
//
// Persistent CTAs, two or four to an SM (the layouts below; one where two rows an SM would not stay in L2:
// 1000 x 131072 f32 takes 206 us with one, 240 with two; 16-bit rows half as long 119 and 115), take rows blockIdx, blockIdx + gridDim, ...  In a CTA
//   - kGroups warps, one for each group below, issue untiled bulk copies of chunks into a ring
//     (mbarriers full / empty), as far ahead as the ring allows.  The ring is a multiple of kGroups
//     chunks, so that each of its places has one copy warp and one group for good.  (One warp for all
//     of them takes about 600 cycles a copy -- its waits and its issue, one after the other -- and
//     held reads to 3.7 TB/s with 8 KB copies.)
//   - kGroups groups of four warps (one to each of the SM's quarters) run the passes, each on chunks
//     of its own in turn.  The second pass of shorter f32 rows runs one row behind the first (lag), so that
//     nothing waits for what lies between a row's two passes; with longer rows the two of each CTA no longer stay in
//     L2 together, all the less the more gradient goes through it.  Policy, 8192 rows (us, with and without lag):
//     bf16 gradient 8000 columns 90 and 98, 15000 130 and 142, 16384 140 and 143; f32 gradient 8000 columns 97 and 111, 10000 117
//     and 130, 12000 144 and 136, 16384 208 and 180.  16-bit rows have four CTAs an SM, which fill each other's gaps: 16384 x 8192
//     130 and 135, but 8192 x 16384 114 and 114, with the bonus 123 and 121, with lists 146 and 128; they run without;
//   - that is the work of kHelpers warps, rows in turn: fetch what the row's loss needs besides the
//     logits (ahead of time), merge the passes' states, hand back the gradient's coefficients, write
//     the row's results, and at last the single entries of a list.
// Every wait is bounded; an expired one raises the CTA's abort flag and the status word, after which
// no copy is issued, nobody waits, and the copies in flight are waited for before the CTA exits.
// --------------------------------------------------------------------------

// How the kernel is laid out: GROUPS of four warps for the passes, a copy warp for each, HELPERS, and
// CTAS of these to an SM; chunks of CHUNK bytes, PLACES of them in the ring; LAG: rows whose bytes and twice their
// gradient's come to no more run with the second pass one row behind the first.
//
// A helper has one place for its row's coefficients.  It writes row i's once every warp has handed in the states
// of row i, so every warp must have read those of its row before by then, row i - HELPERS.  Without lag a warp
// reads row i - 1's ahead of the states of row i.  With lag its order is first(i - 1), second(i - 2), first(i): it has
// read those of row i - 2 and not yet those of row i - 1, so that two helpers are needed.
template <int GROUPS, int HELPERS, int CTAS, int CHUNK, int PLACES, int64_t LAG>
struct Layout {
  static_assert(LAG == 0 || HELPERS >= 2, "the coefficients of a row behind would be overwritten");
  static constexpr int kGroups = GROUPS, kHelpers = HELPERS, kCtas = CTAS, kChunk = CHUNK, kPlaces = PLACES;
  static constexpr int64_t kLag = LAG;
  static constexpr int kGroup = 128;                        // threads of a group
  static constexpr int kPass = GROUPS * kGroup;             // threads of the passes
  static constexpr int kWarps = kPass / 32;
  static constexpr int kThreads = kPass + 128;              // one more group of four: copies, helpers, spare
  static constexpr int kChunkVec = CHUNK / 16;
  static constexpr int kVecPer = kChunkVec / kGroup;        // vectors a thread takes of a chunk
  // registers go where the passes need them: (GROUPS * kRegs + kSpareRegs) * 128, the launch's
  static constexpr int kRegs = GROUPS == 1 ? 80 : 88, kSpareRegs = GROUPS == 1 ? 48 : 64;
  static constexpr int kSmem = (227 - CTAS) * 1024 / CTAS / 128 * 128;  // of each CTA, besides what the system keeps
  static_assert(GROUPS + HELPERS <= 4 && PLACES % GROUPS == 0 && PLACES <= 32, "warps of the fourth; places of one group each, a bit for each");
  static_assert((GROUPS * kRegs + kSpareRegs) * 128 <= 65536 / CTAS / kThreads / 8 * 8 * kThreads, "registers of the launch");
};
// 16-bit rows up to 128 KB, four CTAs of one group: what a row costs whatever its length is paid by four warps
// instead of eight, and three other CTAs fill the gaps (policy 8192 x 32000 bf16: 189 us against 200 for the
// other layout, 1000 x 131072 127 against 115).  One helper: a second one helps sums alone (log-probabilities 8192 x 32000
// bf16: 84 us against 90), and costs where a gradient is written (policy with bonus, 8192 x 12000: 118 against 114) or follows in
// the next launch (preference 16384 x 32000, a third masked: 483 against 454).  Lists take 8 KB chunks (distill 8192 x 32000 bf16: 200 us against
// 207 with 16 KB; policy 197 against 189).
template <bool LIST>
using NarrowLayout = Layout<1, 1, 4, LIST ? 8192 : 16384, LIST ? 6 : 3, 0>;
// Longer rows, and f32 rows, which have half the work to the byte (policy 8192 x 32000 f32: 259 us against 292).
using WideLayout = Layout<2, 2, 2, 16384, 6, 128 * 1024>;
constexpr int64_t kNarrowRow = 128 * 1024;

template <class L>
struct RingShared {
  uint64_t full[L::kPlaces], empty[L::kPlaces];
  // of a helper's row: its base is there; the passes' states are; its coefficients are; its
  // gradient is written
  uint64_t ready[L::kHelpers], states[L::kHelpers], done[L::kHelpers], written[L::kHelpers];
  State warp_state[L::kHelpers][L::kWarps];
  alignas(16) Coef coef[L::kHelpers];
  float base[L::kHelpers];
  int abort;
};

template <class L>
__host__ __device__ constexpr int ring_header() {
  return (int)((sizeof(RingShared<L>) + 127) / 128 * 128);
}

// The bounded wait of common.cuh for warps that run ahead of the passes: it sleeps between tries.
__device__ __forceinline__ bool wait_idle(uint64_t* bar, uint32_t parity, volatile int* abort, int where) {
  if (mbar_try_wait(bar, parity)) return true;
  const uint64_t t0 = globaltimer_ns();
  while (!mbar_try_wait(bar, parity)) {
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
// bulk_load (common.cuh) with an L2 policy.
__device__ __forceinline__ void bulk_load_hint(void* dst, const void* src, uint32_t bytes, uint64_t* bar, uint64_t policy) {
  asm volatile(
      "cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes.L2::cache_hint [%0], [%1], %2, [%3], %4;" ::"r"(smem_u32(dst)),
      "l"(src), "r"(bytes), "r"(smem_u32(bar)), "l"(policy)
      : "memory");
}

// A row's chunks, kept from row to row while the rows' addresses agree modulo 16.
template <typename T, int CHUNK_VEC>
struct Chunks {
  int n, phase;
  int head, tail, nv, chunks;
  __device__ __forceinline__ explicit Chunks(int n_) : n(n_), phase(-1) {}
  __device__ __forceinline__ void at(const T* x) {
    const int p = (int)(reinterpret_cast<uintptr_t>(x) & 15);
    if (p == phase) return;
    phase = p;
    const RowCut<T> cut(x, n);
    head = cut.head;
    tail = cut.tail;
    nv = cut.nv;
    chunks = (nv + CHUNK_VEC - 1) / CHUNK_VEC;
  }
  // the column of the element outside the vectors that thread tid takes, or -1
  __device__ __forceinline__ int edge(int tid) const {
    if (tid >= 32 || (head == 0 && tail == n)) return -1;
    if (tid < head) return tid;
    const int e = tail + tid - 16;
    return tid >= 16 && e < n ? e : -1;
  }
};

// Which of the rows r, r + step, ... are live, asked row by row by a whole warp: 32 rows' masks are
// fetched at a time, so that a row's own is never waited for.
template <class Op>
struct LiveRows {
  const Op& op;
  int64_t rows, step;
  bool backwards;  // row r stands for rows - 1 - r
  uint32_t mask = 0;
  int left = 0;
  __device__ __forceinline__ bool next(int64_t r) {
    if (left == 0) {
      const int64_t q = r + (int64_t)(threadIdx.x & 31) * step;
      mask = __ballot_sync(0xffffffffu, q < rows && op.live(op.pre(backwards ? rows - 1 - q : q)));
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
    at += n;
    while (at >= size) {
      at -= size;
      parity ^= 1;
    }
  }
};

template <class L, class Op, typename TI, typename TO, bool GRAD>
__global__ void __launch_bounds__(L::kThreads, L::kCtas) ring_kernel(RowIn in, RowOut out, Op op, int ring_chunks, int lag) {
  constexpr int N = 16 / sizeof(TI), kGroups = L::kGroups, kHelpers = L::kHelpers, kChunk = L::kChunk, kChunkVec = L::kChunkVec;
  constexpr int kGroup = L::kGroup, kPass = L::kPass, kWarps = L::kWarps, kVecPer = L::kVecPer;
  constexpr bool kSums = !Op::kHasStats;        // a first pass
  constexpr bool kFix = GRAD && Op::kList;
  extern __shared__ __align__(128) char smem[];
  RingShared<L>& sh = *reinterpret_cast<RingShared<L>*>(smem);
  char* ring = smem + ring_header<L>();
  const int slot_bytes = (op.slot_bytes() + 15) & ~15;
  char* slots = ring + (size_t)ring_chunks * kChunk;
  volatile int* abort = &sh.abort;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  // With statistics from an earlier pass over the same rows, the last rows come first: they are what
  // that pass has left in L2.
  const int64_t step = gridDim.x, r0 = blockIdx.x;
  auto nth = [&](int64_t r) { return Op::kHasStats ? in.rows - 1 - r : r; };
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
    }
    sh.abort = 0;
    fence_mbar_init();
  }
  pdl_launch_dependents();
  __syncthreads();
  pdl_wait();

  LiveRows<Op> rows{op, in.rows, step, Op::kHasStats};
  Chunks<TI, kChunkVec> row((int)in.vocab);
  if (warp >= kWarps) {
    setmaxnreg_dec<L::kSpareRegs>();
    if (warp < kWarps + kGroups) {  // ---- copies of one group's chunks
      const int group = warp - kWarps;
      const uint64_t keep = l2_policy_evict_last(), let_go = l2_policy_evict_first();
      Place p;
      int k = 0;  // which group has the next pass's first chunk
      uint32_t used = 0, last_parity = 0;  // bit c: place c has held a copy, and the last one's parity
      bool stop = false;
      auto copy = [&](int64_t r, bool last) {
        const TI* x = static_cast<const TI*>(in.logits) + r * in.ld;
        row.at(x);
        const int c0 = (group - k + kGroups) % kGroups;
        Place at = p;
        at.next(ring_chunks, c0);
        p.next(ring_chunks, row.chunks);
        k = (k + row.chunks) % kGroups;
        if (lane != 0 || stop) return;
        const char* src = reinterpret_cast<const char*>(x + row.head) + (size_t)c0 * kChunk;
        int left = row.nv - c0 * kChunkVec;
        for (int c = c0; c < row.chunks; c += kGroups) {
          // a place's first use waits for the barrier's phase before the first: no wait
          if (!wait_idle(&sh.empty[at.at], at.parity ^ 1, abort, 201)) {
            stop = true;
            return;
          }
          const uint32_t bytes = (uint32_t)min(left, kChunkVec) * 16u;
          mbar_arrive_expect_tx(&sh.full[at.at], bytes);
          bulk_load_hint(ring + (size_t)at.at * kChunk, src, bytes, &sh.full[at.at], last ? let_go : keep);
          used |= 1u << at.at;
          last_parity = (last_parity & ~(1u << at.at)) | (at.parity << at.at);
          at.next(ring_chunks, kGroups);
          src += kGroups * kChunk;
          left -= kGroups * kChunkVec;
        }
      };
      int64_t behind = -1;
      for (int64_t r = r0;; r += step) {  // the order of the passes below
        while (r < in.rows && !rows.next(r)) r += step;
        const bool more = r < in.rows;
        if (kSums && more) copy(nth(r), !GRAD);
        const int64_t due = kSums && lag ? behind : more ? r : -1;
        if (GRAD && due >= 0) copy(nth(due), true);
        if (!more) break;
        behind = r;
      }
      // the last copy into each place has landed before the CTA gives up its shared memory
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
    } else if (warp < kWarps + kGroups + kHelpers) {  // ---- what lies between a row's two passes
      const int h = warp - kWarps - kGroups;
      const float g = GRAD ? (out.dloss ? *out.dloss : 1.f) * out.scale : 0.f;
      int turn = 0;
      uint32_t parity = 0;
      int64_t r = r0;
      auto next_row = [&]() {  // this helper's next row, or past the end
        for (; r < in.rows; r += step) {
          if (!rows.next(r)) continue;
          const bool mine = turn == h;
          if (++turn == kHelpers) turn = 0;
          if (mine) break;
        }
      };
      // Fetches row r into one of the helper's two slots and announces its base.
      auto fetch = [&](int which) {
        const int64_t at = nth(r);
        const TI* x = static_cast<const TI*>(in.logits) + at * in.ld;
        const float base = op.prep(at, op.pre(at), x, in, slots + (2 * h + which) * slot_bytes);
        __syncwarp();
        if (kSums && lane == 0) {
          sh.base[h] = base;
          mbar_arrive(&sh.ready[h]);
        }
      };
      next_row();
      if (r < in.rows) fetch(0);
      while (r < in.rows) {
        const int64_t now = nth(r);
        char* slot = slots + (2 * h + parity) * slot_bytes;
        Norm w;
        if constexpr (kSums) {
          (void)wait_idle(&sh.states[h], parity, abort, 203);
          __syncwarp();
          const State st = lane < kWarps ? sh.warp_state[h][lane] : empty_state(sh.warp_state[h][0].m);
          w = normalise<Op::kEnt>(warp_merge<Op::kEnt, Op::kLogp>(st, in), in);
        } else {
          w = op.state(slot);
          // the passes have read the coefficients of this helper's row before
          (void)wait_idle(&sh.written[h], parity ^ 1, abort, 205);
          __syncwarp();
        }
        const Coef cf = op.finish(now, w, in, g, slot);
        if (lane == 0) {
          sh.coef[h] = cf;
          mbar_arrive(&sh.done[h]);
        }
        op.results(now, w, in, slot);
        r += step;
        next_row();
        if (r < in.rows) fetch((int)(parity ^ 1));  // before the wait for this row's gradient
        if constexpr (kFix) {
          (void)wait_idle(&sh.written[h], parity, abort, 206);
          __syncwarp();
          if (!cf.masked) op.template fix<TO>(cf, static_cast<TO*>(out.dlogits) + now * out.ld, in, slot, lane, 32);
          __syncwarp();
        }
        parity ^= 1;
      }
    }
  } else {  // ---- the passes
    setmaxnreg_inc<L::kRegs>();
    const Pairs2 kk(in);
    const uint32_t group = warp / (kGroup / 32), gtid = tid % kGroup;
    Place p, slot1, slot2;  // of the next pass's first chunk; of the helpers of the first and the second pass
    uint32_t k = 0;         // which group has that chunk
    // This group's first chunk of a pass over `row`, after which p and k are the next pass's.
    auto enter = [&](Place& at) {
      const int c0 = (int)((group - k + kGroups) % kGroups);
      at = p;
      at.next(ring_chunks, c0);
      p.next(ring_chunks, row.chunks);
      k = (k + row.chunks) % kGroups;
      return c0;
    };
    // the first pass of row r: its sums
    auto first = [&](int64_t r) {
      const TI* x = static_cast<const TI*>(in.logits) + r * in.ld;
      row.at(x);
      const int edge = row.edge(tid);
      const float edge_x = edge >= 0 ? DT<TI>::to_f(x[edge]) : 0.f;
      (void)mbar_wait(&sh.ready[slot1.at], slot1.parity, abort, 211);
      State st = empty_state(sh.base[slot1.at]);
      float nc = minus_c(st.m, in);
      using P = Pad<TI, Op::kEnt>;
      Place at;
      const int c0 = enter(at);
      int left = row.nv - c0 * kChunkVec - (int)gtid;
      for (int c = c0; c < row.chunks; c += kGroups) {
        (void)mbar_wait(&sh.full[at.at], at.parity, abort, 209);
        const uint4* v = reinterpret_cast<const uint4*>(ring + (size_t)at.at * kChunk) + gtid;
        Left todo = Left::kAll;
        if (P::kThere || (kVecPer - 1) * kGroup < left) {  // all of the thread's vectors at once
          uint4 raw[kVecPer];
#pragma unroll
          for (int q = 0; q < kVecPer; ++q) {
            raw[q] = v[q * kGroup];  // past the row's end: whatever the chunk holds
            if (P::kThere && q * kGroup >= left) raw[q] = P::vector();
          }
          todo = push_usual<Op, false, TI>(st, nc, raw, kk);
        }
        if (todo != Left::kNothing) {
#pragma unroll 1
          for (int q = 0; q < kVecPer; ++q)
            if (q * kGroup < left) {
              float vals[N];
              unpack16<TI>(v[q * kGroup], vals);
              push<Op::kEnt, Op::kLogp>(st, nc, vals, in, kk, todo == Left::kDot);
            }
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&sh.empty[at.at]);
        at.next(ring_chunks, kGroups);
        left -= kGroups * kChunkVec;
      }
      if (edge >= 0) {
        const float one[1] = {edge_x};
        push<Op::kEnt, Op::kLogp>(st, nc, one, in, kk);
      }
      __syncwarp();
      st = warp_merge<Op::kEnt, Op::kLogp>(st, in);
      // the helper has read the states of its row before
      if constexpr (!GRAD) (void)mbar_wait(&sh.done[slot1.at], slot1.parity ^ 1, abort, 210);
      if (lane == 0) {
        sh.warp_state[slot1.at][warp] = st;
        mbar_arrive(&sh.states[slot1.at]);
      }
      slot1.next(kHelpers);
    };
    // the second pass of row r: its gradient
    auto second = [&](int64_t r) {
      const TI* x = static_cast<const TI*>(in.logits) + r * in.ld;
      row.at(x);
      TO* dx = static_cast<TO*>(out.dlogits) + r * out.ld;
      const int edge = row.edge(tid);
      const bool vec = vector_rows<TO, N>(dx, row.head);
      const float edge_x = edge >= 0 ? DT<TI>::to_f(x[edge]) : 0.f;
      (void)mbar_wait(&sh.done[slot2.at], slot2.parity, abort, 207);
      const Coef cf = sh.coef[slot2.at];
      const uint32_t k_row = k;
      Place first_at;
      const int c0 = enter(first_at);
      // What is the same for a whole row is decided here, not vector by vector.
      auto chunks = [&](auto usual_row) {
        constexpr bool kUsual = decltype(usual_row)::value;
        Place at = first_at;
        int left = row.nv - c0 * kChunkVec - (int)gtid;
        TO* to = dx + row.head + (c0 * kChunkVec + (int)gtid) * N;
        for (int c = c0; c < row.chunks; c += kGroups) {
          (void)mbar_wait(&sh.full[at.at], at.parity, abort, 208);
          const uint4* v = reinterpret_cast<const uint4*>(ring + (size_t)at.at * kChunk) + gtid;
          if constexpr (kUsual) {  // all of the thread's vectors, side by side
            uint4 raw[kVecPer];
#pragma unroll
            for (int q = 0; q < kVecPer; ++q) raw[q] = v[q * kGroup];
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
                unpack16<TI>(v[q * kGroup], vals);
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
          }
          // Released after the chunk's last use.  The arrival orders this warp's accesses of shared memory among
          // ordinary ones, but the next copy writes through the async proxy, and nothing orders that after loads that
          // are still under way: released right after the loads were issued, the copy overtook some of them.  A store
          // that needs a loaded value (in the first pass, the branch on the check of the sums) is not issued before the
          // value is there, and the arrival follows it.  A proxy fence before the arrival would do as well, but waits for more:
          // log-probabilities 8192 x 32000 bf16 took 94 us with it for 89, 2999 x 50257 f16 66 for 57.
          __syncwarp();
          if (lane == 0) mbar_arrive(&sh.empty[at.at]);
          at.next(ring_chunks, kGroups);
          left -= kGroups * kChunkVec;
          to += kGroups * kChunkVec * N;
        }
      };
      if (vec && !cf.big && !cf.masked) chunks(std::true_type());
      else chunks(std::false_type());
      if (edge >= 0) dx[edge] = DT<TO>::from_f(cf.masked ? 0.f : edge == cf.t ? cf.at_t : grad_of<Op::kGradEnt>(edge_x, in.k, cf));
      // the target's entry, by the thread that has stored the vector it lies in
      const uint32_t tv = (uint32_t)(cf.t - row.head) / N;  // not a vector of the row where t < head
      if (tv < (uint32_t)row.nv && tv % kGroup == gtid && (tv / kChunkVec + k_row) % kGroups == group) dx[cf.t] = DT<TO>::from_f(cf.at_t);
      if constexpr (kFix || !kSums) {
        __syncwarp();
        if (lane == 0) mbar_arrive(&sh.written[slot2.at]);
      }
      slot2.next(kHelpers);
    };
    int64_t behind = -1;
    for (int64_t r = r0;; r += step) {
      for (; r < in.rows && !rows.next(r); r += step) {  // masked
        const int64_t at = nth(r);
        if (tid == 0) op.dead(at);
        if constexpr (GRAD) {
          TO* dx = static_cast<TO*>(out.dlogits) + at * out.ld;
          row.at(static_cast<const TI*>(in.logits) + at * in.ld);
          const bool vec = vector_rows<TO, N>(dx, row.head);
          const float zero[N] = {};
          for (int v = tid; v < row.nv; v += kPass) store_at(dx + row.head + v * N, zero, vec);
          const int edge = row.edge(tid);
          if (edge >= 0) dx[edge] = DT<TO>::from_f(0.f);
        }
      }
      const bool more = r < in.rows;
      if constexpr (kSums)
        if (more) first(r);
      if constexpr (GRAD) {
        const int64_t due = kSums && lag ? behind : more ? r : -1;
        if (due >= 0) second(nth(due));
      }
      if (!more) break;
      behind = r;
    }
  }
}

// --------------------------------------------------------------------------
// host
// --------------------------------------------------------------------------

constexpr int64_t kPairRow = 320 * 1024;  // bytes: of longer rows an SM takes one at a time

template <class L, class Op, typename TI, typename TO, bool GRAD>
static cudaError_t launch_ring(cudaStream_t s, const RowIn& in, const RowOut& out, const Op& op, int dev) {
  auto kern = ring_kernel<L, Op, TI, TO, GRAD>;
  static std::atomic<bool> ready[64];  // (set once a device; racing first calls do the same)
  if (!ready[dev].load(std::memory_order_relaxed)) {
    const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, L::kSmem);
    if (e != cudaSuccess) return e;
    ready[dev].store(true, std::memory_order_relaxed);
  }
  const int slots = 2 * L::kHelpers * ((op.slot_bytes() + 15) & ~15);
  int places = (L::kSmem - ring_header<L>() - slots) / L::kChunk;
  places = (places < L::kPlaces ? places : L::kPlaces) / L::kGroups * L::kGroups;
  const size_t smem = (size_t)ring_header<L>() + (size_t)places * L::kChunk + slots;
  const int64_t bytes = in.vocab * (int64_t)sizeof(TI), ctas = (int64_t)num_sms(dev) * (bytes <= kPairRow ? L::kCtas : 1);
  return launch_pdl(kern, dim3((unsigned)(in.rows < ctas ? in.rows : ctas)), dim3(L::kThreads), smem, s, in, out, op, places,
                    GRAD && bytes + 2 * in.vocab * (int64_t)sizeof(TO) <= L::kLag);
}

template <class Op, typename TI, typename TO, bool GRAD>
static int launch_row(cudaStream_t s, const RowIn& in, const RowOut& out, const Op& op, const char* name) {
  const int dev = current_device();
  if (dev < 0 || dev >= 64) return fail(FERRITE_LAUNCH_FAILED, "%s: device ordinal %d", name, dev);
  cudaError_t e;
  const int slot = (op.slot_bytes() + 15) & ~15;
  // The kernel goes by the row's length and type (and a list's), not by how many rows there are, with a
  // gradient or without: so a row's results have the same bits in every call (log-probabilities taken
  // in one batch and compared in another differ by nothing), as long as it starts on a 16-byte boundary.
  const int64_t bytes = in.vocab * (int64_t)sizeof(TI);
  if (bytes <= kShortRow && kShortWarps * slot <= kShortSlots) {
    const int64_t ctas = (in.rows + kShortWarps - 1) / kShortWarps, most = (int64_t)num_sms(dev) * 16;
    e = launch_pdl(short_row_kernel<Op, TI, TO, GRAD>, dim3((unsigned)(ctas < most ? ctas : most)), dim3(kShortWarps * 32), kShortWarps * slot, s,
                   in, out, op);
  } else {
    e = cudaSuccess;
    bool narrow = false;
    if constexpr (sizeof(TI) == 2) {
      narrow = bytes <= kNarrowRow;
      if (narrow) e = launch_ring<NarrowLayout<Op::kList>, Op, TI, TO, GRAD>(s, in, out, op, dev);
    }
    if (!narrow) e = launch_ring<WideLayout, Op, TI, TO, GRAD>(s, in, out, op, dev);
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
