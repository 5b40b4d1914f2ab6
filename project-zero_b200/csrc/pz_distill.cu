// pz_distill.cu — distillation from a teacher's top logits: the loss of a
// student's rows of logits against a short list of ids per row, and its
// gradient.
//
// Per row, with student logits s over V ids, the list's ids j with values
// t_j, temperature T and weight w:
//
//   q_v   = exp(s_v / T) / sum_u exp(s_u / T)
//   LIST: p_j = exp(t_j / T) / sum over the list, rho = 0
//   REST: p_j = exp(t_j) (log-probabilities over the whole vocabulary),
//         rho = max(0, 1 - sum_j p_j), the mass of all other ids together
//   loss  = w T^2 ( sum_j p_j (log p_j - log q_j) + rho (log rho - log r) )
//           r = sum of q over the ids off the list
//   d loss / d s_v = w T (P q_v - p_v)              v on the list
//                  = w T q_v (P - rho / r)          v off it,  P = sum p + rho
//
// An id listed twice counts with the sum of its probabilities.
//
// Everything runs in units of 2: e_v = 2^((s_v - m) c), c = log2(e) / T, m a
// maximum (the difference first, so rows of the type's lowest value keep
// their shape).  Sums of e are fp32, joined in a fixed order: the same call
// gives the same bits.  A thread adds the even and the odd columns apart, 501
// terms each for a row of 128256 in one CTA, 768 for the longest span that a
// CTA's bits allow (196608 columns), and scales the sums once a batch.  REST keeps
// the ids off the list under a maximum of their own, so that log r and
// rho / r hold when the student leaves them next to nothing.  The sum over
// the list, whose terms nearly cancel against log S, is in fp64.
//
// Bound: HBM; loss and gradient together also by what has to follow one
// another within a row (fetch, exchange, store), which five CTAs on an SM do
// not hide altogether.
//   loss      a row per CTA while the rows fill the GPU, parts of one in a
//             cluster otherwise; the next batch of vectors in flight while one
//             is summed.  1024 rows of 128256 f32, nine tenths of them with
//             a weight (the others are not read, here and below): 74 us, 6.4
//             TB/s.
//   gradient  from saved statistics: parts of 64 KB, independent CTAs.  2048
//             rows of 151936 bf16: 190 us, 6.2 TB/s (after a loss of 99 us).
//   both      one read and one write: a row stays on chip between its two
//             passes.  A cluster of up to 8 CTAs takes it, each fetching 32 KB
//             of it into shared memory (cp.async; a thread reads back what it
//             fetched itself), and they exchange maximum and sums through
//             distributed shared memory.  4096 rows of 128256 bf16: 412 us,
//             4.8 TB/s.  Four warps a CTA: with eight, each repeating the
//             row's scalars for half as many columns, it was 566 us, with two
//             495; parts of 64 KB (three CTAs on an SM, not five) 505.
// The list is read by all parts of its row: at most 1024 ids, two barriers.
// Gradient rows that lie at another offset from a 16-byte boundary than the
// logits' are stored an element at a time: 2048 rows of 50257 bf16, logits
// 50304 apart, gradient alone 269 us where its rows are contiguous, 74 where
// they are 50304 apart too.
#include <atomic>

#include "pz_device.cuh"
#include "pz_rowvec.cuh"
#include "pz_status.cuh"

namespace pz {
namespace {

constexpr int kThreads = 128;
constexpr int kWarps = kThreads / 32;
constexpr int kBatch = 4;              // 16-byte vectors that a thread works on at a time
constexpr int kStep = kBatch * kThreads;
constexpr int kEntries = (PZ_TOP_K_MAX + kThreads - 1) / kThreads;  // most list entries of a thread
constexpr int kMaxCluster = 8;         // the portable cluster size
constexpr int kCtasPerSm = 7;
constexpr int kResident = 64 * 1024;   // most bytes of a row that a CTA keeps in shared memory

struct DistillArgs {
  const void *logits;
  int64_t ld;
  int N, V;
  const int32_t *ids;
  const float *values;
  int K;
  int64_t ld_ids, ld_values;
  const int32_t *n_list;
  const float *weight;
  const float *grad_loss;
  float T, c;
  double inv_T;
  int rest;
  float *loss;
  float4 *stats;
  void *grad;
  int64_t ld_grad;
  int parts;  // CTAs per row (the cluster's size in distill_kernel)
  int span;   // vectors per CTA
  int bit_words;  // words of a CTA's bits of listed columns, a multiple of 4
  int resident;   // vectors of the span that stay in shared memory
  int flag_shift; // batches of a thread per flag: 2^flag_shift, so that 32 flags cover the span
};

// 2^x, fp32 results below 2^-126 flushed to zero (they are lost in any sum
// with the 1 that the row's maximum contributes).
__device__ __forceinline__ float exp2_approx(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// A CTA's view of its row's list, in shared memory; entry j belongs to thread
// j % kThreads, which alone reads and writes it once the list is set up.
struct List {
  uint32_t *bits;  // one bit per column of the CTA's span: listed
  uint32_t flags;  // REST: this thread's batches (groups of 2^flag_shift) that hold a listed column
  int32_t *id;     // [K]; -1: not in this CTA's columns, ignored, or a later entry of an id listed twice
  float *p;        // [K] probabilities
  float *log_p;    // [K]
  float *s;        // [K] the student's logits
  float mass;      // sum of p over the whole list, and rho
  float rho;
  bool valid;      // the row has a target
};

// The columns [c0, c1) that a CTA takes of a row whose columns start `shift`
// elements after a 16-byte boundary: the vectors [k0, k1).
template <typename T>
struct Span {
  int k0, k1, c0, c1;
  __device__ __forceinline__ Span(int part, int span, int V, int shift) {
    constexpr int N = RowElem<T>::N;
    const int all = (V + shift + N - 1) / N;
    k0 = min(part * span, all);
    k1 = min(k0 + span, all);
    c0 = k0 * N - shift;  // may lie before column 0
    c1 = k1 * N - shift;
  }
};

// A thread's first entry of the row's list, on its way before anything is
// known about the row.
struct Entry {
  int id, n;
  float value;
  __device__ __forceinline__ Entry(const DistillArgs &A, int64_t row) : id(-1), n(A.K), value(0.0f) {
    const int j = threadIdx.x;
    if (j < A.K) {
      if (A.n_list) n = min(max(A.n_list[row], 0), A.K);
      id = A.ids[row * A.ld_ids + j];
      value = A.values[row * A.ld_values + j];
    }
  }
};

// Reads the row's list: the probabilities and, of the ids in the CTA's
// columns, bits and logits.  Two barriers of the block, the second one last.
template <typename T, bool REST>
__device__ __forceinline__ List read_list(const DistillArgs &A, int64_t row, const Entry &first, const T *x_row,
                                          const Span<T> &sp, unsigned char *smem) {
  __shared__ float s_top[kWarps];
  __shared__ int s_seen[kWarps], s_bad[kWarps];
  __shared__ double s_sum[kWarps];
  __shared__ int s_twice, s_gap;
  __shared__ uint32_t s_flags[REST ? kThreads : 1];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int busy = min((A.K + 31) / 32, kWarps);  // warps with an entry
  List L;
  L.bits = reinterpret_cast<uint32_t *>(smem);
  L.id = reinterpret_cast<int32_t *>(L.bits + A.bit_words);
  L.p = reinterpret_cast<float *>(L.id + A.K);
  L.log_p = L.p + A.K;
  L.s = L.log_p + A.K;
  float top = -INFINITY;
  int seen = 0, bad = 0;
  float own[kEntries];  // logits on their way while the probabilities are worked out
  if (warp < busy) {
    const int32_t *ids = A.ids + row * A.ld_ids;
    const float *values = A.values + row * A.ld_values;
#pragma unroll
    for (int e = 0; e < kEntries; e++) {
      const int j = tid + e * kThreads;
      if (j >= A.K) break;
      int id = e == 0 ? first.id : ids[j];
      float t = e == 0 ? first.value : values[j];
      if (j >= first.n || id < 0 || id >= A.V) {
        id = -1;
        t = -INFINITY;
      } else {
        seen++;
        bad |= t != t;
        top = fmaxf(top, t);
      }
      L.id[j] = id;
      L.log_p[j] = t;
      if (id >= 0 && id >= sp.c0 && id < sp.c1) own[e] = RowElem<T>::get(x_row + id);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, o));
    seen = __reduce_add_sync(0xFFFFFFFFu, seen);
    bad = __any_sync(0xFFFFFFFFu, bad);
    if (lane == 0) {
      s_top[warp] = top;
      s_seen[warp] = seen;
      s_bad[warp] = bad;
    }
  }
  for (int i = tid; i < A.bit_words / 4; i += kThreads) reinterpret_cast<uint4 *>(L.bits)[i] = make_uint4(0u, 0u, 0u, 0u);
  if (tid == 0) s_twice = s_gap = 0;
  if (REST) s_flags[tid] = 0u;
  __syncthreads();
  top = -INFINITY;
  seen = bad = 0;
  for (int i = 0; i < busy; i++) {
    top = fmaxf(top, s_top[i]);
    seen += s_seen[i];
    bad |= s_bad[i];
  }
  // LIST: relative to the largest, the difference before the division by T:
  // values of the type's lowest or far from zero keep what sets them apart.
  // REST: as they are.
  const float base = (REST || !(top > -INFINITY)) ? 0.0f : top;
  // A list that names every id leaves none for rho (what 1 - sum holds then
  // is rounding).
  const bool whole = REST && seen >= A.V;
  if (whole) {
    for (int v = tid; v < A.V; v += kThreads) {
      bool on = false;
      for (int j = 0; j < A.K; j++) on |= L.id[j] == v;
      if (!on) s_gap = 1;
    }
    __syncthreads();  // ids of other CTAs' columns leave the list below
  }
  if (warp < busy) {
    double sum = 0.0;
#pragma unroll
    for (int e = 0; e < kEntries; e++) {
      const int j = tid + e * kThreads;
      if (j >= A.K) break;
      const int id = L.id[j];
      const float t = REST ? L.log_p[j] : __fdiv_rn(__fsub_rn(L.log_p[j], base), A.T);
      const float p = id >= 0 ? expf(t) : 0.0f;
      L.log_p[j] = t;
      L.p[j] = p;
      sum += p;
      if (id >= 0 && id >= sp.c0 && id < sp.c1) {
        const uint32_t bit = 1u << ((id - sp.c0) & 31);
        L.s[j] = own[e];
        if (REST) {
          const int vec = (id - sp.c0) / RowElem<T>::N;
          atomicOr(&s_flags[vec % kThreads], 1u << (vec / kStep >> A.flag_shift));
        }
        if (atomicOr(&L.bits[(id - sp.c0) >> 5], bit) & bit) s_twice = 1;
      } else {
        L.id[j] = -1;
      }
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, o);
    if (lane == 0) s_sum[warp] = sum;
  }
  __syncthreads();
  L.flags = REST ? s_flags[tid] : 0u;
  double sum = 0.0;
  for (int i = 0; i < busy; i++) sum += s_sum[i];
  if (!REST) {
    if (warp < busy) {
      const float inv = static_cast<float>(1.0 / sum), log_sum = logf(static_cast<float>(sum));
      for (int j = tid; j < A.K; j += kThreads) {
        L.p[j] = __fmul_rn(L.p[j], inv);
        L.log_p[j] = __fsub_rn(L.log_p[j], log_sum);
      }
    }
    if (sum == sum) sum = 1.0;  // a NaN value makes the row's outputs NaN
  }
  // (an unordered comparison keeps a NaN sum)
  L.rho = (REST && !(whole && !s_gap) && !(sum >= 1.0)) ? static_cast<float>(1.0 - sum) : 0.0f;
  L.mass = __fadd_rn(static_cast<float>(sum), L.rho);
  // no entries: no target.  LIST with no finite value: none either.
  L.valid = seen > 0 && (REST || top > -INFINITY || bad);
  if (s_twice) {
    // the first entry of an id takes the probabilities of all, in list order
    __syncthreads();
    float joined[kEntries];
#pragma unroll
    for (int e = 0; e < kEntries; e++) {
      const int j = tid + e * kThreads;
      joined[e] = -1.0f;
      if (j < A.K && L.id[j] >= 0) {
        double all = 0.0;
        bool first = true;
        for (int i = 0; i < A.K; i++)
          if (L.id[i] == L.id[j]) {
            first &= i >= j;
            all += L.p[i];
          }
        if (first) joined[e] = static_cast<float>(all);
      }
    }
    __syncthreads();
#pragma unroll
    for (int e = 0; e < kEntries; e++) {
      const int j = tid + e * kThreads;
      if (j < A.K) {
        if (joined[e] == -1.0f) L.id[j] = -1;
        L.p[j] = joined[e];
        L.log_p[j] = logf(joined[e]);
      }
    }
  }
  return L;
}

// The row's columns as a thread sees them: batches of kBatch vectors, kThreads
// apart, from vector `kb + tid` on.  Batches that lie whole in the span and in
// the row (the block's, all alike) take a path without a test per vector.
template <typename T>
struct Columns {
  static constexpr int N = RowElem<T>::N;
  const T *row;
  int V, shift;
  WholeVecs whole;
  Span<T> sp;
  __device__ __forceinline__ Columns(const T *x_row, int V_, int part, int span)
      : row(x_row), V(V_), shift(row_shift(x_row)), whole(whole_vecs<T>(shift, V_)), sp(part, span, V_, shift) {}
  __device__ __forceinline__ bool whole_batch(int kb) const {
    return kb >= whole.first && kb + kStep <= min(sp.k1, whole.last);
  }
  __device__ __forceinline__ bool whole_vec(int k) const { return k >= whole.first && k < whole.last; }
  __device__ __forceinline__ const T *at(int k) const { return row + (k * N - shift); }
  // A batch into registers, -inf where there is no vector.
  __device__ __forceinline__ void load(int kb, uint4 *raw) const {
    const int k = kb + static_cast<int>(threadIdx.x);
    if (whole_batch(kb)) {
      const T *p = at(k);
#pragma unroll
      for (int i = 0; i < kBatch; i++) raw[i] = load16(p + i * kThreads * N);
    } else {
#pragma unroll
      for (int i = 0; i < kBatch; i++) {
        const int v = k + i * kThreads;
        raw[i] = make_uint4(RowElem<T>::kNegInf2, RowElem<T>::kNegInf2, RowElem<T>::kNegInf2, RowElem<T>::kNegInf2);
        if (v < sp.k1) raw[i] = whole_vec(v) ? load16(at(v)) : load_edge(row, V, v * N - shift);
      }
    }
  }
  // The vectors [sp.k0, k_end) into shared memory, asynchronously where they
  // lie whole in the row; every thread fetches those it reads itself.
  __device__ __forceinline__ void fetch(uint4 *to, int k_end) const {
    for (int kb = sp.k0; kb < k_end; kb += kStep) {
      const int k = kb + static_cast<int>(threadIdx.x);
      uint4 *slot = to + (k - sp.k0);
      if (whole_batch(kb) && kb + kStep <= k_end) {
        const T *p = at(k);
#pragma unroll
        for (int i = 0; i < kBatch; i++) copy16(slot + i * kThreads, p + i * kThreads * N);
      } else {
        for (int v = k; v < min(kb + kStep, k_end); v += kThreads, slot += kThreads) {
          if (whole_vec(v))
            copy16(slot, at(v));
          else
            *slot = load_edge(row, V, v * N - shift);
        }
      }
    }
  }
  static __device__ __forceinline__ void copy16(uint4 *to, const T *from) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(static_cast<uint32_t>(__cvta_generic_to_shared(to))),
                 "l"(from)
                 : "memory");
  }
  __device__ __forceinline__ void held(const uint4 *from, int kb, int k_end, uint4 *raw) const {
    const int k = kb + static_cast<int>(threadIdx.x);
    const uint4 *p = from + (k - sp.k0);
    if (kb + kStep <= k_end) {
#pragma unroll
      for (int i = 0; i < kBatch; i++) raw[i] = p[i * kThreads];
    } else {
#pragma unroll
      for (int i = 0; i < kBatch; i++) {
        raw[i] = make_uint4(RowElem<T>::kNegInf2, RowElem<T>::kNegInf2, RowElem<T>::kNegInf2, RowElem<T>::kNegInf2);
        if (k + i * kThreads < k_end) raw[i] = p[i * kThreads];
      }
    }
  }
};

// The same columns of the gradient.
template <typename T>
struct Gradient {
  static constexpr int N = RowElem<T>::N;
  T *row;
  bool aligned;  // a vector of the logits is one of the gradient too
  __device__ __forceinline__ Gradient(T *g_row, int shift)
      : row(g_row),
        aligned(((reinterpret_cast<uintptr_t>(g_row) - static_cast<uintptr_t>(shift) * sizeof(T)) & 15u) == 0) {}
  __device__ __forceinline__ void store(const Columns<T> &C, int kb, int k_end, const uint4 *v) const {
    const int k = kb + static_cast<int>(threadIdx.x);
    if (aligned && C.whole_batch(kb)) {
      T *p = row + (k * N - C.shift);
#pragma unroll
      for (int i = 0; i < kBatch; i++) store16(p + i * kThreads * N, v[i]);
    } else {
#pragma unroll
      for (int i = 0; i < kBatch; i++) {
        const int at = k + i * kThreads;
        if (at < k_end) {
          if (aligned && C.whole_vec(at))
            store16(row + (at * N - C.shift), v[i]);
          else
            store_edge(row, C.V, at * N - C.shift, v[i]);
        }
      }
    }
  }
  __device__ __forceinline__ void zero(const Columns<T> &C) const {
    const uint4 v[kBatch] = {};
    for (int kb = C.sp.k0; kb < C.sp.k1; kb += kStep) store(C, kb, C.sp.k1, v);
  }
};

// A maximum and the sum of e relative to it.
struct MaxSum {
  float m, s;
};
__device__ __forceinline__ float exp_from(float x, float m, float c) {
  return exp2_approx(__fmul_rn(__fsub_rn(x, m), c));
}
// The pairs of the lanes whose index differs in the bits of WIDTH - 1: their
// maximum first, then each sum scaled once (a lane at -inf has the sum 0, or
// NaN, which stays).
template <int WIDTH>
__device__ __forceinline__ MaxSum join_lanes(MaxSum a, float c) {
  float m = a.m;
#pragma unroll
  for (int o = WIDTH / 2; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xFFFFFFFFu, m, o));
  float s = __fmul_rn(a.s, exp_from(a.m, m > -INFINITY ? m : 0.0f, c));
#pragma unroll
  for (int o = WIDTH / 2; o > 0; o >>= 1) s = __fadd_rn(s, __shfl_xor_sync(0xFFFFFFFFu, s, o));
  return MaxSum{m, s};
}
__device__ __forceinline__ MaxSum join(const MaxSum &a, const MaxSum &b, float c) {
  const float m = fmaxf(a.m, b.m), base = m > -INFINITY ? m : 0.0f;
  return MaxSum{m, __fadd_rn(__fmul_rn(a.s, exp_from(a.m, base, c)), __fmul_rn(b.s, exp_from(b.m, base, c)))};
}
template <int WIDTH>
__device__ __forceinline__ double sum_lanes(double x) {
#pragma unroll
  for (int o = WIDTH / 2; o > 0; o >>= 1) x += __shfl_xor_sync(0xFFFFFFFFu, x, o);
  return x;
}

// A CTA's part of its row's sums.
struct RowPart {
  MaxSum row;   // its columns (REST: those off the list)
  MaxSum list;  // REST: its listed ids
  // over its listed ids: sum p, and sum p (log p - (s - ref) / T), ref being
  // the CTA's own maximum: the differences are taken before the sums, which
  // would lose them in rows of the type's lowest value
  double p, l;
  __device__ __forceinline__ float ref() const {
    const float m = fmaxf(row.m, list.m);
    return m > -INFINITY ? m : 0.0f;
  }
};

__device__ __forceinline__ int cluster_rank() {
  int r;
  asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ int cluster_id() {
  int r;
  asm("mov.u32 %0, %%clusterid.x;" : "=r"(r));
  return r;
}
// The row's cluster: all CTAs have to arrive before any passes the wait.
// Threads that wrote nothing for the others arrive without a fence.
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release;" ::: "memory"); }
__device__ __forceinline__ void cluster_arrive_relaxed() {
  asm volatile("barrier.cluster.arrive.relaxed;" ::: "memory");
}
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire;" ::: "memory"); }

// Copies v to the same shared variable of CTA `rank` of the cluster.
__device__ __forceinline__ void put_remote(const RowPart *slot, const RowPart &v, int rank) {
  uint32_t at;
  asm("mapa.shared::cluster.u32 %0, %1, %2;"
      : "=r"(at)
      : "r"(static_cast<uint32_t>(__cvta_generic_to_shared(slot))), "r"(rank));
  static_assert(sizeof(RowPart) == 32, "two 16-byte stores");
  asm volatile("st.shared::cluster.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(at), "f"(v.row.m), "f"(v.row.s), "f"(v.list.m),
               "f"(v.list.s)
               : "memory");
  asm volatile("st.shared::cluster.v2.f64 [%0], {%1, %2};" ::"r"(at + 16), "d"(v.p), "d"(v.l) : "memory");
}

// The row's sums: M and S over all ids, M_off and S_off over those whose
// gradient is the pass along the row's (LIST: all; REST: off the list).
struct RowSums {
  float M, S, M_off, S_off;
};

// What the gradient multiplies e by.
struct GradFactors {
  float M, M_off;
  float q_of_e;  // listed ids, e relative to M: P / S
  float f;       // the others, e relative to M_off: w T (P / S 2^((M_off - M) c) - rho / S_off)
};
__device__ __forceinline__ GradFactors grad_factors(const List &L, const RowSums &R, float c, float by) {
  // a row without any weight (every logit -inf): its gradient is 0
  if (R.S == 0.0f) return GradFactors{R.M, R.M_off, 0.0f, 0.0f};
  GradFactors g{R.M, R.M_off, __fdiv_rn(L.mass, R.S), 0.0f};
  const float off = (L.rho == 0.0f || R.S_off == 0.0f) ? 0.0f : __fdiv_rn(L.rho, R.S_off);
  g.f = __fmul_rn(by, __fsub_rn(__fmul_rn(g.q_of_e, exp_from(R.M_off, R.M, c)), off));
  return g;
}

// The gradient of the listed ids, over what the pass along the row wrote
// there (a barrier before).
template <typename T>
__device__ __forceinline__ void grad_list(const DistillArgs &A, const List &L, const GradFactors &g, T *grad, float by) {
  for (int j = threadIdx.x; j < A.K; j += kThreads) {
    const int id = L.id[j];
    if (id < 0) continue;
    const float e = exp_from(L.s[j], g.M, A.c);
    RowElem<T>::put(grad + id, g.q_of_e == 0.0f ? 0.0f : __fmul_rn(by, __fsub_rn(__fmul_rn(e, g.q_of_e), L.p[j])));
  }
}

// One batch of the pass along the row: e times f.
template <typename T>
__device__ __forceinline__ void grad_batch(uint4 *raw, float m, float c, float f) {
  constexpr int P = RowElem<T>::N / 2;
  const f32x2 m2 = pair(-m, -m), c2 = pair(c, c), f2 = pair(f, f);
#pragma unroll
  for (int i = 0; i < kBatch; i++) {
    f32x2 x[P];
    RowElem<T>::pairs(raw[i], x);
#pragma unroll
    for (int j = 0; j < P; j++) {
      float a, b;
      unpair(mul2(add2(x[j], m2), c2), a, b);
      x[j] = mul2(pair(exp2_approx(a), exp2_approx(b)), f2);
    }
    raw[i] = RowElem<T>::pack_pairs(x);
  }
}

// The batches from kb on, straight from global memory, the next one in flight
// while one is worked on (`now` holds the first).
template <typename T>
__device__ __forceinline__ void grad_stream(const Columns<T> &C, const Gradient<T> &G, const GradFactors &g, float c,
                                            int kb, uint4 *now) {
  uint4 next[kBatch];
  for (; kb < C.sp.k1; kb += 2 * kStep) {
    if (kb + kStep < C.sp.k1) C.load(kb + kStep, next);
    grad_batch<T>(now, g.M_off, c, g.f);
    G.store(C, kb, C.sp.k1, now);
    if (kb + kStep < C.sp.k1) {
      if (kb + 2 * kStep < C.sp.k1) C.load(kb + 2 * kStep, now);
      grad_batch<T>(next, g.M_off, c, g.f);
      G.store(C, kb + kStep, C.sp.k1, next);
    }
  }
}

// One batch into a thread's running maximum and sum (two sums, of the even
// and the odd columns).  REST: listed ids are left out; few batches hold any.
template <typename T, bool REST>
__device__ __forceinline__ void sum_batch(const List &L, const Columns<T> &C, float c, int flag_shift, uint4 *raw,
                                          int kb, float &m, f32x2 &s) {
  constexpr int N = RowElem<T>::N;
  if (REST) {
    if ((L.flags >> ((kb - C.sp.k0) / kStep >> flag_shift)) & 1u) {
#pragma unroll
      for (int i = 0; i < kBatch; i++) {
        const int u = (kb + static_cast<int>(threadIdx.x) + i * kThreads - C.sp.k0) * N;
        const uint32_t on = u < C.sp.c1 - C.sp.c0 ? (L.bits[u >> 5] >> (u & 31)) & ((1u << N) - 1u) : 0u;
        if (on != 0u) {
          float x[N];
          RowElem<T>::unpack(raw[i], x);
#pragma unroll
          for (int j = 0; j < N; j++)
            if ((on >> j) & 1u) x[j] = -INFINITY;
          raw[i] = RowElem<T>::pack(x);
        }
      }
    }
  }
  float top = m;
#pragma unroll
  for (int i = 0; i < kBatch; i++) top = fmaxf(top, RowElem<T>::max(raw[i]));
  const float base = top > -INFINITY ? top : 0.0f;
  const f32x2 m2 = pair(-base, -base), c2 = pair(c, c);
  const float scale = exp_from(m, base, c);
  s = mul2(s, pair(scale, scale));
  m = top;
#pragma unroll
  for (int i = 0; i < kBatch; i++) {
    f32x2 x[N / 2];
    RowElem<T>::pairs(raw[i], x);
#pragma unroll
    for (int j = 0; j < N / 2; j++) {
      float a, b;
      unpair(mul2(add2(x[j], m2), c2), a, b);
      s = add2(s, pair(exp2_approx(a), exp2_approx(b)));
    }
  }
}

template <typename T, bool REST, bool GRAD>
__global__ void __launch_bounds__(kThreads, kCtasPerSm) distill_kernel(const DistillArgs A) {
  __shared__ __align__(16) RowPart s_part[kMaxCluster];
  __shared__ MaxSum s_warp[kWarps][2];
  __shared__ double s_list[kWarps][2];
  __shared__ GradFactors s_factors;
  extern __shared__ __align__(16) unsigned char s_dyn[];
  const int part = cluster_rank();
  const int64_t row = cluster_id();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const Columns<T> C(static_cast<const T *>(A.logits) + row * A.ld, A.V, part, A.span);
  const float w = A.weight ? A.weight[row] : 1.0f;
  const float by = __fmul_rn(w, A.T);

  bool target = w != 0.0f;
  List L;
  uint4 now[kBatch];
  const Entry first(A, row);
  uint4 *held = reinterpret_cast<uint4 *>(s_dyn);
  const int k_held = GRAD ? min(C.sp.k0 + A.resident, C.sp.k1) : C.sp.k0;  // the vectors before stay on chip
  if (target) {
    if (GRAD) C.fetch(held, k_held);
    if (!GRAD) C.load(C.sp.k0, now);
    L = read_list<T, REST>(A, row, first, C.row, C.sp, s_dyn + static_cast<size_t>(A.resident) * 16);
    target = L.valid;
  }
  if (!target) {  // the whole cluster leaves
    if (GRAD) {
      asm volatile("cp.async.wait_all;" ::: "memory");
      Gradient<T>(static_cast<T *>(A.grad) + row * A.ld_grad, C.shift).zero(C);
    }
    if (part == 0 && tid == 0) {
      A.loss[row] = 0.0f;
      if (A.stats) A.stats[row] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    }
    return;
  }
  cluster_arrive_relaxed();

  // running maximum and sum of this thread's columns
  float m = -INFINITY;
  f32x2 s = pair(0.0f, 0.0f);
  {
    uint4 next[kBatch];
    int kb = k_held;
    if (GRAD && kb < C.sp.k1) C.load(kb, now);
    for (; kb < C.sp.k1; kb += 2 * kStep) {
      if (kb + kStep < C.sp.k1) C.load(kb + kStep, next);
      sum_batch<T, REST>(L, C, A.c, A.flag_shift, now, kb, m, s);
      if (kb + kStep < C.sp.k1) {
        if (kb + 2 * kStep < C.sp.k1) C.load(kb + 2 * kStep, now);
        sum_batch<T, REST>(L, C, A.c, A.flag_shift, next, kb + kStep, m, s);
      }
    }
  }
  if (GRAD) {
    asm volatile("cp.async.wait_all;" ::: "memory");  // a thread reads back what it fetched itself
    for (int kb = C.sp.k0; kb < k_held; kb += kStep) {
      C.held(held, kb, k_held, now);
      sum_batch<T, REST>(L, C, A.c, A.flag_shift, now, kb, m, s);
    }
  }
  MaxSum a{m, 0.0f};
  {
    float s0, s1;
    unpair(s, s0, s1);
    a.s = __fadd_rn(s0, s1);
  }
  a = join_lanes<32>(a, A.c);
  // and of its listed ids
  const int busy = min((A.K + 31) / 32, kWarps);
  if (REST && warp < busy) {
    MaxSum listed{-INFINITY, 0.0f};
    for (int j = tid; j < A.K; j += kThreads)
      if (L.id[j] >= 0) listed = join(listed, MaxSum{L.s[j], L.s[j] == -INFINITY ? 0.0f : 1.0f}, A.c);
    listed = join_lanes<32>(listed, A.c);
    if (lane == 0) s_warp[warp][1] = listed;
  }
  if (lane == 0) s_warp[warp][0] = a;
  __syncthreads();
  if (warp < busy) {
    RowPart r;
    r.row = join_lanes<kWarps>(s_warp[lane & (kWarps - 1)][0], A.c);
    r.list = MaxSum{-INFINITY, 0.0f};
    if (REST) r.list = join_lanes<kWarps>((lane & (kWarps - 1)) < busy ? s_warp[lane & (kWarps - 1)][1] : r.list, A.c);
    const double ref = r.ref();
    r.p = r.l = 0.0;
    for (int j = tid; j < A.K; j += kThreads) {
      const float p = L.p[j];
      if (L.id[j] < 0 || p == 0.0f) continue;
      r.p += p;
      r.l += p * (L.log_p[j] - (L.s[j] - ref) * A.inv_T);
    }
    r.p = sum_lanes<32>(r.p);
    r.l = sum_lanes<32>(r.l);
    if (busy > 1) {
      if (lane == 0) {
        s_list[warp][0] = r.p;
        s_list[warp][1] = r.l;
      }
      asm volatile("bar.sync 1, %0;" ::"r"(32 * busy) : "memory");  // of the warps with an entry
      r.p = r.l = 0.0;
      for (int i = 0; i < busy; i++) {
        r.p += s_list[i][0];
        r.l += s_list[i][1];
      }
    }
    if (warp == 0) {
      cluster_wait();  // every CTA of the row runs: its shared memory may be written
      if (lane < A.parts) put_remote(&s_part[part], r, lane);
      cluster_arrive();
    }
  }
  if (warp != 0) {
    cluster_wait();
    cluster_arrive_relaxed();
  }
  cluster_wait();
  if (warp == 0) {
    const RowPart none{{-INFINITY, 0.0f}, {-INFINITY, 0.0f}, 0.0, 0.0};
    const RowPart mine = lane < A.parts ? s_part[lane] : none;
    const MaxSum all = join_lanes<kMaxCluster>(mine.row, A.c);
    RowSums R{all.m, all.s, all.m, all.s};
    if (REST) {
      const MaxSum both = join(all, join_lanes<kMaxCluster>(mine.list, A.c), A.c);
      R.M = both.m;
      R.S = both.s;
    }
    if (!(R.M > -INFINITY)) R.M = 0.0f;
    if (!(R.M_off > -INFINITY)) R.M_off = R.M;
    if (GRAD && lane == 0) s_factors = grad_factors(L, R, A.c, by);
    if (GRAD) asm volatile("bar.arrive 2, %0;" ::"r"(kThreads) : "memory");  // the others go on; the loss can wait
    if (part == 0) {
      const double mass = sum_lanes<kMaxCluster>(mine.p);
      double l = sum_lanes<kMaxCluster>(mine.l - mine.p * ((static_cast<double>(mine.ref()) - R.M) * A.inv_T));
      if (lane == 0) {
        const double T_ = A.T, log_s = log(static_cast<double>(R.S));
        l += mass * log_s;
        if (L.rho != 0.0f)
          l += L.rho * (log(static_cast<double>(L.rho) / R.S_off) + log_s -
                        (static_cast<double>(R.M_off) - R.M) * A.inv_T);
        if (R.S == 0.0f) l = INFINITY;  // every logit is -inf: the student has no distribution
        A.loss[row] = static_cast<float>(static_cast<double>(w) * T_ * T_ * l);
        if (A.stats) A.stats[row] = make_float4(R.M, R.S, R.M_off, R.S_off);
      }
    }
    __syncwarp();
  } else if (GRAD) {
    asm volatile("bar.sync 2, %0;" ::"r"(kThreads) : "memory");
  }
  if constexpr (GRAD) {
    const GradFactors g = s_factors;
    const Gradient<T> G(static_cast<T *>(A.grad) + row * A.ld_grad, C.shift);
    for (int kb = C.sp.k0; kb < k_held; kb += kStep) {
      C.held(held, kb, k_held, now);
      grad_batch<T>(now, g.M_off, A.c, g.f);
      G.store(C, kb, k_held, now);
    }
    if (k_held < C.sp.k1) {
      C.load(k_held, now);
      grad_stream(C, G, g, A.c, k_held, now);
    }
    __syncthreads();
    grad_list(A, L, g, G.row, by);
  }
}

// The gradient from saved statistics: no sums are left to take, so the parts
// of a row are independent CTAs.
template <typename T, bool REST>
__global__ void __launch_bounds__(kThreads, kCtasPerSm) distill_backward_kernel(const DistillArgs A) {
  extern __shared__ __align__(16) unsigned char s_dyn[];
  const int part = static_cast<int>(blockIdx.x) % A.parts;
  const int64_t row = blockIdx.x / A.parts;
  const Columns<T> C(static_cast<const T *>(A.logits) + row * A.ld, A.V, part, A.span);
  const Gradient<T> G(static_cast<T *>(A.grad) + row * A.ld_grad, C.shift);
  const float w = A.weight ? A.weight[row] : 1.0f;
  const float up = A.grad_loss ? A.grad_loss[row] : 1.0f;
  const float4 st = A.stats[row];
  bool target = w != 0.0f;
  List L;
  uint4 now[kBatch];
  const Entry first(A, row);
  if (target) {
    C.load(C.sp.k0, now);
    L = read_list<T, REST>(A, row, first, C.row, C.sp, s_dyn);
    target = L.valid;
  }
  if (!target) {
    G.zero(C);
    return;
  }
  const float by = __fmul_rn(__fmul_rn(w, A.T), up);
  const GradFactors g = grad_factors(L, RowSums{st.x, st.y, st.z, st.w}, A.c, by);
  // (read_list has read the listed logits: the gradient may lie over them)
  grad_stream(C, G, g, A.c, C.sp.k0, now);
  __syncthreads();
  grad_list(A, L, g, G.row, by);
}

// The shared memory of a CTA: the resident vectors, a bit per column of its
// span, and the list.
template <typename T>
size_t distill_smem(DistillArgs &A) {
  A.bit_words = (A.span * RowElem<T>::N + 127) / 128 * 4;
  for (A.flag_shift = 0; (A.span - 1) / kStep >> A.flag_shift >= 32;) A.flag_shift++;
  return static_cast<size_t>(A.resident) * 16 +
         sizeof(uint32_t) * (static_cast<size_t>(A.bit_words) + 4 * static_cast<size_t>(A.K));
}

// CTAs per row, up to 8.  The loss alone: as many as fill one wave of the
// GPU's CTA slots (512 rows of 128256 f32: 42.4 us with two, 49.3 with three,
// 1.5 waves of them); one from there on, two where that leaves the second or
// third wave less than half full (1100 rows: 111 and 101 us; 2048: 155 and
// 160).  With the gradient: 32 KB of a row each, of which five CTAs share an
// SM's shared memory, more while the rows would leave slots empty; a row of
// more than 8 x 64 KB is read a second time beyond that.  Either way so many
// that a CTA's bits of its columns stay within 24 KB.
template <typename T, bool REST, bool GRAD>
cudaError_t launch_distill_as(DistillArgs &A, cudaStream_t st) {
  constexpr int N = RowElem<T>::N;
  const int vecs = (A.V + 2 * N - 2) / N;  // of a row with the largest shift
  const int slots = kCtasPerSm * current_sms(), wave = slots / A.N;
  const int least = (A.V + 24 * 1024 * 8 - 1) / (24 * 1024 * 8);  // by the bits
  const int batches = vecs / kStep;
  int parts;
  if (GRAD) {
    parts = (vecs + 2047) / 2048;
    if (parts < wave) parts = wave < batches ? wave : batches;
  } else {
    const int last = A.N % slots;
    parts = wave > 0 ? wave : A.N < 3 * slots && last > 0 && last < slots / 2 ? 2 : 1;
    parts = parts < batches ? parts : batches;
  }
  parts = parts > least ? parts : least;  // (at least one)
  parts = parts < kMaxCluster ? parts : kMaxCluster;
  A.parts = parts;
  A.span = (vecs + parts - 1) / parts;
  const int most = kResident / 16 / kStep * kStep;
  A.resident = GRAD ? (A.span < most ? A.span : most) : 0;
  const int64_t ctas = static_cast<int64_t>(A.N) * parts;
  if (ctas > 0x7FFFFFFF) return cudaErrorInvalidConfiguration;
  const size_t smem = distill_smem<T>(A);
  static std::atomic<uint64_t> ready{0};  // devices whose attribute is set
  cudaError_t e = allow_smem(reinterpret_cast<const void *>(distill_kernel<T, REST, GRAD>), 112 * 1024, &ready);
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(static_cast<unsigned>(ctas));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = parts;
  at[0].val.clusterDim.y = 1;
  at[0].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  e = cudaLaunchKernelEx(&cfg, distill_kernel<T, REST, GRAD>, A);
  return e != cudaSuccess ? e : cudaGetLastError();
}

template <bool GRAD>
cudaError_t launch_distill(DistillArgs &A, pz_dtype dtype, cudaStream_t st) {
  if (dtype == PZ_DTYPE_F32)
    return A.rest ? launch_distill_as<float, true, GRAD>(A, st) : launch_distill_as<float, false, GRAD>(A, st);
  return A.rest ? launch_distill_as<bf16_t, true, GRAD>(A, st) : launch_distill_as<bf16_t, false, GRAD>(A, st);
}

// The gradient alone: parts of 64 KB, smaller ones while the rows would leave
// SMs without a CTA.
template <typename T>
cudaError_t launch_backward(DistillArgs &A, cudaStream_t st) {
  constexpr int N = RowElem<T>::N;
  const int vecs = (A.V + 2 * N - 2) / N;
  A.parts = (vecs + 4095) / 4096;
  const int wave = kCtasPerSm * current_sms() / A.N, most = vecs / kThreads;
  if (A.parts < wave && A.parts < most) A.parts = wave < most ? wave : most;
  A.span = (vecs + A.parts - 1) / A.parts;
  const int64_t ctas = static_cast<int64_t>(A.N) * A.parts;
  if (ctas > 0x7FFFFFFF) return cudaErrorInvalidConfiguration;
  const size_t smem = distill_smem<T>(A);
  if (A.rest)
    distill_backward_kernel<T, true><<<static_cast<unsigned>(ctas), kThreads, smem, st>>>(A);
  else
    distill_backward_kernel<T, false><<<static_cast<unsigned>(ctas), kThreads, smem, st>>>(A);
  return cudaGetLastError();
}

// Checks what the three entries share and fills the arguments.
pz_status distill_args(const char *who, DistillArgs *A, const void *logits, pz_dtype dtype, int N, int V, int64_t ld,
                       const pz_distill_target *t) {
  static thread_local char msg[160];
  auto bad = [&](pz_status s, const char *why) {
    int n = 0;
    for (const char *p = who; *p && n < 60; p++) msg[n++] = *p;
    for (const char *p = ": "; *p; p++) msg[n++] = *p;
    for (const char *p = why; *p && n < 158; p++) msg[n++] = *p;
    msg[n] = 0;
    return report(s, msg);
  };
  if (!logits || !t || N < 0 || V <= 0 || ld < V) return bad(PZ_ERR_INVALID_ARGS, "null pointer or bad size");
  if (dtype != PZ_DTYPE_F32 && dtype != PZ_DTYPE_BF16) return bad(PZ_ERR_INVALID_ARGS, "bad dtype");
  if (!t->ids || !t->values || t->K <= 0 || t->ld_ids < t->K || t->ld_values < t->K)
    return bad(PZ_ERR_INVALID_ARGS, "the list needs ids, values and row strides of at least K > 0");
  if (t->mode != PZ_DISTILL_LIST && t->mode != PZ_DISTILL_REST) return bad(PZ_ERR_INVALID_ARGS, "bad mode");
  if (!(t->temperature >= 1e-6f && t->temperature <= 1e6f))
    return bad(PZ_ERR_INVALID_ARGS, "temperature outside [1e-6, 1e6]");
  if (misaligned(logits, elem_bytes(dtype)) || misaligned(t->ids, 4) || misaligned(t->values, 4) ||
      misaligned(t->n_list, 4) || misaligned(t->weight, 4))
    return bad(PZ_ERR_INVALID_ARGS, "pointer not aligned to its elements");
  if (t->K > PZ_TOP_K_MAX) return bad(PZ_ERR_UNSUPPORTED, "lists of more than 1024 ids");
  if (V > PZ_DISTILL_MAX_VOCAB) return bad(PZ_ERR_UNSUPPORTED, "more than 2^20 columns");
  A->logits = logits;
  A->ld = ld;
  A->N = N;
  A->V = V;
  A->ids = t->ids;
  A->values = t->values;
  A->K = t->K;
  A->ld_ids = t->ld_ids;
  A->ld_values = t->ld_values;
  A->n_list = t->n_list;
  A->weight = t->weight;
  A->T = t->temperature;
  A->c = static_cast<float>(1.4426950408889634 / static_cast<double>(t->temperature));
  A->inv_T = 1.0 / static_cast<double>(t->temperature);
  A->rest = t->mode == PZ_DISTILL_REST ? 1 : 0;
  return PZ_OK;
}

pz_status distill_grad_args(const char *who, DistillArgs *A, pz_dtype dtype, void *grad, int64_t ld_grad) {
  const size_t es = elem_bytes(dtype);
  if (!grad || ld_grad < A->V || misaligned(grad, es)) return report(PZ_ERR_INVALID_ARGS, who);
  if (A->N > 0 && (grad == A->logits ? ld_grad != A->ld
                                     : overlap(A->logits, rows_bytes(A->N, A->V, A->ld, es), grad,
                                               rows_bytes(A->N, A->V, ld_grad, es))))
    return report(PZ_ERR_INVALID_ARGS, who);
  A->grad = grad;
  A->ld_grad = ld_grad;
  return PZ_OK;
}

}  // namespace
}  // namespace pz

extern "C" {

pz_status pz_distill_forward(const void *logits, pz_dtype dtype, int N, int V, int64_t ld,
                             const pz_distill_target *target, float *loss, float *stats, void *stream) {
  pz::DistillArgs A{};
  pz_status s = pz::distill_args("pz_distill_forward", &A, logits, dtype, N, V, ld, target);
  if (s != PZ_OK) return s;
  if (!loss || pz::misaligned(loss, 4) || pz::misaligned(stats, 16))
    return pz::report(PZ_ERR_INVALID_ARGS, "pz_distill_forward: no loss, or loss or stats (16 bytes) not aligned");
  if (N == 0) return PZ_OK;
  A.loss = loss;
  A.stats = reinterpret_cast<float4 *>(stats);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const cudaError_t e = pz::launch_distill<false>(A, dtype, st);
  return e == cudaSuccess ? PZ_OK : pz::report_cuda(e);
}

pz_status pz_distill_backward(const void *logits, pz_dtype dtype, int N, int V, int64_t ld,
                              const pz_distill_target *target, const float *stats, const float *grad_loss, void *grad,
                              int64_t ld_grad, void *stream) {
  pz::DistillArgs A{};
  pz_status s = pz::distill_args("pz_distill_backward", &A, logits, dtype, N, V, ld, target);
  if (s != PZ_OK) return s;
  if (!stats || pz::misaligned(stats, 16) || pz::misaligned(grad_loss, 4))
    return pz::report(PZ_ERR_INVALID_ARGS, "pz_distill_backward: no stats, or stats (16 bytes) or grad_loss not aligned");
  s = pz::distill_grad_args("pz_distill_backward: grad is the logits' buffer itself (same ld) or apart from it", &A,
                            dtype, grad, ld_grad);
  if (s != PZ_OK || N == 0) return s;
  A.stats = reinterpret_cast<float4 *>(const_cast<float *>(stats));
  A.grad_loss = grad_loss;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const cudaError_t e =
      dtype == PZ_DTYPE_F32 ? pz::launch_backward<float>(A, st) : pz::launch_backward<pz::bf16_t>(A, st);
  return e == cudaSuccess ? PZ_OK : pz::report_cuda(e);
}

pz_status pz_distill_loss_grad(const void *logits, pz_dtype dtype, int N, int V, int64_t ld,
                               const pz_distill_target *target, float *loss, void *grad, int64_t ld_grad,
                               void *stream) {
  pz::DistillArgs A{};
  pz_status s = pz::distill_args("pz_distill_loss_grad", &A, logits, dtype, N, V, ld, target);
  if (s != PZ_OK) return s;
  if (!loss || pz::misaligned(loss, 4))
    return pz::report(PZ_ERR_INVALID_ARGS, "pz_distill_loss_grad: no loss, or loss not aligned");
  s = pz::distill_grad_args("pz_distill_loss_grad: grad is the logits' buffer itself (same ld) or apart from it", &A,
                            dtype, grad, ld_grad);
  if (s != PZ_OK || N == 0) return s;
  A.loss = loss;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const cudaError_t e = pz::launch_distill<true>(A, dtype, st);
  return e == cudaSuccess ? PZ_OK : pz::report_cuda(e);
}

}  // extern "C"
