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
// their shape).  Sums of e are fp32, at most a few hundred terms per thread,
// joined in a fixed order: the same call gives the same bits.  REST keeps
// the ids off the list under a maximum of their own, so that log r and
// rho / r hold when the student leaves them next to nothing.  The sum over
// the list, whose terms nearly cancel against log S, is in fp64.
//
// Bound: HBM.  The loss reads the logits once; the gradient from saved
// statistics reads and writes once; loss and gradient together read once and
// write once, because a row stays on chip between its two passes: a cluster
// of up to 8 CTAs takes a row, each CTA holding 64 KB of it in registers
// (512 threads x 8 vectors of 16 bytes, two CTAs per SM), and they exchange
// maximum and sums through distributed shared memory.  Columns beyond
// 8 x 64 KB are read a second time (from L2, mostly: the rows in flight are
// at most 148 x 2 / 8 of them).
#include "pz_device.cuh"
#include "pz_rowvec.cuh"
#include "pz_status.cuh"

namespace pz {
namespace {

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr int kBatch = 4;              // 16-byte vectors that a thread has in flight
constexpr int kMaxCluster = 8;         // the portable cluster size
constexpr int kCtasPerSm = 4;

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
  int rest;
  float *loss;
  float4 *stats;
  void *grad;
  int64_t ld_grad;
  int parts;  // CTAs per row (the cluster's size in distill_kernel)
  int span;   // vectors per CTA
  int bit_words;  // words of a CTA's bits of listed columns, a multiple of 4
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
  int32_t *id;     // [K]; -1: ignored, or a later entry of an id listed twice
  float *p;        // [K] probabilities
  uint32_t *bits;  // one bit per column of the CTA's span: listed
  double sum_p;
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

// Reads the row's list: ids and probabilities, their sum, rho, and the bits
// of the ids in [c0, c1).  Two barriers of the block, the second one last.
__device__ __forceinline__ List read_list(const DistillArgs &A, int64_t row, int c0, int c1, unsigned char *smem,
                                          int bit_words) {
  __shared__ float s_top[kWarps];
  __shared__ int s_seen[kWarps], s_bad[kWarps];
  __shared__ double s_sum[kWarps];
  __shared__ int s_twice, s_gap;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  List L;
  L.bits = reinterpret_cast<uint32_t *>(smem);
  L.id = reinterpret_cast<int32_t *>(L.bits + bit_words);
  L.p = reinterpret_cast<float *>(L.id + A.K);
  const int32_t *ids = A.ids + row * A.ld_ids;
  const float *values = A.values + row * A.ld_values;
  const int n = A.n_list ? min(max(A.n_list[row], 0), A.K) : A.K;
  float top = -INFINITY;
  int seen = 0, bad = 0;
  for (int j = tid; j < A.K; j += kThreads) {
    int id = ids[j];
    const float v = values[j];
    float t = -INFINITY;
    if (j >= n || id < 0 || id >= A.V) {
      id = -1;
    } else {
      t = A.rest ? v : __fdiv_rn(v, A.T);
      seen++;
      bad |= t != t;
      top = fmaxf(top, t);
    }
    L.id[j] = id;
    L.p[j] = t;
  }
  for (int i = tid; i < bit_words / 4; i += kThreads) reinterpret_cast<uint4 *>(L.bits)[i] = make_uint4(0u, 0u, 0u, 0u);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, o));
  seen = __reduce_add_sync(0xFFFFFFFFu, seen);
  bad = __any_sync(0xFFFFFFFFu, bad);
  if (lane == 0) {
    s_top[warp] = top;
    s_seen[warp] = seen;
    s_bad[warp] = bad;
  }
  if (tid == 0) s_twice = s_gap = 0;
  __syncthreads();
  seen = 0;
  for (int i = 0; i < kWarps; i++) {
    top = fmaxf(top, s_top[i]);
    seen += s_seen[i];
    bad |= s_bad[i];
  }
  // LIST: relative to the largest; REST: as they are
  const float base = (A.rest || !(top > -INFINITY)) ? 0.0f : top;
  double sum = 0.0;
  for (int j = tid; j < A.K; j += kThreads) {
    const int id = L.id[j];
    const float p = id >= 0 ? expf(__fsub_rn(L.p[j], base)) : 0.0f;
    L.p[j] = p;
    sum += p;
    if (id >= 0 && id >= c0 && id < c1) {
      const uint32_t bit = 1u << ((id - c0) & 31);
      if (atomicOr(&L.bits[(id - c0) >> 5], bit) & bit) s_twice = 1;
    }
  }
  // A list that names every id leaves none for rho (what 1 - sum holds then
  // is rounding).
  const bool whole = A.rest && seen >= A.V;
  if (whole) {
    for (int v = tid; v < A.V; v += kThreads) {
      bool on = false;
      for (int j = 0; j < A.K; j++) on |= L.id[j] == v;
      if (!on) s_gap = 1;
    }
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, o);
  if (lane == 0) s_sum[warp] = sum;
  __syncthreads();
  sum = 0.0;
  for (int i = 0; i < kWarps; i++) sum += s_sum[i];
  if (!A.rest) {
    const float inv = static_cast<float>(1.0 / sum);
    for (int j = tid; j < A.K; j += kThreads)
      if (L.id[j] >= 0) L.p[j] = __fmul_rn(L.p[j], inv);
    if (sum == sum) sum = 1.0;  // a NaN value makes the row's outputs NaN
  }
  L.sum_p = sum;
  // (an unordered comparison keeps a NaN sum: the row's outputs are NaN then)
  L.rho = (A.rest && !(whole && !s_gap) && !(sum >= 1.0)) ? static_cast<float>(1.0 - sum) : 0.0f;
  // no entries: no target.  LIST with no finite value: none either.
  L.valid = seen > 0 && (A.rest || top > -INFINITY || bad);
  if (s_twice) {
    // the first entry of an id takes the probabilities of all, in list order
    __syncthreads();
    float joined[PZ_TOP_K_MAX / kThreads];
#pragma unroll
    for (int e = 0; e < PZ_TOP_K_MAX / kThreads; e++) {
      const int j = tid + e * kThreads;
      joined[e] = -1.0f;
      if (j < A.K && L.id[j] >= 0) {
        float all = 0.0f;
        bool first = true;
        for (int i = 0; i < A.K; i++)
          if (L.id[i] == L.id[j]) {
            first &= i >= j;
            all = __fadd_rn(all, L.p[i]);
          }
        if (first) joined[e] = all;
      }
    }
    __syncthreads();
#pragma unroll
    for (int e = 0; e < PZ_TOP_K_MAX / kThreads; e++) {
      const int j = tid + e * kThreads;
      if (j < A.K) {
        if (joined[e] == -1.0f) L.id[j] = -1;
        L.p[j] = joined[e];
      }
    }
  }
  return L;
}

template <typename T>
__device__ __forceinline__ void zero_span(T *row, const Span<T> &sp, int V, bool aligned) {
  constexpr int N = RowElem<T>::N;
  float x[N];
#pragma unroll
  for (int j = 0; j < N; j++) x[j] = 0.0f;
  for (int k = sp.k0 + threadIdx.x; k < sp.k1; k += kThreads)
    store_row_vec<N>(row, V, sp.c0 + (k - sp.k0) * N, x, aligned);
}

// kBatch vectors of the span, from vector k on, kThreads apart.
template <typename T>
__device__ __forceinline__ void load_batch(const T *row, int shift, int V, int k, int k1, uint4 *raw) {
#pragma unroll
  for (int i = 0; i < kBatch; i++)
    if (k + i * kThreads < k1) raw[i] = load_row_vec(row, shift, V, k + i * kThreads);
}

// A maximum and the sum of e relative to it.
struct MaxSum {
  float m, s;
};
__device__ __forceinline__ MaxSum join(const MaxSum &a, const MaxSum &b, float c) {
  MaxSum r;
  r.m = fmaxf(a.m, b.m);
  const float base = r.m > -INFINITY ? r.m : 0.0f;  // a side at -inf has s = 0 (or NaN, which stays)
  r.s = __fadd_rn(__fmul_rn(a.s, exp2_approx(__fmul_rn(__fsub_rn(a.m, base), c))),
                  __fmul_rn(b.s, exp2_approx(__fmul_rn(__fsub_rn(b.m, base), c))));
  return r;
}
__device__ __forceinline__ MaxSum join_warp(MaxSum a, float c) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const MaxSum b{__shfl_xor_sync(0xFFFFFFFFu, a.m, o), __shfl_xor_sync(0xFFFFFFFFu, a.s, o)};
    a = join(a, b, c);
  }
  return a;
}

// A CTA's part of its row's sums (warps hand in `row` and `list`).
struct RowPart {
  MaxSum row;          // its columns (REST: those off the list)
  MaxSum list;         // REST: its listed ids
  // over its listed ids: sum p, sum p log p, and sum p (s - ref), ref being
  // the CTA's own maximum: the differences are taken before the sums, which
  // would lose them in rows of the type's lowest value
  double p, plogp, ps, pad;
  __device__ __forceinline__ float ref() const {
    const float m = fmaxf(row.m, list.m);
    return m > -INFINITY ? m : 0.0f;
  }
};

// The row's cluster: all CTAs have to arrive before any passes the wait.
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire;" ::: "memory"); }

// Copies *v to the same shared variable of CTA `rank` of the cluster.
__device__ __forceinline__ void put_remote(const RowPart *slot, const RowPart &v, int rank) {
  uint32_t at;
  asm("mapa.shared::cluster.u32 %0, %1, %2;"
      : "=r"(at)
      : "r"(static_cast<uint32_t>(__cvta_generic_to_shared(slot))), "r"(rank));
  static_assert(sizeof(RowPart) == 48, "three 16-byte stores");
  asm volatile("st.shared::cluster.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(at), "f"(v.row.m), "f"(v.row.s), "f"(v.list.m),
               "f"(v.list.s)
               : "memory");
  asm volatile("st.shared::cluster.v2.f64 [%0], {%1, %2};" ::"r"(at + 16), "d"(v.p), "d"(v.plogp) : "memory");
  asm volatile("st.shared::cluster.v2.f64 [%0], {%1, %2};" ::"r"(at + 32), "d"(v.ps), "d"(v.pad) : "memory");
}

// The row's sums: M and S over all ids, M_off and S_off over those whose
// gradient is the pass along the row's (LIST: all; REST: off the list).
struct RowSums {
  float M, S, M_off, S_off;
};

// What the passes multiply e by.
struct GradFactors {
  float q_of_e;  // listed ids, e relative to M: P / S
  float f;       // the others, e relative to M_off: w T (P / S 2^((M_off - M) c) - rho / S_off)
};
__device__ __forceinline__ GradFactors grad_factors(const List &L, const RowSums &R, float c, float by) {
  // a row without any weight (every logit -inf): its gradient is 0
  if (R.S == 0.0f) return GradFactors{0.0f, 0.0f};
  const float P = __fadd_rn(static_cast<float>(L.sum_p), L.rho);
  GradFactors g;
  g.q_of_e = __fdiv_rn(P, R.S);
  const float off = (L.rho == 0.0f || R.S_off == 0.0f) ? 0.0f : __fdiv_rn(L.rho, R.S_off);
  const float q = __fmul_rn(g.q_of_e, exp2_approx(__fmul_rn(__fsub_rn(R.M_off, R.M), c)));
  g.f = __fmul_rn(by, __fsub_rn(q, off));
  return g;
}

// One batch of the pass along the row: e times f.
template <typename T>
__device__ __forceinline__ void grad_batch(const uint4 *raw, const Span<T> &sp, int k, int V, T *grad, bool aligned,
                                           float m, float c, float f) {
  constexpr int N = RowElem<T>::N;
#pragma unroll
  for (int i = 0; i < kBatch; i++) {
    const int at = k + i * kThreads;
    if (at < sp.k1) {
      float x[N];
      RowElem<T>::unpack(raw[i], x);
#pragma unroll
      for (int j = 0; j < N; j++) x[j] = __fmul_rn(exp2_approx(__fmul_rn(__fsub_rn(x[j], m), c)), f);
      store_row_vec<N>(grad, V, sp.c0 + (at - sp.k0) * N, x, aligned);
    }
  }
}

// The pass along the row, the next batch in flight while one is worked on;
// then the listed ids get their own gradient over what the pass wrote there.
// Their logits are read before it: the gradient may lie over the logits.
template <typename T>
__device__ __forceinline__ void write_gradient(const DistillArgs &A, const List &L, const Span<T> &sp, const T *row,
                                               int shift, T *grad, bool aligned, const RowSums &R, float by) {
  constexpr int STEP = kBatch * kThreads;
  const GradFactors g = grad_factors(L, R, A.c, by);
  constexpr int E = PZ_TOP_K_MAX / kThreads;
  float own[E];
#pragma unroll
  for (int e = 0; e < E; e++) {
    const int j = static_cast<int>(threadIdx.x) + e * kThreads;
    own[e] = 0.0f;
    if (j < A.K) {
      const int id = L.id[j];
      if (id >= 0 && id >= sp.c0 && id < sp.c1) own[e] = RowElem<T>::get(row + id);
    }
  }
  int k = sp.k0 + static_cast<int>(threadIdx.x);
  uint4 a[kBatch], b[kBatch];
  load_batch(row, shift, A.V, k, sp.k1, a);
  // every listed logit of the span has been read (their values are used
  // below, behind this barrier's wait for the loads)
#pragma unroll
  for (int e = 0; e < E; e++) {
    const float x = exp2_approx(__fmul_rn(__fsub_rn(own[e], R.M), A.c));
    own[e] = __fmul_rn(x, g.q_of_e);
  }
  __syncthreads();
  for (; k < sp.k1; k += 2 * STEP) {
    load_batch(row, shift, A.V, k + STEP, sp.k1, b);
    grad_batch(a, sp, k, A.V, grad, aligned, R.M_off, A.c, g.f);
    load_batch(row, shift, A.V, k + 2 * STEP, sp.k1, a);
    grad_batch(b, sp, k + STEP, A.V, grad, aligned, R.M_off, A.c, g.f);
  }
  __syncthreads();
#pragma unroll
  for (int e = 0; e < E; e++) {
    const int j = static_cast<int>(threadIdx.x) + e * kThreads;
    if (j < A.K) {
      const int id = L.id[j];
      if (id >= 0 && id >= sp.c0 && id < sp.c1)
        RowElem<T>::put(grad + id, g.q_of_e == 0.0f ? 0.0f : __fmul_rn(by, __fsub_rn(own[e], L.p[j])));
    }
  }
}

// One batch into a thread's running maximum and sum.  REST: listed ids are
// left out.
template <typename T>
__device__ __forceinline__ void sum_batch(const DistillArgs &A, const List &L, const Span<T> &sp, uint4 *raw, int k,
                                          MaxSum &a) {
  constexpr int N = RowElem<T>::N;
  float x[N];
  float top = a.m;
#pragma unroll
  for (int i = 0; i < kBatch; i++) {
    const int at = k + i * kThreads;
    if (at >= sp.k1) {
      raw[i] = make_uint4(RowElem<T>::kNegInf2, RowElem<T>::kNegInf2, RowElem<T>::kNegInf2, RowElem<T>::kNegInf2);
    } else if (A.rest) {
      const int u = (at - sp.k0) * N;
      const uint32_t on = (L.bits[u >> 5] >> (u & 31)) & ((1u << N) - 1u);
      if (on != 0u) {
        RowElem<T>::unpack(raw[i], x);
#pragma unroll
        for (int j = 0; j < N; j++)
          if ((on >> j) & 1u) x[j] = -INFINITY;
        raw[i] = RowElem<T>::pack(x);
      }
    }
    RowElem<T>::unpack(raw[i], x);
#pragma unroll
    for (int j = 0; j < N; j++) top = fmaxf(top, x[j]);
  }
  const float base = top > -INFINITY ? top : 0.0f;
  float s = __fmul_rn(a.s, exp2_approx(__fmul_rn(__fsub_rn(a.m, base), A.c)));
#pragma unroll
  for (int i = 0; i < kBatch; i++) {
    RowElem<T>::unpack(raw[i], x);
#pragma unroll
    for (int j = 0; j < N; j++) s = __fadd_rn(s, exp2_approx(__fmul_rn(__fsub_rn(x[j], base), A.c)));
  }
  a = MaxSum{top, s};
}

template <typename T, bool GRAD>
__global__ void __launch_bounds__(kThreads, kCtasPerSm) distill_kernel(const DistillArgs A) {
  constexpr int STEP = kBatch * kThreads;
  __shared__ __align__(16) RowPart s_part[kMaxCluster];
  __shared__ MaxSum s_warp[kWarps][2];
  extern __shared__ __align__(16) unsigned char s_dyn[];
  const int part = static_cast<int>(blockIdx.x) % A.parts;
  const int64_t row = blockIdx.x / A.parts;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const T *x_row = static_cast<const T *>(A.logits) + row * A.ld;
  const int shift = row_shift(x_row);
  const Span<T> sp(part, A.span, A.V, shift);
  T *g_row = GRAD ? static_cast<T *>(A.grad) + row * A.ld_grad : nullptr;
  const bool aligned =
      GRAD && ((reinterpret_cast<uintptr_t>(g_row) - static_cast<uintptr_t>(shift) * sizeof(T)) & 15u) == 0;
  const float w = A.weight ? A.weight[row] : 1.0f;

  bool target = w != 0.0f;
  List L;
  uint4 ra[kBatch], rb[kBatch];
  int k = sp.k0 + tid;
  if (target) {
    load_batch(x_row, shift, A.V, k, sp.k1, ra);
    L = read_list(A, row, sp.c0, sp.c1, s_dyn, A.bit_words);
    target = L.valid;
  }
  if (!target) {  // the whole cluster leaves
    if (GRAD) zero_span(g_row, sp, A.V, aligned);
    if (part == 0 && tid == 0) {
      A.loss[row] = 0.0f;
      if (A.stats) A.stats[row] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    }
    return;
  }
  cluster_arrive();

  // running maximum and sum of this thread's columns
  MaxSum a{-INFINITY, 0.0f};
  for (; k < sp.k1; k += 2 * STEP) {
    load_batch(x_row, shift, A.V, k + STEP, sp.k1, rb);
    sum_batch(A, L, sp, ra, k, a);
    load_batch(x_row, shift, A.V, k + 2 * STEP, sp.k1, ra);
    if (k + STEP < sp.k1) sum_batch(A, L, sp, rb, k + STEP, a);
  }
  // and of its listed ids
  MaxSum listed{-INFINITY, 0.0f};
  if (A.rest) {
    for (int j = tid; j < A.K; j += kThreads) {
      const int id = L.id[j];
      if (id < 0 || id < sp.c0 || id >= sp.c1) continue;
      const float sv = RowElem<T>::get(x_row + id);
      listed = join(listed, MaxSum{sv, sv == -INFINITY ? 0.0f : 1.0f}, A.c);
    }
    listed = join_warp(listed, A.c);
  }
  a = join_warp(a, A.c);
  if (lane == 0) {
    s_warp[warp][0] = a;
    s_warp[warp][1] = listed;
  }
  __syncthreads();
  RowPart r{s_warp[0][0], s_warp[0][1], 0.0, 0.0, 0.0, 0.0};
  for (int i = 1; i < kWarps; i++) {
    r.row = join(r.row, s_warp[i][0], A.c);
    r.list = join(r.list, s_warp[i][1], A.c);
  }
  const double ref = r.ref();
  for (int j = tid; j < A.K; j += kThreads) {
    const int id = L.id[j];
    const float p = L.p[j];
    if (id < 0 || id < sp.c0 || id >= sp.c1 || p == 0.0f) continue;
    r.p += p;
    r.plogp += static_cast<double>(p) * logf(p);
    r.ps += static_cast<double>(p) * (RowElem<T>::get(x_row + id) - ref);
  }
  if (A.K > 32) {  // entries in several warps
    __shared__ double s_list[kWarps][3];
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      r.p += __shfl_xor_sync(0xFFFFFFFFu, r.p, o);
      r.plogp += __shfl_xor_sync(0xFFFFFFFFu, r.plogp, o);
      r.ps += __shfl_xor_sync(0xFFFFFFFFu, r.ps, o);
    }
    if (lane == 0) {
      s_list[warp][0] = r.p;
      s_list[warp][1] = r.plogp;
      s_list[warp][2] = r.ps;
    }
    __syncthreads();
    r.p = r.plogp = r.ps = 0.0;
    for (int i = 0; i < kWarps; i++) {
      r.p += s_list[i][0];
      r.plogp += s_list[i][1];
      r.ps += s_list[i][2];
    }
  } else if (warp == 0) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      r.p += __shfl_xor_sync(0xFFFFFFFFu, r.p, o);
      r.plogp += __shfl_xor_sync(0xFFFFFFFFu, r.plogp, o);
      r.ps += __shfl_xor_sync(0xFFFFFFFFu, r.ps, o);
    }
  }
  cluster_wait();  // every CTA of the row runs: its shared memory may be written
  if (tid < A.parts) put_remote(&s_part[part], r, tid);
  cluster_arrive();
  cluster_wait();
  RowPart all = s_part[0];
  for (int i = 1; i < A.parts; i++) {
    all.row = join(all.row, s_part[i].row, A.c);
    all.list = join(all.list, s_part[i].list, A.c);
  }
  RowSums R{all.row.m, all.row.s, all.row.m, all.row.s};
  if (A.rest) {
    const MaxSum both = join(all.row, all.list, A.c);
    R.M = both.m;
    R.S = both.s;
  }
  if (!(R.M > -INFINITY)) R.M = 0.0f;
  if (!(R.M_off > -INFINITY)) R.M_off = R.M;
  if (part == 0 && tid == 0) {
    const double T_ = A.T, log_s = log(static_cast<double>(R.S));
    double l = 0.0, mass = 0.0;
    for (int i = 0; i < A.parts; i++) {
      const RowPart &q = s_part[i];
      l += q.plogp - (q.ps + q.p * (static_cast<double>(q.ref()) - R.M)) / T_;
      mass += q.p;
    }
    l += mass * log_s;
    if (L.rho != 0.0f)
      l += L.rho * (log(static_cast<double>(L.rho)) - log(static_cast<double>(R.S_off)) + log_s -
                    (static_cast<double>(R.M_off) - R.M) / T_);
    if (R.S == 0.0f) l = INFINITY;  // every logit is -inf: the student has no distribution
    A.loss[row] = static_cast<float>(static_cast<double>(w) * T_ * T_ * l);
    if (A.stats) A.stats[row] = make_float4(R.M, R.S, R.M_off, R.S_off);
  }
  if constexpr (GRAD) write_gradient(A, L, sp, x_row, shift, g_row, aligned, R, __fmul_rn(w, A.T));
}

// The gradient from saved statistics: no sums are left to take, so the parts
// of a row are independent CTAs.
template <typename T>
__global__ void __launch_bounds__(kThreads, kCtasPerSm) distill_backward_kernel(const DistillArgs A) {
  extern __shared__ __align__(16) unsigned char s_dyn[];
  const int part = static_cast<int>(blockIdx.x) % A.parts;
  const int64_t row = blockIdx.x / A.parts;
  const T *x_row = static_cast<const T *>(A.logits) + row * A.ld;
  const int shift = row_shift(x_row);
  const Span<T> sp(part, A.span, A.V, shift);
  T *g_row = static_cast<T *>(A.grad) + row * A.ld_grad;
  const bool aligned = ((reinterpret_cast<uintptr_t>(g_row) - static_cast<uintptr_t>(shift) * sizeof(T)) & 15u) == 0;
  const float w = A.weight ? A.weight[row] : 1.0f;
  const float up = A.grad_loss ? A.grad_loss[row] : 1.0f;
  const float4 st = A.stats[row];
  bool target = w != 0.0f;
  List L;
  if (target) {
    L = read_list(A, row, sp.c0, sp.c1, s_dyn, A.bit_words);
    target = L.valid;
  }
  if (!target) {
    zero_span(g_row, sp, A.V, aligned);
    return;
  }
  write_gradient(A, L, sp, x_row, shift, g_row, aligned, RowSums{st.x, st.y, st.z, st.w},
                 __fmul_rn(__fmul_rn(w, A.T), up));
}

// The shared memory of a CTA: a bit per column of its span, and the list.
template <typename T>
size_t distill_smem(DistillArgs &A) {
  A.bit_words = (A.span * RowElem<T>::N + 127) / 128 * 4;
  return sizeof(uint32_t) * (static_cast<size_t>(A.bit_words) + 2 * static_cast<size_t>(A.K));
}

// CTAs per row.  The loss alone: whole rows while they fill the GPU's CTA
// slots.  With the gradient: 64 KB of a row each, so that the rows in flight
// stay in L2 for their second pass.  Either way more, up to 8, while the rows
// would leave slots empty, and so many that a CTA's bits of its columns
// stay within 24 KB (four CTAs share an SM).
template <typename T, bool GRAD>
cudaError_t launch_distill(DistillArgs &A, cudaStream_t st) {
  constexpr int N = RowElem<T>::N;
  const int vecs = (A.V + 2 * N - 2) / N;  // of a row with the largest shift
  int parts = GRAD ? (vecs + 4095) / 4096 : 1;
  const int bits = (A.V + 24 * 1024 * 8 - 1) / (24 * 1024 * 8);
  parts = parts > bits ? parts : bits;
  while (parts < kMaxCluster && static_cast<int64_t>(A.N) * parts < kCtasPerSm * current_sms() &&
         vecs > parts * kBatch * kThreads)
    parts++;
  parts = parts < kMaxCluster ? parts : kMaxCluster;
  A.parts = parts;
  A.span = (vecs + parts - 1) / parts;
  const int64_t ctas = static_cast<int64_t>(A.N) * parts;
  if (ctas > 0x7FFFFFFF) return cudaErrorInvalidConfiguration;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(static_cast<unsigned>(ctas));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = distill_smem<T>(A);
  cfg.stream = st;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = parts;
  at[0].val.clusterDim.y = 1;
  at[0].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, distill_kernel<T, GRAD>, A);
  return e != cudaSuccess ? e : cudaGetLastError();
}

// The gradient alone: parts of 64 KB.
template <typename T>
cudaError_t launch_backward(DistillArgs &A, cudaStream_t st) {
  constexpr int N = RowElem<T>::N;
  const int vecs = (A.V + 2 * N - 2) / N;
  A.parts = (vecs + 4095) / 4096;
  while (static_cast<int64_t>(A.N) * A.parts < kCtasPerSm * current_sms() && vecs > A.parts * kThreads) A.parts *= 2;
  A.span = (vecs + A.parts - 1) / A.parts;
  const int64_t ctas = static_cast<int64_t>(A.N) * A.parts;
  if (ctas > 0x7FFFFFFF) return cudaErrorInvalidConfiguration;
  const size_t smem = distill_smem<T>(A);
  distill_backward_kernel<T><<<static_cast<unsigned>(ctas), kThreads, smem, st>>>(A);
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
  if (misaligned(logits, elem_bytes(dtype))) return bad(PZ_ERR_INVALID_ARGS, "pointer not aligned to its elements");
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
  if (!loss || pz::misaligned(stats, 16))
    return pz::report(PZ_ERR_INVALID_ARGS, "pz_distill_forward: no loss, or stats not 16-byte aligned");
  if (N == 0) return PZ_OK;
  A.loss = loss;
  A.stats = reinterpret_cast<float4 *>(stats);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const cudaError_t e = dtype == PZ_DTYPE_F32 ? pz::launch_distill<float, false>(A, st)
                                              : pz::launch_distill<pz::bf16_t, false>(A, st);
  return e == cudaSuccess ? PZ_OK : pz::report_cuda(e);
}

pz_status pz_distill_backward(const void *logits, pz_dtype dtype, int N, int V, int64_t ld,
                              const pz_distill_target *target, const float *stats, const float *grad_loss, void *grad,
                              int64_t ld_grad, void *stream) {
  pz::DistillArgs A{};
  pz_status s = pz::distill_args("pz_distill_backward", &A, logits, dtype, N, V, ld, target);
  if (s != PZ_OK) return s;
  if (!stats || pz::misaligned(stats, 16))
    return pz::report(PZ_ERR_INVALID_ARGS, "pz_distill_backward: stats missing or not 16-byte aligned");
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
  if (!loss) return pz::report(PZ_ERR_INVALID_ARGS, "pz_distill_loss_grad: no loss");
  s = pz::distill_grad_args("pz_distill_loss_grad: grad is the logits' buffer itself (same ld) or apart from it", &A,
                            dtype, grad, ld_grad);
  if (s != PZ_OK || N == 0) return s;
  A.loss = loss;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const cudaError_t e = dtype == PZ_DTYPE_F32 ? pz::launch_distill<float, true>(A, st)
                                              : pz::launch_distill<pz::bf16_t, true>(A, st);
  return e == cudaSuccess ? PZ_OK : pz::report_cuda(e);
}

}  // extern "C"
