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

constexpr int kRes = 8;                // vectors of a thread that stay in registers
constexpr int kDistillThreads = 512;
constexpr int kMaxCluster = 8;         // the portable cluster size
constexpr int kBackThreads = 256;

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
};

// 2^x, fp32 results below 2^-126 flushed to zero (they are lost in any sum
// with the 1 that the row's maximum contributes).
__device__ __forceinline__ float exp2_approx(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// What a CTA knows about its row's list.
struct ListShared {
  int32_t id[PZ_TOP_K_MAX];   // -1: ignored
  float p[PZ_TOP_K_MAX];
  float own_p[PZ_TOP_K_MAX];  // probability of the entry's id, at the first entry of an id in this CTA's columns; else -1
  float own_s[PZ_TOP_K_MAX];  // the student's logit there
  double sum_p;
  float rho;
  int valid;                  // the row has a target
  int twice;                  // an id is listed twice in this CTA's columns
};

// Reads the row's list into L: ids, probabilities, their sum and rho.  Warp 0
// works out the probabilities; every thread of the block calls this, and a
// barrier has to follow.
__device__ __forceinline__ void read_list(const DistillArgs &A, int row, ListShared &L) {
  const int tid = threadIdx.x, lane = tid & 31;
  if (tid >= 32) return;
  const int32_t *ids = A.ids + row * A.ld_ids;
  const float *values = A.values + row * A.ld_values;
  const int n = A.n_list ? min(max(A.n_list[row], 0), A.K) : A.K;
  float top = -INFINITY;
  int seen = 0, bad = 0;
  for (int j = lane; j < A.K; j += 32) {
    int id = j < n ? ids[j] : -1;
    if (id >= A.V) id = -1;
    if (id < 0) id = -1;
    float t = -INFINITY;
    if (id >= 0) {
      t = A.rest ? values[j] : __fdiv_rn(values[j], A.T);
      seen++;
      bad |= t != t;
      top = fmaxf(top, t);
    }
    L.id[j] = id;
    L.p[j] = t;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, o));
    seen += __shfl_xor_sync(0xFFFFFFFFu, seen, o);
    bad |= __shfl_xor_sync(0xFFFFFFFFu, bad, o);
  }
  // LIST: relative to the largest; REST: as they are
  const float base = (A.rest || !(top > -INFINITY)) ? 0.0f : top;
  double sum = 0.0;
  for (int j = lane; j < A.K; j += 32) {
    const float p = L.id[j] >= 0 ? expf(__fsub_rn(L.p[j], base)) : 0.0f;
    L.p[j] = p;
    sum += p;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, o);
  if (!A.rest) {
    const float inv = static_cast<float>(1.0 / sum);
    sum = 0.0;
    for (int j = lane; j < A.K; j += 32) {
      if (L.id[j] >= 0) L.p[j] = __fmul_rn(L.p[j], inv);
      sum += L.p[j];
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, o);
  }
  // A list that names every id leaves none for rho (what 1 - sum holds then
  // is rounding).
  bool whole = A.rest && seen >= A.V;
  if (whole) {
    __syncwarp();
    for (int v = lane; v < A.V; v += 32) {
      bool on = false;
      for (int j = 0; j < A.K; j++) on |= L.id[j] == v;
      whole &= on;
    }
    whole = __all_sync(0xFFFFFFFFu, whole);
  }
  if (lane == 0) {
    L.sum_p = sum;  // of the probabilities as they are held
    // (an unordered comparison keeps a NaN sum: the row's outputs are NaN then)
    L.rho = (A.rest && !whole && !(sum >= 1.0)) ? static_cast<float>(1.0 - sum) : 0.0f;
    // no entries: no target.  LIST with no finite value: none either.
    L.valid = seen > 0 && (A.rest || top > -INFINITY || bad);
    L.twice = 0;
  }
}

// The first column of this CTA's span and one past its last, for the row
// whose columns start `shift` elements after a 16-byte boundary.
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

// The list's entries in the columns [c0, c1): one bit per column in `bits`,
// the student's logits in own_s.  The bits are zero before; barriers before
// (read_list) and after.
template <typename T>
__device__ __forceinline__ void mark_list(const DistillArgs &A, ListShared &L, uint32_t *bits, const T *row, int c0,
                                          int c1, int nt) {
  for (int j = threadIdx.x; j < A.K; j += nt) {
    const int id = L.id[j];
    float own = -1.0f;
    if (id >= 0 && id >= c0 && id < c1) {
      const int u = id - c0;
      if (atomicOr(&bits[u >> 5], 1u << (u & 31)) & (1u << (u & 31))) L.twice = 1;
      L.own_s[j] = RowElem<T>::get(row + id);
      own = L.p[j];
    }
    L.own_p[j] = own;
  }
}

// Where an id is listed twice its first entry takes the whole probability,
// in list order.  Called between two barriers.
__device__ __forceinline__ void join_doubles(const DistillArgs &A, ListShared &L, int nt) {
  if (!L.twice) return;
  for (int j = threadIdx.x; j < A.K; j += nt) {
    const int id = L.id[j];
    if (id < 0 || L.own_p[j] == -1.0f) continue;  // outside this CTA's columns
    float sum = 0.0f;
    bool first = true;
    for (int i = 0; i < A.K; i++)
      if (L.id[i] == id) {
        if (i < j) first = false;
        sum = __fadd_rn(sum, L.p[i]);
      }
    L.own_p[j] = first ? sum : -1.0f;
  }
}

template <typename T>
__device__ __forceinline__ void zero_span(T *row, const Span<T> &sp, int V, bool aligned, int nt) {
  constexpr int N = RowElem<T>::N;
  float x[N];
#pragma unroll
  for (int j = 0; j < N; j++) x[j] = 0.0f;
  for (int k = sp.k0 + threadIdx.x; k < sp.k1; k += nt)
    store_row_vec<N>(row, V, sp.c0 + (k - sp.k0) * N, x, aligned);
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

template <typename T>
__device__ __forceinline__ void grad_vec(const uint4 &raw, float m, float c, float f, float *x) {
  constexpr int N = RowElem<T>::N;
  RowElem<T>::unpack(raw, x);
#pragma unroll
  for (int j = 0; j < N; j++) x[j] = __fmul_rn(exp2_approx(__fmul_rn(__fsub_rn(x[j], m), c)), f);
}

// What the passes multiply e by.
struct GradFactors {
  float q_of_e;  // listed ids, e relative to M: P / S
  float f;       // the others, e relative to M_off: w T (P / S 2^((M_off - M) c) - rho / S_off)
};
__device__ __forceinline__ GradFactors grad_factors(const ListShared &L, const RowSums &R, float c, float by) {
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

// The listed ids get their own gradient, over what the pass along the row
// wrote there (a barrier before).
template <typename T>
__device__ __forceinline__ void grad_list(const DistillArgs &A, const ListShared &L, T *grad, float M, float by,
                                          float q_of_e, int nt) {
  for (int j = threadIdx.x; j < A.K; j += nt) {
    const float p = L.own_p[j];
    if (p == -1.0f) continue;
    const float e = exp2_approx(__fmul_rn(__fsub_rn(L.own_s[j], M), A.c));
    RowElem<T>::put(grad + L.id[j], q_of_e == 0.0f ? 0.0f : __fmul_rn(by, __fsub_rn(__fmul_rn(e, q_of_e), p)));
  }
}

template <typename T, bool GRAD>
__global__ void __launch_bounds__(kDistillThreads, 2) distill_kernel(const DistillArgs A) {
  constexpr int N = RowElem<T>::N;
  constexpr int NT = kDistillThreads;
  constexpr int NW = NT / 32;
  __shared__ ListShared L;
  __shared__ __align__(16) RowPart s_part[kMaxCluster];
  __shared__ MaxSum s_warp[NW][2];
  extern __shared__ uint32_t s_bits[];
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
  const float by = __fmul_rn(w, A.T);

  if (w == 0.0f) {  // the whole cluster leaves: the row is not read
    if (GRAD) zero_span(g_row, sp, A.V, aligned, NT);
    if (part == 0 && tid == 0) {
      A.loss[row] = 0.0f;
      if (A.stats) A.stats[row] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    }
    return;
  }
  // The span's batches of kRes vectors per thread, the first one last: it
  // stays in registers for the gradient.
  const int batches = max(1, (sp.k1 - sp.k0 + kRes * NT - 1) / (kRes * NT));
  uint4 raw[kRes];
  auto load = [&](int b) {
#pragma unroll
    for (int i = 0; i < kRes; i++) {
      const int k = sp.k0 + (b * kRes + i) * NT + tid;
      raw[i] = k < sp.k1 ? load_row_vec(x_row, shift, A.V, k)
                         : make_uint4(RowElem<T>::kNegInf2, RowElem<T>::kNegInf2, RowElem<T>::kNegInf2,
                                      RowElem<T>::kNegInf2);
    }
  };
  load(batches - 1);
  for (int i = tid; i < (A.span * N + 31) / 32; i += NT) s_bits[i] = 0u;
  read_list(A, static_cast<int>(row), L);
  __syncthreads();
  if (!L.valid) {
    if (GRAD) zero_span(g_row, sp, A.V, aligned, NT);
    if (part == 0 && tid == 0) {
      A.loss[row] = 0.0f;
      if (A.stats) A.stats[row] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    }
    return;
  }
  cluster_arrive();
  mark_list(A, L, s_bits, x_row, sp.c0, sp.c1, NT);
  __syncthreads();
  join_doubles(A, L, NT);

  // running maximum and sum of this thread's columns
  MaxSum a{-INFINITY, 0.0f};
  for (int b = batches - 1; b >= 0; b--) {
    if (b < batches - 1) load(b);
    float x[N];
    if (A.rest) {  // listed ids leave the sum
#pragma unroll
      for (int i = 0; i < kRes; i++) {
        const int u = ((b * kRes + i) * NT + tid) * N;
        const uint32_t on = u < A.span * N ? (s_bits[u >> 5] >> (u & 31)) & ((1u << N) - 1u) : 0u;
        if (on != 0u) {
          RowElem<T>::unpack(raw[i], x);
#pragma unroll
          for (int j = 0; j < N; j++)
            if ((on >> j) & 1u) x[j] = -INFINITY;
          raw[i] = RowElem<T>::pack(x);
        }
      }
    }
    float top = a.m;
#pragma unroll
    for (int i = 0; i < kRes; i++) {
      RowElem<T>::unpack(raw[i], x);
#pragma unroll
      for (int j = 0; j < N; j++) top = fmaxf(top, x[j]);
    }
    const float base = top > -INFINITY ? top : 0.0f;
    float s = __fmul_rn(a.s, exp2_approx(__fmul_rn(__fsub_rn(a.m, base), A.c)));
#pragma unroll
    for (int i = 0; i < kRes; i++) {
      RowElem<T>::unpack(raw[i], x);
#pragma unroll
      for (int j = 0; j < N; j++) s = __fadd_rn(s, exp2_approx(__fmul_rn(__fsub_rn(x[j], base), A.c)));
    }
    a = MaxSum{top, s};
  }
  // and of its listed ids
  MaxSum listed{-INFINITY, 0.0f};
  if (A.rest) {
    for (int j = tid; j < A.K; j += NT) {
      if (L.own_p[j] == -1.0f) continue;
      const float sv = L.own_s[j];
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
  cluster_wait();  // every CTA of the row runs: its shared memory may be written
  if (warp == 0) {
    RowPart r{s_warp[0][0], s_warp[0][1], 0.0, 0.0, 0.0, 0.0};
    for (int i = 1; i < NW; i++) {
      r.row = join(r.row, s_warp[i][0], A.c);
      r.list = join(r.list, s_warp[i][1], A.c);
    }
    const double ref = r.ref();
    for (int j = lane; j < A.K; j += 32) {
      const float p = L.own_p[j];
      if (p == -1.0f || p == 0.0f) continue;
      r.p += p;
      r.plogp += static_cast<double>(p) * logf(p);
      r.ps += static_cast<double>(p) * (L.own_s[j] - ref);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      r.p += __shfl_xor_sync(0xFFFFFFFFu, r.p, o);
      r.plogp += __shfl_xor_sync(0xFFFFFFFFu, r.plogp, o);
      r.ps += __shfl_xor_sync(0xFFFFFFFFu, r.ps, o);
    }
    if (lane < A.parts) put_remote(&s_part[part], r, lane);
  }
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
    double l = L.sum_p * log_s;
    for (int i = 0; i < A.parts; i++) {
      const RowPart &r = s_part[i];
      l += r.plogp - (r.ps + r.p * (static_cast<double>(r.ref()) - R.M)) / T_;
    }
    if (L.rho != 0.0f)
      l += L.rho * (log(static_cast<double>(L.rho)) - log(static_cast<double>(R.S_off)) + log_s -
                    (static_cast<double>(R.M_off) - R.M) / T_);
    if (R.S == 0.0f) l = INFINITY;  // every logit is -inf: the student has no distribution
    A.loss[row] = static_cast<float>(static_cast<double>(w) * T_ * T_ * l);
    if (A.stats) A.stats[row] = make_float4(R.M, R.S, R.M_off, R.S_off);
  }
  if constexpr (GRAD) {
    const GradFactors g = grad_factors(L, R, A.c, by);
    for (int b = 0; b < batches; b++) {
      if (b > 0) load(b);
#pragma unroll
      for (int i = 0; i < kRes; i++) {
        const int k = sp.k0 + (b * kRes + i) * NT + tid;
        if (k < sp.k1) {
          float x[N];
          grad_vec<T>(raw[i], R.M_off, A.c, g.f, x);
          store_row_vec<N>(g_row, A.V, sp.c0 + (k - sp.k0) * N, x, aligned);
        }
      }
    }
    __syncthreads();
    grad_list(A, L, g_row, R.M, by, g.q_of_e, NT);
  }
}

// The gradient from saved statistics: no sums are left to take, so a row's
// tiles (256 threads x 8 vectors) are independent CTAs.
template <typename T>
__global__ void __launch_bounds__(kBackThreads) distill_backward_kernel(const DistillArgs A) {
  constexpr int N = RowElem<T>::N;
  constexpr int NT = kBackThreads;
  __shared__ ListShared L;
  __shared__ uint32_t s_bits[kRes * NT * N / 32];
  const int part = static_cast<int>(blockIdx.x) % A.parts;
  const int64_t row = blockIdx.x / A.parts;
  const int tid = threadIdx.x;
  const T *x_row = static_cast<const T *>(A.logits) + row * A.ld;
  const int shift = row_shift(x_row);
  const Span<T> sp(part, A.span, A.V, shift);
  T *g_row = static_cast<T *>(A.grad) + row * A.ld_grad;
  const bool aligned = ((reinterpret_cast<uintptr_t>(g_row) - static_cast<uintptr_t>(shift) * sizeof(T)) & 15u) == 0;
  const float w = A.weight ? A.weight[row] : 1.0f;
  if (w == 0.0f) {
    zero_span(g_row, sp, A.V, aligned, NT);
    return;
  }
  uint4 raw[kRes];
#pragma unroll
  for (int i = 0; i < kRes; i++) {
    const int k = sp.k0 + i * NT + tid;
    raw[i] = k < sp.k1 ? load_row_vec(x_row, shift, A.V, k) : make_uint4(0u, 0u, 0u, 0u);
  }
  const float4 st = A.stats[row];
  const float by = __fmul_rn(__fmul_rn(w, A.T), A.grad_loss ? A.grad_loss[row] : 1.0f);
  for (int i = tid; i < kRes * NT * N / 32; i += NT) s_bits[i] = 0u;
  read_list(A, static_cast<int>(row), L);
  __syncthreads();
  if (!L.valid) {
    zero_span(g_row, sp, A.V, aligned, NT);
    return;
  }
  mark_list(A, L, s_bits, x_row, sp.c0, sp.c1, NT);
  __syncthreads();
  join_doubles(A, L, NT);
  const RowSums R{st.x, st.y, st.z, st.w};
  const GradFactors g = grad_factors(L, R, A.c, by);
#pragma unroll
  for (int i = 0; i < kRes; i++) {
    const int k = sp.k0 + i * NT + tid;
    if (k < sp.k1) {
      float x[N];
      grad_vec<T>(raw[i], R.M_off, A.c, g.f, x);
      store_row_vec<N>(g_row, A.V, sp.c0 + (k - sp.k0) * N, x, aligned);
    }
  }
  __syncthreads();
  grad_list(A, L, g_row, R.M, by, g.q_of_e, NT);
}

// CTAs per row: 64 KB of a row each; more, up to 8, while the rows would
// leave SMs without a CTA.
template <typename T, bool GRAD>
cudaError_t launch_distill(DistillArgs &A, cudaStream_t st) {
  constexpr int N = RowElem<T>::N;
  const int vecs = (A.V + 2 * N - 2) / N;  // of a row with the largest shift
  int parts = (vecs + kRes * kDistillThreads - 1) / (kRes * kDistillThreads);
  while (parts < kMaxCluster && static_cast<int64_t>(A.N) * parts < 2 * current_sms() &&
         vecs > parts * kDistillThreads)
    parts++;
  parts = parts < kMaxCluster ? parts : kMaxCluster;
  A.parts = parts;
  A.span = (vecs + parts - 1) / parts;
  const int64_t ctas = static_cast<int64_t>(A.N) * parts;
  if (ctas > 0x7FFFFFFF) return cudaErrorInvalidConfiguration;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(static_cast<unsigned>(ctas));
  cfg.blockDim = dim3(kDistillThreads);
  cfg.dynamicSmemBytes = sizeof(uint32_t) * ((static_cast<size_t>(A.span) * N + 31) / 32);
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

template <typename T>
cudaError_t launch_backward(DistillArgs &A, cudaStream_t st) {
  constexpr int N = RowElem<T>::N;
  const int vecs = (A.V + 2 * N - 2) / N;
  A.span = kRes * kBackThreads;
  A.parts = (vecs + A.span - 1) / A.span;
  const int64_t ctas = static_cast<int64_t>(A.N) * A.parts;
  if (ctas > 0x7FFFFFFF) return cudaErrorInvalidConfiguration;
  distill_backward_kernel<T><<<static_cast<unsigned>(ctas), kBackThreads, 0, st>>>(A);
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
