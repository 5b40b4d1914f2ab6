// pz_rules.cu — pz_process_logits: penalties, biases and grammar masks on
// rows of logits.
//
// Per row and column v, with x the widened logit:
//   penalty   v occurs c > 0 times in the row's history:
//               if (rep != 1) x = x > 0 ? x / rep : x * rep;
//               x = x - (c * freq + pres)
//             the sampler's own steps (penalize, pz_device.cuh), each rounded
//             to fp32, so an fp32 row comes out bit for bit as the sampler
//             sees it after its penalties
//   bias      v is listed in the row's bias list: x = x + b, b being the last
//             entry of that id (a list with an id twice is read as a JSON
//             object with a key twice is)
//   mask      v's bit is 0: x = -inf, whatever x was (NaN and inf included)
//
// Bound: HBM.  Out of place every logit is read and written once (1024 rows of
// 128256 f32: 165 us without rules, 6.4 TB/s of a copy's 6.5; 167 with masks;
// 199, 5.3 TB/s, with 1024 history ids a row, each of which is another 32-byte
// sector to fetch and to write; bf16 into f32 153 with masks and 166 with
// lists too).  In place only the vectors that something changes are touched:
// 4096 rows of 151936 bf16 under masks, half of them random, 343 us; a sector
// that a mask takes part of is read and written whole, 1.65 GB there.  Under
// masks and lists together it is no gain: the 1024 f32 rows 241 us (74 with
// the lists alone, 137 with the masks).  Rows of out that lie at another offset
// from a 16-byte boundary than the logits' are stored an element at a time
// (1024 rows of 128255, odd addresses into rows 128256 apart: f32 184 us
// against 172, bf16 352 against 90).
//
// A CTA takes a part of a row.  Four warps pass along its columns and know
// the mask alone.  Two more work out the listed ids meanwhile: those that lie
// in the CTA's columns go into a hash table in shared memory, which counts how
// often each occurs in the history and remembers its last bias entry (integer
// atomics: the same sums in any order); their new values, computed from the
// input, are stored over what the pass wrote once it is through.  In place
// the pass changes no allowed id, so both ways a value is read before
// anything lies over it.  A part with more distinct ids than the table takes
// is done in classes of the ids' hash, each as small as it needs: histories
// may have any length.
#include "pz_device.cuh"
#include "pz_rowvec.cuh"
#include "pz_status.cuh"

namespace pz {
namespace {

constexpr int kRulesThreads = 128;

struct RulesArgs {
  const void *in;
  void *out;
  int64_t ld_in, ld_out;
  int V;
  int parts;  // CTAs per row; one more counts the mask when n_allowed is given
  int span;   // vectors per CTA
  const pz_sampler_config *cfg;
  const int32_t *hist, *hist_off;
  const int32_t *bias_ids;
  const float *bias_vals;
  const int32_t *bias_off;
  const uint32_t *mask;
  int64_t mask_ld;
  int32_t mask_rows;
  const int32_t *mask_index;
  int32_t *n_allowed;
};

// The row's mask words, or null where the row has none.
__device__ __forceinline__ const uint32_t *mask_row(const RulesArgs &A, int row) {
  if (A.mask == nullptr) return nullptr;
  const int at = A.mask_index ? A.mask_index[row] : row;
  if (at < 0 || at >= A.mask_rows) return nullptr;
  return A.mask + static_cast<int64_t>(at) * A.mask_ld;
}

// Allowed ids of a row: the set bits of its mask among the columns [0, V).
__device__ void count_allowed(const RulesArgs &A, int row) {
  __shared__ int s_sum;
  const uint32_t *m = mask_row(A, row);
  if (m == nullptr) {
    if (threadIdx.x == 0) A.n_allowed[row] = A.V;
    return;
  }
  if (threadIdx.x == 0) s_sum = 0;
  __syncthreads();
  int n = 0;
  const int words = (A.V + 31) / 32;
  for (int i = threadIdx.x; i < words; i += blockDim.x) {
    uint32_t w = m[i];
    if (i == words - 1 && (A.V & 31) != 0) w &= (1u << (A.V & 31)) - 1u;
    n += __popc(w);
  }
  n = __reduce_add_sync(0xFFFFFFFFu, n);
  if ((threadIdx.x & 31) == 0) atomicAdd(&s_sum, n);
  __syncthreads();
  if (threadIdx.x == 0) A.n_allowed[row] = s_sum;
}

constexpr int kSlots = 1024;     // of the hash table
constexpr int kProbes = 32;      // a longer run of taken slots counts as a full table
constexpr int kRulesBatch = 4;   // vectors that a thread has in flight
constexpr int kRulesStep = kRulesBatch * kRulesThreads;

// Threads that work on the lists beside the pass's, and the CTAs per SM that
// go with them.  More of them shorten a CTA's life where the whole batch is
// one wave of CTAs (64 rows of 151936 bf16, 1024 ids each: 17.6 us with 64,
// 12.7 with 128), fewer leave room for more passes where it is many (1024
// rows of 128256 f32: 202 and 216 us).
constexpr int kManyLists = 128, kFewLists = 64;
constexpr int rules_ctas(int lt) { return lt == 0 ? 7 : lt == kManyLists ? 4 : 5; }
constexpr int kQueue = 256;       // of each of their warps

template <int LT>
struct Table {
  int32_t key[kSlots];    // id or -1
  int32_t count[kSlots];  // occurrences in the history
  int32_t last[kSlots];   // last bias entry + 1
  uint16_t slot[kSlots];  // the taken slots, in the order they were taken
  float value[kSlots];    // by that order: the new value
  int2 queue[LT / 32][kQueue];  // ids on their way in, with their places in the lists
  int taken;
  int full;
};

// The lists of a row in the columns [c0, c1).
template <typename Ti, typename To, int LT>
struct Lists {
  const int32_t *hist, *bias_ids;  // of this row
  const float *bias_vals;
  int n_hist, n_bias;
  int c0, c1;
  RowPlan P;
  uint32_t cls = 0;  // the class of ids that is being worked on: those whose hash ends in these bits
  int bits = 0;

  __device__ __forceinline__ Lists(const RulesArgs &A, int row, int c0_, int c1_)
      : hist(nullptr), bias_ids(nullptr), bias_vals(nullptr), n_hist(0), n_bias(0), c0(c0_), c1(c1_), P{} {
    if (A.hist != nullptr) {
      const int from = A.hist_off[row], to = A.hist_off[row + 1];
      P = plan_row(A.cfg[row], A.V);
      hist = A.hist + from;
      n_hist = P.pen_on ? max(to - from, 0) : 0;
    }
    if (A.bias_ids != nullptr) {
      const int from = A.bias_off[row];
      bias_ids = A.bias_ids + from;
      bias_vals = A.bias_vals + from;
      n_bias = max(A.bias_off[row + 1] - from, 0);
    }
  }
  static __device__ __forceinline__ uint32_t hash(int id) {  // odd factor: one to one
    return static_cast<uint32_t>(id) * 0x9E3779B1u;
  }
  // The threads that work on the lists, and their barrier.
  static __device__ __forceinline__ int self() { return static_cast<int>(threadIdx.x) - kRulesThreads; }
  static __device__ __forceinline__ void sync() { asm volatile("bar.sync 1, %0;" ::"r"(LT) : "memory"); }
  // The first n ids of the warp's queue into the table.
  __device__ __forceinline__ void insert(Table<LT> &S, const int2 *queue, int n) const {
    __syncwarp();
    for (int i = threadIdx.x & 31; i < n; i += 32) {
      const int2 e = queue[i];
      uint32_t at = hash(e.x) >> 22;
      static_assert(kSlots == 1 << 10, "the slot is the hash's top 10 bits");
      int tries = 0;
      for (; tries < kProbes; tries++, at = (at + 1) % kSlots) {
        const int was = atomicCAS(&S.key[at], -1, e.x);
        if (was == -1) S.slot[atomicAdd(&S.taken, 1)] = static_cast<uint16_t>(at);
        if (was == -1 || was == e.x) break;
      }
      if (tries == kProbes)
        S.full = 1;
      else if (e.y >= 0)
        atomicMax(&S.last[at], e.y + 1);
      else
        atomicAdd(&S.count[at], 1);
    }
    __syncwarp();
  }
  // The lists' ids of the class into the table: the history's, then the
  // biases', as one list, the next round's ids on their way while one round's
  // are looked at.  Few lie in the CTA's columns: a warp lines its own up
  // first, and the table's atomics run with full warps (64 rows with 2048 ids
  // each, 64 threads: 16.1 us put in as they came, 13.0 lined up).
  __device__ __forceinline__ void fill(Table<LT> &S) const {
    constexpr int G = 4;  // ids of a round
    const uint32_t low = bits >= 32 ? 0xFFFFFFFFu : (1u << bits) - 1u;
    const int64_t n = static_cast<int64_t>(n_hist) + n_bias;
    int2 *queue = S.queue[self() >> 5];
    auto load = [&](int64_t j0, int *id) {
#pragma unroll
      for (int g = 0; g < G; g++) {
        const int64_t j = j0 + g * LT + self();
        id[g] = j < n_hist ? hist[j] : j < n ? bias_ids[j - n_hist] : -1;
      }
    };
    int now[G], next[G];
    int waiting = 0;
    load(0, now);
    for (int64_t j0 = 0; j0 < n; j0 += G * LT) {
      load(j0 + G * LT, next);
#pragma unroll
      for (int g = 0; g < G; g++) {
        const int t = now[g];
        now[g] = next[g];
        const bool here = t >= c0 && t < c1 && (hash(t) & low) == cls;  // (c0 >= 0)
        const uint32_t all = __ballot_sync(0xFFFFFFFFu, here);
        if (here) {
          const int64_t j = j0 + g * LT + self();
          queue[waiting + __popc(all & lanemask_lt())] = make_int2(t, j < n_hist ? -1 : static_cast<int>(j - n_hist));
        }
        waiting += __popc(all);
      }
      if (waiting > kQueue - G * 32) {
        insert(S, queue, waiting);
        waiting = 0;
      }
    }
    insert(S, queue, waiting);
  }
  // The next class that fits the table, from the present one on.
  __device__ __forceinline__ void build(Table<LT> &S) {
    for (;;) {
      for (int i = self(); i < kSlots / 4; i += LT) {
        reinterpret_cast<int4 *>(S.key)[i] = make_int4(-1, -1, -1, -1);
        reinterpret_cast<int4 *>(S.count)[i] = make_int4(0, 0, 0, 0);
        reinterpret_cast<int4 *>(S.last)[i] = make_int4(0, 0, 0, 0);
      }
      if (self() == 0) S.taken = S.full = 0;
      sync();
      fill(S);
      sync();
      if (!S.full) return;
      bits++;  // half of the class (32 bits leave one id)
      sync();
    }
  }
  // To the next class; false when there is none.
  __device__ __forceinline__ bool advance() {
    while (bits > 0 && ((cls >> (bits - 1)) & 1u)) {
      bits--;
      cls &= (1u << bits) - 1u;
    }
    if (bits == 0) return false;
    cls |= 1u << (bits - 1);
    return true;
  }
  // The new values of the taken slots (a slot whose id the mask takes: none).
  __device__ __forceinline__ void gather(Table<LT> &S, const Ti *in, const uint32_t *m) const {
    constexpr int G = 4;  // loads in flight
    const int n = S.taken;
    for (int i0 = self(); i0 < n; i0 += G * LT) {
      float x[G];
      bool on[G];
#pragma unroll
      for (int g = 0; g < G; g++) {
        on[g] = false;
        if (i0 + g * LT < n) {
          const int t = S.key[S.slot[i0 + g * LT]];
          x[g] = RowElem<Ti>::get(in + t);
          on[g] = m == nullptr || ((m[t >> 5] >> (t & 31)) & 1u);
        }
      }
#pragma unroll
      for (int g = 0; g < G; g++) {
        if (i0 + g * LT >= n) continue;
        const int at = S.slot[i0 + g * LT];
        float y = x[g];
        if (S.count[at] > 0) y = penalize(y, S.count[at], P);
        if (S.last[at] > 0) y = __fadd_rn(y, bias_vals[S.last[at] - 1]);
        S.value[i0 + g * LT] = y;
        if (!on[g]) S.key[at] = -1;
      }
    }
  }
  __device__ __forceinline__ void scatter(const Table<LT> &S, To *out) const {
    for (int i = self(); i < S.taken; i += LT) {
      const int t = S.key[S.slot[i]];
      if (t >= 0) RowElem<To>::put(out + t, S.value[i]);
    }
  }
};

// The pass along the columns of the vectors [k0, k1): the mask alone.  A
// thread's vectors are kRulesThreads apart, a multiple of 32 columns, so
// their bits lie at one offset of words a fixed step apart.
template <typename Ti, typename To, bool INPLACE, bool KEEP>
struct MaskPass {
  static constexpr int N = RowElem<Ti>::N;
  static constexpr uint32_t ALL = (1u << N) - 1u;
  static constexpr int WORDS = kRulesThreads * N / 32;  // between a thread's vectors
  static_assert(kRulesThreads * N % 32 == 0, "a thread's vectors share their bit offset");
  const Ti *in;
  To *out;
  const uint32_t *m;
  int V, shift, words, k1;
  WholeVecs whole;
  bool aligned;

  __device__ __forceinline__ bool whole_batch(int kb) const {  // the block's batch from vector kb on
    return kb >= whole.first && kb + kRulesStep <= min(k1, whole.last);
  }
  // The mask bits of the columns [c, c + N).  c may lie up to a vector before
  // column 0; bits outside the words are 0.
  __device__ __forceinline__ uint32_t bits_at(int c) const {
    const int at = c >> 5, off = c & 31;
    uint32_t w = at >= 0 ? __ldg(m + at) >> off : 0u;
    if (off > 32 - N && at + 1 < words) w |= __ldg(m + at + 1) << (32 - off);
    return w & ALL;
  }
  // A batch's mask bits (past its end: all, which changes nothing in place).
  __device__ __forceinline__ void bits(int kb, uint32_t *allow) const {
    const int k = kb + static_cast<int>(threadIdx.x);
    const int c = k * N - shift;
    if (m == nullptr) return;
    if (shift == 0 && whole_batch(kb)) {  // one word holds a vector's bits
      const int off = c & 31;
      const uint32_t *p = m + (c >> 5);
#pragma unroll
      for (int i = 0; i < kRulesBatch; i++) allow[i] = (__ldg(p + i * WORDS) >> off) & ALL;
    } else {
#pragma unroll
      for (int i = 0; i < kRulesBatch; i++)
        allow[i] = k + i * kRulesThreads < k1 ? bits_at(c + i * kRulesThreads * N) : ALL;
    }
  }
  // A batch's vectors; in place only those that keep some of their values.
  __device__ __forceinline__ void data(int kb, const uint32_t *allow, uint4 *raw) const {
    const int k = kb + static_cast<int>(threadIdx.x);
    if (whole_batch(kb)) {
      const Ti *p = in + (k * N - shift);
#pragma unroll
      for (int i = 0; i < kRulesBatch; i++)
        if (!INPLACE || (allow[i] != ALL && allow[i] != 0u)) raw[i] = load16(p + i * kRulesThreads * N);
    } else {
#pragma unroll
      for (int i = 0; i < kRulesBatch; i++)
        if (k + i * kRulesThreads < k1 && (!INPLACE || (allow[i] != ALL && allow[i] != 0u)))
          raw[i] = vec(k + i * kRulesThreads);
    }
  }
  __device__ __forceinline__ uint4 vec(int k) const {
    return k >= whole.first && k < whole.last ? load16(in + (k * N - shift)) : load_edge(in, V, k * N - shift);
  }
  __device__ __forceinline__ void store(int kb, uint4 *raw, const uint32_t *allow) const {
    const int k = kb + static_cast<int>(threadIdx.x);
    if (m != nullptr) {
#pragma unroll
      for (int i = 0; i < kRulesBatch; i++) raw[i] = RowElem<Ti>::keep(raw[i], allow[i]);
    }
    if (whole_batch(kb) && aligned) {
      To *p = out + (k * N - shift);
#pragma unroll
      for (int i = 0; i < kRulesBatch; i++)
        if (!INPLACE || allow[i] != ALL) put(p + i * kRulesThreads * N, raw[i]);
    } else {
#pragma unroll
      for (int i = 0; i < kRulesBatch; i++) {
        const int v = k + i * kRulesThreads;
        if (v >= k1 || (INPLACE && allow[i] == ALL)) continue;
        if (aligned && v >= whole.first && v < whole.last)
          put(out + (v * N - shift), raw[i]);
        else
          put_edge(v * N - shift, raw[i]);
      }
    }
  }
  // KEEP: listed ids are stored over some of it.
  static __device__ __forceinline__ void put16(To *p, const uint4 &v) { KEEP ? store16_keep(p, v) : store16(p, v); }
  static __device__ __forceinline__ void put(To *p, const uint4 &v) {
    if constexpr (sizeof(Ti) == sizeof(To)) {
      put16(p, v);
    } else {
      float x[N];
      RowElem<Ti>::unpack(v, x);
#pragma unroll
      for (int j = 0; j < N; j += RowElem<To>::N) put16(p + j, RowElem<To>::pack(x + j));
    }
  }
  __device__ __forceinline__ void put_edge(int c, const uint4 &v) const {
    if constexpr (sizeof(Ti) == sizeof(To)) {
      store_edge(out, V, c, v);
    } else {
      float x[N];
      RowElem<Ti>::unpack(v, x);
#pragma unroll
      for (int j = 0; j < N; j += RowElem<To>::N) store_edge(out, V, c + j, RowElem<To>::pack(x + j));
    }
  }
  // The next batch's vectors are in flight while one is worked on; in place,
  // where they hang on the mask, the bits of the one after.
  __device__ __forceinline__ void run(int k0) const {
    if (INPLACE && m == nullptr) return;
    uint4 a[kRulesBatch], b[kRulesBatch];
    uint32_t aa[kRulesBatch], ab[kRulesBatch], ac[kRulesBatch];
    bits(k0, aa);
    if (INPLACE && k0 + kRulesStep < k1) bits(k0 + kRulesStep, ab);
    data(k0, aa, a);
    for (int kb = k0; kb < k1; kb += kRulesStep) {
      if (INPLACE) {
        if (kb + 2 * kRulesStep < k1) bits(kb + 2 * kRulesStep, ac);
      } else if (kb + kRulesStep < k1) {
        bits(kb + kRulesStep, ab);
      }
      if (kb + kRulesStep < k1) data(kb + kRulesStep, ab, b);
      store(kb, a, aa);
#pragma unroll
      for (int i = 0; i < kRulesBatch; i++) {
        a[i] = b[i];
        aa[i] = ab[i];
        if (INPLACE) ab[i] = ac[i];
      }
    }
  }
};

// kRulesThreads threads for the pass and LT for the lists (0: there are none).
template <typename Ti, typename To, bool INPLACE, int LT>
__global__ void __launch_bounds__(kRulesThreads + LT, rules_ctas(LT))
    rules_kernel(const RulesArgs A) {
  constexpr int N = RowElem<Ti>::N;
  const int per_row = A.parts + (A.n_allowed != nullptr ? 1 : 0);
  const int row = blockIdx.x / per_row;
  const int part = blockIdx.x - row * per_row;
  if (part == A.parts) {
    count_allowed(A, row);
    return;
  }
  const Ti *in = static_cast<const Ti *>(A.in) + static_cast<int64_t>(row) * A.ld_in;
  To *out = static_cast<To *>(A.out) + static_cast<int64_t>(row) * A.ld_out;
  const int shift = row_shift(in);
  const int all = (A.V + shift + N - 1) / N;
  const int k0 = min(part * A.span, all), k1 = min(k0 + A.span, all);
  if (k0 >= k1) return;
  const uint32_t *m = mask_row(A, row);
  if constexpr (LT > 0) {
    if (threadIdx.x >= kRulesThreads) {
      __shared__ __align__(16) Table<LT> S;
      Lists<Ti, To, LT> L(A, row, max(k0 * N - shift, 0), min(k1 * N - shift, A.V));
      L.build(S);
      L.gather(S, in, m);
      __syncthreads();  // the pass is through
      L.scatter(S, out);
      while (L.advance()) {
        L.sync();
        L.build(S);
        L.gather(S, in, m);
        L.scatter(S, out);
      }
      return;
    }
  }
  const MaskPass<Ti, To, INPLACE, (LT > 0)> pass{
      in, out, m, A.V, shift, (A.V + 31) / 32, k1, whole_vecs<Ti>(shift, A.V),
      ((reinterpret_cast<uintptr_t>(out) - static_cast<uintptr_t>(shift) * sizeof(To)) & 15u) == 0};
  pass.run(k0);
  if (LT > 0) __syncthreads();
}

// Parts of a row: 64 KB (1024 rows of 128256 f32 with history, biases and
// masks: 228 us at 32 KB, 202 at 64 KB, 205 at 128 KB; a row per CTA, a
// thousand streams apart from one another, 264), smaller ones, of at least
// one vector per thread, while they would not fill the GPU's CTA slots.
constexpr int kPartVecs = 4096;
template <typename Ti, typename To, bool INPLACE>
cudaError_t launch_rules(RulesArgs &A, int B, cudaStream_t st) {
  constexpr int N = RowElem<Ti>::N;
  const bool lists = A.hist != nullptr || A.bias_ids != nullptr;
  const int vecs = (A.V + 2 * N - 2) / N;  // of a row with the largest shift
  int parts = (vecs + kPartVecs - 1) / kPartVecs;
  const int most = (vecs + kRulesThreads - 1) / kRulesThreads;
  const int wave = current_sms() * rules_ctas(lists ? kManyLists : 0) / B - (A.n_allowed != nullptr ? 1 : 0);
  const bool one_wave = parts <= wave;
  if (parts < wave) parts = wave < most ? wave : most;
  A.parts = parts;
  A.span = (vecs + parts - 1) / parts;
  const int64_t ctas = static_cast<int64_t>(B) * (parts + (A.n_allowed != nullptr ? 1 : 0));
  if (ctas > 0x7FFFFFFF) return cudaErrorInvalidConfiguration;
  const unsigned grid = static_cast<unsigned>(ctas);
  if (!lists)
    rules_kernel<Ti, To, INPLACE, 0><<<grid, kRulesThreads, 0, st>>>(A);
  else if (one_wave)
    rules_kernel<Ti, To, INPLACE, kManyLists><<<grid, kRulesThreads + kManyLists, 0, st>>>(A);
  else
    rules_kernel<Ti, To, INPLACE, kFewLists><<<grid, kRulesThreads + kFewLists, 0, st>>>(A);
  return cudaGetLastError();
}

}  // namespace
}  // namespace pz

extern "C" pz_status pz_process_logits(const void *logits, pz_dtype dtype, int B, int V, int64_t ld,
                                       const pz_logits_rules *rules, void *out, pz_dtype out_dtype,
                                       int64_t ld_out, int32_t *n_allowed, void *stream) {
  using pz::report;
  if (!logits || !rules || !out || B < 0 || V <= 0 || ld < V || ld_out < V)
    return report(PZ_ERR_INVALID_ARGS, "pz_process_logits: null pointer or bad size");
  if ((dtype != PZ_DTYPE_F32 && dtype != PZ_DTYPE_BF16) ||
      (out_dtype != dtype && out_dtype != PZ_DTYPE_F32))
    return report(PZ_ERR_INVALID_ARGS, "pz_process_logits: out_dtype is dtype or f32");
  if (V > (1 << 30)) return report(PZ_ERR_UNSUPPORTED, "pz_process_logits: more than 2^30 columns");
  const pz_logits_rules &R = *rules;
  if ((R.hist == nullptr) != (R.hist_off == nullptr) || (R.hist && !R.cfg))
    return report(PZ_ERR_INVALID_ARGS, "pz_process_logits: hist comes with hist_off and cfg");
  if ((R.bias_ids == nullptr) != (R.bias_off == nullptr) || (R.bias_ids == nullptr) != (R.bias_vals == nullptr))
    return report(PZ_ERR_INVALID_ARGS, "pz_process_logits: bias_ids, bias_vals and bias_off come together");
  if (R.mask == nullptr ? (R.mask_index != nullptr)
                        : (R.mask_rows < (R.mask_index ? 1 : B) || R.mask_ld < (static_cast<int64_t>(V) + 31) / 32))
    return report(PZ_ERR_INVALID_ARGS, "pz_process_logits: mask rows hold ceil(V/32) words, one row per logits row or per index");
  const size_t es = pz::elem_bytes(dtype), eo = pz::elem_bytes(out_dtype);
  const void *words[] = {R.cfg, R.hist, R.hist_off, R.bias_ids, R.bias_vals, R.bias_off, R.mask, R.mask_index, n_allowed};
  bool crooked = pz::misaligned(logits, es) || pz::misaligned(out, eo);
  for (const void *p : words) crooked |= pz::misaligned(p, 4);
  if (crooked)
    return report(PZ_ERR_INVALID_ARGS, "pz_process_logits: pointer not aligned to its elements");
  if (B == 0) return PZ_OK;
  const bool inplace = out == logits;
  if (inplace ? (out_dtype != dtype || ld_out != ld)
              : pz::overlap(logits, pz::rows_bytes(B, V, ld, es), out, pz::rows_bytes(B, V, ld_out, eo)))
    return report(PZ_ERR_INVALID_ARGS, "pz_process_logits: out is logits itself (same type and ld) or apart from it");
  pz::RulesArgs A{};
  A.in = logits;
  A.out = out;
  A.ld_in = ld;
  A.ld_out = ld_out;
  A.V = V;
  A.cfg = R.cfg;
  A.hist = R.hist;
  A.hist_off = R.hist_off;
  A.bias_ids = R.bias_ids;
  A.bias_vals = R.bias_vals;
  A.bias_off = R.bias_off;
  A.mask = R.mask;
  A.mask_ld = R.mask_ld;
  A.mask_rows = R.mask_rows;
  A.mask_index = R.mask_index;
  A.n_allowed = n_allowed;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  cudaError_t e;
  if (dtype == PZ_DTYPE_F32)
    e = inplace ? pz::launch_rules<float, float, true>(A, B, st) : pz::launch_rules<float, float, false>(A, B, st);
  else if (out_dtype == PZ_DTYPE_F32)
    e = pz::launch_rules<pz::bf16_t, float, false>(A, B, st);
  else
    e = inplace ? pz::launch_rules<pz::bf16_t, pz::bf16_t, true>(A, B, st)
                : pz::launch_rules<pz::bf16_t, pz::bf16_t, false>(A, B, st);
  return e == cudaSuccess ? PZ_OK : pz::report_cuda(e);
}
