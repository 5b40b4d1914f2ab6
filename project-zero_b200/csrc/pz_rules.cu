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
// Bound: HBM.  Out of place every logit is read and written once; in place
// only the vectors that something changes are touched.
//
// One CTA takes a tile of a row's columns.  It first has its logits on their
// way to registers, then reads the whole of the row's history and bias list
// (a few KB, from L2 after the row's first tile) and keeps what falls into
// its columns: a count per column and the index of the last bias entry per
// column, in shared memory, with one bit per column that says whether either
// is there.  Counts per column need no bound on the history's length and no
// hashing, and integer atomics give the same sums in any order.  Every
// vector is then changed by the thread that read it and written once: no
// column has two writers, so the output may be the input.
#include "pz_device.cuh"
#include "pz_rowvec.cuh"
#include "pz_status.cuh"

namespace pz {
namespace {

constexpr int kRulesThreads = 256;

struct RulesArgs {
  const void *in;
  void *out;
  int64_t ld_in, ld_out;
  int V;
  int tiles;  // column tiles per row; one more CTA per row counts the mask when n_allowed is given
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
  __shared__ int s_part[kRulesThreads / 32];
  const uint32_t *m = mask_row(A, row);
  int n = 0;
  if (m != nullptr) {
    const int words = (A.V + 31) / 32;
    for (int i = threadIdx.x; i < words; i += kRulesThreads) {
      uint32_t w = m[i];
      if (i == words - 1 && (A.V & 31) != 0) w &= (1u << (A.V & 31)) - 1u;
      n += __popc(w);
    }
    n = __reduce_add_sync(0xFFFFFFFFu, n);
    if ((threadIdx.x & 31) == 0) s_part[threadIdx.x >> 5] = n;
    __syncthreads();
    n = 0;
    for (int w = 0; w < kRulesThreads / 32; w++) n += s_part[w];
  } else {
    n = A.V;
  }
  if (threadIdx.x == 0) A.n_allowed[row] = n;
}

// VPT vectors of 16 input bytes per thread.  The tile's columns are counted
// from c0, which lies up to one vector before column 0 in the first tile.
template <typename Ti, typename To, int VPT, bool INPLACE, bool LISTS>
__global__ void __launch_bounds__(kRulesThreads) rules_kernel(const RulesArgs A) {
  constexpr int N = RowElem<Ti>::N;
  constexpr int TILE = kRulesThreads * VPT * N;
  constexpr int WORDS = TILE / 32;
  __shared__ uint32_t s_allow[WORDS];
  __shared__ uint32_t s_touch[LISTS ? WORDS : 1];
  extern __shared__ __align__(16) int32_t s_dyn[];  // counts [TILE], last bias entries [TILE]
  const int per_row = A.tiles + (A.n_allowed != nullptr ? 1 : 0);
  const int row = blockIdx.x / per_row;
  const int tile = blockIdx.x - row * per_row;
  const int tid = threadIdx.x;
  if (tile == A.tiles) {
    count_allowed(A, row);
    return;
  }
  const Ti *in = static_cast<const Ti *>(A.in) + static_cast<int64_t>(row) * A.ld_in;
  To *out = static_cast<To *>(A.out) + static_cast<int64_t>(row) * A.ld_out;
  const int shift = row_shift(in);
  const int c0 = tile * TILE - shift;
  if (c0 >= A.V) return;
  const bool aligned = ((reinterpret_cast<uintptr_t>(out) - static_cast<uintptr_t>(shift) * sizeof(To)) & 15u) == 0;
  const int k0 = tile * (kRulesThreads * VPT) + tid;

  uint4 raw[VPT];
  if constexpr (!INPLACE) {
#pragma unroll
    for (int i = 0; i < VPT; i++) raw[i] = load_row_vec(in, shift, A.V, k0 + i * kRulesThreads);
  }

  // the tile's mask bits, moved so that bit j of word i is column c0 + 32 i + j
  const uint32_t *m = mask_row(A, row);
  const int words = (A.V + 31) / 32;
  for (int i = tid; i < WORDS; i += kRulesThreads) {
    uint32_t w = 0xFFFFFFFFu;
    if (m != nullptr) {
      const int c = c0 + 32 * i;
      const int at = c >> 5;  // rounds down for the columns before 0 too
      const uint32_t lo = (at >= 0 && at < words) ? m[at] : 0u;
      const uint32_t hi = ((c & 31) != 0 && at + 1 < words) ? m[at + 1] : 0u;
      w = __funnelshift_r(lo, hi, c & 31);
    }
    s_allow[i] = w;
    if constexpr (LISTS) s_touch[i] = 0u;
  }
  RowPlan P{};
  int32_t *s_cnt = s_dyn;
  int32_t *s_last = s_dyn + (A.hist ? TILE : 0);
  if constexpr (LISTS) {
    const int n = ((A.hist ? TILE : 0) + (A.bias_ids ? TILE : 0)) / 4;
    for (int i = tid; i < n; i += kRulesThreads) reinterpret_cast<int4 *>(s_dyn)[i] = make_int4(0, 0, 0, 0);
    __syncthreads();
    if (A.hist != nullptr) {
      P = plan_row(A.cfg[row], A.V);
      const int h0 = A.hist_off[row], h1 = P.pen_on ? A.hist_off[row + 1] : h0;
      for (int64_t j = static_cast<int64_t>(h0) + tid; j < h1; j += kRulesThreads) {
        const int t = A.hist[j];
        const int u = t - c0;
        if (t >= 0 && t < A.V && u >= 0 && u < TILE) {
          atomicAdd(&s_cnt[u], 1);
          atomicOr(&s_touch[u >> 5], 1u << (u & 31));
        }
      }
    }
    if (A.bias_ids != nullptr) {
      const int b0 = A.bias_off[row], b1 = A.bias_off[row + 1];
      for (int64_t j = static_cast<int64_t>(b0) + tid; j < b1; j += kRulesThreads) {
        const int t = A.bias_ids[j];
        const int u = t - c0;
        if (t >= 0 && t < A.V && u >= 0 && u < TILE) {
          atomicMax(&s_last[u], static_cast<int>(j - b0) + 1);
          atomicOr(&s_touch[u >> 5], 1u << (u & 31));
        }
      }
    }
  }
  __syncthreads();

  constexpr uint32_t ALL = (1u << N) - 1u;
#pragma unroll
  for (int i = 0; i < VPT; i++) {
    const int q = (tid + i * kRulesThreads) * N;  // the vector's first column, from c0
    const int c = c0 + q;
    if (c >= A.V) continue;
    const uint32_t allow = (s_allow[q >> 5] >> (q & 31)) & ALL;
    uint32_t touch = 0u;
    if constexpr (LISTS) touch = (s_touch[q >> 5] >> (q & 31)) & allow;
    uint4 r;
    if constexpr (INPLACE) {
      if (allow == ALL && touch == 0u) continue;
      if (allow != 0u) r = load_row_vec(in, shift, A.V, k0 + i * kRulesThreads);
    } else {
      r = raw[i];
    }
    float x[N];
    if (allow != 0u) RowElem<Ti>::unpack(r, x);
    if constexpr (LISTS) {
      if (touch != 0u) {
#pragma unroll
        for (int j = 0; j < N; j++) {
          if ((touch >> j) & 1u) {
            if (A.hist != nullptr) {
              const int n = s_cnt[q + j];
              if (n > 0) x[j] = penalize(x[j], n, P);
            }
            if (A.bias_ids != nullptr) {
              const int b = s_last[q + j];
              if (b > 0) x[j] = __fadd_rn(x[j], A.bias_vals[A.bias_off[row] + b - 1]);
            }
          }
        }
      }
    }
#pragma unroll
    for (int j = 0; j < N; j++)
      if (!((allow >> j) & 1u)) x[j] = __int_as_float(0xFF800000);
    store_row_vec<N>(out, A.V, c, x, aligned);
  }
}

template <typename Ti, typename To, int VPT, bool INPLACE>
cudaError_t launch_tiles(RulesArgs &A, int B, cudaStream_t st) {
  constexpr int N = RowElem<Ti>::N;
  constexpr int TILE = kRulesThreads * VPT * N;
  A.tiles = static_cast<int>((static_cast<int64_t>(A.V) + N - 1 + TILE - 1) / TILE);
  const int64_t ctas = static_cast<int64_t>(B) * (A.tiles + (A.n_allowed != nullptr ? 1 : 0));
  if (ctas > 0x7FFFFFFF) return cudaErrorInvalidConfiguration;
  const size_t smem = sizeof(int32_t) * TILE * ((A.hist ? 1 : 0) + (A.bias_ids ? 1 : 0));
  if (smem > 0)
    rules_kernel<Ti, To, VPT, INPLACE, true><<<static_cast<unsigned>(ctas), kRulesThreads, smem, st>>>(A);
  else
    rules_kernel<Ti, To, VPT, INPLACE, false><<<static_cast<unsigned>(ctas), kRulesThreads, 0, st>>>(A);
  return cudaGetLastError();
}

// Tiles of 4096 columns; of one vector per thread while the larger ones
// would leave SMs without a CTA.
template <typename Ti, typename To, bool INPLACE>
cudaError_t launch_rules(RulesArgs &A, int B, cudaStream_t st) {
  constexpr int VPT = 4096 / (kRulesThreads * RowElem<Ti>::N);
  if (static_cast<int64_t>(B) * ((A.V + 4095) / 4096) < 2 * current_sms())
    return launch_tiles<Ti, To, 1, INPLACE>(A, B, st);
  return launch_tiles<Ti, To, VPT, INPLACE>(A, B, st);
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
  if (pz::misaligned(logits, es) || pz::misaligned(out, eo) || pz::misaligned(R.mask, 4))
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
