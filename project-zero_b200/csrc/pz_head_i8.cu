// pz_head_i8.cu — the LM head in 8-bit integers: rows quantised with a scale
// of their own, and the product of quantised tokens with a quantised
// classifier.
//
// Quantisation of a row x of K values (tokens and channels alike):
//   top = max |x|;  scale = top / 127;  inv = 127 / top;  q = rint(x * inv)
// each step rounded to fp32, rint to even.  |x * inv| <= 127 (1 + 2^-23), so
// q is in [-127, 127] without a clamp.  A row whose top is below 2^-100
// (127 / top would leave fp32) becomes zeros with scale 0; a row that holds
// an inf or a NaN becomes zeros with scale NaN, so its products are NaN and
// not numbers that look right.
//
// Product: out[m][n] = float(sum_k a[m][k] w[n][k]) * (a_scale[m] * w_scale[n]),
// the sum in 32-bit integers (exact for K < 2^17), then three fp32 roundings,
// and one to bf16 where that is the output.
#include "pz_rowvec.cuh"
#include "pz_status.cuh"

namespace pz {
namespace {

constexpr int kQuantThreads = 256;
constexpr int kQuantRes = 4;  // 16-byte vectors of a row that a thread keeps in registers

struct QuantArgs {
  const void *x;
  int64_t ld;
  int rows, cols;
  int8_t *q;
  int64_t ld_q;
  float *scale;
};

// One CTA per row; the row is read once while it fits the registers
// (16 KB), else a second time from L2.
template <typename T>
__global__ void __launch_bounds__(kQuantThreads) quantize_kernel(const QuantArgs A) {
  constexpr int N = RowElem<T>::N;
  constexpr int NT = kQuantThreads;
  __shared__ float s_top[NT / 32];
  __shared__ int s_bad[NT / 32];
  const int64_t row = blockIdx.x;
  const int tid = threadIdx.x;
  const T *x_row = static_cast<const T *>(A.x) + row * A.ld;
  int8_t *q_row = A.q + row * A.ld_q;
  const int shift = row_shift(x_row);
  const int vecs = (A.cols + shift + N - 1) / N;
  uint4 raw[kQuantRes];
  float top = 0.0f;
  int bad = 0;
  auto look = [&](const uint4 &r, int k) {
    float x[N];
    RowElem<T>::unpack(r, x);
    const int c = k * N - shift;
#pragma unroll
    for (int j = 0; j < N; j++)
      if (c + j >= 0 && c + j < A.cols) {
        bad |= !(fabsf(x[j]) <= 3.402823466e38f);
        top = fmaxf(top, fabsf(x[j]));
      }
  };
#pragma unroll
  for (int i = 0; i < kQuantRes; i++)
    if (tid + i * NT < vecs) raw[i] = load_row_vec(x_row, shift, A.cols, tid + i * NT);
#pragma unroll
  for (int i = 0; i < kQuantRes; i++)
    if (tid + i * NT < vecs) look(raw[i], tid + i * NT);
  for (int k = tid + kQuantRes * NT; k < vecs; k += NT) look(load_row_vec(x_row, shift, A.cols, k), k);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, o));
  bad = __any_sync(0xFFFFFFFFu, bad);
  if ((tid & 31) == 0) {
    s_top[tid >> 5] = top;
    s_bad[tid >> 5] = bad;
  }
  __syncthreads();
  for (int i = 0; i < NT / 32; i++) {
    top = fmaxf(top, s_top[i]);
    bad |= s_bad[i];
  }
  const bool some = !bad && top >= 7.888609052e-31f;  // 2^-100
  const float inv = some ? __fdiv_rn(127.0f, top) : 0.0f;
  if (tid == 0) A.scale[row] = bad ? __int_as_float(0x7FC00000) : some ? __fdiv_rn(top, 127.0f) : 0.0f;
  auto write = [&](const uint4 &r, int k) {
    float x[N];
    RowElem<T>::unpack(r, x);
    const int c = k * N - shift;
    uint32_t w[N / 4];
#pragma unroll
    for (int j = 0; j < N; j++) {
      const int q = some ? __float2int_rn(__fmul_rn(x[j], inv)) : 0;
      const uint32_t b = static_cast<uint32_t>(q & 0xFF) << (8 * (j & 3));
      w[j / 4] = (j & 3) == 0 ? b : (w[j / 4] | b);
    }
    if (shift == 0 && c + N <= A.cols) {
      if constexpr (N == 4)
        *reinterpret_cast<uint32_t *>(q_row + c) = w[0];
      else
        *reinterpret_cast<uint2 *>(q_row + c) = make_uint2(w[0], w[N / 4 - 1]);
    } else {
#pragma unroll
      for (int j = 0; j < N; j++)
        if (c + j >= 0 && c + j < A.cols) q_row[c + j] = static_cast<int8_t>(w[j / 4] >> (8 * (j & 3)));
    }
  };
#pragma unroll
  for (int i = 0; i < kQuantRes; i++)
    if (tid + i * NT < vecs) write(raw[i], tid + i * NT);
  for (int k = tid + kQuantRes * NT; k < vecs; k += NT) write(load_row_vec(x_row, shift, A.cols, k), k);
}

cudaError_t launch_quantize(const QuantArgs &A, pz_dtype dtype, cudaStream_t st) {
  if (dtype == PZ_DTYPE_F32)
    quantize_kernel<float><<<A.rows, kQuantThreads, 0, st>>>(A);
  else
    quantize_kernel<bf16_t><<<A.rows, kQuantThreads, 0, st>>>(A);
  return cudaGetLastError();
}

struct MatmulArgs {
  const int8_t *a;
  const float *a_scale;
  const int8_t *w;
  const float *w_scale;
  int M, N, K;
  int64_t ld_a, ld_w, ld_out;
  void *out;
};

constexpr int kMatRows = 8;

// One warp takes a channel at a time and 8 tokens, 4 products per instruction.
template <typename T>
__global__ void __launch_bounds__(256) matmul_i8_kernel(const MatmulArgs A) {
  const int lane = threadIdx.x & 31;
  const int n = blockIdx.x * 8 + (threadIdx.x >> 5);
  if (n >= A.N) return;
  const int m0 = blockIdx.y * kMatRows;
  const int8_t *w = A.w + static_cast<int64_t>(n) * A.ld_w;
  int acc[kMatRows];
#pragma unroll
  for (int r = 0; r < kMatRows; r++) acc[r] = 0;
  const int whole = A.K / 4;
  for (int k = lane; k < whole; k += 32) {
    const int x = reinterpret_cast<const int *>(w)[k];
#pragma unroll
    for (int r = 0; r < kMatRows; r++)
      if (m0 + r < A.M)
        acc[r] = __dp4a(x, reinterpret_cast<const int *>(A.a + static_cast<int64_t>(m0 + r) * A.ld_a)[k], acc[r]);
  }
  for (int k = whole * 4 + lane; k < A.K; k += 32)
#pragma unroll
    for (int r = 0; r < kMatRows; r++)
      if (m0 + r < A.M) acc[r] += w[k] * A.a[static_cast<int64_t>(m0 + r) * A.ld_a + k];
#pragma unroll
  for (int r = 0; r < kMatRows; r++) {
    const int s = __reduce_add_sync(0xFFFFFFFFu, acc[r]);
    if (lane == 0 && m0 + r < A.M)
      RowElem<T>::put(static_cast<T *>(A.out) + static_cast<int64_t>(m0 + r) * A.ld_out + n,
                      __fmul_rn(__int2float_rn(s), __fmul_rn(A.a_scale[m0 + r], A.w_scale[n])));
  }
}

cudaError_t launch_matmul(const MatmulArgs &A, pz_dtype out_dtype, cudaStream_t st) {
  const dim3 grid((A.N + 7) / 8, (A.M + kMatRows - 1) / kMatRows);
  if (out_dtype == PZ_DTYPE_F32)
    matmul_i8_kernel<float><<<grid, 256, 0, st>>>(A);
  else
    matmul_i8_kernel<bf16_t><<<grid, 256, 0, st>>>(A);
  return cudaGetLastError();
}

pz_status check_quantize(const void *x, pz_dtype dtype, int rows, int cols, int64_t ld, const int8_t *q, int64_t ld_q,
                         const float *scale) {
  if (!x || !q || !scale || rows < 0 || cols <= 0 || ld < cols || ld_q < cols)
    return report(PZ_ERR_INVALID_ARGS, "pz_quantize_rows_i8: null pointer or bad size");
  if (dtype != PZ_DTYPE_F32 && dtype != PZ_DTYPE_BF16)
    return report(PZ_ERR_INVALID_ARGS, "pz_quantize_rows_i8: bad dtype");
  if (misaligned(x, elem_bytes(dtype)) || misaligned(q, 16) || ld_q % 16 != 0 || misaligned(scale, 4))
    return report(PZ_ERR_INVALID_ARGS, "pz_quantize_rows_i8: q and its rows start on 16 bytes, x on its elements");
  return PZ_OK;
}

pz_status check_matmul(const MatmulArgs &A, pz_dtype out_dtype) {
  if (!A.a || !A.a_scale || !A.w || !A.w_scale || !A.out || A.M < 0 || A.N <= 0 || A.K <= 0 || A.ld_a < A.K ||
      A.ld_w < A.K || A.ld_out < A.N)
    return report(PZ_ERR_INVALID_ARGS, "pz_matmul_i8: null pointer or bad size");
  if (out_dtype != PZ_DTYPE_F32 && out_dtype != PZ_DTYPE_BF16)
    return report(PZ_ERR_INVALID_ARGS, "pz_matmul_i8: bad out_dtype");
  if (misaligned(A.a, 16) || misaligned(A.w, 16) || A.ld_a % 16 != 0 || A.ld_w % 16 != 0 || misaligned(A.a_scale, 4) ||
      misaligned(A.w_scale, 4) || misaligned(A.out, elem_bytes(out_dtype)))
    return report(PZ_ERR_INVALID_ARGS, "pz_matmul_i8: 8-bit rows start on 16 bytes, out on its elements");
  if (A.K >= PZ_MATMUL_I8_MAX_K)
    return report(PZ_ERR_UNSUPPORTED, "pz_matmul_i8: K of 2^17 or more may overflow the 32-bit sums");
  return PZ_OK;
}

}  // namespace
}  // namespace pz

extern "C" {

pz_status pz_quantize_rows_i8(const void *x, pz_dtype dtype, int rows, int cols, int64_t ld, int8_t *q, int64_t ld_q,
                              float *scale, void *stream) {
  const pz_status s = pz::check_quantize(x, dtype, rows, cols, ld, q, ld_q, scale);
  if (s != PZ_OK || rows == 0) return s;
  const pz::QuantArgs A{x, ld, rows, cols, q, ld_q, scale};
  const cudaError_t e = pz::launch_quantize(A, dtype, static_cast<cudaStream_t>(stream));
  return e == cudaSuccess ? PZ_OK : pz::report_cuda(e);
}

pz_status pz_matmul_i8(const int8_t *a, int64_t ld_a, const float *a_scale, int M, const int8_t *w, int64_t ld_w,
                       const float *w_scale, int N, int K, void *out, pz_dtype out_dtype, int64_t ld_out,
                       void *stream) {
  const pz::MatmulArgs A{a, a_scale, w, w_scale, M, N, K, ld_a, ld_w, ld_out, out};
  const pz_status s = pz::check_matmul(A, out_dtype);
  if (s != PZ_OK || M == 0) return s;
  const cudaError_t e = pz::launch_matmul(A, out_dtype, static_cast<cudaStream_t>(stream));
  return e == cudaSuccess ? PZ_OK : pz::report_cuda(e);
}

pz_status pz_lm_head_logits_i8(const void *hidden, pz_dtype hidden_dtype, int B, int dim, int64_t ld_hidden,
                               const int8_t *w_q, int64_t ld_w, const float *w_scale, int V, void *logits,
                               pz_dtype logits_dtype, int64_t ld, int8_t *hidden_q, int64_t ld_q, float *hidden_scale,
                               void *stream) {
  pz_status s = pz::check_quantize(hidden, hidden_dtype, B, dim, ld_hidden, hidden_q, ld_q, hidden_scale);
  if (s != PZ_OK) return s;
  const pz::MatmulArgs A{hidden_q, hidden_scale, w_q, w_scale, B, V, dim, ld_q, ld_w, ld, logits};
  s = pz::check_matmul(A, logits_dtype);
  if (s != PZ_OK || B == 0) return s;
  const pz::QuantArgs Q{hidden, ld_hidden, B, dim, hidden_q, ld_q, hidden_scale};
  cudaError_t e = pz::launch_quantize(Q, hidden_dtype, static_cast<cudaStream_t>(stream));
  if (e == cudaSuccess) e = pz::launch_matmul(A, logits_dtype, static_cast<cudaStream_t>(stream));
  return e == cudaSuccess ? PZ_OK : pz::report_cuda(e);
}

}  // extern "C"
