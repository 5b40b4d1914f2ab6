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
#include <cuda.h>

#include <atomic>

#include "pz_epilogue.cuh"
#include "pz_rowvec.cuh"
#include "pz_status.cuh"
#include "pz_tcgen05.cuh"

namespace pz {
namespace {

constexpr int kQuantRes = 4;  // 16-byte vectors of a row that a thread keeps in registers

struct QuantArgs {
  const void *x;
  int64_t ld;
  int rows, cols;
  int8_t *q;
  int64_t ld_q;
  float *scale;
};

// One CTA per row; the row is read once while it fits the registers (64 bytes
// a thread), what is beyond that a second time from L2.  Bound: HBM for rows
// that fit (128256 x 4096 bf16: 235 us, 6.7 TB/s).  To keep the arithmetic under it:
// the maximum of magnitudes carries NaN by itself, and adding 1.5 * 2^23
// rounds to a whole number (to even, as rint does) whose low byte is q.  The
// product and the sum are separate instructions for one value: the packed
// forms for two were joined into one, whose single rounding moves ties
// (63.4999998 became 63 where the rounded product 63.5 gives 64).
template <typename T, int NT>
__global__ void __launch_bounds__(NT) quantize_kernel(const QuantArgs A) {
  constexpr int N = RowElem<T>::N;
  pdl_launch_dependents();  // the product may start fetching its weights
  __shared__ float s_top[NT / 32];
  const int64_t row = blockIdx.x;
  const int tid = threadIdx.x;
  const T *x_row = static_cast<const T *>(A.x) + row * A.ld;
  int8_t *q_row = A.q + row * A.ld_q;
  const int shift = row_shift(x_row);
  const int vecs = (A.cols + shift + N - 1) / N;
  const WholeVecs whole = whole_vecs<T>(shift, A.cols);
  // columns outside the row as 0: they change no maximum
  auto is_whole = [&](int k) { return k >= whole.first && k < whole.last; };
  auto load = [&](int k) {
    return is_whole(k) ? load16(x_row + (k * N - shift)) : load_edge(x_row, A.cols, k * N - shift, 0.0f);
  };
  uint4 raw[kQuantRes];
#pragma unroll
  for (int i = 0; i < kQuantRes; i++) {
    const int k = tid + i * NT;
    raw[i] = is_whole(k) ? load16(x_row + (k * N - shift)) : make_uint4(0u, 0u, 0u, 0u);
  }
  // the edges once every whole vector is on its way: a call between them would hold them up
#pragma unroll
  for (int i = 0; i < kQuantRes; i++)
    if (tid + i * NT < vecs && !is_whole(tid + i * NT)) raw[i] = load(tid + i * NT);
  float top = 0.0f;
#pragma unroll
  for (int i = 0; i < kQuantRes; i++) top = max_nan(top, RowElem<T>::max_abs_nan(raw[i]));
  for (int k = tid + kQuantRes * NT; k < vecs; k += NT) top = max_nan(top, RowElem<T>::max_abs_nan(load(k)));
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) top = max_nan(top, __shfl_xor_sync(0xFFFFFFFFu, top, o));
  if ((tid & 31) == 0) s_top[tid >> 5] = top;
  __syncthreads();
  for (int i = 0; i < NT / 32; i++) top = max_nan(top, s_top[i]);
  const bool bad = !(top <= 3.402823466e38f);  // an infinity or NaN
  const bool some = !bad && top >= 7.888609052e-31f;  // 2^-100
  const float inv = some ? __fdiv_rn(127.0f, top) : 0.0f;
  if (tid == 0) A.scale[row] = bad ? __int_as_float(0x7FC00000) : some ? __fdiv_rn(top, 127.0f) : 0.0f;
  auto write = [&](uint4 r, int k) {
    if (!some) r = make_uint4(0u, 0u, 0u, 0u);  // (inf times 0 is no number)
    float x[N];
    RowElem<T>::unpack(r, x);
    auto whole_number = [&](float v) { return __float_as_uint(__fadd_rn(__fmul_rn(v, inv), 12582912.0f)); };
    uint32_t w[N / 4];
#pragma unroll
    for (int j = 0; j < N / 4; j++) {
      const uint32_t lo = __byte_perm(whole_number(x[4 * j]), whole_number(x[4 * j + 1]), 0x0040);
      const uint32_t hi = __byte_perm(whole_number(x[4 * j + 2]), whole_number(x[4 * j + 3]), 0x0040);
      w[j] = __byte_perm(lo, hi, 0x5410);
    }
    const int c = k * N - shift;
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
  for (int k = tid + kQuantRes * NT; k < vecs; k += NT) write(load(k), k);
}

// 128 threads while their registers hold the row (8 KB), 256 beyond.  Both
// sides, 128 and 256 threads, us: 128256 x 4096 bf16 235 and 357, 32000 x 1000
// bf16 36 and 66, 1024 x 4096 bf16 3.3 and 4.3; 128256 x 8192 bf16 666 and 489,
// 128256 x 6144 bf16 473 and 421, 128256 x 3000 f32 389 and 328, 512 x 4096 f32
// 4.1 and 3.0, 1 x 4096 f32 3.3 and 2.0.  From 8 to about 11 KB the narrow side
// still wins where rows are many (128256 x 2560 f32 272 and 297, 128256 x 5120
// bf16 351 and 391) and loses on a batch of tokens whose rows come from memory
// (1024 x 2560 f32 10.1 and 8.2): tokens are quantised at every call, a
// classifier once.  Threads in a number set at run time to fit each row were
// slower than the better of the two.  Rows of 2 KB are bound by the start and
// the end of a CTA each, 2.5 times their bytes' time.  Rows at odd addresses
// are stored a byte at a time (32000 x 1001 bf16 62 us, 32000 x 1000 37).
template <typename T>
void launch_quantize_as(const QuantArgs &A, cudaStream_t st) {
  constexpr int narrow_cols = 128 * kQuantRes * RowElem<T>::N;
  if (A.cols <= narrow_cols)
    quantize_kernel<T, 128><<<A.rows, 128, 0, st>>>(A);
  else
    quantize_kernel<T, 256><<<A.rows, 256, 0, st>>>(A);
}

cudaError_t launch_quantize(const QuantArgs &A, pz_dtype dtype, cudaStream_t st) {
  if (dtype == PZ_DTYPE_F32)
    launch_quantize_as<float>(A, st);
  else
    launch_quantize_as<bf16_t>(A, st);
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

// ---------------------------------------------------------------------------
// The product on the tensor cores.  out^T = W a^T: a tile is 128 channels
// (the instruction's M, so a decode batch of few tokens still fills it) by
// up to 256 tokens (its N, a multiple of 16).
//
// Few tokens: bound by HBM, every weight read once: a persistent CTA per SM
// keeps about 200 KB of weights and tokens in flight (1 token, dim 2560,
// 128256 channels: 53 us, 6.2 TB/s; 64 tokens, dim 4096, 151936 channels: 108
// us, 6.1 TB/s).  Many tokens: bound by what the SMs fetch from L2 (54 bytes a
// clock each, measured; a tile of 128 x 256 wants 384 bytes per 32768
// products, half a tile in a pair of CTAs 256), and beside it by the tensor
// cores and the power limit (4096 tokens, dim 4096, 128256 channels: 1.42 to
// 1.55 ms, 2.8 to 3.0 POP/s).
//
// Warp 0 issues TMA loads (128 channels x 128 bytes of K and the tokens'
// part, 128-byte swizzle) into a ring of stages; one thread of warp 1 issues
// four tcgen05.mma (K = 32 each) per block; the sums lie in tensor memory,
// two tiles of them, so that the other warps read, scale and store one tile
// while the next is summed.  A lane of the epilogue holds one channel: a
// warp stores 32 neighbouring logits of a token at a time.  Eight warps of
// it (301 tokens, dim 128, 32003 channels, nothing but epilogue: 14.1 us,
// 16.3 with four).
//
// Rows and K past the matrices' ends arrive as zeros.  Every wait is bounded:
// one that runs out (4 s: no work of this kernel takes as long, a GPU that was
// held in between does) ends the CTA once its products are done and its loads
// have landed, with NaN in the outputs it did not reach: every warp of the
// epilogue fills its own tokens.
// ---------------------------------------------------------------------------
using OwnTokens = EpilogueTokens<8>;  // of each of the epilogue's warps
constexpr int kTcWarps = OwnTokens::WARPS;
constexpr int kTcThreads = 64 + 32 * kTcWarps;
constexpr int kTcChannels = 128;
constexpr int kTcTokens = 256;
constexpr int kTcK = 128;             // bytes of K per block; a stage is one or several
constexpr int kTcMaxStages = 12;
constexpr int kTcRing = 200 * 1024;   // shared memory of the ring

struct TcArgs {
  const float *a_scale, *w_scale;
  void *out;
  int64_t ld_out;
  int M, N;
  int nt;          // tokens per tile, a multiple of 16 (PAIR: 32)
  int tok_tiles;
  int tiles;       // channel tiles x tok_tiles
  int k_blocks;    // K in blocks of kTcK
  int sub;         // blocks per stage
  int k_stages;    // stages' worth of K
  int k_steps;     // K in steps of 32
  int stages;
  int cols;        // tensor memory columns, a power of two >= 2 nt
};

// PAIR: clusters of two CTAs (two SMs) sum tiles of 256 channels together,
// each CTA's 128 from its own weights and tokens that lie half in either's
// shared memory, so that a CTA reads half as many tokens.  The leading CTA's
// barriers count both CTAs' loads, it issues the products for both and tells
// both of their end.
template <typename T, bool PAIR>
__global__ void __launch_bounds__(kTcThreads, 1)
    matmul_i8_kernel(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_a, const TcArgs A) {
  extern __shared__ unsigned char s_raw[];
  __shared__ __align__(8) uint64_t s_full[kTcMaxStages], s_empty[kTcMaxStages], s_sum[2], s_free[2], s_drain;
  __shared__ uint32_t s_tmem;
  __shared__ volatile int s_stop;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const uint32_t ring = (smem_addr(s_raw) + 1023u) & ~1023u;
  const uint32_t rank = PAIR ? blockIdx.x & 1u : 0u;
  const int tile0 = PAIR ? blockIdx.x >> 1 : blockIdx.x, tile_step = PAIR ? gridDim.x >> 1 : gridDim.x;
  constexpr int kTileChannels = PAIR ? 2 * kTcChannels : kTcChannels;
  const int a_rows = PAIR ? A.nt / 2 : A.nt;  // tokens in this CTA's shared memory
  const uint32_t w_bytes = kTcChannels * kTcK, a_bytes = static_cast<uint32_t>(a_rows) * kTcK;
  const uint32_t block_bytes = w_bytes + a_bytes, stage_bytes = block_bytes * A.sub;
  const uint32_t full = smem_addr(s_full), empty = smem_addr(s_empty), sum = smem_addr(s_sum), free_ = smem_addr(s_free);

  if (tid == 0) {
    tma_prefetch_map(&map_w);
    tma_prefetch_map(&map_a);
    for (int i = 0; i < A.stages; i++) {
      mbar_init(full + 8 * i, 1);
      mbar_init(empty + 8 * i, 1);
    }
    for (int i = 0; i < 2; i++) {
      mbar_init(sum + 8 * i, 1);
      mbar_init(free_ + 8 * i, PAIR ? 2 * kTcWarps : kTcWarps);
    }
    mbar_init(smem_addr(&s_drain), 1);
    mbar_init_fence();
    s_stop = 0;
  }
  if (warp == 2) tmem_alloc<PAIR>(smem_addr(&s_tmem), static_cast<uint32_t>(A.cols));
  tc_fence_before();
  __syncthreads();
  if (PAIR) pair_sync();  // the other CTA's barriers are set up too
  tc_fence_after();
  const uint32_t tmem = s_tmem;
  int64_t loads = 0;  // stages that this thread has loaded

  if (warp == 0) {
    if (lane == 0) {
      // The weights of the first stages do not depend on what runs before
      // this kernel (the tokens' quantisation): they are on their way first.
      const int mine = (A.tiles - tile0 + tile_step - 1) / tile_step;
      const int64_t total = static_cast<int64_t>(mine) * A.k_stages;
      const int early = static_cast<int>(total < A.stages ? total : A.stages);
      // (one thread feeds the SM: no division, no address worked out twice
      // between two loads)
      const uint32_t lead = PAIR ? remote_addr(full, 0) : full;  // the barriers that count the loads
      auto weights = [&](uint32_t slot, uint32_t bar, int x, int y, int n) {
        if (rank == 0) mbar_expect(bar, (PAIR ? 2 : 1) * block_bytes * n);
        for (int b = 0; b < n; b++, slot += block_bytes, x += kTcK)
          tma_load<PAIR>(slot, &map_w, x, y, bar - full + lead);
      };
      {
        int tile = tile0, ks = 0, y = tile / A.tok_tiles * kTileChannels + rank * kTcChannels;
        for (int i = 0; i < early; i++) {
          weights(ring + i * stage_bytes, full + 8 * i, ks * A.sub * kTcK, y, min(A.sub, A.k_blocks - ks * A.sub));
          if (++ks == A.k_stages) {
            ks = 0;
            tile += tile_step;
            y = tile / A.tok_tiles * kTileChannels + rank * kTcChannels;
          }
        }
      }
      pdl_wait();
      int64_t n = 0;  // (loads)
      uint32_t slot = ring, bar = full, gone = empty, ph = 1;
      const uint32_t ring_end = ring + A.stages * stage_bytes;
      bool ok = true;
      for (int tile = tile0; ok && tile < A.tiles; tile += tile_step) {
        const int yw = tile / A.tok_tiles * kTileChannels + rank * kTcChannels;
        const int ya = tile % A.tok_tiles * A.nt + rank * a_rows;
        for (int kb = 0; kb < A.k_blocks; kb += A.sub) {
          const int blocks = min(A.sub, A.k_blocks - kb);
          int x = kb * kTcK;
          if (n >= early) {
            if (!(ok = mbar_wait(gone, ph, &s_stop))) break;
            weights(slot, bar, x, yw, blocks);
          }
          uint32_t to = slot + w_bytes;
          for (int b = 0; b < blocks; b++, to += block_bytes, x += kTcK)
            tma_load<PAIR>(to, &map_a, x, ya, bar - full + lead);
          n++;
          slot += stage_bytes;
          bar += 8;
          gone += 8;
          if (slot == ring_end) {
            slot = ring;
            bar = full;
            gone = empty;
            ph ^= 1;
          }
        }
      }
      // no commit may be on its way to this CTA's barriers when its memory goes
      for (int64_t i = n < A.stages ? 0 : n - A.stages; ok && PAIR && i < n; i++)
        ok = mbar_wait(empty + 8 * static_cast<uint32_t>(i % A.stages), static_cast<uint32_t>((i / A.stages) & 1), &s_stop);
      loads = n;
    }
    __syncwarp();
  } else if (warp == 1) {
    if (lane == 0 && rank == 0) {
      const uint32_t inst = i8_instruction(kTileChannels, A.nt);
      const int whole = A.k_steps / (kTcK / 32);  // blocks of four steps; the last may have fewer
      const uint64_t block_desc = block_bytes >> 4, a_desc = w_bytes >> 4;
      uint64_t dw = smem_desc(ring);
      const uint64_t dw_end = dw + static_cast<uint64_t>(A.stages) * (stage_bytes >> 4);
      uint32_t bar = full, gone = empty, ph = 0;
      int t = 0;
      bool ok = true;
      for (int tile = tile0; ok && tile < A.tiles; tile += tile_step, t++) {
        const int acc = t & 1;
        if (!(ok = mbar_wait(free_ + 8 * acc, ((t >> 1) & 1) ^ 1, &s_stop))) break;
        tc_fence_after();
        const uint32_t d = tmem + static_cast<uint32_t>(acc * (A.cols / 2));
        bool add = false;
        for (int kb = 0; kb < A.k_blocks; kb += A.sub) {
          if (!(ok = mbar_wait(bar, ph, &s_stop))) break;
          tc_fence_after();
          const int blocks = min(A.sub, A.k_blocks - kb);
          uint64_t w = dw;
          for (int b = 0; b < blocks; b++, w += block_desc) {
            if (kb + b < whole) {
#pragma unroll
              for (int k = 0; k < kTcK / 32; k++) tc_mma_i8<PAIR>(d, w + 2 * k, w + a_desc + 2 * k, inst, add || k > 0);
            } else {
              for (int k = 0; k < A.k_steps - (kb + b) * (kTcK / 32); k++)
                tc_mma_i8<PAIR>(d, w + 2 * k, w + a_desc + 2 * k, inst, add || k > 0);
            }
            add = true;
          }
          tc_commit<PAIR>(gone);
          dw += stage_bytes >> 4;
          bar += 8;
          gone += 8;
          if (dw == dw_end) {
            dw = smem_desc(ring);
            bar = full;
            gone = empty;
            ph ^= 1;
          }
        }
        if (ok) tc_commit<PAIR>(sum + 8 * acc);
      }
      // no product may be under way when the CTA's memory goes, whether or not
      // the epilogue waited for it (where it did, this costs nothing)
      tc_commit<PAIR>(smem_addr(&s_drain));
      volatile int ignore = 0;
      mbar_wait(smem_addr(&s_drain), 0, &ignore);
    }
    __syncwarp();
  } else {
    pdl_wait();
    const int quarter = OwnTokens::quarter(warp);
    const int first = OwnTokens::first(warp - 2);
    const int row = quarter * 32 + lane;
    int t = 0;
    bool ok = true;
    const uint32_t freed = PAIR ? remote_addr(free_, 0) : free_;
    for (int tile = tile0; tile < A.tiles; tile += tile_step, t++) {
      const int acc = t & 1;
      const int n = tile / A.tok_tiles * kTileChannels + rank * kTcChannels + row;
      const int m0 = tile % A.tok_tiles * A.nt;
      T *out = static_cast<T *>(A.out) + static_cast<int64_t>(m0) * A.ld_out + n;
      const int tokens = min(A.nt, A.M - m0);
      // the scales are on their way while the sums are waited for
      const float sw = n < A.N ? A.w_scale[n] : 0.0f;
      float sa = first + lane < tokens ? __ldcg(A.a_scale + m0 + first + lane) : 0.0f;
      if (ok) ok = mbar_wait(sum + 8 * acc, (t >> 1) & 1, &s_stop);
      ok = __all_sync(0xFFFFFFFFu, ok);
      if (!ok) {
        for (int c = first; c < tokens; c += OwnTokens::STEP)
          for (int j = 0; j < OwnTokens::count(c, tokens); j++)
            if (n < A.N) RowElem<T>::put(out + static_cast<int64_t>(c + j) * A.ld_out, __int_as_float(0x7FC00000));
        continue;
      }
      tc_fence_after();
      const uint32_t at = tmem + static_cast<uint32_t>(acc * (A.cols / 2)) + (static_cast<uint32_t>(quarter * 32) << 16);
      // 32 tokens at a time; each lane fetches one token's scale, ahead of
      // the stores that the compiler may not move a load across
      for (int c = first; c < tokens; c += OwnTokens::STEP) {
        int v[32];
        __syncwarp();
        tmem_load32(at + c, v);
        const float here = sa;
        if (c + OwnTokens::STEP + lane < tokens) sa = __ldcg(A.a_scale + m0 + c + OwnTokens::STEP + lane);
        tmem_load_wait();
        float x[32];
#pragma unroll
        for (int j = 0; j < 32; j++)
          x[j] = __fmul_rn(__int2float_rn(v[j]), __fmul_rn(__shfl_sync(0xFFFFFFFFu, here, j), sw));
        T *o = out + static_cast<int64_t>(c) * A.ld_out;
        if (OwnTokens::count(c, tokens) == OwnTokens::RUN) {
          if (n < A.N) {
#pragma unroll
            for (int j = 0; j < 32; j++) RowElem<T>::put(o + j * A.ld_out, x[j]);
          }
        } else {
#pragma unroll
          for (int j = 0; j < 32; j++)
            if (c + j < tokens && n < A.N) RowElem<T>::put(o + j * A.ld_out, x[j]);
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) PAIR ? mbar_arrive_remote(freed + 8 * acc) : mbar_arrive(freed + 8 * acc);
    }
    __syncwarp();
  }
  tc_fence_before();
  __syncthreads();
  // After a stop: no load may be in flight when the CTA's memory goes (the
  // leading CTA waits for both CTAs' loads; without a stop its products have).
  // Only here is it known whether any role stopped.
  if (s_stop && rank == 0 && tid == 0) {
    for (int64_t i = loads < A.stages ? 0 : loads - A.stages; i < loads; i++) {
      volatile int ignore = 0;
      mbar_wait(full + 8 * static_cast<uint32_t>(i % A.stages), static_cast<uint32_t>((i / A.stages) & 1), &ignore);
    }
  }
  if (PAIR && rank == 1 && tid == 32) {  // nor the leading CTA's signal, which arrives here too
    volatile int ignore = 0;
    mbar_wait(smem_addr(&s_drain), 0, &ignore);
  }
  if (PAIR) pair_sync();  // neither CTA's memory or barriers are used by the other any more
  if (warp == 2) {
    tc_fence_after();
    tmem_free<PAIR>(tmem, static_cast<uint32_t>(A.cols));
  }
}

using EncodeTiled = CUresult (*)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *,
                                 const cuuint64_t *, const cuuint32_t *, const cuuint32_t *, CUtensorMapInterleave,
                                 CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

// The driver's encoder, looked up once (the library does not link libcuda).
EncodeTiled encoder() {
  static std::atomic<void *> known{nullptr};
  void *f = known.load(std::memory_order_acquire);
  if (f == nullptr) {
    cudaDriverEntryPointQueryResult how;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &f, cudaEnableDefault, &how) != cudaSuccess ||
        how != cudaDriverEntryPointSuccess)
      return nullptr;
    known.store(f, std::memory_order_release);
  }
  return reinterpret_cast<EncodeTiled>(f);
}

// 8-bit rows of K values as tiles of `box` rows by 128 bytes.
bool encode_rows(CUtensorMap *map, const int8_t *p, int K, int rows, int64_t ld, int box) {
  const EncodeTiled f = encoder();
  if (f == nullptr) return false;
  const cuuint64_t dims[2] = {static_cast<cuuint64_t>(K), static_cast<cuuint64_t>(rows)};
  const cuuint64_t strides[1] = {static_cast<cuuint64_t>(ld)};
  const cuuint32_t size[2] = {kTcK, static_cast<cuuint32_t>(box)}, step[2] = {1, 1};
  return f(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<int8_t *>(p), dims, strides, size, step,
           CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
           CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// after_quantize: launched behind the tokens' quantisation, whose end the
// kernel waits for itself.
template <typename T, bool PAIR>
cudaError_t launch_matmul_as(const MatmulArgs &P, bool after_quantize, cudaStream_t st) {
  TcArgs A{};
  A.a_scale = P.a_scale;
  A.w_scale = P.w_scale;
  A.out = P.out;
  A.ld_out = P.ld_out;
  A.M = P.M;
  A.N = P.N;
  constexpr int UNIT = PAIR ? 32 : 16;  // the instruction's step of tokens
  A.tok_tiles = (P.M + kTcTokens - 1) / kTcTokens;
  A.nt = ((P.M + A.tok_tiles - 1) / A.tok_tiles + UNIT - 1) / UNIT * UNIT;
  const int a_rows = PAIR ? A.nt / 2 : A.nt, channels = PAIR ? 2 * kTcChannels : kTcChannels;
  const int64_t tiles = static_cast<int64_t>((P.N + channels - 1) / channels) * A.tok_tiles;
  if (tiles > 0x3FFFFFFF) return cudaErrorInvalidConfiguration;
  A.tiles = static_cast<int>(tiles);
  A.k_blocks = (P.K + kTcK - 1) / kTcK;
  A.k_steps = (P.K + 31) / 32;
  // Stages of up to a third of the ring: several blocks of K of the same rows
  // at a time, since 128 bytes here and there is slow from HBM (1 token, dim
  // 2560, 128256 channels: 58.6 us at one block a stage, 55.4 at three; 64
  // tokens, dim 4096, 151936 channels: 127 at one, 116 at two, 123 at three;
  // 4096 tokens in pairs: 1815 at one, 1523 at two).
  const int block = (kTcChannels + a_rows) * kTcK;
  A.sub = kTcRing / 3 / block;
  A.k_stages = (A.k_blocks + A.sub - 1) / A.sub;
  const int stage = block * A.sub;
  A.stages = kTcRing / stage < kTcMaxStages ? kTcRing / stage : kTcMaxStages;
  A.cols = 64;  // (the epilogue reads 32 columns at a time)
  while (A.cols < 2 * A.nt) A.cols *= 2;
  CUtensorMap map_w, map_a;
  if (!encode_rows(&map_w, P.w, P.K, P.N, P.ld_w, kTcChannels) || !encode_rows(&map_a, P.a, P.K, P.M, P.ld_a, a_rows))
    return cudaErrorInvalidValue;
  const size_t smem = static_cast<size_t>(A.stages) * stage + 1024;
  static std::atomic<uint64_t> ready{0};  // devices whose attribute is set
  cudaError_t e = allow_smem(reinterpret_cast<const void *>(matmul_i8_kernel<T, PAIR>), kTcRing + 1024, &ready);
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg{};
  const int groups = current_sms() / (PAIR ? 2 : 1);
  cfg.gridDim = dim3(static_cast<unsigned>((A.tiles < groups ? A.tiles : groups) * (PAIR ? 2 : 1)));
  cfg.blockDim = dim3(kTcThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute at[2];
  int n = 0;
  if (after_quantize) {
    at[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[n++].val.programmaticStreamSerializationAllowed = 1;
  }
  if (PAIR) {
    at[n].id = cudaLaunchAttributeClusterDimension;
    at[n].val.clusterDim.x = 2;
    at[n].val.clusterDim.y = 1;
    at[n++].val.clusterDim.z = 1;
  }
  cfg.attrs = at;
  cfg.numAttrs = n;
  e = cudaLaunchKernelEx(&cfg, matmul_i8_kernel<T, PAIR>, map_w, map_a, A);
  return e != cudaSuccess ? e : cudaGetLastError();
}

// Pairs from here on (dim 4096, 128256 channels, bf16 logits: 64 tokens 88.8
// us alone and 88.3 in pairs, 96: 94.0 and 90.9, 256: 132 and 117, 1024: 489
// and 390; dim 1000, 32003 channels: 64: 11.4 and 11.4, 256: 25.4 and 19.1).
constexpr int kPairTokens = 65;
template <typename T>
cudaError_t launch_matmul_to(const MatmulArgs &A, bool after_quantize, cudaStream_t st) {
  return A.M >= kPairTokens ? launch_matmul_as<T, true>(A, after_quantize, st)
                            : launch_matmul_as<T, false>(A, after_quantize, st);
}
cudaError_t launch_matmul(const MatmulArgs &A, pz_dtype out_dtype, bool after_quantize, cudaStream_t st) {
  return out_dtype == PZ_DTYPE_F32 ? launch_matmul_to<float>(A, after_quantize, st)
                                   : launch_matmul_to<bf16_t>(A, after_quantize, st);
}

// Largest sizes that still fit 32-bit indexes when they are rounded up to a
// vector (columns of a row) or a tile (tokens, channels).
constexpr int kMaxCols = 0x7FFFFFFF - 15, kMaxTiled = 0x7FFFFFFF - 255;

pz_status check_quantize(const void *x, pz_dtype dtype, int rows, int cols, int64_t ld, const int8_t *q, int64_t ld_q,
                         const float *scale) {
  if (!x || !q || !scale || rows < 0 || cols <= 0 || ld < cols || ld_q < cols)
    return report(PZ_ERR_INVALID_ARGS, "pz_quantize_rows_i8: null pointer or bad size");
  if (dtype != PZ_DTYPE_F32 && dtype != PZ_DTYPE_BF16)
    return report(PZ_ERR_INVALID_ARGS, "pz_quantize_rows_i8: bad dtype");
  if (misaligned(x, elem_bytes(dtype)) || misaligned(q, 16) || ld_q % 16 != 0 || misaligned(scale, 4))
    return report(PZ_ERR_INVALID_ARGS, "pz_quantize_rows_i8: q and its rows start on 16 bytes, x on its elements");
  if (rows > 0 && overlap(x, rows_bytes(rows, cols, ld, elem_bytes(dtype)), q, rows_bytes(rows, cols, ld_q, 1)))
    return report(PZ_ERR_INVALID_ARGS, "pz_quantize_rows_i8: q lies over x");
  if (cols > kMaxCols) return report(PZ_ERR_UNSUPPORTED, "pz_quantize_rows_i8: more than 2^31 - 16 columns");
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
  if (A.M > 0 && (overlap(A.out, rows_bytes(A.M, A.N, A.ld_out, elem_bytes(out_dtype)), A.w,
                          rows_bytes(A.N, A.K, A.ld_w, 1)) ||
                  overlap(A.out, rows_bytes(A.M, A.N, A.ld_out, elem_bytes(out_dtype)), A.a,
                          rows_bytes(A.M, A.K, A.ld_a, 1))))
    return report(PZ_ERR_INVALID_ARGS, "pz_matmul_i8: out lies over a or w");
  if (A.K >= PZ_MATMUL_I8_MAX_K)
    return report(PZ_ERR_UNSUPPORTED, "pz_matmul_i8: K of 2^17 or more may overflow the 32-bit sums");
  if (A.M > kMaxTiled || A.N > kMaxTiled)
    return report(PZ_ERR_UNSUPPORTED, "pz_matmul_i8: more than 2^31 - 256 rows");
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
  const cudaError_t e = pz::launch_matmul(A, out_dtype, false, static_cast<cudaStream_t>(stream));
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
  if (e == cudaSuccess) e = pz::launch_matmul(A, logits_dtype, true, static_cast<cudaStream_t>(stream));
  return e == cudaSuccess ? PZ_OK : pz::report_cuda(e);
}

}  // extern "C"
