// pz_epilogue.cuh — which part of a tile of sums each warp of the epilogue
// reads, scales and stores.  Host code too: the split is tested on the CPU.
#pragma once

#ifdef __CUDACC__
#define PZ_HOST_DEVICE __host__ __device__ __forceinline__
#else
#define PZ_HOST_DEVICE inline
#endif

namespace pz {

// W warps, four to a group.  Within a group each reads a quarter of tensor
// memory's lanes (the hardware's rule: by the warp's index in the block);
// the groups take runs of 32 tokens in turn.  Every token of every quarter
// has one owner, which also fills it where the sums never came.
template <int W>
struct EpilogueTokens {
  static_assert(W % 4 == 0, "four quarters of tensor memory");
  static constexpr int WARPS = W;
  static constexpr int RUN = 32;           // tokens that a warp takes at a time
  static constexpr int STEP = RUN * W / 4;  // from one of its runs to the next
  static PZ_HOST_DEVICE int quarter(int warp) { return warp & 3; }                 // of the warp with this index in the block
  static PZ_HOST_DEVICE int first(int epilogue_warp) { return epilogue_warp / 4 * RUN; }
  // tokens of the run that starts at c, of a tile of `tokens`
  static PZ_HOST_DEVICE int count(int c, int tokens) { return tokens - c < RUN ? tokens - c : RUN; }
};

}  // namespace pz
