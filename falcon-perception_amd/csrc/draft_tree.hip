// Trees of drafted tokens: which drafts each one sees, its row behind the cached keys and its place in the text.
//
//   mask_j = mask_parent | 1 << j,  depth_j = depth_parent + 1   (a first token: 1 << j and 0)
//
// Bound by latency.  A wavefront has a sequence, a token a lane; the way to the first token is halved in every turn, so that 64 tokens
// in a row take 6 exchanges.  3 sequences of 5 tokens take 1.6 us, 64 of 24 5.4 (28 KB; the launch and two trips to memory).
#include "fp_common.h"

namespace {

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / 64;

__global__ __launch_bounds__(kThreads) void draft_tree_kernel(const int32_t* parents, const void* cached, int cached_i64, int B, int S,
                                                              int64_t* masks, int32_t* input_pos, int32_t* rope_pos) {
  const int b = blockIdx.x * kWaves + (threadIdx.x >> 6), j = threadIdx.x & 63;
  if (b >= B) return;
  const int p = j < S ? parents[static_cast<int64_t>(b) * S + j] : -2;
  const int64_t base = fp::load_index(cached, b, cached_i64);
  const bool child = p >= 0 && p < j;
  // up: the token this far towards the first one; the mask and the steps are of the way there
  int up = child ? p : j, depth = child, none = !(child || p == -1) || base < 0 || base > INT32_MAX - 64;
  uint64_t mask = 1ull << j;
#pragma unroll
  for (int turn = 0; turn < 6; ++turn) {
    mask |= __shfl(mask, up);
    depth += __shfl(depth, up);
    none |= __shfl(none, up);
    up = __shfl(up, up);
  }
  if (j >= S) return;
  const int64_t at = static_cast<int64_t>(b) * S + j;
  masks[at] = none ? 0 : static_cast<int64_t>(mask);
  input_pos[at] = none ? -1 : static_cast<int>(base) + j;
  rope_pos[at] = none ? 0 : static_cast<int>(base) + depth;
}

}  // namespace

extern "C" int fp_draft_tree(const int32_t* parents, const void* cached, int cached_index_type, int32_t B, int32_t S, int64_t* masks,
                             int32_t* input_pos, int32_t* rope_pos, void* stream) {
  if (B < 0 || S <= 0) return fp::fail(FP_ERR_INVALID_ARGUMENT, "fp_draft_tree: bad sizes (B=%d S=%d)", B, S);
  if (S > 64) return fp::fail(FP_ERR_UNSUPPORTED, "fp_draft_tree: at most 64 tokens a tree (got %d)", S);
  if (B > (1 << 26) - kWaves)  // a dispatch holds fewer than 2^32 lanes
    return fp::fail(FP_ERR_UNSUPPORTED, "fp_draft_tree: %d sequences are too many for one call", B);
  if (cached_index_type != FP_INDEX_I32 && cached_index_type != FP_INDEX_I64)
    return fp::fail(FP_ERR_INVALID_ARGUMENT, "fp_draft_tree: cached_index_type %d", cached_index_type);
  if (B == 0) return FP_OK;
  if (!parents || !cached || !masks || !input_pos || !rope_pos)
    return fp::fail(FP_ERR_INVALID_ARGUMENT, "fp_draft_tree: null pointer");
  hipLaunchKernelGGL(draft_tree_kernel, dim3((static_cast<unsigned>(B) + kWaves - 1) / kWaves), dim3(kThreads), 0,
                     static_cast<hipStream_t>(stream), parents, cached, cached_index_type, B, S, masks, input_pos, rope_pos);
  return fp::check_launch("fp_draft_tree");
}
