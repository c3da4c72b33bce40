// Attention of a batch's newest tokens over the paged cache, where sequences of the batch begin with the same keys.
//
//   out[b, h, j] = sum over t <= p of softmax_t(scale q.k_t) v_t,   p = input_pos[b, j]
#include "fp_common.h"

#include <math.h>

namespace {

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / 64;
constexpr int kMaxSequences = 4096;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

struct SharedArgs {
  const char* q;
  int64_t qs_b, qs_h, qs_s;  // bytes
  const char* pool_k;
  const char* pool_v;
  const int64_t* page_table;
  int64_t pt_row_stride;
  const int64_t* batch_idx;
  const void* input_pos;
  int pos_i64;
  char* out;
  int64_t os_b, os_h, os_s;  // bytes
  float* lse;
  const float* sinks;
  int B, S, Hq, Hc;
  fp::PageDiv pd;
  int n_pages, max_batch, pool_pages;
  int64_t n_slots;
  int max_context;
  float qscale;  // scale * log2(e)
};

template <typename T>
__device__ __forceinline__ float wave_sum(T x) {
#pragma unroll
  for (int off = 32; off; off >>= 1) x += __shfl_xor(x, off);
  return x;
}

template <typename E, int D>
__global__ __launch_bounds__(kThreads) void shared_decode_simple(const SharedArgs a) {
  constexpr int V = D / 64;
  __shared__ float s_acc[kWaves][D], s_ml[kWaves][2];
  const int hq = blockIdx.x, b = blockIdx.y / a.S, s = blockIdx.y % a.S, hc = hq / (a.Hq / a.Hc);
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const int64_t trow = a.batch_idx[b];
  int64_t L = fp::load_index(a.input_pos, static_cast<int64_t>(b) * a.S + s, a.pos_i64);
  L = L < 0 || trow < 0 || trow >= a.max_batch ? 0 : L >= a.max_context ? a.max_context : L + 1;
  const E* q = reinterpret_cast<const E*>(a.q + b * a.qs_b + hq * a.qs_h + s * a.qs_s) + lane * V;
  float qv[V], acc[V], m = -INFINITY, l = 0.f;
  for (int i = 0; i < V; ++i) qv[i] = static_cast<float>(q[i]), acc[i] = 0.f;
  for (int64_t t = wave; t < L; t += kWaves) {
    int64_t blk;
    int off;
    a.pd.split(t, blk, off);
    int64_t page = blk < a.n_pages ? a.page_table[trow * a.pt_row_stride + blk] : 0;
    if (page < 0 || page >= a.pool_pages) page = 0;
    const int64_t row = (static_cast<int64_t>(hc) * a.n_slots + page * a.pd.page_size + off) * D + lane * V;
    float x = 0.f;
    for (int i = 0; i < V; ++i) x += qv[i] * static_cast<float>(reinterpret_cast<const E*>(a.pool_k)[row + i]);
    x = wave_sum(x) * a.qscale;
    const float mn = fmaxf(m, x), ms = mn == -INFINITY ? 0.f : mn;
    const float keep = exp2f(m - ms), p = exp2f(x - ms);
    l = l * keep + p;
    for (int i = 0; i < V; ++i) acc[i] = acc[i] * keep + p * static_cast<float>(reinterpret_cast<const E*>(a.pool_v)[row + i]);
    m = mn;
  }
  for (int i = 0; i < V; ++i) s_acc[wave][lane * V + i] = acc[i];
  if (lane == 0) s_ml[wave][0] = m, s_ml[wave][1] = l;
  __syncthreads();
  float mn = -INFINITY, den = 0.f;
  for (int w = 0; w < kWaves; ++w) mn = fmaxf(mn, s_ml[w][0]);
  const float ms = mn == -INFINITY ? 0.f : mn;
  for (int w = 0; w < kWaves; ++w) den += s_ml[w][1] * exp2f(s_ml[w][0] - ms);
  const float lse = (mn + log2f(den)) * kLn2;
  for (int d = threadIdx.x; d < D; d += kThreads) {
    float num = 0.f;
    for (int w = 0; w < kWaves; ++w) num += s_acc[w][d] * exp2f(s_ml[w][0] - ms);
    float o = L == 0 ? 0.f : num / den;
    if (a.sinks && L > 0) o = static_cast<float>(static_cast<E>(o)) / (1.f + expf(a.sinks[hq] - lse));
    reinterpret_cast<E*>(a.out + b * a.os_b + hq * a.os_h + s * a.os_s)[d] = static_cast<E>(o);
  }
  if (threadIdx.x == 0) a.lse[(static_cast<int64_t>(b) * a.Hq + hq) * a.S + s] = L == 0 ? -INFINITY : lse;
}

int check_shape(const char* what, int B, int S, int Hq, int Hc, int D) {
  if (B < 0 || S <= 0 || Hq <= 0 || Hc <= 0 || Hq % Hc != 0)
    return fp::fail(FP_ERR_INVALID_ARGUMENT, "%s: bad sizes (B=%d S=%d Hq=%d Hc=%d)", what, B, S, Hq, Hc);
  const int G = Hq / Hc;
  if (D != 64 && D != 128) return fp::fail(FP_ERR_UNSUPPORTED, "%s: head_dim %d (64 or 128)", what, D);
  if (G != 1 && G != 2 && G != 4 && G != 8)
    return fp::fail(FP_ERR_UNSUPPORTED, "%s: %d query heads per cache head (1, 2, 4 or 8)", what, G);
  if (B > kMaxSequences || S > 1024)
    return fp::fail(FP_ERR_UNSUPPORTED, "%s: at most %d sequences of 1024 tokens (got %d of %d)", what, kMaxSequences, B, S);
  return FP_OK;
}

}  // namespace

extern "C" int64_t fp_shared_decode_plan_bytes(int32_t B, int32_t S, int32_t Hq, int32_t Hc, int32_t D) {
  if (const int rc = check_shape("fp_shared_decode_plan_bytes", B, S, Hq, Hc, D)) return rc;
  return 64;
}

extern "C" int64_t fp_shared_decode_workspace_bytes(int32_t B, int32_t S, int32_t Hq, int32_t Hc, int32_t D) {
  if (const int rc = check_shape("fp_shared_decode_workspace_bytes", B, S, Hq, Hc, D)) return rc;
  return 64;
}

extern "C" int fp_shared_decode_plan(const int64_t* batch_idx, const void* input_pos, int pos_index_type,
                                     const int32_t* prefix_ids, const int32_t* prefix_lens, int32_t B, int32_t S, int32_t Hq,
                                     int32_t Hc, int32_t D, int32_t max_batch, int32_t max_context, void* plan,
                                     int64_t plan_bytes, void* stream) {
  const char* const what = "fp_shared_decode_plan";
  if (const int rc = check_shape(what, B, S, Hq, Hc, D)) return rc;
  if (max_batch <= 0 || max_context <= 0)
    return fp::fail(FP_ERR_INVALID_ARGUMENT, "%s: max_batch %d, max_context %d", what, max_batch, max_context);
  if (pos_index_type != FP_INDEX_I32 && pos_index_type != FP_INDEX_I64)
    return fp::fail(FP_ERR_INVALID_ARGUMENT, "%s: pos_index_type %d", what, pos_index_type);
  if (B == 0) return FP_OK;
  if (!batch_idx || !input_pos || !prefix_ids || !prefix_lens || !plan)
    return fp::fail(FP_ERR_INVALID_ARGUMENT, "%s: null pointer", what);
  if (plan_bytes < fp_shared_decode_plan_bytes(B, S, Hq, Hc, D) || !fp::aligned(plan, 16))
    return fp::fail(FP_ERR_WORKSPACE, "%s: the plan needs %lld bytes, 16-byte aligned (got %lld)", what,
                    static_cast<long long>(fp_shared_decode_plan_bytes(B, S, Hq, Hc, D)), static_cast<long long>(plan_bytes));
  (void)stream;
  return FP_OK;
}

extern "C" int fp_paged_decode_shared(const void* q, int64_t q_stride_b, int64_t q_stride_h, int64_t q_stride_s,
                                      const void* pool_k, const void* pool_v, const int64_t* page_table,
                                      int64_t pt_row_stride, const int64_t* batch_idx, const void* input_pos,
                                      int pos_index_type, void* out, int64_t out_stride_b, int64_t out_stride_h,
                                      int64_t out_stride_s, float* lse, const float* sinks, void* workspace,
                                      int64_t workspace_bytes, const void* plan, int64_t plan_bytes, int32_t B, int32_t S,
                                      int32_t Hq, int32_t Hc, int32_t D, int32_t page_size, int32_t n_pages,
                                      int32_t max_batch, int64_t n_slots, int32_t max_context, float scale, int dtype,
                                      void* stream) {
  const char* const what = "fp_paged_decode_shared";
  if (const int rc = check_shape(what, B, S, Hq, Hc, D)) return rc;
  const int e = fp::elem_bytes(dtype);
  if (e == 0) return fp::fail(FP_ERR_UNSUPPORTED, "%s: dtype code %d", what, dtype);
  if (page_size <= 0 || n_pages <= 0 || max_batch <= 0 || max_context <= 0 || n_slots <= 0 || n_slots / page_size < 1 ||
      n_slots / page_size > INT32_MAX)
    return fp::fail(FP_ERR_INVALID_ARGUMENT, "%s: bad sizes (page_size=%d n_pages=%d max_batch=%d n_slots=%lld max_context=%d)",
                    what, page_size, n_pages, max_batch, static_cast<long long>(n_slots), max_context);
  if (pos_index_type != FP_INDEX_I32 && pos_index_type != FP_INDEX_I64)
    return fp::fail(FP_ERR_INVALID_ARGUMENT, "%s: pos_index_type %d", what, pos_index_type);
  if (B == 0) return FP_OK;
  if (!q || !pool_k || !pool_v || !page_table || !batch_idx || !input_pos || !out || !lse || !plan)
    return fp::fail(FP_ERR_INVALID_ARGUMENT, "%s: null pointer", what);
  if (!fp::aligned(q, 16) || !fp::aligned(pool_k, 16) || !fp::aligned(pool_v, 16) || !fp::aligned(out, 16) ||
      q_stride_b * e % 16 || q_stride_h * e % 16 || q_stride_s * e % 16 || out_stride_b * e % 16 || out_stride_h * e % 16 ||
      out_stride_s * e % 16)
    return fp::fail(FP_ERR_INVALID_ARGUMENT, "%s: rows of q, out and the pools must be 16-byte aligned", what);
  if (plan_bytes < fp_shared_decode_plan_bytes(B, S, Hq, Hc, D))
    return fp::fail(FP_ERR_WORKSPACE, "%s: plan of %lld bytes is too small", what, static_cast<long long>(plan_bytes));
  const int64_t need = fp_shared_decode_workspace_bytes(B, S, Hq, Hc, D);
  if (!workspace || workspace_bytes < need || !fp::aligned(workspace, 16))
    return fp::fail(FP_ERR_WORKSPACE, "%s: workspace of %lld bytes, 16-byte aligned, is needed (got %lld)", what,
                    static_cast<long long>(need), static_cast<long long>(workspace_bytes));
  const SharedArgs a{static_cast<const char*>(q), q_stride_b * e, q_stride_h * e, q_stride_s * e,
                     static_cast<const char*>(pool_k), static_cast<const char*>(pool_v), page_table, pt_row_stride, batch_idx,
                     input_pos, pos_index_type, static_cast<char*>(out), out_stride_b * e, out_stride_h * e, out_stride_s * e,
                     lse, sinks, B, S, Hq, Hc, fp::PageDiv(page_size), n_pages, max_batch,
                     static_cast<int>(n_slots / page_size), n_slots, max_context, scale * kLog2e};
  const dim3 grid(Hq, B * S), block(kThreads);
  const hipStream_t st = static_cast<hipStream_t>(stream);
  const auto go = [&](auto element) {
    using E = decltype(element);
    if (D == 64)
      hipLaunchKernelGGL((shared_decode_simple<E, 64>), grid, block, 0, st, a);
    else
      hipLaunchKernelGGL((shared_decode_simple<E, 128>), grid, block, 0, st, a);
  };
  if (dtype == FP_DTYPE_F32)
    go(float{});
  else if (dtype == FP_DTYPE_BF16)
    go(__bf16{});
  else
    go(_Float16{});
  return fp::check_launch(what);
}
