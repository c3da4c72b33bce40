// The cached rows of the drafts that stand, moved together behind the cached keys in every plane of the pool.
//
//   pool[p, slot(cached_b + i), :] = pool[p, slot(cached_b + path_i), :]   for i < n_b, every plane p (layer, K or V, head)
//
// A path rises, so path_i >= i: a row is written over only where it is read for an earlier place.  A plane's rows are therefore all read
// before the first is written: by one wavefront, which has several planes' rows on their way at once and waits for no other.
//
// The bytes bound it, read and written once: 65 MB (64 sequences, 1 to 7 rows kept of up to 32, 28 layers of 16 heads of 256 bytes) in 14.9 us,
// 4.4 TB/s, of which 3 us pass before the first row's address is known (slot, count, path, page: each in the one before); the smallest
// calls take 3.8 us.  With a workgroup to a plane's rows, a division for every chunk and stores that stay in L2 it was 19.3 us; with 8 chunks
// a lane instead of 4 (half the wavefronts) 19.2; with ordinary stores 16.0 (and 2 us more until the next kernel begins).
#include "fp_common.h"

namespace {

constexpr int kThreads = 256, kWaves = kThreads / 64;
constexpr int kMaxPath = 64;
constexpr int kAhead = 4;  // chunks a lane has on their way
typedef uint32_t v4u __attribute__((ext_vector_type(4)));

struct KeepArgs {
  char* pool;
  const int64_t* page_table;
  int64_t pt_row_stride;
  const int64_t* batch_idx;
  const void* cached;
  int cached_i64;
  const int32_t* path;
  int64_t planes, plane_bytes, n_slots;
  int B, S, n_pages, max_batch, pool_pages;
  int chunks;  // 16-byte chunks of a row
  uint32_t per_row;
  fp::PageDiv pd;
};

// Row of the planes that holds the sequence's token t, -1: none.
__device__ __forceinline__ int64_t slot_of(const KeepArgs& a, int64_t row, int64_t t) {
  int64_t blk;
  int off;
  a.pd.split(t, blk, off);
  if (blk >= a.n_pages) return -1;
  const int64_t page = a.page_table[row * a.pt_row_stride + blk];
  return page < 0 || page >= a.pool_pages ? -1 : page * a.pd.page_size + off;
}

// i / d for i below 2^16 and d above 1, from m = 2^32 / d rounded up.
__device__ __forceinline__ int over(int i, uint32_t m) { return static_cast<int>(__umulhi(static_cast<uint32_t>(i), m)); }

__global__ __launch_bounds__(kThreads) void keep_rows_kernel(const KeepArgs a) {
  __shared__ int64_t s_from[kMaxPath], s_to[kMaxPath];  // byte offsets in a plane
  __shared__ int s_n;
  const int b = blockIdx.y, tid = threadIdx.x;
  const int64_t row = a.batch_idx[b];
  const int64_t base = fp::load_index(a.cached, b, a.cached_i64);
  if (row < 0 || row >= a.max_batch || base < 0 || base > INT32_MAX) return;
  // a slot that an entry before this one names is left to that one
  int twice = 0;
  for (int i = tid; i < b; i += kThreads) twice |= a.batch_idx[i] == row;
  if (tid < 64) {
    const int p = tid < a.S ? a.path[static_cast<int64_t>(b) * a.S + tid] : -1;
    const int before = __shfl_up(p, 1);
    const bool good = p >= 0 && p < a.S && (tid == 0 || p > before);
    const uint64_t bad = ~__ballot(good);
    const int n = bad ? __builtin_ctzll(bad) : 64;
    const int64_t from = tid < n && p > tid ? slot_of(a, row, base + p) : -1, to = from >= 0 ? slot_of(a, row, base + tid) : -1;
    const uint64_t moved = __ballot(to >= 0);
    if (to >= 0) {
      const int at = __builtin_popcountll(moved & ((1ull << tid) - 1));
      s_from[at] = from * a.chunks * 16;
      s_to[at] = to * a.chunks * 16;
    }
    if (tid == 0) s_n = __builtin_popcountll(moved);
  }
  if (__syncthreads_or(twice)) return;
  const int n = s_n;
  if (n == 0) return;
  // A wavefront takes the rows of some planes at once, or those of one plane in turns in the order of the path: what one turn writes is
  // read by no turn after it.
  const int lane = tid & 63, wave = tid >> 6;
  const int room = 64 * kAhead;  // chunks
  const int rows = min(n, room / a.chunks), items = rows * a.chunks, at_once = rows < n ? 1 : room / items;
  const uint32_t per_plane = 0xffffffffu / static_cast<uint32_t>(items) + 1;
  const int64_t n_waves = static_cast<int64_t>(gridDim.x) * kWaves;
  for (int64_t plane0 = (static_cast<int64_t>(blockIdx.x) * kWaves + wave) * at_once; plane0 < a.planes; plane0 += n_waves * at_once) {
    char* const base_of = a.pool + plane0 * a.plane_bytes;
    const int here = static_cast<int>(min<int64_t>(a.planes - plane0, at_once)) * items;
    for (int r0 = 0; r0 < n; r0 += rows) {
      v4u chunk[kAhead];
      char* to[kAhead];
#pragma unroll
      for (int k = 0; k < kAhead; ++k) {
        const int i = lane + k * 64;
        const int plane = items == 1 ? i : over(i, per_plane), rest = i - plane * items;
        const int turn = a.chunks == 1 ? rest : over(rest, a.per_row), c = rest - turn * a.chunks, r = r0 + turn;
        to[k] = nullptr;
        if (i < here && r < n) {
          char* const at = base_of + plane * a.plane_bytes + c * 16;
          chunk[k] = *reinterpret_cast<const v4u*>(at + s_from[r]);
          to[k] = at + s_to[r];
        }
      }
      asm volatile("s_waitcnt vmcnt(0)" : : : "memory");  // every row has been read
#pragma unroll
      for (int k = 0; k < kAhead; ++k)
        if (to[k]) __builtin_nontemporal_store(chunk[k], reinterpret_cast<v4u*>(to[k]));
    }
  }
}

}  // namespace

extern "C" int fp_keep_rows(void* pool, const int64_t* page_table, int64_t pt_row_stride, const int64_t* batch_idx, const void* cached,
                            int cached_index_type, const int32_t* path, int32_t B, int32_t S, int64_t n_planes, int64_t n_slots,
                            int32_t D, int32_t page_size, int32_t n_pages, int32_t max_batch, int dtype, void* stream) {
  const char* const what = "fp_keep_rows";
  const int e = fp::elem_bytes(dtype);
  if (e == 0) return fp::fail(FP_ERR_UNSUPPORTED, "%s: dtype code %d", what, dtype);
  if (B < 0 || S <= 0 || n_planes < 0 || n_slots < 0 || page_size <= 0 || n_pages <= 0 || max_batch <= 0 || D <= 0 || (D * static_cast<int64_t>(e)) % 16 != 0)
    return fp::fail(FP_ERR_INVALID_ARGUMENT, "%s: bad sizes (B=%d S=%d planes=%lld n_slots=%lld D=%d page_size=%d n_pages=%d max_batch=%d)",
                    what, B, S, static_cast<long long>(n_planes), static_cast<long long>(n_slots), D, page_size, n_pages, max_batch);
  if (S > kMaxPath || B > 65535 || D * static_cast<int64_t>(e) > kThreads * 16)
    return fp::fail(FP_ERR_UNSUPPORTED, "%s: at most 65535 sequences, %d rows of each and %d bytes a row (got %d, %d, %lld)", what, kMaxPath,
                    kThreads * 16, B, S, static_cast<long long>(D) * e);
  if (cached_index_type != FP_INDEX_I32 && cached_index_type != FP_INDEX_I64)
    return fp::fail(FP_ERR_INVALID_ARGUMENT, "%s: cached_index_type %d", what, cached_index_type);
  if (n_slots / page_size > INT32_MAX) return fp::fail(FP_ERR_UNSUPPORTED, "%s: n_slots=%lld", what, static_cast<long long>(n_slots));
  if (B == 0 || n_planes == 0 || n_slots == 0) return FP_OK;
  if (!pool || !page_table || !batch_idx || !cached || !path) return fp::fail(FP_ERR_INVALID_ARGUMENT, "%s: null pointer", what);
  if (!fp::aligned(pool, 16)) return fp::fail(FP_ERR_INVALID_ARGUMENT, "%s: the pool must be 16-byte aligned", what);
  const int64_t row_bytes = static_cast<int64_t>(D) * e;
  const KeepArgs a{static_cast<char*>(pool), page_table, pt_row_stride, batch_idx, cached, cached_index_type, path, n_planes,
                   n_slots * row_bytes, n_slots, B, S, n_pages, max_batch, static_cast<int>(n_slots / page_size),
                   static_cast<int>(row_bytes / 16), 0xffffffffu / static_cast<uint32_t>(row_bytes / 16) + 1, fp::PageDiv(page_size)};
  int64_t x = (16ll * fp::compute_units() + B - 1) / B;
  if (x > (n_planes + kWaves - 1) / kWaves) x = (n_planes + kWaves - 1) / kWaves;
  hipLaunchKernelGGL(keep_rows_kernel, dim3(static_cast<unsigned>(x), static_cast<unsigned>(B)), dim3(kThreads), 0,
                     static_cast<hipStream_t>(stream), a);
  return fp::check_launch(what);
}
