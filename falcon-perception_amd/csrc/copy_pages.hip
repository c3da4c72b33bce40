// Copy of the first rows of pages to other pages, in every plane of a pool.
//
//   pool[p, dst_i * P + t, :] = pool[p, src_i * P + t, :]   for t < rows_i, every plane p (layer, K or V, head)
//
// HBM-bound: every byte is read once and written once.  A workgroup copies one entry's rows of one plane, which are
// contiguous on both sides, 16 bytes a lane and 32 KB on their way at once; the stores go past the caches, which the sources of
// several forks are read from.  24 pages through 28 layers of 16 heads, D 128, bf16 (678 MB read and written): 116 us, 5.8 TB/s, where a
// large copy reaches 5.2 on this GPU; with plain stores 143, one chunk at a time 138, with non-temporal loads as well 148.
#include "fp_common.h"

namespace {

constexpr int kThreads = 256;
typedef uint32_t v4u __attribute__((ext_vector_type(4)));

struct CopyArgs {
  char* pool;
  const int64_t* src;
  const int64_t* dst;
  const int32_t* rows;
  int64_t planes, plane_bytes, page_bytes, pool_pages;
  int n, page_size, row_bytes;
};

__device__ __forceinline__ bool valid_entry(const CopyArgs& a, int64_t src, int64_t dst, int rows) {
  return src >= 0 && src < a.pool_pages && dst >= 0 && dst < a.pool_pages && rows > 0;
}

// Whether entry i is copied: its page must be nobody's source and not the destination of an entry before it, so that what
// the launch writes does not depend on the order of its workgroups.
__device__ __forceinline__ bool takes_part(const CopyArgs& a, int i, int64_t dst) {
  int clash = 0;
  for (int j = threadIdx.x; j < a.n; j += kThreads) {
    const int64_t s = a.src[j], d = a.dst[j];
    if (valid_entry(a, s, d, a.rows[j]) && (s == dst || (j < i && d == dst))) clash = 1;
  }
  return !__syncthreads_or(clash);
}

constexpr int kAhead = 8;  // chunks a thread has on their way: 32 KB a workgroup

__global__ __launch_bounds__(kThreads) void copy_pages_kernel(const CopyArgs a) {
  const int i = blockIdx.y;
  const int64_t src = a.src[i], dst = a.dst[i];
  int rows = a.rows[i];
  if (!valid_entry(a, src, dst, rows)) return;
  if (rows > a.page_size) rows = a.page_size;
  const int64_t bytes = static_cast<int64_t>(rows) * a.row_bytes;
  bool asked = false;
  for (int64_t p = blockIdx.x; p < a.planes; p += gridDim.x) {
    const char* const from = a.pool + p * a.plane_bytes + src * a.page_bytes;
    char* const to = a.pool + p * a.plane_bytes + dst * a.page_bytes;
    for (int64_t at0 = threadIdx.x * 16; at0 - threadIdx.x * 16 < bytes; at0 += kAhead * kThreads * 16) {
      v4u chunk[kAhead];
#pragma unroll
      for (int k = 0; k < kAhead; ++k) {
        const int64_t at = at0 + k * kThreads * 16;
        if (at < bytes) chunk[k] = *reinterpret_cast<const v4u*>(from + at);
      }
      if (!asked) {  // the first chunks are on their way meanwhile
        if (!takes_part(a, i, dst)) return;
        asked = true;
      }
#pragma unroll
      for (int k = 0; k < kAhead; ++k) {
        const int64_t at = at0 + k * kThreads * 16;
        if (at < bytes) __builtin_nontemporal_store(chunk[k], reinterpret_cast<v4u*>(to + at));
      }
    }
  }
}

}  // namespace

extern "C" int fp_copy_pages(void* pool, const int64_t* src, const int64_t* dst, const int32_t* rows, int32_t n,
                             int64_t n_planes, int64_t n_slots, int32_t D, int32_t page_size, int dtype, void* stream) {
  const int e = fp::elem_bytes(dtype);
  if (e == 0) return fp::fail(FP_ERR_UNSUPPORTED, "fp_copy_pages: dtype code %d", dtype);
  if (n < 0 || n_planes < 0 || n_slots < 0 || page_size <= 0 || D <= 0 || (D * e) % 16 != 0)
    return fp::fail(FP_ERR_INVALID_ARGUMENT, "fp_copy_pages: bad sizes (n=%d planes=%lld n_slots=%lld D=%d page_size=%d)", n,
                    static_cast<long long>(n_planes), static_cast<long long>(n_slots), D, page_size);
  if (n > 65535) return fp::fail(FP_ERR_UNSUPPORTED, "fp_copy_pages: at most 65535 pages a call (got %d)", n);
  if (n == 0 || n_planes == 0 || n_slots == 0) return FP_OK;
  if (!pool || !src || !dst || !rows) return fp::fail(FP_ERR_INVALID_ARGUMENT, "fp_copy_pages: null pointer");
  if (!fp::aligned(pool, 16)) return fp::fail(FP_ERR_INVALID_ARGUMENT, "fp_copy_pages: the pool must be 16-byte aligned");
  const int64_t row_bytes = static_cast<int64_t>(D) * e;
  const CopyArgs a{static_cast<char*>(pool), src, dst, rows, n_planes, n_slots * row_bytes, page_size * row_bytes,
                   n_slots / page_size, n, page_size, static_cast<int>(row_bytes)};
  const int64_t x = n_planes < 65535 ? n_planes : 65535;
  hipLaunchKernelGGL(copy_pages_kernel, dim3(static_cast<unsigned>(x), static_cast<unsigned>(n)), dim3(kThreads), 0,
                     static_cast<hipStream_t>(stream), a);
  return fp::check_launch("fp_copy_pages");
}
