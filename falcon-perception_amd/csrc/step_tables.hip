// Page tables, packed rows and slot map of a step, from the lengths of its requests.
//
// Replaces the host loop over PagedKVCache.reserve (paged_attention.py:115-164), one upload and two index writes a
// request, and the host lists of batch_idx / input_pos of a packed prefill step (paged_inference.py:637-672).
//   have_b = ceil(old_b / P), of a fork floor(old_b / P);  need_b = ceil(new_b / P) - have_b, at least 0
//   off_b, start_b = sums over the requests before b of need and of the rows new - old, padded to row_multiple
//   table[slot_b, have_b + i] = free[count - off_b - need_b + i]   (the pages that reserve, called in turn, pops)
//   row start_b + j -> (slot_b, old_b + j, page * P + position % P)
//
// Bound by latency for a decode step (one launch: load, scan, store) and by the stores of the rows (20 bytes each) for an
// admission step.  One launch: every workgroup works out the sums of all requests by itself - 16 to 32 bytes a request, from L2 -
// instead of waiting for a launch that does; nothing that one workgroup writes is read by another.  64 requests of one token: 6.0 us;
// 48 forks, 16 thousand rows: 7.0; 1000 requests, 2 million rows, 41 MB: 20.2, about 8
// of them before the first row.
#include "fp_common.h"

namespace {

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / 64;
constexpr int kMaxRequests = 4096;
constexpr int kMaxSlots = 1 << 17;
constexpr int64_t kLdsBytes = 160 * 1024;  // of a CU
typedef int64_t v2l __attribute__((ext_vector_type(2)));
typedef int v4i __attribute__((ext_vector_type(4)));

struct TablesArgs {
  const int64_t* slots;
  const void* old_lens;
  const void* new_lens;
  int lens_i64;
  const int64_t* parents;  // optional
  const int64_t* free_pages;
  const int32_t* free_count;
  int64_t* page_table;
  int64_t pt_row_stride;
  int64_t* inverse;  // optional
  int64_t inv_row_stride, inv_cols;
  int64_t* batch_idx;
  int32_t* input_pos;
  int64_t* slot_map;
  int32_t* row_starts;
  int32_t* free_left;
  int64_t* copy_src;
  int64_t* copy_dst;
  int32_t* copy_rows;
  int32_t* status;
  int B, max_rows, row_multiple, columns, max_batch, n_free;
  int wide;  // the rows' arrays are 16-byte aligned
  fp::PageDiv pd;
};

// What the rows of a request need of it, in LDS.
struct Record {
  int slot, old_len, new_len, have;
};

struct Request {
  int64_t slot, parent;
  int64_t old_len, new_len;
  int64_t have, blocks;
  int tail;  // tokens of a fork's prefix behind its whole pages
  __device__ int64_t need() const { return blocks > have ? blocks - have : 0; }
};

__device__ __forceinline__ Request load_request(const TablesArgs& a, int b) {
  Request r;
  r.slot = a.slots[b];
  r.parent = a.parents ? a.parents[b] : 0;
  r.old_len = fp::load_index(a.old_lens, b, a.lens_i64);
  r.new_len = fp::load_index(a.new_lens, b, a.lens_i64);
  int64_t blk, end;
  int off, rest;
  a.pd.split(r.old_len < 0 ? 0 : r.old_len, blk, off);
  a.pd.split(r.new_len < 0 ? 0 : r.new_len, end, rest);
  r.have = blk + (r.parent <= 0 && off > 0);
  r.blocks = end + (rest > 0);
  r.tail = r.parent > 0 ? off : 0;
  return r;
}

__device__ __forceinline__ int64_t padded_rows(const TablesArgs& a, const Request& r) {
  const int64_t n = r.new_len - r.old_len;
  if (a.row_multiple == 1) return n;
  return (n + a.row_multiple - 1) / a.row_multiple * a.row_multiple;
}

__device__ __forceinline__ int64_t pages_of_request(const TablesArgs& a, const Record& r) {
  int64_t end;
  int rest;
  a.pd.split(r.new_len, end, rest);
  end += rest > 0;
  return end > r.have ? end - r.have : 0;
}

// page of block c of a request: its own row, its parent's or the free list, none of which this launch writes there
__device__ __forceinline__ int64_t page_of(const TablesArgs& a, const Request& r, int64_t c, int64_t first_free) {
  if (c >= r.have) return a.free_pages[first_free + c - r.have];
  return a.page_table[(r.parent > 0 ? r.parent : r.slot) * a.pt_row_stride + c];
}

template <int kRows>  // neighbours that a thread has
__global__ __launch_bounds__(kThreads) void step_tables_kernel(const TablesArgs a) {
  extern __shared__ __attribute__((aligned(16))) int s_mem[];
  int* const s_start = s_mem;                      // [B + 1] first row of every request
  int* const s_free = s_mem + a.B + 1;             // [B] pages taken by the requests before
  uint32_t* const s_named = reinterpret_cast<uint32_t*>(s_free + a.B);  // bit per slot: named by a request
  Record* const s_rec = reinterpret_cast<Record*>(s_mem + (2 * a.B + 1 + (a.max_batch + 31) / 32 + 3) / 4 * 4);
  const int words = (a.max_batch + 31) / 32;
  __shared__ int64_t s_sum[kWaves][2];
  __shared__ int s_bad;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  for (int i = tid; i < words; i += kThreads) s_named[i] = 0;
  if (tid == 0) s_bad = 0;
  __syncthreads();

  // sums: consecutive requests a thread, then over the lanes and the wavefronts.  64 bits: lengths that do not fit are refused below
  const int per = (a.B + kThreads - 1) / kThreads;
  const int b0 = tid * per, b1 = min(a.B, b0 + per);
  const int64_t count = *a.free_count;
  int64_t rows = 0, pages = 0;
  int bad = count < 0 || count > a.n_free ? 8 : 0;
  for (int b4 = b0; b4 < b1; b4 += 4) {
    Request four[4];  // on their way together
#pragma unroll
    for (int k = 0; k < 4; ++k) four[k] = load_request(a, min(b4 + k, b1 - 1));
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int b = b4 + k;
      if (b >= b1) break;
      const Request& r = four[k];
      if (r.slot <= 0 || r.slot >= a.max_batch || r.parent >= a.max_batch || r.old_len < 0 || r.new_len < r.old_len ||
          r.new_len > INT32_MAX) {
        bad |= 8;
        continue;
      }
      const uint32_t bit = 1u << (r.slot & 31);
      if (atomicOr(&s_named[r.slot >> 5], bit) & bit) bad |= 8;  // a slot that two requests name
      if (r.blocks > a.columns) bad |= 2;
      const int64_t n = padded_rows(a, r);
      if (n > a.max_rows) bad |= 4;
      rows += n;
      pages += r.need();
      s_start[b] = static_cast<int>(n);  // its own rows and pages for now, below those of the requests before it
      s_free[b] = static_cast<int>(r.need());
      s_rec[b] = Record{static_cast<int>(r.slot), static_cast<int>(r.old_len), static_cast<int>(r.new_len), static_cast<int>(r.have)};
    }
  }
  int64_t rows_upto = rows, pages_upto = pages;
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) {
    const int64_t x = __shfl_up(rows_upto, off), y = __shfl_up(pages_upto, off);
    if (lane >= off) rows_upto += x, pages_upto += y;
  }
  if (lane == 63) s_sum[wave][0] = rows_upto, s_sum[wave][1] = pages_upto;
  __syncthreads();
  int64_t rows_all = 0, pages_all = 0;
  rows_upto -= rows, pages_upto -= pages;
#pragma unroll
  for (int w = 0; w < kWaves; ++w) {
    if (w < wave) rows_upto += s_sum[w][0], pages_upto += s_sum[w][1];
    rows_all += s_sum[w][0], pages_all += s_sum[w][1];
  }
  if (rows_all > a.max_rows) bad |= 4;
  if (pages_all > count) bad |= 1;
  if (!bad) {  // else nothing is done
    for (int b = b0; b < b1; ++b) {
      const int64_t parent = a.parents ? a.parents[b] : 0;
      if (parent > 0 && s_named[parent >> 5] >> (parent & 31) & 1) bad |= 8;
      const int n = s_start[b], need = s_free[b];
      s_start[b] = static_cast<int>(rows_upto);
      s_free[b] = static_cast<int>(pages_upto);
      rows_upto += n;
      pages_upto += need;
    }
  }
  if (bad) atomicOr(&s_bad, bad);
  if (tid == 0) s_start[a.B] = static_cast<int>(rows_all);
  __syncthreads();
  bad = s_bad;
  const int n_rows = bad ? 0 : static_cast<int>(rows_all);

  if (blockIdx.x == 0) {
    for (int b = tid; b <= a.B; b += kThreads) a.row_starts[b] = bad ? 0 : s_start[b];
    if (tid == 0) {
      *a.status = bad;
      *a.free_left = static_cast<int>(count - (bad ? 0 : pages_all));
    }
  }

  // rows of the table: a wavefront a request
  for (int b = blockIdx.x * kWaves + wave; b < a.B; b += gridDim.x * kWaves) {
    int64_t src = -1, dst = -1;
    int n_copy = 0;
    if (!bad) {
      const Request r = load_request(a, b);
      const int64_t first = count - s_free[b] - r.need();
      const bool fork = r.parent > 0;
      for (int64_t c = (fork ? 0 : r.have) + lane; c < r.blocks; c += 64) {
        const int64_t page = page_of(a, r, c, first);
        a.page_table[r.slot * a.pt_row_stride + c] = page;
        if (a.inverse && page >= 0 && page < a.inv_cols) a.inverse[r.slot * a.inv_row_stride + page] = c;
      }
      if (r.tail > 0) {
        src = a.page_table[r.parent * a.pt_row_stride + r.have];
        dst = a.free_pages[first];
        n_copy = r.tail;
      }
    }
    if (lane == 0) {
      a.copy_src[b] = src;
      a.copy_dst[b] = dst;
      a.copy_rows[b] = n_copy;
    }
  }

  // packed rows
  const int64_t stride = static_cast<int64_t>(gridDim.x) * kThreads * kRows;
  for (int64_t row0 = (static_cast<int64_t>(blockIdx.x) * kThreads + tid) * kRows; row0 < a.max_rows; row0 += stride) {
    int64_t slot[kRows] = {}, where[kRows] = {};
    int pos[kRows] = {};
    if (row0 < n_rows) {
      int lo = 0, hi = a.B - 1;  // the last request that starts at or before the row
      while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (s_start[mid] <= row0) lo = mid; else hi = mid - 1;
      }
      Record r = s_rec[lo];
      int64_t blk_now = -1, page = 0;
#pragma unroll
      for (int k = 0; k < kRows; ++k) {
        const int64_t row = row0 + k;
        if (row >= n_rows) break;
        if (row >= s_start[lo + 1]) {
          do ++lo; while (row >= s_start[lo + 1]);
          r = s_rec[lo];
          blk_now = -1;
        }
        const int64_t p = r.old_len + (row - s_start[lo]);
        if (p >= r.new_len) continue;
        int64_t blk;
        int off;
        a.pd.split(p, blk, off);
        if (blk != blk_now) {
          blk_now = blk;
          // behind the blocks it has, the free list; else its own row, which this launch does not write there (a fork's rows begin
          // behind its shared blocks)
          const int64_t need = pages_of_request(a, r);
          page = (blk >= r.have ? a.free_pages[count - s_free[lo] - need + blk - r.have]
                                : a.page_table[r.slot * a.pt_row_stride + blk]) * a.pd.page_size;
        }
        slot[k] = r.slot;
        pos[k] = static_cast<int>(p);
        where[k] = page + off;
      }
    }
    bool stored = false;
    if constexpr (kRows == 4) {
      if (a.wide && row0 + 4 <= a.max_rows) {
        v2l* const to_slot = reinterpret_cast<v2l*>(a.batch_idx + row0);
        v2l* const to_where = reinterpret_cast<v2l*>(a.slot_map + row0);
        __builtin_nontemporal_store(v2l{slot[0], slot[1]}, to_slot);
        __builtin_nontemporal_store(v2l{slot[2], slot[3]}, to_slot + 1);
        __builtin_nontemporal_store(v2l{where[0], where[1]}, to_where);
        __builtin_nontemporal_store(v2l{where[2], where[3]}, to_where + 1);
        __builtin_nontemporal_store(v4i{pos[0], pos[1], pos[2], pos[3]}, reinterpret_cast<v4i*>(a.input_pos + row0));
        stored = true;
      }
    }
    if (!stored) {
#pragma unroll
      for (int k = 0; k < kRows; ++k) {
        if (row0 + k >= a.max_rows) break;
        a.batch_idx[row0 + k] = slot[k];
        a.input_pos[row0 + k] = pos[k];
        a.slot_map[row0 + k] = where[k];
      }
    }
  }
}

}  // namespace

extern "C" int fp_step_tables(const int64_t* slots, const void* old_lens, const void* new_lens, int len_index_type,
                              const int64_t* parents, const int64_t* free_pages, const int32_t* free_count, int32_t n_free,
                              int64_t* page_table, int64_t pt_row_stride, int64_t* inverse, int64_t inv_row_stride,
                              int64_t inv_cols, int64_t* batch_idx, int32_t* input_pos, int64_t* slot_map,
                              int32_t* row_starts, int32_t* free_left, int64_t* copy_src, int64_t* copy_dst,
                              int32_t* copy_rows, int32_t* status, int32_t B, int32_t max_rows, int32_t row_multiple,
                              int32_t page_size, int32_t n_pages, int32_t max_batch, void* stream) {
  if (B < 0 || max_rows < 0 || row_multiple <= 0 || page_size <= 0 || n_pages <= 0 || max_batch <= 0 || n_free < 0)
    return fp::fail(FP_ERR_INVALID_ARGUMENT, "fp_step_tables: bad sizes (B=%d max_rows=%d row_multiple=%d page_size=%d "
                    "n_pages=%d max_batch=%d n_free=%d)", B, max_rows, row_multiple, page_size, n_pages, max_batch, n_free);
  if (len_index_type != FP_INDEX_I32 && len_index_type != FP_INDEX_I64)
    return fp::fail(FP_ERR_INVALID_ARGUMENT, "fp_step_tables: len_index_type %d", len_index_type);
  if (B > kMaxRequests || max_batch > kMaxSlots)
    return fp::fail(FP_ERR_UNSUPPORTED, "fp_step_tables: at most %d requests and %d slots (got %d and %d)", kMaxRequests,
                    kMaxSlots, B, max_batch);
  if (!free_count || !free_left || !status || !row_starts || (n_free > 0 && !free_pages) || !page_table ||
      (B > 0 && (!slots || !old_lens || !new_lens || !copy_src || !copy_dst || !copy_rows)) ||
      (max_rows > 0 && (!batch_idx || !input_pos || !slot_map)))
    return fp::fail(FP_ERR_INVALID_ARGUMENT, "fp_step_tables: null pointer");
  if (free_left == free_count)
    return fp::fail(FP_ERR_INVALID_ARGUMENT, "fp_step_tables: free_left may not be free_count: every workgroup reads that one");
  const TablesArgs a{slots, old_lens, new_lens, len_index_type, parents, free_pages, free_count, page_table, pt_row_stride,
                     inverse, inv_row_stride, inv_cols, batch_idx, input_pos, slot_map, row_starts, free_left, copy_src,
                     copy_dst, copy_rows, status, B, max_rows, row_multiple, n_pages, max_batch, n_free,
                     fp::aligned(batch_idx, 16) && fp::aligned(input_pos, 16) && fp::aligned(slot_map, 16), fp::PageDiv(page_size)};
  // A row a thread while that many threads run at once: a decode step's rows belong to as many requests, whose numbers four rows of one
  // thread would fetch one after the other (64 requests: 5.9 us, 7.8 with four).  Beyond, four: mostly one request and one page, and
  // stores of 16 bytes past the caches (1000 requests, 2 million rows, 41 MB: a row a thread 35 us, four 22.6, stores past the caches
  // 21.5, three workgroups a CU 20.3).  Every workgroup reads all requests, so there are no more of them than run at once.
  const size_t lds = (2 * static_cast<size_t>(B) + 1 + (max_batch + 31) / 32 + 3) / 4 * 16 + B * sizeof(Record);
  const bool few = max_rows <= 2ll * fp::compute_units() * kThreads;
  const int64_t fit = kLdsBytes / (lds + 1024), a_cu = few ? 2 : fit < 1 ? 1 : fit > 3 ? 3 : fit, most = a_cu * fp::compute_units();
  const int64_t turns = few ? max_rows : (max_rows + 3) / 4, work = turns > 64ll * B ? turns : 64ll * B;
  int64_t grid = (work + kThreads - 1) / kThreads;
  grid = grid < 1 ? 1 : grid > most ? most : grid;
  const auto go = [&](auto kernel) {
    if (lds > 64 * 1024 && hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize,
                                               static_cast<int>(lds)) != hipSuccess)
      return;  // the launch below would be refused: check_launch says so
    hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>(grid)), dim3(kThreads), lds, static_cast<hipStream_t>(stream), a);
  };
  few ? go(step_tables_kernel<1>) : go(step_tables_kernel<4>);
  return fp::check_launch("fp_step_tables");
}
