// Verification of drafted tokens: which of them the target model's distribution lets stand, and the token behind them.
//
//   w_i = exp((x_i - max x) / T), Z = sum of w, x the logits of the row of a token
// From the first token on, a token's children are looked at in rising order; R are the weights of those refused before:
//   child c stands if  u_c (Z - R) < w[token_c]                          (the drafts are given)
//                      u_c q[token_c] Z < w[token_c]                      (the drafts were drawn from q)
// Behind the last that stands one more token is drawn: the first i whose cumulative weight is above u_0 times the total, of
//   w without the refused tokens, or of max(0, w / Z - q).
//
// Which token that is depends on sums over the whole vocabulary to the last bits: next to the border between two tokens, and with
// 65536 of them there is always one near, sums in 32 bits would answer by the order they are taken in.  So the row that is drawn from is
// weighed in 64 bits, the exponential to 2^-51.  All other rows have to say no more than on which side of a draft's weight u (Z - R) lies:
//  * rows: every row's maximum and sum, a chunk a workgroup, from one read of the logits.  Weights in 32 bits, off by kBand at
//    most, summed in 64.
//  * walk: every workgroup puts the chunks of its request's rows together and walks down the tree; a comparison within kBand of its
//    border is made again with the row's sum in 64 bits (a few in a million).  Then it sums the weights of its pieces of the row that the walk
//    ends at, and the last workgroup of a request draws; the drawn token's logarithm is by that sum.  Where the drafts were drawn, Z is known
//    only then: until then a piece has the sums of w and of q over the tokens that surely have something left, and one with a token within kBand
//    of its border (every 100 pieces, if p and q have nothing to do with each other) is weighed again by the last workgroup.
// The first launch sets the counters of the second to 0: nothing is kept between calls.
//
// Rows is bound by the logits' bytes: 64 requests of 3 to 8 rows of 65536 in 32 bits, 92 MB, 19.7 us (4.7 TB/s), 32 of 17 to 33 in 16 bits, 104 MB,
// 24.6 us (4.2 TB/s: an exponential for every two bytes; 0.3 of it to find which rows the walk can reach).  With all weights in 64 bits the two were
// 60.7 and 50.4 us.  Walk is a line of trips and of f64 instructions: of the first 25.0 us, 2.7 until a request's rows are put together, 1.6 the walk,
// 8.5 the 25 MB of the rows that are drawn from and of their drafts' probabilities (35 instructions a token, 14 of them f64 products), 2 until the last
// workgroup has the sums, 2 for the pieces of which it was not sure, and the draw; of the second 15.5.  One request of 5 rows: 3.7 and 11.5 us.
#include "fp_common.h"

#include <math.h>

namespace {

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / 64;
constexpr int kMaxTokens = 64;
// What a row's sum may be off by, relatively.  A weight 2^-p in 32 bits is off by 2 p 2^-24 ln 2 (the exponent and the rate
// rounded) and 2^-23 (the exponential), sums of 8 by 3 * 2^-24.  Weights of 2^-p are V 2^-p of a whole of 1 or more, so p counts up to
// log2 V, 24: 2.3e-6 in all.
constexpr float kBand = 0x1p-18f;
typedef uint32_t v4u __attribute__((ext_vector_type(4)));

struct BF16 {
  static constexpr int kBytes = 2, kVec = 8;
  static __device__ __forceinline__ float get(v4u v, int i) {
    return __uint_as_float(i & 1 ? v[i >> 1] & 0xffff0000u : v[i >> 1] << 16);
  }
  static __device__ __forceinline__ float at(const char* p) {
    return __uint_as_float(static_cast<uint32_t>(*reinterpret_cast<const uint16_t*>(p)) << 16);
  }
};
struct F16 {
  static constexpr int kBytes = 2, kVec = 8;
  static __device__ __forceinline__ float get(v4u v, int i) {
    return static_cast<float>(__builtin_bit_cast(_Float16, static_cast<uint16_t>(v[i >> 1] >> (i & 1) * 16)));
  }
  static __device__ __forceinline__ float at(const char* p) { return static_cast<float>(*reinterpret_cast<const _Float16*>(p)); }
};
struct F32 {
  static constexpr int kBytes = 4, kVec = 4;
  static __device__ __forceinline__ float get(v4u v, int i) { return __uint_as_float(v[i]); }
  static __device__ __forceinline__ float at(const char* p) { return *reinterpret_cast<const float*>(p); }
};

struct Part {   // of a chunk of a row
  double sum;   // of the weights, by `peak`
  float peak;
  int best;     // the first place of `peak`, where the request is greedy
};
struct Piece {  // of 64 vectors of the row that is drawn from
  double all;   // the weights
  double kept, taken;  // of the tokens that surely have something left: weights, and the draft's probabilities; kept < 0: of some it is not sure
};

struct VerifyArgs {
  const char* logits;
  int64_t ls_b, ls_s;  // bytes
  const int64_t* tokens;
  const int32_t* parents;
  const float* uniforms;
  const float* temperatures;  // optional [B]
  const char* probs;          // optional
  int64_t ps_b, ps_s;         // bytes
  int probs_dtype;
  int32_t* accepted;
  int32_t* path;
  int64_t* answer;
  float* logprobs;
  Part* parts;     // [B * S, chunks]
  Piece* sums;     // [B, pieces]
  double* rests;   // [B, pieces]: what is left of them
  int* arrivals;   // [B]
  int B, S, V;
  int chunks, chunk_vectors;  // of a row, and of a chunk
  int draws, pieces;          // workgroups of a request, and pieces of 64 vectors
};

// 2^t for t below 1000 (0 for NaN): t = n + f, 2^f by its Chebyshev interpolation of degree 10 on [-1/2, 1/2], off by 2^-51.
__device__ __forceinline__ double power2(double t) {
  t = fmax(t, -1100.0);
  const double n = rint(t), f = t - n;
  double p = 0x1.e6063f7217bc6p-28;
  p = fma(p, f, 0x1.b675bca4eeebbp-24);
  p = fma(p, f, 0x1.62bfd47773353p-20);
  p = fma(p, f, 0x1.ffcb54062e698p-17);
  p = fma(p, f, 0x1.430913096fd9fp-13);
  p = fma(p, f, 0x1.5d87fe9d7a584p-10);
  p = fma(p, f, 0x1.3b2ab6fba1ddap-7);
  p = fma(p, f, 0x1.c6b08d703ce49p-5);
  p = fma(p, f, 0x1.ebfbdff82c598p-3);
  p = fma(p, f, 0x1.62e42fefa3a19p-1);
  p = fma(p, f, 1.0);
  return ldexp(p, static_cast<int>(n));
}

constexpr double kLog2e = 0x1.71547652b82fep+0;

// A token's weight next to the largest logit's 1.  NaN weighs nothing, and neither does anything in a row without a logit above -inf.
__device__ __forceinline__ double weight(float x, float peak, double rate) {
  if (x == peak) return peak == -INFINITY ? 0.0 : 1.0;
  return power2((static_cast<double>(x) - static_cast<double>(peak)) * rate);
}

// The same for many tokens of a row, without a branch between them where the largest logit is finite.
struct Weights {
  float peak;
  double rate;
  bool plain;
  __device__ Weights(float peak, double rate) : peak(peak), rate(rate), plain(__builtin_amdgcn_readfirstlane(fabsf(peak) < INFINITY)) {}
  __device__ __forceinline__ double operator()(float x) const {
    return plain ? power2((static_cast<double>(x) - static_cast<double>(peak)) * rate) : weight(x, peak, rate);
  }
};

__device__ __forceinline__ float heat_of(const VerifyArgs& a, int b) { return a.temperatures ? a.temperatures[b] : 1.f; }

// Whether the walk can reach row j, which is the same for all lanes: up from there, in scalar registers.
__device__ __forceinline__ bool is_reachable(int parent, int j) {
  while (j > 0) {
    const int above = __builtin_amdgcn_readlane(parent, j);
    if (above < 0 || above >= j) return false;
    j = above;
  }
  return __builtin_amdgcn_readlane(parent, 0) == -1;
}

// A row: elements in front of the first whole 16 bytes, whole ones, elements behind them.
template <typename E>
struct Row {
  const char* at;
  int head, vectors, tail;
  __device__ Row(const char* p, int V) : at(p) {
    head = min(V, static_cast<int>((16 - (reinterpret_cast<uintptr_t>(p) & 15)) & 15) / E::kBytes);
    vectors = (V - head) / E::kVec;
    tail = V - head - vectors * E::kVec;
  }
  __device__ v4u load(int v) const {
    return *reinterpret_cast<const v4u*>(at + (head + static_cast<int64_t>(v) * E::kVec) * E::kBytes);
  }
  __device__ float one(int64_t i) const { return E::at(at + i * E::kBytes); }
  __device__ int behind() const { return head + vectors * E::kVec; }  // first element behind the whole ones
};

// The rows that the walk can reach from row 0, a bit each, for all lanes; lane j holds the parent of row j, -2 if there is none.  A turn for
// every level of the tree.
__device__ __forceinline__ uint64_t reachable(int parent, int lane) {
  uint64_t rows = __ballot(lane == 0 && parent == -1);
  for (uint64_t more = rows; more;) {
    more = __ballot(parent >= 0 && parent < lane && (rows >> (parent & 63) & 1)) & ~rows;
    rows |= more;
  }
  return rows;
}

// Sum over the lanes up to this one, without a trip through LDS (row_shr:1, 2, 4, 8, then row_bcast:15, 31).
template <int kControl, int kRows>
__device__ __forceinline__ double from_lane(double x) {
  const uint64_t bits = __builtin_bit_cast(uint64_t, x);
  const uint32_t lo = __builtin_amdgcn_update_dpp(0, static_cast<int>(bits), kControl, kRows, 0xf, false);
  const uint32_t hi = __builtin_amdgcn_update_dpp(0, static_cast<int>(bits >> 32), kControl, kRows, 0xf, false);
  return __builtin_bit_cast(double, static_cast<uint64_t>(hi) << 32 | lo);
}
__device__ __forceinline__ double scan_lanes(double x) {
  x += from_lane<0x111, 0xf>(x);
  x += from_lane<0x112, 0xf>(x);
  x += from_lane<0x114, 0xf>(x);
  x += from_lane<0x118, 0xf>(x);
  x += from_lane<0x142, 0xa>(x);
  x += from_lane<0x143, 0xc>(x);
  return x;
}
__device__ __forceinline__ double lane_of(double x, int lane) {
  const uint64_t bits = __builtin_bit_cast(uint64_t, x);
  const uint32_t lo = __builtin_amdgcn_readlane(static_cast<int>(bits), lane), hi = __builtin_amdgcn_readlane(static_cast<int>(bits >> 32), lane);
  return __builtin_bit_cast(double, static_cast<uint64_t>(hi) << 32 | lo);
}
__device__ __forceinline__ double sum_lanes(double x) { return lane_of(scan_lanes(x), 63); }

template <typename T, typename Op>
__device__ __forceinline__ T reduce_lanes(T x, int width, Op op) {
  for (int d = 1; d < width; d <<= 1) x = op(x, __shfl_xor(x, d));
  return x;
}

// The elements of a row that belong to its v-th vector, in order, to f(x, i, place in the vector): of the first one those in front of it,
// too, and of the last one those behind (place -1).
template <typename E, typename F>
__device__ __forceinline__ void each(const Row<E>& r, int v, const v4u& x, F f) {
  if (r.head > 0 && v == 0)
    for (int i = 0; i < r.head; ++i) f(r.one(i), i, -1);
  if (v < r.vectors)
#pragma unroll
    for (int i = 0; i < E::kVec; ++i) f(E::get(x, i), r.head + v * E::kVec + i, i);
  if (r.tail > 0 && v == max(r.vectors - 1, 0))
    for (int i = 0; i < r.tail; ++i) f(r.one(r.behind() + i), r.behind() + i, -1);
}

// ---------------------------------------------------------------------------------------------------------------- rows
// A thread has G vectors at a time, the next ones on their way meanwhile, and weighs by a logit of its own that moves only when a larger one
// is more than 2^kSlack heavier: no exchange between threads before the end of the chunk.  An exponent is x rate - shift in one
// instruction, rate and shift in 32 bits: the weights are next to 2^reference, which has in 64 bits what the two were rounded by.  An
// infinity that is not below, or NaN, makes a thread's sum NaN, and it weighs once more.  (32 requests of 17 to 33 rows of 65536 in 16 bits: 24.2 us,
// 26.2 with a difference, a product and a bound for NaN.)
constexpr double kSlack = 20.0;
constexpr double kFar = 0x1p22;  // a shift up to this is rounded by 1/4 at most

template <typename E, int G>
__global__ __launch_bounds__(kThreads) void verify_rows_kernel(const VerifyArgs a) {
  __shared__ float s_peak[kWaves];
  __shared__ int s_best[kWaves];
  __shared__ double s_sum[kWaves];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const uint32_t row = blockIdx.x / static_cast<uint32_t>(a.chunks), b = row / static_cast<uint32_t>(a.S);
  const int c = blockIdx.x - row * a.chunks, j = row - b * a.S;
  if (c == 0 && j == 0 && tid == 0) a.arrivals[b] = 0;
  const float heat = heat_of(a, b);
  if (!is_reachable(lane < a.S ? a.parents[static_cast<int64_t>(b) * a.S + lane] : -2, j)) return;
  const Row<E> r(a.logits + b * a.ls_b + j * a.ls_s, a.V);
  const int v_end = min((c + 1) * a.chunk_vectors, r.vectors);
  int v = c * a.chunk_vectors + tid;
  const bool greedy = !(heat > 0.f);
  const double rate = kLog2e / (greedy ? 1.0 : heat);
  const float rate32 = static_cast<float>(rate), slack = static_cast<float>(kSlack / rate);

  float peak = -INFINITY, by = -INFINITY, shift = 0.f;  // by: what the thread weighs by
  int best = INT32_MAX;
  double sum = 0.0, reference = 0.0;
  const auto load = [&](v4u (&x)[G], int v) {
#pragma unroll
    for (int k = 0; k < G; ++k) {
      x[k] = v4u{0, 0, 0, 0};
      if (v + k * kThreads < v_end) x[k] = r.load(v + k * kThreads);
    }
  };
  const auto grow = [&](float top) {  // of the elements to come
    if (top > by + slack) {
      shift = top * rate32;
      const double next = static_cast<double>(shift) + static_cast<double>(top) * (rate - static_cast<double>(rate32));
      sum = by == -INFINITY ? 0.0 : sum * power2(reference - next);  // (nothing weighs anything before: NaN alone)
      reference = next;
      by = top;
    }
  };
  v4u x[G];
  load(x, v);
  for (; v < v_end; v += G * kThreads) {
    v4u next[G];
    load(next, v + G * kThreads);
    float top = -INFINITY;
#pragma unroll
    for (int k = 0; k < G; ++k)
      if (k == 0 || v + k * kThreads < v_end)
#pragma unroll
        for (int i = 0; i < E::kVec; ++i) top = fmaxf(top, E::get(x[k], i));
    if (greedy && top > peak) {
#pragma unroll
      for (int k = G - 1; k >= 0; --k)
        if (v + k * kThreads < v_end)
#pragma unroll
          for (int i = E::kVec - 1; i >= 0; --i) best = E::get(x[k], i) == top ? r.head + (v + k * kThreads) * E::kVec + i : best;
    }
    peak = fmaxf(peak, top);
    grow(top);
#pragma unroll
    for (int k = 0; k < G; ++k)
      if (k == 0 || v + k * kThreads < v_end) {
        float w[E::kVec];
#pragma unroll
        for (int i = 0; i < E::kVec; ++i) w[i] = __builtin_amdgcn_exp2f(fmaf(E::get(x[k], i), rate32, -shift));  // (-inf: 0)
#pragma unroll
        for (int d = 1; d < E::kVec; d *= 2)
#pragma unroll
          for (int i = 0; i < E::kVec; i += 2 * d) w[i] += w[i + d];
        sum += w[0];
      }
#pragma unroll
    for (int k = 0; k < G; ++k) x[k] = next[k];
  }
  // the elements outside the whole 16 bytes: the first chunk's first threads and the last one's next 8
  int loose = -1;
  if (c == 0 && tid < r.head) loose = tid;
  if (c == a.chunks - 1 && tid >= 8 && tid - 8 < r.tail) loose = r.behind() + tid - 8;
  if (loose >= 0) {
    const float y = r.one(loose);
    if (y > peak || (y == peak && loose < best)) best = loose;
    peak = fmaxf(peak, y);
    grow(y);
    sum += power2(static_cast<double>(y) * rate - reference);
  }
  float all = reduce_lanes(peak, 64, [](float p, float q) { return fmaxf(p, q); });
  if (lane == 0) s_peak[wave] = all;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kWaves; ++w) all = fmaxf(all, s_peak[w]);
  if (fabs(all * rate) < kFar && rate > 0x1p-40 && rate < 0x1p40 && fabs(sum) < INFINITY) {
    sum = by == -INFINITY ? 0.0 : sum * power2(reference - static_cast<double>(all) * rate);
  } else {  // infinite and far logits, NaN, temperatures out of all measure: once more, in 64 bits
    sum = loose >= 0 ? weight(r.one(loose), all, rate) : 0.0;
    for (int u = c * a.chunk_vectors + tid; u < v_end; u += kThreads) {
#pragma nounroll
      for (int i = 0; i < E::kVec; ++i) sum += weight(r.one(r.head + u * E::kVec + i), all, rate);
    }
  }
  sum = sum_lanes(sum);
  if (greedy) best = reduce_lanes(peak == all ? best : INT32_MAX, 64, [](int p, int q) { return min(p, q); });
  if (lane == 0) {
    s_sum[wave] = sum;
    s_best[wave] = best;
  }
  __syncthreads();
  if (tid == 0) {
    for (int w = 1; w < kWaves; ++w) sum += s_sum[w], best = min(best, s_best[w]);
    a.parts[blockIdx.x] = Part{sum, all, best};
  }
}

// ----------------------------------------------------------------------------------------------------------- decisions
__device__ __forceinline__ float probability(const VerifyArgs& a, const char* row, int64_t i) {
  return a.probs_dtype == FP_DTYPE_F32 ? F32::at(row + i * 4) : a.probs_dtype == FP_DTYPE_BF16 ? BF16::at(row + i * 2) : F16::at(row + i * 2);
}

__device__ __forceinline__ void publish(double* p, double x) {
  __hip_atomic_store(reinterpret_cast<uint64_t*>(p), __builtin_bit_cast(uint64_t, x), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ double take(const double* p) {
  return __builtin_bit_cast(double, __hip_atomic_load(reinterpret_cast<const uint64_t*>(p), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT));
}

// log p of a token with logit x; slope: 1 / temperature
__device__ __forceinline__ float log_share(float x, float peak, double slope, double total) {
  return static_cast<float>((x == peak ? 0.0 : (static_cast<double>(x) - static_cast<double>(peak)) * slope) - log(total));
}

// Sums of three numbers over the lanes: of the first in lanes 0 to 15, of the second in 16 to 31, of the third in 32 to 47.  While lanes of
// the first halves add to one number, those of the second add to another: 21 instructions instead of the 90 of three sums.
__device__ __forceinline__ double add_halves(double x, double y) {  // x in lanes 0 to 31, y in 32 to 63
  const uint64_t p = __builtin_bit_cast(uint64_t, x), q = __builtin_bit_cast(uint64_t, y);
  const auto lo = __builtin_amdgcn_permlane32_swap(static_cast<uint32_t>(p), static_cast<uint32_t>(q), false, false);
  const auto hi = __builtin_amdgcn_permlane32_swap(static_cast<uint32_t>(p >> 32), static_cast<uint32_t>(q >> 32), false, false);
  return __builtin_bit_cast(double, static_cast<uint64_t>(hi[0]) << 32 | lo[0]) + __builtin_bit_cast(double, static_cast<uint64_t>(hi[1]) << 32 | lo[1]);
}
__device__ __forceinline__ double add_rows(double x, double y) {  // x in lanes 0 to 15 and 32 to 47, y in the others
  const uint64_t p = __builtin_bit_cast(uint64_t, x), q = __builtin_bit_cast(uint64_t, y);
  const auto lo = __builtin_amdgcn_permlane16_swap(static_cast<uint32_t>(p), static_cast<uint32_t>(q), false, false);
  const auto hi = __builtin_amdgcn_permlane16_swap(static_cast<uint32_t>(p >> 32), static_cast<uint32_t>(q >> 32), false, false);
  return __builtin_bit_cast(double, static_cast<uint64_t>(hi[0]) << 32 | lo[0]) + __builtin_bit_cast(double, static_cast<uint64_t>(hi[1]) << 32 | lo[1]);
}
__device__ __forceinline__ double sum_three(double x, double y, double z) {
  double s = add_rows(add_halves(x, z), add_halves(y, 0.0));
  s += from_lane<0xb1, 0xf>(s);   // quad_perm: the neighbour,
  s += from_lane<0x4e, 0xf>(s);   // the other pair of four,
  s += from_lane<0x141, 0xf>(s);  // row_half_mirror: the other four of eight,
  s += from_lane<0x140, 0xf>(s);  // row_mirror: the other eight
  return s;
}

constexpr int kHeldEach = 4, kHeld = kHeldEach * kThreads;  // pieces whose sums the last workgroup holds in LDS
struct DrawShared {
  double all[kHeld], kept[kHeld], taken[kHeld];
  double sum[kWaves], total[kWaves], rest[kWaves];
  int place, flag;
  double refused;  // weights of the tokens refused at the row that is drawn from
};

__device__ __forceinline__ double sum_threads(double x, double (&part)[kWaves]) {  // a part once between two barriers
  x = sum_lanes(x);
  if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = x;
  __syncthreads();
  return part[0] + part[1] + part[2] + part[3];
}

// Weights are summed by pieces of 64 vectors, a wavefront's.  The last workgroup of a request runs what follows alone, its instructions come from
// memory as they are needed: loops, not copies of their bodies.

// Whether this is the last of `n` workgroups whose sums are on their way.
__device__ __forceinline__ bool last_to_arrive(int* counter, int n, int* flag) {
  asm volatile("s_waitcnt vmcnt(0)" : : : "memory");  // this wavefront's have arrived
  __syncthreads();
  if (threadIdx.x == 0) *flag = __hip_atomic_fetch_add(counter, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == n - 1;
  __syncthreads();
  return *flag != 0;
}

// Elements of a piece, by threads; and the first and the end of piece k: what is in front of the whole 16 bytes is the first one's, what is behind
// them the last one's.
template <typename E>
constexpr int elements_each() { return (64 * E::kVec + 2 * (E::kVec - 1) + kThreads - 1) / kThreads; }
template <typename E>
__device__ __forceinline__ int2 piece_range(const Row<E>& r, int V, int k) {
  const int pieces = max((r.vectors + 63) / 64, 1);
  return int2{k == 0 ? 0 : r.head + k * 64 * E::kVec, k == pieces - 1 ? V : r.head + (k + 1) * 64 * E::kVec};
}

// The first token at which the weights of the row pass u times their total: sum_of(k) the sum of piece k of n, weigh(x, i, load(i)) the weight
// of token i.  What it is goes to answer(token, x), by one thread; -1 if nothing weighs anything.  Only a piece that weighs something is chosen:
// behind the last of them the sums up to a lane, which every lane adds up in another order, still differ in their last bits, and a goal of the whole
// total (u = 1) lies among them.
template <typename E, typename S, typename L, typename W, typename A>
__device__ __forceinline__ void draw(const Row<E>& r, int V, double total, S sum_of, int n, float u, DrawShared& sh, L load, W weigh, A answer) {
  constexpr int kEach = elements_each<E>();
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  // by every wavefront, which all get the same
  const double goal = (u < 0.f ? 0.0 : static_cast<double>(u)) * total;  // (NaN passes nothing: the last token)
  double before = 0.0, before_last = 0.0;
  int part = -1, last = -1;
#pragma nounroll
  for (int k0 = 0; k0 < n && part < 0; k0 += 64) {
    const double s = k0 + lane < n ? sum_of(k0 + lane) : 0.0, upto = scan_lanes(s);
    const uint64_t some = __ballot(s > 0.0), past = some & __ballot(before + upto > goal);
    if (past) {
      const int l = __builtin_ctzll(past);
      part = k0 + l;
      before += lane_of(upto - s, l);
    } else {
      if (some) {
        const int l = 63 - __builtin_clzll(some);
        last = k0 + l;
        before_last = before + lane_of(upto - s, l);
      }
      before += lane_of(upto, 63);
    }
  }
  if (part < 0) part = last, before = before_last;
  if (part < 0) {
    if (tid == 0) answer(-1, 0.f);
    return;
  }
  const int2 range = piece_range(r, V, part);
  const int mine = range.x + tid * kEach, end = range.y;
  double w[kEach], sum = 0.0;
  float x[kEach], with[kEach];
  int found = -1;
  float its = 0.f;
#pragma unroll
  for (int i = 0; i < kEach; ++i) {
    x[i] = mine + i < end ? r.one(mine + i) : 0.f;
    with[i] = mine + i < end ? load(mine + i) : 0.f;
  }
#pragma unroll
  for (int i = 0; i < kEach; ++i) {
    w[i] = mine + i < end ? weigh(x[i], mine + i, with[i]) : 0.0;
    sum += w[i];
    found = w[i] > 0.0 ? mine + i : found;  // the last that weighs something
    its = w[i] > 0.0 ? x[i] : its;
  }
  const double upto = scan_lanes(sum);
  if (lane == 63) sh.sum[wave] = upto;
  if (tid == 0) sh.place = INT32_MAX;
  __syncthreads();
  double at = before;
#pragma unroll
  for (int k = 0; k < kWaves - 1; ++k) at += k < wave ? sh.sum[k] : 0.0;
  at += upto - sum;
  if (sum > 0.0 && at + sum > goal) {
    bool done = false;
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
      at += w[i];
      const bool here = !done && w[i] > 0.0 && at > goal;
      found = here ? mine + i : found;
      its = here ? x[i] : its;
      done |= here;
    }
    atomicMin(&sh.place, found);
  }
  __syncthreads();
  if (sh.place == INT32_MAX) {  // u at its very end: the last token that weighs something
    __syncthreads();
    if (tid == 0) sh.place = -1;
    __syncthreads();
    if (found >= 0) atomicMax(&sh.place, found);
    __syncthreads();
  }
  if (sh.place < 0) {  // not a token of the piece
    if (tid == 0) answer(-1, 0.f);
    return;
  }
  if (found == sh.place) answer(found, its);
}

// Element i0 .. of a row of the draft's probabilities; `aligned`: kVec of them at once
template <int kVec>
__device__ __forceinline__ void load_probs(const VerifyArgs& a, const char* row, int64_t i0, bool aligned, float (&out)[kVec]) {
  if (aligned && a.probs_dtype == FP_DTYPE_F32) {
#pragma unroll
    for (int h = 0; h < kVec / 4; ++h) {
      const v4u four = *reinterpret_cast<const v4u*>(row + (i0 + h * 4) * 4);
#pragma unroll
      for (int i = 0; i < 4; ++i) out[h * 4 + i] = F32::get(four, i);
    }
  } else if (aligned) {
    uint32_t two[kVec / 2];
    if constexpr (kVec == 8) {
      const v4u all = *reinterpret_cast<const v4u*>(row + i0 * 2);
#pragma unroll
      for (int i = 0; i < 4; ++i) two[i] = all[i];
    } else {
      const uint2 all = *reinterpret_cast<const uint2*>(row + i0 * 2);
      two[0] = all.x, two[1] = all.y;
    }
    const bool bf16 = a.probs_dtype == FP_DTYPE_BF16;
#pragma unroll
    for (int i = 0; i < kVec; ++i) {
      const v4u pack = {two[i / 2], 0, 0, 0};
      out[i] = bf16 ? BF16::get(pack, i & 1) : F16::get(pack, i & 1);
    }
  } else {
#pragma unroll
    for (int i = 0; i < kVec; ++i) out[i] = probability(a, row, i0 + i);
  }
}

template <typename E>
__global__ __launch_bounds__(kThreads) void verify_walk_kernel(const VerifyArgs a) {
  __shared__ float s_peak[kMaxTokens];
  __shared__ int s_best[kMaxTokens];
  __shared__ double s_total[kMaxTokens];
  __shared__ int s_out[kMaxTokens];  // refused tokens
  __shared__ int s_node, s_count, s_n_out, s_refused, s_again;
  __shared__ DrawShared sh;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const uint32_t b = blockIdx.x / static_cast<uint32_t>(a.draws);
  const int c = blockIdx.x - b * a.draws, S = a.S;
  const int64_t first = static_cast<int64_t>(b) * S;
  const float heat = heat_of(a, b), u0 = a.uniforms[first];
  const bool greedy = !(heat > 0.f);
  const double rate = kLog2e / (greedy ? 1.0 : heat), slope = 1.0 / (greedy ? 1.0 : heat);

  // a token a lane
  const int parent = lane < S ? a.parents[first + lane] : -2;
  const int64_t token = lane < S ? a.tokens[first + lane] : -1;
  const float u = lane < S ? a.uniforms[first + lane] : 0.f;

  // every row's maximum and sum, `per` lanes a row: the first chunks are on their way before it is known which rows are reached
  int per = 64;
  while (per > kThreads / S) per >>= 1;
  const int mine = tid / per, row = mine < S ? mine : 0;
  const Part* const parts = a.parts + (first + row) * a.chunks;
  Part t = parts[min(tid % per, a.chunks - 1)];
  const uint64_t rows = reachable(parent, lane);
  const bool there = rows & 1;
  const bool is_row = mine < S && (rows >> row & 1);
  const bool child = lane > 0 && (rows >> lane & 1), known = token >= 0 && token < a.V;
  const int at = child ? parent : 0, name = known ? static_cast<int>(token) : -1;
  float x = -INFINITY;
  double q = 0.0;
  if (wave == 0 && child && known) {
    x = E::at(a.logits + b * a.ls_b + at * a.ls_s + token * E::kBytes);
    if (a.probs) q = probability(a, a.probs + b * a.ps_b + at * a.ps_s, token);
  }
  if (tid % per >= a.chunks || !is_row) t = Part{0.0, -INFINITY, INT32_MAX};
  if (is_row) {
    for (int k = tid % per + per; k < a.chunks; k += per) {
      const Part p = parts[k];
      if (p.peak > t.peak) {
        t.sum = t.sum * weight(t.peak, p.peak, rate) + p.sum;
        t.best = p.best;
        t.peak = p.peak;
      } else {
        t.sum += p.sum * weight(p.peak, t.peak, rate);
        if (p.peak == t.peak) t.best = min(t.best, p.best);
      }
    }
  }
  {
    const float peak = reduce_lanes(t.peak, per, [](float p, float q) { return fmaxf(p, q); });
    const double total = reduce_lanes(t.sum * weight(t.peak, peak, rate), per, [](double p, double q) { return p + q; });
    const int best = greedy ? reduce_lanes(t.peak == peak ? t.best : INT32_MAX, per, [](int p, int q) { return min(p, q); }) : 0;
    if (is_row && tid % per == 0) {
      s_peak[row] = peak;
      s_total[row] = total;
      s_best[row] = peak == -INFINITY ? -1 : best;
    }
  }
  __syncthreads();
  if (!there) {
    if (c == 0 && tid < S) {
      a.path[first + tid] = -1;
      a.answer[first + tid] = -1;
      a.logprobs[first + tid] = 0.f;
      if (tid == 0) a.accepted[b] = 0;
    }
    return;
  }

  // the walk down the tree
  uint64_t exact = 0;  // rows whose sums are in 64 bits
  const double w = wave == 0 && child && known ? weight(x, s_peak[at], rate) : 0.0;
  for (;;) {
    if (wave == 0) {
      int node = 0, count = 0, path = lane == 0 ? 0 : -1, again = -1;  // path: its lane-th row
      double refused = 0.0;
      for (bool stands = true; stands;) {
        // the children in turn: what those refused weigh, the same token once
        const double z = s_total[node], doubt = exact >> node & 1 ? -1.0 : kBand * z;
        const int best = s_best[node];
        refused = 0.0;
        bool out = false;  // this lane's token is refused at this node
        stands = false;
        for (uint64_t left = __ballot(child && parent == node); left && !stands && again < 0; left &= left - 1) {
          const int i = __builtin_ctzll(left), token_i = __builtin_amdgcn_readlane(name, i);
          if (greedy) {
            stands = token_i >= 0 && token_i == best;
          } else if (a.probs) {
            const double side = lane_of(static_cast<double>(u) * q, i) * z, w_i = lane_of(w, i);
            if (w_i > 0.0 && fabs(side - w_i) <= (doubt < 0.0 ? -1.0 : kBand * side)) again = node;
            stands = again < 0 && w_i > 0.0 && side < w_i;
          } else if (token_i >= 0 && __ballot(out && name == token_i) == 0) {
            const double side = lane_of(static_cast<double>(u), i) * (z - refused), w_i = lane_of(w, i);
            if (w_i > 0.0 && fabs(side - w_i) <= doubt) again = node;
            stands = again < 0 && w_i > 0.0 && side < w_i;
            refused += w_i;
          }
          if (a.probs && !stands) break;  // of drafts that were drawn the first child only
          out |= lane == i;
          if (stands) {
            node = i;
            ++count;
            if (lane == count) path = i;
          }
        }
      }
      const bool here = child && parent == node, gone = here && known;
      const uint64_t out = __ballot(gone);
      if (gone) s_out[__builtin_popcountll(out & ((1ull << lane) - 1))] = name;
      const bool any = __ballot(here) != 0;
      if (lane == 0) {
        s_node = node;
        s_count = count;
        s_n_out = __builtin_popcountll(out);
        s_refused = any;
        s_again = again;
        sh.refused = refused;
      }
      if (c == 0 && again < 0) {
        // the token of path[lane + 1] answers at place lane; the last place is the drawn one's
        const int next = __shfl_down(path, 1);
        const int from = lane < count ? next : 0;
        const int64_t says_token = __shfl(token, from);
        const float its = __shfl(x, from);
        const int under = __shfl(at, from);
        if (lane < S) {
          a.path[first + lane] = path;
          if (lane != count) {
            const bool says = lane < count;
            a.answer[first + lane] = says ? says_token : -1;
            a.logprobs[first + lane] = says ? log_share(its, s_peak[under], slope, s_total[under]) : 0.f;
          }
        }
        if (lane == 0) a.accepted[b] = count;
      }
    }
    __syncthreads();
    const int again = s_again;
    if (again < 0) break;
    // too near to its border: the row's sum once more, in 64 bits
    const Row<E> r(a.logits + b * a.ls_b + again * a.ls_s, a.V);
    const float peak = s_peak[again];
    const Weights weigh(peak, rate);
    double sum = 0.0;
    for (int v = tid; v < max(r.vectors, 1); v += kThreads)
      each<E>(r, v, v < r.vectors ? r.load(v) : v4u{0, 0, 0, 0}, [&](float y, int, int) { sum += weigh(y); });
    sum = sum_lanes(sum);
    if (lane == 0) sh.sum[wave] = sum;
    __syncthreads();
    if (tid == 0) s_total[again] = sh.sum[0] + sh.sum[1] + sh.sum[2] + sh.sum[3];
    exact |= 1ull << again;
    __syncthreads();
  }

  const int node = s_node, count = s_count;
  const float peak = s_peak[node];
  const double total = s_total[node];
  double whole = total;  // what the drawn token's logarithm is by: the sum in 64 bits, as soon as that is known
  const Row<E> r(a.logits + b * a.ls_b + node * a.ls_s, a.V);
  const auto answer = [&](int token, float x) {
    a.answer[first + count] = token;
    a.logprobs[first + count] = token < 0 ? 0.f : log_share(x, peak, slope, whole);
  };
  if (greedy || peak == -INFINITY) {
    if (c == 0 && tid == 0) answer(s_best[node], peak);
    return;
  }
  const int n_out = a.probs ? 0 : s_n_out;
  const Weights weights(peak, rate);
  Piece* const sums = a.sums + static_cast<int64_t>(b) * a.pieces;
  const int step = a.draws * kWaves;
  if (!(a.probs && s_refused)) {
    const auto is_out = [&](int i) {  // refused
      bool out = false;
#pragma nounroll
      for (int k = 0; k < n_out; ++k) out |= s_out[k] == i;
      return out;
    };
    int piece = c * kWaves + wave;
    v4u x = {0, 0, 0, 0};
    if (piece * 64 + lane < r.vectors) x = r.load(piece * 64 + lane);
    for (; piece < a.pieces; piece += step) {
      const int v = piece * 64 + lane;
      v4u next = {0, 0, 0, 0};
      if (v + step * 64 < r.vectors) next = r.load(v + step * 64);
      uint32_t out = 0;  // the vector's refused tokens, a bit each
#pragma nounroll
      for (int k = 0; k < n_out; ++k) {
        const uint32_t place = s_out[k] - (r.head + v * E::kVec);
        if (place < E::kVec) out |= 1u << place;
      }
      double sum = 0.0;
      each<E>(r, v, x, [&](float y, int i, int place) {
        const double w = weights(y);
        sum += (place >= 0 ? out >> place & 1 : is_out(i)) ? 0.0 : w;
      });
      sum = sum_lanes(sum);
      if (lane == 0) publish(&sums[piece].all, sum);
      x = next;
    }
    if (!last_to_arrive(a.arrivals + b, a.draws, &sh.flag)) return;
    double all[kHeldEach], total = 0.0;
#pragma unroll
    for (int i = 0; i < kHeldEach; ++i) all[i] = take(&sums[min(i * kThreads + tid, a.pieces - 1)].all);
#pragma unroll
    for (int i = 0; i < kHeldEach; ++i) {
      sh.all[i * kThreads + tid] = all[i];
      total += i * kThreads + tid < a.pieces ? all[i] : 0.0;
    }
#pragma nounroll
    for (int k = kHeld + tid; k < a.pieces; k += kThreads) total += take(&sums[k].all);
    total = sum_threads(total, sh.total);
    whole = total + sh.refused;
    draw<E>(r, a.V, total, [&](int k) { return k < kHeld ? sh.all[k] : take(&sums[k].all); }, a.pieces, u0, sh,
            [](int) { return 0.f; }, [&](float y, int i, float) { return is_out(i) ? 0.0 : weights(y); }, answer);
    return;
  }

  // max(0, w / Z - q)
  const char* const probs = a.probs + b * a.ps_b + node * a.ps_s;
  const int pe = a.probs_dtype == FP_DTYPE_F32 ? 4 : 2;
  const bool aligned = reinterpret_cast<uintptr_t>(probs + r.head * pe) % (E::kVec * pe < 16 ? E::kVec * pe : 16) == 0;
  const double about = 1.0 / total;
  {
    int piece = c * kWaves + wave;
    v4u x = {0, 0, 0, 0};
    float q[E::kVec] = {};
    const auto load = [&](int v, v4u& x, float (&q)[E::kVec]) {
      if (v >= r.vectors) return;
      x = r.load(v);
      load_probs<E::kVec>(a, probs, r.head + static_cast<int64_t>(v) * E::kVec, aligned, q);
    };
    load(piece * 64 + lane, x, q);
    for (; piece < a.pieces; piece += step) {
      const int v = piece * 64 + lane;
      v4u next = {0, 0, 0, 0};
      float q_next[E::kVec] = {};
      load(v + step * 64, next, q_next);
      Piece sum = {0.0, 0.0, 0.0};
      bool unsure = false;
      each<E>(r, v, x, [&](float y, int i, int place) {
        const double w = weights(y), taken = place >= 0 ? q[place] : probability(a, probs, i), left = w * about - taken;
        sum.all += w;
        const bool kept = left > 0.0;
        sum.kept += kept ? w : 0.0;
        sum.taken += kept ? taken : 0.0;
        unsure |= fabs(left) <= 4.0 * kBand * taken && taken > 0.0;  // (NaN is not left)
      });
      const double its = sum_three(sum.all, sum.kept, sum.taken);
      const bool again = __ballot(unsure) != 0;
      if (lane % 16 == 0 && lane < 48) publish(&sums[piece].all + lane / 16, again && lane == 16 ? -1.0 : its);
      x = next;
#pragma unroll
      for (int i = 0; i < E::kVec; ++i) q[i] = q_next[i];
    }
  }
  if (!last_to_arrive(a.arrivals + b, a.draws, &sh.flag)) return;
  double all[kHeldEach], kept[kHeldEach], taken[kHeldEach], sum = 0.0, rest = 0.0;
#pragma unroll
  for (int i = 0; i < kHeldEach; ++i) {  // all of them on their way at once
    const Piece* const its = sums + min(i * kThreads + tid, a.pieces - 1);
    all[i] = take(&its->all), kept[i] = take(&its->kept), taken[i] = take(&its->taken);
  }
#pragma unroll
  for (int i = 0; i < kHeldEach; ++i) {
    const int k = i * kThreads + tid;
    sh.all[k] = all[i], sh.kept[k] = kept[i], sh.taken[k] = taken[i];
    sum += k < a.pieces ? all[i] : 0.0;
  }
#pragma nounroll
  for (int k = kHeld + tid; k < a.pieces; k += kThreads) sum += take(&sums[k].all);
  whole = sum_threads(sum, sh.total);
  const double share = 1.0 / whole;
  const auto left_of = [&](float y, float q) { return fmax(0.0, weights(y) * share - static_cast<double>(q)); };
  // what is left of every piece, in place of what was kept; those of which it was not sure by the wavefront that found it
  double* const rests = a.rests + static_cast<int64_t>(b) * a.pieces;
  const auto set_rest = [&](int k, double x) {
    rest += x;
    if (k < kHeld)
      sh.kept[k] = x;
    else
      publish(rests + k, x);
  };
  const int rounds = (a.pieces + kThreads - 1) / kThreads;
#pragma nounroll
  for (int round = 0; round < rounds; ++round) {
    const int k = round * kThreads + tid;
    bool unsure = false;
    if (k < a.pieces) {
      const double kept = k < kHeld ? sh.kept[k] : take(&sums[k].kept), taken = k < kHeld ? sh.taken[k] : take(&sums[k].taken);
      unsure = kept < 0.0;
      if (!unsure) set_rest(k, fmax(0.0, kept * share - taken));
    }
    for (uint64_t again = __ballot(unsure); again; again &= again - 1) {
      const int piece = round * kThreads + wave * 64 + __builtin_ctzll(again);
      const int2 range = piece_range(r, a.V, piece);
      float y[E::kVec + 1], q[E::kVec + 1];  // (up to 2 (kVec - 1) more than 64 vectors)
#pragma unroll
      for (int i = 0; i <= E::kVec; ++i) {
        const int at = min(range.x + i * 64 + lane, range.y - 1);
        y[i] = r.one(at), q[i] = probability(a, probs, at);
      }
      double sum = 0.0;
#pragma unroll
      for (int i = 0; i <= E::kVec; ++i) sum += range.x + i * 64 + lane < range.y ? left_of(y[i], q[i]) : 0.0;
      sum = sum_lanes(sum);
      if (lane == 0) set_rest(piece, sum);
    }
  }
  asm volatile("s_waitcnt vmcnt(0)" : : : "memory");
  const double left = sum_threads(rest, sh.rest);
  const bool own = !(left > 0.0);  // nothing is left: the target's own distribution
  draw<E>(r, a.V, own ? whole : left,
          [&](int k) { return k < kHeld ? own ? sh.all[k] : sh.kept[k] : take(own ? &sums[k].all : rests + k); }, a.pieces, u0, sh,
          [&](int i) { return probability(a, probs, i); }, [&](float y, int, float q) { return own ? weights(y) : left_of(y, q); }, answer);
}

constexpr int kRowVectors = 16;  // vectors a thread of the largest cut of rows
struct Cut {
  int nv, chunks;
};
// Vectors a thread: as many as leave `wanted` workgroups, `most` at most.
Cut cut_of(int64_t rows, int V, int vec, int most, int64_t wanted) {
  const int64_t vectors = (static_cast<int64_t>(V) + vec - 1) / vec;
  Cut c{most, 0};
  for (;; c.nv /= 2) {
    c.chunks = static_cast<int>((vectors + kThreads * c.nv - 1) / (kThreads * c.nv));
    if (c.nv == 1 || rows * c.chunks >= wanted) return c;
  }
}
int64_t rows_wanted() { return 6ll * fp::compute_units(); }
Cut rows_cut(int B, int S, int V, int vec) { return cut_of(static_cast<int64_t>(B) * S, V, vec, kRowVectors, rows_wanted()); }
// Chunks of up to this many rows of up to V logits: those of the largest cut, or, of a smaller one, less than twice what was wanted (the cut of twice
// its size made too few).
int64_t most_chunks(int64_t rows, int V, int vec) {
  const int64_t vectors = (static_cast<int64_t>(V) + vec - 1) / vec;
  const int64_t largest = rows * ((vectors + kThreads * kRowVectors - 1) / (kThreads * kRowVectors)), smallest = rows * ((vectors + kThreads - 1) / kThreads);
  const int64_t finer = 2 * rows_wanted() < smallest ? 2 * rows_wanted() : smallest;
  return largest > finer ? largest : finer;
}
// Workgroups of a request for the row that is drawn from: four pieces each, more where there are two for every CU without.
Cut draw_cut(int B, int V, int vec) { return cut_of(B, V, vec, 4, 2ll * fp::compute_units()); }
int pieces_of(int V, int vec) { return static_cast<int>((static_cast<int64_t>(V) + vec * 64 - 1) / (vec * 64)); }

// Whether both launches, a workgroup a chunk of a row and a workgroup a request's share of the row that is drawn from, are of fewer than 2^32 lanes.
bool one_launch(int B, int S, int V, int vec) {
  const int64_t rows = static_cast<int64_t>(B) * S * rows_cut(B, S, V, vec).chunks, draws = static_cast<int64_t>(B) * draw_cut(B, V, vec).chunks;
  return (rows > draws ? rows : draws) < (1ll << 32) / kThreads;
}
int too_many(const char* what, int B, int S, int V) {
  return fp::fail(FP_ERR_UNSUPPORTED, "%s: %d requests of %d rows of %d logits are too many for one call", what, B, S, V);
}
int check_shape(const char* what, int B, int S, int V) {
  if (B < 0 || S <= 0 || V <= 0) return fp::fail(FP_ERR_INVALID_ARGUMENT, "%s: bad sizes (B=%d S=%d V=%d)", what, B, S, V);
  if (S > kMaxTokens || V > 1 << 24)
    return fp::fail(FP_ERR_UNSUPPORTED, "%s: at most %d tokens a request and a vocabulary of %d (got %d and %d)", what, kMaxTokens, 1 << 24, S, V);
  if (!one_launch(B, S, V, 8)) return too_many(what, B, S, V);  // of 16 bits; fp_verify_drafts knows its type
  return FP_OK;
}

struct Layout {
  int64_t parts, sums, rests, bytes;
};
Layout layout_of(int64_t B, int64_t chunks, int64_t pieces) {
  Layout l;
  l.parts = (B * 4 + 15) / 16 * 16;
  l.sums = l.parts + chunks * static_cast<int64_t>(sizeof(Part));
  l.rests = l.sums + B * pieces * static_cast<int64_t>(sizeof(Piece));
  l.bytes = l.rests + B * pieces * 8;
  return l;
}
// What any call of this size or smaller, in any type, needs: fewer requests are cut finer and can have more chunks.
int64_t workspace_of(int B, int S, int V) {
  int64_t most = 0;
  for (const int vec : {4, 8}) {
    const int64_t n = layout_of(B, most_chunks(static_cast<int64_t>(B) * S, V, vec), pieces_of(V, vec)).bytes;
    most = n > most ? n : most;
  }
  return most;
}

}  // namespace

extern "C" int64_t fp_verify_drafts_workspace_bytes(int32_t B, int32_t S, int32_t V) {
  if (const int rc = check_shape("fp_verify_drafts_workspace_bytes", B, S, V)) return rc;
  return workspace_of(B, S, V);
}

extern "C" int fp_verify_drafts(const void* logits, int64_t logits_stride_b, int64_t logits_stride_s, int dtype, const int64_t* tokens,
                                const int32_t* parents, const float* uniforms, const float* temperatures, const void* draft_probs,
                                int64_t probs_stride_b, int64_t probs_stride_s, int probs_dtype, int32_t* accepted, int32_t* path,
                                int64_t* answer, float* logprobs, void* workspace, int64_t workspace_bytes, int32_t B, int32_t S,
                                int32_t V, void* stream) {
  const char* const what = "fp_verify_drafts";
  if (const int rc = check_shape(what, B, S, V)) return rc;
  const int e = fp::elem_bytes(dtype), pe = draft_probs ? fp::elem_bytes(probs_dtype) : 4;
  if (e == 0 || pe == 0) return fp::fail(FP_ERR_UNSUPPORTED, "%s: dtype code %d", what, e == 0 ? dtype : probs_dtype);
  if (!one_launch(B, S, V, 16 / e)) return too_many(what, B, S, V);
  if (B == 0) return FP_OK;
  if (!logits || !tokens || !parents || !uniforms || !accepted || !path || !answer || !logprobs)
    return fp::fail(FP_ERR_INVALID_ARGUMENT, "%s: null pointer", what);
  if (!fp::aligned(logits, e) || !fp::aligned(draft_probs, pe))
    return fp::fail(FP_ERR_INVALID_ARGUMENT, "%s: logits and draft_probs must be aligned to their elements", what);
  const Cut rows = rows_cut(B, S, V, 16 / e), draw = draw_cut(B, V, 16 / e);
  const int pieces = pieces_of(V, 16 / e);
  const Layout l = layout_of(B, static_cast<int64_t>(B) * S * rows.chunks, pieces);
  const int64_t needed = workspace_of(B, S, V);
  if (!workspace || workspace_bytes < needed || !fp::aligned(workspace, 16))
    return fp::fail(FP_ERR_WORKSPACE, "%s: workspace of %lld bytes, 16-byte aligned, is needed (got %lld)", what,
                    static_cast<long long>(needed), static_cast<long long>(workspace_bytes));
  char* const ws = static_cast<char*>(workspace);
  const VerifyArgs a{static_cast<const char*>(logits), logits_stride_b * e, logits_stride_s * e, tokens, parents, uniforms, temperatures,
                     static_cast<const char*>(draft_probs), probs_stride_b * pe, probs_stride_s * pe, probs_dtype, accepted, path, answer,
                     logprobs, reinterpret_cast<Part*>(ws + l.parts), reinterpret_cast<Piece*>(ws + l.sums),
                     reinterpret_cast<double*>(ws + l.rests), reinterpret_cast<int*>(ws), B, S, V, rows.chunks, rows.nv * kThreads, draw.chunks,
                     pieces};
  const hipStream_t st = static_cast<hipStream_t>(stream);
  const auto go = [&](auto kernel, int64_t grid) {
    hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>(grid)), dim3(kThreads), 0, st, a);
    return fp::check_launch(what);
  };
  const auto launch = [&](auto element) {
    using E = decltype(element);
    const int64_t grid = static_cast<int64_t>(B) * S * rows.chunks;
    const int rc = rows.nv >= 4 ? go(verify_rows_kernel<E, 4>, grid) : rows.nv == 2 ? go(verify_rows_kernel<E, 2>, grid) : go(verify_rows_kernel<E, 1>, grid);
    // (the second reads what the first writes)
    return rc != FP_OK ? rc : go(verify_walk_kernel<E>, static_cast<int64_t>(B) * draw.chunks);
  };
  return dtype == FP_DTYPE_F32 ? launch(F32{}) : dtype == FP_DTYPE_BF16 ? launch(BF16{}) : launch(F16{});
}
