// Verification of drafted tokens: which of them the target model's distribution lets stand, and the token behind them.
//
//   w_i = exp((x_i - max x) / T), Z = sum of w, x the logits of the row of a token
// From the first token on, a token's children are looked at in rising order; R are the weights of those refused before:
//   child c stands if  u_c (Z - R) < w[token_c]                          (the drafts are given)
//                      u_c q[token_c] Z < w[token_c]                      (the drafts were drawn from q)
// Behind the last that stands one more token is drawn: the first i whose cumulative weight is above u_0 times the total, of
//   w without the refused tokens, or of max(0, w / Z - q).
// Which token that is depends on sums over the whole vocabulary to the last bits: next to the border between two tokens, and with
// 65536 of them there is always one near, sums in 32 bits would answer by the order they are taken in.  Weights and sums are
// in 64 bits, the exponential to 2^-51 (a polynomial; on this GPU as many instructions a second as in 32 bits).
//
// Two launches.  The first has every row's maximum and sum, a chunk a workgroup, from one read of the logits.  In the second every
// workgroup puts the chunks of its request's rows together, walks down the tree and sums the weights of a chunk of the row it ends at; the
// last one of a request draws.  The first launch sets the counters of the second to 0: nothing is kept between calls.
#include "fp_common.h"

#include <math.h>

namespace {

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / 64;
constexpr int kMaxTokens = 64;
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
struct Sums {   // of a chunk of the row that is drawn from
  double left;  // what is drawn from
  double all;   // the weights themselves
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
  Part* parts;   // [B * S, chunks]
  Sums* sums;    // [B, draws]
  int* arrivals;  // [B]
  int B, S, V, chunks, draws;
};

// 2^t for t <= 0 (0 for NaN): t = n + f, 2^f by its Chebyshev interpolation of degree 10 on [-1/2, 1/2], off by 2^-51.
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

__device__ __forceinline__ float heat_of(const VerifyArgs& a, int b) { return a.temperatures ? a.temperatures[b] : 1.f; }

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

// Whether row j of the request is a token that can be reached.
__device__ __forceinline__ bool is_token(int j, int parent) { return j == 0 ? parent == -1 : parent >= 0 && parent < j; }

template <typename T, typename Op>
__device__ __forceinline__ T reduce_lanes(T x, int width, Op op) {
  for (int d = 1; d < width; d <<= 1) x = op(x, __shfl_xor(x, d));
  return x;
}

// ---------------------------------------------------------------------------------------------------------------- rows
template <typename E, int NV>  // vectors a thread
__global__ __launch_bounds__(kThreads) void verify_rows_kernel(const VerifyArgs a) {
  __shared__ float s_peak[kWaves];
  __shared__ int s_best[kWaves];
  __shared__ double s_sum[kWaves];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const uint32_t row = blockIdx.x / static_cast<uint32_t>(a.chunks), b = row / static_cast<uint32_t>(a.S);
  const int c = blockIdx.x - row * a.chunks, j = row - b * a.S;
  if (c == 0 && j == 0 && tid == 0) a.arrivals[b] = 0;
  if (!is_token(j, a.parents[row]) || a.parents[static_cast<int64_t>(b) * a.S] != -1) return;
  const Row<E> r(a.logits + b * a.ls_b + j * a.ls_s, a.V);
  const int v0 = c * (kThreads * NV) + tid;
  v4u x[NV];
#pragma unroll
  for (int k = 0; k < NV; ++k)
    if (v0 + k * kThreads < r.vectors) x[k] = r.load(v0 + k * kThreads);
  // the elements outside the whole 16 bytes: the first chunk's first threads and the last one's next 8
  int extra = -1;
  if (c == 0 && tid < r.head) extra = tid;
  if (c == a.chunks - 1 && tid >= 8 && tid - 8 < r.tail) extra = r.behind() + tid - 8;
  const float loose = extra >= 0 ? r.one(extra) : -INFINITY;
  const float heat = heat_of(a, b);

  float peak = fmaxf(loose, -INFINITY);
#pragma unroll
  for (int k = 0; k < NV; ++k)
    if (v0 + k * kThreads < r.vectors)
#pragma unroll
      for (int i = 0; i < E::kVec; ++i) peak = fmaxf(peak, E::get(x[k], i));
  peak = reduce_lanes(peak, 64, [](float p, float q) { return fmaxf(p, q); });
  if (lane == 0) s_peak[wave] = peak;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kWaves; ++w) peak = fmaxf(peak, s_peak[w]);

  int best = INT32_MAX;
  if (!(heat > 0.f)) {
    if (loose == peak && extra >= 0) best = extra;
#pragma unroll
    for (int k = 0; k < NV; ++k)
      if (v0 + k * kThreads < r.vectors)
#pragma unroll
        for (int i = 0; i < E::kVec; ++i)
          if (E::get(x[k], i) == peak) best = min(best, r.head + (v0 + k * kThreads) * E::kVec + i);
    best = reduce_lanes(best, 64, [](int p, int q) { return min(p, q); });
  }
  double sum = 0.0;
  if (fabsf(peak) < INFINITY) {
    const double rate = kLog2e / (heat > 0.f ? heat : 1.0), top = peak;
    if (extra >= 0) sum = power2((loose - top) * rate);
#pragma unroll
    for (int k = 0; k < NV; ++k)
      if (v0 + k * kThreads < r.vectors)
#pragma unroll
        for (int i = 0; i < E::kVec; ++i) sum += power2((E::get(x[k], i) - top) * rate);
  } else if (peak > 0.f) {  // only infinite logits count
    sum = extra >= 0 && loose == peak;
#pragma unroll
    for (int k = 0; k < NV; ++k)
      if (v0 + k * kThreads < r.vectors)
#pragma unroll
        for (int i = 0; i < E::kVec; ++i) sum += E::get(x[k], i) == peak;
  }
  sum = reduce_lanes(sum, 64, [](double p, double q) { return p + q; });
  if (lane == 0) {
    s_sum[wave] = sum;
    s_best[wave] = best;
  }
  __syncthreads();
  if (tid == 0) {
    for (int w = 1; w < kWaves; ++w) sum += s_sum[w], best = min(best, s_best[w]);
    a.parts[blockIdx.x] = Part{sum, peak, best};
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

// What the row that is drawn from weighs, element by element.
struct Drawn {
  const char* probs;   // of the draft, null: not taken away
  float peak;
  double rate, share;  // share: 1 / Z
};

template <typename E, int NV>
__global__ __launch_bounds__(kThreads) void verify_draw_kernel(const VerifyArgs a) {
  constexpr int kVectors = kThreads * NV, kMarks = kVectors * E::kVec + 2 * 8;
  __shared__ float s_peak[kMaxTokens];
  __shared__ int s_best[kMaxTokens];
  __shared__ double s_total[kMaxTokens];
  __shared__ int64_t s_out[kMaxTokens];             // refused tokens
  __shared__ uint32_t s_mark[(kMarks + 31) / 32];   // of the chunk's elements
  __shared__ int s_node, s_count, s_n_out, s_refused, s_flag, s_place;
  __shared__ double s_sum[kWaves][2];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const uint32_t b = blockIdx.x / static_cast<uint32_t>(a.draws);
  const int c = blockIdx.x - b * a.draws, S = a.S;
  const int64_t first = static_cast<int64_t>(b) * S;
  const bool there = a.parents[first] == -1;
  const float heat = heat_of(a, b);
  const bool greedy = !(heat > 0.f);
  const double rate = kLog2e / (greedy ? 1.0 : heat), slope = 1.0 / (greedy ? 1.0 : heat);

  // every row's maximum and sum: `per` lanes a row
  int per = 64;
  while (per > kThreads / S) per >>= 1;
  for (int j = tid / per; j < S; j += kThreads / per) {
    Part t{0.0, -INFINITY, INT32_MAX};
    if (there && is_token(j, a.parents[first + j])) {
      const Part* const parts = a.parts + (first + j) * a.chunks;
      for (int k = tid % per; k < a.chunks; k += per) {
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
    const float peak = reduce_lanes(t.peak, per, [](float p, float q) { return fmaxf(p, q); });
    const double total = reduce_lanes(t.sum * weight(t.peak, peak, rate), per, [](double p, double q) { return p + q; });
    const int best = reduce_lanes(t.peak == peak ? t.best : INT32_MAX, per, [](int p, int q) { return min(p, q); });
    if (tid % per == 0) {
      s_peak[j] = peak;
      s_total[j] = total;
      s_best[j] = peak == -INFINITY ? -1 : best;
    }
  }
  __syncthreads();

  // the walk down the tree: a token a lane
  if (wave == 0) {
    const int parent = lane < S ? a.parents[first + lane] : -2;
    const int64_t token = lane < S ? a.tokens[first + lane] : -1;
    const float u = lane < S ? a.uniforms[first + lane] : 0.f;
    const bool child = there && lane > 0 && lane < S && parent >= 0 && parent < lane, known = token >= 0 && token < a.V;
    const int at = child ? parent : 0;
    double w = 0.0, q = 0.0;
    float x = -INFINITY;
    if (child && known) {
      x = E::at(a.logits + b * a.ls_b + at * a.ls_s + token * E::kBytes);
      if (a.probs) q = probability(a, a.probs + b * a.ps_b + at * a.ps_s, token);
      w = weight(x, s_peak[at], rate);
    }
    double refused = 0.0;
    bool eldest = true;
    for (int i = 1; i < S; ++i) {  // the siblings before this token: what they weigh, the same token once
      const bool sibling = i < lane && __builtin_amdgcn_readlane(parent, i) == parent;
      const int64_t name = __shfl(token, i);
      const double theirs = __shfl(w, i);
      if (sibling) {
        eldest = false;
        if (name == token) w = 0.0; else refused += theirs;
      }
    }
    const double z = s_total[at];
    const bool takes = child && known && (greedy ? token == s_best[at] : a.probs ? eldest && u * q * z < w : u * (z - refused) < w);
    int node = 0, count = 0, mine = lane == 0 ? 0 : -1;  // mine: the lane-th of the path
    if (there) {
      for (;;) {
        const uint64_t stand = __ballot(takes && parent == node);
        if (stand == 0) break;
        node = __builtin_ctzll(stand);
        ++count;
        if (lane == count) mine = node;
      }
    }
    const uint64_t out = __ballot(child && known && parent == node);
    if (child && known && parent == node) s_out[__builtin_popcountll(out & ((1ull << lane) - 1))] = token;
    const bool any = __ballot(child && parent == node) != 0;
    if (lane == 0) {
      s_node = node;
      s_count = count;
      s_n_out = __builtin_popcountll(out);
      s_refused = any;
    }
    if (c == 0) {
      // the token of path[lane + 1] answers at place lane; the last place is the drawn one's
      const int next = __shfl_down(mine, 1);
      const int from = lane < count ? next : 0;
      const int64_t name = __shfl(token, from);
      const float its = __shfl(x, from);
      const int under = __shfl(at, from);
      if (lane < S) {
        a.path[first + lane] = there ? mine : -1;
        if (lane != count || !there) {
          const bool says = there && lane < count;
          a.answer[first + lane] = says ? name : -1;
          const float peak = s_peak[under];
          a.logprobs[first + lane] = says ? static_cast<float>((its == peak ? 0.0 : (static_cast<double>(its) - peak) * slope) - log(s_total[under])) : 0.f;
        }
      }
      if (lane == 0) a.accepted[b] = count;
    }
  }
  __syncthreads();
  if (!there) return;
  const int node = s_node, count = s_count;
  const Row<E> r(a.logits + b * a.ls_b + node * a.ls_s, a.V);
  const auto answer = [&](int64_t token) {
    a.answer[first + count] = token;
    float says = 0.f;
    if (token >= 0) {
      const float x = r.one(token), peak = s_peak[node];
      says = static_cast<float>((x == peak ? 0.0 : (static_cast<double>(x) - peak) * slope) - log(s_total[node]));
    }
    a.logprobs[first + count] = says;
  };
  if (greedy || s_peak[node] == -INFINITY) {
    if (c == 0 && tid == 0) answer(s_best[node]);
    return;
  }

  const Drawn drawn{a.probs && s_refused ? a.probs + b * a.ps_b + node * a.ps_s : nullptr, s_peak[node], rate, 1.0 / s_total[node]};
  const int n_out = a.probs ? 0 : s_n_out;
  // Marks of the refused tokens among the elements of a chunk: those in front of the whole 16 bytes have the first 8 places, those behind
  // them the next 8.
  const auto mark = [&](int chunk) {
    if (n_out == 0) return;
    __syncthreads();
    for (int i = tid; i < (kMarks + 31) / 32; i += kThreads) s_mark[i] = 0;
    __syncthreads();
    if (tid < n_out) {
      const int64_t t = s_out[tid], inside = t - r.head - static_cast<int64_t>(chunk) * kVectors * E::kVec;
      int place = -1;
      if (t < r.head)
        place = chunk == 0 ? static_cast<int>(t) : -1;
      else if (t >= r.behind())
        place = chunk == a.draws - 1 ? static_cast<int>(8 + t - r.behind()) : -1;
      else if (inside >= 0 && inside < kVectors * E::kVec)
        place = static_cast<int>(16 + inside);
      if (place >= 0) atomicOr(&s_mark[place >> 5], 1u << (place & 31));
    }
    __syncthreads();
  };
  const auto marked = [&](int place) { return n_out > 0 && (s_mark[place >> 5] >> (place & 31) & 1); };
  // weight of element i of the row, whose place among the marks is given
  const auto left_of = [&](float x, int64_t i, int place, bool take_away) {
    if (marked(place)) return 0.0;
    const double w = weight(x, drawn.peak, drawn.rate);
    return take_away ? fmax(0.0, w * drawn.share - static_cast<double>(probability(a, drawn.probs, i))) : w;
  };

  mark(c);
  {
    double left = 0.0, all = 0.0;
    const auto add = [&](float x, int64_t i, int place) {
      const double w = left_of(x, i, place, false);
      all += w;
      if (drawn.probs) left += fmax(0.0, w * drawn.share - static_cast<double>(probability(a, drawn.probs, i)));
    };
    v4u x[NV];
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const int v = c * kVectors + k * kThreads + tid;
      if (v < r.vectors) x[k] = r.load(v);
    }
    if (c == 0 && tid < r.head) add(r.one(tid), tid, tid);
    if (c == a.draws - 1 && tid >= 8 && tid - 8 < r.tail) add(r.one(r.behind() + tid - 8), r.behind() + tid - 8, tid);
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const int v = c * kVectors + k * kThreads + tid;
      if (v < r.vectors)
#pragma unroll
        for (int i = 0; i < E::kVec; ++i)
          add(E::get(x[k], i), r.head + static_cast<int64_t>(v) * E::kVec + i, 16 + (k * kThreads + tid) * E::kVec + i);
    }
    const auto plus = [](double p, double q) { return p + q; };
    all = reduce_lanes(all, 64, plus);
    left = reduce_lanes(left, 64, plus);
    if (lane == 0) s_sum[wave][0] = drawn.probs ? left : all, s_sum[wave][1] = all;
    __syncthreads();
    if (tid == 0) {
      Sums* const to = a.sums + static_cast<int64_t>(b) * a.draws + c;
      publish(&to->left, s_sum[0][0] + s_sum[1][0] + s_sum[2][0] + s_sum[3][0]);
      publish(&to->all, s_sum[0][1] + s_sum[1][1] + s_sum[2][1] + s_sum[3][1]);
      asm volatile("s_waitcnt vmcnt(0)" : : : "memory");  // they have arrived before the count does
      s_flag = __hip_atomic_fetch_add(a.arrivals + b, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == a.draws - 1;
    }
    __syncthreads();
    if (!s_flag) return;
  }

  // The last workgroup of the request: the chunk in which the cumulative weight passes u_0 times the total, by one wavefront
  __shared__ int s_chunk, s_all;
  __shared__ double s_before, s_goal;
  if (wave == 0) {
    const Sums* const sums = a.sums + static_cast<int64_t>(b) * a.draws;
    double left = 0.0, all = 0.0;
    for (int k = lane; k < a.draws; k += 64) left += take(&sums[k].left), all += take(&sums[k].all);
    const auto plus = [](double p, double q) { return p + q; };
    left = reduce_lanes(left, 64, plus);
    all = reduce_lanes(all, 64, plus);
    const bool whole = !(left > 0.0);  // nothing is left: the target's own distribution
    const float u = a.uniforms[first];
    const double goal = (u < 0.f ? 0.0 : static_cast<double>(u)) * (whole ? all : left);  // (NaN passes nothing: the last token)
    double before = 0.0;
    int chunk = -1, last = -1;
    double before_last = 0.0;
    for (int k0 = 0; k0 < a.draws && chunk < 0; k0 += 64) {
      const int k = k0 + lane;
      const double s = k < a.draws ? take(whole ? &sums[k].all : &sums[k].left) : 0.0;
      double upto = s;
#pragma unroll
      for (int d = 1; d < 64; d <<= 1) {
        const double y = __shfl_up(upto, d);
        if (lane >= d) upto += y;
      }
      const uint64_t past = __ballot(before + upto > goal), some = __ballot(s > 0.0);
      if (past) {
        const int l = __builtin_ctzll(past);
        chunk = k0 + l;
        before += __shfl(upto - s, l);
      } else {
        if (some) {
          const int l = 63 - __builtin_clzll(some);
          last = k0 + l;
          before_last = before + __shfl(upto - s, l);
        }
        before += __shfl(upto, 63);
      }
    }
    if (lane == 0) {
      s_chunk = chunk >= 0 ? chunk : last;
      s_before = chunk >= 0 ? before : before_last;
      s_goal = goal;
      s_all = whole;
      s_place = -1;
    }
  }
  __syncthreads();
  const int chunk = s_chunk;
  if (chunk < 0) {  // every token is refused
    if (tid == 0) answer(-1);
    return;
  }
  const bool take_away = drawn.probs && !s_all;
  mark(chunk);
  // its elements in order, a segment at a time: those in front, the vectors by rows of threads, those behind
  double before = s_before;
  const double goal = s_goal;
  int last = -1;  // of this thread's elements, the last that weighs something
  for (int seg = 0; seg < NV + 2; ++seg) {
    int n = 0, place = 0;
    int64_t i0 = 0;
    float x[E::kVec];
    if (seg == 0) {
      if (chunk == 0 && tid < r.head) n = 1, i0 = tid, place = tid;
    } else if (seg == NV + 1) {
      if (chunk == a.draws - 1 && tid < r.tail) n = 1, i0 = r.behind() + tid, place = 8 + tid;
    } else {
      const int v = chunk * kVectors + (seg - 1) * kThreads + tid;
      if (v < r.vectors) n = E::kVec, i0 = r.head + static_cast<int64_t>(v) * E::kVec, place = 16 + ((seg - 1) * kThreads + tid) * E::kVec;
    }
    double w[E::kVec], sum = 0.0;
    if (n == 1) x[0] = r.one(i0);
    if (n > 1) {
      const v4u all = *reinterpret_cast<const v4u*>(r.at + i0 * E::kBytes);
#pragma unroll
      for (int i = 0; i < E::kVec; ++i) x[i] = E::get(all, i);
    }
#pragma unroll
    for (int i = 0; i < E::kVec; ++i) {
      w[i] = i < n ? left_of(x[i], i0 + i, place + i, take_away) : 0.0;
      sum += w[i];
      if (w[i] > 0.0) last = static_cast<int>(i0 + i);
    }
    double upto = sum;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const double y = __shfl_up(upto, d);
      if (lane >= d) upto += y;
    }
    __syncthreads();  // the segment before has been read
    if (lane == 63) s_sum[wave][0] = upto;
    __syncthreads();
    double ahead = before;
    for (int k = 0; k < wave; ++k) ahead += s_sum[k][0];
    for (int k = 0; k < kWaves; ++k) before += s_sum[k][0];
    // the thread in which the weight passes the goal: the first one whose elements reach beyond it
    double at = ahead + (upto - sum);
    if (sum > 0.0 && at + sum > goal) {
      int found = -1;
#pragma unroll
      for (int i = 0; i < E::kVec; ++i) {
        at += w[i];
        if (found < 0 && w[i] > 0.0 && at > goal) found = static_cast<int>(i0 + i);
      }
      if (found >= 0) atomicMin(reinterpret_cast<uint32_t*>(&s_place), static_cast<uint32_t>(found));
    }
    __syncthreads();
    if (s_place >= 0) break;
  }
  if (s_place < 0) {  // u_0 at the very end: the last token that weighs something
    last = reduce_lanes(last, 64, [](int p, int q) { return max(p, q); });
    __syncthreads();
    if (lane == 0) atomicMax(&s_place, last);
    __syncthreads();
  }
  if (tid == 0) answer(s_place);
}

struct Cut {
  int nv, chunks;
};
// Vectors a thread: as many as leave `wanted` workgroups, 8 (rows) or 4 (draws) at most.
Cut cut_of(int64_t rows, int V, int vec, int most, int64_t wanted) {
  const int64_t vectors = (static_cast<int64_t>(V) + vec - 1) / vec;
  Cut c{most, 0};
  for (;; c.nv /= 2) {
    c.chunks = static_cast<int>((vectors + kThreads * c.nv - 1) / (kThreads * c.nv));
    if (c.nv == 1 || rows * c.chunks >= wanted) return c;
  }
}
Cut rows_cut(int B, int S, int V, int vec) { return cut_of(static_cast<int64_t>(B) * S, V, vec, 8, 4ll * fp::compute_units()); }
Cut draw_cut(int B, int V, int vec) { return cut_of(B, V, vec, 4, 2ll * fp::compute_units()); }

int check_shape(const char* what, int B, int S, int V) {
  if (B < 0 || S <= 0 || V <= 0) return fp::fail(FP_ERR_INVALID_ARGUMENT, "%s: bad sizes (B=%d S=%d V=%d)", what, B, S, V);
  if (S > kMaxTokens || V > 1 << 24)
    return fp::fail(FP_ERR_UNSUPPORTED, "%s: at most %d tokens a request and a vocabulary of %d (got %d and %d)", what, kMaxTokens, 1 << 24, S, V);
  // one launch of workgroups of a chunk of a row each
  if (static_cast<int64_t>(B) * S * ((V + kThreads * 4ll - 1) / (kThreads * 4)) > INT32_MAX)
    return fp::fail(FP_ERR_UNSUPPORTED, "%s: %d requests of %d rows of %d logits are too many for one call", what, B, S, V);
  return FP_OK;
}

struct Layout {
  int64_t parts, sums, bytes;
};
Layout layout_of(int B, int S, int64_t chunks, int64_t draws) {
  Layout l;
  l.parts = (static_cast<int64_t>(B) * 4 + 15) / 16 * 16;
  l.sums = l.parts + static_cast<int64_t>(B) * S * chunks * sizeof(Part);
  l.bytes = l.sums + B * draws * static_cast<int64_t>(sizeof(Sums));
  return l;
}

}  // namespace

extern "C" int64_t fp_verify_drafts_workspace_bytes(int32_t B, int32_t S, int32_t V) {
  if (const int rc = check_shape("fp_verify_drafts_workspace_bytes", B, S, V)) return rc;
  int64_t most = 0;
  for (const int vec : {4, 8}) {
    const int64_t n = layout_of(B, S, rows_cut(B, S, V, vec).chunks, draw_cut(B, V, vec).chunks).bytes;
    most = n > most ? n : most;
  }
  return most;
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
  if (B == 0) return FP_OK;
  if (!logits || !tokens || !parents || !uniforms || !accepted || !path || !answer || !logprobs)
    return fp::fail(FP_ERR_INVALID_ARGUMENT, "%s: null pointer", what);
  if (!fp::aligned(logits, e) || !fp::aligned(draft_probs, pe))
    return fp::fail(FP_ERR_INVALID_ARGUMENT, "%s: logits and draft_probs must be aligned to their elements", what);
  const Cut rows = rows_cut(B, S, V, 16 / e), draw = draw_cut(B, V, 16 / e);
  const Layout l = layout_of(B, S, rows.chunks, draw.chunks);
  if (!workspace || workspace_bytes < l.bytes || !fp::aligned(workspace, 16))
    return fp::fail(FP_ERR_WORKSPACE, "%s: workspace of %lld bytes, 16-byte aligned, is needed (got %lld)", what,
                    static_cast<long long>(l.bytes), static_cast<long long>(workspace_bytes));
  char* const ws = static_cast<char*>(workspace);
  const VerifyArgs a{static_cast<const char*>(logits), logits_stride_b * e, logits_stride_s * e, tokens, parents, uniforms, temperatures,
                     static_cast<const char*>(draft_probs), probs_stride_b * pe, probs_stride_s * pe, probs_dtype, accepted, path, answer,
                     logprobs, reinterpret_cast<Part*>(ws + l.parts), reinterpret_cast<Sums*>(ws + l.sums), reinterpret_cast<int*>(ws), B, S, V,
                     rows.chunks, draw.chunks};
  const hipStream_t st = static_cast<hipStream_t>(stream);
  const auto go = [&](auto kernel, int64_t grid) {
    hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>(grid)), dim3(kThreads), 0, st, a);
  };
  const auto launch = [&](auto element) {
    using E = decltype(element);
    const int64_t grid = static_cast<int64_t>(B) * S * rows.chunks;
    switch (rows.nv) {
      case 8: go(verify_rows_kernel<E, 8>, grid); break;
      case 4: go(verify_rows_kernel<E, 4>, grid); break;
      case 2: go(verify_rows_kernel<E, 2>, grid); break;
      default: go(verify_rows_kernel<E, 1>, grid);
    }
    const int64_t draws = static_cast<int64_t>(B) * draw.chunks;
    switch (draw.nv) {
      case 4: go(verify_draw_kernel<E, 4>, draws); break;
      case 2: go(verify_draw_kernel<E, 2>, draws); break;
      default: go(verify_draw_kernel<E, 1>, draws);
    }
  };
  if (dtype == FP_DTYPE_F32)
    launch(F32{});
  else if (dtype == FP_DTYPE_BF16)
    launch(BF16{});
  else
    launch(F16{});
  return fp::check_launch(what);
}
