// Attention of a batch's newest tokens over the paged cache, where sequences of the batch begin with the same keys.
//
//   out[b, h, j] = sum over t <= p of softmax_t(scale q.k_t) v_t,   p = input_pos[b, j]
// The softmax over a sequence's keys is two: over the prefix that its group shares and over the keys behind it, joined by
// their maxima and sums.  Over the prefix all rows of the group - its sequences' tokens times the query heads of a cached
// head - are the columns of one matrix product, so that a shared key is read once for up to 64 rows, not once a sequence.
//
// Three launches: the plan once per step, then for every layer the products and the join.
//  * Plan (one workgroup): finds the groups, leaves out members whose prefix is too short, and makes tiles of up to 64 rows over
//    one range of keys: the prefix of a group by its rows, the keys behind it by the rows of one sequence.  The tiles' keys, in units of 64, are laid end to end and
//    cut evenly over two workgroups a CU, so a workgroup streams the same number of keys whatever the lengths are; a tile
//    that a cut goes through leaves a partial result for each of its pieces.
//  * Products: a workgroup of 4 wavefronts takes the pieces of its cut, one cached head.  The wavefronts have the same rows
//    and take the stages of keys in turn, each from a ring of its own in LDS that global_load_lds fills, without a barrier:
//      S^T = K Q^T    keys are the M rows of the matrix product and queries its columns, so a lane has the scores of
//                     one query and a K operand read from LDS serves up to four blocks of 16 columns
//      O^T += V^T P^T  P^T is in the B operand's layout as the scores leave the first product; V^T comes out of LDS
//                     through the transpose read (fp32: by reading four neighbours of a row for four blocks of O^T).
//                     Of 16-bit types a probability is the sum of two numbers of the type, which one product of depth 32
//                     takes against 16 keys twice: rounded once to 16 bits they cost f16 most of its precision
//    The states of the four wavefronts meet in LDS at the end of a piece.
//  * Join: a row's pieces, by their maxima and sums, in 32 bits.
//
// Bound by HBM where the keys are many.  64 sequences, most on one of 9 prefixes, 16 query heads on 8 cached ones, D 128, bf16, 473 MB a
// layer: products 81.5 us (5.8 TB/s; a large copy reaches 5.2 on this GPU), join 5.0, plan 10.9 once a step; fp_paged_decode, which
// reads a prefix once a sequence, takes 141.  192 sequences on 8 prefixes of up to 12288 keys, 4 query heads a cached one, 2.0 GB a layer:
// 330 us, 6.0 TB/s (1153 once a sequence).  Small batches are bound by the trips to memory in front of the first key and by two
// launches (3 sequences, 1.5 MB: 8.9 and 4.1 us), many tokens a sequence by LDS and the instructions between the matrix products
// (40 sequences of 24 tokens, 11.6 GFLOP: 46 us).
#include "decode_common.h"

#include <math.h>

namespace {

using fp_decode::fast_exp2;
using fp_decode::kLn2;
using fp_decode::kLog2e;
using fp_decode::safe_max;

// The sink gate (model.py:122-128) in 32 bits: the product is rounded once, when it is stored.
__device__ __forceinline__ float gated(float o, float lse, const float* sinks, int h) {
  return sinks == nullptr ? o : o / (1.f + __expf(sinks[h] - lse));
}

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / 64;
constexpr int kMaxSequences = 1536;
constexpr int kMaxRows = 1 << 20;      // B * S * heads of a group
constexpr int kMaxContext = 1 << 21;   // with the rows: units of all tiles fit 31 bits
constexpr int kTileRows = 64;
constexpr int kUnit = 64;              // keys: what the cut is made of
constexpr int kMinUnits = 3;           // a workgroup's share at least
constexpr int kSegPages = 1024;        // page ids held in LDS
constexpr float kMaxSlack = 6.f;       // the reference point of the exponentials may lag the maximum by this much (log2)
constexpr int kMagic = 0x5ade0001;

typedef uint32_t v4u __attribute__((ext_vector_type(4)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef short s16x4 __attribute__((ext_vector_type(4)));

// ------------------------------------------------------------------------------------------------------------ plan
// ints: header, sequences, tokens of the groups and of the other sequences, each token's place, workgroups, tiles
struct Header {
  int magic, B, S, Hq, Hc, max_batch, max_context;
  int n_wg;     // workgroups that have a share
  int n_tiles;
  int pad[7];
};
struct Sequence {
  int slot, keys;      // -1: not a slot; keys any of its tokens sees
  int prefix_tile;     // first tile of its group, -1: shares with nobody
  int prefix_row;      // its first row among the group's
  int own_tile;        // first tile of the keys behind the prefix, -1: none
  int pad[3];
  // one token a sequence: workspace row of its first head, rows from piece to piece, pieces; of the prefix and of its own keys.  The
  // join has them with this record instead of a trip to memory later (4.5 -> 4.3 us a layer).
  int at, step, n, own_at, own_step, own_n;
  int pad2[2];
};
struct Tile {
  int slot;            // row of the page table
  int base;            // place of its group's or sequence's first token in the list
  int row0, n_rows;    // of the group's or the sequence's rows
  int t_begin, t_end;  // keys
  int n_pieces;
  int part;            // workspace row of the first piece's first row; piece after piece
  int shared;          // of a group
  int lead;            // units that stand for what it costs before its first key and behind its last
  int again;           // other tiles read the same keys
  int next;            // the tile behind it on the axis that it is cut on
};
struct Share {
  int tile, offset, units;  // first tile, units of it (lead included) that belong to workgroups before, units to do
  int piece;                // of the first tile; the others begin here
  Tile first;               // the first tile itself: a trip to memory less
};

struct Layout {
  int n_wg, max_tiles, rows;  // rows: of a sequence and cached head
  int64_t seqs, tokens, place, shares, tiles, bytes;  // byte offsets
  int64_t part_rows;
};

Layout layout_of(int B, int S, int Hq, int Hc) {
  Layout l;
  l.n_wg = 2 * fp::compute_units() / Hc;
  if (l.n_wg < 1) l.n_wg = 1;
  l.rows = S * (Hq / Hc);
  // ceil(rows / 64) summed over groups of two or more; every sequence's own
  l.max_tiles = static_cast<int>(static_cast<int64_t>(B) * l.rows / kTileRows + B / 2 + 1 +
                                 static_cast<int64_t>(B) * ((l.rows + kTileRows - 1) / kTileRows));
  const int64_t list = (static_cast<int64_t>(B) * S * 4 + 15) / 16 * 16;
  l.seqs = sizeof(Header);
  l.tokens = l.seqs + static_cast<int64_t>(B) * sizeof(Sequence);
  l.place = l.tokens + list;
  l.shares = l.place + list;
  l.tiles = l.shares + static_cast<int64_t>(l.n_wg) * sizeof(Share);
  l.bytes = l.tiles + static_cast<int64_t>(l.max_tiles) * sizeof(Tile);
  l.part_rows = 4ll * B * l.rows + static_cast<int64_t>(kTileRows) * l.n_wg;
  return l;
}

// A token of the lists: sequence and place in it (kMaxSequences and kMaxRows bound both).
constexpr int kTokenShift = 20;
static_assert(kMaxSequences <= 1 << (31 - kTokenShift) && kMaxRows <= 1 << kTokenShift, "a token is one int");

struct PlanArgs {
  const int64_t* batch_idx;
  const void* input_pos;
  int pos_i64;
  const int32_t* ids;
  const int32_t* lens;
  int B, S, Hq, Hc, group, max_batch, max_context, n_wg;
  char* plan;
  int64_t seqs, tokens, place, shares, tiles;
};

// What a tile costs before its first key and behind its last, in units.
__device__ __forceinline__ int lead_of(int rows) { return rows <= 16 ? 2 : rows <= 32 ? 3 : 6; }

__device__ __forceinline__ int units_of(int keys) { return (keys + kUnit - 1) / kUnit; }

// last i of 0 .. n - 1 with at[i] <= x (at[0] is 0)
__device__ __forceinline__ int last_at_or_below(const int* at, int n, int x) {
  int lo = 0, hi = n - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (at[mid] <= x) lo = mid; else hi = mid - 1;
  }
  return lo;
}

// keys that token j of sequence b sees, 0: no token
__device__ __forceinline__ int plan_keys(const PlanArgs& a, int b, int j) {
  const int64_t p = fp::load_index(a.input_pos, static_cast<int64_t>(b) * a.S + j, a.pos_i64) + 1;
  return p < 0 ? 0 : p > a.max_context ? a.max_context : static_cast<int>(p);
}

// Sums over the threads before this one and over all, of N numbers a thread.
template <int N>
__device__ __forceinline__ void block_sums(const int (&x)[N], int (&before)[N], int (&total)[N], int* s_sum) {
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), n_waves = blockDim.x >> 6;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const int up = fp_decode::scan_lanes(x[i]);
    if (lane == 63) s_sum[wave * N + i] = up;
    before[i] = up - x[i];
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < N; ++i) {  // the wavefronts' sums, one a lane
    const int y = lane < n_waves ? s_sum[lane * N + i] : 0, up = fp_decode::scan_lanes(y);
    total[i] = __builtin_amdgcn_readlane(up, 63);
    before[i] += __builtin_amdgcn_readlane(up, wave) - __builtin_amdgcn_readlane(y, wave);
  }
  __syncthreads();
}

constexpr int kPlanArrays = 23;

__global__ __launch_bounds__(1024) void shared_plan_kernel(const PlanArgs a) {
  extern __shared__ int s_mem[];
  const int Bp = (a.B + 3) & ~3;
  int* const s_id = s_mem;             // prefix id, 0: none
  int* const s_keys = s_id + Bp;       // keys the sequence's tokens see
  int* const s_len = s_keys + Bp;      // its prefix length
  int* const s_tok = s_len + Bp;       // its tokens
  int* const s_shared = s_tok + Bp;    // shared keys of its group, 0: none
  int* const s_count = s_shared + Bp;  // tokens of the group, at its first sequence (its leader), elsewhere 0
  int* const s_rank = s_count + Bp;    // tokens of the members before
  int* const s_lead = s_rank + Bp;
  int* const s_slot = s_lead + Bp;
  int* const s_ptile = s_slot + Bp;    // sums over the sequences before: tiles of prefixes,
  int* const s_base = s_ptile + Bp;    //   tokens of groups or of sequences that share nothing: place in the list
  int* const s_stile = s_base + Bp;    //   tiles of own keys,
  int* const s_unit = s_stile + Bp;    //   units of prefixes that are cut with everything else,
  int* const s_own = s_unit + Bp;      //   units of own keys,
  int* const s_wide = s_own + Bp;      // place of a group of several tiles in the lists of these:
  int* const s_at = s_wide + Bp;       //   its first sequence,
  int* const s_n = s_at + Bp;          //   its tiles,
  int* const s_u = s_n + Bp;           //   units of each, with the lead
  int* const s_lu = s_u + Bp;          //   the lead,
  int* const s_pos = s_lu + Bp;        //   its place on the axis of its kind,
  int* const s_end = s_pos + Bp;       //   length of that axis, at the first of a kind, elsewhere 0,
  int* const s_next = s_end + Bp;      //   the next of its kind, -1: none,
  int* const s_part = s_next + Bp;     //   pieces of the groups before
  __shared__ int s_sum[16 * 7], s_pick[1], s_turn[2];
  const int tid = threadIdx.x, n_thr = blockDim.x, lane = tid & 63, wave = tid >> 6, n_waves = n_thr / 64;
  Sequence* const seqs = reinterpret_cast<Sequence*>(a.plan + a.seqs);
  // until the sums below, these three hold a group's sequences, shortest prefix length and most keys, at its first sequence
  int* const s_members = s_ptile;
  int* const s_shortest = s_base;
  int* const s_longest = s_stile;
  // and these its longest prefix length, the most units that a length spares, and that length
  int* const s_furthest = s_unit;
  int* const s_best = s_own;
  int* const s_cut = s_wide;
  for (int b = tid; b < Bp; b += n_thr) {
    const int64_t slot = b < a.B ? a.batch_idx[b] : -1;
    const bool valid = slot >= 0 && slot < a.max_batch;
    const int keys = a.S == 1 && valid ? plan_keys(a, b, 0) : 0;
    const int id = valid ? max(a.ids[slot], 0) : 0, length = valid ? max(a.lens[slot], 0) : 0;
    s_id[b] = length >= kUnit ? id : 0;
    s_len[b] = length;
    s_keys[b] = keys;
    s_tok[b] = keys > 0;
    s_slot[b] = valid ? static_cast<int>(slot) : -1;
    s_lead[b] = b;
    s_rank[b] = s_count[b] = s_members[b] = s_longest[b] = s_furthest[b] = 0;
    s_shortest[b] = INT32_MAX;
  }
  if (tid < 2) s_turn[tid] = 0;
  __syncthreads();
  if (a.S > 1) {
    for (int i = tid; i < a.B * a.S; i += n_thr) {
      const int b = static_cast<uint32_t>(i) / static_cast<uint32_t>(a.S), keys = s_slot[b] < 0 ? 0 : plan_keys(a, b, i - b * a.S);
      if (keys > 0) {
        atomicMax(&s_keys[b], keys);
        atomicAdd(&s_tok[b], 1);
      }
    }
    __syncthreads();
  }

  // Groups.  The first sequence with the same id leads, and a sequence's place is behind the tokens of those before it: sequences
  // look at all before them, four at a time, some threads a sequence.  A sequence without a token belongs to no group.
  const auto usable = [&](int b) { return min(s_len[b], s_longest[s_lead[b]]) / kUnit; };  // units of its prefix
  const auto mixed = [&](int lead) {
    return s_members[lead] > 2 && min(s_shortest[lead], s_longest[lead]) / kUnit < min(s_furthest[lead], s_longest[lead]) / kUnit;
  };
  for (int turn = 0;; ++turn) {
    const int wide = (a.B + 63) & ~63, parts = max(1, n_thr / wide), part = tid / wide;
    const int quads = (Bp / 4 + parts - 1) / parts;  // that a thread looks at
    for (int b = parts > 1 ? tid - part * wide : tid; b < a.B && part < parts; b += n_thr) {
      const int id = s_tok[b] > 0 ? s_id[b] : 0;
      if (id == 0) continue;
      int lead = b, rank = 0;
      const int from = parts > 1 ? part * quads * 4 : 0, to = min(b, from + quads * 4);
      for (int j = from; j < to; j += 4) {
        const i32x4 ids = *reinterpret_cast<const i32x4*>(s_id + j), toks = *reinterpret_cast<const i32x4*>(s_tok + j);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int tokens = ids[i] == id && j + i < b ? toks[i] : 0;
          rank += tokens;
          lead = min(lead, tokens > 0 ? j + i : b);
        }
      }
      if (lead < b) atomicMin(&s_lead[b], lead);
      if (rank > 0) atomicAdd(&s_rank[b], rank);
    }
    __syncthreads();
    for (int b = tid; b < a.B; b += n_thr) {
      if (s_id[b] == 0 || s_tok[b] == 0) continue;
      const int lead = s_lead[b];
      atomicAdd(&s_count[lead], s_tok[b]);
      atomicAdd(&s_members[lead], 1);
      atomicMin(&s_shortest[lead], s_len[b]);
      atomicMax(&s_furthest[lead], s_len[b]);
      atomicMax(&s_longest[lead], s_keys[b]);
    }
    __syncthreads();
    for (int b = tid; b < a.B; b += n_thr) {
      // Whole units: what is behind them counts as each one's own, up to 63 keys that are read once a sequence.  Own keys then begin
      // with a stage that lies in one page; from anywhere else they would be staged row by row (64 sequences on 9 pictures: 86 us a
      // layer instead of 82).
      const int lead = s_lead[b], members = s_members[lead], shortest = s_shortest[lead], longest = s_longest[lead], furthest = s_furthest[lead];
      const int shared = members >= 2 ? min(shortest, longest) / kUnit * kUnit : 0;
      const bool shares = s_tok[b] > 0 && s_id[b] > 0 && shared > 0;
      s_shared[b] = shares ? shared : 0;
      if (!shares) s_rank[b] = 0;
      if (!shares || lead != b) s_count[b] = 0;
      if (turn == 0 && members > 2 && shared < min(furthest, longest) / kUnit * kUnit) s_turn[0] = 1;
    }
    __syncthreads();
    if (__builtin_expect(turn == 1 || s_turn[0] == 0, 1)) break;

    // The shortest prefix length is what all of a group share.  Where lengths differ, those take part whose length is at least the
    // one that spares most keys, length * (members of that length or more - 1), and the others share with nobody: a single short one
    // would leave the others little or nothing.  The members of such groups, sorted by leader and length, say how many there are; the second
    // turn makes the groups without those that were left out.  (The plan of 128 sequences of four groups: 11.8 us where lengths are alike,
    // 21.2 where a fifth of them is short; of 1536 282 and 518.)
    int* const s_sorted = s_n;  // as many as the next power of two, below 2 B, of the 7 B behind it
    int n_sort = 1;
    while (n_sort < a.B) n_sort *= 2;
    const auto of_mixed = [&](int b) { return s_id[b] > 0 && s_tok[b] > 0 && mixed(s_lead[b]); };
    constexpr int kLengthBits = 16;
    static_assert(kMaxContext / kUnit < 1 << kLengthBits && kMaxSequences < 1 << (31 - kLengthBits), "leader and length are one int");
    for (int b = tid; b < a.B; b += n_thr) {
      s_best[b] = 0;
      s_cut[b] = INT32_MAX;
    }
    for (int i = tid; i < n_sort; i += n_thr) s_sorted[i] = i < a.B && of_mixed(i) ? s_lead[i] << kLengthBits | usable(i) : INT32_MAX;
    __syncthreads();
    for (int k = 2; k <= n_sort; k *= 2)
      for (int j = k / 2; j > 0; j /= 2) {
        for (int i = tid; i < n_sort; i += n_thr) {
          const int at = i ^ j;
          if (at < i) continue;
          const int x = s_sorted[i], y = s_sorted[at];
          if ((x > y) == ((i & k) == 0)) {
            s_sorted[i] = y;
            s_sorted[at] = x;
          }
        }
        __syncthreads();
      }
    const auto spared = [&](int i, int* lead, int* units) {  // by the length at place i
      *lead = s_sorted[i] >> kLengthBits, *units = s_sorted[i] & ((1 << kLengthBits) - 1);
      int begin = 0, end = i;  // the leader's first place
      while (begin < end) {
        const int mid = (begin + end) >> 1;
        if (s_sorted[mid] >= *lead << kLengthBits) end = mid; else begin = mid + 1;
      }
      return *units * (begin + s_members[*lead] - i - 1);
    };
    int lead, units;
    for (int i = tid; i < a.B; i += n_thr)
      if (s_sorted[i] != INT32_MAX) {
        const int keys = spared(i, &lead, &units);
        atomicMax(&s_best[lead], keys);
      }
    __syncthreads();
    for (int i = tid; i < a.B; i += n_thr)
      if (s_sorted[i] != INT32_MAX && spared(i, &lead, &units) == s_best[lead]) atomicMin(&s_cut[lead], units);
    __syncthreads();
    for (int b = tid; b < a.B; b += n_thr)
      if (of_mixed(b) && usable(b) < s_cut[s_lead[b]]) {
        s_id[b] = 0;
        s_turn[1] = 1;
      }
    __syncthreads();
    if (s_turn[1] == 0) break;
    for (int b = tid; b < a.B; b += n_thr) {
      s_lead[b] = b;
      s_rank[b] = s_count[b] = s_members[b] = s_longest[b] = s_furthest[b] = 0;
      s_shortest[b] = INT32_MAX;
    }
    __syncthreads();
  }

  const auto lead_for = [&](int tokens) { return lead_of(tokens * a.group); };
  const auto tiles_of = [&](int tokens) { return (tokens * a.group + kTileRows - 1) / kTileRows; };
  // sums over the sequences before, consecutive ones a thread
  const int per = (a.B + n_thr - 1) / n_thr, b0 = min(a.B, tid * per), b1 = min(a.B, b0 + per);
  int x[7] = {0, 0, 0, 0, 0, 0, 0}, before[7], total[7];
  const auto add = [&](int b) {
    const int c = s_count[b], own = s_keys[b] - s_shared[b];
    if (c > 0) {
      x[0] += tiles_of(c);
      x[1] += c;
      x[4] += tiles_of(c) * (lead_for(c) + units_of(s_shared[b]));
      x[5] += tiles_of(c) > 1;
    }
    if (own > 0) {
      x[2] += tiles_of(s_tok[b]);
      x[4] += tiles_of(s_tok[b]) * (lead_for(s_tok[b]) + units_of(own));
    }
    if (s_shared[b] == 0) x[3] += s_tok[b];
    x[6] += s_tok[b];
  };
  for (int b = b0; b < b1; ++b) add(b);
  block_sums(x, before, total, s_sum);
  const int p_tiles = total[0], n_tiles = p_tiles + total[2], shared_tokens = total[1], n_multi = total[5], all_units = total[4];
#pragma unroll
  for (int i = 0; i < 7; ++i) x[i] = before[i];
  for (int b = b0; b < b1; ++b) {
    s_ptile[b] = x[0];
    s_base[b] = s_shared[b] > 0 ? x[1] : shared_tokens + x[3];  // of a group: right at its leader
    s_stile[b] = x[2];
    s_len[b] = x[6];  // tokens of the sequences before; the prefix lengths are no longer needed
    if (s_count[b] > 0 && tiles_of(s_count[b]) > 1) {
      s_wide[b] = x[5];
      s_at[x[5]] = b;
      s_n[x[5]] = tiles_of(s_count[b]);
      s_lu[x[5]] = lead_for(s_count[b]);
      s_u[x[5]] = lead_for(s_count[b]) + units_of(s_shared[b]);
    }
    add(b);
  }
  if (tid == 0) s_pick[0] = -1;
  __syncthreads();

  // The cut: `len` units a workgroup.  Prefixes of several tiles are cut apart from everything else: those with the same number of tiles
  // lie on one axis, every cut of it is a workgroup for each of the tiles, and these run at the same time and find what the first of
  // them loads in their XCD's L2.  (With its tiles one behind the other all of them read the keys from beyond L2.)  That takes a few
  // more workgroups, so `len` is the shortest of 64 lengths, a lane each, for which there are enough.
  for (int m = tid; m < n_multi; m += n_thr) {
    const int n = s_n[m];
    int pos = 0, all = 0, next = -1, first = 1;
    for (int i = 0; i < n_multi; ++i) {
      if (s_n[i] != n) continue;
      const int u = s_u[i];
      all += u;
      if (i < m) {
        pos += u;
        first = 0;
      } else if (i > m && next < 0) {
        next = i;
      }
    }
    s_pos[m] = pos;
    s_end[m] = first ? all : 0;
    s_next[m] = next;
  }
  __syncthreads();
  const int shortest_len = max(kMinUnits, (all_units + a.n_wg - 1) / a.n_wg);
  const auto cuts = [](int units, int len) { return units > 0 ? (units - 1) / len + 1 : 0; };  // (two such sums may pass 31 bits)
  const auto length_at = [&](int i) {  // the i-th of the 64: up to three times the shortest, at most everything
    return static_cast<int>(min(static_cast<int64_t>(max(kMinUnits, all_units)), shortest_len + (static_cast<int64_t>(shortest_len) * i + 31) / 32));
  };
  if (wave == 0 && n_multi > 0) {
    const int len = length_at(lane);
    int need = 0, rest = all_units;
    for (int m = 0; m < n_multi; ++m) {
      need += s_n[m] * cuts(s_end[m], len);
      rest -= s_n[m] * s_u[m];
    }
    const unsigned long long enough = __ballot(need + cuts(rest, len) <= a.n_wg);
    if (enough != 0 && lane == 0) s_pick[0] = __builtin_ctzll(enough);
  }
  __syncthreads();
  const int pick = s_pick[0];
  const bool apart = pick >= 0;  // else there are too many kinds of groups: all on one axis
  const int len = apart ? length_at(pick) : shortest_len;
  const auto pieces_at = [&](int m) {  // of a tile: from the cut of its first key to that of its last
    return (s_pos[m] + s_u[m] - 1) / len - (s_pos[m] + s_lu[m]) / len + 1;
  };
  int wg0 = 0, wide_parts = 0;  // workgroups and pieces of these prefixes
  if (apart) {
    for (int m = 0; m < n_multi; ++m) {
      if (tid == 0) s_part[m] = wide_parts;
      wg0 += s_n[m] * cuts(s_end[m], len);
      wide_parts += s_n[m] * pieces_at(m);
    }
  }
  const auto stands_apart = [&](int b) { return apart && tiles_of(s_count[b]) > 1; };
  int y[2] = {0, 0}, y_before[2], y_total[2];
  const auto add_cut = [&](int b) {
    const int c = s_count[b], own = s_keys[b] - s_shared[b];
    if (c > 0 && !stands_apart(b)) y[0] += tiles_of(c) * (lead_for(c) + units_of(s_shared[b]));
    if (own > 0) y[1] += tiles_of(s_tok[b]) * (lead_for(s_tok[b]) + units_of(own));
  };
  for (int b = b0; b < b1; ++b) add_cut(b);
  block_sums(y, y_before, y_total, s_sum);
  const int prefix_units = y_total[0], units = prefix_units + y_total[1];
  const int n_wg = wg0 + cuts(units, len);
  y[0] = y_before[0], y[1] = y_before[1];
  for (int b = b0; b < b1; ++b) {
    s_unit[b] = y[0];
    s_own[b] = y[1];
    add_cut(b);
  }
  __syncthreads();

  if (tid == 0) {
    Header* const h = reinterpret_cast<Header*>(a.plan);
    h->magic = kMagic;
    h->B = a.B, h->S = a.S, h->Hq = a.Hq, h->Hc = a.Hc, h->max_batch = a.max_batch, h->max_context = a.max_context;
    h->n_wg = n_wg, h->n_tiles = n_tiles;
  }
  int* const tokens = reinterpret_cast<int*>(a.plan + a.tokens);
  int* const place = reinterpret_cast<int*>(a.plan + a.place);
  const auto base_of = [&](int b) { return s_shared[b] > 0 ? s_base[s_lead[b]] + s_rank[b] : s_base[b]; };
  if (a.S == 1)
    for (int b = tid; b < a.B; b += n_thr)
      if (s_tok[b] > 0) tokens[base_of(b)] = b << kTokenShift;
  if (a.S > 1) {
    for (int b = wave; b < a.B; b += n_waves) {
      int n = 0;
      const int base = base_of(b), all = s_tok[b];
      for (int j0 = 0; j0 < a.S; j0 += 64) {
        const int j = j0 + lane;
        const bool on = all > 0 && j < a.S && plan_keys(a, b, j) > 0;
        const unsigned long long who = __ballot(on);
        const int at = n + __popcll(who & ((1ull << lane) - 1));
        if (on && at < all) tokens[base + at] = b << kTokenShift | j;
        if (j < a.S) place[b * a.S + j] = on ? at : -1;
        n += __popcll(who);
      }
    }
  }
  // Workspace rows.  Prefixes that are cut apart: 64 a piece.  Behind them, along the other axis: those of the tiles before, each once, and
  // 64 for every cut up to a tile's first key.
  const int rest_part = kTileRows * wide_parts;
  const auto tile_at = [&](int i) {
    Tile t;
    int n_units, from, rows_before;
    if (i < p_tiles) {
      const int b = last_at_or_below(s_ptile, a.B, i), k = i - s_ptile[b], n = tiles_of(s_count[b]);
      n_units = units_of(s_shared[b]);
      t.lead = lead_for(s_count[b]);
      t.base = s_base[b];
      t.slot = s_slot[b];
      t.row0 = k * kTileRows;
      t.n_rows = min(kTileRows, s_count[b] * a.group - t.row0);
      t.t_begin = 0;
      t.t_end = s_shared[b];
      t.shared = 1;
      t.again = n > 1;
      if (stands_apart(b)) {
        const int m = s_wide[b], next = s_next[m];
        t.n_pieces = pieces_at(m);
        t.part = kTileRows * (s_part[m] + k * t.n_pieces);
        t.next = next < 0 ? n_tiles : s_ptile[s_at[next]] + k;
        return t;
      }
      from = s_unit[b] + k * (t.lead + n_units);
      const int end = from + t.lead + n_units;
      t.next = k + 1 < n ? i + 1 : end < prefix_units ? s_ptile[last_at_or_below(s_unit, a.B, end)] : p_tiles;
      rows_before = s_base[b] * a.group + t.row0;
    } else {
      const int b = last_at_or_below(s_stile, a.B, i - p_tiles), k = i - p_tiles - s_stile[b];
      n_units = units_of(s_keys[b] - s_shared[b]);
      t.lead = lead_for(s_tok[b]);
      from = prefix_units + s_own[b] + k * (t.lead + n_units);
      t.base = base_of(b);
      t.slot = s_slot[b];
      t.row0 = k * kTileRows;
      t.n_rows = min(kTileRows, s_tok[b] * a.group - t.row0);
      t.t_begin = s_shared[b];
      t.t_end = s_keys[b];
      t.shared = 0;
      t.again = tiles_of(s_tok[b]) > 1;
      t.next = i + 1;
      rows_before = (shared_tokens + s_len[b]) * a.group + t.row0;
    }
    const int first = (from + t.lead) / len;
    t.n_pieces = (from + t.lead + n_units - 1) / len - first + 1;
    t.part = rest_part + rows_before + kTileRows * first;
    return t;
  };
  // Shares, tiles, and two items a sequence: its prefix and its own keys.  Lanes of all three work out the tile that they need together
  // (in a branch for each they would do so one after the other: 16 sequences 11.2 us instead of 8.6).
  for (int i = tid; i < n_wg + n_tiles + 2 * a.B; i += n_thr) {
    const int k = i - n_wg - n_tiles, b = k >> 1;
    const bool is_share = i < n_wg, is_tile = !is_share && k < 0, of_own = k & 1;
    int index = -1, offset = 0, units_to_do = 0, piece = 0;
    if (is_share) {
      int start, from;  // of the first tile's first key and of this workgroup, on their axis
      if (i < wg0) {
        int m = 0, rest = i;  // the first group of the kind, workgroups of the kind before this one
        for (;; ++m) {
          const int here = s_n[m] * cuts(s_end[m], len);
          if (rest < here) break;
          rest -= here;
        }
        const int n = s_n[m], all = s_end[m];
        from = rest / n * len;
        while (s_pos[m] + s_u[m] <= from) m = s_next[m];
        index = s_ptile[s_at[m]] + rest % n;
        offset = from - s_pos[m];
        units_to_do = min(len, all - from);
        start = s_pos[m] + s_lu[m];
      } else {
        from = (i - wg0) * len;
        units_to_do = min(len, units - from);
        const bool own = from >= prefix_units;
        const int at = own ? from - prefix_units : from, of = last_at_or_below(own ? s_own : s_unit, a.B, at);
        const int lead = lead_for(own ? s_tok[of] : s_count[of]);
        const int n = lead + units_of(own ? s_keys[of] - s_shared[of] : s_shared[of]), off = at - (own ? s_own : s_unit)[of];
        index = (own ? p_tiles + s_stile[of] : s_ptile[of]) + off / n;
        offset = off % n;
        start = from - offset + lead;
      }
      piece = max(0, from / len - start / len);
    } else if (is_tile) {
      index = i - n_wg;
    } else if (of_own) {
      index = s_keys[b] > s_shared[b] ? p_tiles + s_stile[b] : -1;
    } else {
      index = s_shared[b] > 0 ? s_ptile[s_lead[b]] + s_rank[b] * a.group / kTileRows : -1;
    }
    Tile t{};
    if (index >= 0) t = tile_at(index);
    if (is_share) {
      reinterpret_cast<Share*>(a.plan + a.shares)[i] = Share{index, offset, units_to_do, piece, t};
    } else if (is_tile) {
      reinterpret_cast<Tile*>(a.plan + a.tiles)[index] = t;
    } else if (of_own) {
      seqs[b].own_tile = index;
      seqs[b].own_at = t.part, seqs[b].own_step = t.n_rows, seqs[b].own_n = t.n_pieces;
    } else {
      const int row = s_rank[b] * a.group;
      seqs[b].slot = s_slot[b], seqs[b].keys = s_keys[b];
      seqs[b].prefix_tile = index < 0 ? -1 : index - row / kTileRows, seqs[b].prefix_row = row;
      seqs[b].at = t.part + row % kTileRows, seqs[b].step = t.n_rows, seqs[b].n = t.n_pieces;
    }
  }
}

// -------------------------------------------------------------------------------------------------------- products
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
  int group, group_shift;  // query heads of a cached head
  const char* plan;
  int64_t seqs, tokens, place, shares, tiles;
  float* ws_acc;  // [part rows, Hc, D]
  float* ws_ml;   // [part rows, Hc, 2]
};

struct BF16 {
  using type = __bf16;
  typedef __bf16 vec8 __attribute__((ext_vector_type(8)));
  static constexpr int kBytes = 2;
  // sets the elements of w that are infinite or NaN to 0; whether there are any
  static __device__ __forceinline__ bool drop_infinities(uint32_t& w) {
    const bool lo = (w & 0x7f80u) == 0x7f80u, hi = (w & 0x7f800000u) == 0x7f800000u;
    w &= (lo ? 0u : 0xffffu) | (hi ? 0u : 0xffff0000u);
    return lo || hi;
  }
  // Added to the exponents: the probabilities stay at 1 and below although the reference point lags the maximum, so that a product
  // with the largest V of the type stays in fp32.
  static constexpr float kHeadroom = -kMaxSlack;
  static __device__ __forceinline__ f32x4 mfma_k32(const v4u& a, const v4u& b, const f32x4& c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(vec8, a), __builtin_bit_cast(vec8, b), c, 0, 0, 0);
  }
  static __device__ __forceinline__ uint32_t pack2(float lo, float hi) {
    typedef __bf16 vec2 __attribute__((ext_vector_type(2)));
    const vec2 v = {static_cast<__bf16>(lo), static_cast<__bf16>(hi)};
    return __builtin_bit_cast(uint32_t, v);
  }
  // p0 and p1 as sums of two numbers of the type, none below 0 (and above it where p is), so that against an infinite V element
  // they give infinity: truncated, and what is left over, with 2^-23 of p on top.
  static __device__ __forceinline__ void split(float p0, float p1, uint32_t& hi, uint32_t& lo) {
    const uint32_t b0 = __float_as_uint(p0), b1 = __float_as_uint(p1);
    hi = __builtin_amdgcn_perm(b1, b0, 0x07060302);
    lo = pack2(fmaf(p0, 1.f + 0x1p-23f, -__uint_as_float(b0 & 0xffff0000u)), fmaf(p1, 1.f + 0x1p-23f, -__uint_as_float(b1 & 0xffff0000u)));
  }
};
struct F16 {
  using type = _Float16;
  typedef _Float16 vec8 __attribute__((ext_vector_type(8)));
  static constexpr int kBytes = 2;
  static __device__ __forceinline__ bool drop_infinities(uint32_t& w) {
    const bool lo = (w & 0x7c00u) == 0x7c00u, hi = (w & 0x7c000000u) == 0x7c000000u;
    w &= (lo ? 0u : 0xffffu) | (hi ? 0u : 0xffff0000u);
    return lo || hi;
  }
  // probabilities up to 2^(8 + kMaxSlack): below the largest f16, and small ones stay normal numbers longer
  static constexpr float kHeadroom = 8.f;
  static __device__ __forceinline__ f32x4 mfma_k32(const v4u& a, const v4u& b, const f32x4& c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(vec8, a), __builtin_bit_cast(vec8, b), c, 0, 0, 0);
  }
  static __device__ __forceinline__ uint32_t pack2(float lo, float hi) {
    typedef _Float16 vec2 __attribute__((ext_vector_type(2)));
    const vec2 v = {static_cast<_Float16>(lo), static_cast<_Float16>(hi)};
    return __builtin_bit_cast(uint32_t, v);
  }
  // As above.  Neither part of a p above 0 is below the smallest number of the type, 2^-24, where a wavefront's largest p is 2^8 or more
  // (kHeadroom): each key of vanishing weight counts for up to 2^-31 of the largest one's.  A wavefront has a quarter of a piece's stages,
  // so in a context of n keys they come to n * 2^-33 of the largest |V| at most, 2^-12 at kMaxContext, half of what rounding an f16 of
  // that size may cost.
  static __device__ __forceinline__ void split(float p0, float p1, uint32_t& hi, uint32_t& lo) {
    const float l0 = fminf(p0 * 0x1p+102f, 0x1p-24f), l1 = fminf(p1 * 0x1p+102f, 0x1p-24f);
    const auto h = __builtin_amdgcn_cvt_pkrtz(fmaxf(p0, l0), fmaxf(p1, l1));
    hi = __builtin_bit_cast(uint32_t, h);
    lo = pack2(fmaxf(p0 - static_cast<float>(h[0]), l0), fmaxf(p1 - static_cast<float>(h[1]), l1));
  }
};
struct F32 {
  using type = float;
  static constexpr int kBytes = 4;
  static constexpr float kHeadroom = -kMaxSlack;
  static __device__ __forceinline__ bool drop_infinities(uint32_t& w) {
    const bool odd = (w & 0x7f800000u) == 0x7f800000u;
    if (odd) w = 0;
    return odd;
  }
};

__device__ __forceinline__ s16x4 lds_read_tr(const char* p) {
  return __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)(p));
}

// fp::load_to_lds for rows that no other workgroup reads (non-temporal).
__device__ __forceinline__ void load_once(const char* base, uint32_t offset, uint32_t own, uint32_t constant) {
  asm volatile("s_add_u32 m0, %0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %2, %3 nt"
               : : "s"(own), "s"(constant), "v"(offset), "s"(base) : "memory", "scc");
}

// this wavefront's staging loads but the `kLater` issued last have landed in LDS
template <int kLater>
__device__ __forceinline__ void wait_staged() {
  asm volatile("s_waitcnt vmcnt(%0)" : : "n"(kLater) : "memory");
}

// Stages: TS rows of K, then TS rows of V.  16-byte chunk c of K's row r sits at c ^ k_swz(r) (the score product reads one chunk of
// 16 consecutive rows); of 16-bit V, 32-byte region c of row r at c ^ v_swz(r) (a transpose read takes one region of 16
// rows); fp32's V is read along its rows and stays in order.
template <typename E, int D>
struct Geo {
  static constexpr bool k16 = E::kBytes == 2;
  static constexpr int ROWB = D * E::kBytes;
  static constexpr int CPR = ROWB / 16;            // 16-byte chunks of a row
  static constexpr int R32 = ROWB / 32;
  static constexpr int RPI = 64 / CPR;             // rows of one load instruction
  static constexpr int TS = ROWB == 128 ? 32 : 16;  // keys of a stage
  static constexpr int HALF = TS * ROWB;           // bytes of a stage's K
  static constexpr int NI = HALF / 1024;           // load instructions of a stage's K
  static constexpr int NB = TS / 16;               // blocks of 16 keys
  static constexpr int DB = D / 16;                // blocks of 16 rows of O^T
  static constexpr int QV = ROWB / 64;             // 16-byte operand registers of a query row
  static constexpr bool QTAIL = k16 && D == 128;
  static constexpr int RING = 2 * 2 * HALF;        // two stages a wavefront
  static constexpr int PASS = RING / (16 * D * 4) < 4 ? RING / (16 * D * 4) : 4;  // column blocks whose states fit a ring
  static __device__ __forceinline__ int k_swz(int r) { return CPR == 8 ? (r >> 1) & 7 : r & 15; }
  static __device__ __forceinline__ int v_swz(int r) { return !k16 ? 0 : CPR == 16 ? r & 7 : (r >> 1) & 3; }
};

template <typename E>
__device__ __forceinline__ void store4(char* p, const f32x4& v) {
  if constexpr (E::kBytes == 4)
    *reinterpret_cast<f32x4*>(p) = v;
  else
    *reinterpret_cast<uint2*>(p) = uint2{E::pack2(v[0], v[1]), E::pack2(v[2], v[3])};
}

// keys of token j of sequence b
__device__ __forceinline__ int keys_of(const SharedArgs& a, int b, int j) {
  const int64_t p = fp::load_index(a.input_pos, static_cast<int64_t>(b) * a.S + j, a.pos_i64) + 1;
  return p < 0 ? 0 : p > a.max_context ? a.max_context : static_cast<int>(p);
}

template <typename E, int D>
struct Shared {
  using G = Geo<E, D>;
  __attribute__((aligned(1024))) char ring[kWaves][G::RING];
  int pages[kSegPages];
  __attribute__((aligned(8))) float ml[kWaves][kTileRows][2];
  float joined[kTileRows][2];    // maximum and sum of all wavefronts
  int limit[kWaves][kTileRows];  // keys of the columns' rows, each wavefront's own copy
  __attribute__((aligned(16))) v4u q_tail[G::QTAIL ? 4 * 64 : 1];  // last quarter of the query rows, by column block and lane
  int tainted;  // an element of V that is not finite was left out
};

// This lane's number, worked out where it is used: kept through the loop over the keys it would be a register of the loop, and so
// would all that follows from it.
__device__ __forceinline__ int lane_id() {
  int x;
  asm volatile("v_mbcnt_lo_u32_b32 %0, -1, 0\n\tv_mbcnt_hi_u32_b32 %0, -1, %0" : "=v"(x));
  return x;
}

// The kernel's arguments (its first parameter) read again where they are used: scalar registers that carried them through the
// loop over the keys would be spilled into vector registers.
__device__ __forceinline__ const SharedArgs& reread() {
  auto p = (const __attribute__((address_space(4))) SharedArgs*)__builtin_amdgcn_kernarg_segment_ptr();
  asm volatile("" : "+s"(p));
  return *(const SharedArgs*)p;
}

// Token and head of row r of a tile.
__device__ __forceinline__ void find_row(const SharedArgs& a, const Tile& tile, int r, int* b, int* j, int* g) {
  const int x = tile.row0 + r, token = reinterpret_cast<const int*>(a.plan + a.tokens)[tile.base + (x >> a.group_shift)];
  *b = token >> kTokenShift;
  *j = token & ((1 << kTokenShift) - 1);
  *g = x & (a.group - 1);
}

// What the products left out of row r: the infinities and NaN of the V rows of keys [t0, t1) that it sees, elements 4 c .. 4 c + 3.
template <typename E, int D>
__device__ __forceinline__ void add_infinities(const SharedArgs& a, const Tile& tile, int r, int t0, int t1,
                                                         const char* vplane, int c, f32x4& num) {
  int b, j, g;
  find_row(a, tile, r, &b, &j, &g);
  const int end = min(t1, keys_of(a, b, j));
  for (int t = t0; t < end; ++t) {
    int64_t blk;
    int off;
    a.pd.split(t, blk, off);
    int64_t page = blk < a.n_pages ? a.page_table[static_cast<int64_t>(tile.slot) * a.pt_row_stride + blk] : 0;
    if (page < 0 || page >= a.pool_pages) page = 0;
    const char* const at = vplane + ((page * a.pd.page_size + off) * D + c * 4) * E::kBytes;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const float v = static_cast<float>(reinterpret_cast<const typename E::type*>(at)[k]);
      if (!(fabsf(v) < INFINITY)) num[k] += v;
    }
  }
}

// A barrier of the workgroup behind this wavefront's LDS instructions.  (__syncthreads also waits for stores to global memory, 1 to 2 us
// for partial results that nobody here reads.)
__device__ __forceinline__ void lds_barrier() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" : : : "memory"); }

// One piece: the rows of a tile over its keys [t0, t1).  CB blocks of 16 columns.
template <typename E, int D, int CB>
__device__ __forceinline__ void run_piece(const SharedArgs& a, Shared<E, D>& sh, const int wave, const Tile& tile, const int piece,
                                          const int t0, const int t1) {
  using G = Geo<E, D>;
  const int hc = blockIdx.x;
  const bool prefix = tile.shared != 0;
  char* const ring = sh.ring[wave];
  const uint32_t lds_ring = fp::lds_address(ring);
  const char* const kplane = a.pool_k + static_cast<int64_t>(hc) * a.n_slots * G::ROWB;
  const char* const vplane = a.pool_v + static_cast<int64_t>(hc) * a.n_slots * G::ROWB;
  const int64_t* const table = a.page_table + static_cast<int64_t>(tile.slot) * a.pt_row_stride;

  // the page ids of the first segment are on their way before the rows are asked for
  int64_t early = 0;
  {
    int64_t first, last;
    int unused;
    a.pd.split(t0, first, unused);
    a.pd.split(t1 - 1, last, unused);
    const int64_t blk = first + wave * 64 + lane_id();
    if (blk <= last && blk < a.n_pages) early = table[blk];
  }

  // rows: query operands and limits of this lane's columns.  A column without a row repeats row 0, sees everything and is not stored.
  // Of four column blocks at head_dim 128 the last quarter of the query rows stays in LDS: with it the registers would not hold the rest.
  constexpr bool kTail = CB == 4 && G::QTAIL;
  constexpr int QR = kTail ? G::QV - 1 : G::QV;
  v4u q[CB][QR], tail = {0, 0, 0, 0};
  int64_t pos[CB];
  int least = INT32_MAX;
  {
    // two trips to memory: the tokens, then what they name
    const int lane = lane_id(), col = lane & 15, grp = lane >> 4;
    const SharedArgs& a = reread();
    const int* const tokens = reinterpret_cast<const int*>(a.plan + a.tokens) + tile.base;
    int x[CB], token[CB];
#pragma unroll
    for (int cb = 0; cb < CB; ++cb) {
      const int r = cb * 16 + col;
      x[cb] = tile.row0 + (r < tile.n_rows ? r : 0);
      token[cb] = tokens[x[cb] >> a.group_shift];
    }
    const auto at = [&](int cb) { return static_cast<int64_t>(token[cb] >> kTokenShift) * a.S + (token[cb] & ((1 << kTokenShift) - 1)); };
    if (a.pos_i64) {
#pragma unroll
      for (int cb = 0; cb < CB; ++cb) pos[cb] = static_cast<const int64_t*>(a.input_pos)[at(cb)];
    } else {
#pragma unroll
      for (int cb = 0; cb < CB; ++cb) pos[cb] = static_cast<const int32_t*>(a.input_pos)[at(cb)];
    }
#pragma unroll
    for (int cb = 0; cb < CB; ++cb) {
      const int b = token[cb] >> kTokenShift, j = token[cb] & ((1 << kTokenShift) - 1), h = hc * a.group + (x[cb] & (a.group - 1));
      const char* const src = a.q + b * a.qs_b + h * a.qs_h + j * a.qs_s + grp * 16;
#pragma unroll
      for (int kk = 0; kk < QR; ++kk) q[cb][kk] = *reinterpret_cast<const v4u*>(src + kk * 64);
      if (kTail && cb == wave) tail = *reinterpret_cast<const v4u*>(src + QR * 64);  // a block a wavefront
    }
    __builtin_amdgcn_sched_barrier(0);  // all of them are on their way before the first is waited for
  }
  if (wave == 0 && lane_id() == 0) sh.tainted = 0;  // ahead of the barriers of the first segment

  f32x4 o[CB][G::DB];
  float m[CB], l[CB];
#pragma unroll
  for (int cb = 0; cb < CB; ++cb) {
    m[cb] = -INFINITY;
    l[cb] = 0.f;
#pragma unroll
    for (int db = 0; db < G::DB; ++db) o[cb][db] = f32x4{0.f, 0.f, 0.f, 0.f};
  }

  const bool aligned_pages = a.pd.page_size % G::TS == 0;

  for (int seg0 = t0; seg0 < t1;) {
    int64_t blk0;
    int off0, seg1 = t1;
    a.pd.split(seg0, blk0, off0);
    {
      const int64_t room = (blk0 + kSegPages) * a.pd.page_size - seg0;
      if (room < t1 - seg0) seg1 = seg0 + static_cast<int>(room) / (kWaves * G::TS) * (kWaves * G::TS);
      int64_t last;
      int unused;
      a.pd.split(seg1 - 1, last, unused);
      lds_barrier();  // the page ids before are no longer read
      for (int i = wave * 64 + lane_id(); i <= static_cast<int>(last - blk0); i += kThreads) {
        int64_t page = 0;
        if (seg0 == t0 && i < kThreads)
          page = early;
        else if (blk0 + i < a.n_pages)
          page = table[blk0 + i];
        if (page < 0 || page >= a.pool_pages) page = 0;  // as paged_decode: the reserved page
        sh.pages[i] = static_cast<int>(page);
      }
      lds_barrier();
    }

    // pool row of the first key of a stage that lies in one page and in the segment, -1: not such a stage
    const auto locate = [&](int c0) {
      if (!aligned_pages || c0 % G::TS != 0 || c0 + G::TS > seg1) return static_cast<int64_t>(-1);
      const int blk = a.pd.shift >= 0 ? c0 >> a.pd.shift : c0 / a.pd.page_size;
      const int page = __builtin_amdgcn_readfirstlane(sh.pages[blk - static_cast<int>(blk0)]);
      return static_cast<int64_t>(page) * a.pd.page_size + (c0 - blk * a.pd.page_size);
    };
    const auto issue = [&](int64_t slot, int c0, uint32_t stage) {
      // Instruction i brings rows i * RPI + lrow, position lpos of each.  The permutations of a row are those of i * RPI and of lrow
      // together, so a load's offset is one exclusive or and one sum away from the first one's.
      const int at = lane_id(), lrow = at / G::CPR, lpos = at % G::CPR;
      const uint32_t k_at = lrow * G::ROWB + (lpos ^ G::k_swz(lrow)) * 16, v_at = lrow * G::ROWB + (lpos ^ G::v_swz(lrow) * 2) * 16;
      if (slot >= 0) {
        const char* const k = kplane + slot * G::ROWB;
        const char* const v = vplane + slot * G::ROWB;
        if (tile.again) {  // other tiles read these rows, too
#pragma unroll
          for (int i = 0; i < G::NI; ++i) fp::load_to_lds(k, (k_at ^ (G::k_swz(i * G::RPI) * 16)) + i * 1024, stage, i * 1024);
#pragma unroll
          for (int i = 0; i < G::NI; ++i) fp::load_to_lds(v, (v_at ^ (G::v_swz(i * G::RPI) * 32)) + i * 1024, stage, G::HALF + i * 1024);
        } else {
#pragma unroll
          for (int i = 0; i < G::NI; ++i) load_once(k, (k_at ^ (G::k_swz(i * G::RPI) * 16)) + i * 1024, stage, i * 1024);
#pragma unroll
          for (int i = 0; i < G::NI; ++i) load_once(v, (v_at ^ (G::v_swz(i * G::RPI) * 32)) + i * 1024, stage, G::HALF + i * 1024);
        }
      } else {  // pages that do not hold whole stages, the last keys: row by row.  A row past the range repeats its last one and is masked
#pragma nounroll
        for (int i = 0; i < G::NI; ++i) {  // one at a time: their addresses would be registers of the whole loop
          const int t = min(c0 + i * G::RPI + lrow, seg1 - 1);
          int64_t blk;
          int off;
          a.pd.split(t, blk, off);
          const int64_t row = (static_cast<int64_t>(sh.pages[blk - blk0]) * a.pd.page_size + off) * G::ROWB;
          fp::load_to_lds(kplane + row + ((lpos ^ G::k_swz(i * G::RPI + lrow)) * 16), stage + i * 1024, 0u);
          fp::load_to_lds(vplane + row + ((lpos ^ G::v_swz(i * G::RPI + lrow) * 2) * 16), stage + G::HALF + i * 1024, 0u);
        }
      }
    };

    // stages wave, wave + 4, ... of the segment
    const int n_stages = (seg1 - seg0 + G::TS - 1) / G::TS;
    if (wave < n_stages) issue(locate(seg0 + wave * G::TS), seg0 + wave * G::TS, lds_ring);
    if (wave + kWaves < n_stages) issue(locate(seg0 + (wave + kWaves) * G::TS), seg0 + (wave + kWaves) * G::TS, lds_ring + 2 * G::HALF);
    if (seg0 == t0) {  // the rows' limits, now that the first stages are on their way
      const int lane = lane_id(), col = lane & 15, max_context = a.max_context;
#pragma unroll
      for (int cb = 0; cb < CB; ++cb) {
        const int r = cb * 16 + col;
        const int64_t keys = pos[cb] < 0 ? 0 : pos[cb] >= max_context ? max_context : pos[cb] + 1;
        const int lim = r < tile.n_rows ? static_cast<int>(keys) : INT32_MAX;
        least = min(least, lim);
        if (lane < 16) sh.limit[wave][cb * 16 + col] = lim;
      }
      least = -fp::wave_max(-least);
      if constexpr (kTail) {
        sh.q_tail[wave * 64 + lane] = tail;
        lds_barrier();
      }
    }
    // The query rows are waited for here.  At their first use, inside the loop over the stages, the wait would be one of every stage, and
    // for the stages on their way, too, of which the compiler does not know.
#pragma unroll
    for (int cb = 0; cb < CB; ++cb)
#pragma unroll
      for (int kk = 0; kk < QR; ++kk) asm volatile("" : "+v"(q[cb][kk]));
#pragma nounroll
    for (int s = wave, buf = 0; s < n_stages; s += kWaves, buf ^= 1) {
      const int c0 = seg0 + s * G::TS;
      char* const k_lds = ring + buf * 2 * G::HALF;
      char* const v_lds = k_lds + G::HALF;
      const int64_t next = s + 2 * kWaves < n_stages ? locate(c0 + 2 * kWaves * G::TS) : -1;
      if (s + kWaves < n_stages) wait_staged<2 * G::NI>(); else wait_staged<0>();
      // scores of this lane's columns: keys 16 * blk + 4 * grp + 0 .. 3
      f32x4 sc[CB][G::NB];
      const int lane_now = lane_id();
#pragma unroll
      for (int blk = 0; blk < G::NB; ++blk) {
#pragma unroll
        for (int cb = 0; cb < CB; ++cb) sc[cb][blk] = f32x4{0.f, 0.f, 0.f, 0.f};
        const int r = blk * 16 + (lane_now & 15);
        const uint32_t at = r * G::ROWB + ((lane_now >> 4) ^ G::k_swz(r)) * 16;
        constexpr int kAhead = CB == 4 ? 2 : 4;  // operands on their way ahead of the products that use them
        v4u ahead[G::QV];
#pragma unroll
        for (int kk = 0; kk < kAhead && kk < G::QV; ++kk) ahead[kk] = *reinterpret_cast<const v4u*>(k_lds + (at ^ (kk * 64)));
#pragma unroll
        for (int kk = 0; kk < G::QV; ++kk) {
          if (kk + kAhead < G::QV) ahead[kk + kAhead] = *reinterpret_cast<const v4u*>(k_lds + (at ^ ((kk + kAhead) * 64)));
          __builtin_amdgcn_sched_barrier(0);
          const v4u ka = ahead[kk];
#pragma unroll
          for (int cb = 0; cb < CB; ++cb) {
            if constexpr (G::k16) {
              const v4u qb = kk < QR ? q[cb][kk < QR ? kk : 0] : sh.q_tail[cb * 64 + lane_now];
              sc[cb][blk] = E::mfma_k32(ka, qb, sc[cb][blk]);
            } else {
#pragma unroll
              for (int e = 0; e < 4; ++e)
                sc[cb][blk] = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(ka[e]), __uint_as_float(q[cb][kk][e]), sc[cb][blk], 0, 0, 0);
            }
          }
        }
#pragma unroll
        for (int cb = 0; cb < CB; ++cb) sc[cb][blk] *= a.qscale;
      }
      if (c0 + G::TS > min(seg1, least)) {
#pragma unroll
        for (int cb = 0; cb < CB; ++cb) {
          const int end = min(sh.limit[wave][cb * 16 + (lane_now & 15)], seg1);
#pragma unroll
          for (int blk = 0; blk < G::NB; ++blk)
#pragma unroll
            for (int j = 0; j < 4; ++j)
              if (c0 + blk * 16 + (lane_now >> 4) * 4 + j >= end) sc[cb][blk][j] = -INFINITY;
        }
        // V rows past the range become 0: a probability of 0 against an infinity would be NaN.  So do the elements that are not
        // finite of rows which only some columns see; these columns get them at the end.
#pragma nounroll
        for (int i = 0; i < G::NI; ++i) {
          const int t = c0 + i * G::RPI + lane_now / G::CPR;
          if (t < least) continue;
          v4u* const at = reinterpret_cast<v4u*>(v_lds + i * 1024 + lane_now * 16);
          v4u w = {0, 0, 0, 0};
          if (t < seg1) {
            w = *at;
            bool odd = false;
#pragma unroll
            for (int c = 0; c < 4; ++c) {
              uint32_t two = w[c];
              odd |= E::drop_infinities(two);
              w[c] = two;
            }
            if (!odd) continue;
            sh.tainted = 1;
          }
          *at = w;
        }
        asm volatile("" : : : "memory");  // a wavefront's LDS instructions are executed in order
      }
      // The first V operands leave LDS while the exponentials are worked out, where there are registers for them.
      constexpr int kReadsV = G::k16 ? G::NB * G::DB : G::NB * 4 * (D / 64);  // reads of a stage
      constexpr int kAheadV = CB == 4 ? 2 : 8 < kReadsV ? 8 : kReadsV;
      const auto read_v = [&](int n) {
        if constexpr (G::k16) {
          // lanes 4 j + c of a 16-lane block name elements 4 c .. of key 4 * grp + j and receive element `col` of the four keys
          const int r = n / G::DB * 16 + (lane_now >> 4) * 4 + ((lane_now & 15) >> 2);
          return lds_read_tr(v_lds + ((r * G::ROWB + G::v_swz(r) * 32 + (lane_now & 3) * 8) ^ (n % G::DB * 32)));
        } else {
          const int r = n / (D / 64) / 4 * 16 + (lane_now >> 4) * 4 + n / (D / 64) % 4;
          return *reinterpret_cast<const f32x4*>(v_lds + r * G::ROWB + n % (D / 64) * 256 + (lane_now & 15) * 16);
        }
      };
      decltype(read_v(0)) v_ahead[kAheadV];
      const auto first_v = [&] {
#pragma unroll
        for (int n = 0; n < kAheadV; ++n) v_ahead[n] = read_v(n);
      };
      if constexpr (CB < 4) first_v();
      // Reference point of the exponentials, per column: moves only when the column's maximum has outgrown it by kMaxSlack, so most
      // stages need no exchange between the lanes of a column and no rescale.
      float cand[CB];
      bool grown = false;
#pragma unroll
      for (int cb = 0; cb < CB; ++cb) {
        cand[cb] = sc[cb][0][0];
#pragma unroll
        for (int blk = 0; blk < G::NB; ++blk)
#pragma unroll
          for (int j = 0; j < 4; ++j) cand[cb] = fmaxf(cand[cb], sc[cb][blk][j]);
        grown |= cand[cb] > m[cb] + (E::kHeadroom + kMaxSlack);
      }
      if (__any(grown)) {
#pragma unroll
        for (int cb = 0; cb < CB; ++cb) {
          cand[cb] = fmaxf(cand[cb], __shfl_xor(cand[cb], 16));
          cand[cb] = fmaxf(cand[cb], __shfl_xor(cand[cb], 32));
          if (cand[cb] > m[cb] + (E::kHeadroom + kMaxSlack)) {
            const float m_new = cand[cb] - E::kHeadroom, alpha = fast_exp2(m[cb] - m_new);
            l[cb] *= alpha;
#pragma unroll
            for (int db = 0; db < G::DB; ++db) o[cb][db] *= alpha;
            m[cb] = m_new;
          }
        }
      }
#pragma unroll
      for (int cb = 0; cb < CB; ++cb) {
        const float ms = safe_max(m[cb]);  // no key above -inf so far: its probabilities are 0
#pragma unroll
        for (int blk = 0; blk < G::NB; ++blk)
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            sc[cb][blk][j] = fast_exp2(sc[cb][blk][j] - ms);
            l[cb] += sc[cb][blk][j];
          }
      }
      if constexpr (CB == 4) first_v();
      if constexpr (G::k16) {
#pragma unroll
        for (int blk = 0; blk < G::NB; ++blk) {
          // 16 keys and the same 16 again: the probabilities are the sum of two parts of 16 bits, of which one product takes both
          v4u pb[CB];
#pragma unroll
          for (int cb = 0; cb < CB; ++cb) {
            uint32_t hi[2], lo[2];
#pragma unroll
            for (int j = 0; j < 2; ++j) E::split(sc[cb][blk][2 * j], sc[cb][blk][2 * j + 1], hi[j], lo[j]);
            pb[cb] = v4u{hi[0], hi[1], lo[0], lo[1]};
          }
#pragma unroll
          for (int db = 0; db < G::DB; ++db) {
            const uint2 half = __builtin_bit_cast(uint2, v_ahead[(blk * G::DB + db) % kAheadV]);
            const v4u va = {half.x, half.y, half.x, half.y};
#pragma unroll
            for (int cb = 0; cb < CB; ++cb) o[cb][db] = E::mfma_k32(va, pb[cb], o[cb][db]);
            if (blk * G::DB + db + kAheadV < G::NB * G::DB) v_ahead[(blk * G::DB + db) % kAheadV] = read_v(blk * G::DB + db + kAheadV);
            __builtin_amdgcn_sched_barrier(0);
          }
        }
      } else {
        // element e of four neighbours of a V row is the operand of block e of O^T: row i of block 4 h + e is d = 64 h + 4 i + e
#pragma unroll
        for (int n = 0; n < kReadsV; ++n) {
          const int h = n % (D / 64), j = n / (D / 64) % 4, blk = n / (D / 64) / 4;
          const f32x4 va = v_ahead[n % kAheadV];
#pragma unroll
          for (int cb = 0; cb < CB; ++cb)
#pragma unroll
            for (int e = 0; e < 4; ++e)
              o[cb][4 * h + e] = __builtin_amdgcn_mfma_f32_16x16x4f32(va[e], sc[cb][blk][j], o[cb][4 * h + e], 0, 0, 0);
          if (n + kAheadV < kReadsV) v_ahead[n % kAheadV] = read_v(n + kAheadV);
          __builtin_amdgcn_sched_barrier(0);
        }
      }
      if (s + 2 * kWaves < n_stages) {
        asm volatile("s_waitcnt lgkmcnt(0)" : : : "memory");  // every operand of this stage has left LDS
        issue(next, c0 + 2 * kWaves * G::TS, lds_ring + buf * 2 * G::HALF);
      }
    }
    seg0 = seg1;
  }

  const int lane = lane_id(), tid = wave * 64 + lane, col = lane & 15, grp = lane >> 4;
  // The wavefronts' states meet in LDS: maxima and sums first, then the accumulators, scaled to the common maximum, PASS column blocks
  // at a time, chunks permuted against bank conflicts.
#pragma unroll
  for (int cb = 0; cb < CB; ++cb) {
    l[cb] += __shfl_xor(l[cb], 16);
    l[cb] += __shfl_xor(l[cb], 32);
    if (grp == 0) *reinterpret_cast<float2*>(sh.ml[wave][cb * 16 + col]) = float2{m[cb], l[cb]};
  }
  lds_barrier();
  {
    float2 ml[CB][kWaves];
#pragma unroll
    for (int cb = 0; cb < CB; ++cb)
#pragma unroll
      for (int w = 0; w < kWaves; ++w) ml[cb][w] = *reinterpret_cast<const float2*>(sh.ml[w][cb * 16 + col]);
    __builtin_amdgcn_sched_barrier(0);  // all reads on their way
#pragma unroll
    for (int cb = 0; cb < CB; ++cb) {
      float mn = -INFINITY, den = 0.f;
#pragma unroll
      for (int w = 0; w < kWaves; ++w) mn = fmaxf(mn, ml[cb][w].x);
      const float ms = safe_max(mn);
#pragma unroll
      for (int w = 0; w < kWaves; ++w) den += ml[cb][w].y * fast_exp2(ml[cb][w].x - ms);
      if (wave == 0 && grp == 0) *reinterpret_cast<float2*>(sh.joined[cb * 16 + col]) = float2{mn, den};
      const float scale = fast_exp2(m[cb] - ms);
#pragma unroll
      for (int db = 0; db < G::DB; ++db) o[cb][db] *= scale;
    }
  }
  const SharedArgs& e = reread();
  const bool sole = !prefix && tile.n_pieces == 1 && tile.t_begin == 0;  // nothing to join: the result itself
  constexpr int C4 = D / 4;  // 16-byte chunks of a row of O
#pragma unroll
  for (int cb0 = 0; cb0 < CB; cb0 += G::PASS) {
    if (cb0 > 0) lds_barrier();  // the pass before has been read
#pragma unroll
    for (int i = 0; i < G::PASS && cb0 + i < CB; ++i) {
      const int cb = cb0 + i;
      f32x4* const acc = reinterpret_cast<f32x4*>(ring) + (i * 16 + col) * C4;
#pragma unroll
      for (int db = 0; db < G::DB; ++db) {
        if constexpr (G::k16) {
          acc[(db * 4 + grp) ^ col] = o[cb][db];
        } else if (db % 4 == 0) {
#pragma unroll
          for (int j = 0; j < 4; ++j)
            acc[(db * 4 + grp * 4 + j) ^ col] = f32x4{o[cb][db][j], o[cb][db + 1][j], o[cb][db + 2][j], o[cb][db + 3][j]};
        }
      }
    }
    lds_barrier();
    // a thread has one chunk of every kStep-th row
    constexpr int kRows = G::PASS < CB ? G::PASS * 16 : CB * 16, kStep = kThreads / C4, kTurns = kRows / kStep;
    const int c = tid % C4, row0 = tid / C4, r0 = cb0 * 16 + row0;
    f32x4 num[kTurns];
    float2 ml[kTurns];
#pragma unroll
    for (int k = 0; k < kTurns; ++k) {
      const int row = row0 + k * kStep;
      ml[k] = *reinterpret_cast<const float2*>(sh.joined[cb0 * 16 + row]);
      num[k] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int w = 0; w < kWaves; ++w) num[k] += reinterpret_cast<const f32x4*>(sh.ring[w])[row * C4 + (c ^ (row & 15))];
    }
    if (sh.tainted) {
#pragma nounroll
      for (int k = 0; k < kTurns; ++k)
        if (r0 + k * kStep < tile.n_rows) {
          f32x4 more = {0.f, 0.f, 0.f, 0.f};
          add_infinities<E, D>(e, tile, r0 + k * kStep, max(t0, least), t1, e.pool_v + static_cast<int64_t>(hc) * e.n_slots * G::ROWB, c, more);
#pragma unroll
          for (int n = 0; n < kTurns; ++n)
            if (n == k) num[n] += more;
        }
    }
    if (sole) {
#pragma unroll
      for (int k = 0; k < kTurns; ++k) {
        if (r0 + k * kStep >= tile.n_rows) break;
        int b, j, g;
        find_row(e, tile, r0 + k * kStep, &b, &j, &g);
        const int h = hc * e.group + g;
        const bool any = keys_of(e, b, j) > 0;
        const float lse = (ml[k].x + log2f(ml[k].y)) * kLn2;
        f32x4 res;
#pragma unroll
        for (int n = 0; n < 4; ++n) res[n] = any ? gated(num[k][n] / ml[k].y, lse, e.sinks, h) : 0.f;
        store4<E>(e.out + b * e.os_b + h * e.os_h + j * e.os_s + c * 4 * E::kBytes, res);
        if (c == 0) e.lse[(static_cast<int64_t>(b) * e.Hq + h) * e.S + j] = any ? lse : -INFINITY;
      }
    } else {
      const int64_t first = (static_cast<int64_t>(tile.part) + static_cast<int64_t>(piece) * tile.n_rows + r0) * e.Hc + hc;
      float* const acc = e.ws_acc + first * D + c * 4;
      float* const mls = e.ws_ml + first * 2;
      const int64_t step = static_cast<int64_t>(kStep) * e.Hc;
#pragma unroll
      for (int k = 0; k < kTurns; ++k) {
        if (r0 + k * kStep >= tile.n_rows) break;
        *reinterpret_cast<f32x4*>(acc + k * step * D) = num[k];
        if (c == 0) *reinterpret_cast<float2*>(mls + k * step * 2) = ml[k];
      }
    }
  }
}

__device__ __forceinline__ bool plan_fits(const SharedArgs& a, const Header& h) {
  return h.magic == kMagic && h.B == a.B && h.S == a.S && h.Hq == a.Hq && h.Hc == a.Hc && h.max_batch == a.max_batch &&
         h.max_context == a.max_context;
}

// A record of the plan, which no launch that reads it writes: scalar loads.
template <typename T>
__device__ __forceinline__ T load_record(const char* p) {
  typedef const __attribute__((address_space(4))) int* ints;
  const ints from = (ints)p;
  T t;
  int* const to = reinterpret_cast<int*>(&t);
#pragma unroll
  for (int i = 0; i < static_cast<int>(sizeof(T) / 4); ++i) to[i] = from[i];
  return t;
}

template <typename E, int D>
__global__ __launch_bounds__(kThreads, (sizeof(Shared<E, D>) <= 80 * 1024 ? 2 : 1)) void shared_products_kernel(const SharedArgs a) {
  __shared__ Shared<E, D> sh;
  const int w = blockIdx.y;
  const Header h = load_record<Header>(a.plan);
  const Share share = load_record<Share>(a.plan + a.shares + w * static_cast<int64_t>(sizeof(Share)));
  if (!plan_fits(a, h) || w >= h.n_wg) return;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  int left = share.units, offset = share.offset, piece = share.piece;
  bool busy = false;
  Tile t = share.first;
  for (int i = share.tile;;) {
    const int all = units_of(t.t_end - t.t_begin);
    const int from = max(0, offset - t.lead), to = min(all, offset + left - t.lead);
    const int t0 = t.t_begin + from * kUnit, t1 = min(t.t_end, t.t_begin + to * kUnit);
    left -= t.lead + all - offset;
    offset = 0;
    if (to > from) {
      if (busy) lds_barrier();  // the piece before has left LDS
      busy = true;
      if (t.n_rows <= 16)
        run_piece<E, D, 1>(a, sh, wave, t, piece, t0, t1);
      else if (t.n_rows <= 32)
        run_piece<E, D, 2>(a, sh, wave, t, piece, t0, t1);
      else
        run_piece<E, D, 4>(a, sh, wave, t, piece, t0, t1);
    }
    i = t.next;
    if (left <= 0 || i >= h.n_tiles) break;
    piece = 0;
    t = load_record<Tile>(a.plan + a.tiles + i * static_cast<int64_t>(sizeof(Tile)));
  }
}

// ------------------------------------------------------------------------------------------------------------ join
// D / 4 lanes have a row, kBatch of its pieces on their way at once.  A row has as many pieces as its keys are cut into, up to one a
// workgroup.  kWide: a workgroup has one row, and where that has more pieces than a batch all of its groups of lanes take some, so
// that they are one trip to memory.
constexpr int kBatch = 8;
// Up to here a row a workgroup: 4 sequences on a prefix of 16000 keys, 64 pieces a row, 16 heads, D 128: a layer 28.3 -> 20.7 us; with pieces in
// one batch it costs 0.2 us a layer (16 sequences, 256 rows) and with 6144 rows 10.
constexpr int kWideRows = 2048;
template <typename E, int D, bool kWide>
__global__ __launch_bounds__(kThreads) void shared_join_kernel(const SharedArgs a) {
  constexpr int LPR = D / 4, kGroups = kThreads / LPR, kRowsHere = kWide ? 1 : kGroups;
  __shared__ float2 s_ml[kGroups];
  __shared__ f32x4 s_acc[kWide ? kGroups : 1][LPR];
  const int c = threadIdx.x % LPR, group = threadIdx.x / LPR, here = kWide ? 0 : group, part = kWide ? group : 0;
  // (32 bits: a division of 64 is a thousand cycles in front of the first load)
  const uint32_t rows = static_cast<uint32_t>(a.B * a.S) * a.Hq, row = blockIdx.x * kRowsHere + here;
  if (row >= rows) return;
  const uint32_t bj = row / static_cast<uint32_t>(a.Hq);
  const int h = static_cast<int>(row - bj * a.Hq);
  const int b = a.S == 1 ? static_cast<int>(bj) : static_cast<int>(bj / static_cast<uint32_t>(a.S)), j = static_cast<int>(bj) - b * a.S;
  const Header head = *reinterpret_cast<const Header*>(a.plan);
  const bool fits = plan_fits(a, head);
  const Sequence s = reinterpret_cast<const Sequence*>(a.plan + a.seqs)[b];
  const int keys = keys_of(a, b, j);
  const int64_t slot = a.batch_idx[b];
  const bool valid = slot >= 0 && slot < a.max_batch;
  const int at_b = !fits || a.S == 1 ? 0 : reinterpret_cast<const int*>(a.plan + a.place)[bj];  // place among the sequence's tokens
  const bool missing = at_b < 0;
  // of another step: the plan
  const bool foreign = !fits || (valid && (s.slot != slot || keys > s.keys || (keys > 0 && missing))) || (!valid && s.slot >= 0);
  const bool any = !foreign && valid && keys > 0;
  float m = -INFINITY, den = 0.f;
  f32x4 num = {0.f, 0.f, 0.f, 0.f};
  bool shared_out = false;
  if (any) {
    const Tile* const tiles = reinterpret_cast<const Tile*>(a.plan + a.tiles);
    const int hc = h >> a.group_shift, x = (at_b << a.group_shift) + (h & (a.group - 1));
    // the prefix's pieces, then those of its own keys
    int n_shared = 0, n_own = 0;
    int64_t at = 0, step = 0, own_at = 0, own_step = 0;  // rows of the workspace
    if (a.S == 1) {
      n_shared = s.n, n_own = s.own_n;
      at = s.at + x, step = s.step;
      own_at = s.own_at + x, own_step = s.own_step;
    } else {
      if (s.prefix_tile >= 0) {
        const int rr = s.prefix_row + x;
        const Tile t = tiles[s.prefix_tile + rr / kTileRows];
        n_shared = t.n_pieces;
        at = t.part + rr % kTileRows;
        step = t.n_rows;
      }
      if (s.own_tile >= 0) {
        const Tile t = tiles[s.own_tile + x / kTileRows];
        n_own = t.n_pieces;
        own_at = t.part + x % kTileRows;
        own_step = t.n_rows;
      }
    }
    if (n_shared == 0 && n_own == 1) return;  // stored already
    const int n = n_shared + n_own;
    shared_out = kWide && n > kBatch;
    if (!shared_out && part > 0) return;
    const int stride = shared_out ? kGroups : 1;
    for (int k0 = part; k0 < n; k0 += kBatch * stride) {
      float2 ml[kBatch];
      f32x4 acc[kBatch];
#pragma unroll
      for (int i = 0; i < kBatch; ++i) {
        const int k = min(k0 + i * stride, n - 1);
        const int64_t p = (k < n_shared ? at + k * step : own_at + (k - n_shared) * own_step) * a.Hc + hc;
        ml[i] = *reinterpret_cast<const float2*>(a.ws_ml + p * 2);
        acc[i] = *reinterpret_cast<const f32x4*>(a.ws_acc + p * D + c * 4);
      }
      float mn = m;
#pragma unroll
      for (int i = 0; i < kBatch; ++i) mn = fmaxf(mn, k0 + i * stride < n ? ml[i].x : -INFINITY);
      const float ms = safe_max(mn), keep = fast_exp2(m - ms);
      den *= keep;
      num *= keep;
#pragma unroll
      for (int i = 0; i < kBatch; ++i) {
        if (k0 + i * stride >= n) break;
        const float w = fast_exp2(ml[i].x - ms);
        den += ml[i].y * w;
        num += acc[i] * w;
      }
      m = mn;
    }
  } else if (part > 0) {
    return;
  }
  if (kWide && shared_out) {
    if (c == 0) s_ml[part] = float2{m, den};
    s_acc[part][c] = num;
    __syncthreads();
    if (part > 0) return;
    float2 ml[kGroups];
    f32x4 acc[kGroups];
#pragma unroll
    for (int i = 0; i < kGroups; ++i) ml[i] = s_ml[i], acc[i] = s_acc[kWide ? i : 0][c];
#pragma unroll
    for (int i = 1; i < kGroups; ++i) m = fmaxf(m, ml[i].x);
    const float ms = safe_max(m);
    den = 0.f;
    num = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < kGroups; ++i) {
      const float w = fast_exp2(ml[i].x - ms);
      den += ml[i].y * w;
      num += acc[i] * w;
    }
  }
  f32x4 res = {0.f, 0.f, 0.f, 0.f};
  float lse = -INFINITY;
  if (foreign) {
    lse = NAN;
    res = f32x4{NAN, NAN, NAN, NAN};
  } else if (any) {
    lse = (m + log2f(den)) * kLn2;
#pragma unroll
    for (int k = 0; k < 4; ++k) res[k] = gated(num[k] / den, lse, a.sinks, h);
  }
  store4<E>(a.out + b * a.os_b + h * a.os_h + j * a.os_s + c * 4 * E::kBytes, res);
  if (c == 0) a.lse[(static_cast<int64_t>(b) * a.Hq + h) * a.S + j] = lse;
}

template <typename E, int D>
void launch(const SharedArgs& a, int n_wg, hipStream_t st) {
  hipLaunchKernelGGL((shared_products_kernel<E, D>), dim3(a.Hc, n_wg), dim3(kThreads), 0, st, a);
  const int64_t rows = static_cast<int64_t>(a.B) * a.S * a.Hq;
  const auto join = [&](auto kernel, int here) {
    hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>((rows + here - 1) / here)), dim3(kThreads), 0, st, a);
  };
  if (rows <= kWideRows)
    join(shared_join_kernel<E, D, true>, 1);
  else
    join(shared_join_kernel<E, D, false>, kThreads / (D / 4));
}

int check_shape(const char* what, int B, int S, int Hq, int Hc, int D) {
  if (B < 0 || S <= 0 || Hq <= 0 || Hc <= 0 || Hq % Hc != 0)
    return fp::fail(FP_ERR_INVALID_ARGUMENT, "%s: bad sizes (B=%d S=%d Hq=%d Hc=%d)", what, B, S, Hq, Hc);
  const int G = Hq / Hc;
  if (D != 64 && D != 128) return fp::fail(FP_ERR_UNSUPPORTED, "%s: head_dim %d (64 or 128)", what, D);
  if (G != 1 && G != 2 && G != 4 && G != 8)
    return fp::fail(FP_ERR_UNSUPPORTED, "%s: %d query heads per cache head (1, 2, 4 or 8)", what, G);
  if (B > kMaxSequences || static_cast<int64_t>(B) * S * G > kMaxRows || static_cast<int64_t>(B) * S * Hq > INT32_MAX)
    return fp::fail(FP_ERR_UNSUPPORTED, "%s: at most %d sequences and %d rows a cached head (got %d of %d tokens, %d heads)", what,
                    kMaxSequences, kMaxRows, B, S, G);
  return FP_OK;
}

}  // namespace

extern "C" int64_t fp_shared_decode_plan_bytes(int32_t B, int32_t S, int32_t Hq, int32_t Hc, int32_t D) {
  if (const int rc = check_shape("fp_shared_decode_plan_bytes", B, S, Hq, Hc, D)) return rc;
  return layout_of(B, S, Hq, Hc).bytes;
}

extern "C" int64_t fp_shared_decode_workspace_bytes(int32_t B, int32_t S, int32_t Hq, int32_t Hc, int32_t D) {
  if (const int rc = check_shape("fp_shared_decode_workspace_bytes", B, S, Hq, Hc, D)) return rc;
  return layout_of(B, S, Hq, Hc).part_rows * Hc * (D + 2) * static_cast<int64_t>(sizeof(float));
}

extern "C" int fp_shared_decode_plan(const int64_t* batch_idx, const void* input_pos, int pos_index_type,
                                     const int32_t* prefix_ids, const int32_t* prefix_lens, int32_t B, int32_t S, int32_t Hq,
                                     int32_t Hc, int32_t D, int32_t max_batch, int32_t max_context, void* plan,
                                     int64_t plan_bytes, void* stream) {
  const char* const what = "fp_shared_decode_plan";
  if (const int rc = check_shape(what, B, S, Hq, Hc, D)) return rc;
  if (max_batch <= 0 || max_context <= 0)
    return fp::fail(FP_ERR_INVALID_ARGUMENT, "%s: max_batch %d, max_context %d", what, max_batch, max_context);
  if (max_context > kMaxContext)
    return fp::fail(FP_ERR_UNSUPPORTED, "%s: max_context %d, at most %d", what, max_context, kMaxContext);
  if (pos_index_type != FP_INDEX_I32 && pos_index_type != FP_INDEX_I64)
    return fp::fail(FP_ERR_INVALID_ARGUMENT, "%s: pos_index_type %d", what, pos_index_type);
  if (B == 0) return FP_OK;
  if (!batch_idx || !input_pos || !prefix_ids || !prefix_lens || !plan)
    return fp::fail(FP_ERR_INVALID_ARGUMENT, "%s: null pointer", what);
  if (plan_bytes < fp_shared_decode_plan_bytes(B, S, Hq, Hc, D) || !fp::aligned(plan, 16))
    return fp::fail(FP_ERR_WORKSPACE, "%s: the plan needs %lld bytes, 16-byte aligned (got %lld)", what,
                    static_cast<long long>(fp_shared_decode_plan_bytes(B, S, Hq, Hc, D)), static_cast<long long>(plan_bytes));
  const Layout l = layout_of(B, S, Hq, Hc);
  const PlanArgs a{batch_idx, input_pos, pos_index_type, prefix_ids, prefix_lens, B, S, Hq, Hc, Hq / Hc, max_batch, max_context,
                   l.n_wg, static_cast<char*>(plan), l.seqs, l.tokens, l.place, l.shares, l.tiles};
  // as many as there are shares, tiles and sequences to write: 64 sequences 2 us less with 512 than with 256, a few no more
  const int threads = S > 1 || B > 64 ? 1024 : B > 24 ? 512 : 256;
  const size_t lds = kPlanArrays * static_cast<size_t>((B + 3) & ~3) * sizeof(int);
  if (lds > 64 * 1024) {
    const hipError_t allowed = hipFuncSetAttribute(reinterpret_cast<const void*>(shared_plan_kernel),
                                                   hipFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(lds));
    if (allowed != hipSuccess) return fp::fail(FP_ERR_LAUNCH, "%s: %s", what, hipGetErrorString(allowed));
  }
  hipLaunchKernelGGL(shared_plan_kernel, dim3(1), dim3(threads), lds, static_cast<hipStream_t>(stream), a);
  return fp::check_launch(what);
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
  if (max_context > kMaxContext)
    return fp::fail(FP_ERR_UNSUPPORTED, "%s: max_context %d, at most %d", what, max_context, kMaxContext);
  if (pos_index_type != FP_INDEX_I32 && pos_index_type != FP_INDEX_I64)
    return fp::fail(FP_ERR_INVALID_ARGUMENT, "%s: pos_index_type %d", what, pos_index_type);
  if (B == 0) return FP_OK;
  if (!q || !pool_k || !pool_v || !page_table || !batch_idx || !input_pos || !out || !lse || !plan)
    return fp::fail(FP_ERR_INVALID_ARGUMENT, "%s: null pointer", what);
  if (!fp::aligned(q, 16) || !fp::aligned(pool_k, 16) || !fp::aligned(pool_v, 16) || !fp::aligned(out, 16) ||
      q_stride_b * e % 16 || q_stride_h * e % 16 || q_stride_s * e % 16 || out_stride_b * e % 16 || out_stride_h * e % 16 ||
      out_stride_s * e % 16)
    return fp::fail(FP_ERR_INVALID_ARGUMENT, "%s: rows of q, out and the pools must be 16-byte aligned", what);
  if (plan_bytes < fp_shared_decode_plan_bytes(B, S, Hq, Hc, D) || !fp::aligned(plan, 16))
    return fp::fail(FP_ERR_WORKSPACE, "%s: plan of %lld bytes is too small, or not 16-byte aligned", what, static_cast<long long>(plan_bytes));
  const int64_t need = fp_shared_decode_workspace_bytes(B, S, Hq, Hc, D);
  if (!workspace || workspace_bytes < need || !fp::aligned(workspace, 16))
    return fp::fail(FP_ERR_WORKSPACE, "%s: workspace of %lld bytes, 16-byte aligned, is needed (got %lld)", what,
                    static_cast<long long>(need), static_cast<long long>(workspace_bytes));
  const Layout l = layout_of(B, S, Hq, Hc);
  const int G = Hq / Hc;
  float* const acc = static_cast<float*>(workspace);
  const SharedArgs a{static_cast<const char*>(q), q_stride_b * e, q_stride_h * e, q_stride_s * e,
                     static_cast<const char*>(pool_k), static_cast<const char*>(pool_v), page_table, pt_row_stride, batch_idx,
                     input_pos, pos_index_type, static_cast<char*>(out), out_stride_b * e, out_stride_h * e, out_stride_s * e,
                     lse, sinks, B, S, Hq, Hc, fp::PageDiv(page_size), n_pages, max_batch,
                     static_cast<int>(n_slots / page_size), n_slots, max_context, scale * kLog2e, G, fp::log2_exact(G),
                     static_cast<const char*>(plan), l.seqs, l.tokens, l.place, l.shares, l.tiles, acc, acc + l.part_rows * Hc * D};
  const hipStream_t st = static_cast<hipStream_t>(stream);
  const auto go = [&](auto element) {
    using E = decltype(element);
    if (D == 64)
      launch<E, 64>(a, l.n_wg, st);
    else
      launch<E, 128>(a, l.n_wg, st);
  };
  if (dtype == FP_DTYPE_F32)
    go(F32{});
  else if (dtype == FP_DTYPE_BF16)
    go(BF16{});
  else
    go(F16{});
  return fp::check_launch(what);
}
