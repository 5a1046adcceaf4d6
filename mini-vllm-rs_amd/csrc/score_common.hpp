// What the kernels of mvr_score.h share on the device: a request's lengths, the
// keys that a query row sees, and the score of a pair.
#pragma once

#include "row_helpers.hpp"
#include "score_attention.hpp"

#include <math.h>

#include <type_traits>

namespace mvr {
namespace {

struct ScoreSeq {
  int seq_len, q_start, q_len;
};

// The tables' loads, an absent table's from one that is there, go out together.
__device__ __forceinline__ ScoreSeq load_score_seq(const ScoreTables& t, int b) {
  typedef const_i32 word;
  const word* any = (const word*)(t.cu_q_lens ? t.cu_q_lens : t.seq_lens ? t.seq_lens : t.block_tables);
  const int seq_len = *(t.seq_lens ? (const word*)t.seq_lens + b : any);
  const int q_start = *(t.cu_q_lens ? (const word*)t.cu_q_lens + b : any);
  const int q_end = *(t.cu_q_lens ? (const word*)t.cu_q_lens + b + 1 : any);
  ScoreSeq s;
  // Clamped to the bounds that the host has checked tables for.  (Rows of a request of
  // length 0 see nothing, but they are rows.)
  s.seq_len = max(t.seq_lens ? min(seq_len, t.max_seq_len) : t.max_seq_len, 0);
  s.q_start = t.cu_q_lens ? q_start : 0;
  s.q_len = max(t.cu_q_lens ? min(q_end - q_start, t.max_q_len) : t.max_q_len, 0);
  return s;
}

// One query row: its slot, the keys [lo, lo + width) that it sees (of no key: lo =
// width = 0), and its head's slope.  Rows of a (request, KV head) are numbered token
// by token, the query heads of a token next to each other: a tile of them spans few
// tokens, whose ranges of keys are nearly one.
struct ScoreRow {
  int pos, lo, width;
  float slope_log2;
};

// prefix: of the request, 0 for none (prefix_of).
__device__ __forceinline__ int prefix_of(const ScoreRules& r, int b) {
  return r.prefix_lens ? ((const const_i32*)r.prefix_lens)[b] : 0;
}

__device__ __forceinline__ int first_key_of(const ScoreRules& r, int token) { return r.first_keys ? r.first_keys[token] : 0; }
__device__ __forceinline__ float slope_of(const ScoreRules& r, int q_head) { return r.slopes ? r.slopes[q_head] : 0.f; }

__device__ __forceinline__ ScoreRow score_row(const ScoreRules& r, const ScoreSeq& s, int prefix, int i, int first_key,
                                              float slope) {
  ScoreRow row;
  row.pos = s.seq_len - s.q_len + i;
  // (Slots below 0, of a request shorter than its query, and negative table entries count as
  // 0 here: no difference leaves 32 bits.)
  int hi = max(max(row.pos + 1, prefix), 0), lo = max(first_key, 0);
  if (r.window > 0) lo = max(lo, max(row.pos, 0) - (r.window - 1));
  hi = min(hi, s.seq_len);
  row.width = max(hi - lo, 0);
  row.lo = row.width ? lo : 0;
  row.slope_log2 = slope * 1.4426950408889634f;
  return row;
}

__device__ __forceinline__ ScoreRow score_row(const ScoreRules& r, const ScoreSeq& s, int prefix, int q_head, int i) {
  return score_row(r, s, prefix, i, first_key_of(r, s.q_start + i), slope_of(r, q_head));
}

__device__ __forceinline__ bool sees(const ScoreRow& row, int key) {
  return (uint32_t)(key - row.lo) < (uint32_t)row.width;
}

// Over the 16 lanes of a DPP row, by rotations: every lane gets the result.
template <typename Op>
__device__ __forceinline__ int row16_reduce(int v, Op op) {
  v = op(v, __builtin_amdgcn_update_dpp(v, v, 0x128, 0xf, 0xf, false)); // row_ror:8
  v = op(v, __builtin_amdgcn_update_dpp(v, v, 0x124, 0xf, 0xf, false));
  v = op(v, __builtin_amdgcn_update_dpp(v, v, 0x122, 0xf, 0xf, false));
  return op(v, __builtin_amdgcn_update_dpp(v, v, 0x121, 0xf, 0xf, false));
}

__device__ __forceinline__ float row16_sum(float v) {
  auto turned = [](float x, auto by) {
    const int bits = __float_as_int(x);
    return __int_as_float(__builtin_amdgcn_update_dpp(bits, bits, decltype(by)::value, 0xf, 0xf, false));
  };
  v += turned(v, std::integral_constant<int, 0x128>()); // row_ror:8
  v += turned(v, std::integral_constant<int, 0x124>());
  v += turned(v, std::integral_constant<int, 0x122>());
  return v + turned(v, std::integral_constant<int, 0x121>());
}

// The keys that any row of a wavefront sees, [begin, end), and those that all do,
// [all_begin, all_end) (empty where a row sees none): the latter need no masks.
struct KeyRange {
  int begin, end, all_begin, all_end;
};

__device__ __forceinline__ void add_row(KeyRange& k, const ScoreRow& row) {
  if (row.width) {
    k.begin = min(k.begin, row.lo);
    k.end = max(k.end, row.lo + row.width);
  }
  k.all_begin = max(k.all_begin, row.lo);
  k.all_end = min(k.all_end, row.lo + row.width);
}

__device__ __forceinline__ KeyRange no_rows() { return {INT32_MAX, 0, 0, INT32_MAX}; }

// Over the query rows of 16 lanes, or of 32 (the other lanes hold the same ones); nothing
// seen: begin = end = 0.
template <int kLanes>
__device__ __forceinline__ KeyRange rows_range(const KeyRange& mine) {
  auto least = [](int a, int b) { return min(a, b); };
  auto most = [](int a, int b) { return max(a, b); };
  auto over = [](int v, auto op) {
    v = row16_reduce(v, op);
    const int first = __builtin_amdgcn_readfirstlane(v);
    return kLanes == 16 ? first : op(first, __builtin_amdgcn_readlane(v, 16));
  };
  KeyRange k = {over(mine.begin, least), over(mine.end, most), over(mine.all_begin, most), over(mine.all_end, least)};
  if (k.end == 0) k.begin = 0;
  return k;
}

// N dot products q . k of one row to scores in log2 units less `minus`,
// x = score * log2(e) - minus; element e is key key0 + offset(e), the offsets constants.
// What the rules lack is left out by branches that all lanes take alike.
//
// A cap costs 7 operations a score while all of them lie in the polynomial's range (those
// of a model that caps them mostly do): its coefficients hold scale, cap and log2(e).
// Past it tanh(y) = 1 - 2 / (e^2y + 1), off by 2^-21 at most; that takes an exponential
// and a reciprocal, 16 cycles each, and loses small values to cancellation, so the scores
// in range take the polynomial also where others are past it: a score is the same number
// whatever the others are.
template <int N, typename Offset>
__device__ __forceinline__ void to_scores(const ScoreRules& r, const ScoreRow& row, float minus, float (&x)[N], int key0,
                                          Offset offset) {
  if (r.cap_log2 > 0.f) {
    float top = 0.f;
#pragma unroll
    for (int e = 0; e < N; e++) top = fmaxf(top, fabsf(x[e]));
    // (A NaN among scores in range takes either way as a NaN.)
    auto in_range = [&](float s, float p) {
      const float u = s * s;
#pragma unroll
      for (int k = 4; k >= 0; k--) p = fmaf(p, u, r.cap_poly[k]);
      return fmaf(s, p, -minus);
    };
    if (__any(!(top <= r.cap_poly_limit))) {
#pragma unroll
      for (int e = 0; e < N; e++) {
        // (One at a time, and nothing that both ways compute, or all scores, worked out
        // before: the other way sets the registers.)
        __builtin_amdgcn_sched_barrier(0);
        float s = x[e], p;
        asm volatile("v_mov_b32 %0, %2" : "=v"(p), "+v"(s) : "s"(r.cap_poly[5]));
        const float ey = __builtin_amdgcn_exp2f(s * r.cap_exp_scale);
        const float past = fmaf(r.cap_log2, fmaf(-2.f, __builtin_amdgcn_rcpf(ey + 1.f), 1.f), -minus);
        x[e] = fabsf(s) <= r.cap_poly_limit ? in_range(s, p) : past;
      }
    } else {
#pragma unroll
      for (int e = 0; e < N; e++) x[e] = in_range(x[e], r.cap_poly[5]);
    }
  } else {
#pragma unroll
    for (int e = 0; e < N; e++) x[e] = fmaf(x[e], r.scale_log2, -minus);
  }
  if (r.slopes) {
    float away = (float)(key0 - row.pos);
    asm volatile("" : "+v"(away)); // (or every element's distance is held over the key loop)
#pragma unroll
    for (int e = 0; e < N; e++) x[e] = fmaf(-row.slope_log2, fabsf(away + (float)offset(e)), x[e]);
  }
}

// `instead` in the place of the scores that the row does not see.
template <int N, typename Offset>
__device__ __forceinline__ void mask_scores(const ScoreRow& row, float (&x)[N], int key0, Offset offset, float instead) {
  int from = key0 - row.lo;
  asm volatile("" : "+v"(from)); // (as above)
#pragma unroll
  for (int e = 0; e < N; e++) x[e] = (uint32_t)(from + offset(e)) < (uint32_t)row.width ? x[e] : instead;
}

// Both.  What the row does not see is taken out before a cap too, whose way to the tanh
// depends on the largest score.
template <int N, typename Offset>
__device__ __forceinline__ void to_masked_scores(const ScoreRules& r, const ScoreRow& row, float minus, float (&x)[N],
                                                 int key0, Offset offset) {
  if (r.cap_log2 > 0.f) mask_scores(row, x, key0, offset, 0.f);
  to_scores(r, row, minus, x, key0, offset);
  mask_scores(row, x, key0, offset, -INFINITY);
}

// The running maximum of a row is where its largest probability is 2^kTopStart, and moves
// once one would exceed 2^kTopLimit: those that enter a product in F16, whose least step
// is 2^-24, are then counted down to some 2^-31 of the largest, which a long cache may
// hold millions of.  (F16 ends at 2^16.)
constexpr float kTopStart = 7.f, kTopLimit = 15.f;

constexpr int kScoreWaves = 4; // wavefronts per block

// Row tile `rt` of request b and KV head h, in place `place`.
struct ScoreTile {
  int b, h, rt;
  int64_t place;
};

// Packed: the last request whose places begin at or before place `at` of its head, by 64
// requests at a time.
template <int kTileRows>
__device__ __forceinline__ int packed_request(const ScoreTables& t, int at, int& begin) {
  auto begin_of = [&](int b) { return (int)((int64_t)t.cu_q_lens[b] * t.group_size / kTileRows) + b; };
  int b = 0;
  for (int n = t.num_seqs; n > 1;) {
    const int step = (n + kWaveSize - 1) / kWaveSize, mine = b + lane_id() * step;
    const int upto = __popcll(__ballot(mine < b + n && begin_of(min(mine, t.num_seqs - 1)) <= at));
    const int skip = max(upto - 1, 0) * step;
    b += skip;
    n = min(step, n - skip);
  }
  b = __builtin_amdgcn_readfirstlane(b);
  begin = __builtin_amdgcn_readfirstlane(begin_of(b));
  return b;
}

// The tile of place `at` of group `group`.  (Its rt may lie behind the request's last tile,
// or before its first where cu_q_lens does not begin at 0.)
template <int kTileRows>
__device__ __forceinline__ ScoreTile tile_at(const ScoreAttentionParams& p, int group, int at) {
  ScoreTile x;
  x.place = (int64_t)group * p.row_tiles + at;
  if (p.packed) {
    int begin;
    x.b = packed_request<kTileRows>(p.t, at, begin);
    x.h = group;
    x.rt = at - begin;
  } else {
    x.b = group / p.t.num_kv_heads;
    x.h = group - x.b * p.t.num_kv_heads;
    x.rt = at;
  }
  return x;
}

template <int kTileRows>
__device__ __forceinline__ bool has_rows(const ScoreTile& x, int rows) {
  return x.rt >= 0 && (int64_t)x.rt * kTileRows < rows;
}

// A block's item: part `part` of the tile of a place.  Items are numbered group by group,
// within one from the last place: the last row tiles first, which a causal mask leaves
// the most keys.  Runs of p.run items go to one XCD (workgroups are dealt to the 8 XCDs
// round-robin): neighbours read the same keys, through one L2.  Every other round deals
// them backwards, so that no XCD gets the longer run of each round.
struct ScoreItem {
  int group, at, part;
};

__device__ __forceinline__ ScoreItem block_item(const ScoreAttentionParams& p) {
  const uint32_t xcd = blockIdx.x % kScoreXcds, of_xcd = blockIdx.x / kScoreXcds, run = (uint32_t)p.run;
  const uint32_t round = of_xcd / run, turn = round % 2 ? kScoreXcds - 1 - xcd : xcd;
  const uint32_t item = (round * kScoreXcds + turn) * run + (of_xcd - round * run);
  const uint32_t inner = (uint32_t)(p.row_tiles * p.parts);
  const uint32_t group = item / inner, rest = item - group * inner, at = rest / (uint32_t)p.parts;
  return {(int)group, p.row_tiles - 1 - (int)at, (int)(rest - at * p.parts)};
}

__device__ __forceinline__ int groups_of(const ScoreAttentionParams& p) {
  return p.packed ? p.t.num_kv_heads : p.t.num_seqs * p.t.num_kv_heads;
}

// First unit of part `part` (of `parts`, 64 at most) of `units`.
__device__ __forceinline__ int part_begin(int part, int units, int parts) {
  return (int)((uint32_t)part * (uint32_t)units / (uint32_t)parts);
}

__device__ __forceinline__ int units_of(const KeyRange& k) {
  return (k.end + kScoreUnitTokens - 1) / kScoreUnitTokens - k.begin / kScoreUnitTokens;
}

// log of sum_j e^score_j from the row's maximum (log2 units) and sum; a row without a
// key, whose sum is 0: -infinity.
__device__ __forceinline__ void store_lse(const ScoreRules& r, int head, int token, float m, float sum) {
  if (r.lse) r.lse[(int64_t)head * r.lse_stride_head + token] = 0.69314718055994531f * (m + __builtin_amdgcn_logf(sum));
}

} // namespace
} // namespace mvr
