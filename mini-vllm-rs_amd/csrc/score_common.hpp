// What the kernels of mvr_score.h share on the device: a request's lengths, the
// keys that a query row sees, and the score of a pair.
#pragma once

#include "row_helpers.hpp"
#include "score_attention.hpp"

#include <math.h>

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
  // Clamped to the bounds that the host has checked tables for.
  s.seq_len = t.seq_lens ? min(seq_len, t.max_seq_len) : t.max_seq_len;
  s.q_start = t.cu_q_lens ? q_start : 0;
  s.q_len = t.cu_q_lens ? min(q_end - q_start, t.max_q_len) : t.max_q_len;
  if (s.seq_len <= 0 || s.q_len <= 0) s.seq_len = s.q_len = 0;
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

__device__ __forceinline__ ScoreRow score_row(const ScoreTables& t, const ScoreRules& r, const ScoreSeq& s, int b,
                                              int q_head, int i) {
  ScoreRow row;
  row.pos = s.seq_len - s.q_len + i;
  int hi = row.pos + 1, lo = 0;
  if (r.prefix_lens) hi = max(hi, r.prefix_lens[b]);
  if (r.first_keys) lo = max(lo, r.first_keys[s.q_start + i]);
  if (r.window > 0) lo = max(lo, row.pos - (r.window - 1));
  hi = min(hi, s.seq_len);
  row.width = max(hi - lo, 0);
  row.lo = row.width ? lo : 0;
  row.slope_log2 = r.slopes ? r.slopes[q_head] * 1.4426950408889634f : 0.f;
  return row;
}

__device__ __forceinline__ bool sees(const ScoreRow& row, int key) {
  return (uint32_t)(key - row.lo) < (uint32_t)row.width;
}

// Smallest, largest over the 64 lanes.
__device__ __forceinline__ int wave_min(int v) {
#pragma unroll
  for (int x = 32; x; x >>= 1) v = min(v, __shfl_xor(v, x));
  return __builtin_amdgcn_readfirstlane(v);
}
__device__ __forceinline__ int wave_max(int v) {
#pragma unroll
  for (int x = 32; x; x >>= 1) v = max(v, __shfl_xor(v, x));
  return __builtin_amdgcn_readfirstlane(v);
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

// Over the wavefront's lanes; nothing seen: begin = end = 0.
__device__ __forceinline__ KeyRange wave_range(const KeyRange& mine) {
  KeyRange k = {wave_min(mine.begin), wave_max(mine.end), wave_max(mine.all_begin), wave_min(mine.all_end)};
  if (k.end == 0) k.begin = 0;
  return k;
}

// tanh(y) / y for |y| <= kTanhPolynomial as a polynomial in u = y^2 that is off by
// 4.4e-9 of it at most (least squares, reweighted towards the largest error); in 32
// bits y * P(u) is within 1.0e-7.  A form with exponentials takes an e^x and a
// reciprocal, 16 cycles each, and loses the small values to cancellation.
constexpr float kTanhPolynomial = 0.625f;
__device__ __forceinline__ float tanh_over(float u) {
  float p = -0.005704979412257671f;
  p = fmaf(p, u, 0.020639080554246902f);
  p = fmaf(p, u, -0.05373971164226532f);
  p = fmaf(p, u, 0.13331441581249237f);
  p = fmaf(p, u, -0.3333328068256378f);
  return fmaf(p, u, 1.0f);
}

// tanh(y), any y: past the polynomial's range 1 - 2 / (e^2|y| + 1), there 0.55 at
// least, so the difference loses no more than one bit.
__device__ __forceinline__ float tanh_any(float y) {
  const float a = fabsf(y);
  const float e = __builtin_amdgcn_exp2f(a * 2.8853900817779268f);
  const float big = copysignf(fmaf(-2.f, __builtin_amdgcn_rcpf(e + 1.f), 1.f), y);
  return a <= kTanhPolynomial ? y * tanh_over(y * y) : big; // (a NaN: big, which is one)
}

// N dot products q . k of one row to scores in log2 units, x = score * log2(e);
// key(e): the key of element e.  What the rules lack is left out by branches that all
// lanes take alike.
template <int N, typename Key>
__device__ __forceinline__ void to_scores(const ScoreRules& r, const ScoreRow& row, float (&x)[N], Key key) {
  if (r.cap_log2 > 0.f) {
    float top = 0.f;
#pragma unroll
    for (int e = 0; e < N; e++) top = fmaxf(top, fabsf(x[e]));
    // (Most scores of a model that caps them are far below the cap.  A NaN among
    // finite scores takes either way as a NaN.)
    if (__any(!(top * r.cap_scale <= kTanhPolynomial))) {
#pragma unroll
      for (int e = 0; e < N; e++) x[e] = r.cap_log2 * tanh_any(x[e] * r.cap_scale);
    } else {
#pragma unroll
      for (int e = 0; e < N; e++) {
        const float y = x[e] * r.cap_scale;
        x[e] = x[e] * r.scale_log2 * tanh_over(y * y);
      }
    }
  } else {
#pragma unroll
    for (int e = 0; e < N; e++) x[e] *= r.scale_log2;
  }
  if (r.slopes) {
#pragma unroll
    for (int e = 0; e < N; e++) x[e] = fmaf(-row.slope_log2, fabsf((float)(key(e) - row.pos)), x[e]);
  }
}

// log of sum_j e^score_j from the row's maximum (log2 units) and sum; a row without a
// key, whose sum is 0: -infinity.
__device__ __forceinline__ void store_lse(const ScoreRules& r, int head, int token, float m, float sum) {
  if (r.lse) r.lse[(int64_t)head * r.lse_stride_head + token] = 0.69314718055994531f * (m + __builtin_amdgcn_logf(sum));
}

} // namespace
} // namespace mvr
