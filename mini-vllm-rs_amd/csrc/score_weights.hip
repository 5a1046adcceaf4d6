// The weight that cached keys get from query rows, for gfx950 (MI355X, CDNA4).
//
// For key j of a (request, KV head):
//   w_j <- (j < fresh_from ? decay * w_j : 0) + sum over the rows that see j of e^(x_j - L)
// with a row's score x_j and log-sum-exp L as in score_attention.hip.  With every row's
// L known, keys need nothing of each other: a wavefront holds the rows of its keys (64
// of 256 bytes, fewer of longer rows) in registers and takes the query rows past them 16
// at a time; S^T = K Q^T leaves a query row in a lane, so that a row's range, slope and L
// are one register each, and its sums over rows add up lane by lane: the 16 lanes of a
// row tile are summed once, at the end.
//
// Bound by HBM where rows are few (every key is read once, all of a wavefront's loads in
// flight together: 64 single tokens on 8,192, 28/4 heads of 128 F16, 112 us, 4.8 TB/s), by
// the exponentials and the cap where they are many (4 of 32 on 6,000, capped: 24.5 us, with
// 32 keys to a wavefront 28.1).  Each weight has one
// writer and one order of its sum.
#include "score_common.hpp"

namespace mvr {
namespace {

constexpr int kWaves = 4; // wavefronts per block

// Wavefronts per SIMD.  (F32 rows from 512 bytes on hold their queries twice, with the next
// tile's, in up to 128 registers.)
template <typename T, int D>
constexpr int weights_waves() {
  return sizeof(T) == 4 && D >= 128 ? 2 : 3;
}

// SPLIT: the block's wavefronts hold the same keys and take every fourth row tile each
// (their sums add up in LDS); else they hold keys of their own.
template <typename Tr, int D, bool SPLIT>
__global__ __launch_bounds__(kWaveSize* kWaves, (weights_waves<typename Tr::elem, D>())) void score_weights_kernel(
    ScoreWeightsParams p, int blocks_per_pair) {
  typedef typename Tr::elem T;
  constexpr int kUnit = weights_unit_tokens(sizeof(T), D), kChunks = kUnit / kChunkTokens;
  constexpr int kRowStep = SPLIT ? 16 * kWaves : 16;
  const ScoreTables& t = p.t;
  const int l = lane_id(), g = l >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWaveSize);
  const int pair = (int)(blockIdx.x / (unsigned)blocks_per_pair), block = (int)(blockIdx.x - (unsigned)pair * blocks_per_pair);
  const int key0 = (SPLIT ? block : block * kWaves + wave) * kUnit;
  const int b = pair / t.num_kv_heads, h = pair - b * t.num_kv_heads;
  const ScoreSeq s = load_score_seq(t, b);
  if (key0 >= s.seq_len || s.q_len == 0) return; // (SPLIT: the whole block)
  const int rows = t.group_size * s.q_len, prefix = prefix_of(p.r, b);

  // Lane l holds the page entry of key key0 + l (lanes past the last key that key's).
  const int my_key = min(key0 + l % kUnit, s.seq_len - 1);
  auto page_div = [&](int x) { return (int)(((uint64_t)(uint32_t)x * t.page_magic) >> t.page_magic_shift); };
  const uint32_t entry = (uint32_t)t.block_tables[(int64_t)b * t.block_table_stride + page_div(my_key)];

  // The next row tile's queries and rows are on their way while one is computed.
  struct Rows {
    typename Tr::qreg_t q[Tr::kQRegs];
    int i, first_key;
    float slope, lse;
    bool valid;
  };
  int token = (16 * (SPLIT ? wave : 0) + (l & 15)) / t.group_size; // the lane's row of the next tile: token and head
  int in_group = 16 * (SPLIT ? wave : 0) + (l & 15) - token * t.group_size;
  const int token_step = kRowStep / t.group_size, group_step = kRowStep - token_step * t.group_size;
  auto load_rows = [&](Rows& r) {
    r.valid = token < s.q_len;
    const int i = r.valid ? token : 0, head = h * t.group_size + (r.valid ? in_group : 0);
    token += token_step;
    in_group += group_step;
    if (in_group >= t.group_size) {
      in_group -= t.group_size;
      token++;
    }
    r.lse = p.r.lse[(int64_t)head * p.r.lse_stride_head + s.q_start + i];
    r.i = i;
    r.first_key = first_key_of(p.r, s.q_start + i);
    r.slope = slope_of(p.r, head);
    Tr::load_q(static_cast<const T*>(t.q) + (int64_t)head * t.q_stride_head + (int64_t)(s.q_start + i) * t.q_stride_token,
               r.valid, g, r.q);
  };
  Rows next;
  int rho0 = SPLIT ? 16 * wave : 0;
  if (rho0 < rows) load_rows(next);

  const uint32_t page = min(entry, t.last_page);
  const uint32_t in_page = (uint32_t)(my_key - page_div(my_key) * t.page_size);
  const uint64_t slot = ((uint64_t)page * t.num_kv_heads + h) * (uint32_t)t.page_size + in_page; // of all pools' slots
  typename Tr::kreg_t k[kChunks][Tr::kLoads];
#pragma unroll
  for (int c = 0; c < kChunks; c++) {
    const int from = 4 * (16 * c + (l & 15));
    const uint32_t lo = (uint32_t)__builtin_amdgcn_ds_bpermute(from, (int)(uint32_t)slot);
    const uint32_t hi = (uint32_t)__builtin_amdgcn_ds_bpermute(from, (int)(uint32_t)(slot >> 32));
    Tr::load_k_row(static_cast<const T*>(t.key_pool) + (((uint64_t)hi << 32) | lo) * D, l, k[c]);
  }
  // What the key had, and whether it is the lane's to write.
  const bool writes = l < kUnit && key0 + l < s.seq_len && entry <= t.last_page && (!SPLIT || wave == 0);
  const int fresh = p.fresh_from ? ((const const_i32*)p.fresh_from)[b] : s.seq_len - s.q_len;
  const bool keeps = writes && my_key < fresh && p.decay != 0.f;
  const float had = keeps ? p.weights[slot] : 0.f;
  __shared__ uint64_t slots[kWaves][kWaveSize]; // (each lane's own: no register holds it over the rows)
  slots[wave][l] = slot;

  float acc[4 * kChunks];
#pragma unroll
  for (int v = 0; v < 4 * kChunks; v++) acc[v] = 0.f;

  for (; rho0 < rows; rho0 += kRowStep) {
    Rows r = next;
    if (rho0 + kRowStep < rows) load_rows(next);
    ScoreRow row = score_row(p.r, s, prefix, r.i, r.first_key, r.slope);
    if (!r.valid || r.lse == -INFINITY) row.width = 0;
    const float lse_log2 = r.lse * 1.4426950408889634f;
    const int end = row.lo + row.width;
    if (!__any(row.width && end > key0 && row.lo < key0 + kUnit)) continue;
    const bool masked = __any(end < key0 + kUnit || row.lo > key0); // some row does not see all the keys
    float x[4 * kChunks];
#pragma unroll
    for (int c = 0; c < kChunks; c++) {
      const float4v sc = Tr::qk(k[c], r.q);
#pragma unroll
      for (int e = 0; e < 4; e++) x[4 * c + e] = sc[e];
    }
    auto offset = [](int e) { return 16 * (e >> 2) + (e & 3); };
    if (masked)
      to_masked_scores(p.r, row, lse_log2, x, key0 + 4 * g, offset);
    else
      to_scores(p.r, row, lse_log2, x, key0 + 4 * g, offset);
#pragma unroll
    for (int e = 0; e < 4 * kChunks; e++) acc[e] += __builtin_amdgcn_exp2f(x[e]);
  }

  // acc[4 c + e] of lane 16 g + n: key 16 c + 4 g + e, rows n modulo 16.  Summed over a
  // group's lanes, the lane l takes key l's.
  const int want = 4 * (l >> 4) + (l & 3); // (of group (l & 15) / 4)
  float mine = 0.f;
#pragma unroll
  for (int v = 0; v < 4 * kChunks; v++) {
    const float sum = row16_sum(acc[v]);
    mine = (l & 15) == v ? sum : mine;
  }
  float got = __shfl(mine, 16 * ((l & 15) >> 2) + want);
  if constexpr (SPLIT) {
    __shared__ float sums[kWaves][kWaveSize];
    sums[wave][l] = got;
    __syncthreads();
    got = ((sums[0][l] + sums[1][l]) + sums[2][l]) + sums[3][l];
  }
  if (writes) p.weights[slots[wave][l]] = (keeps ? p.decay * had : 0.f) + got;
}

template <typename Tr, int D>
hipError_t launch(const ScoreWeightsParams& p, bool split, hipStream_t stream) {
  constexpr int kUnit = weights_unit_tokens(sizeof(typename Tr::elem), D);
  const int64_t units = ((int64_t)p.t.max_seq_len + kUnit - 1) / kUnit, blocks = (units + kWaves - 1) / kWaves;
  const int64_t pairs = (int64_t)p.t.num_seqs * p.t.num_kv_heads;
  const dim3 block(kWaveSize * kWaves);
  if (split)
    hipLaunchKernelGGL((score_weights_kernel<Tr, D, true>), dim3((unsigned)(pairs * units)), block, 0, stream, p, (int)units);
  else
    hipLaunchKernelGGL((score_weights_kernel<Tr, D, false>), dim3((unsigned)(pairs * blocks)), block, 0, stream, p, (int)blocks);
  return hipGetLastError();
}

template <int D>
hipError_t launch_type(const ScoreWeightsParams& p, int dtype, bool split, hipStream_t stream) {
  return dtype == 1 ? launch<F16Traits<D>, D>(p, split, stream) : launch<F32Traits<D>, D>(p, split, stream);
}

} // namespace

hipError_t launch_score_weights(const ScoreWeightsParams& params, int dtype, int head_dim, bool split, hipStream_t stream) {
  switch (head_dim) {
  case 32: return launch_type<32>(params, dtype, split, stream);
  case 64: return launch_type<64>(params, dtype, split, stream);
  case 96: return launch_type<96>(params, dtype, split, stream);
  case 128: return launch_type<128>(params, dtype, split, stream);
  case 160: return launch_type<160>(params, dtype, split, stream);
  case 192: return launch_type<192>(params, dtype, split, stream);
  case 224: return launch_type<224>(params, dtype, split, stream);
  case 256: return launch_type<256>(params, dtype, split, stream);
  default: return hipErrorInvalidValue;
  }
}

} // namespace mvr
