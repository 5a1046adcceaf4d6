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
// flight together), by the exponentials where they are many.  Each weight has one
// writer and one order of its sum.
#include "score_common.hpp"

namespace mvr {
namespace {

constexpr int kWaves = 4; // wavefronts per block

template <typename Tr, int D>
__global__ __launch_bounds__(kWaveSize* kWaves) void score_weights_kernel(ScoreWeightsParams p, int blocks_per_pair) {
  typedef typename Tr::elem T;
  constexpr int kUnit = weights_unit_tokens(sizeof(T), D), kChunks = kUnit / kChunkTokens;
  const ScoreTables& t = p.t;
  const int l = lane_id(), g = l >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWaveSize);
  const int pair = (int)(blockIdx.x / (unsigned)blocks_per_pair);
  const int unit = (int)(blockIdx.x - (unsigned)pair * blocks_per_pair) * kWaves + wave;
  const int b = pair / t.num_kv_heads, h = pair - b * t.num_kv_heads;
  const ScoreSeq s = load_score_seq(t, b);
  const int key0 = unit * kUnit;
  if (key0 >= s.seq_len) return;
  const int rows = t.group_size * s.q_len;

  // Lane l holds the page entry of key key0 + l (lanes past the last key that key's).
  const int my_key = min(key0 + l % kUnit, s.seq_len - 1);
  auto page_div = [&](int x) { return (int)(((uint64_t)(uint32_t)x * t.page_magic) >> t.page_magic_shift); };
  const uint32_t entry = (uint32_t)t.block_tables[(int64_t)b * t.block_table_stride + page_div(my_key)];
  const uint32_t page = min(entry, t.last_page);
  const uint32_t in_page = (uint32_t)(my_key - page_div(my_key) * t.page_size);
  const uint64_t slot = ((uint64_t)page * t.num_kv_heads + h) * (uint32_t)t.page_size + in_page; // of all pools' slots
  // What the key had, and whether it is the lane's to write.
  const bool writes = l < kUnit && key0 + l < s.seq_len && entry <= t.last_page;
  const int fresh = p.fresh_from ? ((const const_i32*)p.fresh_from)[b] : s.seq_len - s.q_len;
  const bool keeps = writes && my_key < fresh && p.decay != 0.f;
  const float had = keeps ? p.weights[slot] : 0.f;

  typename Tr::kreg_t k[kChunks][Tr::kLoads];
#pragma unroll
  for (int c = 0; c < kChunks; c++) {
    const int from = 4 * (16 * c + (l & 15));
    const uint32_t lo = (uint32_t)__builtin_amdgcn_ds_bpermute(from, (int)(uint32_t)slot);
    const uint32_t hi = (uint32_t)__builtin_amdgcn_ds_bpermute(from, (int)(uint32_t)(slot >> 32));
    Tr::load_k_row(static_cast<const T*>(t.key_pool) + (((uint64_t)hi << 32) | lo) * D, l, k[c]);
  }

  float acc[kChunks][4];
#pragma unroll
  for (int c = 0; c < kChunks; c++)
#pragma unroll
    for (int e = 0; e < 4; e++) acc[c][e] = 0.f;

  for (int rho0 = 0; rho0 < rows; rho0 += 16) {
    const int rho = rho0 + (l & 15);
    const bool valid = rho < rows;
    const int i = valid ? rho / t.group_size : 0, head = h * t.group_size + (valid ? rho - i * t.group_size : 0);
    ScoreRow row = score_row(t, p.r, s, b, head, i);
    const float lse = valid ? p.r.lse[(int64_t)head * p.r.lse_stride_head + s.q_start + i] : 0.f;
    if (!valid || lse == -INFINITY) row.width = 0;
    const float lse_log2 = lse * 1.4426950408889634f;
    KeyRange range = no_rows();
    add_row(range, row);
    range = wave_range(range);
    if (range.end <= key0 || range.begin >= key0 + kUnit) continue;
    typename Tr::qreg_t q[Tr::kQRegs];
    Tr::load_q(static_cast<const T*>(t.q) + (int64_t)head * t.q_stride_head + (int64_t)(s.q_start + i) * t.q_stride_token,
               valid, g, q);
    const bool masked = range.all_begin > key0 || range.all_end < key0 + kUnit;
#pragma unroll
    for (int c = 0; c < kChunks; c++) {
      const float4v sc = Tr::qk(k[c], q);
      float x[4] = {sc[0], sc[1], sc[2], sc[3]};
      const int first = key0 + 16 * c + 4 * g;
      to_scores(p.r, row, x, [&](int e) { return first + e; });
#pragma unroll
      for (int e = 0; e < 4; e++) {
        float w = __builtin_amdgcn_exp2f(x[e] - lse_log2);
        if (masked) w = sees(row, first + e) ? w : 0.f;
        acc[c][e] += w;
      }
    }
  }

  // acc[c][e] of lane 16 g + n: key 16 c + 4 g + e, rows n modulo 16.  Four steps, each
  // of which adds one half of the values to the other lane's half, leave lane 16 g + n
  // with the sum of value n.
  float sum[16];
#pragma unroll
  for (int v = 0; v < 16; v++) sum[v] = v < 4 * kChunks ? acc[v / 4 % kChunks][v % 4] : 0.f;
#pragma unroll
  for (int half = 8; half; half >>= 1) {
    const bool upper = l & half;
#pragma unroll
    for (int v = 0; v < half; v++) {
      const float give = upper ? sum[v] : sum[v + half], keep = upper ? sum[v + half] : sum[v];
      sum[v] = keep + __shfl_xor(give, half);
    }
  }
  // Value n = 4 c + e of lane group g is key 16 c + 4 g + e.
  const int c = l >> 4, in_chunk = l & 15;
  const float got = __shfl(sum[0], 16 * (in_chunk >> 2) + 4 * c + (in_chunk & 3));
  if (writes) p.weights[slot] = (keeps ? p.decay * had : 0.f) + got;
}

template <typename Tr, int D>
hipError_t launch(const ScoreWeightsParams& p, hipStream_t stream) {
  constexpr int kUnit = weights_unit_tokens(sizeof(typename Tr::elem), D);
  const int64_t units = ((int64_t)p.t.max_seq_len + kUnit - 1) / kUnit, blocks = (units + kWaves - 1) / kWaves;
  const int64_t pairs = (int64_t)p.t.num_seqs * p.t.num_kv_heads;
  hipLaunchKernelGGL((score_weights_kernel<Tr, D>), dim3((unsigned)(pairs * blocks)), dim3(kWaveSize * kWaves), 0, stream,
                     p, (int)blocks);
  return hipGetLastError();
}

template <int D>
hipError_t launch_type(const ScoreWeightsParams& p, int dtype, hipStream_t stream) {
  return dtype == 1 ? launch<F16Traits<D>, D>(p, stream) : launch<F32Traits<D>, D>(p, stream);
}

} // namespace

hipError_t launch_score_weights(const ScoreWeightsParams& params, int dtype, int head_dim, hipStream_t stream) {
  switch (head_dim) {
  case 32: return launch_type<32>(params, dtype, stream);
  case 64: return launch_type<64>(params, dtype, stream);
  case 96: return launch_type<96>(params, dtype, stream);
  case 128: return launch_type<128>(params, dtype, stream);
  case 160: return launch_type<160>(params, dtype, stream);
  case 192: return launch_type<192>(params, dtype, stream);
  case 224: return launch_type<224>(params, dtype, stream);
  case 256: return launch_type<256>(params, dtype, stream);
  default: return hipErrorInvalidValue;
  }
}

} // namespace mvr
