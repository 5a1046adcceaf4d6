// Attention over a paged cache with bent and masked scores, for gfx950 (MI355X, CDNA4).
//
// Row (token at slot p, query head h) of a request sees the keys lo <= j < hi and
// its output is
//   sum_j e^(x_j - m) v_j / sum_j e^(x_j - m),   m = max_j x_j,
//   x_j = cap * tanh(scale * q . k_j / cap) - slope_h * |p - j|
// (0 where it sees none), its log-sum-exp m + log sum_j e^(x_j - m).  One pass over
// the keys keeps the running maximum and sum of each row in 32 bits (exp2 domain), and
// the results of disjoint key ranges merge exactly:  o = sum_p 2^(m_p - m) o_p, l
// likewise.
//
// What a row sees is one interval of keys, whatever the rules: the causal mask, a
// window, a document and a prefix each move one of its ends.  A row tile loads the keys
// between its rows' first and last, and masks are looked at only in the chunks that not
// every row sees whole.
#include "score_common.hpp"

#include <type_traits>

namespace mvr {
namespace {

// ---------------------------------------------------------------------------
// Key streaming: a block of 4 wavefronts per item, 16 rows, each wavefront its share
// of the part's 16-token chunks straight from the cache; their results merge in LDS.
//
// For rows that are few: bound by HBM where there are blocks enough (32/8 heads of 128 F16:
// 64 single tokens on 300 to 8,192 201 us, 5.2 TB/s; 32 of them with a window of 4,096
// 94 us, 5.7 TB/s), else by the chunks that follow each other in a wavefront, some 1 us
// each (one token on 512, 2 KV heads of 64 F32: 12.2 us whole, 8.8 in 8 parts with their
// merge).  8 and 16 wavefronts to a block: 11.1 and 12.1, whole.  For more rows key tiles
// win: 4 requests of 8 tokens on 2,000 14.1 us here and 19.1 in tiles of 64 rows, of 16
// tokens 20.7 and 20.3, of 32 23.8 and 21.5 (32/8 heads of 128 F16).
// ---------------------------------------------------------------------------
// Chunks of one step: two of F16, whose softmax and products are then one of 32 keys;
// F32 rows hold twice the registers.
template <typename Tr>
constexpr int step_chunks() {
  return sizeof(typename Tr::elem) == 4 ? 1 : 2;
}

// TP: page sizes that are not a multiple of 16, where every token row has a page of its
// own to look up.
template <typename Tr, int D, bool TP>
__global__ __launch_bounds__(kWaveSize* kScoreWaves, (score_stream_blocks_per_cu(sizeof(typename Tr::elem) == 2, D))) void score_stream_kernel(
    ScoreAttentionParams p) {
  typedef typename Tr::elem T;
  constexpr int kTileRows = 16, C = step_chunks<Tr>(), kMergeStride = D + 4;
  constexpr size_t kTileBytes = (size_t)kScoreWaves * C * kChunkTokens * D * sizeof(T);
  constexpr size_t kMergeBytes = (size_t)kScoreWaves * kTileRows * (kMergeStride + 2) * sizeof(float);
  __shared__ __attribute__((aligned(16))) char lds_raw[kTileBytes > kMergeBytes ? kTileBytes : kMergeBytes];
  float* const merge_o = reinterpret_cast<float*>(lds_raw);
  float* const merge_ml = merge_o + kScoreWaves * kTileRows * kMergeStride;

  const int l = lane_id(), g = l >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWaveSize);
  T* const lds = reinterpret_cast<T*>(lds_raw) + (size_t)wave * C * kChunkTokens * D;
  const ScoreItem it = block_item(p);
  const ScoreTables& t = p.t;
  if (it.group >= groups_of(p)) return;
  const ScoreTile tile = tile_at<kTileRows>(p, it.group, it.at);
  const int b = tile.b, h = tile.h;
  const ScoreSeq s = load_score_seq(t, b);
  const int rows = t.group_size * s.q_len;
  if (!has_rows<kTileRows>(tile, rows)) return;

  // The lane's row.
  const int rho = tile.rt * kTileRows + (l & 15);
  const bool valid = rho < rows;
  const int i = valid ? rho / t.group_size : 0, head = h * t.group_size + (valid ? rho - i * t.group_size : 0);
  typename Tr::qreg_t q[Tr::kQRegs];
  Tr::load_q(static_cast<const T*>(t.q) + (int64_t)head * t.q_stride_head + (int64_t)(s.q_start + i) * t.q_stride_token,
             valid, g, q);
  const ScoreRow row = score_row(p.r, s, prefix_of(p.r, b), head, i);
  KeyRange range = no_rows();
  if (valid) add_row(range, row);
  range = rows_range<16>(range);

  // The part's chunks, and the wavefront's.
  const int units = units_of(range), unit0 = range.begin / kScoreUnitTokens;
  const int parts = max(1, min(p.parts, (units + p.part_units - 1) / p.part_units));
  if (it.part >= parts) return;
  if (p.parts > 1 && it.part == 0 && threadIdx.x == 0) p.tile_parts[tile.place] = parts;
  constexpr int kUnitChunks = kScoreUnitTokens / kChunkTokens;
  const int n_chunks = (range.end + kChunkTokens - 1) / kChunkTokens;
  const int part0 = kUnitChunks * (unit0 + part_begin(it.part, units, parts));
  const int part1 = min(kUnitChunks * (unit0 + part_begin(it.part + 1, units, parts)), n_chunks);
  const int k0 = part0 + (int)((int64_t)(part1 - part0) * wave / kScoreWaves);
  const int k1 = part0 + (int)((int64_t)(part1 - part0) * (wave + 1) / kScoreWaves);
  // What the lane's row sees of them.  (A chunk past k1 is seen by nobody.)
  ScoreRow mine = row;
  mine.lo = max(row.lo, k0 * kChunkTokens);
  mine.width = max(0, min(row.lo + row.width, k1 * kChunkTokens) - mine.lo);

  float m = -INFINITY, lsum = 0.f;
  float4v o[D / 16];
#pragma unroll
  for (int n = 0; n < D / 16; n++) o[n] = float4v{0.f, 0.f, 0.f, 0.f};

  const T* kpool = static_cast<const T*>(t.key_pool);
  const T* vpool = static_cast<const T*>(p.value_pool);
  const int32_t* bt = t.block_tables + (int64_t)b * t.block_table_stride;
  auto page_div = [&](int x) { return (int)(((uint64_t)(uint32_t)x * t.page_magic) >> t.page_magic_shift); };
  const uint32_t page_rows = (uint32_t)(t.num_kv_heads * t.page_size), head_rows = (uint32_t)(h * t.page_size);

  // Loads of the C chunks from k on (past k1 the last one again, an L2 hit, rather than
  // a branch).  TP: lane l % 32 holds the page entry of token l % 32, read a step ahead;
  // the lanes get their rows' pages from it.  Rows past the last key read the last
  // key's row (masked, and zeroed in LDS).
  auto token_of = [&](int k, int c, int r) { return min(min(k + c, k1 - 1) * kChunkTokens + r, s.seq_len - 1); };
  auto load_entry = [&](int k) { return (uint32_t)bt[page_div(token_of(k, (l >> 4) % C, l & 15))]; };
  uint32_t entry = 0, next_entry = 0; // TP
  uint64_t chunk_off[C];              // otherwise: element offsets of the chunks
  auto look_up = [&](int k) {
    if constexpr (TP) {
      entry = min(next_entry, t.last_page);
      next_entry = load_entry(k + C);
    } else {
#pragma unroll
      for (int c = 0; c < C; c++) {
        const int x = min(k + c, k1 - 1) * kChunkTokens, pi = page_div(x);
        const uint32_t page = min((uint32_t)((const const_i32*)bt)[__builtin_amdgcn_readfirstlane(pi)], t.last_page);
        chunk_off[c] = ((uint64_t)page * page_rows + head_rows + (uint32_t)(x - pi * t.page_size)) * D;
      }
    }
  };
  auto row_off = [&](int k, int c, int r) { // TP: element offset of a token row of chunk c
    const int x = token_of(k, c, r);
    const uint32_t page = (uint32_t)__builtin_amdgcn_ds_bpermute(4 * (16 * c + r), (int)entry);
    return ((uint64_t)page * page_rows + head_rows + (uint32_t)(x - page_div(x) * t.page_size)) * D;
  };
  // (The lane index is opaque in these, so that the rows' offsets are worked out where
  // they are used and not held, and spilled, over the key loop.)
  auto opaque_lane = [&]() {
    int le = l;
    asm volatile("" : "+v"(le));
    return le;
  };
  auto load_k = [&](int k, typename Tr::kreg_t (&kr)[C][Tr::kLoads]) {
    const int le = opaque_lane();
#pragma unroll
    for (int c = 0; c < C; c++) {
      if constexpr (TP)
        Tr::load_k_row(kpool + row_off(k, c, le & 15), le, kr[c]);
      else
        Tr::load_k(kpool + chunk_off[c], le, kr[c]);
    }
  };
  auto load_v = [&](int k, typename Tr::vreg_t (&vr)[C][Tr::kLoads]) {
    const int le = opaque_lane();
#pragma unroll
    for (int c = 0; c < C; c++) {
      if constexpr (TP) {
#pragma unroll
        for (int u = 0; u < Tr::kLoads; u++)
          vr[c][u] = Tr::load_v_row(vpool + row_off(k, c, Tr::v_row(le, u)), le, u);
      } else {
        Tr::load_v(vpool + chunk_off[c], le, vr[c]);
      }
    }
  };

  // Scores to probabilities.  The running maximum moves, and what the row holds is
  // rescaled, only where a score exceeds it by enough.
  auto softmax = [&](float (&x)[4 * C]) {
    float mx = -INFINITY;
#pragma unroll
    for (int e = 0; e < 4 * C; e++) mx = fmaxf(mx, x[e]);
    mx = row_max(mx);
    const bool grow = mx > m + kTopLimit || (m == -INFINITY && mx != -INFINITY);
    if (__any(grow)) {
      const float m_new = grow ? mx - kTopStart : m;
      const float alpha = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m - m_new);
#pragma unroll
      for (int n = 0; n < D / 16; n++) o[n] *= alpha;
      lsum *= alpha;
      m = m_new;
    }
    const float m_use = m == -INFINITY ? 0.f : m;
#pragma unroll
    for (int e = 0; e < 4 * C; e++) {
      x[e] = __builtin_amdgcn_exp2f(x[e] - m_use);
      lsum += x[e];
    }
  };
  // O^T += V^T P^T of the chunks.  F16: two chunks in one product of 32 keys, lane group
  // g with tokens 4 g .. + 4 of each.  P enters as hi + lo, two F16 numbers whose sum is
  // p but for 2^-20 of it (or 2^-24): both are cut towards 0, p - hi is
  // exact in 32 bits.  (With hi alone outputs are up to 1.8 times as far from the formula
  // as those of a form that holds 32 bits; the second product costs nothing where HBM is
  // the bound.)
  auto pv = [&](int le, const float (&pr)[4 * C]) {
    if constexpr (sizeof(T) == 2) {
      half8 hi, lo;
      float minus = -1.f;
      asm("" : "+s"(minus)); // (opaque: conversion and difference are one v_fma_mix)
#pragma unroll
      for (int e = 0; e < 8; e += 2) {
        const half2v x = __builtin_bit_cast(half2v, __builtin_amdgcn_cvt_pkrtz(pr[e], pr[e + 1]));
        const half2v rest = __builtin_bit_cast(
            half2v, __builtin_amdgcn_cvt_pkrtz(fmaf((float)x[0], minus, pr[e]), fmaf((float)x[1], minus, pr[e + 1])));
        hi[e] = x[0];
        hi[e + 1] = x[1];
        lo[e] = rest[0];
        lo[e + 1] = rest[1];
      }
      const int r = 4 * (le >> 4) + ((le & 15) >> 2), sw = Tr::swz(r);
#pragma unroll
      for (int n = 0; n < D / 16; n++) {
        T* at = lds + r * D + ((n ^ sw) * 16) + 4 * (le & 3);
        const short4v ra = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_short4*)at);
        const short4v rb = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_short4*)(at + kChunkTokens * D));
        const half8 vt = __builtin_bit_cast(half8, __builtin_shufflevector(ra, rb, 0, 1, 2, 3, 4, 5, 6, 7));
        o[n] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vt, lo, o[n], 0, 0, 0);
        o[n] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vt, hi, o[n], 0, 0, 0);
      }
    } else {
#pragma unroll
      for (int c = 0; c < C; c++) {
        float p4[1][4];
#pragma unroll
        for (int e = 0; e < 4; e++) p4[0][e] = pr[4 * c + e];
        float4v (&o1)[1][D / 16] = reinterpret_cast<float4v(&)[1][D / 16]>(o);
        Tr::template pv<1>(lds + c * kChunkTokens * D, le, p4, o1);
      }
    }
  };

  typename Tr::kreg_t kbuf[C][Tr::kLoads];
  typename Tr::vreg_t vbuf[C][Tr::kLoads];
  // One step: the C chunks from k on, whose K and V are in kbuf and vbuf; the next ones
  // are requested as soon as their registers are free.
  auto step = [&](int k, auto masked) {
    constexpr bool kMasked = decltype(masked)::value; // some row does not see all of them
    const int le = opaque_lane();
    float x[4 * C];
#pragma unroll
    for (int c = 0; c < C; c++) {
      const float4v sc = Tr::qk(kbuf[c], q);
#pragma unroll
      for (int e = 0; e < 4; e++) x[4 * c + e] = sc[e];
    }
    look_up(k + C);
    load_k(k + C, kbuf);
    bool bad = false;
    asm volatile("" ::: "memory");
#pragma unroll
    for (int c = 0; c < C; c++) {
      int tokens = kChunkTokens;
      if constexpr (kMasked) {
        tokens = k + c < k1 ? min(s.seq_len - (k + c) * kChunkTokens, kChunkTokens) : 0;
#pragma unroll
        for (int u = 0; u < Tr::kLoads; u++) bad |= Tr::v_row(le, u) < tokens && any_non_finite(vbuf[c][u]);
      }
      Tr::stage_v(lds + c * kChunkTokens * D, le, tokens, vbuf[c]);
    }
    load_v(k + C, vbuf);
    const int first = k * kChunkTokens + 4 * g;
    auto offset = [](int e) { return 16 * (e >> 2) + (e & 3); };
    if constexpr (kMasked)
      to_masked_scores(p.r, mine, 0.f, x, first, offset);
    else
      to_scores(p.r, mine, 0.f, x, first, offset);
    softmax(x);
    // The V tiles are written by this wavefront's own lanes: wait for the LDS writes
    // before reads of other lanes' rows.
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    if constexpr (kMasked) {
      // A V row may hold infinities and NaN: in a product, 0 times one of those would
      // reach the rows that do not see the key.  They are added to the rows that see
      // them one by one, and cleared before the product.
      if (__any(bad)) {
        for (int at = 0; at < C * kChunkTokens; at++) {
          const bool seen = sees(mine, k * kChunkTokens + at);
#pragma unroll
          for (int n = 0; n < D / 16; n++) {
            // The lane's dims 16 n + 4 g + e of the token, where stage_v put them.
            const T* src = lds + at * D + (n ^ Tr::swz(at & 15)) * 16 + 4 * g;
#pragma unroll
            for (int e = 0; e < 4; e++) {
              const float v = non_finite_part(src[e]);
              o[n][e] += seen ? v : 0.f;
            }
          }
        }
        for (int at = l; at < C * kChunkTokens * D; at += kWaveSize) lds[at] = finite_or_zero(lds[at]);
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      }
    }
    pv(le, x);
  };

  if (k0 < k1) {
    if constexpr (TP) next_entry = load_entry(k0);
    look_up(k0);
    load_k(k0, kbuf);
    load_v(k0, vbuf);
    // Steps whose keys every row sees lie in the middle.
    const int clear0 = (range.all_begin + kChunkTokens - 1) / kChunkTokens, clear1 = min(range.all_end / kChunkTokens, k1);
    for (int k = k0; k < k1;) {
      if (k >= clear0)
        for (; k + C <= clear1; k += C) step(k, std::false_type());
      if (k >= k1) break;
      step(k, std::true_type());
      k += C;
    }
  }

  // Every wavefront's rows into LDS over the V tiles, then they are merged, a thread per
  // 4 elements.
  __syncthreads();
  const float ltot = row_sum(lsum);
  float* mine_o = merge_o + (wave * kTileRows + (l & 15)) * kMergeStride;
#pragma unroll
  for (int n = 0; n < D / 16; n++) *reinterpret_cast<float4v*>(mine_o + 16 * n + 4 * g) = o[n];
  if (g == 0) {
    merge_ml[(wave * kTileRows + (l & 15)) * 2 + 0] = m;
    merge_ml[(wave * kTileRows + (l & 15)) * 2 + 1] = ltot;
  }
  __syncthreads();
  constexpr int kCells = kTileRows * (D / 4); // float4 of the tile
  for (int c = threadIdx.x; c < kCells; c += kScoreWaves * kWaveSize) {
    const int rr = c / (D / 4), d = 4 * (c % (D / 4));
    const int at = tile.rt * kTileRows + rr;
    if (at >= rows) break; // rows grow with c
    float mmax = -INFINITY;
#pragma unroll
    for (int j = 0; j < kScoreWaves; j++) mmax = fmaxf(mmax, merge_ml[(j * kTileRows + rr) * 2]);
    const float m_use = mmax == -INFINITY ? 0.f : mmax;
    float4v acc = {0.f, 0.f, 0.f, 0.f};
    float sum = 0.f;
#pragma unroll
    for (int j = 0; j < kScoreWaves; j++) {
      const float w = __builtin_amdgcn_exp2f(merge_ml[(j * kTileRows + rr) * 2] - m_use);
      sum += w * merge_ml[(j * kTileRows + rr) * 2 + 1];
      acc += w * *reinterpret_cast<const float4v*>(merge_o + (j * kTileRows + rr) * kMergeStride + d);
    }
    if (parts > 1) {
      const int64_t prow = (tile.place * p.parts + it.part) * kTileRows + rr;
      *reinterpret_cast<float4v*>(p.partial_o + prow * D + d) = acc;
      if (d == 0) {
        p.partial_ml[prow * 2 + 0] = mmax;
        p.partial_ml[prow * 2 + 1] = sum;
      }
    } else {
      const int ti = at / t.group_size, r = at - ti * t.group_size;
      T* dst = static_cast<T*>(p.out) + (int64_t)(h * t.group_size + r) * p.out_stride_head +
               (int64_t)(s.q_start + ti) * p.out_stride_token + d;
      Tr::store_out(dst, acc * inverse_sum(sum));
      if (d == 0) store_lse(p.r, h * t.group_size + r, s.q_start + ti, mmax, sum);
    }
  }
}

// out = sum_j 2^(m_j - M) o_j / sum_j 2^(m_j - M) l_j over the parts of each row tile
// that was split; one thread per 4 elements, 4 parts' loads in flight, one pass with a
// running maximum.  Bound by its launch and a chain of loads: 3.3 us for a row of 8 parts,
// 5.5 for 512 tiles of 16 rows, 8.5 for 144 of 128 rows in 4 parts.
template <typename Tr, int D, int kTileRows>
__global__ __launch_bounds__(256) void score_merge_kernel(ScoreAttentionParams p) {
  typedef typename Tr::elem T;
  constexpr int kAhead = 4;
  constexpr int kTileBlocks = (kTileRows * (D / 4) + 255) / 256;
  const int c = (int)(blockIdx.x % kTileBlocks) * 256 + threadIdx.x;
  const int rr = c / (D / 4), d = 4 * (c % (D / 4));
  const int place = (int)(blockIdx.x / kTileBlocks), group = place / p.row_tiles;
  const ScoreTile tile = tile_at<kTileRows>(p, group, place - group * p.row_tiles);
  const int b = tile.b, h = tile.h;
  const ScoreSeq s = load_score_seq(p.t, b);
  if (!has_rows<kTileRows>(tile, p.t.group_size * s.q_len)) return; // (its parts were not counted)
  const int rho = tile.rt * kTileRows + rr;
  const int parts = ((const const_i32*)p.tile_parts)[place];
  if (parts <= 1 || rr >= kTileRows || rho >= p.t.group_size * s.q_len) return;
  const int64_t row0 = tile.place * p.parts * kTileRows + rr;
  float4v acc = {0.f, 0.f, 0.f, 0.f};
  float sum = 0.f, m = -INFINITY;
  for (int j0 = 0; j0 < parts; j0 += kAhead) {
    float2v ml[kAhead];
    float4v o[kAhead];
#pragma unroll
    for (int u = 0; u < kAhead; u++) { // (past the last part: the last again, not counted)
      const int64_t row = row0 + (int64_t)min(j0 + u, parts - 1) * kTileRows;
      ml[u] = *reinterpret_cast<const float2v*>(p.partial_ml + row * 2);
      o[u] = *reinterpret_cast<const float4v*>(p.partial_o + row * D + d);
    }
    float m_new = m;
#pragma unroll
    for (int u = 0; u < kAhead; u++) m_new = fmaxf(m_new, ml[u][0]);
    const float m_use = m_new == -INFINITY ? 0.f : m_new;
    const float alpha = __builtin_amdgcn_exp2f(m - m_use);
    acc *= alpha;
    sum *= alpha;
#pragma unroll
    for (int u = 0; u < kAhead; u++) {
      if (j0 + u >= parts) continue; // (no weight of 0: its rows may hold an infinity)
      const float w = __builtin_amdgcn_exp2f(ml[u][0] - m_use);
      sum += w * ml[u][1];
      acc += w * o[u];
    }
    m = m_new;
  }
  const int i = rho / p.t.group_size, head = h * p.t.group_size + (rho - i * p.t.group_size);
  T* dst = static_cast<T*>(p.out) + (int64_t)head * p.out_stride_head + (int64_t)(s.q_start + i) * p.out_stride_token + d;
  Tr::store_out(dst, acc * inverse_sum(sum));
  if (d == 0) store_lse(p.r, head, s.q_start + i, m, sum);
}

template <typename Tr, int D>
hipError_t launch_stream(const ScoreAttentionPlan& plan, const ScoreAttentionParams& p, hipStream_t stream) {
  const dim3 grid(score_blocks(p)), block(kWaveSize * kScoreWaves);
  if (p.t.page_size % kChunkTokens == 0)
    hipLaunchKernelGGL((score_stream_kernel<Tr, D, false>), grid, block, 0, stream, p);
  else
    hipLaunchKernelGGL((score_stream_kernel<Tr, D, true>), grid, block, 0, stream, p);
  return hipGetLastError();
}

template <typename Tr, int D, int kTileRows>
hipError_t launch_merge(const ScoreAttentionPlan& plan, const ScoreAttentionParams& p, hipStream_t stream) {
  constexpr int kTileBlocks = (kTileRows * (D / 4) + 255) / 256;
  const dim3 grid((unsigned)(kTileBlocks * score_groups(p.packed, p.t.num_seqs, p.t.num_kv_heads) * p.row_tiles));
  hipLaunchKernelGGL((score_merge_kernel<Tr, D, kTileRows>), grid, dim3(256), 0, stream, p);
  return hipGetLastError();
}

template <typename Tr, int D>
hipError_t launch_dim(const ScoreAttentionPlan& plan, const ScoreAttentionParams& p, int dtype, hipStream_t stream) {
  const hipError_t err =
      plan.tile_rows == 16 ? launch_stream<Tr, D>(plan, p, stream) : launch_score_tiles(plan, p, dtype, D, stream);
  if (err != hipSuccess || plan.parts == 1) return err;
  switch (plan.tile_rows) {
  case 16: return launch_merge<Tr, D, 16>(plan, p, stream);
  case 64: return launch_merge<Tr, D, 64>(plan, p, stream);
  default: return launch_merge<Tr, D, 128>(plan, p, stream);
  }
}

template <int D>
hipError_t launch_type(const ScoreAttentionPlan& plan, const ScoreAttentionParams& p, int dtype, hipStream_t stream) {
  return dtype == 1 ? launch_dim<F16Traits<D>, D>(plan, p, dtype, stream) : launch_dim<F32Traits<D>, D>(plan, p, dtype, stream);
}

} // namespace

hipError_t launch_score_attention(const ScoreAttentionPlan& plan, const ScoreAttentionParams& params, int dtype,
                                  int head_dim, hipStream_t stream) {
  switch (head_dim) {
  case 32: return launch_type<32>(plan, params, dtype, stream);
  case 64: return launch_type<64>(plan, params, dtype, stream);
  case 96: return launch_type<96>(plan, params, dtype, stream);
  case 128: return launch_type<128>(plan, params, dtype, stream);
  case 160: return launch_type<160>(plan, params, dtype, stream);
  case 192: return launch_type<192>(plan, params, dtype, stream);
  case 224: return launch_type<224>(plan, params, dtype, stream);
  case 256: return launch_type<256>(plan, params, dtype, stream);
  default: return hipErrorInvalidValue;
  }
}

} // namespace mvr
