// Attention with bent and masked scores of many rows per KV head, for gfx950: key tiles
// in LDS, 32x32 MFMAs.  The mathematics is score_attention.hip's.
//
// A block of 4 wavefronts holds a row tile of 32 * RW rows of one (request, KV head), 32
// rows per wavefront, in G = 4 / RW groups of RW wavefronts that hold the same rows and
// take alternating key tiles.  Each step stages G key tiles of K and V in LDS, loaded
// straight from the pages (buffer_load ... lds) one step or more ahead; every wavefront of
// a group reads them from there, so a key's bytes leave the cache once per row tile.
//   S^T = K Q^T   K from LDS as the A operand, Q^T in registers; a lane holds row l % 32, so
//                 that its range, slope and sums are one register each;
//   O^T += V^T P^T  V through transposing LDS reads (F16), P^T from the S^T registers.
// Rows are numbered token by token, so a tile's rows see nearly the same keys: it loads
// those that any of them sees, tests masks in the steps at the ends only, and a wavefront
// whose rows see nothing of a step leaves it out.
//
// Bound by the vector unit and the matrix pipe in turn: a score takes its scale,
// exponential, sum and rounding, and a cap as many operations again, while the two
// products of its 32 x 32 block take the matrix pipe half that time.  28/4 heads of 128
// F16: a prompt of 8,192 549 us, 0.88 PFLOP/s; four of 256 on 2,048 with a cap 57.6 us,
// 0.56.  F32 by the matrix pipe: three of 217 on up to 1,218 130 us, 75% busy in the CUs
// that have a block.
//
// 64 rows (two groups) where rows are few, 128 where a key's bytes should serve more of
// them, in 4 wavefronts, two blocks to a CU, or in 8, one, where blocks are fewer than
// CUs.  32/8 heads of 128 F16, unsplit, 64 rows, 128, 128 in 8 wavefronts: 32 requests of
// 16 tokens on 4,000 102, 107 and 100 us (16 rows streamed: 179); a prompt of 2,000 57, 59
// and 57 (170); documents of 1,500 in a prompt of 6,000 178, 163 and 183 (163 to 172 in 128
// on other days).
#include "key_tiles.hpp"
#include "score_common.hpp"

#include <type_traits>

namespace mvr {
namespace {

// W: wavefronts.  S: LDS stages; S - 1 steps' loads are in flight while a step is computed.
template <int D, typename T, int RW, int W, int PAGES, int S>
__global__ __launch_bounds__(kWaveSize* W, (score_tile_waves_per_simd(32 * RW, W, sizeof(T) == 2, D))) void score_tile_kernel(
    ScoreAttentionParams p) {
  typedef Tile<D, T, RW, W> TL;
  constexpr bool kF32 = TL::kF32;
  constexpr int kTileTokens = TL::kTileTokens, kSub = TL::kSub, G = TL::kGroups;
  constexpr int kTileRows = 32 * RW;
  typedef typename std::conditional<kF32, float4v, half8>::type qfrag_t;
  constexpr int kQFrags = kF32 ? D / 8 : D / 16;
  // One object per stage and operand: the compiler follows the loads into LDS by
  // object, so a read of one stage does not wait for another's.
  __shared__ __attribute__((aligned(16))) T k_lds0[TL::kElems], k_lds1[TL::kElems], k_lds2[TL::kElems],
      k_lds3[TL::kElems];
  __shared__ __attribute__((aligned(16))) T v_lds0[TL::kElems], v_lds1[TL::kElems], v_lds2[TL::kElems],
      v_lds3[TL::kElems];
  __shared__ float ml_xfer[RW][2][64]; // hand-off between groups (O goes through the stages)
  __shared__ __attribute__((aligned(16))) int non_finite[S][W]; // by stage: what each wavefront loaded holds any
  static_assert(S >= 2 && S <= 4, "2, 3 or 4 stages");
  T* const k_st[4] = {k_lds0, k_lds1, k_lds2, k_lds3};
  T* const v_st[4] = {v_lds0, v_lds1, v_lds2, v_lds3};

  const int l = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int rw = wave % RW, grp = wave / RW, hh = l >> 5;
  const ScoreItem it = block_item(p);
  const ScoreTables& t = p.t;
  if (it.group >= groups_of(p)) return;
  const ScoreTile tile = tile_at<kTileRows>(p, it.group, it.at);
  const int b = tile.b, h = tile.h;
  const ScoreSeq s = load_score_seq(t, b);
  const int rows = t.group_size * s.q_len;
  if (!has_rows<kTileRows>(tile, rows)) return;

  // The lane's row: query token i, query head of the KV head's group.
  auto row_at = [&](int rho, int& i, int& head) {
    const bool valid = rho < rows;
    i = valid ? rho / t.group_size : 0;
    head = h * t.group_size + (valid ? rho - i * t.group_size : 0);
    return valid;
  };
  const int rho0 = tile.rt * kTileRows + rw * 32; // the wavefront's first row
  const bool live = rho0 < rows;                // it has rows
  ScoreRow row;
  // Q^T as the B operand: lane l holds row l % 32, dims 16 st + 8 hh .. + 8 (F32: 8 st + 4 hh .. + 4).
  qfrag_t q[kQFrags];
  KeyRange mine = no_rows(); // what the wavefront's rows see
  {
    int token, head;
    const bool valid = row_at(rho0 + (l & 31), token, head);
    const T* qrow = static_cast<const T*>(t.q) + (int64_t)head * t.q_stride_head + (int64_t)(s.q_start + token) * t.q_stride_token;
    constexpr int kFragDims = kF32 ? 8 : 16;
#pragma unroll
    for (int st = 0; st < kQFrags; st++)
      q[st] = valid ? *reinterpret_cast<const qfrag_t*>(qrow + kFragDims * st + (kFragDims / 2) * hh) : qfrag_t{};
    row = score_row(p.r, s, prefix_of(p.r, b), head, token);
    if (valid) add_row(mine, row);
  }
  mine = rows_range<32>(mine);
  // And the block's.
  __shared__ int ranges[RW][4];
  if (grp == 0 && l == 0) {
    ranges[rw][0] = mine.end ? mine.begin : INT32_MAX;
    ranges[rw][1] = mine.end;
    ranges[rw][2] = mine.all_begin;
    ranges[rw][3] = mine.all_end;
  }
  __syncthreads();
  KeyRange range = no_rows();
#pragma unroll
  for (int w = 0; w < RW; w++)
    range = {min(range.begin, ranges[w][0]), max(range.end, ranges[w][1]), max(range.all_begin, ranges[w][2]),
             min(range.all_end, ranges[w][3])};
  auto uniform = [](int v) { return __builtin_amdgcn_readfirstlane(v); };
  range = {uniform(range.end ? range.begin : 0), uniform(range.end), uniform(range.all_begin), uniform(range.all_end)};

  // The part's key tiles [j0, j1).
  const int units = units_of(range), unit0 = range.begin / kScoreUnitTokens;
  const int parts = max(1, min(p.parts, (units + p.part_units - 1) / p.part_units));
  if (it.part >= parts) return;
  if (p.parts > 1 && it.part == 0 && threadIdx.x == 0) p.tile_parts[tile.place] = parts;
  constexpr int kUnitTiles = kScoreUnitTokens / kTileTokens;
  const int n_tiles = (range.end + kTileTokens - 1) / kTileTokens;
  const int j0 = kUnitTiles * (unit0 + part_begin(it.part, units, parts));
  const int j1 = min(kUnitTiles * (unit0 + part_begin(it.part + 1, units, parts)), n_tiles);

  float16v o[D / 32];
#pragma unroll
  for (int n = 0; n < D / 32; n++)
#pragma unroll
    for (int e = 0; e < 16; e++) o[n][e] = 0.f;
  float m = -INFINITY, lsum = 0.f;

  // Staging.  Wavefront w fills the stage's token rows from w * kWaveTokens on;
  // its load u writes LDS chunks (w * kLoads + u) * 64 + lane, and each lane reads
  // the chunk of the row that the swizzle puts there.
  const const_i32* bt = (const const_i32*)(t.block_tables) + (int64_t)b * t.block_table_stride;
  auto page_div = [&](int x) { return (int)(((uint64_t)(uint32_t)x * t.page_magic) >> t.page_magic_shift); };
  constexpr uint32_t kRowBytes = D * (uint32_t)sizeof(T);
  const uint32_t page_rows = (uint32_t)(t.num_kv_heads * t.page_size), head_rows = (uint32_t)(h * t.page_size);
  auto rows_at = [&](uint32_t page, uint32_t at) {
    return ((uint64_t)min(page, t.last_page) * page_rows + (head_rows + at)) * kRowBytes;
  };
  // Bytes from the wavefront's first token row (kWholeLoads: the load's; kAnyPages: within the row).
  constexpr int kLoadTokens = PAGES == kWholeLoads ? 64 / TL::kChunksPerRow : 1;
  static_assert(PAGES != kWholeLoads || 64 % TL::kChunksPerRow == 0, "loads of whole token rows");
  uint32_t off_k[TL::kLoads], off_v[TL::kLoads];
#pragma unroll
  for (int u = 0; u < TL::kLoads; u++) {
    const int P = (wave * TL::kLoads + u) * 64 + l;
    const int tr = P / TL::kChunksPerRow, cs = P % TL::kChunksPerRow;
    const int dt = PAGES == kRuns ? tr - wave * TL::kWaveTokens : PAGES == kWholeLoads ? l / TL::kChunksPerRow : 0;
    off_k[u] = (uint32_t)(dt * D + TL::kChunkElems * (cs ^ TL::kswz(tr))) * sizeof(T);
    off_v[u] = (uint32_t)(dt * D + TL::kChunkElems * (2 * ((cs >> 1) ^ TL::vswz(tr)) + (cs & 1))) * sizeof(T);
  }
  const int n_steps = (j1 - j0 + G - 1) / G, last_step = n_steps - 1;
  const int last_key = s.seq_len - 1;
  // First token of the wavefront's load u in step si (kRuns: of all its loads), or
  // the last key past the end (those tokens are masked).
  auto first_token = [&](int si, int u) {
    return min((j0 + G * si) * kTileTokens + wave * TL::kWaveTokens + u * kLoadTokens, last_key);
  };
  // Block-table entries are read a step ahead of their loads: waiting for a scalar
  // load would also wait for every LDS read in flight.
  struct Entries {
    uint32_t page[PAGES == kWholeLoads ? TL::kLoads : 1];
  };
  auto fetch_pages = [&](int si) {
    Entries e{};
    if constexpr (PAGES == kRuns) e.page[0] = (uint32_t)bt[page_div(first_token(si, 0))];
    if constexpr (PAGES == kWholeLoads) {
#pragma unroll
      for (int u = 0; u < TL::kLoads; u++) e.page[u] = (uint32_t)bt[page_div(first_token(si, u))];
    }
    return e;
  };
  auto issue_stage = [&](int si, const Entries& entries, T* kb, T* vb) __attribute__((always_inline)) {
    const char* kpool = static_cast<const char*>(t.key_pool);
    const char* vpool = static_cast<const char*>(p.value_pool);
    if constexpr (PAGES == kAnyPages) {
      // A load's tokens may lie in several pages, which take their lanes in turn.
      // Lanes of tokens past the last key go with the last page, whose bound reads them
      // as zeros.
      const int last_page_index = page_div(last_key);
#pragma unroll
      for (int u = 0; u < TL::kLoads; u++) {
        const int P = (wave * TL::kLoads + u) * 64;
        const int t0 = (j0 + G * si) * kTileTokens;
        const int key = t0 + (P + l) / TL::kChunksPerRow;
        const int page_index = min(page_div(key), last_page_index);
        const uint32_t row_off = (uint32_t)(key - page_index * t.page_size) * kRowBytes;
        const int first = min(page_div(t0 + P / TL::kChunksPerRow), last_page_index);
        const int last = min(page_div(t0 + (P + 63) / TL::kChunksPerRow), last_page_index);
        for (int pi = first; pi <= last; pi++) { // wave-uniform
          const uint64_t at = rows_at((uint32_t)bt[pi], 0);
          const uint32_t bytes = (uint32_t)min(t.page_size, s.seq_len - pi * t.page_size) * kRowBytes;
          if (page_index == pi) {
            load_to_lds16(kpool + at, bytes, row_off + off_k[u], kb + P * TL::kChunkElems);
            load_to_lds16(vpool + at, bytes, row_off + off_v[u], vb + P * TL::kChunkElems);
          }
        }
      }
    } else {
      // All wave-uniform: a run's first token, its page row, and the bytes from
      // there to the run's end, or the end of the keys.
      constexpr int kRunTokens = PAGES == kRuns ? TL::kWaveTokens : kLoadTokens;
      uint64_t at = 0;
      uint32_t bytes = 0;
#pragma unroll
      for (int u = 0; u < TL::kLoads; u++) {
        if (u == 0 || PAGES == kWholeLoads) {
          const int key = first_token(si, u);
          at = rows_at(entries.page[PAGES == kWholeLoads ? u : 0], (uint32_t)(key - page_div(key) * t.page_size));
          bytes = (uint32_t)min(s.seq_len - key, kRunTokens) * kRowBytes;
        }
        const int dst = (wave * TL::kLoads + u) * 64 * TL::kChunkElems;
        load_to_lds16(kpool + at, bytes, off_k[u], kb + dst);
        load_to_lds16(vpool + at, bytes, off_v[u], vb + dst);
      }
    }
  };

  // LDS read offsets within the group's rows of a stage.  K: token l % 32, chunk
  // 2 st + hh.  V (F16): step u reads rows 16 u + 4 hh + ... through the
  // transposing read; V (F32): D/32 consecutive elements of one row.
  const int gbase = grp * kTileTokens * D;
  constexpr int kKReads = kF32 ? D / 8 : D / 16;
  constexpr int kKOffs = kKReads > 8 ? 8 : kKReads;
  int rk[kKOffs];
#pragma unroll
  for (int st = 0; st < kKOffs; st++)
    rk[st] = gbase + (l & 31) * D + TL::kChunkElems * ((2 * st + hh) ^ TL::kswz(l & 31));
  int rv[kF32 ? 1 : D / 32];
  if constexpr (kF32) {
    rv[0] = gbase + 4 * hh * D + (D / 32) * (l & 31);
  } else {
#pragma unroll
    for (int n = 0; n < D / 32; n++) {
      const int vr = 4 * hh + ((l & 15) >> 2), col = 32 * n + 16 * ((l >> 4) & 1) + 4 * (l & 3);
      rv[n] = gbase + vr * D + ((col >> 4) ^ TL::vswz(vr)) * 16 + (col & 15);
    }
  }

  auto qk = [&](const T* kb, float16v (&acc)[kSub]) __attribute__((always_inline)) {
#pragma unroll
    for (int c = 0; c < kSub; c++)
#pragma unroll
      for (int e = 0; e < 16; e++) acc[c][e] = 0.f;
    if constexpr (kF32) {
#pragma unroll
      for (int st = 0; st < kKReads; st++) {
        const float4v kf = *reinterpret_cast<const float4v*>(kb + rk[st % kKOffs] + (st / kKOffs) * 64);
#pragma unroll
        for (int c = 0; c < 4; c++) acc[0] = __builtin_amdgcn_mfma_f32_32x32x2f32(kf[c], q[st][c], acc[0], 0, 0, 0);
      }
    } else {
#pragma unroll
      for (int st = 0; st < D / 16; st++)
#pragma unroll
        for (int c = 0; c < kSub; c++)
          acc[c] = __builtin_amdgcn_mfma_f32_32x32x16_f16(
              *reinterpret_cast<const half8*>(kb + rk[st % kKOffs] + (st / kKOffs) * 128 + 32 * c * D), q[st], acc[c],
              0, 0, 0);
    }
  };
  // In block c the lane holds tokens 32 c + 8 (e / 4) + 4 hh + e % 4 of its row.
  // Scores less the running maximum (log2 units), which moves, and O and the sum with it,
  // only where a score exceeds it by enough; then P = 2^x in place, and its sum.
  // F16: the product with V takes P rounded to F16 (half a step, 2^-11 of p), the sum
  // holds 32 bits.  Outputs are 1.4 times as far from the formula as with all of P (2.9e-4
  // of them against 2.1e-4, the rounding of the output itself).  A second product, with
  // what the rounding leaves, is the matrix pipe's half again: four of 256 on 2,048 with a
  // cap 57.5 -> 65.1 us, documents 163 -> 193, a prompt of 8,192 537 -> 711 (interleaved
  // with the exponentials 704), 32 requests of 16 tokens on 4,000 102 -> 104.  The
  // streaming kernel, bound by HBM, has it.
  auto softmax = [&](float16v (&sc)[kSub], int first, bool masked) __attribute__((always_inline)) { // first: the tile's first key
    float x[16 * kSub];
#pragma unroll
    for (int e = 0; e < 16 * kSub; e++) x[e] = sc[e / 16][e % 16];
    auto offset = [](int e) { return 32 * (e / 16) + 8 * (e % 16 / 4) + e % 4; };
    const bool cap = masked && p.r.cap_log2 > 0.f; // (as to_masked_scores, its code once)
    if (cap) mask_scores(row, x, first + 4 * hh, offset, 0.f);
    to_scores(p.r, row, m == -INFINITY ? 0.f : m, x, first + 4 * hh, offset);
    if (masked) mask_scores(row, x, first + 4 * hh, offset, -INFINITY);
    float mx = -INFINITY;
#pragma unroll
    for (int e = 0; e < 16 * kSub; e += 4) mx = fmaxf(mx, fmaxf(fmaxf(x[e], x[e + 1]), fmaxf(x[e + 2], x[e + 3])));
    const auto sw = __builtin_amdgcn_permlane32_swap(__float_as_uint(mx), __float_as_uint(mx), false, false);
    mx = fmaxf(__uint_as_float(sw[0]), __uint_as_float(sw[1]));
    const bool grow = mx > kTopLimit || (m == -INFINITY && mx != -INFINITY);
    if (__any(grow)) {
      const float up = grow ? mx - kTopStart : 0.f;
      const float alpha = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(-up);
#pragma unroll
      for (int n = 0; n < D / 32; n++) o[n] *= alpha;
      lsum *= alpha;
      m = grow ? (m == -INFINITY ? up : m + up) : m;
#pragma unroll
      for (int e = 0; e < 16 * kSub; e++) x[e] -= up;
    }
    float psum = 0.f;
#pragma unroll
    for (int e = 0; e < 16 * kSub; e++) {
      x[e] = __builtin_amdgcn_exp2f(x[e]);
      psum += x[e];
      sc[e / 16][e % 16] = x[e];
    }
    lsum += psum;
  };
  // Probabilities e and e + 1 of block c as the product with V takes them.
  auto halves = [&](const float16v (&sc)[kSub], int c, int e) {
    return __builtin_convertvector((float2v{sc[c][e], sc[c][e + 1]}), half2v);
  };
  auto pv = [&](const T* vb, const float16v (&sc)[kSub]) __attribute__((always_inline)) {
    if constexpr (kF32) {
      // Product e pairs tokens 8 (e / 4) + e % 4 and + 4, which the lane halves
      // hold; O^T block n holds dims (D / 32) * row + n.
#pragma unroll
      for (int e = 0; e < 16; e++) {
        const T* src = vb + rv[0] + (8 * (e >> 2) + (e & 3)) * D;
#pragma unroll
        for (int n = 0; n < D / 32; n++) o[n] = __builtin_amdgcn_mfma_f32_32x32x2f32(src[n], sc[0][e], o[n], 0, 0, 0);
      }
    } else {
      half8 pb[2 * kSub];
#pragma unroll
      for (int u = 0; u < 2 * kSub; u++)
#pragma unroll
        for (int e = 0; e < 8; e += 2) {
          const half2v p2 = halves(sc, u >> 1, 8 * (u & 1) + e);
          pb[u][e] = p2[0];
          pb[u][e + 1] = p2[1];
        }
#pragma unroll
      for (int n = 0; n < D / 32; n++)
#pragma unroll
        for (int u = 0; u < 2 * kSub; u++) {
          const short4v ra = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_short4*)(vb + rv[n] + 16 * D * u));
          const short4v rb = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_short4*)(vb + rv[n] + 16 * D * u + 8 * D));
          const half8 vt = __builtin_bit_cast(half8, __builtin_shufflevector(ra, rb, 0, 1, 2, 3, 4, 5, 6, 7));
          o[n] = __builtin_amdgcn_mfma_f32_32x32x16_f16(vt, pb[u], o[n], 0, 0, 0);
        }
    }
  };
  // A V row may hold infinities and NaN: in a product, 0 times one of those
  // would reach the rows that do not see the key.  Each wavefront looks
  // at what it loaded as it lands; where a stage holds any, they are added to the
  // rows that see them one by one, and cleared before the product.
  auto clear_non_finite = [&](T* vb) __attribute__((always_inline)) {
#pragma unroll 1
    for (int c = wave; c < TL::kElems / TL::kChunkElems / 64; c += W) {
      qfrag_t* at = reinterpret_cast<qfrag_t*>(vb + (c * 64 + l) * TL::kChunkElems);
      qfrag_t x = *at;
#pragma unroll
      for (int e = 0; e < TL::kChunkElems; e++) x[e] = finite_or_zero(x[e]);
      *at = x;
    }
  };
  auto add_non_finite = [&](const T* vb, int first) __attribute__((always_inline)) {
    for (int at = 0; at < kTileTokens; at++) {
      const bool seen = sees(row, first + at);
      const T* src = vb + gbase + at * D;
#pragma unroll
      for (int n = 0; n < D / 32; n++) {
        __builtin_amdgcn_sched_barrier(0); // (a block's reads at a time)
#pragma unroll
        for (int e = 0; e < 16; e++) {
          const int er = 8 * (e >> 2) + 4 * hh + (e & 3);
          const int d = kF32 ? (D / 32) * er + n : 32 * n + er; // O^T's dim in o[n][e]
          const float x = non_finite_part(kF32 ? src[d] : src[((d >> 4) ^ TL::vswz(at)) * 16 + (d & 15)]);
          o[n][e] += seen ? x : 0.f;
        }
      }
    }
  };

  // Every stage starts zeroed: a lane past its bound reads zeros, and should it
  // leave its bytes unwritten instead, they hold zeros or keys of this call.
#pragma unroll
  for (int a = 0; a < S; a++)
#pragma unroll
    for (int u = 0; u < TL::kLoads; u++) {
      const int e = ((wave * TL::kLoads + u) * 64 + l) * TL::kChunkElems;
      *reinterpret_cast<u32x4*>(k_st[a] + e) = u32x4{0u, 0u, 0u, 0u};
      *reinterpret_cast<u32x4*>(v_st[a] + e) = u32x4{0u, 0u, 0u, 0u};
    }
  __builtin_amdgcn_s_waitcnt(0xC07F); // lgkmcnt(0)
  // Steps [clear0, clear1), in whole rounds of S: every row of the block sees all of their
  // keys.  The others look at masks, wavefront by wavefront.
  const int all0 = (range.all_begin + kTileTokens - 1) / kTileTokens, all1 = min(range.all_end / kTileTokens, j1);
  const int clear0 = (max(all0 - j0, 0) + G * S - 1) / (G * S) * S;
  const int clear1 = clear0 + max(0, (all1 - j0) / G - clear0) / S * S;
  // Step si's stage lands: this wavefront's loads of it (the S - 2 steps after it
  // stay in flight; loads by page as many as there are pages, so there all), then
  // everybody's.
  auto land = [&](int si, auto stage) __attribute__((always_inline)) {
    constexpr int st = decltype(stage)::value;
    wait_loads<PAGES == kAnyPages ? 0 : (S - 2) * 2 * TL::kLoads>();
    if (si < clear0 || si >= clear1) {
      bool bad = false;
#pragma unroll
      for (int u = 0; u < TL::kLoads; u++)
        bad |= any_non_finite(
            *reinterpret_cast<const qfrag_t*>(v_st[st] + ((wave * TL::kLoads + u) * 64 + l) * TL::kChunkElems));
      non_finite[st][wave] = __any(bad);
    }
    stage_barrier();
  };
  Entries next_pages{};
  if (n_steps > 0) { // (no row of the tile may see a key: nothing is loaded then)
#pragma unroll
    for (int a = 0; a < S - 1; a++) issue_stage(min(a, last_step), fetch_pages(min(a, last_step)), k_st[a], v_st[a]);
    next_pages = fetch_pages(min(S - 1, last_step));
    land(0, std::integral_constant<int, 0>());
  }

  // Step si reads stage si % S; meanwhile step si + S - 1 lands in the stage that
  // step si - 1 read, whose readers met at the last barrier.  (Loads past the last
  // step repeat it, into stages that nobody reads again.)
  auto clear_step = [&](int si, auto stage) __attribute__((always_inline)) {
    constexpr int st = decltype(stage)::value, into = (st + S - 1) % S;
    issue_stage(min(si + S - 1, last_step), next_pages, k_st[into], v_st[into]);
    if (live) {
      float16v sc[kSub];
      qk(k_st[st], sc);
      softmax(sc, (j0 + G * si + grp) * kTileTokens, false);
      pv(v_st[st], sc);
    }
    next_pages = fetch_pages(min(si + S, last_step));
    land(si + 1, std::integral_constant<int, (st + 1) % S>());
  };
  auto masked_step = [&](int si, auto stage) __attribute__((always_inline)) {
    constexpr int st = decltype(stage)::value, into = (st + S - 1) % S;
    issue_stage(min(si + S - 1, last_step), next_pages, k_st[into], v_st[into]);
    const int j = j0 + G * si + grp, first = j * kTileTokens;
    const bool works = j < j1 && first < mine.end && first + kTileTokens > mine.begin;
    int4v flags = *reinterpret_cast<const int4v*>(non_finite[st]);
    if constexpr (W == 8) flags |= *reinterpret_cast<const int4v*>(non_finite[st] + 4);
    const bool bad = __builtin_amdgcn_readfirstlane(flags[0] | flags[1] | flags[2] | flags[3]);
    float16v sc[kSub];
    if (works) {
      qk(k_st[st], sc);
      softmax(sc, first, first < mine.all_begin || first + kTileTokens > mine.all_end);
    }
    if (bad) { // the whole block: every wavefront has read the stage before it is cleared, and meets it cleared
      if (works) add_non_finite(v_st[st], first);
      stage_barrier();
      clear_non_finite(v_st[st]);
      stage_barrier();
    }
    if (works) pv(v_st[st], sc);
    next_pages = fetch_pages(min(si + S, last_step));
    land(si + 1, std::integral_constant<int, (st + 1) % S>());
  };
#define MVR_STAGE(K) std::integral_constant<int, K>()
  // (Each stage is named statically.)
  for (int si = 0; si < n_steps;) {
    if (si == clear0) {
      for (; si < clear1; si += S) {
        clear_step(si, MVR_STAGE(0));
        clear_step(si + 1, MVR_STAGE(1));
        if constexpr (S >= 3) clear_step(si + 2, MVR_STAGE(2));
        if constexpr (S == 4) clear_step(si + 3, MVR_STAGE(3));
      }
      if (si >= n_steps) break;
    }
    masked_step(si, MVR_STAGE(0));
    if (si + 1 < n_steps) masked_step(si + 1, MVR_STAGE(1));
    if constexpr (S >= 3) {
      if (si + 2 < n_steps) masked_step(si + 2, MVR_STAGE(2));
    }
    if constexpr (S == 4) {
      if (si + 3 < n_steps) masked_step(si + 3, MVR_STAGE(3));
    }
    si += S;
  }
#undef MVR_STAGE
  // Every load has landed, everybody's, before the stages are used again.
  wait_loads<0>();
  __syncthreads();

  // Group 1 hands its state to group 0: part n of O of row wavefront rw as 4 x 64
  // float4, 1024 floats from float (n * RW + rw) * 1024 of the stages.
  if constexpr (G == 2) {
    constexpr int kStageFloats = TL::kElems * (int)sizeof(T) / 4;
    static_assert((D / 32) * RW * 1024 <= 4 * kStageFloats && kStageFloats % 1024 == 0, "O exceeds the stages");
    auto xfer = [&](int n) {
      const int f = (n * RW + rw) * 1024, obj = f / kStageFloats;
      T* base = obj == 0 ? k_lds0 : obj == 1 ? k_lds1 : obj == 2 ? v_lds0 : v_lds1;
      return reinterpret_cast<float4v*>(reinterpret_cast<float*>(base) + f % kStageFloats) + l;
    };
    if (grp == 1) {
#pragma unroll
      for (int n = 0; n < D / 32; n++)
#pragma unroll
        for (int a = 0; a < 4; a++)
          xfer(n)[64 * a] = float4v{o[n][4 * a], o[n][4 * a + 1], o[n][4 * a + 2], o[n][4 * a + 3]};
      ml_xfer[rw][0][l] = m;
      ml_xfer[rw][1][l] = lsum;
    }
    __syncthreads();
    if (grp == 0) {
      const float m1 = ml_xfer[rw][0][l], mm = fmaxf(m, m1);
      const float a0 = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m - mm);
      const float a1 = m1 == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m1 - mm);
#pragma unroll
      for (int n = 0; n < D / 32; n++)
#pragma unroll
        for (int a = 0; a < 4; a++) {
          const float4v x = xfer(n)[64 * a];
#pragma unroll
          for (int c = 0; c < 4; c++) o[n][4 * a + c] = a0 * o[n][4 * a + c] + a1 * x[c];
        }
      lsum = a0 * lsum + a1 * ml_xfer[rw][1][l];
      m = mm;
    }
    if (grp == 1) return;
  }
  const float ltot = lsum + __shfl_xor(lsum, 32);
  // (The lane's row is worked out anew: no register holds it over the key loop.)
  int le = l & 31;
  asm volatile("" : "+v"(le));
  int token, head;
  if (!row_at(rho0 + le, token, head)) return;
  // Lane holds dims 32 n + 8 (e / 4) + 4 hh + e % 4 of its row (F32: (D / 32) *
  // (8 (e / 4) + 4 hh + e % 4) + n).
  auto put = [&](auto* dst, float scale) __attribute__((always_inline)) {
#pragma unroll
    for (int n = 0; n < D / 32; n++)
#pragma unroll
      for (int a = 0; a < 4; a++) {
        if constexpr (kF32) {
#pragma unroll
          for (int c = 0; c < 4; c++) dst[(D / 32) * (8 * a + 4 * hh + c) + n] = o[n][4 * a + c] * scale;
        } else {
          typedef typename std::remove_reference<decltype(*dst)>::type out_t;
          typedef out_t out4 __attribute__((ext_vector_type(4)));
          const float4v v = float4v{o[n][4 * a], o[n][4 * a + 1], o[n][4 * a + 2], o[n][4 * a + 3]} * scale;
          *reinterpret_cast<out4*>(dst + 32 * n + 8 * a + 4 * hh) = __builtin_convertvector(v, out4);
        }
      }
  };
  if (parts > 1) {
    const int64_t prow = (tile.place * p.parts + it.part) * kTileRows + rw * 32 + le;
    put(p.partial_o + prow * D, 1.f);
    if (hh == 0) {
      p.partial_ml[prow * 2 + 0] = m;
      p.partial_ml[prow * 2 + 1] = ltot;
    }
  } else {
    put(static_cast<T*>(p.out) + (int64_t)head * p.out_stride_head + (int64_t)(s.q_start + token) * p.out_stride_token,
        inverse_sum(ltot));
    if (hh == 0) store_lse(p.r, head, s.q_start + token, m, ltot);
  }
}

template <int D, typename T, int RW, int W>
constexpr int stage_bytes() { // of K and V
  return 2 * Tile<D, T, RW, W>::kElems * (int)sizeof(T);
}

template <int D, typename T, int RW, int W, int S>
hipError_t launch_stages(const ScoreAttentionPlan& plan, const ScoreAttentionParams& p, hipStream_t stream) {
  typedef Tile<D, T, RW, W> TL;
  const dim3 grid(score_blocks(p)), block(kWaveSize * W);
  if (p.t.page_size % kChunkTokens == 0) { // a wavefront's 8 or 16 tokens lie in one page
    hipLaunchKernelGGL((score_tile_kernel<D, T, RW, W, kRuns, S>), grid, block, 0, stream, p);
    return hipGetLastError();
  }
  if constexpr (D == 64 || D == 128) {
    if (p.t.page_size % (64 / TL::kChunksPerRow) == 0) {
      hipLaunchKernelGGL((score_tile_kernel<D, T, RW, W, kWholeLoads, S>), grid, block, 0, stream, p);
      return hipGetLastError();
    }
  }
  // (Its loads are waited for as a whole: two stages.)
  hipLaunchKernelGGL((score_tile_kernel<D, T, RW, W, kAnyPages, 2>), grid, block, 0, stream, p);
  return hipGetLastError();
}

// Stages: as many as two blocks per CU leave room for, 4 at most (2 at head_dim 128).
template <int D, typename T, int RW, int W>
hipError_t launch_rows(const ScoreAttentionPlan& plan, const ScoreAttentionParams& p, hipStream_t stream) {
  constexpr int kBytes = stage_bytes<D, T, RW, W>() * kTileWaves / W;
  constexpr int kStages = 78 * 1024 / kBytes >= 4 ? 4 : 78 * 1024 / kBytes >= 3 ? 3 : 2;
  return launch_stages<D, T, RW, W, kStages>(plan, p, stream);
}

template <int D, typename T>
hipError_t launch_type(const ScoreAttentionPlan& plan, const ScoreAttentionParams& p, hipStream_t stream) {
  if constexpr (D <= 128) {
    if (plan.tile_rows == 64) return launch_rows<D, T, 2, 4>(plan, p, stream);
    if (plan.waves == 8) return launch_rows<D, T, 4, 8>(plan, p, stream);
  }
  return launch_rows<D, T, 4, 4>(plan, p, stream);
}

template <int D>
hipError_t launch_dim(const ScoreAttentionPlan& plan, const ScoreAttentionParams& p, int dtype, hipStream_t stream) {
  return dtype == 1 ? launch_type<D, half_t>(plan, p, stream) : launch_type<D, float>(plan, p, stream);
}

} // namespace

hipError_t launch_score_tiles(const ScoreAttentionPlan& plan, const ScoreAttentionParams& params, int dtype,
                              int head_dim, hipStream_t stream) {
  switch (head_dim) {
  case 32: return launch_dim<32>(plan, params, dtype, stream);
  case 64: return launch_dim<64>(plan, params, dtype, stream);
  case 96: return launch_dim<96>(plan, params, dtype, stream);
  case 128: return launch_dim<128>(plan, params, dtype, stream);
  case 160: return launch_dim<160>(plan, params, dtype, stream);
  case 192: return launch_dim<192>(plan, params, dtype, stream);
  case 224: return launch_dim<224>(plan, params, dtype, stream);
  case 256: return launch_dim<256>(plan, params, dtype, stream);
  default: return hipErrorInvalidValue;
  }
}

} // namespace mvr
