// Attention of drafted trees with many rows per KV head, for gfx950: key tiles
// in LDS, 32x32 MFMAs.  The mathematics is draft_attention.hip's.
//
// A block of 4 wavefronts holds a row tile of 32 * RW grouped rows of one
// (request, KV head), 32 rows per wavefront, in G = 4 / RW groups of RW
// wavefronts that hold the same rows and take alternating key tiles of TT
// tokens.  Each step stages G key tiles of K and V in LDS, loaded straight from
// the pages (buffer_load ... lds) one step ahead; every wavefront of a group
// reads them from there, so a key's bytes leave the cache once per row tile.
//   S^T = K Q^T   v_mfma_f32_32x32x16_f16 (F32: 32x32x2): K from LDS as the A
//                 operand, Q^T in registers; a lane holds row l % 32, so the
//                 softmax needs one cross-lane step;
//   O^T += V^T P^T  V through transposing LDS reads (F16), P^T from the S^T
//                 registers as it is.
// The running maximum moves, and O is rescaled, only where a score exceeds it by
// more than 2^8: P stays below 2^8 in F16, and sums are 32 bits.
//
// Bound by HBM on long contexts (64 requests of 32 drafts on 8,192 keys, 32 / 8
// heads of 128, F16: 398 us in a loop of calls, 5.5 TB/s, 380 to 450 with the card's
// state; the matrix pipe is 38% busy), else by a step's chain of product, softmax,
// product: a block of 128 rows takes 1.38 us per 64 keys alone on its CU, 448 blocks
// on 256 CUs take 2.02 (0.93 PFLOP/s), which is why two blocks share a CU rather
// than one with deeper stages.  Beside its steps a block
// takes some 5 us more than a launch: scan, Q and masks, first loads, draft steps,
// stores.
#include "draft_common.hpp"
#include "key_tiles.hpp"

#include <type_traits>

namespace mvr {
namespace {

// S: LDS stages; S - 1 steps' loads are in flight while a step is computed.
template <int D, typename T, int RW, int PAGES, int S>
__device__ __forceinline__ void tile_item(const DraftAttentionParams& p, const DraftItem& it, int64_t slot) {
  typedef Tile<D, T, RW> TL;
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
  __shared__ __attribute__((aligned(16))) int non_finite[S][kDraftWaves]; // by stage: what each wavefront loaded holds any
  static_assert(S >= 2 && S <= 4, "2, 3 or 4 stages");
  T* const k_st[4] = {k_lds0, k_lds1, k_lds2, k_lds3};
  T* const v_st[4] = {v_lds0, v_lds1, v_lds2, v_lds3};

  const int l = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int rw = wave % RW, grp = wave / RW, hh = l >> 5;
  const DraftSeq& s = it.s;
  const int rows = p.group_size * s.q_len, prefix = s.seq_len - s.q_len;

  // The part's key tiles [j0, j1).
  constexpr int kUnitTiles = kDraftUnitTokens / kTileTokens;
  const int units = key_units_of(s), n_tiles = (s.seq_len + kTileTokens - 1) / kTileTokens;
  const int j0 = kUnitTiles * (int)((int64_t)it.part * units / it.parts);
  const int j1 = min(kUnitTiles * (int)((int64_t)(it.part + 1) * units / it.parts), n_tiles);
  if (j0 >= j1) return; // (never: parts are of a unit at least; the whole block)

  // The lane's row: query head r of the group, draft i.
  auto row_of = [&](bool& valid, int& r, int& i) {
    const int rho = it.rt * kTileRows + rw * 32 + (l & 31);
    valid = rho < rows;
    r = valid ? rho / s.q_len : 0;
    i = valid ? rho - r * s.q_len : 0;
  };
  const bool live = it.rt * kTileRows + rw * 32 < rows; // the wavefront has rows

  // Q^T as the B operand: lane l holds row l % 32, dims 16 st + 8 hh .. + 8 (F32: 8 st + 4 hh .. + 4).
  qfrag_t q[kQFrags];
  {
    bool valid;
    int r, i;
    row_of(valid, r, i);
    const T* qrow = static_cast<const T*>(p.q) + (int64_t)(it.h * p.group_size + r) * p.q_stride_head +
                    (int64_t)(s.q_start + i) * p.q_stride_token;
    constexpr int kFragDims = kF32 ? 8 : 16;
#pragma unroll
    for (int st = 0; st < kQFrags; st++)
      q[st] = valid ? *reinterpret_cast<const qfrag_t*>(qrow + kFragDims * st + (kFragDims / 2) * hh) : qfrag_t{};
  }
  RowMask row_mask; // (its first words now: they are there when the drafts are)
  {
    bool valid;
    int r, i;
    row_of(valid, r, i);
    row_mask = load_row_mask(p, s, i);
  }

  float16v o[D / 32];
#pragma unroll
  for (int n = 0; n < D / 32; n++)
#pragma unroll
    for (int e = 0; e < 16; e++) o[n][e] = 0.f;
  float m = -INFINITY, lsum = 0.f;

  // Staging.  Wavefront w fills the stage's token rows from w * kWaveTokens on;
  // its load u writes LDS chunks (w * kLoads + u) * 64 + lane, and each lane reads
  // the chunk of the row that the swizzle puts there.
  const const_i32* bt = (const const_i32*)(p.block_tables) + (int64_t)it.b * p.block_table_stride;
  auto page_div = [&](int t) { return (int)(((uint64_t)(uint32_t)t * p.page_magic) >> p.page_magic_shift); };
  constexpr uint32_t kRowBytes = D * (uint32_t)sizeof(T);
  const uint32_t page_rows = (uint32_t)(p.num_kv_heads * p.page_size), head_rows = (uint32_t)(it.h * p.page_size);
  auto rows_at = [&](uint32_t page, uint32_t row) {
    return ((uint64_t)min(page, p.last_page) * page_rows + (head_rows + row)) * kRowBytes;
  };
  // Bytes from the wavefront's first token row (kWholeLoads: the load's; kAnyPages: within the row).
  constexpr int kLoadTokens = PAGES == kWholeLoads ? 64 / TL::kChunksPerRow : 1;
  static_assert(PAGES != kWholeLoads || 64 % TL::kChunksPerRow == 0, "loads of whole token rows");
  uint32_t off_k[TL::kLoads], off_v[TL::kLoads];
#pragma unroll
  for (int u = 0; u < TL::kLoads; u++) {
    const int P = (wave * TL::kLoads + u) * 64 + l;
    const int t = P / TL::kChunksPerRow, cs = P % TL::kChunksPerRow;
    const int dt = PAGES == kRuns ? t - wave * TL::kWaveTokens : PAGES == kWholeLoads ? l / TL::kChunksPerRow : 0;
    off_k[u] = (uint32_t)(dt * D + TL::kChunkElems * (cs ^ TL::kswz(t))) * sizeof(T);
    off_v[u] = (uint32_t)(dt * D + TL::kChunkElems * (2 * ((cs >> 1) ^ TL::vswz(t)) + (cs & 1))) * sizeof(T);
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
  auto issue_stage = [&](int si, const Entries& entries, T* kb, T* vb) {
    const char* kpool = static_cast<const char*>(p.key_pool);
    const char* vpool = static_cast<const char*>(p.value_pool);
    if constexpr (PAGES == kAnyPages) {
      // A load's tokens may lie in several pages, which take their lanes in turn.
      // Lanes of tokens past
      // the last key go with the last page, whose bound reads them as zeros.
      const int last_page_index = page_div(last_key);
#pragma unroll
      for (int u = 0; u < TL::kLoads; u++) {
        const int P = (wave * TL::kLoads + u) * 64;
        const int t0 = (j0 + G * si) * kTileTokens;
        const int t = t0 + (P + l) / TL::kChunksPerRow;
        const int page_index = min(page_div(t), last_page_index);
        const uint32_t row_off = (uint32_t)(t - page_index * p.page_size) * kRowBytes;
        const int first = min(page_div(t0 + P / TL::kChunksPerRow), last_page_index);
        const int last = min(page_div(t0 + (P + 63) / TL::kChunksPerRow), last_page_index);
        for (int pi = first; pi <= last; pi++) { // wave-uniform
          const uint64_t at = rows_at((uint32_t)bt[pi], 0);
          const uint32_t bytes = (uint32_t)min(p.page_size, s.seq_len - pi * p.page_size) * kRowBytes;
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
          const int t = first_token(si, u);
          at = rows_at(entries.page[PAGES == kWholeLoads ? u : 0], (uint32_t)(t - page_div(t) * p.page_size));
          bytes = (uint32_t)min(s.seq_len - t, kRunTokens) * kRowBytes;
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
      const int row = 4 * hh + ((l & 15) >> 2), col = 32 * n + 16 * ((l >> 4) & 1) + 4 * (l & 3);
      rv[n] = gbase + row * D + ((col >> 4) ^ TL::vswz(row)) * 16 + (col & 15);
    }
  }
  const float sl2 = p.scale_log2;

  auto qk = [&](const T* kb, float16v (&acc)[kSub]) {
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
  auto softmax_max = [&](const float16v (&sc)[kSub]) {
    float mx = -INFINITY;
#pragma unroll
    for (int c = 0; c < kSub; c++)
#pragma unroll
      for (int e = 0; e < 16; e += 4)
        mx = fmaxf(mx, fmaxf(fmaxf(sc[c][e], sc[c][e + 1]), fmaxf(sc[c][e + 2], sc[c][e + 3])));
    mx *= sl2; // (scale > 0 keeps the order)
    const auto sw = __builtin_amdgcn_permlane32_swap(__float_as_uint(mx), __float_as_uint(mx), false, false);
    mx = fmaxf(__uint_as_float(sw[0]), __uint_as_float(sw[1]));
    const bool grow = mx > m + kRescaleThreshold || (m == -INFINITY && mx != -INFINITY);
    if (__any(grow)) {
      const float m_new = grow ? mx : m;
      const float alpha = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m - m_new);
#pragma unroll
      for (int n = 0; n < D / 32; n++) o[n] *= alpha;
      lsum *= alpha;
      m = m_new;
    }
  };
  // Probabilities e and e + 1 of block c as the product with V takes them.
  auto halves = [&](const float16v (&sc)[kSub], int c, int e) {
    return __builtin_convertvector((float2v{sc[c][e], sc[c][e + 1]}), half2v);
  };
  // P = 2^(s * scale - m) in place, and its sum.  F16: the product with V takes P
  // rounded to F16 (half a step, 2^-11 of p, so outputs are 1.1 to 1.4 times as far
  // from the formula as those of a form that holds 32 bits), and the sum is of the
  // rounded P: the weights of the keys add up to 1, and values that are all equal come
  // back as they are.  A second product for what the rounding leaves, as the streaming
  // kernel has, costs a quarter here (64 requests of 32 drafts on 8,192 keys 394 -> 493
  // us, 16 of 128 on 1,024 48 -> 62), v_dot2 for the sum 0 to 3%.
  auto exps = [&](float16v (&sc)[kSub]) {
    const float neg_m = m == -INFINITY ? 0.f : -m;
    float psum = 0.f;
#pragma unroll
    for (int c = 0; c < kSub; c++)
#pragma unroll
      for (int e = 0; e < 16; e += 2) {
        sc[c][e] = __builtin_amdgcn_exp2f(fmaf(sc[c][e], sl2, neg_m));
        sc[c][e + 1] = __builtin_amdgcn_exp2f(fmaf(sc[c][e + 1], sl2, neg_m));
        if constexpr (kF32) {
          psum += sc[c][e];
          psum += sc[c][e + 1];
        } else {
          psum = __builtin_amdgcn_fdot2(halves(sc, c, e), half2v{1, 1}, psum, false);
        }
      }
    lsum += psum;
  };
  auto pv = [&](const T* vb, const float16v (&sc)[kSub]) {
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
  // A draft's V may hold infinities and NaN: in a product, 0 times one of those
  // would reach the rows that do not see the draft.  Each wavefront looks
  // at what it loaded as it lands; where a stage holds any, they are added to the
  // rows that see them one by one, and cleared before the product.
  auto clear_non_finite = [&](T* vb) {
#pragma unroll 1
    for (int c = wave; c < TL::kElems / TL::kChunkElems / 64; c += kDraftWaves) {
      qfrag_t* at = reinterpret_cast<qfrag_t*>(vb + (c * 64 + l) * TL::kChunkElems);
      qfrag_t x = *at;
#pragma unroll
      for (int e = 0; e < TL::kChunkElems; e++) x[e] = finite_or_zero(x[e]);
      *at = x;
    }
  };
  auto add_non_finite = [&](const T* vb, const uint32_t (&bits)[kSub]) {
    for (int t = 0; t < kTileTokens; t++) {
      const bool sees = (bits[kSub == 1 ? 0 : t >> 5] >> (t & 31)) & 1;
      const T* row = vb + gbase + t * D;
#pragma unroll
      for (int n = 0; n < D / 32; n++) {
        __builtin_amdgcn_sched_barrier(0); // (a block's reads at a time)
#pragma unroll
        for (int e = 0; e < 16; e++) {
          const int at = 8 * (e >> 2) + 4 * hh + (e & 3);
          const int d = kF32 ? (D / 32) * at + n : 32 * n + at; // O^T's dim in o[n][e]
          const float x = non_finite_part(kF32 ? row[d] : row[((d >> 4) ^ TL::vswz(t)) * 16 + (d & 15)]);
          o[n][e] += sees ? x : 0.f;
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
  // Tiles j < clear_tiles end before the drafts and need no masks: whole rounds of
  // S steps of them come first.
  const int clear_tiles = min(j1, max(prefix, 0) / kTileTokens);
  const int clear_steps = max(0, (clear_tiles - j0) / G) / S * S;
  // Step si's stage lands: this wavefront's loads of it (the S - 2 steps after it
  // stay in flight; loads by page as many as there are pages, so there all), then
  // everybody's.
  auto land = [&](int si, auto stage) {
    constexpr int st = decltype(stage)::value;
    wait_loads<PAGES == kAnyPages ? 0 : (S - 2) * 2 * TL::kLoads>();
    if (si >= clear_steps) {
      bool bad = false;
#pragma unroll
      for (int u = 0; u < TL::kLoads; u++)
        bad |= any_non_finite(
            *reinterpret_cast<const qfrag_t*>(v_st[st] + ((wave * TL::kLoads + u) * 64 + l) * TL::kChunkElems));
      non_finite[st][wave] = __any(bad);
    }
    stage_barrier();
  };
#pragma unroll
  for (int a = 0; a < S - 1; a++) issue_stage(min(a, last_step), fetch_pages(min(a, last_step)), k_st[a], v_st[a]);
  Entries next_pages = fetch_pages(min(S - 1, last_step));
  land(0, std::integral_constant<int, 0>());

  // Step si reads stage si % S; meanwhile step si + S - 1 lands in the stage that
  // step si - 1 read, whose readers met at the last barrier.  (Loads past the last
  // step repeat it, into stages that nobody reads again.)
  auto clear_step = [&](int si, auto stage) {
    constexpr int st = decltype(stage)::value, into = (st + S - 1) % S;
    issue_stage(min(si + S - 1, last_step), next_pages, k_st[into], v_st[into]);
    if (live) {
      float16v sc[kSub];
      qk(k_st[st], sc);
      softmax_max(sc);
      exps(sc);
      pv(v_st[st], sc);
    }
    next_pages = fetch_pages(min(si + S, last_step));
    land(si + 1, std::integral_constant<int, (st + 1) % S>());
  };
  auto draft_step = [&](int si, auto stage) {
    constexpr int st = decltype(stage)::value, into = (st + S - 1) % S;
    issue_stage(min(si + S - 1, last_step), next_pages, k_st[into], v_st[into]);
    const int j = j0 + G * si + grp;
    const bool works = live && j < j1;
    const int4v flags = *reinterpret_cast<const int4v*>(non_finite[st]);
    const bool bad = __builtin_amdgcn_readfirstlane(flags[0] | flags[1] | flags[2] | flags[3]);
    float16v sc[kSub];
    uint32_t bits[kSub];
    if (works) {
      qk(k_st[st], sc);
#pragma unroll
      for (int c = 0; c < kSub; c++) {
        bits[c] = visible_bits(row_mask, j * kTileTokens + 32 * c - prefix);
        const uint32_t mine = bits[c] >> (4 * hh);
#pragma unroll
        for (int e = 0; e < 16; e++) sc[c][e] = (mine >> (8 * (e >> 2) + (e & 3))) & 1 ? sc[c][e] : -INFINITY;
      }
      softmax_max(sc);
      exps(sc);
    }
    if (bad) { // the whole block: every wavefront has read the stage before it is cleared, and meets it cleared
      if (works) add_non_finite(v_st[st], bits);
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
  for (int si = 0; si < clear_steps; si += S) {
    clear_step(si, MVR_STAGE(0));
    clear_step(si + 1, MVR_STAGE(1));
    if constexpr (S >= 3) clear_step(si + 2, MVR_STAGE(2));
    if constexpr (S == 4) clear_step(si + 3, MVR_STAGE(3));
  }
  for (int si = clear_steps; si < n_steps; si += S) {
    draft_step(si, MVR_STAGE(0));
    if (si + 1 >= n_steps) break;
    draft_step(si + 1, MVR_STAGE(1));
    if constexpr (S >= 3) {
      if (si + 2 >= n_steps) break;
      draft_step(si + 2, MVR_STAGE(2));
    }
    if constexpr (S == 4) {
      if (si + 3 >= n_steps) break;
      draft_step(si + 3, MVR_STAGE(3));
    }
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
  bool valid;
  int r, i;
  row_of(valid, r, i);
  if (!valid) return;
  // Lane holds dims 32 n + 8 (e / 4) + 4 hh + e % 4 of its row (F32: (D / 32) *
  // (8 (e / 4) + 4 hh + e % 4) + n).
  auto put = [&](auto* dst, float scale) {
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
  if (it.parts > 1) {
    const int64_t prow = slot * kTileRows + rw * 32 + (l & 31);
    put(p.partial_o + prow * D, 1.f);
    if (hh == 0) {
      p.partial_ml[prow * 2 + 0] = m;
      p.partial_ml[prow * 2 + 1] = ltot;
    }
  } else {
    put(static_cast<T*>(p.out) + (int64_t)(it.h * p.group_size + r) * p.out_stride_head +
            (int64_t)(s.q_start + i) * p.out_stride_token,
        inverse_sum(ltot));
  }
}

template <int D, typename T, int RW>
constexpr int stage_bytes() { // of K and V
  return 2 * Tile<D, T, RW>::kElems * (int)sizeof(T);
}

template <int D, typename T, int RW, int PAGES, int S>
__global__ __launch_bounds__(kWaveSize* kDraftWaves, (draft_blocks_per_cu(32 * RW, sizeof(T) == 2, D))) void draft_tile_kernel(
    DraftAttentionParams p) {
  constexpr int kTileRows = 32 * RW;
  // (One call of tile_item: its code, twice, would crowd the instruction cache.)
  for (int w = first_item(p);; w += gridDim.x) {
    const DraftItem it = find_item<kTileRows>(p, w);
    if (it.b >= p.num_seqs) break;
    if (it.rt < row_tiles_of<kTileRows>(p, it.s)) tile_item<D, T, RW, PAGES, S>(p, it, w);
    __syncthreads(); // the LDS is used again
  }
}

template <int D, typename T, int RW, int S>
hipError_t launch_stages(const DraftAttentionPlan& plan, const DraftAttentionParams& p, hipStream_t stream) {
  typedef Tile<D, T, RW> TL;
  const dim3 grid((unsigned)plan.blocks), block(kWaveSize * kDraftWaves);
  if (p.page_size % kChunkTokens == 0) { // a wavefront's 8 or 16 tokens lie in one page
    hipLaunchKernelGGL((draft_tile_kernel<D, T, RW, kRuns, S>), grid, block, 0, stream, p);
    return hipGetLastError();
  }
  if constexpr (D == 64 || D == 128) {
    if (p.page_size % (64 / TL::kChunksPerRow) == 0) {
      hipLaunchKernelGGL((draft_tile_kernel<D, T, RW, kWholeLoads, S>), grid, block, 0, stream, p);
      return hipGetLastError();
    }
  }
  // (Its loads are waited for as a whole: two stages.)
  hipLaunchKernelGGL((draft_tile_kernel<D, T, RW, kAnyPages, 2>), grid, block, 0, stream, p);
  return hipGetLastError();
}

// Stages: as many as two blocks per CU leave room for, 4 at most (2 at head_dim
// 128).  4 stages and one block per CU there made no difference, 112 blocks of 33
// steps included (39.5 us): a lone block's step waits for its own chain of product,
// softmax and product, not for its loads.
template <int D, typename T, int RW>
hipError_t launch_rows(const DraftAttentionPlan& plan, const DraftAttentionParams& p, hipStream_t stream) {
  constexpr int kBytes = stage_bytes<D, T, RW>();
  constexpr int kStages = 78 * 1024 / kBytes >= 4 ? 4 : 78 * 1024 / kBytes >= 3 ? 3 : 2;
  return launch_stages<D, T, RW, kStages>(plan, p, stream);
}

template <int D>
hipError_t launch_dim(const DraftAttentionPlan& plan, const DraftAttentionParams& p, int dtype, hipStream_t stream) {
  if (plan.tile_rows == 128)
    return dtype == 1 ? launch_rows<D, half_t, 4>(plan, p, stream) : launch_rows<D, float, 4>(plan, p, stream);
  if constexpr (D <= 128) {
    if (plan.tile_rows == 64)
      return dtype == 1 ? launch_rows<D, half_t, 2>(plan, p, stream) : launch_rows<D, float, 2>(plan, p, stream);
  }
  return hipErrorInvalidValue;
}

} // namespace

hipError_t launch_draft_tiles(const DraftAttentionPlan& plan, const DraftAttentionParams& params, int dtype,
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
