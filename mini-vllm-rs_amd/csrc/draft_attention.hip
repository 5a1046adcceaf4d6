// Attention of drafted trees over a paged cache, for gfx950 (MI355X, CDNA4).
//
// Request b has n = seq_len keys, its q_len drafts in the last slots; c = n -
// q_len.  With s_j = scale * q . k_j, query i's output is
//   sum_j e^(s_j - m) v_j / sum_j e^(s_j - m),   m = max_j s_j,
// over the keys j < c and the draft slots j - c whose bit is set in the query's
// mask row; 0 where there are none.  One pass over the keys keeps the running
// maximum and sum of each row in 32 bits (exp2 domain), and the results of
// disjoint key ranges merge exactly:  o = sum_p 2^(m_p - m) o_p,  l likewise.
//
// The masks matter to the key chunks that hold drafts only: all the others are
// seen by every row, and take no mask, no test and no table read.
#include "draft_common.hpp"

#include <type_traits>

namespace mvr {
namespace {

// ---------------------------------------------------------------------------
// Key streaming: a block of 4 wavefronts per item, 16 * NB rows, each wavefront
// its share of the part's 16-token chunks straight from the cache; their
// results merge in LDS.
//
// Bound by HBM where blocks are many (64 requests of 1 token on 500..3,500 keys,
// 32 / 8 heads of 128, F16: 110 us, 5.1 TB/s), by a block's own steps where they
// are few: keys go to registers, not through LDS, so that no wavefront waits for
// another until the end, and up to four blocks of different items share a CU.  16
// rows are what one 16x16 product takes; 8-wavefront blocks were no faster, and
// from some 32 rows on the products of 16 cost more than key tiles in LDS do.
// ---------------------------------------------------------------------------
// Chunks of one step: two of F16, whose softmax and products are then one of 32
// keys (2 x 100 rows on 100 keys 14.8 -> 12.5 us; long contexts as before); F32
// rows hold twice the registers (with two chunks 8 x 8 on 2,000 keys 40.5 -> 45.9).
template <typename Tr>
constexpr int step_chunks() {
  return sizeof(typename Tr::elem) == 4 ? 1 : 2;
}

// TP: page sizes that are not a multiple of 16, where every token row has a page
// of its own to look up.
template <typename Tr, int D, int NB, bool TP>
__device__ __forceinline__ void stream_item(const DraftAttentionParams& p, const DraftItem& it, int64_t slot,
                                            int wave, char* lds_raw) {
  typedef typename Tr::elem T;
  constexpr int kTileRows = 16 * NB;
  constexpr int kMergeStride = D + 4;
  constexpr int kUnitChunks = kDraftUnitTokens / kChunkTokens;
  constexpr int C = step_chunks<Tr>();
  float* const merge_o = reinterpret_cast<float*>(lds_raw);
  float* const merge_ml = merge_o + kDraftWaves * kTileRows * kMergeStride;

  int l = lane_id();
  asm volatile("" : "+v"(l)); // (an item's own: what is worked out from it is not held over the item loop)
  const int g = l >> 4;
  T* lds = reinterpret_cast<T*>(lds_raw) + (size_t)wave * C * kChunkTokens * D;
  const DraftSeq& s = it.s;
  const int rows = p.group_size * s.q_len;
  const int prefix = s.seq_len - s.q_len;

  // The wavefront's chunks.
  const int units = key_units_of(s), n_chunks = (s.seq_len + kChunkTokens - 1) / kChunkTokens;
  const int part0 = kUnitChunks * (int)((int64_t)it.part * units / it.parts);
  const int part1 = min(kUnitChunks * (int)((int64_t)(it.part + 1) * units / it.parts), n_chunks);
  const int k0 = part0 + (int)((int64_t)(part1 - part0) * wave / kDraftWaves);
  const int k1 = part0 + (int)((int64_t)(part1 - part0) * (wave + 1) / kDraftWaves);

  // The lane's row in row block nb.
  auto row_of = [&](int nb, bool& valid, int& r, int& i) {
    const int rho = it.rt * kTileRows + nb * 16 + (l & 15);
    valid = rho < rows;
    r = valid ? rho / s.q_len : 0;
    i = valid ? rho - r * s.q_len : 0;
  };
  typename Tr::qreg_t q[NB][Tr::kQRegs];
#pragma unroll
  for (int nb = 0; nb < NB; nb++) {
    bool valid;
    int r, i;
    row_of(nb, valid, r, i);
    const T* qrow = static_cast<const T*>(p.q) + (int64_t)(it.h * p.group_size + r) * p.q_stride_head +
                    (int64_t)(s.q_start + i) * p.q_stride_token;
    Tr::load_q(qrow, valid, g, q[nb]);
  }

  float m[NB], lsum[NB];
  float4v o[NB][D / 16];
#pragma unroll
  for (int nb = 0; nb < NB; nb++) {
    m[nb] = -INFINITY;
    lsum[nb] = 0.f;
#pragma unroll
    for (int n = 0; n < D / 16; n++) o[nb][n] = float4v{0.f, 0.f, 0.f, 0.f};
  }

  const T* kpool = static_cast<const T*>(p.key_pool);
  const T* vpool = static_cast<const T*>(p.value_pool);
  const int32_t* bt = p.block_tables + (int64_t)it.b * p.block_table_stride;
  auto page_div = [&](int t) { return (int)(((uint64_t)(uint32_t)t * p.page_magic) >> p.page_magic_shift); };
  const uint32_t page_rows = (uint32_t)(p.num_kv_heads * p.page_size), head_rows = (uint32_t)(it.h * p.page_size);

  // Loads of the C chunks from k on (past k1 the last one again, an L2 hit, rather
  // than a branch).  TP: lane l % 32 holds the page entry of token l % 32, read a
  // step ahead; the lanes get their rows' pages from it.  Rows past the last key
  // read the last key's row (masked, and zeroed in LDS).
  auto token_of = [&](int k, int c, int row) { return min(min(k + c, k1 - 1) * kChunkTokens + row, s.seq_len - 1); };
  auto load_entry = [&](int k) { return (uint32_t)bt[page_div(token_of(k, (l >> 4) % C, l & 15))]; };
  uint32_t entry = 0, next_entry = 0; // TP
  uint64_t chunk_off[C];              // otherwise: element offsets of the chunks
  auto look_up = [&](int k) {
    if constexpr (TP) {
      entry = min(next_entry, p.last_page);
      next_entry = load_entry(k + C);
    } else {
#pragma unroll
      for (int c = 0; c < C; c++) {
        const int t = min(k + c, k1 - 1) * kChunkTokens, pi = page_div(t);
        const uint32_t page = min((uint32_t)((const const_i32*)bt)[__builtin_amdgcn_readfirstlane(pi)], p.last_page);
        chunk_off[c] = ((uint64_t)page * page_rows + head_rows + (uint32_t)(t - pi * p.page_size)) * D;
      }
    }
  };
  auto row_off = [&](int k, int c, int row) { // TP: element offset of a token row of chunk c
    const int t = token_of(k, c, row);
    const uint32_t page = (uint32_t)__builtin_amdgcn_ds_bpermute(4 * (16 * c + row), (int)entry);
    return ((uint64_t)page * page_rows + head_rows + (uint32_t)(t - page_div(t) * p.page_size)) * D;
  };
  // (The lane index is opaque in these, so that the rows' offsets are worked out
  // where they are used and not held, and spilled, over the key loop.)
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

  // Scores of one row block to probabilities.  The running maximum moves, and what
  // the row holds is rescaled, only where a score exceeds it by more than 2^8.
  auto softmax = [&](int nb, float4v (&sc)[C]) {
    float mx = -INFINITY;
#pragma unroll
    for (int c = 0; c < C; c++) mx = fmaxf(mx, fmaxf(fmaxf(sc[c][0], sc[c][1]), fmaxf(sc[c][2], sc[c][3])));
    mx = row_max(mx * p.scale_log2); // (scale > 0 keeps the order)
    const bool grow = mx > m[nb] + kRescaleThreshold || (m[nb] == -INFINITY && mx != -INFINITY);
    if (__any(grow)) {
      const float m_new = grow ? mx : m[nb];
      const float alpha = m[nb] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m[nb] - m_new);
#pragma unroll
      for (int n = 0; n < D / 16; n++) o[nb][n] *= alpha;
      lsum[nb] *= alpha;
      m[nb] = m_new;
    }
    const float neg_m = m[nb] == -INFINITY ? 0.f : -m[nb];
#pragma unroll
    for (int c = 0; c < C; c++)
#pragma unroll
      for (int i = 0; i < 4; i++) {
        sc[c][i] = __builtin_amdgcn_exp2f(fmaf(sc[c][i], p.scale_log2, neg_m));
        lsum[nb] += sc[c][i];
      }
  };
  // O^T += V^T P^T of the chunks.  F16: two chunks in one product of 32 keys, lane
  // group g with tokens 4 g .. + 4 of each.  P enters as hi + lo, two F16 numbers
  // whose sum is p but for 2^-20 of it (2^-24 where that is more): both are cut
  // towards 0, p - hi is exact in 32 bits.  With hi alone, off by up to 2^-11 p, calls
  // of few rows came out 1.4 times as far from the formula as a form that holds 32
  // bits, and up to 1.8 times.  The second product is free where HBM is the bound (64
  // requests of 1 token on 500..3,500 keys 110.6 -> 110.5 us), and costs 0 to 5% where
  // a block's steps are (1 x 16 on 1,000 9.2 -> 9.7).
  auto pv = [&](int le, const float4v (&pr)[NB][C]) {
    if constexpr (sizeof(T) == 2) {
      half8 hi[NB], lo[NB];
      float minus = -1.f;
      asm("" : "+s"(minus)); // (opaque: conversion and difference are one v_fma_mix)
#pragma unroll
      for (int nb = 0; nb < NB; nb++)
#pragma unroll
        for (int e = 0; e < 8; e += 2) {
          const float a = pr[nb][e >> 2][e & 3], b = pr[nb][e >> 2][(e & 3) + 1];
          const half2v h = __builtin_bit_cast(half2v, __builtin_amdgcn_cvt_pkrtz(a, b));
          const half2v rest = __builtin_bit_cast(
              half2v, __builtin_amdgcn_cvt_pkrtz(fmaf((float)h[0], minus, a), fmaf((float)h[1], minus, b)));
          hi[nb][e] = h[0];
          hi[nb][e + 1] = h[1];
          lo[nb][e] = rest[0];
          lo[nb][e + 1] = rest[1];
        }
      const int row = 4 * (le >> 4) + ((le & 15) >> 2), sw = Tr::swz(row);
#pragma unroll
      for (int n = 0; n < D / 16; n++) {
        T* at = lds + row * D + ((n ^ sw) * 16) + 4 * (le & 3);
        const short4v ra = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_short4*)at);
        const short4v rb = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_short4*)(at + kChunkTokens * D));
        const half8 vt = __builtin_bit_cast(half8, __builtin_shufflevector(ra, rb, 0, 1, 2, 3, 4, 5, 6, 7));
#pragma unroll
        for (int nb = 0; nb < NB; nb++) {
          o[nb][n] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vt, lo[nb], o[nb][n], 0, 0, 0);
          o[nb][n] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vt, hi[nb], o[nb][n], 0, 0, 0);
        }
      }
    } else {
#pragma unroll
      for (int c = 0; c < C; c++) {
        float p4[NB][4];
#pragma unroll
        for (int nb = 0; nb < NB; nb++)
#pragma unroll
          for (int i = 0; i < 4; i++) p4[nb][i] = pr[nb][c][i];
        Tr::template pv<NB>(lds + c * kChunkTokens * D, le, p4, o);
      }
    }
  };

  typename Tr::kreg_t kbuf[C][Tr::kLoads];
  typename Tr::vreg_t vbuf[C][Tr::kLoads];
  // One step: the C chunks from k on, whose K and V are in kbuf and vbuf; the next
  // ones are requested as soon as their registers are free.
  auto step = [&](int k, const RowMask (&mask)[NB], auto drafts) {
    constexpr bool kDrafts = decltype(drafts)::value; // may hold drafts, or chunks past k1
    const int le = opaque_lane();
    float4v sc[NB][C];
#pragma unroll
    for (int nb = 0; nb < NB; nb++)
#pragma unroll
      for (int c = 0; c < C; c++) sc[nb][c] = Tr::qk(kbuf[c], q[nb]);
    look_up(k + C);
    load_k(k + C, kbuf);
    bool bad = false;
    asm volatile("" ::: "memory");
#pragma unroll
    for (int c = 0; c < C; c++) {
      int tokens = kChunkTokens;
      if constexpr (kDrafts) {
        tokens = k + c < k1 ? min(s.seq_len - (k + c) * kChunkTokens, kChunkTokens) : 0;
#pragma unroll
        for (int u = 0; u < Tr::kLoads; u++) bad |= Tr::v_row(le, u) < tokens && any_non_finite(vbuf[c][u]);
      }
      Tr::stage_v(lds + c * kChunkTokens * D, le, tokens, vbuf[c]);
    }
    load_v(k + C, vbuf);
    uint32_t vis[NB]; // kDrafts: of the step's tokens
#pragma unroll
    for (int nb = 0; nb < NB; nb++) {
      if constexpr (kDrafts) {
        vis[nb] = visible_bits(mask[nb], k * kChunkTokens - prefix);
        if (C == 1 || k + 1 >= k1) vis[nb] &= 0xffffu;
#pragma unroll
        for (int c = 0; c < C; c++)
#pragma unroll
          for (int i = 0; i < 4; i++) sc[nb][c][i] = (vis[nb] >> (16 * c + 4 * g + i)) & 1 ? sc[nb][c][i] : -INFINITY;
      }
      softmax(nb, sc[nb]);
    }
    // The V tiles are written by this wavefront's own lanes: wait for the LDS
    // writes before reads of other lanes' rows.
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    if constexpr (kDrafts) {
      // A draft's V may hold infinities and NaN: in a product, 0 times one of those
      // would reach the rows that do not see the draft.  They are added to the rows
      // that see them one by one, and cleared before the product.
      if (__any(bad)) {
        const int tokens = min(min(k + C, k1) * kChunkTokens, s.seq_len) - k * kChunkTokens;
        for (int t = 0; t < tokens; t++) {
#pragma unroll
          for (int n = 0; n < D / 16; n++) {
            // The lane's dims 16 n + 4 g + e of token t, where stage_v put them.
            const T* src = lds + t * D + (n ^ Tr::swz(t & 15)) * 16 + 4 * g;
#pragma unroll
            for (int e = 0; e < 4; e++) {
              const float x = non_finite_part(src[e]);
#pragma unroll
              for (int nb = 0; nb < NB; nb++) o[nb][n][e] += (vis[nb] >> t) & 1 ? x : 0.f;
            }
          }
        }
        for (int i = l; i < C * kChunkTokens * D; i += kWaveSize) lds[i] = finite_or_zero(lds[i]);
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      }
    }
    pv(le, sc);
  };

  if (k0 < k1) {
    RowMask mask[NB];
    if constexpr (TP) next_entry = load_entry(k0);
    look_up(k0);
    load_k(k0, kbuf);
    load_v(k0, vbuf);
    int k = k0;
    const int plain_end = min(k1, max(prefix, 0) / kChunkTokens); // chunks before it hold no draft
    for (; k + C <= plain_end; k += C) step(k, mask, std::false_type());
    if (k < k1) {
#pragma unroll
      for (int nb = 0; nb < NB; nb++) {
        bool valid;
        int r, i;
        row_of(nb, valid, r, i);
        mask[nb] = load_row_mask(p, s, i);
      }
      for (; k < k1; k += C) step(k, mask, std::true_type());
    }
  }

  // Every wavefront's rows into LDS over the V tiles, then they are merged, a
  // thread per 4 elements.
  __syncthreads();
#pragma unroll
  for (int nb = 0; nb < NB; nb++) {
    const float ltot = row_sum(lsum[nb]);
    const int rr = nb * 16 + (l & 15);
    float* dst = merge_o + (wave * kTileRows + rr) * kMergeStride;
#pragma unroll
    for (int n = 0; n < D / 16; n++) *reinterpret_cast<float4v*>(dst + 16 * n + 4 * g) = o[nb][n];
    if (g == 0) {
      merge_ml[(wave * kTileRows + rr) * 2 + 0] = m[nb];
      merge_ml[(wave * kTileRows + rr) * 2 + 1] = ltot;
    }
  }
  __syncthreads();
  constexpr int kCells = kTileRows * (D / 4); // float4 of the tile
  // (The thread's index is counted anew: no register holds it over the key loop.)
  int none = 0;
  asm volatile("" : "+s"(none));
  const int first_cell = wave * kWaveSize + __builtin_amdgcn_mbcnt_hi(~0u, __builtin_amdgcn_mbcnt_lo(~0u, none));
  for (int c = first_cell; c < kCells; c += kDraftWaves * kWaveSize) {
    const int rr = c / (D / 4), d = 4 * (c % (D / 4));
    const int rho = it.rt * kTileRows + rr;
    if (rho >= rows) break; // rows grow with c
    float mmax = -INFINITY;
#pragma unroll
    for (int j = 0; j < kDraftWaves; j++) mmax = fmaxf(mmax, merge_ml[(j * kTileRows + rr) * 2]);
    const float m_use = mmax == -INFINITY ? 0.f : mmax;
    float4v acc = {0.f, 0.f, 0.f, 0.f};
    float sum = 0.f;
#pragma unroll
    for (int j = 0; j < kDraftWaves; j++) {
      const float w = __builtin_amdgcn_exp2f(merge_ml[(j * kTileRows + rr) * 2] - m_use);
      sum += w * merge_ml[(j * kTileRows + rr) * 2 + 1];
      acc += w * *reinterpret_cast<const float4v*>(merge_o + (j * kTileRows + rr) * kMergeStride + d);
    }
    if (it.parts > 1) {
      const int64_t prow = slot * kTileRows + rr;
      *reinterpret_cast<float4v*>(p.partial_o + prow * D + d) = acc;
      if (d == 0) {
        p.partial_ml[prow * 2 + 0] = mmax;
        p.partial_ml[prow * 2 + 1] = sum;
      }
    } else {
      const int r = rho / s.q_len, i = rho - r * s.q_len;
      T* dst = static_cast<T*>(p.out) + (int64_t)(it.h * p.group_size + r) * p.out_stride_head +
               (int64_t)(s.q_start + i) * p.out_stride_token + d;
      Tr::store_out(dst, acc * inverse_sum(sum));
    }
  }
}

typedef __attribute__((address_space(4))) DraftAttentionParams const_params;

template <typename Tr, int D, int NB, bool TP>
__global__ __launch_bounds__(kWaveSize* kDraftWaves, (draft_blocks_per_cu(16 * NB, sizeof(typename Tr::elem) == 2, D))) void draft_stream_kernel(
    DraftAttentionParams) {
  constexpr int kTileRows = 16 * NB;
  constexpr size_t kTileBytes = (size_t)kDraftWaves * step_chunks<Tr>() * kChunkTokens * D * sizeof(typename Tr::elem);
  constexpr size_t kMergeBytes = (size_t)kDraftWaves * kTileRows * (D + 4 + 2) * sizeof(float);
  __shared__ __attribute__((aligned(16))) char lds_raw[kTileBytes > kMergeBytes ? kTileBytes : kMergeBytes];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWaveSize);
  // (One round, unless the device tables hold more than the host planned for.)
  // The parameters are read again each round: held over the loop, they and what is
  // worked out from them do not fit the registers.
  for (int round = 0;; round++) {
    auto args = (const const_params*)__builtin_amdgcn_kernarg_segment_ptr();
    asm volatile("" : "+s"(args));
    const DraftAttentionParams& p = *(const DraftAttentionParams*)args;
    const int w = first_item(p) + round * gridDim.x;
    const DraftItem it = find_item<kTileRows>(p, w);
    if (it.b >= p.num_seqs) break;
    if (it.rt < row_tiles_of<kTileRows>(p, it.s)) stream_item<Tr, D, NB, TP>(p, it, w, wave, lds_raw);
    __syncthreads(); // the LDS is used again
  }
}

// out = sum_j 2^(m_j - M) o_j / sum_j 2^(m_j - M) l_j over the parts of each row
// tile that was split; one thread per 4 elements, 4 parts' loads in flight, one
// pass with a running maximum.  A launch's own time: 4 to 6 us for 8 to 1,024 blocks.
template <typename Tr, int D, int kTileRows>
__global__ __launch_bounds__(256) void draft_merge_kernel(DraftAttentionParams p) {
  typedef typename Tr::elem T;
  constexpr int kAhead = 4;
  constexpr int kTileBlocks = (kTileRows * (D / 4) + 255) / 256;
  const int c = (int)(blockIdx.x % kTileBlocks) * 256 + threadIdx.x;
  const int rr = c / (D / 4), d = 4 * (c % (D / 4));
  int tile = (int)(blockIdx.x / kTileBlocks);
  const int rt = tile % p.row_tiles;
  tile /= p.row_tiles;
  const int h = tile % p.num_kv_heads, b = tile / p.num_kv_heads;
  // Items before the request's, and of the whole call.
  int base = 0, total = 0;
  DraftSeq s = {0, 0, 0};
  for (int b0 = 0; b0 < p.num_seqs; b0 += kWaveSize) {
    DraftSeq sl;
    const int n = items_of_lane<kTileRows>(p, b0, true, sl);
    const int incl = wave_inclusive_sum(n);
    if (b >= b0 && b < b0 + kWaveSize) {
      base = total + __builtin_amdgcn_readlane(incl - n, b - b0);
      s = uniform_seq(sl, b - b0);
    }
    total += __builtin_amdgcn_readlane(incl, kWaveSize - 1);
  }
  if (total > p.max_items) return; // nothing was split
  const int tiles = row_tiles_of<kTileRows>(p, s), parts = parts_of(p, s, true);
  const int rho = rt * kTileRows + rr;
  if (parts <= 1 || rr >= kTileRows || rho >= p.group_size * s.q_len) return;
  const int64_t stride = (int64_t)p.num_kv_heads * tiles * kTileRows; // rows from one part to the next
  const int64_t row0 = ((int64_t)base + h * tiles + rt) * kTileRows + rr;
  float4v acc = {0.f, 0.f, 0.f, 0.f};
  float sum = 0.f, m = -INFINITY;
  for (int j0 = 0; j0 < parts; j0 += kAhead) {
    float2v ml[kAhead];
    float4v o[kAhead];
#pragma unroll
    for (int u = 0; u < kAhead; u++) { // (past the last part: the last again, not counted)
      const int64_t row = row0 + min(j0 + u, parts - 1) * stride;
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
  const int r = rho / s.q_len, i = rho - r * s.q_len;
  T* dst = static_cast<T*>(p.out) + (int64_t)(h * p.group_size + r) * p.out_stride_head +
           (int64_t)(s.q_start + i) * p.out_stride_token + d;
  Tr::store_out(dst, acc * inverse_sum(sum));
}

template <typename Tr, int D, int NB>
hipError_t launch_stream(const DraftAttentionPlan& plan, const DraftAttentionParams& p, hipStream_t stream) {
  const dim3 grid((unsigned)plan.blocks), block(kWaveSize * kDraftWaves);
  if (p.page_size % kChunkTokens == 0)
    hipLaunchKernelGGL((draft_stream_kernel<Tr, D, NB, false>), grid, block, 0, stream, p);
  else
    hipLaunchKernelGGL((draft_stream_kernel<Tr, D, NB, true>), grid, block, 0, stream, p);
  return hipGetLastError();
}

template <typename Tr, int D, int kTileRows>
hipError_t launch_merge(const DraftAttentionParams& p, hipStream_t stream) {
  constexpr int kTileBlocks = (kTileRows * (D / 4) + 255) / 256;
  const dim3 grid((unsigned)kTileBlocks * (unsigned)(p.num_seqs * p.num_kv_heads * p.row_tiles));
  hipLaunchKernelGGL((draft_merge_kernel<Tr, D, kTileRows>), grid, dim3(256), 0, stream, p);
  return hipGetLastError();
}

template <typename Tr, int D>
hipError_t launch_dim(const DraftAttentionPlan& plan, const DraftAttentionParams& p, int dtype, hipStream_t stream) {
  hipError_t err = hipErrorInvalidValue;
  if (plan.tile_rows == 16) err = launch_stream<Tr, D, 1>(plan, p, stream);
  if constexpr (D <= 128) {
    if (plan.tile_rows == 32) err = launch_stream<Tr, D, 2>(plan, p, stream);
  }
  if (plan.tile_rows >= 64) err = launch_draft_tiles(plan, p, dtype, D, stream);
  if (err != hipSuccess || plan.max_items == 0) return err;
  switch (plan.tile_rows) {
  case 16: return launch_merge<Tr, D, 16>(p, stream);
  case 32: return launch_merge<Tr, D, 32>(p, stream);
  case 64: return launch_merge<Tr, D, 64>(p, stream);
  default: return launch_merge<Tr, D, 128>(p, stream);
  }
}

template <int D>
hipError_t launch_type(const DraftAttentionPlan& plan, const DraftAttentionParams& p, int dtype, hipStream_t stream) {
  return dtype == 1 ? launch_dim<F16Traits<D>, D>(plan, p, dtype, stream) : launch_dim<F32Traits<D>, D>(plan, p, dtype, stream);
}

} // namespace

hipError_t launch_draft_attention(const DraftAttentionPlan& plan, const DraftAttentionParams& params, int dtype,
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
