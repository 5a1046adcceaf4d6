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
#include "draft_attention.hpp"

#include "chunk_traits.hpp"
#include "wave_scan.hpp"

#include <math.h>

namespace mvr {
namespace {

constexpr int kDraftWaves = 4; // wavefronts per block
constexpr int kXcds = 8;

struct DraftSeq {
  int seq_len, q_start, q_len;
};

// The tables' loads, an absent table's from one that is there, go out together.
__device__ __forceinline__ DraftSeq load_draft_seq(const DraftAttentionParams& p, int b) {
  const int32_t* any = p.cu_q_lens ? p.cu_q_lens : p.seq_lens ? p.seq_lens : p.block_tables;
  const int seq_len = *(p.seq_lens ? p.seq_lens + b : any);
  const int q_start = *(p.cu_q_lens ? p.cu_q_lens + b : any);
  const int q_end = *(p.cu_q_lens ? p.cu_q_lens + b + 1 : any);
  DraftSeq s;
  // Clamped to the bounds that the host has checked tables and masks for.
  s.seq_len = p.seq_lens ? min(seq_len, p.max_seq_len) : p.max_seq_len;
  s.q_start = p.cu_q_lens ? q_start : 0;
  s.q_len = p.cu_q_lens ? min(q_end - q_start, p.max_q_len) : p.max_q_len;
  if (s.seq_len <= 0 || s.q_len <= 0) s.seq_len = s.q_len = 0;
  return s;
}

__device__ __forceinline__ DraftSeq uniform_seq(const DraftSeq& s, int src) {
  auto lane = [&](int v) { return __builtin_amdgcn_readlane(v, src); };
  return DraftSeq{lane(s.seq_len), lane(s.q_start), lane(s.q_len)};
}

template <int kTileRows>
__device__ __forceinline__ int row_tiles_of(const DraftAttentionParams& p, const DraftSeq& s) {
  return (p.group_size * s.q_len + kTileRows - 1) / kTileRows;
}

__device__ __forceinline__ int key_units_of(const DraftSeq& s) {
  return (s.seq_len + kDraftUnitTokens - 1) / kDraftUnitTokens;
}

// Parts of each of a request's row tiles (at least 1; only meaningful where it
// has rows).
__device__ __forceinline__ int parts_of(const DraftAttentionParams& p, const DraftSeq& s, bool split) {
  if (!split) return 1;
  return min((key_units_of(s) + p.part_units - 1) / p.part_units, kDraftMaxParts);
}

// Work of one block: part `part` of `parts` of row tile (b, h, rt).
struct DraftItem {
  int b, h, rt, part, parts;
  DraftSeq s;
};

// Items are numbered request by request, within a request part by part, KV head
// by KV head, and the row tiles of one (KV head, part), which read the same keys,
// next to each other.  One request per lane, 64 at a time.
struct DraftScan {
  int total;   // items of the whole call
  bool split;  // false: more items than slots, every row tile is one item
};

template <int kTileRows>
__device__ __forceinline__ int items_of_lane(const DraftAttentionParams& p, int b0, bool split, DraftSeq& s) {
  const int b = b0 + lane_id();
  s = load_draft_seq(p, min(b, p.num_seqs - 1));
  return b < p.num_seqs ? row_tiles_of<kTileRows>(p, s) * parts_of(p, s, split) * p.num_kv_heads : 0;
}

template <int kTileRows>
__device__ __forceinline__ int count_items(const DraftAttentionParams& p, bool split) {
  int total = 0;
  for (int b0 = 0; b0 < p.num_seqs; b0 += kWaveSize) {
    DraftSeq s;
    total += __builtin_amdgcn_readlane(wave_inclusive_sum(items_of_lane<kTileRows>(p, b0, split, s)), kWaveSize - 1);
  }
  return total;
}

// The request of item w and the item's number within it (false: no such item).
template <int kTileRows>
__device__ __forceinline__ bool find_request(const DraftAttentionParams& p, int w, bool split, int& b_out, int& local,
                                             DraftSeq& s_out) {
  for (int b0 = 0; b0 < p.num_seqs; b0 += kWaveSize) {
    DraftSeq s;
    const int n = items_of_lane<kTileRows>(p, b0, split, s);
    const int incl = wave_inclusive_sum(n);
    const int sum = __builtin_amdgcn_readlane(incl, kWaveSize - 1);
    if (w < sum) {
      const int src = __builtin_ctzll(__ballot(w < incl));
      b_out = b0 + src;
      local = w - __builtin_amdgcn_readlane(incl - n, src);
      s_out = uniform_seq(s, src);
      return true;
    }
    w -= sum;
  }
  return false;
}

// Block index -> item number: the blocks of one XCD (workgroups are dealt to
// the 8 XCDs round-robin) take a contiguous range of items, so that the row
// tiles of one (KV head, part) find each other's keys in that XCD's L2.
__device__ __forceinline__ int xcd_item(int block, int blocks) {
  const int xcd = block % kXcds, per = blocks / kXcds, more = blocks % kXcds;
  return xcd * per + min(xcd, more) + block / kXcds;
}

// Visibility of the 32 keys from slot `off` of the drafts on (negative: keys
// before the drafts, which every row sees), from the row's mask.
struct RowMask {
  const uint32_t* words; // the row's mask words
  uint32_t w0, w1;       // the first two
  int q_len;
};

__device__ __forceinline__ uint32_t mask_word(const RowMask& m, int k) {
  const int bits = m.q_len - 32 * k; // that belong to drafts
  if (bits <= 0) return 0;
  const uint32_t w = k == 0 ? m.w0 : k == 1 ? m.w1 : m.words[k];
  return bits >= 32 ? w : w & ((1u << bits) - 1);
}

__device__ __forceinline__ RowMask load_row_mask(const DraftAttentionParams& p, const DraftSeq& s, bool valid, int i) {
  RowMask m;
  m.words = p.masks + (int64_t)(s.q_start + i) * p.mask_words;
  m.q_len = valid ? s.q_len : 0; // a row that is none sees no draft
  m.w0 = valid ? m.words[0] : 0;
  m.w1 = valid && s.q_len > 32 ? m.words[1] : 0;
  return m;
}

__device__ __forceinline__ uint32_t visible_bits(const RowMask& m, int off) {
  if (off <= -32) return ~0u;
  if (off < 0) return (mask_word(m, 0) << -off) | ((1u << -off) - 1);
  const int k = off >> 5, sh = off & 31;
  const uint32_t lo = mask_word(m, k) >> sh;
  return sh ? lo | mask_word(m, k + 1) << (32 - sh) : lo;
}

// 0 for a row without a key (its sum is 0: no exponential was added), else 1 / sum.
__device__ __forceinline__ float inverse_sum(float sum) { return __float_as_uint(sum) == 0 ? 0.f : 1.f / sum; }

__device__ __forceinline__ bool any_non_finite(const half8& v) {
  typedef unsigned int u32x4 __attribute__((ext_vector_type(4)));
  const u32x4 x = __builtin_bit_cast(u32x4, v);
  bool bad = false;
#pragma unroll
  for (int e = 0; e < 4; e++) bad |= (x[e] & 0x7c00u) == 0x7c00u || (x[e] & 0x7c000000u) == 0x7c000000u;
  return bad;
}

__device__ __forceinline__ bool any_non_finite(const float4v& v) {
  bool bad = false;
#pragma unroll
  for (int e = 0; e < 4; e++) bad |= (__float_as_uint(v[e]) & 0x7f800000u) == 0x7f800000u;
  return bad;
}

// One value of V split into its finite part and whether it is +infinity (or
// NaN) or -infinity (or NaN): what a row that sees it gets, and only such a row.
template <typename T>
struct SplitValue {
  T finite, plus, minus;
};
__device__ __forceinline__ SplitValue<half_t> split_value(half_t v) {
  const uint16_t x = __builtin_bit_cast(uint16_t, v);
  const bool bad = (x & 0x7c00u) == 0x7c00u, nan = bad && (x & 0x3ffu);
  return {bad ? (half_t)0 : v, bad && (nan || !(x & 0x8000u)) ? (half_t)1 : (half_t)0,
          bad && (nan || (x & 0x8000u)) ? (half_t)1 : (half_t)0};
}
__device__ __forceinline__ SplitValue<float> split_value(float v) {
  const uint32_t x = __float_as_uint(v);
  const bool bad = (x & 0x7f800000u) == 0x7f800000u, nan = bad && (x & 0x7fffffu);
  return {bad ? 0.f : v, bad && (nan || !(x >> 31)) ? 1.f : 0.f, bad && (nan || (x >> 31)) ? 1.f : 0.f};
}

__device__ __forceinline__ void add_infinities(float4v& o, const float4v& plus, const float4v& minus) {
#pragma unroll
  for (int e = 0; e < 4; e++) {
    if (plus[e] > 0.f) o[e] += INFINITY;
    if (minus[e] > 0.f) o[e] -= INFINITY;
  }
}

// O^T += V^T P^T of a chunk whose V holds an infinity or a NaN: a masked key's
// 0 * infinity would reach every row of the product, so the finite values are
// multiplied by P and the others by the rows' visibility (1 or 0).
template <int D>
struct GuardedPv {
  template <int NB>
  __device__ static void run(F16Traits<D>, half_t* lds, int l, const float (&p)[NB][4], const uint32_t (&vis)[NB],
                             float4v (&o)[NB][D / 16]) {
    const int g = l >> 4, qd = l & 15;
    const int row = 4 * g + (qd >> 2);
    const int sw = F16Traits<D>::swz(row);
#pragma unroll
    for (int n = 0; n < D / 16; n++) {
      half_t* addr = lds + row * D + ((n ^ sw) * 16) + 4 * (qd & 3);
      const half4 vt = __builtin_bit_cast(half4, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_short4*)(addr)));
      half4 fin, plus, minus;
#pragma unroll
      for (int e = 0; e < 4; e++) {
        const SplitValue<half_t> sv = split_value(vt[e]);
        fin[e] = sv.finite, plus[e] = sv.plus, minus[e] = sv.minus;
      }
#pragma unroll
      for (int nb = 0; nb < NB; nb++) {
        half4 pb, seen;
#pragma unroll
        for (int e = 0; e < 4; e++) {
          pb[e] = (half_t)p[nb][e];
          seen[e] = (vis[nb] >> e) & 1 ? (half_t)1 : (half_t)0;
        }
        const float4v zero = {0.f, 0.f, 0.f, 0.f};
        o[nb][n] = __builtin_amdgcn_mfma_f32_16x16x16f16(fin, pb, o[nb][n], 0, 0, 0);
        add_infinities(o[nb][n], __builtin_amdgcn_mfma_f32_16x16x16f16(plus, seen, zero, 0, 0, 0),
                       __builtin_amdgcn_mfma_f32_16x16x16f16(minus, seen, zero, 0, 0, 0));
      }
    }
  }

  template <int NB>
  __device__ static void run(F32Traits<D>, float* lds, int l, const float (&p)[NB][4], const uint32_t (&vis)[NB],
                             float4v (&o)[NB][D / 16]) {
    const int g = l >> 4, qd = l & 15;
#pragma unroll
    for (int n = 0; n < D / 16; n++) {
      float4v plus[NB], minus[NB];
#pragma unroll
      for (int nb = 0; nb < NB; nb++) plus[nb] = minus[nb] = float4v{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int j = 0; j < 4; j++) {
        const int row = 4 * g + j;
        const SplitValue<float> sv = split_value(lds[row * D + ((n ^ F32Traits<D>::swz(row)) * 16) + qd]);
#pragma unroll
        for (int nb = 0; nb < NB; nb++) {
          const float seen = (vis[nb] >> j) & 1 ? 1.f : 0.f;
          o[nb][n] = __builtin_amdgcn_mfma_f32_16x16x4f32(sv.finite, p[nb][j], o[nb][n], 0, 0, 0);
          plus[nb] = __builtin_amdgcn_mfma_f32_16x16x4f32(sv.plus, seen, plus[nb], 0, 0, 0);
          minus[nb] = __builtin_amdgcn_mfma_f32_16x16x4f32(sv.minus, seen, minus[nb], 0, 0, 0);
        }
      }
#pragma unroll
      for (int nb = 0; nb < NB; nb++) add_infinities(o[nb][n], plus[nb], minus[nb]);
    }
  }
};

// ---------------------------------------------------------------------------
// Key streaming: a block of 4 wavefronts per item, 16 * NB rows, each wavefront
// its share of the part's 16-token chunks straight from the cache; their
// results merge in LDS.
// ---------------------------------------------------------------------------
// Chunks in flight per wavefront: two, one where two would not fit the registers
// (F32 rows of more than 128 elements hold a chunk of K and V in 160 to 256).
template <typename Tr, int D>
constexpr int stream_depth() {
  return sizeof(typename Tr::elem) == 4 && D > 128 ? 1 : 2;
}

// Blocks per CU (wavefronts per SIMD) that the registers allow without scratch.
// Rows with a page of their own (TP) hold an address each.
template <typename Tr, int D, int NB, bool TP>
constexpr int stream_blocks() {
  if (sizeof(typename Tr::elem) == 2) return D <= 64 ? 4 - NB : D <= 96 ? (TP ? 3 - NB : 2) : D <= 128 ? 3 - NB : D <= 160 ? 2 : 1;
  return D <= 64 || (D <= 96 && NB == 1) ? 2 : 1;
}

// TP: page sizes that are not a multiple of 16, where every token row has a page
// of its own to look up.
template <typename Tr, int D, int NB, bool TP>
__device__ __forceinline__ void stream_item(const DraftAttentionParams& p, const DraftItem& it, int64_t slot,
                                            char* lds_raw) {
  typedef typename Tr::elem T;
  constexpr int kTileRows = 16 * NB;
  constexpr int kMergeStride = D + 4;
  constexpr int kUnitChunks = kDraftUnitTokens / kChunkTokens;
  constexpr int kDepth = stream_depth<Tr, D>();
  float* const merge_o = reinterpret_cast<float*>(lds_raw);
  float* const merge_ml = merge_o + kDraftWaves * kTileRows * kMergeStride;

  const int l = lane_id(), g = l >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWaveSize);
  T* lds = reinterpret_cast<T*>(lds_raw) + (size_t)wave * kChunkTokens * D;
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

  // TP: the lane's K row is token l % 16 of the chunk; its page entry is read a
  // chunk ahead, and the V rows' pages come from the lanes that hold them.  Rows
  // past the last key read the last key's row (masked, and zeroed in LDS).
  auto load_entry = [&](int k) { return (uint32_t)bt[page_div(min(k * kChunkTokens + (l & 15), s.seq_len - 1))]; };
  uint32_t next_entry = 0;
  auto load_chunk = [&](int k, typename Tr::kreg_t (&kr)[Tr::kLoads], typename Tr::vreg_t (&vr)[Tr::kLoads]) {
    if constexpr (TP) {
      // (The lane index is opaque here, so that the rows' numbers are worked out
      // where they are used and not held, and spilled, over the key loop.)
      int le = l;
      asm volatile("" : "+v"(le));
      const uint32_t entry = min(next_entry, p.last_page);
      next_entry = load_entry(min(k + 1, k1 - 1));
      auto at = [&](int token_row, uint32_t page) {
        const int t = min(k * kChunkTokens + token_row, s.seq_len - 1);
        return ((uint64_t)page * page_rows + head_rows + (uint32_t)(t - page_div(t) * p.page_size)) * D;
      };
      Tr::load_k_row(kpool + at(le & 15, entry), le, kr);
#pragma unroll
      for (int u = 0; u < Tr::kLoads; u++) {
        const int row = Tr::v_row(le, u);
        vr[u] = Tr::load_v_row(vpool + at(row, (uint32_t)__shfl((int)entry, row)), le, u);
      }
    } else {
      const int t = k * kChunkTokens, pi = page_div(t);
      const uint32_t page = min((uint32_t)((const const_i32*)bt)[__builtin_amdgcn_readfirstlane(pi)], p.last_page);
      const uint64_t off = ((uint64_t)page * page_rows + head_rows + (uint32_t)(t - pi * p.page_size)) * D;
      Tr::load_k(kpool + off, l, kr);
      Tr::load_v(vpool + off, l, vr);
    }
  };

  // Scores of one row block to probabilities; rescales what the row holds.
  auto softmax = [&](int nb, const float (&sv)[4], float (&pr)[4]) {
    const float mx = wave_max_across_groups(fmaxf(fmaxf(sv[0], sv[1]), fmaxf(sv[2], sv[3])));
    const float m_new = fmaxf(m[nb], mx);
    const float m_use = m_new == -INFINITY ? 0.f : m_new;
    const float alpha = __builtin_amdgcn_exp2f(m[nb] - m_use);
    float psum = 0.f;
#pragma unroll
    for (int i = 0; i < 4; i++) {
      pr[i] = __builtin_amdgcn_exp2f(sv[i] - m_use);
      psum += pr[i];
    }
    lsum[nb] = lsum[nb] * alpha + psum;
    m[nb] = m_new;
#pragma unroll
    for (int n = 0; n < D / 16; n++) o[nb][n] *= alpha;
  };

  // A chunk before the drafts: every row sees all of it.
  auto process = [&](const typename Tr::kreg_t (&kr)[Tr::kLoads], const typename Tr::vreg_t (&vr)[Tr::kLoads]) {
    asm volatile("" ::: "memory");
    Tr::stage_v(lds, l, kChunkTokens, vr);
    float pr[NB][4];
#pragma unroll
    for (int nb = 0; nb < NB; nb++) {
      const float4v sc = Tr::qk(kr, q[nb]);
      const float sv[4] = {sc[0] * p.scale_log2, sc[1] * p.scale_log2, sc[2] * p.scale_log2, sc[3] * p.scale_log2};
      softmax(nb, sv, pr[nb]);
    }
    // The V tile is written by this wavefront's own lanes: wait for the LDS
    // writes before the transposed reads of other lanes' rows.
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    Tr::template pv<NB>(lds, l, pr, o);
  };

  // Any chunk, under the rows' masks.
  auto process_drafts = [&](int k, const RowMask (&mask)[NB], const typename Tr::kreg_t (&kr)[Tr::kLoads],
                            const typename Tr::vreg_t (&vr)[Tr::kLoads]) {
    const int tok0 = k * kChunkTokens;
    asm volatile("" ::: "memory");
    Tr::stage_v(lds, l, s.seq_len - tok0, vr);
    bool bad = false;
#pragma unroll
    for (int u = 0; u < Tr::kLoads; u++) bad |= Tr::v_row(l, u) < s.seq_len - tok0 && any_non_finite(vr[u]);
    uint32_t vis[NB]; // of the lane's 4 tokens
    float pr[NB][4];
#pragma unroll
    for (int nb = 0; nb < NB; nb++) {
      const float4v sc = Tr::qk(kr, q[nb]);
      vis[nb] = visible_bits(mask[nb], tok0 - prefix) >> (4 * g);
      float sv[4];
#pragma unroll
      for (int i = 0; i < 4; i++) sv[i] = (vis[nb] >> i) & 1 ? sc[i] * p.scale_log2 : -INFINITY;
      softmax(nb, sv, pr[nb]);
    }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    if (__any(bad))
      GuardedPv<D>::template run<NB>(Tr{}, lds, l, pr, vis, o);
    else
      Tr::template pv<NB>(lds, l, pr, o);
  };

  // kDepth chunks in flight; a tail past k1 reloads chunk k1 - 1 (an L2 hit)
  // rather than branching.  Whole rounds of chunks before the drafts first.
  typename Tr::kreg_t kbuf[kDepth][Tr::kLoads];
  typename Tr::vreg_t vbuf[kDepth][Tr::kLoads];
  if (k0 < k1) {
    if constexpr (TP) next_entry = load_entry(k0);
#pragma unroll
    for (int i = 0; i < kDepth; i++) load_chunk(min(k0 + i, k1 - 1), kbuf[i], vbuf[i]);
    int k = k0;
    const int plain_end = min(k1, max(prefix, 0) / kChunkTokens); // chunks before it hold no draft
    for (; k + kDepth <= plain_end; k += kDepth) {
#pragma unroll
      for (int i = 0; i < kDepth; i++) {
        process(kbuf[i], vbuf[i]);
        load_chunk(min(k + i + kDepth, k1 - 1), kbuf[i], vbuf[i]);
      }
    }
    if (k < k1) {
      RowMask mask[NB];
#pragma unroll
      for (int nb = 0; nb < NB; nb++) {
        bool valid;
        int r, i;
        row_of(nb, valid, r, i);
        mask[nb] = load_row_mask(p, s, valid, i);
      }
      for (; k < k1; k += kDepth) {
#pragma unroll
        for (int i = 0; i < kDepth; i++) {
          if (k + i < k1) {
            process_drafts(k + i, mask, kbuf[i], vbuf[i]);
            load_chunk(min(k + i + kDepth, k1 - 1), kbuf[i], vbuf[i]);
          }
        }
      }
    }
  }

  // Every wavefront's rows into LDS over the V tiles, then rows wave, wave + 4,
  // ... are merged, a lane per 4 elements (the lanes past D / 4 re-read the last).
  __syncthreads();
#pragma unroll
  for (int nb = 0; nb < NB; nb++) {
    const float ltot = wave_sum_across_groups(lsum[nb]);
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
  for (int c = threadIdx.x; c < kCells; c += kDraftWaves * kWaveSize) {
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

template <typename Tr, int D, int NB, bool TP>
__global__ __launch_bounds__(kWaveSize* kDraftWaves, (stream_blocks<Tr, D, NB, TP>())) void draft_stream_kernel(
    DraftAttentionParams p) {
  constexpr int kTileRows = 16 * NB;
  constexpr size_t kTileBytes = (size_t)kDraftWaves * kChunkTokens * D * sizeof(typename Tr::elem);
  constexpr size_t kMergeBytes = (size_t)kDraftWaves * kTileRows * (D + 4 + 2) * sizeof(float);
  __shared__ __attribute__((aligned(16))) char lds_raw[kTileBytes > kMergeBytes ? kTileBytes : kMergeBytes];
  const int first = xcd_item(blockIdx.x, gridDim.x);
  if (p.part_units == 0) {
    DraftItem it;
    it.rt = first % p.row_tiles;
    it.h = (first / p.row_tiles) % p.num_kv_heads;
    it.b = first / (p.row_tiles * p.num_kv_heads);
    it.part = 0, it.parts = 1;
    it.s = uniform_seq(load_draft_seq(p, it.b), 0);
    if (it.rt < row_tiles_of<kTileRows>(p, it.s)) stream_item<Tr, D, NB, TP>(p, it, 0, lds_raw);
    return;
  }
  const bool split = count_items<kTileRows>(p, true) <= p.max_items;
  // (One round, unless the device tables hold more than the host planned for.)
  for (int w = first;; w += gridDim.x) {
    DraftItem it;
    int local;
    if (!find_request<kTileRows>(p, w, split, it.b, local, it.s)) break;
    const int tiles = row_tiles_of<kTileRows>(p, it.s);
    it.rt = local % tiles;
    it.h = (local / tiles) % p.num_kv_heads;
    it.part = local / (tiles * p.num_kv_heads);
    it.parts = parts_of(p, it.s, split);
    stream_item<Tr, D, NB, TP>(p, it, w, lds_raw);
    __syncthreads(); // the LDS is used again
  }
}

// out = sum_j 2^(m_j - M) o_j / sum_j 2^(m_j - M) l_j over the parts of each row
// tile that was split; one thread per 4 elements.
template <typename Tr, int D, int kTileRows>
__global__ __launch_bounds__(256) void draft_merge_kernel(DraftAttentionParams p) {
  typedef typename Tr::elem T;
  const int c = blockIdx.x * 256 + threadIdx.x;
  const int rr = c / (D / 4), d = 4 * (c % (D / 4));
  int tile = blockIdx.y;
  const int rt = tile % p.row_tiles;
  tile /= p.row_tiles;
  const int h = tile % p.num_kv_heads, b = tile / p.num_kv_heads;
  // Items before the request's, and of the whole call.
  int base = 0, total = 0;
  for (int b0 = 0; b0 < p.num_seqs; b0 += kWaveSize) {
    DraftSeq sl;
    const int n = items_of_lane<kTileRows>(p, b0, true, sl);
    const int incl = wave_inclusive_sum(n);
    if (b >= b0 && b < b0 + kWaveSize) base = total + __builtin_amdgcn_readlane(incl - n, b - b0);
    total += __builtin_amdgcn_readlane(incl, kWaveSize - 1);
  }
  if (total > p.max_items) return; // nothing was split
  const DraftSeq s = load_draft_seq(p, b);
  const int tiles = row_tiles_of<kTileRows>(p, s), parts = parts_of(p, s, true);
  const int rho = rt * kTileRows + rr;
  if (parts <= 1 || rr >= kTileRows || rho >= p.group_size * s.q_len) return;
  const int64_t stride = (int64_t)p.num_kv_heads * tiles * kTileRows; // rows from one part to the next
  const int64_t row0 = ((int64_t)base + h * tiles + rt) * kTileRows + rr;
  float mmax = -INFINITY;
  for (int j = 0; j < parts; j++) mmax = fmaxf(mmax, p.partial_ml[(row0 + j * stride) * 2]);
  const float m_use = mmax == -INFINITY ? 0.f : mmax;
  float4v acc = {0.f, 0.f, 0.f, 0.f};
  float sum = 0.f;
  for (int j = 0; j < parts; j++) {
    const float2v ml = *reinterpret_cast<const float2v*>(p.partial_ml + (row0 + j * stride) * 2);
    const float w = __builtin_amdgcn_exp2f(ml[0] - m_use);
    sum += w * ml[1];
    acc += w * *reinterpret_cast<const float4v*>(p.partial_o + (row0 + j * stride) * D + d);
  }
  const int r = rho / s.q_len, i = rho - r * s.q_len;
  T* dst = static_cast<T*>(p.out) + (int64_t)(h * p.group_size + r) * p.out_stride_head +
           (int64_t)(s.q_start + i) * p.out_stride_token + d;
  Tr::store_out(dst, acc * inverse_sum(sum));
}

template <typename Tr, int D, int NB>
hipError_t launch_rows(const DraftAttentionPlan& plan, const DraftAttentionParams& p, hipStream_t stream) {
  const dim3 grid((unsigned)plan.blocks), block(kWaveSize * kDraftWaves);
  if (p.page_size % kChunkTokens == 0)
    hipLaunchKernelGGL((draft_stream_kernel<Tr, D, NB, false>), grid, block, 0, stream, p);
  else
    hipLaunchKernelGGL((draft_stream_kernel<Tr, D, NB, true>), grid, block, 0, stream, p);
  hipError_t err = hipGetLastError();
  if (err != hipSuccess || plan.max_items == 0) return err;
  constexpr int kCells = 16 * NB * (D / 4);
  const dim3 merge((kCells + 255) / 256, (unsigned)(p.num_seqs * p.num_kv_heads * p.row_tiles));
  hipLaunchKernelGGL((draft_merge_kernel<Tr, D, 16 * NB>), merge, dim3(256), 0, stream, p);
  return hipGetLastError();
}

template <typename Tr, int D>
hipError_t launch_dim(const DraftAttentionPlan& plan, const DraftAttentionParams& p, hipStream_t stream) {
  if (plan.tile_rows == 16) return launch_rows<Tr, D, 1>(plan, p, stream);
  if constexpr (D <= 128) {
    if (plan.tile_rows == 32) return launch_rows<Tr, D, 2>(plan, p, stream);
  }
  return hipErrorInvalidValue;
}

template <int D>
hipError_t launch_type(const DraftAttentionPlan& plan, const DraftAttentionParams& p, int dtype, hipStream_t stream) {
  return dtype == 1 ? launch_dim<F16Traits<D>, D>(plan, p, stream) : launch_dim<F32Traits<D>, D>(plan, p, stream);
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
