// What the drafted-tree attention kernels share: the requests' lengths, which
// part of which row tile a block works on, the rows' masks.
#pragma once

#include "draft_attention.hpp"
#include "row_helpers.hpp"
#include "wave_scan.hpp"

#include <math.h>

namespace mvr {
namespace {

constexpr int kDraftWaves = 4; // wavefronts per block

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
template <int kTileRows>
__device__ __forceinline__ int items_of_lane(const DraftAttentionParams& p, int b0, bool split, DraftSeq& s) {
  const int b = b0 + lane_id();
  s = load_draft_seq(p, min(b, p.num_seqs - 1));
  return b < p.num_seqs ? row_tiles_of<kTileRows>(p, s) * parts_of(p, s, split) * p.num_kv_heads : 0;
}

// The request of item w (b = num_seqs: no such item), the item's number within it,
// and the items of the whole call.
struct FoundRequest {
  int b, local, total;
  DraftSeq s;
};

template <int kTileRows>
__device__ __forceinline__ FoundRequest find_request(const DraftAttentionParams& p, int w, bool split) {
  FoundRequest f = {p.num_seqs, 0, 0, DraftSeq{0, 0, 0}};
  for (int b0 = 0; b0 < p.num_seqs; b0 += kWaveSize) {
    DraftSeq s;
    const int n = items_of_lane<kTileRows>(p, b0, split, s);
    const int incl = wave_inclusive_sum(n);
    const int sum = __builtin_amdgcn_readlane(incl, kWaveSize - 1), at = w - f.total;
    if (at >= 0 && at < sum) {
      const int src = __builtin_ctzll(__ballot(at < incl));
      f.b = b0 + src;
      f.local = at - __builtin_amdgcn_readlane(incl - n, src);
      f.s = uniform_seq(s, src);
    }
    f.total += sum;
  }
  return f;
}

// The request that is `rank`-th by length, longest first, among the 64 that its
// number falls among.
__device__ __forceinline__ int request_of_rank(const DraftAttentionParams& p, int rank, DraftSeq& s) {
  const int l = lane_id(), b0 = rank & ~(kWaveSize - 1), n = min(kWaveSize, p.num_seqs - b0);
  const DraftSeq sl = load_draft_seq(p, b0 + min(l, n - 1));
  const uint32_t key = l < n ? (uint32_t)key_units_of(sl) * kWaveSize + (kWaveSize - 1 - l) : 0; // all different
  int longer = l < n ? 0 : kWaveSize;
#pragma unroll 1
  for (int j = 0; j < n; j++) longer += (uint32_t)__builtin_amdgcn_readlane((int)key, j) > key;
  const int at = __builtin_ctzll(__ballot(longer == rank - b0));
  s = uniform_seq(sl, at);
  return b0 + at;
}

// Item w of the call (b = num_seqs: past the last one).  Calls that are not split
// have an item for every request, KV head and row tile of the longest request
// (rt past the request's own row tiles: no work), and no scan: blocks w % 8, which
// run on one XCD, take the (request, KV head) pairs that are w % 8 modulo 8, row
// tile by row tile.  Requests of unequal lengths load the XCDs alike that way, and
// with by_length the longest start first (F16, 64 requests of 60 drafts on
// 300..4,000 keys, 28 / 4 heads of 128: 190 -> 164 us; F32, 40 of 10 on 100..1,500,
// 24 / 8 heads: 96 -> 81).
template <int kTileRows>
__device__ __forceinline__ DraftItem find_item(const DraftAttentionParams& p, int w) {
  if (p.part_units == 0) {
    const uint32_t of_xcd = (uint32_t)w / kDraftXcds, eight = of_xcd / (uint32_t)p.row_tiles;
    const uint32_t pair = eight * kDraftXcds + (uint32_t)w % kDraftXcds;
    const int rank = (int)(pair / (uint32_t)p.num_kv_heads);
    DraftItem it = {p.num_seqs, (int)pair - rank * p.num_kv_heads, (int)(of_xcd - eight * p.row_tiles), 0, 1, {0, 0, 0}};
    if (rank >= p.num_seqs) return it;
    if (p.by_length) {
      it.b = request_of_rank(p, rank, it.s);
    } else {
      it.b = rank;
      it.s = uniform_seq(load_draft_seq(p, rank), 0);
    }
    return it;
  }
  FoundRequest f = find_request<kTileRows>(p, w, true);
  const bool split = f.total <= p.max_items;
  if (!split) f = find_request<kTileRows>(p, w, false); // more items than slots: every row tile is one
  const int tiles = max(row_tiles_of<kTileRows>(p, f.s), 1), parts = parts_of(p, f.s, split);
  const int rest = f.local / tiles;
  return DraftItem{f.b, rest % p.num_kv_heads, f.local % tiles, rest / p.num_kv_heads, parts, f.s};
}

// The block's first item.  In a split call the blocks of one XCD (workgroups are
// dealt to the 8 XCDs round-robin) take a contiguous range of items, so that the
// row tiles of one (KV head, part) find each other's keys in that XCD's L2.
__device__ __forceinline__ int first_item(const DraftAttentionParams& p) {
  const uint32_t block = blockIdx.x, blocks = gridDim.x;
  if (p.part_units == 0) return (int)block;
  const uint32_t xcd = block % kDraftXcds, per = blocks / kDraftXcds, more = blocks % kDraftXcds;
  return (int)(xcd * per + min(xcd, more) + block / kDraftXcds);
}

// Visibility of the 32 keys from slot `off` of the drafts on (negative: keys
// before the drafts, which every row sees), from the row's mask.
struct RowMask {
  const uint32_t* masks;
  int mask_words, row;
  uint32_t w0, w1; // the first two words
  int q_len;
};

__device__ __forceinline__ uint32_t mask_word(const RowMask& m, int k) {
  const int bits = m.q_len - 32 * k; // that belong to drafts
  if (bits <= 0) return 0;
  int row = m.row;
  asm volatile("" : "+v"(row)); // (or the address is held over the key loop)
  const uint32_t w = k == 0 ? m.w0 : k == 1 ? m.w1 : m.masks[(int64_t)row * m.mask_words + k];
  return bits >= 32 ? w : w & ((1u << bits) - 1);
}

// (A tile row past the request's last is given row 0's: what it comes to is not stored.)
__device__ __forceinline__ RowMask load_row_mask(const DraftAttentionParams& p, const DraftSeq& s, int i) {
  RowMask m;
  m.masks = p.masks;
  m.mask_words = p.mask_words;
  m.row = s.q_start + i;
  m.q_len = s.q_len;
  const uint32_t* words = m.masks + (int64_t)m.row * m.mask_words;
  m.w0 = words[0];
  m.w1 = s.q_len > 32 ? words[1] : 0;
  return m;
}

__device__ __forceinline__ uint32_t visible_bits(const RowMask& m, int off) {
  if (off <= -32) return ~0u;
  if (off < 0) return (mask_word(m, 0) << -off) | ((1u << -off) - 1);
  const int k = off >> 5, sh = off & 31;
  const uint32_t lo = mask_word(m, k) >> sh;
  return sh ? lo | mask_word(m, k + 1) << (32 - sh) : lo;
}

} // namespace
} // namespace mvr
