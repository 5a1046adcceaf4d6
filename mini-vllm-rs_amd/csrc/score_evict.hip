// The cut of a cache to the tokens that got most attention, for gfx950 (MI355X, CDNA4):
// which tokens stay, and the moves of those that stay past the new length.
#include "score_attention.hpp"

#include <limits.h>

#include <type_traits>

#include "cache_rows.hpp"
#include "wave_scan.hpp"

namespace mvr {
namespace {

typedef __attribute__((address_space(4))) int32_t const_i32;

constexpr int kWave = 64;

// ---------------------------------------------------------------------------
// Which tokens stay: a block per (layer, request, KV head).
//
// Ranks become a search for one number.  A token's key is 2^32 - 1 where it is
// protected, else its weight's bits in an order that ascends with the weight (a NaN's is
// -infinity's; 0, below all, for tokens in pages outside the pool).  The keep-th largest
// key T is found digit by digit from the top, with a histogram of the digit of the keys
// that share the digits found before; tokens above T stay, and of those at T the lowest
// slots, as many as are missing.  What stays past slot `keep` and what goes below it are
// as many, and are paired in ascending order.
//
// The weights are read once, and their keys held in LDS for the passes over them; a
// thread takes four slots at a time, with one 16-byte access each to weights, positions
// and keys where pages hold whole fours (VEC; 8 heads of 32 requests of 8,000 tokens, 4
// layers: 38 us, in 6-token pages 44).  Not bound by the bytes: by a block's own chain
// of steps where blocks are few (2 heads of 1,040 tokens in 24 layers: 6.7 us), by the
// vector unit, some 100 instructions per four slots and pass, where they are many (8 heads
// of 16 requests of 1,500 to 8,000 tokens in 8 layers: 30.5 us, the bytes' 8.3).
// ---------------------------------------------------------------------------
constexpr int kDigitBits = 11, kDigits = 3, kBins = 1 << kDigitBits;
constexpr int kFour = 4; // slots of a thread at a time
// Keys that LDS holds beside the histogram: of four blocks to a CU, or of two.  Requests
// that may be longer read weights and positions anew in each pass (the same 8,000 tokens,
// where max_seq_len lets them be longer: 50 us).
constexpr int kFewKeys = 8128, kManyKeys = 17408;

typedef int int4v __attribute__((ext_vector_type(4)));
typedef float float4v __attribute__((ext_vector_type(4)));

__device__ __forceinline__ uint32_t ascending(float w) {
  const int x = __float_as_int(w != w ? -INFINITY : w + 0.f); // (-0 is 0)
  return (uint32_t)(x ^ (x >> 31 | INT_MIN));
}

// Lanes below this one that are in `lanes`, and `more`.
__device__ __forceinline__ int lanes_before(uint64_t lanes, int more) {
  return __builtin_amdgcn_mbcnt_hi((uint32_t)(lanes >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)lanes, more));
}

template <int kSelectThreads, int kHeldKeys, bool VEC>
__global__ __launch_bounds__(kSelectThreads, 8) void select_tokens_kernel(SelectTokensParams p) {
  constexpr bool HELD = kHeldKeys > 0;
  constexpr int kSelectWaves = kSelectThreads / kWave, kThreadBins = kBins / kSelectThreads;
  static_assert(kFour * kSelectThreads <= kSelectStep, "slots are counted in 32 bits");
  __shared__ int bins[kBins];
  __shared__ int wave_counts[kSelectWaves][4];
  __shared__ int found[2]; // digit, keys above it
  __shared__ __attribute__((aligned(16))) uint32_t held[kHeldKeys + kFour];
  const int tid = threadIdx.x, l = tid % kWave, wave = __builtin_amdgcn_readfirstlane(tid / kWave);
  // The KV heads of one table follow each other on one XCD (workgroups are dealt to the 8
  // XCDs round-robin): their weights share cache lines.
  const unsigned of_xcd = blockIdx.x / 8, eight = of_xcd / (unsigned)p.num_kv_heads;
  const int table = (int)(eight * 8 + blockIdx.x % 8), h = (int)(of_xcd - eight * p.num_kv_heads);
  if (table >= p.num_layers * p.num_seqs) return;
  const int row = table * p.num_kv_heads + h, b = table % p.num_seqs;
  const const_i32* lens = (const const_i32*)p.seq_lens;
  const int n = max(0, min(lens[b], p.max_seq_len));
  const int next = p.next_positions ? ((const const_i32*)p.next_positions)[b] : n;
  const int kept = p.kept_lens ? min(((const const_i32*)p.kept_lens)[b], n) : 0;
  int keep = max(0, min(((const const_i32*)p.keep_lens)[b], n));
  if (min(keep, n - keep) > p.max_moves) keep = n; // (its moves might not fit)
  if (table < p.num_seqs && h == 0 && tid == 0 && p.new_seq_lens) p.new_seq_lens[b] = keep;
  const bool cut = keep != n && keep != 0; // (else nothing goes, or nothing stays)
  const int last_from = (int)max((int64_t)next - p.recent, (int64_t)INT_MIN); // positions of the last `recent`
  int32_t* const count = p.num_moves + row;
  if (!cut && tid == 0) *count = 0;

  const int32_t* bt = p.block_tables + (int64_t)table * p.block_table_stride;
  const uint32_t page_rows = (uint32_t)(p.num_kv_heads * p.page_size);
  const int head_rows = h * p.page_size;
  // Index of slot t in the pools, or -1.
  auto index_of = [&](int t) -> int64_t {
    const int pi = (int)(((uint64_t)(uint32_t)t * p.page_magic) >> p.page_magic_shift), page = bt[pi];
    if (page < 0 || page >= p.num_pages) return -1;
    return (int64_t)((uint64_t)(uint32_t)page * page_rows + (uint32_t)(head_rows + (t - pi * p.page_size)));
  };
  // Keys of slots t, t + stride, ... (VEC: stride 1; 0 past the last one, and in pages
  // outside the pool), and where `writes` is set the positions of those that were appended
  // since the last cut.
  auto read_four = [&](int t, int stride, bool writes, uint32_t (&key)[kFour]) __attribute__((always_inline)) {
    int64_t at[kFour];
    float w[kFour];
    int pos[kFour];
    if constexpr (VEC) {
      const int64_t first = index_of(t), some = max(first, (int64_t)0);
      const float4v w4 = *reinterpret_cast<const float4v*>(p.weights + some);
      int4v pos4 = {0, 0, 0, 0};
      if (t < kept) pos4 = *reinterpret_cast<const int4v*>(p.positions + some);
#pragma unroll
      for (int j = 0; j < kFour; j++) {
        at[j] = first < 0 ? -1 : first + j;
        w[j] = w4[j];
        pos[j] = pos4[j];
      }
    } else {
#pragma unroll
      for (int j = 0; j < kFour; j++) at[j] = index_of(min(t + stride * j, n - 1));
#pragma unroll
      for (int j = 0; j < kFour; j++) {
        const int64_t some = max(at[j], (int64_t)0);
        w[j] = p.weights[some];
        pos[j] = 0;
        if (t + stride * j < kept) pos[j] = p.positions[some];
      }
    }
    int4v fresh;
    bool all = at[0] >= 0 && t + kFour <= n;
#pragma unroll
    for (int j = 0; j < kFour; j++) {
      const int slot = t + stride * j;
      fresh[j] = next - (n - slot);
      all &= slot >= kept;
      if (slot >= kept) pos[j] = fresh[j];
      const bool guarded = pos[j] < p.first || pos[j] >= last_from;
      key[j] = slot >= n || at[j] < 0 ? 0 : guarded ? ~0u : ascending(w[j]);
    }
    if (!writes) return;
    if (VEC && all) {
      *reinterpret_cast<int4v*>(p.positions + at[0]) = fresh;
    } else {
#pragma unroll
      for (int j = 0; j < kFour; j++)
        if (t + stride * j < n && t + stride * j >= kept && at[j] >= 0) p.positions[at[j]] = fresh[j];
    }
  };
  auto keys_of = [&](int t, uint32_t (&key)[kFour]) {
    if constexpr (HELD) {
      const int4v x = *reinterpret_cast<const int4v*>(held + t);
#pragma unroll
      for (int j = 0; j < kFour; j++) key[j] = (uint32_t)x[j];
    } else {
      read_four(t, 1, false, key);
    }
  };
  for (int i = tid; i < kBins; i += kSelectThreads) bins[i] = 0;
  const int t_begin = HELD && cut ? 0 : max(kept, 0) / kFour * kFour;
  if constexpr (VEC || !HELD) {
    for (int t = t_begin + kFour * tid; t < n; t += kFour * kSelectThreads) {
      uint32_t key[kFour];
      read_four(t, 1, true, key);
      if (HELD && cut) *reinterpret_cast<int4v*>(held + t) = int4v{(int)key[0], (int)key[1], (int)key[2], (int)key[3]};
    }
  } else { // (a slot's neighbours to the lanes beside)
    for (int t = t_begin + tid; t < n; t += kFour * kSelectThreads) {
      uint32_t key[kFour];
      read_four(t, kSelectThreads, true, key);
#pragma unroll
      for (int j = 0; j < kFour; j++)
        if (cut && t + kSelectThreads * j < n) held[t + kSelectThreads * j] = key[j];
    }
  }
  if (!cut) return;
  __syncthreads();

  // The keep-th largest key.
  uint32_t prefix = 0, known = 0; // digits found, and which bits they are
  int missing = keep;             // of the keys with those digits, the missing-th largest is T
  for (int digit = kDigits - 1; digit >= 0; digit--) {
    const int shift = digit * kDigitBits;
    for (int t = kFour * tid; t < n; t += kFour * kSelectThreads) {
      uint32_t key[kFour];
      keys_of(t, key);
#pragma unroll
      for (int j = 0; j < kFour; j++)
        if (t + j < n && (key[j] & known) == prefix) atomicAdd(&bins[(key[j] >> shift) & (kBins - 1)], 1);
    }
    __syncthreads();
    // Keys above each bin: a scan from the top, kThreadBins bins per thread.
    const int top = kBins - 1 - kThreadBins * tid;
    int in_bin[kThreadBins], mine = 0;
#pragma unroll
    for (int i = 0; i < kThreadBins; i++) {
      mine += in_bin[i] = bins[top - i];
      bins[top - i] = 0; // (for the next digit)
    }
    const int incl = wave_inclusive_sum(mine);
    if (l == kWave - 1) wave_counts[wave][0] = incl;
    __syncthreads();
    const int waves_upto = wave_inclusive_sum(l < kSelectWaves ? wave_counts[l][0] : 0); // lane l: wavefronts 0 .. l
    int above = incl - mine + (wave ? __builtin_amdgcn_readlane(waves_upto, max(wave - 1, 0)) : 0);
#pragma unroll
    for (int i = 0; i < kThreadBins; i++) {
      if (above < missing && above + in_bin[i] >= missing) {
        found[0] = top - i;
        found[1] = above;
      }
      above += in_bin[i];
    }
    __syncthreads();
    prefix |= (uint32_t)found[0] << shift;
    known |= (uint32_t)(kBins - 1) << shift;
    missing -= found[1];
  }
  // Tokens above T stay, and the first `missing` at T.  Each wavefront looks at a run of
  // slots of its own.  What its run holds: tokens at T, those of them below slot `keep`,
  // tokens below T in slots below `keep`, tokens above T in the others.
  constexpr int kWaveSlots = kFour * kWave;
  const int run = (n + kSelectWaves * kWaveSlots - 1) / (kSelectWaves * kWaveSlots) * kWaveSlots;
  const int t0 = min(wave * run, n), t1 = min(t0 + run, n);
  int ties = 0, low_ties = 0, holes = 0, movers = 0;
  for (int base = t0; base < t1; base += kWaveSlots) {
    const int t = base + kFour * l;
    uint32_t key[kFour] = {0, 0, 0, 0};
    if (t < t1) keys_of(t, key);
    if (base + kWaveSlots <= min(t1, keep)) { // whole, in slots below `keep`
#pragma unroll
      for (int j = 0; j < kFour; j++) {
        const int at_t = __popcll(__ballot(key[j] == prefix));
        ties += at_t;
        low_ties += at_t;
        holes += __popcll(__ballot(key[j] < prefix));
      }
    } else {
#pragma unroll
      for (int j = 0; j < kFour; j++) {
        const bool in = t + j < t1, low = t + j < keep, tie = in && key[j] == prefix;
        ties += __popcll(__ballot(tie));
        low_ties += __popcll(__ballot(tie && low));
        holes += __popcll(__ballot(in && key[j] < prefix && low));
        movers += __popcll(__ballot(in && key[j] > prefix && !low));
      }
    }
  }
  if (l == 0) {
    wave_counts[wave][0] = ties;
    wave_counts[wave][1] = low_ties;
    wave_counts[wave][2] = holes;
    wave_counts[wave][3] = movers;
  }
  __syncthreads();
  // The runs before it (lane l: run l): of a run's tokens at T the first ones stay, which
  // are those below `keep` first.
  const bool is_run = l < kSelectWaves;
  const int at_t = is_run ? wave_counts[l][0] : 0, low = is_run ? wave_counts[l][1] : 0;
  const int ties_before = wave_inclusive_sum(at_t) - at_t, stay = max(0, min(missing - ties_before, at_t));
  const int goes_in = is_run ? wave_counts[l][2] + low - min(low, stay) : 0;
  const int comes_from = is_run ? wave_counts[l][3] + max(0, stay - low) : 0;
  const int holes_upto = wave_inclusive_sum(goes_in), movers_upto = wave_inclusive_sum(comes_from);
  int my_ties = __builtin_amdgcn_readlane(ties_before, wave);
  int my_hole = __builtin_amdgcn_readlane(holes_upto - goes_in, wave);
  int my_mover = __builtin_amdgcn_readlane(movers_upto - comes_from, wave);
  const int all = __builtin_amdgcn_readlane(holes_upto, kSelectWaves - 1);
  if (tid == 0) *count = all;
  int32_t* const moves = p.moves + (int64_t)row * p.max_moves * 2;
  for (int base = t0; base < t1; base += kWaveSlots) {
    const int t = base + kFour * l;
    uint32_t key[kFour] = {0, 0, 0, 0};
    if (t < t1) keys_of(t, key);
    uint64_t tie[kFour], any_ties = 0;
#pragma unroll
    for (int j = 0; j < kFour; j++) any_ties |= tie[j] = __ballot(t + j < t1 && key[j] == prefix);
    bool hole[kFour], mover[kFour];
    uint64_t holes_at[kFour], movers_at[kFour];
    int rank = my_ties; // of the lane's next token at T
    if (any_ties) {
#pragma unroll
      for (int j = 0; j < kFour; j++) {
        rank = lanes_before(tie[j], rank);
        my_ties += __popcll(tie[j]);
      }
    }
#pragma unroll
    for (int j = 0; j < kFour; j++) {
      const bool in = t + j < t1, at_t = in && key[j] == prefix;
      const bool stays = key[j] > prefix || (at_t && rank < missing);
      rank += at_t;
      holes_at[j] = __ballot(hole[j] = in && t + j < keep && !stays);
      movers_at[j] = __ballot(mover[j] = in && t + j >= keep && stays);
    }
    int to = my_hole, from = my_mover;
#pragma unroll
    for (int j = 0; j < kFour; j++) {
      to = lanes_before(holes_at[j], to);
      from = lanes_before(movers_at[j], from);
      my_hole += __popcll(holes_at[j]);
      my_mover += __popcll(movers_at[j]);
    }
#pragma unroll
    for (int j = 0; j < kFour; j++) {
      if (hole[j]) moves[2 * (int64_t)to++ + 1] = t + j;
      if (mover[j]) moves[2 * (int64_t)from++] = t + j;
    }
  }
}

// ---------------------------------------------------------------------------
// Moves: a wavefront takes 32 moves of a (layer, request, KV head) at a time.  Its lanes
// look up the pages of all their slots at once, then share the rows' vectors out among
// them, a batch of K and V in flight together.  No slot is both a source and a target,
// so rows move in any order.  Bound by HBM where there are many: 180,000 rows of 256
// bytes of K and V in random pages 47.2 us, 3.9 TB/s read and written (a large copy: 5.1);
// 16 moves to a wavefront 48.1 (rows of 128 and 512 bytes 22.4 and 45.8, with 16 22.9 and
// 46.5), 8 vectors to a batch 49.5.
// ---------------------------------------------------------------------------
constexpr int kMoveThreads = 256, kMoveWaves = kMoveThreads / kWave;
constexpr int kWaveMoves = kWave / 2;

template <typename V>
__global__ __launch_bounds__(kMoveThreads) void move_tokens_kernel(MoveTokensParams p, int row_vecs, int blocks_per_row) {
  constexpr int kBatch = 4;
  const int row = (int)(blockIdx.x / (unsigned)blocks_per_row), piece = (int)(blockIdx.x - (unsigned)row * blocks_per_row);
  const int table = row / p.num_kv_heads, h = row - table * p.num_kv_heads;
  const int l = threadIdx.x % kWave, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int count = min(((const const_i32*)p.num_moves)[row], p.max_moves);
  const int32_t* bt = p.block_tables + (int64_t)table * p.block_table_stride;
  const int32_t* moves = p.moves + (int64_t)row * p.max_moves * 2;
  const int64_t slots = (int64_t)p.block_table_stride * p.page_size;
  V* const kpool = static_cast<V*>(p.key_pool);
  V* const vpool = static_cast<V*>(p.value_pool);
  for (int j0 = (piece * kMoveWaves + wave) * kWaveMoves; j0 < count; j0 += blocks_per_row * kMoveWaves * kWaveMoves) {
    const int n = min(kWaveMoves, count - j0);
    // Lanes 2 j and 2 j + 1: index in the pools of move j's source and target, or -1.
    int64_t index = -1;
    if (l < 2 * n) {
      const int t = moves[2 * (int64_t)j0 + l];
      if (t >= 0 && t < slots) {
        const int pi = (int)(((uint64_t)(uint32_t)t * p.page_magic) >> p.page_magic_shift);
        const int64_t page = bt[pi];
        if (page >= 0 && page < p.num_pages) index = (page * p.num_kv_heads + h) * p.page_size + (t - pi * p.page_size);
      }
    }
    auto index_of = [&](int lane) {
      const uint32_t lo = (uint32_t)__shfl((int)(uint32_t)index, lane), hi = (uint32_t)__shfl((int)(index >> 32), lane);
      return (int64_t)(((uint64_t)hi << 32) | lo);
    };
    const int64_t other = index_of(l ^ 1);
    if (l % 2 == 0 && index >= 0 && other >= 0) {
      if (p.weights) p.weights[other] = p.weights[index];
      if (p.positions) p.positions[other] = p.positions[index];
    }
    const int64_t vecs = (int64_t)n * row_vecs;
    for (int64_t v0 = 0; v0 < vecs; v0 += kWave * kBatch) {
      V k[kBatch], v[kBatch];
      int64_t dst[kBatch];
#pragma unroll
      for (int u = 0; u < kBatch; u++) {
        const int64_t at = v0 + l + kWave * u;
        // (32 rows of 2^31 bytes at most: their vectors are counted in 64 bits only where
        // rows are that long.)
        const int j = at >= vecs ? 0 : vecs <= INT_MAX ? (int)((unsigned)at / (unsigned)row_vecs) : (int)(at / row_vecs);
        const int64_t from = index_of(2 * j), to = index_of(2 * j + 1), c = at - (int64_t)j * row_vecs;
        dst[u] = at < vecs && from >= 0 && to >= 0 ? to * row_vecs + c : -1;
        if (dst[u] >= 0) {
          k[u] = kpool[from * row_vecs + c];
          v[u] = vpool[from * row_vecs + c];
        }
      }
#pragma unroll
      for (int u = 0; u < kBatch; u++)
        if (dst[u] >= 0) {
          kpool[dst[u]] = k[u];
          vpool[dst[u]] = v[u];
        }
    }
  }
}

} // namespace

hipError_t launch_select_tokens(const SelectTokensParams& params, int compute_units, hipStream_t stream) {
  const int64_t eights = ((int64_t)params.num_layers * params.num_seqs + 7) / 8;
  const int64_t blocks = eights * 8 * params.num_kv_heads;
  const dim3 grid((unsigned)blocks);
  const bool vec = params.page_size % kFour == 0 && ((uintptr_t)params.weights | (uintptr_t)params.positions) % 16 == 0;
  auto launch = [&](auto threads, auto held) {
    constexpr int kThreads = decltype(threads)::value, kHeld = decltype(held)::value;
    if (vec)
      hipLaunchKernelGGL((select_tokens_kernel<kThreads, kHeld, true>), grid, dim3(kThreads), 0, stream, params);
    else
      hipLaunchKernelGGL((select_tokens_kernel<kThreads, kHeld, false>), grid, dim3(kThreads), 0, stream, params);
  };
  // More blocks than CUs hold of the large ones at once: small ones, whose passes then
  // overlap.  (128 heads of 1,500 to 8,000 tokens in 8 layers, 1,024 blocks: 30.5 us in
  // small blocks and 32.7 in large ones; 16 heads of 8,000, 128 blocks: 14.6 and 12.7.)
  if (params.max_seq_len <= kFewKeys && blocks > 2 * compute_units)
    launch(std::integral_constant<int, 512>(), std::integral_constant<int, kFewKeys>());
  else if (params.max_seq_len <= kManyKeys)
    launch(std::integral_constant<int, 1024>(), std::integral_constant<int, kManyKeys>());
  else
    launch(std::integral_constant<int, 1024>(), std::integral_constant<int, 0>());
  return hipGetLastError();
}

hipError_t launch_move_tokens(const MoveTokensParams& params, int64_t row_bytes, hipStream_t stream) {
  const int64_t rows = (int64_t)params.num_layers * params.num_seqs * params.num_kv_heads;
  // Blocks for all of a row's moves at once, but no more than some tens of rounds of them.
  constexpr int kBlockMoves = kMoveWaves * kWaveMoves;
  const int64_t pieces = ((int64_t)params.max_moves + kBlockMoves - 1) / kBlockMoves;
  constexpr int kMostBlocks = kMoveStep / kBlockMoves;
  const int blocks_per_row = (int)std::max<int64_t>(1, std::min<int64_t>(pieces, kMostBlocks / rows));
  return with_vector(row_bytes, params.key_pool, params.value_pool, [&](auto v, int row_vecs) {
    hipLaunchKernelGGL(move_tokens_kernel<decltype(v)>, dim3((unsigned)(rows * blocks_per_row)), dim3(kMoveThreads), 0,
                       stream, params, row_vecs, blocks_per_row);
    return hipGetLastError();
  });
}

} // namespace mvr
