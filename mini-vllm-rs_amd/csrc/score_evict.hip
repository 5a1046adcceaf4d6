// The cut of a cache to the tokens that got most attention, for gfx950 (MI355X, CDNA4):
// which tokens stay, and the moves of those that stay past the new length.
#include "score_attention.hpp"

#include <limits.h>

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
// protected, else its weight's bits in an order that ascends with the weight (0 for a
// NaN, as for -infinity).  The keep-th largest key T is found digit by digit from the
// top, with a histogram of the digit of the keys that share the digits found before;
// tokens above T stay, and of those at T the lowest slots, as many as are missing.  What
// stays past slot `keep` and what goes below it are as many, and are paired in ascending
// order.
//
// Bound by the block's own chain of steps, not by the bytes: the weights are read once,
// and their keys held in LDS for the passes over them.
// ---------------------------------------------------------------------------
constexpr int kSelectThreads = 1024, kSelectWaves = kSelectThreads / kWave;
constexpr int kDigitBits = 11, kDigits = 3, kBins = 1 << kDigitBits;
// Keys that LDS holds: two blocks to a CU beside the histograms.  Requests that may be
// longer read weights and positions anew in each pass.
constexpr int kHeldKeys = 17408;

__device__ __forceinline__ uint32_t ascending(float w) {
  const uint32_t x = __float_as_uint(w);
  if (w != w || x == 0xff800000u) return 0; // NaN, -infinity
  return w == 0.f ? 0x80000000u : x >> 31 ? ~x : x | 0x80000000u;
}

template <bool HELD>
__global__ __launch_bounds__(kSelectThreads, 8) void select_tokens_kernel(SelectTokensParams p) {
  __shared__ int bins[kBins];
  __shared__ int wave_counts[kSelectWaves][4];
  __shared__ int found[2]; // digit, keys above it
  __shared__ uint32_t keys[HELD ? kHeldKeys : 1];
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
  const int kept = p.kept_lens ? ((const const_i32*)p.kept_lens)[b] : 0;
  int keep = max(0, min(((const const_i32*)p.keep_lens)[b], n));
  if (min(keep, n - keep) > p.max_moves) keep = n; // (its moves might not fit)
  if (table < p.num_seqs && h == 0 && tid == 0 && p.new_seq_lens) p.new_seq_lens[b] = keep;
  const bool cut = keep != n && keep != 0; // (else nothing goes, or nothing stays)

  const int32_t* bt = p.block_tables + (int64_t)table * p.block_table_stride;
  // Index of slot t in the pools, or -1.
  auto index_of = [&](int t) -> int64_t {
    const int pi = (int)(((uint64_t)(uint32_t)t * p.page_magic) >> p.page_magic_shift);
    const int64_t page = bt[pi];
    if (page < 0 || page >= p.num_pages) return -1;
    return (page * p.num_kv_heads + h) * p.page_size + (t - pi * p.page_size);
  };
  auto key_at = [&](int pos, float w) { return pos < p.first || pos >= (int64_t)next - p.recent ? ~0u : ascending(w); };
  // (Of slots in pages outside the pool: the lowest key.)
  auto read_key = [&](int t) -> uint32_t {
    const int64_t at = index_of(t);
    return at < 0 ? 0 : key_at(t >= kept ? next - (n - t) : p.positions[at], p.weights[at]);
  };
  auto key_of = [&](int t) -> uint32_t {
    if constexpr (HELD)
      return keys[t];
    else
      return read_key(t);
  };
  for (int i = tid; i < kBins; i += kSelectThreads) bins[i] = 0;
  // Positions of what was appended since the last cut; the keys.  A thread's page entries,
  // then its weights and positions, are on their way together.
  constexpr int kAhead = 4;
  for (int t0 = HELD && cut ? tid : max(kept, 0) + tid; t0 < n; t0 += kAhead * kSelectThreads) {
    int64_t at[kAhead];
    float w[kAhead];
    int pos[kAhead];
#pragma unroll
    for (int u = 0; u < kAhead; u++) at[u] = index_of(min(t0 + u * kSelectThreads, n - 1));
    if (HELD && cut) {
#pragma unroll
      for (int u = 0; u < kAhead; u++) {
        const int64_t some = max(at[u], (int64_t)0);
        w[u] = p.weights[some];
        pos[u] = p.positions[some];
      }
    }
#pragma unroll
    for (int u = 0; u < kAhead; u++) {
      const int t = t0 + u * kSelectThreads;
      if (t >= n) break;
      const int fresh = next - (n - t);
      if (HELD && cut) keys[t] = at[u] < 0 ? 0 : key_at(t >= kept ? fresh : pos[u], w[u]);
      if (t >= kept && at[u] >= 0) p.positions[at[u]] = fresh;
    }
  }
  int32_t* const count = p.num_moves + row;
  if (!cut) {
    if (tid == 0) *count = 0;
    return;
  }
  __syncthreads();

  // The keep-th largest key.
  uint32_t prefix = 0, known = 0; // digits found, and which bits they are
  int missing = keep;             // of the keys with those digits, the missing-th largest is T
  for (int digit = kDigits - 1; digit >= 0; digit--) {
    const int shift = digit * kDigitBits;
    for (int t0 = wave * kWave; t0 < n; t0 += kSelectThreads) {
      const int t = t0 + l;
      const uint32_t key = t < n ? key_of(t) : 0;
      const bool in = t < n && (key & known) == prefix;
      const int bin = (int)((key >> shift) & (kBins - 1));
      // (Lanes of one bin, as those of equal weights are, add up first: atomics on one
      // address take their lanes in turn.)
      const uint64_t lanes = __ballot(in);
      if (lanes == 0) continue;
      const int some = __builtin_amdgcn_readlane(bin, __builtin_ctzll(lanes));
      if (__ballot(in && bin != some) == 0) {
        if (l == 0) atomicAdd(&bins[some], (int)__popcll(lanes));
      } else if (in) {
        atomicAdd(&bins[bin], 1);
      }
    }
    __syncthreads();
    // Keys above each bin: a scan from the top, two bins per thread.
    const int top = kBins - 1 - 2 * tid;
    const int c0 = bins[top], c1 = bins[top - 1];
    const int incl = wave_inclusive_sum(c0 + c1);
    if (l == kWave - 1) wave_counts[wave][0] = incl;
    bins[top] = bins[top - 1] = 0; // (for the next digit)
    __syncthreads();
    const int before = wave_inclusive_sum(l < kSelectWaves ? wave_counts[l][0] : 0); // lane l: wavefronts 0 .. l's
    const int above = incl - c0 - c1 + (wave ? __builtin_amdgcn_readlane(before, max(wave - 1, 0)) : 0);
    if (above < missing && above + c0 >= missing) {
      found[0] = top;
      found[1] = above;
    } else if (above + c0 < missing && above + c0 + c1 >= missing) {
      found[0] = top - 1;
      found[1] = above + c0;
    }
    __syncthreads();
    prefix |= (uint32_t)found[0] << shift;
    known |= (uint32_t)(kBins - 1) << shift;
    missing -= found[1];
  }
  // Tokens above T stay, and the first `missing` at T.  Each wavefront looks at a run of
  // slots of its own.  What its run holds: tokens at T, those of them below slot `keep`,
  // tokens below T in slots below `keep`, tokens above T in the others.
  const int run = (n + kSelectThreads - 1) / kSelectThreads * kWave;
  const int t0 = min(wave * run, n), t1 = min(t0 + run, n);
  const uint64_t lower = (1ull << l) - 1;
  int ties = 0, low_ties = 0, holes = 0, movers = 0;
  for (int t = t0; t < t1; t += kWave) {
    const bool in = t + l < t1, low = t + l < keep;
    const uint32_t key = in ? key_of(t + l) : 0;
    ties += (int)__popcll(__ballot(in && key == prefix));
    low_ties += (int)__popcll(__ballot(in && key == prefix && low));
    holes += (int)__popcll(__ballot(in && key < prefix && low));
    movers += (int)__popcll(__ballot(in && key > prefix && !low));
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
  const int at = is_run ? wave_counts[l][0] : 0, low = is_run ? wave_counts[l][1] : 0;
  const int ties_before = wave_inclusive_sum(at) - at, stay = max(0, min(missing - ties_before, at));
  const int goes_in = is_run ? wave_counts[l][2] + low - min(low, stay) : 0;
  const int comes_from = is_run ? wave_counts[l][3] + max(0, stay - low) : 0;
  const int holes_upto = wave_inclusive_sum(goes_in), movers_upto = wave_inclusive_sum(comes_from);
  int my_before = __builtin_amdgcn_readlane(ties_before, wave);
  int my_hole = __builtin_amdgcn_readlane(holes_upto - goes_in, wave);
  int my_mover = __builtin_amdgcn_readlane(movers_upto - comes_from, wave);
  const int all = __builtin_amdgcn_readlane(holes_upto, kSelectWaves - 1);
  if (tid == 0) *count = all;
  int32_t* const moves = p.moves + (int64_t)row * p.max_moves * 2;
  for (int t = t0; t < t1; t += kWave) {
    const bool in = t + l < t1;
    const uint32_t key = in ? key_of(t + l) : 0;
    const uint64_t tie = __ballot(in && key == prefix);
    const bool stays = key > prefix || (key == prefix && my_before + (int)__popcll(tie & lower) < missing);
    const bool hole = in && t + l < keep && !stays, mover = in && t + l >= keep && stays;
    const uint64_t hole_lanes = __ballot(hole), mover_lanes = __ballot(mover);
    if (hole) moves[2 * (int64_t)(my_hole + (int)__popcll(hole_lanes & lower)) + 1] = t + l;
    if (mover) moves[2 * (int64_t)(my_mover + (int)__popcll(mover_lanes & lower))] = t + l;
    my_hole += (int)__popcll(hole_lanes);
    my_mover += (int)__popcll(mover_lanes);
    my_before += (int)__popcll(tie);
  }
}

// ---------------------------------------------------------------------------
// Moves: a wavefront takes 32 moves of a (layer, request, KV head) at a time.  Its lanes
// look up the pages of all their slots at once, then share the rows' vectors out among
// them, a batch of K and V in flight together.  No slot is both a source and a target,
// so rows move in any order.  Bound by HBM where there are many.
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

hipError_t launch_select_tokens(const SelectTokensParams& params, hipStream_t stream) {
  const int64_t eights = ((int64_t)params.num_layers * params.num_seqs + 7) / 8;
  const dim3 grid((unsigned)(eights * 8 * params.num_kv_heads)), block(kSelectThreads);
  if (params.max_seq_len <= kHeldKeys)
    hipLaunchKernelGGL(select_tokens_kernel<true>, grid, block, 0, stream, params);
  else
    hipLaunchKernelGGL(select_tokens_kernel<false>, grid, block, 0, stream, params);
  return hipGetLastError();
}

hipError_t launch_move_tokens(const MoveTokensParams& params, int64_t row_bytes, hipStream_t stream) {
  const int64_t rows = (int64_t)params.num_layers * params.num_seqs * params.num_kv_heads;
  // Blocks for all of a row's moves at once, but no more than some tens of rounds of them.
  constexpr int kBlockMoves = kMoveWaves * kWaveMoves;
  const int64_t pieces = ((int64_t)params.max_moves + kBlockMoves - 1) / kBlockMoves;
  const int blocks_per_row = (int)std::max<int64_t>(1, std::min<int64_t>(pieces, 65536 / rows));
  return with_vector(row_bytes, params.key_pool, params.value_pool, [&](auto v, int row_vecs) {
    hipLaunchKernelGGL(move_tokens_kernel<decltype(v)>, dim3((unsigned)(rows * blocks_per_row)), dim3(kMoveThreads), 0,
                       stream, params, row_vecs, blocks_per_row);
    return hipGetLastError();
  });
}

} // namespace mvr
