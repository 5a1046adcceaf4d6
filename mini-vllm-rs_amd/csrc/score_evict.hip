// The cut of a cache to the tokens that got most attention, for gfx950 (MI355X, CDNA4):
// which tokens stay, and the moves of those that stay past the new length.
#include "score_attention.hpp"

#include <limits.h>

#include "cache_rows.hpp"

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
// A weight is read once per digit, from the cache after the first time; the block's own
// chain of steps is the bound, not the bytes.
// ---------------------------------------------------------------------------
constexpr int kSelectThreads = 1024, kSelectWaves = kSelectThreads / kWave;
constexpr int kDigitBits = 11, kDigits = 3, kBins = 1 << kDigitBits;

__device__ __forceinline__ uint32_t ascending(float w) {
  const uint32_t x = __float_as_uint(w);
  if (w != w || x == 0xff800000u) return 0; // NaN, -infinity
  return w == 0.f ? 0x80000000u : x >> 31 ? ~x : x | 0x80000000u;
}

__global__ __launch_bounds__(kSelectThreads) void select_tokens_kernel(SelectTokensParams p) {
  __shared__ int bins[kBins];
  __shared__ int wave_counts[kSelectWaves][2];
  __shared__ int found[2]; // digit, keys above it
  const int tid = threadIdx.x, l = tid % kWave, wave = __builtin_amdgcn_readfirstlane(tid / kWave);
  const int row = blockIdx.x;
  const int table = row / p.num_kv_heads, h = row - table * p.num_kv_heads, b = table % p.num_seqs;
  const const_i32* lens = (const const_i32*)p.seq_lens;
  const int n = max(0, min(lens[b], p.max_seq_len));
  const int next = p.next_positions ? ((const const_i32*)p.next_positions)[b] : n;
  const int kept = p.kept_lens ? ((const const_i32*)p.kept_lens)[b] : 0;
  int keep = max(0, min(((const const_i32*)p.keep_lens)[b], n));
  if (min(keep, n - keep) > p.max_moves) keep = n; // (its moves might not fit)
  if (table < p.num_seqs && h == 0 && tid == 0 && p.new_seq_lens) p.new_seq_lens[b] = keep;

  const int32_t* bt = p.block_tables + (int64_t)table * p.block_table_stride;
  // Index of slot t in the pools, or -1.
  auto index_of = [&](int t) -> int64_t {
    const int pi = (int)(((uint64_t)(uint32_t)t * p.page_magic) >> p.page_magic_shift);
    const int64_t page = bt[pi];
    if (page < 0 || page >= p.num_pages) return -1;
    return (page * p.num_kv_heads + h) * p.page_size + (t - pi * p.page_size);
  };
  // Positions of what was appended since the last cut.
  for (int t = max(kept, 0) + tid; t < n; t += kSelectThreads) {
    const int64_t at = index_of(t);
    if (at >= 0) p.positions[at] = next - (n - t);
  }
  int32_t* const count = p.num_moves + row;
  if (keep == n || keep == 0) { // nothing goes, or nothing stays
    if (tid == 0) *count = 0;
    return;
  }
  // (Of slots in pages outside the pool: the lowest key.)
  auto key_of = [&](int t) -> uint32_t {
    const int64_t at = index_of(t);
    if (at < 0) return 0;
    const int pos = t >= kept ? next - (n - t) : p.positions[at];
    if (pos < p.first || pos >= (int64_t)next - p.recent) return ~0u;
    return ascending(p.weights[at]);
  };

  // The keep-th largest key.
  uint32_t prefix = 0, known = 0; // digits found, and which bits they are
  int missing = keep;             // of the keys with those digits, the missing-th largest is T
  for (int digit = kDigits - 1; digit >= 0; digit--) {
    const int shift = digit * kDigitBits;
    for (int i = tid; i < kBins; i += kSelectThreads) bins[i] = 0;
    __syncthreads();
    for (int t = tid; t < n; t += kSelectThreads) {
      const uint32_t key = key_of(t);
      if ((key & known) == prefix) atomicAdd(&bins[(key >> shift) & (kBins - 1)], 1);
    }
    __syncthreads();
    // Keys above each bin: a scan from the top, two bins per thread.
    const int top = kBins - 1 - 2 * tid;
    const int c0 = bins[top], c1 = bins[top - 1];
    int incl = c0 + c1;
#pragma unroll
    for (int d = 1; d < kWave; d <<= 1) {
      const int x = __shfl_up(incl, d);
      if (l >= d) incl += x;
    }
    if (l == kWave - 1) wave_counts[wave][0] = incl;
    __syncthreads();
    int above = incl - c0 - c1;
    for (int w = 0; w < wave; w++) above += wave_counts[w][0];
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
    __syncthreads(); // (before bins and found are written again)
  }
  // Tokens above T stay, and the first `missing` at T.  Each wavefront looks at a run of
  // slots of its own; counts of the runs before it come from a first pass.
  const int run = (n + kSelectThreads - 1) / kSelectThreads * kWave;
  const int t0 = min(wave * run, n), t1 = min(t0 + run, n);
  int ties = 0;
  for (int t = t0; t < t1; t += kWave) {
    const bool tie = t + l < t1 && key_of(t + l) == prefix;
    ties += __popcll(__ballot(tie));
  }
  if (l == 0) wave_counts[wave][0] = ties;
  __syncthreads();
  int ties_before = 0;
  for (int w = 0; w < wave; w++) ties_before += wave_counts[w][0];
  __syncthreads();
  const uint64_t lower = (1ull << l) - 1;
  auto stays = [&](int t, int& before) { // slots t + l
    const bool in = t + l < t1;
    const uint32_t key = in ? key_of(t + l) : 0;
    const uint64_t tie = __ballot(in && key == prefix);
    const bool stay = in && (key > prefix || (key == prefix && before + (int)__popcll(tie & lower) < missing));
    before += (int)__popcll(tie);
    return stay;
  };
  int before = ties_before, holes = 0, movers = 0;
  for (int t = t0; t < t1; t += kWave) {
    const bool stay = stays(t, before);
    holes += (int)__popcll(__ballot(t + l < min(keep, t1) && !stay));
    movers += (int)__popcll(__ballot(t + l >= keep && stay));
  }
  if (l == 0) {
    wave_counts[wave][0] = holes;
    wave_counts[wave][1] = movers;
  }
  __syncthreads();
  holes = movers = 0;
  int all = 0;
  for (int w = 0; w < kSelectWaves; w++) {
    if (w == wave) holes = all;
    all += wave_counts[w][0];
  }
  for (int w = 0; w < wave; w++) movers += wave_counts[w][1];
  if (tid == 0) *count = all;
  int32_t* const moves = p.moves + (int64_t)row * p.max_moves * 2;
  before = ties_before;
  for (int t = t0; t < t1; t += kWave) {
    const bool stay = stays(t, before);
    const bool hole = t + l < min(keep, t1) && !stay, mover = t + l >= keep && stay;
    const uint64_t hole_lanes = __ballot(hole), mover_lanes = __ballot(mover);
    if (hole) moves[2 * (int64_t)(holes + (int)__popcll(hole_lanes & lower)) + 1] = t + l;
    if (mover) moves[2 * (int64_t)(movers + (int)__popcll(mover_lanes & lower))] = t + l;
    holes += (int)__popcll(hole_lanes);
    movers += (int)__popcll(mover_lanes);
  }
}

// ---------------------------------------------------------------------------
// Moves: blocks of a (layer, request, KV head), each a stride of its moves.  Bound by
// HBM where there are many; no slot is both a source and a target, so rows move in any
// order.
// ---------------------------------------------------------------------------
constexpr int kMoveThreads = 256;

template <typename V>
__global__ __launch_bounds__(kMoveThreads) void move_tokens_kernel(MoveTokensParams p, int row_vecs, int blocks_per_row) {
  const int row = (int)(blockIdx.x / (unsigned)blocks_per_row), piece = (int)(blockIdx.x - (unsigned)row * blocks_per_row);
  const int table = row / p.num_kv_heads, h = row - table * p.num_kv_heads;
  const int count = min(((const const_i32*)p.num_moves)[row], p.max_moves);
  const int32_t* bt = p.block_tables + (int64_t)table * p.block_table_stride;
  const int2* moves = reinterpret_cast<const int2*>(p.moves) + (int64_t)row * p.max_moves;
  const int64_t slots = (int64_t)p.block_table_stride * p.page_size;
  // Index of a slot in the pools, or -1.
  auto index_of = [&](int t) -> int64_t {
    if (t < 0 || t >= slots) return -1;
    const int64_t page = bt[t / p.page_size];
    if (page < 0 || page >= p.num_pages) return -1;
    return (page * p.num_kv_heads + h) * p.page_size + t % p.page_size;
  };
  const int l = threadIdx.x % kWave, wave = threadIdx.x / kWave;
  V* const kpool = static_cast<V*>(p.key_pool);
  V* const vpool = static_cast<V*>(p.value_pool);
  for (int j = piece * (kMoveThreads / kWave) + wave; j < count; j += blocks_per_row * (kMoveThreads / kWave)) {
    const int2 move = moves[j];
    const int64_t from = index_of(move.x), to = index_of(move.y);
    if (from < 0 || to < 0) continue;
    for (int64_t v = l; v < row_vecs; v += kWave) {
      const V k = kpool[from * row_vecs + v], w = vpool[from * row_vecs + v];
      kpool[to * row_vecs + v] = k;
      vpool[to * row_vecs + v] = w;
    }
    if (l == 0 && p.weights) p.weights[to] = p.weights[from];
    if (l == 1 && p.positions) p.positions[to] = p.positions[from];
  }
}

} // namespace

hipError_t launch_select_tokens(const SelectTokensParams& params, hipStream_t stream) {
  const int64_t rows = (int64_t)params.num_layers * params.num_seqs * params.num_kv_heads;
  hipLaunchKernelGGL(select_tokens_kernel, dim3((unsigned)rows), dim3(kSelectThreads), 0, stream, params);
  return hipGetLastError();
}

hipError_t launch_move_tokens(const MoveTokensParams& params, int64_t row_bytes, hipStream_t stream) {
  const int64_t rows = (int64_t)params.num_layers * params.num_seqs * params.num_kv_heads;
  const int blocks_per_row = (int)std::max<int64_t>(1, std::min<int64_t>((params.max_moves + 3) / 4, 4096 / rows));
  return with_vector(row_bytes, params.key_pool, params.value_pool, [&](auto v, int row_vecs) {
    hipLaunchKernelGGL(move_tokens_kernel<decltype(v)>, dim3((unsigned)(rows * blocks_per_row)), dim3(kMoveThreads), 0,
                       stream, params, row_vecs, blocks_per_row);
    return hipGetLastError();
  });
}

} // namespace mvr
