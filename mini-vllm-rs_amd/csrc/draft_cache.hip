// The cache side of drafted trees for gfx950 (MI355X, CDNA4): norm, rotation and
// append of new rows, compaction of an accepted path, copies of pages.
//
// All three move rows once: they are bound by HBM where a call has many rows,
// and by the chain of dependent table loads (request, lengths, page, row) where
// it has few.
#include "cache_rows.hpp"

#include <math.h>

namespace mvr {
namespace {

typedef _Float16 half_t;
typedef half_t half4 __attribute__((ext_vector_type(4)));
typedef float float4v __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(4))) int32_t const_i32;

constexpr int kThreads = 256;
constexpr int kWave = 64;
constexpr int kItem = 8; // elements (4 rotation pairs) per thread

__device__ __forceinline__ float4v load4(const float* p) { return *reinterpret_cast<const float4v*>(p); }
__device__ __forceinline__ float4v load4(const half_t* p) {
  return __builtin_convertvector(*reinterpret_cast<const half4*>(p), float4v);
}
__device__ __forceinline__ void store4(float* p, float4v v) { *reinterpret_cast<float4v*>(p) = v; }
__device__ __forceinline__ void store4(half_t* p, float4v v) {
  *reinterpret_cast<half4*>(p) = __builtin_convertvector(v, half4);
}

// The request that holds packed token n and its bounds: the largest b with cu[b]
// <= n (empty requests before it share its start); b = num_seqs behind the last
// one.  A search of the ascending table with one entry per lane and round: one
// round up to 63 requests, whose bounds are then in registers.
struct TokenRequest {
  int b, start, end;
};

__device__ __forceinline__ TokenRequest request_of(const int32_t* cu, int num_seqs, int n) {
  const int l = __lane_id();
  int lo = 0, len = num_seqs + 1; // entries [lo, lo + len) hold the border; those before are <= n
  while (len > kWave) {
    const int step = (len + kWave - 1) / kWave, end = lo + len, at = lo + l * step;
    const int below = __popcll(__ballot(at < end && cu[min(at, end - 1)] <= n)); // probes that are <= n
    if (below == 0) return {-1, 0, 0}; // (only a table that does not start at 0)
    lo += (below - 1) * step;
    len = min(step, end - lo);
  }
  const int entry = cu[lo + min(l, len - 1)];
  const int below = __builtin_amdgcn_readfirstlane(__popcll(__ballot(l < len && entry <= n)));
  const int b = lo + below - 1;
  if (b < 0 || b >= num_seqs) return {b, 0, 0};
  const int start = __builtin_amdgcn_readlane(entry, max(below - 1, 0));
  const int end = below < len ? __builtin_amdgcn_readlane(entry, below) : ((const const_i32*)cu)[b + 1];
  return {b, below > 0 ? start : ((const const_i32*)cu)[b], end};
}

// Norm, rotation and append.  A group of 2^k >= D/8 lanes per row, 8 elements (the
// 4 pairs they rotate as) per lane: the row's mean square is a butterfly over its
// lanes, and nothing is read twice.  A wavefront holds 64 / 2^k rows of one token
// (query heads, then KV heads for K, then for V) and looks the token up by itself,
// while its rows are on their way.
//
// Bound by that chain of dependent loads (request, length, page, store): 1,024
// tokens of 36 rows take 8.3 us in F16 at D=128, where HBM needs 3.9 and a launch
// that does next to nothing 3.5.  Two row groups per wavefront: 8.2, and 1 us more
// for 64 tokens.
template <typename T, int ROPE>
__global__ __launch_bounds__(kThreads) void norm_rope_append_kernel(NormRopeAppendParams p, int lanes_log2,
                                                                    int token_waves) {
  const int64_t unit = (int64_t)blockIdx.x * (kThreads / kWave) + __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int n = (int)(unit / token_waves);
  if (n >= p.total_q) return;
  const int D = p.head_dim, lanes = 1 << lanes_log2, l = threadIdx.x % kWave;
  const int row = ((int)(unit % token_waves) << (6 - lanes_log2)) + (l >> lanes_log2);
  const int j = l & (lanes - 1);
  const int rows = p.num_q_heads + 2 * p.num_kv_heads;
  const bool active = row < rows && j < D / kItem;
  const int kind = row < p.num_q_heads ? 0 : row < p.num_q_heads + p.num_kv_heads ? 1 : 2; // Q, K, V
  const int h = kind == 0 ? row : kind == 1 ? row - p.num_q_heads : row - p.num_q_heads - p.num_kv_heads;
  // The lane's pairs are (lo[e], hi[e]) (Neox), or the neighbours in lo, hi.
  const int lo_off = kind == 2 || ROPE == 1 ? kItem * j : 4 * j;
  const int hi_off = kind == 2 || ROPE == 1 ? kItem * j + 4 : D / 2 + 4 * j;
  float4v lo = {0.f, 0.f, 0.f, 0.f}, hi = lo, wlo = {1.f, 1.f, 1.f, 1.f}, whi = wlo;
  const T* weight = static_cast<const T*>(kind == 0 ? p.q_weight : kind == 1 ? p.k_weight : nullptr);
  if (active) {
    const T* src = kind == 0 ? static_cast<const T*>(p.q) + h * p.q_stride_head + n * p.q_stride_token
                 : kind == 1 ? static_cast<const T*>(p.k) + h * p.k_stride_head + n * p.k_stride_token
                             : static_cast<const T*>(p.v) + h * p.v_stride_head + n * p.v_stride_token;
    lo = load4(src + lo_off);
    hi = load4(src + hi_off);
    if (weight) {
      wlo = load4(weight + lo_off);
      whi = load4(weight + hi_off);
    }
  }

  // The rotation's factors go out as soon as the position is known: with positions
  // now, without them beside the page's look-up.
  float4v c = {0.f, 0.f, 0.f, 0.f}, s = c;
  auto load_factors = [&](int pos) {
    if (!active || kind == 2) return;
    const int64_t at = (int64_t)min(max(pos, 0), p.rope_len - 1) * (D / 2) + 4 * j;
    c = load4(static_cast<const T*>(p.cos_table) + at);
    s = load4(static_cast<const T*>(p.sin_table) + at);
  };
  int pos = 0;
  if (p.positions) {
    pos = ((const const_i32*)p.positions)[n];
    load_factors(pos);
  }
  TokenRequest r = {0, 0, p.total_q};
  if (p.cu_q_lens) r = request_of(p.cu_q_lens, p.num_seqs, n);
  if (r.b < 0 || r.b >= p.num_seqs) return; // behind the last request (a padded batch)
  const int seq_len = p.seq_lens ? ((const const_i32*)p.seq_lens)[r.b] : p.max_seq_len;
  const int slot = seq_len - (r.end - r.start) + (n - r.start);
  if (!p.positions) {
    pos = slot;
    load_factors(pos);
  }
  // Only tables that break the contract hold such values: nothing is written.
  if (slot < 0 || slot >= p.max_seq_len || pos < 0 || pos >= p.rope_len) return;
  const int64_t page = ((const const_i32*)p.block_tables)[(int64_t)r.b * p.block_table_stride + slot / p.page_size];
  if (page < 0 || page >= p.num_pages) return;

  if (weight) {
    float ss = 0.f;
#pragma unroll
    for (int e = 0; e < 4; e++) ss = fmaf(lo[e], lo[e], fmaf(hi[e], hi[e], ss));
    for (int off = lanes >> 1; off >= 1; off >>= 1) ss += __shfl_xor(ss, off);
    const float inv = 1.f / sqrtf(ss / (float)D + p.eps);
    lo = lo * inv * wlo;
    hi = hi * inv * whi;
  }
  if (!active) return;
  const int64_t at = ((page * p.num_kv_heads + h) * p.page_size + slot % p.page_size) * D;
  T* dst = kind == 0 ? static_cast<T*>(p.q_out) + h * p.q_out_stride_head + n * p.q_out_stride_token
         : kind == 1 ? static_cast<T*>(p.key_pool) + at
                     : static_cast<T*>(p.value_pool) + at;
  if (kind != 2) {
    float4v ylo, yhi;
    if (ROPE == 0) {
      ylo = lo * c - hi * s;
      yhi = lo * s + hi * c;
    } else {
#pragma unroll
      for (int e = 0; e < 2; e++) {
        ylo[2 * e] = lo[2 * e] * c[e] - lo[2 * e + 1] * s[e];
        ylo[2 * e + 1] = lo[2 * e] * s[e] + lo[2 * e + 1] * c[e];
        yhi[2 * e] = hi[2 * e] * c[e + 2] - hi[2 * e + 1] * s[e + 2];
        yhi[2 * e + 1] = hi[2 * e] * s[e + 2] + hi[2 * e + 1] * c[e + 2];
      }
    }
    lo = ylo;
    hi = yhi;
  }
  store4(dst + lo_off, lo);
  store4(dst + hi_off, hi);
}

template <typename T>
hipError_t launch_append(const NormRopeAppendParams& p, int rope_type, hipStream_t stream) {
  const int lanes_log2 = append_row_lanes_log2(p.head_dim);
  const int token_waves = append_token_waves(p.num_q_heads + 2 * p.num_kv_heads, p.head_dim);
  const int64_t units = (int64_t)p.total_q * token_waves;
  const dim3 grid((unsigned)((units + kThreads / kWave - 1) / (kThreads / kWave)));
  if (rope_type == 0)
    hipLaunchKernelGGL((norm_rope_append_kernel<T, 0>), grid, dim3(kThreads), 0, stream, p, lanes_log2, token_waves);
  else
    hipLaunchKernelGGL((norm_rope_append_kernel<T, 1>), grid, dim3(kThreads), 0, stream, p, lanes_log2, token_waves);
  return hipGetLastError();
}

// Compaction.  A wavefront per (layer, request, KV head) moves the rows of that
// head's path in both pools.  64 path entries at a time, one per lane, look up
// their rows; then the rows move in batches that fit the registers, all of a batch
// read before any of it is written.  Indices ascend, so a row's source lies at or
// behind its destination, and behind every destination of the batches before:
// whatever is written, its old content has been read.
//
// Rows of 256 bytes in random pages: 32 requests of 20..64 drafts in 32 layers (78
// MB) take 21.7 us, 3.6 TB/s where a large copy reaches 4.9; all wavefronts are
// resident at once, so the chain of lengths, path, pages and rows shows once.
constexpr int kBatch = 4; // vectors per lane, pool and batch

__device__ __forceinline__ int64_t shfl64(int64_t v, int src) {
  const int lo = __shfl((int)v, src), hi = __shfl((int)(v >> 32), src);
  return ((int64_t)hi << 32) | (uint32_t)lo;
}

template <typename V>
__global__ __launch_bounds__(kThreads) void compact_drafts_kernel(CompactDraftsParams p, int row_vecs, int64_t units) {
  const int64_t unit = (int64_t)blockIdx.x * (kThreads / kWave) + __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  if (unit >= units) return;
  const int l = threadIdx.x % kWave;
  const int h = (int)(unit % p.num_kv_heads);
  const int64_t table = unit / p.num_kv_heads; // layer * num_seqs + request
  const int b = (int)(table % p.num_seqs);
  // The path's first indices are on their way while the lengths are.
  const int32_t* accepted = p.accepted + (int64_t)b * p.max_accepted;
  int next = accepted[min(l, p.max_accepted - 1)], carry = -1;
  const const_i32* cu = (const const_i32*)p.cu_q_lens + b;
  const int seq_len = ((const const_i32*)p.seq_lens)[b], q_start = cu[0], q_end = cu[1];
  const int accepted_len = ((const const_i32*)p.accepted_lens)[b];
  const int q_len = q_end - q_start, first = seq_len - q_len;
  const int count = max(0, min(accepted_len, min(q_len, p.max_accepted)));
  if (table < p.num_seqs && h == 0 && l == 0 && p.new_seq_lens) p.new_seq_lens[b] = first + count;
  if (first < 0 || q_len <= 0 || seq_len > p.max_seq_len) return; // (a broken table)
  V* const kpool = static_cast<V*>(p.key_pool);
  V* const vpool = static_cast<V*>(p.value_pool);
  const int32_t* bt = p.block_tables + table * p.block_table_stride;
  // First vector of the row at cache slot t, or -1.
  auto row_at = [&](int t) -> int64_t {
    const int64_t page = bt[t / p.page_size];
    if (page < 0 || page >= p.num_pages) return -1;
    return ((page * p.num_kv_heads + h) * p.page_size + t % p.page_size) * (int64_t)row_vecs;
  };
  const int batch_rows = max(1, kWave * kBatch / row_vecs);
  for (int j0 = 0; j0 < count; j0 += kWave) {
    const int j = j0 + l;
    const int s = j < count ? next : -1, up = __shfl_up(s, 1), before = l > 0 ? up : carry;
    carry = __builtin_amdgcn_readlane(s, kWave - 1);
    if (j0 + kWave < count) next = accepted[min(j + kWave, count - 1)];
    int64_t from = -1, to = -1;
    if (s > j && s < q_len && s > before) { // (s == j is in place)
      from = row_at(first + s);
      to = row_at(first + j);
    }
    if (from < 0 || to < 0) from = to = -1;
    const int n = min(kWave, count - j0);
    for (int r0 = 0; r0 < n; r0 += batch_rows) {
      const int64_t vecs = (int64_t)min(batch_rows, n - r0) * row_vecs;
      // (One pass, but for rows of more vectors than a batch holds: two different
      // rows, copied piece by piece.)
      for (int64_t v0 = 0; v0 < vecs; v0 += kWave * kBatch) {
        V k[kBatch], v[kBatch];
        int64_t dst[kBatch];
#pragma unroll
        for (int u = 0; u < kBatch; u++) {
          const int64_t at = v0 + l + kWave * u;
          const bool in = at < vecs;
          const int rr = in ? (batch_rows == 1 ? 0 : (int)((unsigned)at / (unsigned)row_vecs)) : 0;
          const int64_t src = shfl64(from, r0 + rr), row = shfl64(to, r0 + rr), c = at - (int64_t)rr * row_vecs;
          dst[u] = in && row >= 0 ? row + c : -1;
          if (dst[u] >= 0) {
            k[u] = kpool[src + c];
            v[u] = vpool[src + c];
          }
        }
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); // the batch is in registers
#pragma unroll
        for (int u = 0; u < kBatch; u++)
          if (dst[u] >= 0) {
            kpool[dst[u]] = k[u];
            vpool[dst[u]] = v[u];
          }
      }
    }
  }
}

// Copies of pages.  A block per piece of kCopyVecs * 256 vectors of one page's
// leading tokens, K and V in turn; all of a thread's loads before its stores.
// Bound by HBM: 3,500 pages of 32 KiB in 50.6 us, 4.5 TB/s.
constexpr int kCopyVecs = kCopyPieceVecs / kThreads;

template <typename V>
__global__ __launch_bounds__(kThreads) void copy_pages_kernel(CopyPagesParams p, int row_vecs, int pieces) {
  const int64_t block = blockIdx.x;
  const int piece = (int)(block % pieces);
  const int64_t i = block / pieces / 2;
  V* pool = static_cast<V*>(block / pieces % 2 ? p.value_pool : p.key_pool);
  const int64_t src = ((const const_i32*)p.src_pages)[i], dst = ((const const_i32*)p.dst_pages)[i];
  const int tokens = p.tokens ? min(max(((const const_i32*)p.tokens)[i], 0), p.page_size) : p.page_size;
  if (src < 0 || src >= p.num_pages || dst < 0 || dst >= p.num_pages) return;
  const unsigned per_head = (unsigned)tokens * row_vecs, head_stride = (unsigned)p.page_size * row_vecs;
  const unsigned vecs = per_head * p.num_kv_heads;
  const unsigned v0 = (unsigned)piece * kCopyVecs * kThreads + threadIdx.x;
  const V* from = pool + src * ((int64_t)head_stride * p.num_kv_heads);
  V* to = pool + dst * ((int64_t)head_stride * p.num_kv_heads);
  V held[kCopyVecs];
  unsigned at[kCopyVecs];
#pragma unroll
  for (int u = 0; u < kCopyVecs; u++) {
    const unsigned v = v0 + u * kThreads;
    if (v < vecs) {
      at[u] = v / per_head * head_stride + v % per_head;
      held[u] = from[at[u]];
    }
  }
#pragma unroll
  for (int u = 0; u < kCopyVecs; u++)
    if (v0 + u * kThreads < vecs) to[at[u]] = held[u];
}

} // namespace

hipError_t launch_norm_rope_append(const NormRopeAppendParams& params, int dtype, int rope_type, hipStream_t stream) {
  return dtype == 1 ? launch_append<half_t>(params, rope_type, stream) : launch_append<float>(params, rope_type, stream);
}

hipError_t launch_compact_drafts(const CompactDraftsParams& params, int64_t row_bytes, hipStream_t stream) {
  const int64_t units = (int64_t)params.num_layers * params.num_seqs * params.num_kv_heads;
  const unsigned blocks = (unsigned)((units + kThreads / kWave - 1) / (kThreads / kWave));
  return with_vector(row_bytes, params.key_pool, params.value_pool, [&](auto v, int row_vecs) {
    hipLaunchKernelGGL(compact_drafts_kernel<decltype(v)>, dim3(blocks), dim3(kThreads), 0, stream, params, row_vecs, units);
    return hipGetLastError();
  });
}

hipError_t launch_copy_pages(const CopyPagesParams& params, int64_t row_bytes, hipStream_t stream) {
  return with_vector(row_bytes, params.key_pool, params.value_pool, [&](auto v, int row_vecs) {
    const int64_t pieces =
        copy_pages_pieces((int64_t)params.num_kv_heads * params.page_size, row_bytes, params.key_pool, params.value_pool);
    hipLaunchKernelGGL(copy_pages_kernel<decltype(v)>, dim3((unsigned)(2 * pieces * params.num_copies)), dim3(kThreads),
                       0, stream, params, row_vecs, (int)pieces);
    return hipGetLastError();
  });
}

} // namespace mvr
