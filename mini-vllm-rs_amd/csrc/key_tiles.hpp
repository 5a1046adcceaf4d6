// Key tiles in LDS: how the attention kernels of many rows (draft_tiles.hip,
// score_tiles.hip) lay them out and load them straight from the pages.
#pragma once

#include "row_helpers.hpp"

namespace mvr {
namespace {

constexpr int kTileWaves = 4; // wavefronts per block, but where a kernel takes more

typedef float float16v __attribute__((ext_vector_type(16)));
typedef int int4v __attribute__((ext_vector_type(4)));
typedef unsigned int u32x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) void lds_void;

// 16 bytes per lane at `base` + the lane's byte offset straight into LDS at lds
// + 16 * lane; lanes past `bytes` read zeros.  `base` and `lds` are wave-uniform.
// Raw buffer (stride 0), dword 3 = 0x00020000: untyped 32-bit data.
__device__ __forceinline__ void load_to_lds16(const void* base, uint32_t bytes, uint32_t offset, void* lds) {
  const __amdgpu_buffer_rsrc_t rsrc =
      __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(base), (short)0, (int)bytes, 0x00020000);
  __builtin_amdgcn_raw_ptr_buffer_load_lds(rsrc, (lds_void*)lds, 16, offset, 0, 0, 0);
}

// Waits until at most kNewer of this wavefront's tile loads are in flight.  (The
// compiler's own s_waitcnt, so that its count of the loads stays exact; the empty
// asm keeps memory accesses on their side.)
template <int kNewer>
__device__ __forceinline__ void wait_loads() {
  static_assert(kNewer < 64, "vmcnt has 6 bits");
  __builtin_amdgcn_s_waitcnt((kNewer & 0xF) | ((kNewer >> 4) << 14) | (0x7 << 4) | (0xF << 8)); // vmcnt alone
  asm volatile("" ::: "memory");
}

// Waits for this wavefront's LDS accesses (tile loads stay in flight), then meets
// the others.
__device__ __forceinline__ void stage_barrier() {
  asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

// A block's row tile of 32 * RW rows in W / RW groups of wavefronts, which take
// alternating key tiles.
template <int D, typename T, int RW, int W = kTileWaves>
struct Tile {
  static constexpr bool kF32 = sizeof(T) == 4;
  static constexpr int kGroups = W / RW;
  static constexpr int kTileTokens = kF32 || (kGroups > 1 && W == kTileWaves) ? 32 : 64;
  static constexpr int kSub = kTileTokens / 32;             // S^T blocks of 32 tokens
  static constexpr int kStageTokens = kTileTokens * kGroups; // one tile per group
  static constexpr int kChunkElems = 16 / (int)sizeof(T);
  static constexpr int kChunksPerRow = D / kChunkElems; // 16-byte chunks per token row
  static constexpr int kElems = kStageTokens * D;       // of K, or V, per stage
  static constexpr int kLoads = kStageTokens * kChunksPerRow / (W * kWaveSize); // per thread and operand
  static constexpr int kWaveTokens = kStageTokens / W; // consecutive tokens that a wavefront stages
  static_assert(kLoads * W * kWaveSize == kStageTokens * kChunksPerRow, "whole loads");
  // LDS swizzles, so that the lanes of one read fall into different banks: K by
  // 16-byte chunks with the row (inside groups of the row's largest power of
  // two), F16 V by 32-byte pieces (a transposing read takes 4 rows x 2 pieces at
  // a time).
  static constexpr int kSwzGroup = (kChunksPerRow & -kChunksPerRow) < 16 ? (kChunksPerRow & -kChunksPerRow) : 16;
  __device__ static __forceinline__ int kswz(int t) { return t & (kSwzGroup - 1); }
  __device__ static __forceinline__ int vswz(int t) {
    return kF32 ? 0 : D % 128 == 0 ? 2 * (t & 3) : D % 64 == 0 ? (t & 3) : (t & 1);
  }
};

// How a wavefront's loads find their pages: its run of 8 or 16 tokens lies in one
// page (page sizes that are multiples of 16), or every load's whole token rows do
// (multiples of the rows that 64 lanes of 16 bytes cover), or neither.
enum PageRuns { kRuns, kWholeLoads, kAnyPages };

} // namespace
} // namespace mvr
