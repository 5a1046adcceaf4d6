// Types and dtype traits of the kernels that stream 16-token chunks of the
// cache through one wavefront (paged_attention.hip, draft_attention.hip): how a
// chunk is loaded, multiplied and staged.
#pragma once

#include "paged_attention_kernels.hpp"

namespace mvr {
namespace {

typedef _Float16 half_t;
typedef half_t half8 __attribute__((ext_vector_type(8)));
typedef half_t half4 __attribute__((ext_vector_type(4)));
typedef short short4v __attribute__((ext_vector_type(4)));
typedef float float4v __attribute__((ext_vector_type(4)));
typedef float float2v __attribute__((ext_vector_type(2)));

typedef __attribute__((address_space(3))) short4v lds_short4;
typedef __attribute__((address_space(4))) int32_t const_i32;

__device__ __forceinline__ int lane_id() { return __lane_id(); }

__device__ __forceinline__ float wave_max_across_groups(float v) {
  // Lanes l, l^16, l^32, l^48 hold the same query row.
  v = fmaxf(v, __shfl_xor(v, 16));
  v = fmaxf(v, __shfl_xor(v, 32));
  return v;
}

__device__ __forceinline__ float wave_sum_across_groups(float v) {
  v += __shfl_xor(v, 16);
  v += __shfl_xor(v, 32);
  return v;
}

// ---------------------------------------------------------------------------
// dtype traits: how a 16-token chunk is loaded, multiplied and staged.
// ---------------------------------------------------------------------------

template <int D>
struct F16Traits {
  typedef half_t elem;
  static constexpr int kLoads = D / 32;   // 16-byte K loads (and V loads) per lane per chunk
  static constexpr int kQRegs = D / 32;   // half8 Q operand registers per row block
  typedef half8 kreg_t;
  typedef half8 vreg_t;
  typedef half8 qreg_t;

  // 16-row tiles: 3 wavefronts per SIMD; 32-row tiles: 2 (wider heads: 2, then 1).
  template <int NB>
  static constexpr int min_blocks() { return D <= 128 ? (NB == 1 ? 3 : 2) : D <= 192 ? 2 : 1; }

  // 32-byte pieces of an LDS row: D/16; XOR swizzle spreads 16 rows over
  // banks (within aligned groups of 8 or 4 pieces, so every piece stays in
  // its row; none where D/16 is not a multiple of 4).
  __device__ static __forceinline__ int swz(int t) {
    return D % 128 == 0 ? (t & 7) : D % 64 == 0 ? ((t >> 1) & 3) : 0;
  }

  __device__ static __forceinline__ void load_q(const half_t* row, bool valid, int g, qreg_t (&q)[kQRegs]) {
#pragma unroll
    for (int s = 0; s < kQRegs; s++) {
      q[s] = valid ? *reinterpret_cast<const half8*>(row + 8 * g + 32 * s) : half8{};
    }
  }

  __device__ static __forceinline__ void load_k(const half_t* slab, int l, kreg_t (&k)[kLoads]) {
    const half_t* row = slab + (l & 15) * D + 8 * (l >> 4);
#pragma unroll
    for (int s = 0; s < kLoads; s++) k[s] = *reinterpret_cast<const half8*>(row + 32 * s);
  }

  __device__ static __forceinline__ void load_v(const half_t* slab, int l, vreg_t (&v)[kLoads]) {
#pragma unroll
    for (int u = 0; u < kLoads; u++) {
      const int ci = l + 64 * u; // 16-byte chunk of the 16 x D slab
      v[u] = *reinterpret_cast<const half8*>(slab + 8 * ci);
    }
  }

  // Pages that do not hold whole 16-token chunks: the same loads through a
  // pointer to each token row (K: the lane's row is l & 15; V: load u reads
  // token row v_row(l, u) at column v_col(l, u)).
  __device__ static __forceinline__ void load_k_row(const half_t* row, int l, kreg_t (&k)[kLoads]) {
#pragma unroll
    for (int s = 0; s < kLoads; s++) k[s] = *reinterpret_cast<const half8*>(row + 8 * (l >> 4) + 32 * s);
  }
  __device__ static __forceinline__ int v_row(int l, int u) { return (l + 64 * u) / (D / 8); }
  __device__ static __forceinline__ int v_col(int l, int u) { return 8 * ((l + 64 * u) % (D / 8)); }
  __device__ static __forceinline__ vreg_t load_v_row(const half_t* row, int l, int u) {
    return *reinterpret_cast<const half8*>(row + v_col(l, u));
  }

  __device__ static __forceinline__ void stage_v(half_t* lds, int l, int tok_valid, const vreg_t (&v)[kLoads]) {
#pragma unroll
    for (int u = 0; u < kLoads; u++) {
      const int ci = l + 64 * u;
      const int t = ci / (D / 8), c = ci % (D / 8);
      const int piece = (c >> 1) ^ swz(t);
      // Slots past the sequence end may hold anything (unwritten pages);
      // zero them so 0-weight * garbage cannot produce NaN.
      half8 val = t < tok_valid ? v[u] : half8{};
      *reinterpret_cast<half8*>(lds + t * D + piece * 16 + (c & 1) * 8) = val;
    }
  }

  __device__ static __forceinline__ float4v qk(const kreg_t (&k)[kLoads], const qreg_t (&q)[kQRegs]) {
    float4v acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int s = 0; s < kLoads; s++) acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(k[s], q[s], acc, 0, 0, 0);
    return acc;
  }

  template <int NB>
  __device__ static __forceinline__ void pv(half_t* lds, int l, const float (&p)[NB][4], float4v (&o)[NB][D / 16]) {
    half4 pb[NB];
#pragma unroll
    for (int nb = 0; nb < NB; nb++) pb[nb] = half4{(half_t)p[nb][0], (half_t)p[nb][1], (half_t)p[nb][2], (half_t)p[nb][3]};
    const int g = l >> 4, qd = l & 15;
    const int row = 4 * g + (qd >> 2);
    const int sw = swz(row);
#pragma unroll
    for (int n = 0; n < D / 16; n++) {
      half_t* addr = lds + row * D + ((n ^ sw) * 16) + 4 * (qd & 3);
      short4v raw = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_short4*)(addr));
      half4 vt = __builtin_bit_cast(half4, raw);
#pragma unroll
      for (int nb = 0; nb < NB; nb++) o[nb][n] = __builtin_amdgcn_mfma_f32_16x16x16f16(vt, pb[nb], o[nb][n], 0, 0, 0);
    }
  }

  __device__ static __forceinline__ void store_out(half_t* dst, float4v v) {
    half4 h = {(half_t)v[0], (half_t)v[1], (half_t)v[2], (half_t)v[3]};
    *reinterpret_cast<half4*>(dst) = h;
  }
};

template <int D>
struct F32Traits {
  typedef float elem;
  static constexpr int kLoads = D / 16; // 16-byte loads per lane per chunk
  static constexpr int kQRegs = D / 16;
  typedef float4v kreg_t;
  typedef float4v vreg_t;
  typedef float4v qreg_t;

  template <int NB>
  static constexpr int min_blocks() {
    return D == 128 ? (NB == 1 ? 2 : 1) : D <= 64 ? (NB == 1 ? 3 : 2) : D <= 128 ? 2 : 1;
  }

  // 64-byte pieces (16 floats) of an LDS row; rows 4g+j of the four lane
  // groups land in four different pieces (none where D/16 is not a multiple
  // of 4, so that every piece stays in its row).
  __device__ static __forceinline__ int swz(int t) { return (D / 16) % 4 == 0 ? ((t >> 2) & 3) : 0; }

  __device__ static __forceinline__ void load_q(const float* row, bool valid, int g, qreg_t (&q)[kQRegs]) {
#pragma unroll
    for (int u = 0; u < kQRegs; u++) {
      q[u] = valid ? *reinterpret_cast<const float4v*>(row + 16 * u + 4 * g) : float4v{0.f, 0.f, 0.f, 0.f};
    }
  }

  __device__ static __forceinline__ void load_k(const float* slab, int l, kreg_t (&k)[kLoads]) {
    const float* row = slab + (l & 15) * D + 4 * (l >> 4);
#pragma unroll
    for (int u = 0; u < kLoads; u++) k[u] = *reinterpret_cast<const float4v*>(row + 16 * u);
  }

  __device__ static __forceinline__ void load_v(const float* slab, int l, vreg_t (&v)[kLoads]) {
#pragma unroll
    for (int u = 0; u < kLoads; u++) v[u] = *reinterpret_cast<const float4v*>(slab + 4 * (l + 64 * u));
  }

  __device__ static __forceinline__ void load_k_row(const float* row, int l, kreg_t (&k)[kLoads]) {
#pragma unroll
    for (int u = 0; u < kLoads; u++) k[u] = *reinterpret_cast<const float4v*>(row + 4 * (l >> 4) + 16 * u);
  }
  __device__ static __forceinline__ int v_row(int l, int u) { return (l + 64 * u) / (D / 4); }
  __device__ static __forceinline__ int v_col(int l, int u) { return 4 * ((l + 64 * u) % (D / 4)); }
  __device__ static __forceinline__ vreg_t load_v_row(const float* row, int l, int u) {
    return *reinterpret_cast<const float4v*>(row + v_col(l, u));
  }

  __device__ static __forceinline__ void stage_v(float* lds, int l, int tok_valid, const vreg_t (&v)[kLoads]) {
#pragma unroll
    for (int u = 0; u < kLoads; u++) {
      const int ci = l + 64 * u;
      const int t = ci / (D / 4), c = ci % (D / 4);
      const int piece = (c >> 2) ^ swz(t);
      float4v val = t < tok_valid ? v[u] : float4v{0.f, 0.f, 0.f, 0.f};
      *reinterpret_cast<float4v*>(lds + t * D + piece * 16 + (c & 3) * 4) = val;
    }
  }

  __device__ static __forceinline__ float4v qk(const kreg_t (&k)[kLoads], const qreg_t (&q)[kQRegs]) {
    float4v acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int u = 0; u < kLoads; u++) {
#pragma unroll
      for (int e = 0; e < 4; e++) acc = __builtin_amdgcn_mfma_f32_16x16x4f32(k[u][e], q[u][e], acc, 0, 0, 0);
    }
    return acc;
  }

  template <int NB>
  __device__ static __forceinline__ void pv(float* lds, int l, const float (&p)[NB][4], float4v (&o)[NB][D / 16]) {
    const int g = l >> 4, qd = l & 15;
#pragma unroll
    for (int n = 0; n < D / 16; n++) {
#pragma unroll
      for (int j = 0; j < 4; j++) {
        const int row = 4 * g + j;
        const float vt = lds[row * D + ((n ^ swz(row)) * 16) + qd];
#pragma unroll
        for (int nb = 0; nb < NB; nb++) o[nb][n] = __builtin_amdgcn_mfma_f32_16x16x4f32(vt, p[nb][j], o[nb][n], 0, 0, 0);
      }
    }
  }

  __device__ static __forceinline__ void store_out(float* dst, float4v v) { *reinterpret_cast<float4v*>(dst) = v; }
};

} // namespace
} // namespace mvr
