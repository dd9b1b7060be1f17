// A wave's part of the loop over 64-key tiles in LDS that dense attention (attn_dense.hip) and
// that of shared prefixes (paged_prefix.hip) walk: 32 query rows, S^T = K Q^T and O^T += V^T P^T
// on 32x32x16 matrix instructions.  A tile is 64 rows of D values in chunks of 16 bytes, chunk p
// of row R at p ^ chunk_swizzle<D>(R).
#pragma once
#include "attn_common.h"
#include "mfma.h"

namespace va {

template <typename T, int D> struct DenseTile {
  using M = Mfma<T>;
  using vec = typename M::vec;
  static constexpr int kRowBytes = 2 * D;
  static constexpr int kTileBytes = kTileKeys * kRowBytes;  // one K (or V) tile
  static constexpr int kChunks = D / 8;                     // 16-byte chunks per row
  static constexpr int kRowsPerCopy = 1024 / kRowBytes;     // rows per 1 KB copy
  static constexpr int kCopies = kTileBytes / 1024 / 4;     // per wave of four and tile
  static constexpr int NQK = D / 16;   // QK MFMAs per 32 keys
  static constexpr int NB = D / 32;    // output blocks of 32 features
  static constexpr int NPV = 4 * NB;   // PV MFMAs per tile (16 keys each)

  // LDS read offsets (see attn_mfma.hip): K row l32 (+ 32 for the second half of the tile),
  // chunk 2s + hh = k ^ 32s; V^T rows 8r + 4hh + j (+ 16 per MFMA step), features 32i + ...:
  // v[r] ^ 64i.
  struct Offsets {
    uint32_t k, v[2];
    __device__ explicit Offsets(int lane) {
      const int l32 = lane % 32, hh = lane / 32;
      k = uint32_t(l32 * kRowBytes + 16 * (hh ^ chunk_swizzle<D>(l32)));
      const int j = (lane % 16) / 4, g2 = 2 * ((lane / 16) % 2) + (lane % 4) / 2;
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        const int R = 8 * r + 4 * hh + j;
        v[r] = uint32_t(R * kRowBytes + 16 * (g2 ^ chunk_swizzle<D>(R)) + 8 * (lane % 2));
      }
    }
  };

  // Operand of QK MFMA i.
  __device__ static vec kread(const unsigned char* kb, uint32_t k, int i) {
    return __builtin_bit_cast(vec, *reinterpret_cast<const uint4*>(
                                       kb + (k ^ uint32_t(32 * (i % NQK))) +
                                       i / NQK * 32 * kRowBytes));
  }
  // Of PV MFMA f: 16 keys of step f / NB, features [32 (f % NB), +32).
  __device__ static vec vread(const unsigned char* vb, uint32_t v0, uint32_t v1, int f) {
    const int sub = f / NB, i = f % NB;
    const unsigned char* p0 = vb + (v0 ^ uint32_t(64 * i)) + sub * 16 * kRowBytes;
    const unsigned char* p1 = vb + (v1 ^ uint32_t(64 * i)) + sub * 16 * kRowBytes;
    const s16x4_t lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
        (__attribute__((address_space(3))) s16x4_t*)(p0));
    const s16x4_t hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
        (__attribute__((address_space(3))) s16x4_t*)(p1));
    const s16x4_t both[2] = {lo, hi};
    return __builtin_bit_cast(vec, both);
  }

  // S^T of a tile's two 32-key halves; the copies go out between the MFMAs.  Slot of
  // sc[hf][e]: key 32hf + 8(e/4) + 4hh + e%4 of query row l32.
  template <typename F>
  __device__ static __forceinline__ void scores(const unsigned char* kb, uint32_t k,
                                                const vec (&q)[NQK], f32x16_t (&sc)[2],
                                                F&& copies) {
    constexpr int kAhead = 2;
    asm volatile("" : "+v"(k));  // the offsets are rebuilt, not kept
    vec a[2 * NQK];
#pragma unroll
    for (int i = 0; i < kAhead; ++i) a[i] = kread(kb, k, i);
#pragma unroll
    for (int hf = 0; hf < 2; ++hf)
#pragma unroll
      for (int e = 0; e < 16; ++e) sc[hf][e] = 0.f;
    __builtin_amdgcn_s_setprio(2);
#pragma unroll
    for (int i = 0; i < 2 * NQK; ++i) {
      __builtin_amdgcn_sched_barrier(0);
      if (i + kAhead < 2 * NQK) a[i + kAhead] = kread(kb, k, i + kAhead);
      sc[i / NQK] = M::run(a[i], q[i % NQK], sc[i / NQK]);
      static_for<kCopies>([&](auto c) {
        if (c * 2 * NQK / kCopies == i) copies(c);
      });
    }
    __builtin_amdgcn_sched_barrier(0);
    __builtin_amdgcn_s_setprio(0);
  }

  // A tile's PV MFMAs: multiply(f, V's operand), then the copies that are due, then sum(f).
  template <typename F, typename G, typename S>
  __device__ static __forceinline__ void values(const unsigned char* vb, uint32_t v0, uint32_t v1,
                                                F&& multiply, G&& copies, S&& sum) {
    constexpr int kAhead = 2;
    vec a[NPV];
#pragma unroll
    for (int f = 0; f < kAhead; ++f) a[f] = vread(vb, v0, v1, f);
    __builtin_amdgcn_s_setprio(1);
#pragma unroll
    for (int f = 0; f < NPV; ++f) {
      __builtin_amdgcn_sched_barrier(0);
      if (f + kAhead < NPV) a[f + kAhead] = vread(vb, v0, v1, f + kAhead);
      multiply(f, a[f]);
      static_for<kCopies>([&](auto c) {
        if (c * NPV / kCopies == f) copies(c);
      });
      sum(f);
    }
    __builtin_amdgcn_sched_barrier(0);
    __builtin_amdgcn_s_setprio(0);
  }
};

}  // namespace va
