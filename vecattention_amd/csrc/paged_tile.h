// The matrix-core form of decode attention over a paged cache, as a work-group's
// function: that of paged_attn.hip's kernels, and of the rows' own keys beside the
// prefixes that they share (paged_prefix.hip).
#pragma once
#include <type_traits>

#include "common.h"
#include "lanes.h"
#include "mfma.h"
#include "paged_ops.h"

namespace va {

constexpr int kPagedThreads = 256, kPagedWaves = kPagedThreads / 64;

__device__ inline float2* part_ml(const PagedArgs& a, int64_t slot) {
  return reinterpret_cast<float2*>(a.part) + slot * a.rows;
}
__device__ inline float* part_row(const PagedArgs& a, int64_t slot, int64_t row) {
  return a.part + 4 * int64_t(a.groups) * a.rows + (slot * a.rows + row) * a.D;
}

// Where a work-group's share begins and ends, and the request of its first unit.
struct Place {
  PagedShare share;
  uint32_t number;   // of the share
  uint32_t begin, end;
  uint32_t base;     // first unit of the request
  int32_t request, keys;
};
struct PlaceLds {
  uint32_t sum[kPagedWaves], base;
  int32_t request, keys;
};

// The share of a work-group.  Neighbouring work-groups take shares a quarter of
// all apart: consecutive shares belong to one kv head for long, whose rows lie in
// the same part of every token's and keep to some of the memory channels, and the
// shares that start first got ahead of the others (36 to 44 us at one request of
// 131072 keys).  us in order / in quarters: 32 + 8 heads, 131072 keys 114 / 102;
// 16 + 16 heads, 40000 keys 75.3 / 68.9; 8 requests up to 32768 keys 47.4 / 45.5.
__device__ inline uint32_t share_number(const PagedArgs& a, uint32_t block) {
  const uint32_t quarter = uint32_t(a.groups) / 4;
  return block < 4 * quarter ? block % 4 * quarter + block / 4 : block;
}

// The keys that a row's own pass skips: with kState, those it shares.
template <bool kState>
__device__ inline int32_t skipped(const PagedArgs& a, int64_t n, int64_t capacity) {
  if constexpr (kState) {
    const int32_t shared = shared_keys(a.prefix_lens[n], capacity), len = a.lens[n];
    return len <= 0 ? 0 : shared < len ? shared : len;
  }
  return 0;
}
// The keys of a row's pass (paged_keys).
template <bool kState>
__device__ inline int32_t row_keys(const PagedArgs& a, int64_t n, int64_t capacity) {
  const int32_t keys = paged_keys(a.lens[n], capacity);
  return kState && keys > 0 ? keys - skipped<kState>(a, n, capacity) : keys;
}

// Sums the units of the requests (every work-group does, N lengths from L2) and
// finds the request of the share's first unit.
template <int kUnit, bool kState = false>
__device__ inline Place locate(const PagedArgs& a, PlaceLds& lds, uint32_t block) {
  const int64_t capacity = a.M * a.page;
  if (a.N <= 64) {  // a lane a request, in every wave by itself
    const int lane = threadIdx.x % 64;
    const int32_t keys = lane < a.N ? row_keys<kState>(a, lane, capacity) : 0;
    const uint32_t mine = lane < a.N ? a.per_request * paged_units(keys, kUnit) : 0;
    const uint32_t sum = uint32_t(wave_inclusive_sum(int(mine)));
    const PagedShare share(uint32_t(__builtin_amdgcn_readlane(int(sum), 63)), uint32_t(a.groups));
    const uint32_t number = share_number(a, block), begin = share.begin(number);
    const uint64_t here = __ballot(begin >= sum - mine && begin < sum);
    const int at = here ? __builtin_ctzll(here) : 0;  // none: the share is empty
    return Place{share,
                 number,
                 begin,
                 share.begin(number + 1),
                 uint32_t(__builtin_amdgcn_readlane(int(sum - mine), at)),
                 at,
                 __builtin_amdgcn_readlane(keys, at)};
  }
  const int32_t N = int32_t(a.N), per = (N + kPagedThreads - 1) / kPagedThreads;
  const int32_t lo = int32_t(threadIdx.x) * per;
  uint32_t mine = 0;
  int32_t keys = 0;
  for (int32_t i = lo; i < lo + per && i < N; ++i) {
    keys = row_keys<kState>(a, i, capacity);
    mine += a.per_request * paged_units(keys, kUnit);
  }
  const int lane = threadIdx.x % 64, w = threadIdx.x / 64;
  const uint32_t sum = uint32_t(wave_inclusive_sum(int(mine)));
  if (lane == 63) lds.sum[w] = sum;
  __syncthreads();
  uint32_t at = sum - mine, total = 0;
#pragma unroll
  for (int i = 0; i < kPagedWaves; ++i) {
    if (i < w) at += lds.sum[i];
    total += lds.sum[i];
  }
  const PagedShare share(total, uint32_t(a.groups));
  const uint32_t number = share_number(a, block);
  const uint32_t begin = share.begin(number);
  if (begin >= at && begin < at + mine)
    for (int32_t i = lo; i < lo + per && i < N; ++i) {
      if (per > 1) keys = row_keys<kState>(a, i, capacity);
      const uint32_t n = a.per_request * paged_units(keys, kUnit);
      if (begin < at + n) {
        lds.request = i;
        lds.base = at;
        lds.keys = keys;
        break;
      }
      at += n;
    }
  __syncthreads();
  return Place{share, number, begin, share.begin(number + 1), lds.base, lds.request, lds.keys};
}

// w * x for a weight that is not zero, but may be too small for fp32: what is
// infinite or not a number stays so.
__device__ inline float weighed(float w, float x) {
  return w != 0.f ? w * x : __builtin_fabsf(x) < __builtin_inff() ? 0.f : x;
}

// Merges the waves' states of a segment's rows and writes them: to the output
// (`whole`), or to a partial slot; with kState to the rows' states where the segment
// begins here (`whole`).  sO[wave][row][stride], sm/sl[wave][row]; kV features of a row
// a thread.
template <typename T, int kV, int kThreads = kPagedThreads, int kStates = kPagedWaves,
          bool kState = false>
__device__ inline void finish(const PagedArgs& a, int D, const float* sO, int rstride,
                              int wstride, const float* sm, const float* sl, int mstride, int rows,
                              bool whole, int64_t slot, int64_t request, int64_t head, bool empty,
                              bool bad) {
  typedef float vec __attribute__((ext_vector_type(kV)));
  const int pieces = D / kV;
  for (int i = threadIdx.x; i < rows * pieces; i += kThreads) {
    const int r = i / pieces, f = (i - r * pieces) * kV;
    float lw[kStates], mw[kStates], m = -__builtin_inff();
    vec ow[kStates];
#pragma unroll
    for (int w = 0; w < kStates; ++w) {
      lw[w] = sl[w * mstride + r];
      mw[w] = sm[w * mstride + r];
      ow[w] = *reinterpret_cast<const vec*>(sO + w * wstride + r * rstride + f);
    }
#pragma unroll
    for (int w = 0; w < kStates; ++w)
      if (!(lw[w] == 0.f)) m = __builtin_fmaxf(m, mw[w]);
    float l = 0.f;
    vec o = vec(0.f);
#pragma unroll
    for (int w = 0; w < kStates; ++w) {
      const float c = __builtin_amdgcn_exp2f(mw[w] - m);
      if (lw[w] == 0.f) continue;  // no key seen, or none of any weight
      l += c * lw[w];
      if (c != 0.f) {
        o += c * ow[w];
      } else {
#pragma unroll
        for (int e = 0; e < kV; ++e) o[e] += weighed(c, ow[w][e]);
      }
    }
    if (bad) l = __builtin_nanf("");
    if (kState && whole) {
      const int64_t row = request * a.Hk * a.G + head + r;
      if (f == 0) a.state_ml[row] = make_float2(m, l);
      *reinterpret_cast<vec*>(a.state + row * a.D + f) = o;
    } else if (whole) {
      // No key: 0.  Keys without weight (scores of -infinity alone): 0/0, as the formula has it.
      struct alignas(sizeof(T) * kV) Row { T x[kV]; } y;
#pragma unroll
      for (int e = 0; e < kV; ++e) y.x[e] = Round<T>::store(empty ? 0.f : o[e] / l);
      *reinterpret_cast<Row*>(static_cast<T*>(a.out) + request * a.on + (head + r) * a.oh + f) = y;
    } else {
      if (f == 0) part_ml(a, slot)[r] = make_float2(m, l);
      *reinterpret_cast<vec*>(part_row(a, slot, r) + f) = o;
    }
  }
}

// The matrix-core form: head_dim 64 or 128, 16-byte aligned rows.  A wave takes
// kKeys keys a step and up to 16 query heads of a kv head:
//   S^T = K Q^T     rows: keys, columns: query heads
//   O^T += V^T P^T  rows: features, columns: query heads
// in 16x16 tiles, so that the lane that gets a score (key 4*kg + i of its tile,
// head c; kg = lane / 16, c = lane % 16) holds that weight where the second
// product wants it, and every row of K and V goes from memory to the registers
// of the lane that multiplies it: K's as operand rows, V's with lane c holding
// features [c*D/16, ..) of its keys, which makes row c of product m feature
// c*D/16 + m; the pairing of keys is then a byte permutation in registers.  Nothing
// but the waves' results at a segment's end goes through LDS.
//
// 16-bit types round a weight to 8 (11) bits, which would cost as much accuracy
// as the output's own rounding: it goes in as two parts, high + low.  bf16 has the
// exponents of fp32: to 2^-18 of the weight.  fp16 ends at 2^-24, and beside one key of
// great weight the others' would be lost: its high part is that of 2^7 weights (at
// most 2^15), its low part is held 2^12 times larger still and is summed by itself,
// so that a weight is good to 2^-22 of itself or 2^-44, whatever is more, and a wave's
// greatest weight is 1 or more.  (One sum for both parts would end at 2^-32, and keys
// 24 nats below the greatest would be gone.)
//
// Infinite values would meet weights of 0 and give NaN where they may not: the low
// part of a weight (or one below 0), the weight of a key past the last, whose row
// is the last key's, and weights too small for their type.  A wave whose sums hold
// a NaN repeats its keys with zeros for rows past the last key and for values that
// are not finite, so that all other sums come out as before, bit for bit; those
// values go in by a product of their own, with a weight of 1 for every key that has
// one, however small.
typedef float f32x4_t __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4_t __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2_t __attribute__((ext_vector_type(2)));

template <typename T> struct Mfma16;
template <> struct Mfma16<bf16_t> {
  typedef __bf16 e;
  typedef bf16x8_t vec;
  __device__ static f32x4_t run(vec a, vec b, f32x4_t c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
  }
};
template <> struct Mfma16<f16_t> {
  typedef _Float16 e;
  typedef f16x8_t vec;
  __device__ static f32x4_t run(vec a, vec b, f32x4_t c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
  }
};

// Max and sum over the four lanes that hold a column (lanes c, c + 16, ..).
__device__ inline float column_max(float x) {
  const uint32_t u = float_to_bits(x);
  const auto p = __builtin_amdgcn_permlane16_swap(u, u, false, false);
  return max_halves(__builtin_fmaxf(bits_to_float(p[0]), bits_to_float(p[1])));
}
__device__ inline float column_sum(float x) {
  const uint32_t u = float_to_bits(x);
  const auto p = __builtin_amdgcn_permlane16_swap(u, u, false, false);
  return sum_halves(bits_to_float(p[0]) + bits_to_float(p[1]));
}

// LDS accesses of a wave's lanes before it come before those after it.  The
// hardware keeps a wave's LDS accesses in order; this keeps the compiler from
// moving a lane's load ahead of the store of another lane.
__device__ inline void wave_fence() {
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
}

constexpr int kTileHeads = 16;
template <typename T> constexpr int kStepKeys = sizeof(T) == 2 ? 32 : 16;
template <typename T> constexpr int kTileUnit = kPagedWaves * kStepKeys<T>;  // when split

// Places of a step's keys: page id and first key of the page for each tile of
// 16 keys, which lie in one page when the page size is a multiple of 16.
template <int kTiles> struct Pages {
  int32_t id[kTiles];
  uint32_t first[kTiles];
};

// Two waves a SIMD: 256 registers each, so that the products' results stay in
// vector registers.  In accumulation registers the compiler (ROCm 7.2) left out
// the wait before one of them was read behind a branch, and a quarter of the
// scores were stale.
//
// kForm: the units are dealt to work-groups of four waves, or a work-group takes a
// whole segment, with eight waves or one, and there is nothing to merge afterwards.
// kStream: the values are read past the caches.
enum PagedForm : int { kFormSplit = 4, kFormWhole = 8, kFormShort = 1 };  // and its waves
//
// kState: a row's keys from `skipped` on, and states instead of outputs.
template <typename T, int D, PagedForm kForm> struct TileLds {
  static constexpr int kWaves = kForm, kStates = kWaves < kPagedWaves ? kWaves : kPagedWaves;
  static constexpr int kStride = D + 4, kKeys = kStepKeys<T>;
  PlaceLds place;
  __align__(16) float sO[kStates][kTileHeads][kStride];
  float sm[kStates][kTileHeads], sl[kStates][kTileHeads];
  int sbad[kWaves];
  int2 srow[kWaves][kKeys];        // (page, row) of a step's keys, any page size
};
template <typename T, int D, bool kWholeTiles, PagedForm kForm, bool kStream, bool kState = false>
__device__ __forceinline__ void paged_tile(const PagedArgs& a, TileLds<T, D, kForm>& lds,
                                           uint32_t block) {
  constexpr bool k16 = sizeof(T) == 2, kSplit = kForm == kFormSplit;
  constexpr int kWaves = kForm, kStates = TileLds<T, D, kForm>::kStates;
  constexpr int kKeys = kStepKeys<T>, kTiles = kKeys / 16, kUnit = kWaves * kKeys;
  constexpr int kF = D / 16;                       // features of a lane in a row of V
  constexpr int kKL = k16 ? D / 32 : D / 16;       // 16-byte loads of a lane in a row of K
  constexpr int kVW = kF * int(sizeof(T)) / 4;     // words of a lane in a row of V
  constexpr int kStride = TileLds<T, D, kForm>::kStride;
  constexpr bool kApart = std::is_same_v<T, f16_t>;  // the low parts are summed by themselves
  auto& sO = lds.sO;
  auto& sm = lds.sm;
  auto& sl = lds.sl;
  auto& sbad = lds.sbad;
  auto& srow = lds.srow;
  const int lane = threadIdx.x % 64;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
  const int kg = lane / 16, c = lane % 16;
  const int64_t capacity = a.M * a.page;
  const uint32_t page = uint32_t(a.page);
  Place pl{PagedShare(1, 1), 0, 0, 0, 0, 0, 0};
  if constexpr (kSplit) {
    pl = locate<kUnit, kState>(a, lds.place, block);
  } else {
    pl.request = int32_t(block / uint32_t(a.per_request));
    pl.keys = row_keys<kState>(a, pl.request, capacity);
    pl.begin = (block - pl.request * a.per_request) * paged_units(pl.keys, kUnit);
    pl.end = pl.begin + 1;  // all of the segment's units
  }
  const uint32_t begin = pl.begin, end = pl.end;
  int64_t req = pl.request;
  int32_t keys = pl.keys;
  uint32_t base = pl.base;
  for (uint32_t u = begin; u < end;) {
    const uint32_t units = paged_units(keys, kUnit);
    const uint32_t seg = (u - base) / units, c0 = (u - base) - seg * units;
    const uint32_t count = kSplit && end - u < units - c0 ? end - u : units - c0;
    const int32_t hk = int32_t(seg) / a.tiles, r0 = (int32_t(seg) - hk * a.tiles) * a.rows;
    const int rows = int(a.G - r0 < a.rows ? a.G - r0 : a.rows);
    const int32_t* table = a.table + req * a.table_stride;
    const T* kbase = static_cast<const T*>(a.k) + hk * a.kh;
    const T* vbase = static_cast<const T*>(a.v) + hk * a.vh;

    // The queries: column c, features as K's lanes hold them.
    u32x4_t q[kKL];
    {
      const T* qr = static_cast<const T*>(a.q) + req * a.qn + (hk * a.G + r0 + c) * a.qh;
#pragma unroll
      for (int s = 0; s < kKL; ++s)
        q[s] = c < rows ? *reinterpret_cast<const u32x4_t*>(qr + (s * 4 + kg) * (16 / sizeof(T)))
                        : u32x4_t{0, 0, 0, 0};
    }
    bool bad = keys < 0;
    const uint32_t skip = uint32_t(skipped<kState>(a, req, capacity));
    const uint32_t last = skip + (keys > 0 ? uint32_t(keys) - 1 : 0);
    const uint32_t first = skip + c0 * kUnit + wave * kKeys;
    int steps = 0;
    if (keys > 0 && first <= last) {
      const uint32_t left = (last - first) / kUnit + 1;
      steps = int(left < count ? left : count);
    }

    // Page entries are read a step ahead of the rows they place: `fetch` issues
    // the reads, `place` puts them to use.  Ids that are no pages read page 0.
    Pages<kTiles> pg, ahead;
    int32_t id_ahead = 0;    // any page size: of the lane's key
    uint32_t in_ahead = 0;
    u32x4_t kr[kTiles][kKL];
    uint32_t vr[kTiles * 4][kVW];
    auto fetch = [&](uint32_t key0) {
      if constexpr (kWholeTiles) {
#pragma unroll
        for (int t = 0; t < kTiles; ++t) {
          const uint32_t p = a.by_page.div(key0 + 16 * t < last ? key0 + 16 * t : last);
          ahead.id[t] = table[p];
          ahead.first[t] = p * page;
        }
      } else {
        const uint32_t k0 = key0 + lane % kKeys < last ? key0 + lane % kKeys : last;
        const uint32_t p = a.by_page.div(k0);
        id_ahead = table[p];
        in_ahead = k0 - p * page;
      }
    };
    auto place = [&]() {
      if constexpr (kWholeTiles) {
        pg = ahead;
#pragma unroll
        for (int t = 0; t < kTiles; ++t)
          if (pg.id[t] < 0 || pg.id[t] >= a.num_pages) {
            bad = true;
            pg.id[t] = 0;
          }
      } else {
        const bool page0 = id_ahead < 0 || id_ahead >= a.num_pages;
        bad |= page0;
        wave_fence();  // the step before has been read
        if (lane < kKeys) srow[wave][lane] = make_int2(page0 ? 0 : id_ahead, int(in_ahead));
        wave_fence();
      }
    };
    // Row `r` of tile t of the step at key0: keys past the last read the last one.
    auto row_of = [&](const T* from, int64_t sp, int64_t sn, uint32_t key0, int t, uint32_t r) {
      if constexpr (kWholeTiles) {
        const uint32_t k0 = key0 + 16 * t + r < last ? key0 + 16 * t + r : last;
        return from + pg.id[t] * sp + (k0 - pg.first[t]) * uint32_t(sn);
      } else {
        const int2 at = srow[wave][16 * t + r];
        return from + at.x * sp + uint32_t(at.y) * uint32_t(sn);
      }
    };
    auto load_k = [&](uint32_t key0) {
#pragma unroll
      for (int t = 0; t < kTiles; ++t) {
        const T* row = row_of(kbase, a.kp, a.kn, key0, t, c);
#pragma unroll
        for (int s = 0; s < kKL; ++s)
          kr[t][s] = *reinterpret_cast<const u32x4_t*>(row + (s * 4 + kg) * (16 / sizeof(T)));
      }
    };
    auto load_v = [&](uint32_t key0) {
#pragma unroll
      for (int j = 0; j < kTiles * 4; ++j) {
        const T* row = row_of(vbase, a.vp, a.vn, key0, j / 4, 4 * kg + j % 4) + c * kF;
#pragma unroll
        for (int w = 0; w < kVW; w += kVW < 4 ? kVW : 4) {
          if constexpr (kVW >= 4) {
            const u32x4_t* at = reinterpret_cast<const u32x4_t*>(
                reinterpret_cast<const uint32_t*>(row) + w);
            const u32x4_t x = kStream ? __builtin_nontemporal_load(at) : *at;
            vr[j][w] = x[0], vr[j][w + 1] = x[1], vr[j][w + 2] = x[2], vr[j][w + 3] = x[3];
          } else {
            const u32x2_t* at = reinterpret_cast<const u32x2_t*>(row);
            const u32x2_t x = kStream ? __builtin_nontemporal_load(at) : *at;
            vr[j][0] = x[0], vr[j][1] = x[1];
          }
        }
      }
    };

    f32x4_t acc[kF], low[kApart ? kF : 1];
    float m, l;
    auto walk = [&](auto again) {
      constexpr bool repeat = decltype(again)::value;
      m = -__builtin_inff();
      l = 0.f;
#pragma unroll
      for (int f = 0; f < kF; ++f) {
        acc[f] = f32x4_t{0.f, 0.f, 0.f, 0.f};
        if constexpr (kApart) low[f] = f32x4_t{0.f, 0.f, 0.f, 0.f};
      }
      if (steps > 0) {
        fetch(first);
        place();
        fetch(first + kUnit);
        load_k(first);
        load_v(first);
      }
      for (int i = 0; i < steps; ++i) {
        const uint32_t key0 = first + uint32_t(i) * kUnit;
        f32x4_t s[kTiles];
#pragma unroll
        for (int t = 0; t < kTiles; ++t) {
          s[t] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int x = 0; x < kKL; ++x) {
            if constexpr (k16) {
              typedef typename Mfma16<T>::vec vec;
              s[t] = Mfma16<T>::run(__builtin_bit_cast(vec, kr[t][x]),
                                    __builtin_bit_cast(vec, q[x]), s[t]);
            } else {
#pragma unroll
              for (int e = 0; e < 4; ++e)
                s[t] = __builtin_amdgcn_mfma_f32_16x16x4f32(
                    bits_to_float(kr[t][x][e]), bits_to_float(q[x][e]), s[t], 0, 0, 0);
            }
          }
        }
        if (i + 1 < steps) {
          place();
          fetch(key0 + 2 * kUnit);
          load_k(key0 + kUnit);
        }
        float p[kTiles * 4], top = -__builtin_inff();
#pragma unroll
        for (int j = 0; j < kTiles * 4; ++j) {
          p[j] = s[j / 4][j % 4] * a.scale_log2;
          if (key0 + 16 * (j / 4) + 4 * kg + j % 4 > last) p[j] = -__builtin_inff();
          top = __builtin_fmaxf(top, p[j]);  // a NaN score stays out of m and poisons its weight
        }
        top = column_max(top);
        // m trails the maximum by at most 8: weights stay within 2^8.  The difference is exact
        // where it is near that; m + 8 rounds at scores of 2^27, to m + 16.
        if (__any(top - m > 8.f)) {
          const float mn = __builtin_fmaxf(m, top);
          const float f = __builtin_amdgcn_exp2f(m - (mn == -__builtin_inff() ? 0.f : mn));
          m = mn;
          l *= f;
#pragma unroll
          for (int x = 0; x < kF; ++x) {
            if constexpr (kApart) low[x] *= f;
            if constexpr (!repeat)
              acc[x] *= f;
            else
#pragma unroll
              for (int e = 0; e < 4; ++e) acc[x][e] = weighed(f, acc[x][e]);
          }
        }
        const float ms = m == -__builtin_inff() ? 0.f : m;
        float seen[kTiles * 4];  // 1 for a key that has a weight
#pragma unroll
        for (int j = 0; j < kTiles * 4; ++j) {
          if constexpr (repeat) seen[j] = p[j] != -__builtin_inff() ? 1.f : 0.f;
          p[j] = __builtin_amdgcn_exp2f(p[j] - ms);
          l += p[j];
        }
        if constexpr (repeat) {
#pragma unroll
          for (int j = 0; j < kTiles * 4; ++j)
            if (key0 + 16 * (j / 4) + 4 * kg + j % 4 > last)
#pragma unroll
              for (int w = 0; w < kVW; ++w) vr[j][w] = 0;
        }
        if constexpr (k16) {
          typedef typename Mfma16<T>::vec vec;
          typedef typename Mfma16<T>::e elem;
          vec hi, lo, one;
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            if constexpr (repeat) one[j] = elem(seen[j]);
            if constexpr (kApart) {
              hi[j] = elem(p[j] * 0x1p7f);
              lo[j] = elem(__builtin_fmaf(p[j], 0x1p19f, -0x1p12f * float(hi[j])));
            } else {
              hi[j] = elem(p[j]);
              lo[j] = elem(p[j] - float(hi[j]));
            }
          }
#pragma unroll
          for (int x = 0; x < kF; ++x) {
            // Feature x of the lane's eight keys: halves of words x / 2.
            const uint32_t sel = x % 2 ? 0x07060302u : 0x05040100u;
            u32x4_t av, odd;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              av[j] = __builtin_amdgcn_perm(vr[2 * j + 1][x / 2], vr[2 * j][x / 2], sel);
              if constexpr (repeat) {  // the halves whose exponent has every bit set
                constexpr uint32_t kExp = kApart ? 0x7c00u : 0x7f80u;
                odd[j] = ((av[j] & kExp) == kExp ? av[j] & 0xffffu : 0u) |
                         ((av[j] >> 16 & kExp) == kExp ? av[j] & 0xffff0000u : 0u);
                av[j] ^= odd[j];
              }
            }
            acc[x] = Mfma16<T>::run(__builtin_bit_cast(vec, av), hi, acc[x]);
            f32x4_t& rest = kApart ? low[kApart ? x : 0] : acc[x];
            rest = Mfma16<T>::run(__builtin_bit_cast(vec, av), lo, rest);
            if constexpr (repeat)
              acc[x] = Mfma16<T>::run(__builtin_bit_cast(vec, odd), one, acc[x]);
          }
        } else {
#pragma unroll
          for (int x = 0; x < kF; ++x)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              uint32_t v = vr[j][x], odd = 0;
              if constexpr (repeat) {
                odd = (v & 0x7f800000u) == 0x7f800000u ? v : 0u;
                v ^= odd;
              }
              acc[x] = __builtin_amdgcn_mfma_f32_16x16x4f32(bits_to_float(v), p[j], acc[x], 0, 0,
                                                            0);
              if constexpr (repeat)
                acc[x] = __builtin_amdgcn_mfma_f32_16x16x4f32(bits_to_float(odd), seen[j], acc[x],
                                                              0, 0, 0);
            }
        }
        if (i + 1 < steps) load_v(key0 + kUnit);
      }
      if constexpr (kApart) {
#pragma unroll
        for (int x = 0; x < kF; ++x)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            acc[x][e] = __builtin_fmaf(low[x][e], 0x1p-19f, acc[x][e] * 0x1p-7f);
      }
    };
    walk(std::false_type{});
    bool nan = false;
#pragma unroll
    for (int x = 0; x < kF; ++x)
#pragma unroll
      for (int e = 0; e < 4; ++e) nan |= acc[x][e] != acc[x][e];
    if (__any(nan)) walk(std::true_type{});
    l = column_sum(l);

    if (u > begin) lds_barrier();  // the segment before has been read
    if (__any(bad)) bad = true;
    if (lane == 0) sbad[wave] = bad;
    if constexpr (kForm == kFormWhole) {
      // The upper four waves' states join those of the lower four, lane by lane.
      f32x4_t* upper = reinterpret_cast<f32x4_t*>(&sO[0][0][0]) + (wave % kPagedWaves) * 64 * kF;
      if (wave >= kPagedWaves) {
#pragma unroll
        for (int x = 0; x < kF; ++x) upper[x * 64 + lane] = acc[x];
        if (kg == 0) {
          sm[wave - kPagedWaves][c] = m;
          sl[wave - kPagedWaves][c] = l;
        }
      }
      lds_barrier();
      if (wave < kPagedWaves) {
        const float mu = sm[wave][c], lu = sl[wave][c];
        const float mn = lu == 0.f ? m : l == 0.f ? mu : __builtin_fmaxf(m, mu);
        const float f = l == 0.f ? 0.f : __builtin_amdgcn_exp2f(m - mn);
        const float g = lu == 0.f ? 0.f : __builtin_amdgcn_exp2f(mu - mn);
#pragma unroll
        for (int x = 0; x < kF; ++x) {
          const f32x4_t up = upper[x * 64 + lane];
#pragma unroll
          for (int e = 0; e < 4; ++e)
            acc[x][e] = (l == 0.f ? 0.f : weighed(f, acc[x][e])) +
                        (lu == 0.f ? 0.f : weighed(g, up[e]));
        }
        l = f * l + g * lu;
        m = mn;
      }
      lds_barrier();
    }
    if (wave < kStates) {
#pragma unroll
      for (int e = 0; e < 4; ++e)
#pragma unroll
        for (int x = 0; x < kF; x += 4)
          *reinterpret_cast<f32x4_t*>(&sO[wave][c][(4 * kg + e) * kF + x]) =
              f32x4_t{acc[x][e], acc[x + 1][e], acc[x + 2][e], acc[x + 3][e]};
      if (kg == 0) {
        sm[wave][c] = m;
        sl[wave][c] = l;
      }
    }
    lds_barrier();
    bool any_bad = false;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) any_bad |= sbad[w] != 0;
    finish<T, 4, 64 * kWaves, kStates, kState>(
        a, D, &sO[0][0][0], kStride, kTileHeads * kStride, &sm[0][0], &sl[0][0], kTileHeads, rows,
        kState ? c0 == 0 : count == units, 2 * int64_t(pl.number) + (!kState && u > begin), req,
        hk * a.G + r0, keys == 0, any_bad);
    if (!kSplit) break;
    if (c0 == 0 && threadIdx.x == 0)
      a.split[req * a.per_request + seg] =
          count == units ? make_int2(-1, -1)
                         : make_int2(2 * int(pl.number) + (u > begin),
                                     int(pl.share.owner(u + units - 1)));
    u += count;
    if (u < end && u == base + units * a.per_request) {
      base = u;
      keys = row_keys<kState>(a, ++req, capacity);
    }
  }
}

}  // namespace va
