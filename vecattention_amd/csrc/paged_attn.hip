// Decode attention over a paged cache: for each request n and query head h,
//   out[n, h] = sum_j softmax_j(q[n, h] . K[n, j, g] * scale) V[n, j, g],
//   g = h / (Hq / Hk), j < lens[n],
// with an online softmax (running maximum m and sum l, in log2 units).  The
// keys of all requests are cut into units that are dealt evenly to the
// work-groups (PagedShare in paged.h), whatever the lengths are: they are known
// to the GPU only.  A work-group walks its share segment by segment; the rows of
// a segment it holds whole go to the output, the others to its partial slots,
// which a second launch merges in order (no atomics: the same lengths give the
// same bits).
//
// Partial slots: work-group w writes the segment its share begins with to slot
// 2w, and a later one its share ends in to slot 2w + 1.  Slot s holds `rows` pairs
// (m, l), and `rows` unnormalised fp32 rows of D.  The work-group that a segment
// begins in leaves the segment's first slot and last work-group for the merge.
#include "common.h"
#include "lanes.h"
#include "mfma.h"
#include "paged_ops.h"

#include <type_traits>

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
__device__ inline uint32_t share_number(const PagedArgs& a) {
  const uint32_t quarter = uint32_t(a.groups) / 4;
  return blockIdx.x < 4 * quarter ? blockIdx.x % 4 * quarter + blockIdx.x / 4 : blockIdx.x;
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
__device__ inline Place locate(const PagedArgs& a, PlaceLds& lds) {
  const int64_t capacity = a.M * a.page;
  if (a.N <= 64) {  // a lane a request, in every wave by itself
    const int lane = threadIdx.x % 64;
    const int32_t keys = lane < a.N ? row_keys<kState>(a, lane, capacity) : 0;
    const uint32_t mine = lane < a.N ? a.per_request * paged_units(keys, kUnit) : 0;
    const uint32_t sum = uint32_t(wave_inclusive_sum(int(mine)));
    const PagedShare share(uint32_t(__builtin_amdgcn_readlane(int(sum), 63)), uint32_t(a.groups));
    const uint32_t number = share_number(a), begin = share.begin(number);
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
  const uint32_t number = share_number(a);
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

// Any head_dim up to 256, type, stride and alignment: a wave per key, lane l
// holds the features l, l + 64, ..
constexpr int kRowTile = 4;     // query heads of a tile
constexpr int kRowUnit = 128;   // keys of a unit: 32 for each wave
constexpr int kRowMaxD = 256;
template <typename T, int NF>
__global__ __launch_bounds__(kPagedThreads) void paged_row_kernel(PagedArgs a) {
  __shared__ PlaceLds place;
  __shared__ float sO[kPagedWaves][kRowTile][kRowMaxD], sm[kPagedWaves][kRowTile],
      sl[kPagedWaves][kRowTile];
  __shared__ int sbad[kPagedWaves];
  const int lane = threadIdx.x % 64, wave = threadIdx.x / 64;
  const Place pl = locate<kRowUnit>(a, place);
  const uint32_t begin = pl.begin, end = pl.end;
  const int64_t capacity = a.M * a.page;
  int64_t req = pl.request;
  int32_t keys = pl.keys;
  uint32_t base = pl.base;
  for (uint32_t u = begin; u < end;) {
    const uint32_t units = paged_units(keys, kRowUnit);
    const uint32_t seg = (u - base) / units, c0 = (u - base) - seg * units;
    const uint32_t count = end - u < units - c0 ? end - u : units - c0;
    const int32_t hk = int32_t(seg) / a.tiles, r0 = (int32_t(seg) - hk * a.tiles) * a.rows;
    const int rows = int(a.G - r0 < a.rows ? a.G - r0 : a.rows);
    float q[kRowTile][NF], acc[kRowTile][NF], m[kRowTile], l[kRowTile];
#pragma unroll
    for (int r = 0; r < kRowTile; ++r) {
      m[r] = -__builtin_inff();
      l[r] = 0.f;
#pragma unroll
      for (int j = 0; j < NF; ++j) {
        const int f = lane + 64 * j;
        acc[r][j] = 0.f;
        q[r][j] = r < rows && f < a.D
                      ? to_f32(static_cast<const T*>(
                            a.q)[req * a.qn + (hk * a.G + r0 + r) * a.qh + f])
                      : 0.f;
      }
    }
    bool bad = keys < 0;
    for (int64_t c = c0; c < int64_t(c0) + count; ++c) {
      const int64_t k0 = c * kRowUnit + wave * 32;
      const int64_t k1 = k0 + 32 < keys ? k0 + 32 : keys;
      for (int64_t key = k0; key < k1; ++key) {
        const uint32_t p = a.by_page.div(uint32_t(key)), in = uint32_t(key) - p * uint32_t(a.page);
        int64_t id = a.table[req * a.table_stride + p];
        if (id < 0 || id >= a.num_pages) {
          bad = true;
          id = 0;
        }
        const T* kr = static_cast<const T*>(a.k) + id * a.kp + in * a.kn + hk * a.kh;
        const T* vr = static_cast<const T*>(a.v) + id * a.vp + in * a.vn + hk * a.vh;
        float kf[NF], vf[NF];
#pragma unroll
        for (int j = 0; j < NF; ++j) {
          const int f = lane + 64 * j;
          kf[j] = f < a.D ? to_f32(kr[f]) : 0.f;
          vf[j] = f < a.D ? to_f32(vr[f]) : 0.f;
        }
#pragma unroll
        for (int r = 0; r < kRowTile; ++r) {
          if (r >= rows) break;
          float s = 0.f;
#pragma unroll
          for (int j = 0; j < NF; ++j) s += q[r][j] * kf[j];
#pragma unroll
          for (int d = 1; d < 64; d <<= 1) s += __shfl_xor(s, d);
          s *= a.scale_log2;
          const float mnew = __builtin_fmaxf(m[r], s);  // NaN scores poison p, not m
          const float ms = mnew == -__builtin_inff() ? 0.f : mnew;
          const float c1 = __builtin_amdgcn_exp2f(m[r] - ms), p1 = __builtin_amdgcn_exp2f(s - ms);
          l[r] = l[r] * c1 + p1;
          const bool seen = s != -__builtin_inff();  // else a weight of 0 indeed
#pragma unroll
          for (int j = 0; j < NF; ++j)
            acc[r][j] = weighed(c1, acc[r][j]) + (seen ? weighed(p1, vf[j]) : p1 * vf[j]);
          m[r] = mnew;
        }
      }
    }
    if (u > begin) lds_barrier();  // the segment before has been read
#pragma unroll
    for (int r = 0; r < kRowTile; ++r) {
#pragma unroll
      for (int j = 0; j < NF; ++j) sO[wave][r][lane + 64 * j] = acc[r][j];
      if (lane == 0) {
        sm[wave][r] = m[r];
        sl[wave][r] = l[r];
      }
    }
    if (lane == 0) sbad[wave] = bad;
    lds_barrier();
    finish<T, 1>(a, int(a.D), &sO[0][0][0], kRowMaxD, kRowTile * kRowMaxD, &sm[0][0], &sl[0][0],
                 kRowTile, rows, count == units, 2 * int64_t(pl.number) + (u > begin), req,
                 hk * a.G + r0, keys == 0, sbad[0] || sbad[1] || sbad[2] || sbad[3]);
    if (c0 == 0 && threadIdx.x == 0)
      a.split[req * a.per_request + seg] =
          count == units ? make_int2(-1, -1)
                         : make_int2(2 * int(pl.number) + (u > begin),
                                     int(pl.share.owner(u + units - 1)));
    u += count;
    if (u < end && u == base + units * a.per_request) {
      base = u;
      keys = paged_keys(a.lens[++req], capacity);
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
template <typename T, int D, bool kWholeTiles, PagedForm kForm, bool kStream, bool kState = false>
__global__ __launch_bounds__(64 * kForm, 2) void paged_tile_kernel(PagedArgs a) {
  constexpr bool k16 = sizeof(T) == 2, kSplit = kForm == kFormSplit;
  constexpr int kWaves = kForm, kStates = kWaves < kPagedWaves ? kWaves : kPagedWaves;
  constexpr int kKeys = kStepKeys<T>, kTiles = kKeys / 16, kUnit = kWaves * kKeys;
  constexpr int kF = D / 16;                       // features of a lane in a row of V
  constexpr int kKL = k16 ? D / 32 : D / 16;       // 16-byte loads of a lane in a row of K
  constexpr int kVW = kF * int(sizeof(T)) / 4;     // words of a lane in a row of V
  constexpr int kStride = D + 4;
  constexpr bool kApart = std::is_same_v<T, f16_t>;  // the low parts are summed by themselves
  __shared__ PlaceLds place;
  __shared__ __align__(16) float sO[kStates][kTileHeads][kStride];
  __shared__ float sm[kStates][kTileHeads], sl[kStates][kTileHeads];
  __shared__ int sbad[kWaves];
  __shared__ int2 srow[kWaves][kKeys];        // (page, row) of a step's keys, any page size
  const int lane = threadIdx.x % 64;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
  const int kg = lane / 16, c = lane % 16;
  const int64_t capacity = a.M * a.page;
  const uint32_t page = uint32_t(a.page);
  Place pl{PagedShare(1, 1), 0, 0, 0, 0, 0, 0};
  if constexpr (kSplit) {
    pl = locate<kUnit, kState>(a, place);
  } else {
    pl.request = int32_t(blockIdx.x / uint32_t(a.per_request));
    pl.keys = row_keys<kState>(a, pl.request, capacity);
    pl.begin = (blockIdx.x - pl.request * a.per_request) * paged_units(pl.keys, kUnit);
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

// Maximum and sum over the wave, in every lane.  As row_sum's steps: pairs, quads'
// halves, the mirrored quad and half of a DPP row; then across the four rows.
template <int kCtrl> __device__ inline float dpp_of(float x) {
  return bits_to_float(uint32_t(
      __builtin_amdgcn_update_dpp(0, int(float_to_bits(x)), kCtrl, 0xf, 0xf, false)));
}
__device__ inline float wave_max(float x) {
  x = __builtin_fmaxf(x, dpp_of<0xb1>(x));
  x = __builtin_fmaxf(x, dpp_of<0x4e>(x));
  x = __builtin_fmaxf(x, dpp_of<0x141>(x));
  x = __builtin_fmaxf(x, dpp_of<0x140>(x));
  return column_max(x);
}
__device__ inline float wave_sum(float x) {
  x += dpp_of<0xb1>(x);
  x += dpp_of<0x4e>(x);
  x += dpp_of<0x141>(x);
  x += dpp_of<0x140>(x);
  return column_sum(x);
}

// Rows of segments that several work-groups share: one work-group per
// (segment, row).  The partials' weights 2^(m - M) go to LDS; kV features a thread,
// as many partials side by side as that leaves threads for, U of each thread's in
// flight (the first ones while the weights are computed); then their sums, always
// in the same order: across a wave's lanes in registers, then across the waves.  With
// many partials 32 features a work-group keep all loads in flight at once (128 of 128
// features, 28 rows: 6.3 -> 4.6 us).  kF: the features of a work-group, 0 for all of them.
constexpr int kMostGroups = 2048;
template <typename T, int kF, int kV, int kThreads>
__global__ __launch_bounds__(kThreads) void paged_merge_kernel(PagedArgs a) {
  typedef float vec __attribute__((ext_vector_type(kV)));
  constexpr int U = 4, kWaves = kThreads / 64;
  __shared__ float weight[kMostGroups + 1];
  __shared__ vec sacc[kThreads];
  __shared__ float top[kWaves], den[kWaves];
  const int2 split = a.split[blockIdx.x];
  if (split.x < 0) return;  // written whole
  const uint32_t r = blockIdx.y, n = blockIdx.x / a.per_request;
  const uint32_t s = blockIdx.x - n * a.per_request, hk = s / a.tiles;
  const uint32_t head = (s - hk * a.tiles) * a.rows + r;
  if (head >= a.G) return;
  const int w0 = split.x / 2, parts = split.y - w0 + 1;
  const int lanes = (kF ? kF : int(a.D)) / kV, side = kThreads / lanes;
  const int p = threadIdx.x / lanes, c0 = threadIdx.x - p * lanes;
  const int c = c0 + (kF ? int(blockIdx.z) * lanes : 0);
  auto slot = [&](int i) { return int64_t(i == 0 ? split.x : 2 * (w0 + i)); };
  // Reads past the last partial read it again, with no weight.
  vec x[U];
  auto load = [&](int from) {
#pragma unroll
    for (int i = 0; i < U; ++i) {
      const int at = from + p + i * side < parts ? from + p + i * side : parts - 1;
      x[i] = reinterpret_cast<const vec*>(part_row(a, slot(at), r))[c];
    }
  };
  const int me = threadIdx.x;
  float2 mine = me < parts ? part_ml(a, slot(me))[r] : make_float2(0.f, 0.f);
  load(0);
  float m = mine.y == 0.f ? -__builtin_inff() : mine.x;
  for (int i = me + kThreads; i < parts; i += kThreads) {
    const float2 ml = part_ml(a, slot(i))[r];
    if (!(ml.y == 0.f)) m = __builtin_fmaxf(m, ml.x);
  }
  m = wave_max(m);
  if constexpr (kWaves > 1) {
    if (me % 64 == 0) top[me / 64] = m;
    lds_barrier();
#pragma unroll
    for (int w = 0; w < kWaves; ++w) m = __builtin_fmaxf(m, top[w]);
  }
  float l = 0.f;
  for (int i = me; i < parts; i += kThreads) {
    if (i != me) mine = part_ml(a, slot(i))[r];
    const float f = __builtin_amdgcn_exp2f(mine.x - m);
    weight[i] = mine.y == 0.f ? -1.f : f;  // -1: no weight at all
    l += mine.y == 0.f ? 0.f : f * mine.y;
  }
  l = wave_sum(l);
  if (me % 64 == 0) den[me / 64] = l;
  lds_barrier();
  vec acc = vec(0.f);
  for (int from = 0;; from += U * side) {
    vec y[U];
#pragma unroll
    for (int i = 0; i < U; ++i) y[i] = x[i];
    const bool more = from + U * side < parts;
    if (more) load(from + U * side);
#pragma unroll
    for (int i = 0; i < U; ++i) {
      const int at = from + p + i * side;
      const float f = at < parts ? weight[at] : -1.f;
      if (f > 0.f) acc += f * y[i];
      if (f == 0.f)
#pragma unroll
        for (int e = 0; e < kV; ++e) acc[e] += weighed(f, y[i][e]);
    }
    if (!more) break;
  }
  if constexpr (kF) {  // across the wave in registers, then the waves
    constexpr int kLanes = kF / kV;
    static_assert(kLanes == 8 || kLanes == 16 || kLanes == 32, "lanes of a row in a wave");
#pragma unroll
    for (int e = 0; e < kV; ++e) {
      if constexpr (kLanes == 8) acc[e] += dpp_of<0x128>(acc[e]);  // row_ror:8
      acc[e] = kLanes == 32 ? sum_halves(acc[e]) : column_sum(acc[e]);
    }
    if constexpr (kWaves > 1) {
      if (me % 64 < kLanes) sacc[me / 64 * kLanes + c0] = acc;
      lds_barrier();
    }
    if (p != 0) return;
#pragma unroll
    for (int w = 1; w < kWaves; ++w) acc += sacc[w * kLanes + c0];
  } else {
    sacc[me] = acc;
    lds_barrier();
    if (p != 0) return;
#pragma unroll 4
    for (int i = 1; i < side; ++i) acc += sacc[i * lanes + c0];
  }
  l = 0.f;
#pragma unroll
  for (int w = 0; w < kWaves; ++w) l += den[w];
  T* out = static_cast<T*>(a.out) + n * a.on + (hk * a.G + head) * a.oh + c * kV;
#pragma unroll
  for (int i = 0; i < kV; ++i) out[i] = Round<T>::store(acc[i] / l);
}

static int64_t round256(int64_t x) { return (x + 255) / 256 * 256; }

// Whether the matrix-core form takes these rows: whole 16-byte pieces, and
// offsets within a page of 31 bits.
bool paged_tile_form(int dtype, const PagedArgs& a) {
  if (a.D != 64 && a.D != 128) return false;
  const int64_t es = dtype == kF32 ? 4 : 2, piece = 16 / es;
  for (const void* p : {a.q, a.k, a.v})
    if (reinterpret_cast<uintptr_t>(p) % 16) return false;
  for (int64_t s : {a.qn, a.qh, a.kp, a.kn, a.kh, a.vp, a.vn, a.vh})
    if (s < 0 || s % piece) return false;
  if (reinterpret_cast<uintptr_t>(a.out) % (4 * es) || a.on % 4 || a.oh % 4) return false;
  for (int64_t s : {a.kn, a.vn})
    if (s >= (int64_t(1) << 31) / a.page) return false;
  return true;
}

// The work for `unit` keys a unit and `tile` heads a tile; its workspace bytes.
static int64_t plan_form(PagedArgs& a, int64_t unit, int64_t tile, int64_t groups) {
  a.tiles = int32_t((a.G + tile - 1) / tile);
  a.rows = int32_t((a.G + a.tiles - 1) / a.tiles);
  const int64_t longest = (a.M * a.page + unit - 1) / unit;
  if (longest >= int64_t(1) << 31) return -1;  // nor does the product overflow
  const int64_t most = a.N * a.Hk * a.tiles * (longest > 1 ? longest : 1);  // units, at most
  if (most >= (int64_t(1) << 31)) return -1;
  a.groups = int32_t(most < groups ? most : groups);
  a.per_request = int32_t(a.Hk * a.tiles);
  a.by_page = FastDiv(uint32_t(a.page));
  // Pairs and rows of 2 * groups partial slots, and a pair for each segment.
  return round256(2 * int64_t(a.groups) * a.rows * (8 + 4 * a.D)) +
         round256(8 * a.N * a.per_request);
}
static int64_t plan_tiles(int dtype, PagedArgs& a) {
  return plan_form(a, dtype == kF32 ? kTileUnit<float> : kTileUnit<bf16_t>, kTileHeads, 512);
}
static int64_t plan_rows(PagedArgs& a) { return plan_form(a, kRowUnit, kRowTile, kMostGroups); }

int64_t paged_attn_workspace(int dtype, PagedArgs a) {
  // Which form runs depends on the tensors' alignment too: enough for either.
  const int64_t rows = plan_rows(a), tiles = plan_tiles(dtype, a);
  return rows < 0 || tiles < 0 ? -1 : rows > tiles ? rows : tiles;
}

// The form, by the segments and by the most keys that the tables allow a request.
// A work-group a segment saves the merge and its launch, but takes the segment's
// keys alone: eight waves up to 256 KB of keys and values, up to 512 KB where the
// segments fill the GPU; one wave where they more than fill it and have few keys,
// of which eight waves would get none or a step each.  us, split and merged / eight
// waves / one wave, 28 + 4 heads of 128 in bf16:
//   1 request, 512 keys 10.7 / 9.7 / -, 1024 keys 10.7 / 14.4 / -
//   64 requests, 1024 keys 23.2 / 18.3 / -, 2048 keys 29.9 / 32.8 / -
//   96 requests, 32 keys - / 9.8 / 6.6, 256 keys - / 16.3 / 16.5
//   256 requests, 32 keys - / 21.1 / 9.4, 384 keys - / 39.8 / 31.8
//   1000 requests, 384 keys 124 / - / 101.
static PagedForm paged_form(int dtype, const PagedArgs& a) {
  const int64_t segments = a.N * a.per_request, keys = a.M * a.page;
  const int64_t bytes = keys * a.D * (dtype == kF32 ? 8 : 4);
  if ((segments > 256 && keys <= 256 && bytes <= 128 << 10) ||
      (segments >= 1024 && keys <= 384 && bytes <= 256 << 10))
    return kFormShort;
  if (segments < 2048 && bytes <= (segments < 256 ? 256 << 10 : 512 << 10)) return kFormWhole;
  return kFormSplit;
}

template <typename T, int D, PagedForm kForm, bool kStream>
static void launch_tiles(const PagedArgs& a, hipStream_t stream) {
  const dim3 grid{unsigned(kForm == kFormSplit ? a.groups : a.N * a.per_request)};
  const dim3 block{64 * kForm};
  if (a.page % 16 == 0)
    hipLaunchKernelGGL((paged_tile_kernel<T, D, true, kForm, kStream>), grid, block, 0, stream, a);
  else
    hipLaunchKernelGGL((paged_tile_kernel<T, D, false, kForm, kStream>), grid, block, 0, stream,
                       a);
}
// Values that the Infinity Cache could not hold until the next step, if the tables
// are full, are read past it (not keys: their rows are read in pieces of 64 bytes).
// us without / with: 1 request, 131072 keys 60.6 / 57.3; 64 requests 101 / 93.6; 8
// requests 45.2 / 40.5; 19 requests in fp32, 225 MB in turns, 23.7 / 24.9.
template <typename T, int D>
static void launch_form(PagedForm form, const PagedArgs& a, hipStream_t stream) {
  if (form == kFormShort)
    launch_tiles<T, D, kFormShort, false>(a, stream);
  else if (form == kFormWhole)
    launch_tiles<T, D, kFormWhole, false>(a, stream);
  else if (2 * a.N * a.Hk * a.M * a.page * D * int64_t(sizeof(T)) > (256 << 20))
    launch_tiles<T, D, kFormSplit, true>(a, stream);
  else
    launch_tiles<T, D, kFormSplit, false>(a, stream);
}

template <typename T, int kF, int kV, int kThreads>
static void launch_merge(const PagedArgs& a, hipStream_t stream) {
  hipLaunchKernelGGL((paged_merge_kernel<T, kF, kV, kThreads>),
                     dim3(unsigned(a.N * a.per_request), unsigned(a.rows),
                          unsigned(kF ? a.D / kF : 1)),
                     dim3(kThreads), 0, stream, a);
}

template <typename T>
static hipError_t launch_paged_t(int dtype, PagedArgs& a, void* workspace, hipStream_t stream) {
  const bool tiles = paged_tile_form(dtype, a);
  const int64_t need = tiles ? plan_tiles(dtype, a) : plan_rows(a);
  if (need < 0) return hipErrorInvalidValue;
  a.part = static_cast<float*>(workspace);
  a.split = reinterpret_cast<int2*>(static_cast<char*>(workspace) + need -
                                    round256(8 * a.N * a.per_request));
  if (tiles) {
    const PagedForm form = paged_form(dtype, a);
    a.D == 64 ? launch_form<T, 64>(form, a, stream) : launch_form<T, 128>(form, a, stream);
    if (form != kFormSplit) return hipGetLastError();
  } else {
    const dim3 grid{unsigned(a.groups)}, block{kPagedThreads};
    if (a.D <= 64)
      hipLaunchKernelGGL((paged_row_kernel<T, 1>), grid, block, 0, stream, a);
    else if (a.D <= 128)
      hipLaunchKernelGGL((paged_row_kernel<T, 2>), grid, block, 0, stream, a);
    else
      hipLaunchKernelGGL((paged_row_kernel<T, 4>), grid, block, 0, stream, a);
  }
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  // One wave a row where segments have few partials (64 requests of up to 16384 keys
  // 6.3 -> 5.3 us), four waves to 32 features where they may have many.
  const bool few = a.groups <= 8 * a.N * a.per_request;
  if (a.D == 64 && few)
    launch_merge<T, 64, 4, 64>(a, stream);
  else if (a.D == 128 && few)
    launch_merge<T, 128, 4, 64>(a, stream);
  else if (a.D % 32 == 0)
    launch_merge<T, 32, 4, 256>(a, stream);
  else if (a.D % 4 == 0)
    launch_merge<T, 0, 4, 256>(a, stream);
  else
    launch_merge<T, 0, 1, 256>(a, stream);
  return hipGetLastError();
}

// States of the rows' own keys: always dealt evenly, since the tables' width says
// nothing about how many there are.
int64_t paged_states_workspace(int dtype, PagedArgs& a) { return plan_tiles(dtype, a); }

template <typename T, int D>
static void launch_states(const PagedArgs& a, hipStream_t stream) {
  const dim3 grid{unsigned(a.groups)}, block{64 * kFormSplit};
  if (a.page % 16 == 0)
    hipLaunchKernelGGL((paged_tile_kernel<T, D, true, kFormSplit, false, true>), grid, block, 0,
                       stream, a);
  else
    hipLaunchKernelGGL((paged_tile_kernel<T, D, false, kFormSplit, false, true>), grid, block, 0,
                       stream, a);
}

hipError_t launch_paged_states(int dtype, PagedArgs& a, hipStream_t stream) {
  const bool wide = a.D == 128;
  if (dtype == kBF16)
    wide ? launch_states<bf16_t, 128>(a, stream) : launch_states<bf16_t, 64>(a, stream);
  else
    wide ? launch_states<f16_t, 128>(a, stream) : launch_states<f16_t, 64>(a, stream);
  return hipGetLastError();
}

hipError_t launch_paged_attn(int dtype, PagedArgs a, void* workspace, hipStream_t stream) {
  if (dtype == kBF16) return launch_paged_t<bf16_t>(dtype, a, workspace, stream);
  if (dtype == kF16) return launch_paged_t<f16_t>(dtype, a, workspace, stream);
  return launch_paged_t<float>(dtype, a, workspace, stream);
}

}  // namespace va
