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
#include "paged_tile.h"

namespace va {

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
  const Place pl = locate<kRowUnit>(a, place, blockIdx.x);
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

template <typename T, int D, bool kWholeTiles, PagedForm kForm, bool kStream>
__global__ __launch_bounds__(64 * kForm, 2) void paged_tile_kernel(PagedArgs a) {
  __shared__ TileLds<T, D, kForm> lds;
  paged_tile<T, D, kWholeTiles, kForm, kStream>(a, lds, blockIdx.x);
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

// States of rows' own keys: always dealt evenly, since the tables' width says nothing
// about how many there are, to one work-group a CU, which the prefixes' work-groups
// join (paged_prefix.hip).
int64_t paged_states_workspace(int dtype, PagedArgs& a) {
  return plan_form(a, dtype == kF32 ? kTileUnit<float> : kTileUnit<bf16_t>, kTileHeads, 256);
}

hipError_t launch_paged_attn(int dtype, PagedArgs a, void* workspace, hipStream_t stream) {
  if (dtype == kBF16) return launch_paged_t<bf16_t>(dtype, a, workspace, stream);
  if (dtype == kF16) return launch_paged_t<f16_t>(dtype, a, workspace, stream);
  return launch_paged_t<float>(dtype, a, workspace, stream);
}

}  // namespace va
