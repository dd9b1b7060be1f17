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
// Partial slots: work-group w writes the segment its share begins with (begun
// before) to slot 2w, and a later one its share ends in to slot 2w + 1.  Slot s
// holds `rows` pairs (m, l), and `rows` unnormalised fp32 rows of D.
#include "common.h"
#include "lanes.h"
#include "paged_ops.h"

namespace va {

constexpr int kPagedThreads = 256, kPagedWaves = kPagedThreads / 64;

__device__ inline float2* part_ml(const PagedArgs& a, int64_t slot) {
  return reinterpret_cast<float2*>(a.part) + slot * a.rows;
}
__device__ inline float* part_row(const PagedArgs& a, int64_t slot, int64_t row) {
  return a.part + (4 * a.groups * a.rows + 3) / 4 * 4 + (slot * a.rows + row) * a.D;
}

// Where a work-group's share begins.
struct Place {
  int64_t total, request, start;  // units of all requests; the first request and its first unit
};

// Sums the units of the requests (every work-group does, N lengths from L2) and
// finds the request of the share's first unit.  The first work-group leaves
// the sums for the merge.
template <int kUnit>
__device__ inline Place locate(const PagedArgs& a, int64_t (*lds)[2]) {
  const int64_t capacity = a.M * a.page, per_segment = a.Hk * a.tiles;
  const int64_t per = (a.N + kPagedThreads - 1) / kPagedThreads;
  const int64_t lo = threadIdx.x * per < a.N ? threadIdx.x * per : a.N;
  const int64_t hi = lo + per < a.N ? lo + per : a.N;
  int64_t mine = 0;
  for (int64_t i = lo; i < hi; ++i)
    mine += per_segment * paged_units(paged_keys(a.lens[i], capacity), kUnit);
  const int lane = threadIdx.x % 64, w = threadIdx.x / 64;
  int64_t sum = mine;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const int64_t u = __shfl_up(sum, d);
    if (lane >= d) sum += u;
  }
  if (lane == 63) lds[w][0] = sum;
  __syncthreads();
  int64_t before = 0, total = 0;
#pragma unroll
  for (int i = 0; i < kPagedWaves; ++i) {
    if (i < w) before += lds[i][0];
    total += lds[i][0];
  }
  int64_t at = before + sum - mine;
  const int64_t begin = PagedShare(total, a.groups).begin(blockIdx.x);
  const bool first = blockIdx.x == 0;
  __syncthreads();
  if (first || (begin >= at && begin < at + mine))
    for (int64_t i = lo; i < hi; ++i) {
      const int64_t n = per_segment * paged_units(paged_keys(a.lens[i], capacity), kUnit);
      if (first) a.start[i] = at;
      if (begin >= at && begin < at + n) {
        lds[0][0] = i;
        lds[0][1] = at;
      }
      at += n;
    }
  if (first && threadIdx.x == 0) a.start[a.N] = total;
  __syncthreads();
  return Place{total, lds[0][0], lds[0][1]};
}

// Merges the waves' states of a segment's rows and writes them: to the output
// (`whole`), or to a partial slot.  sO[wave][row][stride], sm/sl[wave][row].
template <typename T>
__device__ inline void finish(const PagedArgs& a, const float* sO, int rstride, int wstride,
                              const float* sm, const float* sl, int mstride, int rows, bool whole,
                              int64_t slot, int64_t request, int64_t head, bool empty, bool bad) {
  for (int i = threadIdx.x; i < rows * int(a.D); i += kPagedThreads) {
    const int r = i / int(a.D), f = i % int(a.D);
    float m = -__builtin_inff();
#pragma unroll
    for (int w = 0; w < kPagedWaves; ++w)
      if (!(sl[w * mstride + r] == 0.f)) m = __builtin_fmaxf(m, sm[w * mstride + r]);
    float l = 0.f, o = 0.f;
#pragma unroll
    for (int w = 0; w < kPagedWaves; ++w) {
      const float lw = sl[w * mstride + r];
      if (lw == 0.f) continue;  // no key seen, or none of any weight
      const float c = __builtin_amdgcn_exp2f(sm[w * mstride + r] - m);
      l += c * lw;
      o += c * sO[w * wstride + r * rstride + f];
    }
    if (bad) l = __builtin_nanf("");
    if (whole) {
      // No key: 0.  Keys without weight (scores of -infinity alone): 0/0, as the formula has it.
      T* out = static_cast<T*>(a.out) + request * a.on + (head + r) * a.oh;
      out[f] = Round<T>::store(empty ? 0.f : o / l);
    } else {
      if (f == 0) part_ml(a, slot)[r] = make_float2(m, l);
      part_row(a, slot, r)[f] = o;
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
  __shared__ int64_t place[kPagedWaves][2];
  __shared__ float sO[kPagedWaves][kRowTile][kRowMaxD], sm[kPagedWaves][kRowTile],
      sl[kPagedWaves][kRowTile];
  __shared__ int sbad;
  const int lane = threadIdx.x % 64, wave = threadIdx.x / 64;
  const Place pl = locate<kRowUnit>(a, place);
  const PagedShare share(pl.total, a.groups);
  const int64_t begin = share.begin(blockIdx.x), end = share.begin(blockIdx.x + 1);
  const int64_t capacity = a.M * a.page;
  int64_t req = pl.request, base = pl.start;
  for (int64_t u = begin; u < end;) {
    const int32_t keys = paged_keys(a.lens[req], capacity);
    const int64_t units = paged_units(keys, kRowUnit);
    const int64_t seg = (u - base) / units, c0 = (u - base) % units;
    const int64_t count = end - u < units - c0 ? end - u : units - c0;
    const int64_t hk = seg / a.tiles, r0 = seg % a.tiles * a.rows;
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
    for (int64_t c = c0; c < c0 + count; ++c) {
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
#pragma unroll
          for (int j = 0; j < NF; ++j) acc[r][j] = acc[r][j] * c1 + p1 * vf[j];
          m[r] = mnew;
        }
      }
    }
    if (threadIdx.x == 0) sbad = 0;
    __syncthreads();
    if (bad) sbad = 1;
#pragma unroll
    for (int r = 0; r < kRowTile; ++r) {
#pragma unroll
      for (int j = 0; j < NF; ++j) sO[wave][r][lane + 64 * j] = acc[r][j];
      if (lane == 0) {
        sm[wave][r] = m[r];
        sl[wave][r] = l[r];
      }
    }
    __syncthreads();
    finish<T>(a, &sO[0][0][0], kRowMaxD, kRowTile * kRowMaxD, &sm[0][0], &sl[0][0], kRowTile,
              rows, count == units, 2 * int64_t(blockIdx.x) + (u > begin), req, hk * a.G + r0,
              keys == 0, sbad != 0);
    __syncthreads();
    u += count;
    if (u == base + units * a.Hk * a.tiles) {
      base = u;
      ++req;
    }
  }
}

// Rows of segments that several work-groups share: one work-group of 256
// threads per (segment, row); the partials go in the work-groups' order.
template <typename T>
__global__ __launch_bounds__(kPagedThreads) void paged_merge_kernel(PagedArgs a) {
  const int64_t seg = blockIdx.x, r = blockIdx.y, per_request = a.Hk * a.tiles;
  const int64_t n = seg / per_request, s = seg % per_request;
  const int64_t hk = s / a.tiles, head = s % a.tiles * a.rows + r;
  if (head >= a.G) return;
  const int64_t base = a.start[n], units = (a.start[n + 1] - base) / per_request;
  const int64_t u0 = base + s * units, u1 = u0 + units;
  const PagedShare share(a.start[a.N], a.groups);
  const int64_t w0 = share.owner(u0), w1 = share.owner(u1 - 1);
  if (w0 == w1) return;  // written whole
  const int64_t first = 2 * w0 + (share.begin(w0) < u0);
  for (int f = threadIdx.x; f < a.D; f += kPagedThreads) {
    float m = -__builtin_inff();
    for (int64_t w = w0; w <= w1; ++w) {
      const float2 ml = part_ml(a, w == w0 ? first : 2 * w)[r];
      if (!(ml.y == 0.f)) m = __builtin_fmaxf(m, ml.x);
    }
    float l = 0.f, o = 0.f;
    for (int64_t w = w0; w <= w1; ++w) {
      const int64_t slot = w == w0 ? first : 2 * w;
      const float2 ml = part_ml(a, slot)[r];
      if (ml.y == 0.f) continue;
      const float c = __builtin_amdgcn_exp2f(ml.x - m);
      l += c * ml.y;
      o += c * part_row(a, slot, r)[f];
    }
    T* out = static_cast<T*>(a.out) + n * a.on + (hk * a.G + head) * a.oh;
    out[f] = Round<T>::store(o / l);
  }
}

static int64_t round256(int64_t x) { return (x + 255) / 256 * 256; }

int64_t plan_paged_attn(int dtype, PagedArgs& a) {
  (void)dtype;
  const int64_t unit = kRowUnit, tile = kRowTile;
  a.tiles = (a.G + tile - 1) / tile;
  a.rows = (a.G + a.tiles - 1) / a.tiles;
  const int64_t longest = (a.M * a.page + unit - 1) / unit;
  const int64_t most = a.N * a.Hk * a.tiles * (longest > 1 ? longest : 1);  // units, at most
  if (most >= (int64_t(1) << 31)) return -1;
  a.groups = most < 2048 ? most : 2048;
  a.by_page = FastDiv(uint32_t(a.page));
  // Pairs and rows of 2 * groups partial slots, and the requests' first units.
  return round256((4 * a.groups * a.rows + 3) / 4 * 16 + 2 * a.groups * a.rows * a.D * 4) +
         round256(8 * (a.N + 1));
}

template <typename T>
static hipError_t launch_paged_t(const PagedArgs& a, hipStream_t stream) {
  const dim3 grid{unsigned(a.groups)}, block{kPagedThreads};
  if (a.D <= 64)
    hipLaunchKernelGGL((paged_row_kernel<T, 1>), grid, block, 0, stream, a);
  else if (a.D <= 128)
    hipLaunchKernelGGL((paged_row_kernel<T, 2>), grid, block, 0, stream, a);
  else
    hipLaunchKernelGGL((paged_row_kernel<T, 4>), grid, block, 0, stream, a);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  hipLaunchKernelGGL(paged_merge_kernel<T>, dim3(unsigned(a.N * a.Hk * a.tiles), unsigned(a.rows)),
                     block, 0, stream, a);
  return hipGetLastError();
}

hipError_t launch_paged_attn(int dtype, PagedArgs a, void* workspace, hipStream_t stream) {
  const int64_t need = plan_paged_attn(dtype, a);
  if (need < 0) return hipErrorInvalidValue;
  a.part = static_cast<float*>(workspace);
  a.start = reinterpret_cast<int64_t*>(static_cast<char*>(workspace) + need -
                                       round256(8 * (a.N + 1)));
  if (dtype == kBF16) return launch_paged_t<bf16_t>(a, stream);
  if (dtype == kF16) return launch_paged_t<f16_t>(a, stream);
  return launch_paged_t<float>(a, stream);
}

}  // namespace va
