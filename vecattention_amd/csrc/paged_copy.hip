// Pages of a key-value cache to other pages of it, in up to 32 layers with one launch:
// the tails of forked rows and the moves of a compaction.  A copy of whole rows:
// HBM for many pages, latency for a few.  A page is cut into pieces of 16 bytes
// (of one element where strides or addresses allow no more), numbered along the
// smaller of its row and head strides, and a work-group copies kPer of them to a
// thread, all loads before the stores.
//
// us, 1500 pages of 32 KB in eight caches (786 MB read and written): 233 with every
// piece's place found by two divisions, which made it 70 us of arithmetic; 158 (5.0 TB/s,
// a large copy's rate) where pages are blocks without gaps, whose pieces need none.  Last
// pages of eight rows in 4 layers: 5.1, the launch.  An empty entry costs a work-group an
// iteration in every cache: 50000 of them 43 in 4 layers, 279 in 28.
#include "common.h"
#include "paged_ops.h"

namespace va {

namespace {

constexpr int kThreads = 256, kPer = 8;

typedef uint32_t u32x4_t __attribute__((ext_vector_type(4)));

struct Pieces {
  FastDiv by_part, by_inner;  // pieces of a head's row; heads (rows) of a page
  uint32_t parts, inner, total;
  bool rows_inner;
  int64_t sp[2], sn[2], sh[2];  // strides in pieces
};

// kLinear: piece k of a page lies at k.  kStream: the pages are stored past the caches.
template <typename P, bool kLinear, bool kStream>
__global__ __launch_bounds__(kThreads) void copy_pages_kernel(CopyArgs a, Pieces pc,
                                                              uint32_t units, uint32_t most) {
  // Unit u of entry e, for the cache blockIdx.y.
  const int kind = blockIdx.y >= unsigned(a.caches / 2);
  P* cache = static_cast<P*>(a.cache[blockIdx.y]);
  const int64_t sp = pc.sp[kind], sn = pc.sn[kind], sh = pc.sh[kind];
  for (uint32_t w = blockIdx.x; w < most; w += gridDim.x) {
    const uint32_t e = units == 1 ? w : w / units, u = w - e * units;
    const int32_t src = a.src[e], dst = a.dst[e];
    if (!is_page(src, a.num_pages) || !is_page(dst, a.num_pages) || src == dst) continue;
    int32_t rows = a.rows ? a.rows[e] : a.page;
    if (rows > a.page) rows = a.page;
    if (rows <= 0) continue;
    const P* from = cache + src * sp;
    P* to = cache + dst * sp;
    P x[kPer];
    uint32_t k[kPer];
    int64_t at[kPer];
    bool take[kPer];
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      k[i] = (u * kPer + i) * kThreads + threadIdx.x;
      take[i] = k[i] < pc.total;
      at[i] = k[i];
    }
    if (!kLinear || rows < a.page) {
#pragma unroll
      for (int i = 0; i < kPer; ++i) {
        const uint32_t line = pc.by_part.div(k[i]), part = k[i] - line * pc.parts;
        const uint32_t outer = pc.by_inner.div(line), inner = line - outer * pc.inner;
        const uint32_t row = pc.rows_inner ? inner : outer, head = pc.rows_inner ? outer : inner;
        take[i] = take[i] && int32_t(row) < rows;
        if (!kLinear) at[i] = row * sn + head * sh + part;
      }
    }
#pragma unroll
    for (int i = 0; i < kPer; ++i)
      if (take[i]) x[i] = from[at[i]];
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      if (!take[i]) continue;
      if constexpr (kStream)
        __builtin_nontemporal_store(x[i], to + at[i]);
      else
        to[at[i]] = x[i];
    }
  }
}

template <typename P, bool kLinear>
void launch_form(const CopyArgs& a, const Pieces& pc, hipStream_t stream) {
  const uint32_t units = (pc.total + kPer * kThreads - 1) / (kPer * kThreads);
  const int64_t most = a.C * units;
  const dim3 grid{unsigned(most < 2048 ? most : 2048), unsigned(a.caches)}, block{kThreads};
  // Pages that the Infinity Cache could not hold until they are read again.
  if (int64_t(a.C) * pc.total * int64_t(sizeof(P)) * a.caches > (256 << 20))
    hipLaunchKernelGGL((copy_pages_kernel<P, kLinear, true>), grid, block, 0, stream, a, pc, units,
                       uint32_t(most));
  else
    hipLaunchKernelGGL((copy_pages_kernel<P, kLinear, false>), grid, block, 0, stream, a, pc,
                       units, uint32_t(most));
}

template <typename P>
hipError_t launch_pieces(const CopyArgs& a, int width, hipStream_t stream) {
  Pieces pc;
  pc.parts = uint32_t(a.D / width);
  pc.rows_inner = a.sn[0] < a.sh[0];
  pc.inner = uint32_t(pc.rows_inner ? a.page : a.heads);
  pc.total = uint32_t(a.page) * uint32_t(a.heads) * pc.parts;
  pc.by_part = FastDiv(pc.parts);
  pc.by_inner = FastDiv(pc.inner);
  bool linear = true;
  for (int i = 0; i < 2; ++i) {
    const int64_t inner = pc.rows_inner ? a.sn[i] : a.sh[i];
    const int64_t outer = pc.rows_inner ? a.sh[i] : a.sn[i];
    pc.sp[i] = a.sp[i] / width;
    pc.sn[i] = a.sn[i] / width;
    pc.sh[i] = a.sh[i] / width;
    linear = linear && (inner == a.D || pc.inner == 1) &&
             (outer == int64_t(pc.inner) * a.D || a.page * int64_t(a.heads) == pc.inner);
  }
  if (linear)
    launch_form<P, true>(a, pc, stream);
  else
    launch_form<P, false>(a, pc, stream);
  return hipGetLastError();
}

}  // namespace

hipError_t launch_copy_kv(int dtype, const CopyArgs& a, hipStream_t stream) {
  const int64_t es = dtype == kF32 ? 4 : 2, whole = 16 / es;
  bool aligned = a.D % whole == 0;
  for (int i = 0; i < a.caches; ++i)
    aligned = aligned && reinterpret_cast<uintptr_t>(a.cache[i]) % 16 == 0;
  for (int i = 0; i < 2; ++i)
    aligned = aligned && a.sp[i] % whole == 0 && a.sn[i] % whole == 0 && a.sh[i] % whole == 0;
  if (aligned) return launch_pieces<u32x4_t>(a, int(whole), stream);
  if (es == 4) return launch_pieces<uint32_t>(a, 1, stream);
  return launch_pieces<uint16_t>(a, 1, stream);
}

}  // namespace va
