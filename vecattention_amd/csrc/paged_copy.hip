// Pages of a key-value cache to other pages of it, in all layers with one launch:
// the tails of forked rows and the moves of a compaction.  A copy of whole rows:
// HBM for many pages, latency for a few.  A page is cut into pieces of 16 bytes
// (of one element where strides or addresses allow no more), numbered along the
// smaller of its row and head strides, and a work-group copies kPer of them to a
// thread, all loads before the stores.
#include "common.h"
#include "paged_ops.h"

namespace va {

namespace {

constexpr int kThreads = 256, kPer = 8;

struct Pieces {
  FastDiv by_part, by_inner;  // pieces of a head's row; heads (rows) of a page
  uint32_t parts, inner, total;
  bool rows_inner;
};

template <typename P>
__global__ __launch_bounds__(kThreads) void copy_pages_kernel(CopyArgs a, Pieces pc, int width,
                                                              uint32_t units, uint32_t most) {
  // Unit u of entry e, for the cache blockIdx.y.
  const int half = a.caches / 2, kind = blockIdx.y >= unsigned(half);
  P* cache = static_cast<P*>(a.cache[blockIdx.y]);
  const int64_t sp = a.sp[kind] / width, sn = a.sn[kind] / width, sh = a.sh[kind] / width;
  for (uint32_t w = blockIdx.x; w < most; w += gridDim.x) {
    const uint32_t e = w / units, u = w - e * units;
    const int32_t src = a.src[e], dst = a.dst[e];
    if (!is_page(src, a.num_pages) || !is_page(dst, a.num_pages) || src == dst) continue;
    const int32_t asked = a.rows ? a.rows[e] : a.page;
    const int32_t rows = asked < a.page ? asked : a.page;
    if (rows <= 0) continue;
    const P* from = cache + src * sp;
    P* to = cache + dst * sp;
    P x[kPer];
    int64_t at[kPer];
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const uint32_t k = (u * kPer + i) * kThreads + threadIdx.x;
      at[i] = -1;
      if (k >= pc.total) continue;
      const uint32_t line = pc.by_part.div(k), part = k - line * pc.parts;
      const uint32_t outer = pc.by_inner.div(line), inner = line - outer * pc.inner;
      const uint32_t row = pc.rows_inner ? inner : outer, head = pc.rows_inner ? outer : inner;
      if (int32_t(row) >= rows) continue;
      at[i] = row * sn + head * sh + part;
      x[i] = from[at[i]];
    }
#pragma unroll
    for (int i = 0; i < kPer; ++i)
      if (at[i] >= 0) to[at[i]] = x[i];
  }
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
  const uint32_t units = (pc.total + kPer * kThreads - 1) / (kPer * kThreads);
  const int64_t most = a.C * units;
  hipLaunchKernelGGL((copy_pages_kernel<P>),
                     dim3(unsigned(most < 2048 ? most : 2048), unsigned(a.caches)), dim3(kThreads),
                     0, stream, a, pc, width, units, uint32_t(most));
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
  if (aligned) return launch_pieces<uint4>(a, int(whole), stream);
  if (es == 4) return launch_pieces<uint32_t>(a, 1, stream);
  return launch_pieces<uint16_t>(a, 1, stream);
}

}  // namespace va
