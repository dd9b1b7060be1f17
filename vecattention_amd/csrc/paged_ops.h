// Arguments and launches of the paged-cache operators.
#pragma once
#include "common.h"
#include "paged.h"

namespace va {

hipError_t launch_paged_plan(const int32_t* kv_lens, const int32_t* new_lens, int64_t N,
                             int32_t* table, int64_t table_stride, int64_t M,
                             const int32_t* free_pages, int64_t F, const int32_t* free_head,
                             int64_t page, int64_t tokens, int32_t* kv_out, int32_t* indptr,
                             int64_t* slots, int64_t* positions, int32_t* requests,
                             int64_t* taken, uint32_t* workspace, hipStream_t stream);
int64_t plan_workspace_bytes(int64_t N);

constexpr int kRopeAxes = 4;

struct RopeRows {   // rows of one tensor: row (b, h, s) at base + b*sb + h*sh + s*ss
  const void* x;
  int64_t sb, sh, ss;
  void* y;
  int64_t tb, th, ts;
};
struct RopeArgs {
  RopeRows q, k;          // k.y is null where the keys go to the cache
  const void* v;          // values of the tokens (cache form): row (h, s)
  int64_t vh, vs;
  void *kc, *vc;          // caches: row (page, in, h) at page*p + in*n + h*h
  int64_t kp, kn, kh, vp, vn, vch;
  const int64_t* slots;
  int64_t num_slots;
  uint32_t page;
  int64_t B, S;
  int Hq, Hk, D, rot;
  const int64_t* positions;   // (axis, b, s) at axis*pa + b*pb + s
  int64_t pa, pb;
  int axes, section_end[kRopeAxes];
  const float* inv_freq;
  const void *qw, *kw;        // norm weights or null
  int w_f32;                  // the weights are fp32, whatever the rows are
  float eps, scaling;
  bool adjacent;
};
constexpr int kRopeMaxD = 512;
hipError_t launch_rope(int dtype, const RopeArgs& a, hipStream_t stream);

struct WriteArgs {
  const void *k, *v;          // row (t, h) at t*ks + h*kh
  int64_t ks, kh, vs, vh;
  void *kc, *vc;
  int64_t kp, kn, kch, vp, vn, vch;
  const int64_t* slots;
  int64_t num_slots;
  uint32_t page;
  int64_t T;
  int Hk, D;
};
hipError_t launch_write_kv(int dtype, const WriteArgs& a, hipStream_t stream);

// Decode attention over pages.  Row (page, in, h) of the keys at
// page*kp + in*kn + h*kh, of the values at page*vp + in*vn + h*vh; query row
// (n, h) at n*qn + h*qh, output row at n*on + h*oh (elements).
struct PagedArgs {
  const void *q, *k, *v;
  void* out;
  int64_t qn, qh, kp, kn, kh, vp, vn, vh, on, oh;
  const int32_t* table;
  int64_t table_stride, M;   // M page entries a row
  const int32_t* lens;
  int64_t N, Hk, G;          // G query heads per kv head
  int64_t D, page, num_pages;
  float scale_log2;
  int32_t tiles, rows;       // tiles of at most `rows` query heads per kv head
  int32_t groups;            // work-groups the units are dealt to
  int32_t per_request;       // segments of a request: Hk * tiles
  float* part;               // partial rows, see paged_attn.hip
  int2* split;               // per segment: first slot and last work-group, -1 written whole
  FastDiv by_page;
};
// Workspace bytes for these sizes (N, Hk, G, D, M, page), -1 where the units do
// not fit 31 bits.
int64_t paged_attn_workspace(int dtype, PagedArgs a);
hipError_t launch_paged_attn(int dtype, PagedArgs a, void* workspace, hipStream_t stream);

}  // namespace va
