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

// The next step's rows from this one's (paged_share.hip).
struct ForkArgs {
  const int32_t *kv_lens, *keep, *parents;  // (N), (R) or null, (R)
  const int32_t* table;
  int64_t table_stride, N, R, M;
  const int32_t* shares;
  int64_t P;
  const int32_t* free_pages;
  int64_t F;
  const int32_t* free_head;
  uint32_t page;
  int32_t *kv_out, *table_out, *shares_out, *free_out, *head_out;
  int32_t *copy_src, *copy_dst, *copy_rows;
};
constexpr int64_t kForkMostRows = 65536;
int64_t fork_workspace_bytes(int64_t R, int64_t P);
hipError_t launch_paged_fork(const ForkArgs& a, void* workspace, hipStream_t stream);

struct CompactArgs {
  const int32_t* kv_lens;
  const int32_t* table;
  int64_t table_stride, N, M;
  const int32_t* shares;
  int64_t P;
  const int32_t* free_pages;
  int64_t F;
  const int32_t* free_head;
  uint32_t page;
  int32_t *table_out, *shares_out, *free_out, *head_out;
  int32_t *copy_src, *copy_dst, *num_moves;
};
int64_t compact_workspace_bytes(int64_t P);
hipError_t launch_paged_compact(const CompactArgs& a, void* workspace, hipStream_t stream);

struct PrefixArgs {
  const int32_t* kv_lens;
  const int32_t* table;
  int64_t table_stride, N, M;
  const int32_t* ids;  // or null
  uint32_t page;
  int32_t *prefix_lens, *group_rows;
};
constexpr int64_t kPrefixMostRows = 65536;
int64_t prefix_workspace_bytes(int64_t N);
hipError_t launch_paged_prefix(const PrefixArgs& a, void* workspace, hipStream_t stream);

// Rows of pages to other pages of each of `caches` caches, half of them with the
// strides of the keys, the others with those of the values.
constexpr int kCopyCaches = 64;
struct CopyArgs {
  void* cache[kCopyCaches];
  int32_t caches;
  int64_t sp[2], sn[2], sh[2];  // page, row and head strides of keys and values
  const int32_t *src, *dst, *rows;
  int64_t C, num_pages;
  int32_t page, heads, D;
};
hipError_t launch_copy_kv(int dtype, const CopyArgs& a, hipStream_t stream);

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
  // Attention of rows that share their first keys (paged_prefix.hip): those keys of
  // row n, and the rows of the group that begins there.  Its kernels leave states (m,
  // l) and unnormalised rows of D: `state` one for each (request, query head).
  const int32_t *prefix_lens, *group_rows;
  float2* state_ml;
  float* state;
};

// Keys of a prefix that are computed for its rows together: whole tiles of them.
constexpr int kPrefixTile = 64;
__host__ __device__ inline int32_t shared_keys(int32_t prefix, int64_t capacity) {
  const int64_t n = prefix < capacity ? prefix : capacity;
  return n <= 0 ? 0 : int32_t(n / kPrefixTile * kPrefixTile);
}
// Workspace bytes for these sizes (N, Hk, G, D, M, page), -1 where the units do
// not fit 31 bits.
int64_t paged_attn_workspace(int dtype, PagedArgs a);
hipError_t launch_paged_attn(int dtype, PagedArgs a, void* workspace, hipStream_t stream);

// Whether the matrix-core form takes these tensors; its work for the states of every
// row's own keys (from shared_keys on), and the bytes of the partial rows.
bool paged_tile_form(int dtype, const PagedArgs& a);
int64_t paged_states_workspace(int dtype, PagedArgs& a);

int64_t prefix_attn_workspace(int dtype, PagedArgs a);
hipError_t launch_prefix_attn(int dtype, PagedArgs a, void* workspace, hipStream_t stream);

}  // namespace va
