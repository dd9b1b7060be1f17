// Plan of a step over a paged key-value cache: from the lengths of the requests
// and the tokens each adds, the pages they take from the free list, the block
// tables with those pages, and for every new token its request, position and
// slot (formulas: PlanRow and plan_slot in paged.h).
//
// Two exclusive prefix sums over the requests (new tokens, new pages) decide
// everything; a token then needs the request that holds it, a binary search in
// the first sum.  The sums cost less than a second launch: every work-group
// takes them for itself, with the results in LDS, and handles its share of the
// tokens and of the new pages.  A token of a new page reads the page's id from
// the free list, not from the table entry that another work-group writes, so
// the work-groups are independent.  Past kPlanLds requests the sums no longer
// fit and a launch of one work-group leaves them in the workspace.
#include "common.h"
#include "paged_ops.h"

namespace va {

constexpr int kPlanLds = 2048;       // requests whose sums fit the LDS of a work-group (32 KB)
constexpr int kPlanThreads = 256;

struct PlanArgs {
  const int32_t* kv_lens;
  const int32_t* new_lens;
  int64_t N;
  int32_t* table;
  int64_t table_stride, M;
  const int32_t* free_pages;
  int64_t F;
  const int32_t* free_head;
  uint32_t page;
  int64_t tokens;
  int32_t* kv_out;
  int32_t* indptr;
  int64_t* slots;
  int64_t* positions;
  int32_t* requests;
  int64_t* taken;
};

__device__ inline PlanRow plan_row(const PlanArgs& a, int64_t i) {
  return PlanRow(a.kv_lens[i], a.new_lens[i], a.page, uint32_t(a.M));
}

// Exclusive sums of (x, y) over the work-group, and their totals in *tx, *ty.
template <int kThreads>
__device__ inline void block_exclusive(int64_t& x, int64_t& y, int64_t* tx, int64_t* ty,
                                       int64_t (*wave)[2]) {
  const int lane = threadIdx.x % 64, w = threadIdx.x / 64;
  int64_t sx = x, sy = y;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const int64_t ux = __shfl_up(sx, d), uy = __shfl_up(sy, d);
    if (lane >= d) {
      sx += ux;
      sy += uy;
    }
  }
  if (lane == 63) {
    wave[w][0] = sx;
    wave[w][1] = sy;
  }
  __syncthreads();
  int64_t bx = 0, by = 0, ax = 0, ay = 0;
#pragma unroll
  for (int i = 0; i < kThreads / 64; ++i) {
    if (i < w) {
      bx += wave[i][0];
      by += wave[i][1];
    }
    ax += wave[i][0];
    ay += wave[i][1];
  }
  x = bx + sx - x;
  y = by + sy - y;
  *tx = ax;
  *ty = ay;
}

// Outputs of one request: the length after the step and the row start.
__device__ inline void plan_request(const PlanArgs& a, int64_t i, const PlanRow& r,
                                    int64_t first_token) {
  const uint32_t end = r.len + r.fresh;
  a.kv_out[i] = int32_t(end < 0x7fffffffu ? end : 0x7fffffffu);
  a.indptr[i] = int32_t(first_token < 0x7fffffff ? first_token : 0x7fffffff);
}

// Largest i in [0, n) with start[i] <= x, where start[0] = 0 <= x < start[n]:
// the request that holds x (requests that hold nothing are passed over).
__device__ inline int64_t holder(const int64_t* start, int64_t n, int64_t x) {
  int64_t lo = 0, hi = n;
  while (hi - lo > 1) {
    const int64_t mid = (lo + hi) >> 1;
    if (start[mid] <= x)
      lo = mid;
    else
      hi = mid;
  }
  return lo;
}

// The work-group's tokens and pages.  tok, pag: the sums, with the totals at [N].
__device__ inline void plan_fill(const PlanArgs& a, const int64_t* tok, const int64_t* pag) {
  const int64_t threads = int64_t(gridDim.x) * kPlanThreads;
  const int64_t me = int64_t(blockIdx.x) * kPlanThreads + threadIdx.x;
  const int64_t head = a.free_head ? int64_t(*a.free_head) : 0;
  const int64_t ntok = tok[a.N], npag = pag[a.N];
  for (int64_t t = me; t < a.tokens; t += threads) {
    int64_t slot = -1, pos = 0;
    int32_t req = -1;
    if (t < ntok) {
      const int64_t i = holder(tok, a.N, t);
      const PlanRow r = plan_row(a, i);
      const uint32_t p = r.len + uint32_t(t - tok[i]);
      slot = plan_slot(r, p, a.page, uint32_t(a.M), a.table + i * a.table_stride, a.free_pages,
                       a.F, head + pag[i]);
      pos = p;
      req = int32_t(i);
    }
    a.slots[t] = slot;
    a.positions[t] = pos;
    a.requests[t] = req;
  }
  for (int64_t g = me; g < npag; g += threads) {
    const int64_t i = holder(pag, a.N, g);
    const PlanRow r = plan_row(a, i);
    a.table[i * a.table_stride + r.held + (g - pag[i])] = free_page(a.free_pages, a.F, head + g);
  }
  if (me == 0) {
    a.indptr[a.N] = int32_t(ntok < 0x7fffffff ? ntok : 0x7fffffff);
    *a.taken = npag;
  }
}

__global__ __launch_bounds__(kPlanThreads) void plan_kernel(PlanArgs a) {
  __shared__ int64_t tok[kPlanLds + 1], pag[kPlanLds + 1];
  __shared__ int64_t wave[kPlanThreads / 64][2];
  const int64_t per = (a.N + kPlanThreads - 1) / kPlanThreads;
  const int64_t lo = threadIdx.x * per < a.N ? threadIdx.x * per : a.N;
  const int64_t hi = lo + per < a.N ? lo + per : a.N;
  int64_t x = 0, y = 0, tx, ty;
  for (int64_t i = lo; i < hi; ++i) {
    const PlanRow r = plan_row(a, i);
    x += r.fresh;
    y += r.need;
  }
  block_exclusive<kPlanThreads>(x, y, &tx, &ty, wave);
  for (int64_t i = lo; i < hi; ++i) {
    const PlanRow r = plan_row(a, i);
    tok[i] = x;
    pag[i] = y;
    if (blockIdx.x == 0) plan_request(a, i, r, x);
    x += r.fresh;
    y += r.need;
  }
  if (threadIdx.x == 0) {
    tok[a.N] = tx;
    pag[a.N] = ty;
  }
  __syncthreads();
  plan_fill(a, tok, pag);
}

// More requests than LDS holds: the sums of all of them, kThreads at a time.
constexpr int kScanThreads = 1024;
__global__ __launch_bounds__(kScanThreads) void plan_scan_kernel(PlanArgs a, int64_t* tok,
                                                                 int64_t* pag) {
  __shared__ int64_t wave[kScanThreads / 64][2];
  int64_t bx = 0, by = 0;
  for (int64_t base = 0; base < a.N; base += kScanThreads) {
    const int64_t i = base + threadIdx.x;
    const PlanRow r = i < a.N ? plan_row(a, i) : PlanRow(0, 0, 1, 0);
    int64_t x = r.fresh, y = r.need, tx, ty;
    block_exclusive<kScanThreads>(x, y, &tx, &ty, wave);
    if (i < a.N) {
      tok[i] = bx + x;
      pag[i] = by + y;
      plan_request(a, i, r, bx + x);
    }
    bx += tx;
    by += ty;
    __syncthreads();  // `wave` is written again
  }
  if (threadIdx.x == 0) {
    tok[a.N] = bx;
    pag[a.N] = by;
  }
}
__global__ __launch_bounds__(kPlanThreads) void plan_fill_kernel(PlanArgs a, const int64_t* tok,
                                                                 const int64_t* pag) {
  plan_fill(a, tok, pag);
}

int64_t plan_workspace_bytes(int64_t N) { return N <= kPlanLds ? 0 : 16 * (N + 1); }

hipError_t launch_paged_plan(const int32_t* kv_lens, const int32_t* new_lens, int64_t N,
                             int32_t* table, int64_t table_stride, int64_t M,
                             const int32_t* free_pages, int64_t F, const int32_t* free_head,
                             int64_t page, int64_t tokens, int32_t* kv_out, int32_t* indptr,
                             int64_t* slots, int64_t* positions, int32_t* requests,
                             int64_t* taken, int64_t* workspace, hipStream_t stream) {
  const PlanArgs a{kv_lens, new_lens, N,      table,  table_stride, M,         free_pages, F,
                   free_head, uint32_t(page), tokens, kv_out,       indptr,    slots,
                   positions, requests,       taken};
  // Four tokens a thread: fewer repeat the sums more often, more leave CUs idle.
  int64_t groups = (tokens + 4 * kPlanThreads - 1) / (4 * kPlanThreads);
  if (groups < 1) groups = 1;
  if (groups > 4096) groups = 4096;
  if (N <= kPlanLds) {
    hipLaunchKernelGGL(plan_kernel, dim3(unsigned(groups)), dim3(kPlanThreads), 0, stream, a);
  } else {
    hipLaunchKernelGGL(plan_scan_kernel, dim3(1), dim3(kScanThreads), 0, stream, a, workspace,
                       workspace + (N + 1));
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    hipLaunchKernelGGL(plan_fill_kernel, dim3(unsigned(groups)), dim3(kPlanThreads), 0, stream, a,
                       workspace, workspace + (N + 1));
  }
  return hipGetLastError();
}

}  // namespace va
