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

constexpr int kPlanLds = 2048;       // requests whose sums fit the LDS of a work-group (16 KB)
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
  uint32_t token_groups;
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

__device__ inline int64_t plan_head(const PlanArgs& a) {
  return a.free_head ? int64_t(*a.free_head) : 0;
}

// Sums that end at 2^31 - 1 (still associative, for values up to that): no token
// or entry behind it is ever looked up.
constexpr uint32_t kMost = 0x7fffffffu;
__device__ inline uint32_t plus(uint32_t a, uint32_t b) {
  const uint32_t s = a + b;
  return s < kMost ? s : kMost;
}
// As wave_inclusive_sum (lanes.h), with plus.
__device__ inline uint32_t wave_inclusive_plus(uint32_t x) {
#define VA_STEP(ctrl, rows) \
  x = plus(x, uint32_t(__builtin_amdgcn_update_dpp(0, int(x), ctrl, rows, 0xf, false)))
  VA_STEP(0x111, 0xf);  // row_shr:1, 2, 4, 8
  VA_STEP(0x112, 0xf);
  VA_STEP(0x114, 0xf);
  VA_STEP(0x118, 0xf);
  VA_STEP(0x142, 0xa);  // row_bcast:15 -> rows 1, 3
  VA_STEP(0x143, 0xc);  // row_bcast:31 -> rows 2, 3
#undef VA_STEP
  return x;
}

// Exclusive sums of x and of y over the work-group, and their totals.
template <int kThreads>
__device__ inline void block_exclusive(uint32_t& x, uint32_t& y, uint32_t* tx, uint32_t* ty,
                                       uint2* wave) {
  const int lane = threadIdx.x % 64, w = threadIdx.x / 64;
  const uint32_t sx = wave_inclusive_plus(x), sy = wave_inclusive_plus(y);
  if (lane == 63) wave[w] = make_uint2(sx, sy);
  __syncthreads();
  uint32_t bx = 0, by = 0;
  *tx = *ty = 0;
#pragma unroll
  for (int i = 0; i < kThreads / 64; ++i) {
    if (i < w) {
      bx = plus(bx, wave[i].x);
      by = plus(by, wave[i].y);
    }
    *tx = plus(*tx, wave[i].x);
    *ty = plus(*ty, wave[i].y);
  }
  // Exclusive: the lane before's sum.
  const uint32_t ex = __shfl_up(sx, 1), ey = __shfl_up(sy, 1);
  x = plus(bx, lane ? ex : 0u);
  y = plus(by, lane ? ey : 0u);
}

// Outputs of one request: the length after the step and the row start.
__device__ inline void plan_request(const PlanArgs& a, int64_t i, const PlanRow& r,
                                    uint32_t first_token) {
  a.kv_out[i] = int32_t(plus(r.len, r.fresh));
  a.indptr[i] = int32_t(first_token);
}

// Largest i in [0, n) with start[i] <= x, where start[0] = 0 <= x < start[n]:
// the request that holds x (requests that hold nothing are passed over).
__device__ inline uint32_t holder(const uint32_t* start, uint32_t n, uint32_t x) {
  uint32_t lo = 0, hi = n;
  while (hi - lo > 1) {
    const uint32_t mid = (lo + hi) >> 1;
    if (start[mid] <= x)
      lo = mid;
    else
      hi = mid;
  }
  return lo;
}

// The work-group's share.  tok, pag: the sums, with the totals at [N].  The first
// `token_groups` work-groups take the tokens, kRun in a row to a thread, which makes
// one search, one division for each request and page that they reach, and 16-byte
// stores (steps of single tokens: kRun 1, all searches at once); the others take the
// new pages.
template <int kRun>
__device__ inline void plan_fill(const PlanArgs& a, const uint32_t* tok, const uint32_t* pag,
                                 int64_t head) {
  const uint32_t N = uint32_t(a.N);
  const uint32_t ntok = tok[N], npag = pag[N];
  if (blockIdx.x >= a.token_groups) {
    const uint32_t threads = (gridDim.x - a.token_groups) * kPlanThreads;
    const uint32_t me = (blockIdx.x - a.token_groups) * kPlanThreads + threadIdx.x;
    for (uint32_t g = me; g < npag; g += threads) {
      const uint32_t i = holder(pag, N, g);
      const PlanRow r = plan_row(a, i);
      a.table[int64_t(i) * a.table_stride + r.held + (g - pag[i])] =
          free_page(a.free_pages, a.F, head + g);
    }
    if (me == 0) {
      a.indptr[N] = int32_t(ntok);
      *a.taken = npag;
    }
    return;
  }
  const int64_t step = int64_t(a.token_groups) * kPlanThreads * kRun;
  for (int64_t t0 = (int64_t(blockIdx.x) * kPlanThreads + threadIdx.x) * kRun; t0 < a.tokens;
       t0 += step) {
    uint32_t i = 0, next = 0, pos = 0, left = 0;  // request, its last token + 1, tokens left in page
    int64_t slot = -1;
    int64_t slots[kRun], positions[kRun];
    int32_t requests[kRun];
#pragma unroll
    for (int e = 0; e < kRun; ++e) {
      const uint32_t t = uint32_t(t0 + e);
      const bool real = t0 + e < a.tokens && t < ntok;
      if (real) {
        if (e == 0 || t >= next || left == 0) {
          if (e == 0 || t >= next) i = holder(tok, N, t);
          next = tok[i + 1];
          const PlanRow r = plan_row(a, i);
          pos = r.len + (t - tok[i]);
          slot = plan_slot(r, pos, a.page, uint32_t(a.M), a.table + int64_t(i) * a.table_stride,
                           a.free_pages, a.F, head + pag[i]);
          left = a.page - pos % a.page - 1;
        } else {
          ++pos;
          --left;
          slot = slot < 0 ? -1 : slot + 1;
        }
      }
      slots[e] = real ? slot : -1;
      positions[e] = real ? int64_t(pos) : 0;
      requests[e] = real ? int32_t(i) : -1;
    }
    if (kRun == 4 && t0 + kRun <= a.tokens) {
      typedef int64_t long2_t __attribute__((ext_vector_type(2)));
      typedef int32_t int4_t __attribute__((ext_vector_type(4)));
#pragma unroll
      for (int e = 0; e + 1 < kRun; e += 2) {
        *reinterpret_cast<long2_t*>(a.slots + t0 + e) = long2_t{slots[e], slots[e + 1]};
        *reinterpret_cast<long2_t*>(a.positions + t0 + e) =
            long2_t{positions[e], positions[e + 1]};
      }
      *reinterpret_cast<int4_t*>(a.requests + t0) =
          int4_t{requests[0], requests[1 % kRun], requests[2 % kRun], requests[3 % kRun]};
    } else {
#pragma unroll
      for (int e = 0; e < kRun; ++e) {
        if (t0 + e >= a.tokens) break;
        a.slots[t0 + e] = slots[e];
        a.positions[t0 + e] = positions[e];
        a.requests[t0 + e] = requests[e];
      }
    }
  }
}

template <int kRun>
__global__ __launch_bounds__(kPlanThreads) void plan_kernel(PlanArgs a) {
  __shared__ uint32_t tok[kPlanLds + 1], pag[kPlanLds + 1];
  __shared__ uint2 wave[kPlanThreads / 64];
  const int per = int(a.N + kPlanThreads - 1) / kPlanThreads;
  const int lo = int(threadIdx.x) * per, N = int(a.N);
  const int64_t head = plan_head(a);
  uint32_t x = 0, y = 0, tx, ty;
  for (int i = lo; i < lo + per && i < N; ++i) {
    const PlanRow r = plan_row(a, i);
    tok[i] = r.fresh;  // read by this thread alone, below
    pag[i] = r.need;
    x = plus(x, r.fresh);
    y = plus(y, r.need);
  }
  block_exclusive<kPlanThreads>(x, y, &tx, &ty, wave);
  for (int i = lo; i < lo + per && i < N; ++i) {
    const uint32_t fresh = tok[i], need = pag[i];
    tok[i] = x;
    pag[i] = y;
    if (blockIdx.x == 0) plan_request(a, i, plan_row(a, i), x);
    x = plus(x, fresh);
    y = plus(y, need);
  }
  if (threadIdx.x == 0) {
    tok[N] = tx;
    pag[N] = ty;
  }
  __syncthreads();
  plan_fill<kRun>(a, tok, pag, head);
}

// More requests than LDS holds: the sums of all of them, kThreads at a time.
constexpr int kScanThreads = 1024;
__global__ __launch_bounds__(kScanThreads) void plan_scan_kernel(PlanArgs a, uint32_t* tok,
                                                                 uint32_t* pag) {
  __shared__ uint2 wave[kScanThreads / 64];
  uint32_t bx = 0, by = 0;
  for (int64_t base = 0; base < a.N; base += kScanThreads) {
    const int64_t i = base + threadIdx.x;
    const PlanRow r = i < a.N ? plan_row(a, i) : PlanRow(0, 0, 1, 0);
    uint32_t x = r.fresh, y = r.need, tx, ty;
    block_exclusive<kScanThreads>(x, y, &tx, &ty, wave);
    if (i < a.N) {
      tok[i] = plus(bx, x);
      pag[i] = plus(by, y);
      plan_request(a, i, r, plus(bx, x));
    }
    bx = plus(bx, tx);
    by = plus(by, ty);
    __syncthreads();  // `wave` is written again
  }
  if (threadIdx.x == 0) {
    tok[a.N] = bx;
    pag[a.N] = by;
  }
}
__global__ __launch_bounds__(kPlanThreads) void plan_fill_kernel(PlanArgs a, const uint32_t* tok,
                                                                 const uint32_t* pag) {
  plan_fill<1>(a, tok, pag, plan_head(a));
}

int64_t plan_workspace_bytes(int64_t N) { return N <= kPlanLds ? 0 : 8 * (N + 1); }

hipError_t launch_paged_plan(const int32_t* kv_lens, const int32_t* new_lens, int64_t N,
                             int32_t* table, int64_t table_stride, int64_t M,
                             const int32_t* free_pages, int64_t F, const int32_t* free_head,
                             int64_t page, int64_t tokens, int32_t* kv_out, int32_t* indptr,
                             int64_t* slots, int64_t* positions, int32_t* requests,
                             int64_t* taken, uint32_t* workspace, hipStream_t stream) {
  // Steps of single tokens, or prompts among them, whose tokens are stored by fours.
  const bool whole = (reinterpret_cast<uintptr_t>(slots) | reinterpret_cast<uintptr_t>(positions) |
                      reinterpret_cast<uintptr_t>(requests)) % 16 == 0;
  const int run = N <= kPlanLds && tokens > 4 * N && whole ? 4 : 1;
  int64_t groups = (tokens + run * kPlanThreads - 1) / (run * kPlanThreads);
  if (groups < 1) groups = 1;
  if (groups > 4096) groups = 4096;
  int64_t page_groups = (tokens / page + N + 4 * kPlanThreads - 1) / (4 * kPlanThreads);
  if (page_groups < 1) page_groups = 1;
  if (page_groups > 1024) page_groups = 1024;
  const PlanArgs a{kv_lens,   new_lens,       N,
                   table,     table_stride,   M,
                   free_pages, F,             free_head,
                   uint32_t(page), uint32_t(groups), tokens,
                   kv_out,    indptr,         slots,
                   positions, requests,       taken};
  const dim3 grid{unsigned(groups + page_groups)}, block{kPlanThreads};
  if (N > kPlanLds) {
    hipLaunchKernelGGL(plan_scan_kernel, dim3(1), dim3(kScanThreads), 0, stream, a, workspace,
                       workspace + (N + 1));
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    hipLaunchKernelGGL(plan_fill_kernel, grid, block, 0, stream, a, workspace,
                       workspace + (N + 1));
  } else if (run == 4) {
    hipLaunchKernelGGL(plan_kernel<4>, grid, block, 0, stream, a);
  } else {
    hipLaunchKernelGGL(plan_kernel<1>, grid, block, 0, stream, a);
  }
  return hipGetLastError();
}

}  // namespace va
