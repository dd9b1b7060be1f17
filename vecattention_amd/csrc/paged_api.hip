// C entry points of the paged-cache operators: argument checks and launches
// (declarations: include/vecattn.h).
#include "../../include/vecattn.h"
#include "paged_ops.h"

namespace va {
int api_error(int code, const char* fmt, ...);
}

namespace {

using va::api_error;

bool dtype_ok(int dtype) { return dtype == VA_F32 || dtype == VA_BF16 || dtype == VA_F16; }

int launched(hipError_t e, const char* what) {
  return e == hipSuccess ? VA_OK : api_error(VA_ERR_HIP, "%s: %s", what, hipGetErrorString(e));
}

constexpr int64_t kInt31 = int64_t(1) << 31;

// page_size and num_pages of a cache: slots are counted in 62 bits, a token's
// place in 31.
int check_pages(int64_t num_pages, int64_t page_size) {
  if (page_size <= 0 || page_size >= kInt31)
    return api_error(VA_ERR_ARG, "page_size %lld", (long long)page_size);
  if (num_pages <= 0 || num_pages >= kInt31)
    return api_error(VA_ERR_ARG, "a cache of %lld pages", (long long)num_pages);
  return VA_OK;
}

// The rotation's and norms' part of the arguments.
int set_rotation(va::RopeArgs& a, int64_t D, int64_t rot, const int64_t* positions, int64_t pa,
                 int64_t pb, int64_t axes, const int64_t* sections, const float* inv_freq,
                 const void* qw, const void* kw, int dtype, int wdtype, float eps, float scaling,
                 int adjacent) {
  if (D > va::kRopeMaxD)
    return api_error(VA_ERR_UNSUPPORTED, "head_dim %lld > %d", (long long)D, va::kRopeMaxD);
  if (rot <= 0 || rot % 2 || rot > D)
    return api_error(VA_ERR_ARG, "rotary_dim %lld of head_dim %lld", (long long)rot, (long long)D);
  if (!positions || !inv_freq) return api_error(VA_ERR_ARG, "null positions or inv_freq");
  if (axes < 1 || axes > va::kRopeAxes)
    return api_error(VA_ERR_UNSUPPORTED, "%lld position axes: 1 to %d", (long long)axes,
                     va::kRopeAxes);
  if (axes > 1 && !sections) return api_error(VA_ERR_ARG, "position axes without their sections");
  int64_t end = 0;
  for (int64_t i = 0; i < axes; ++i) {
    const int64_t n = axes == 1 ? rot / 2 : sections[i];
    if (n < 0 || n > rot / 2 - end)
      return api_error(VA_ERR_ARG, "sections do not add up to rotary_dim / 2 = %lld",
                       (long long)(rot / 2));
    end += n;
    a.section_end[i] = int(end);
  }
  if (end != rot / 2)
    return api_error(VA_ERR_ARG, "sections do not add up to rotary_dim / 2 = %lld",
                     (long long)(rot / 2));
  if ((qw || kw) && wdtype != dtype && wdtype != VA_F32)
    return api_error(VA_ERR_ARG, "norm weights of type %d for rows of type %d", wdtype, dtype);
  a.D = int(D);
  a.rot = int(rot);
  a.positions = positions;
  a.pa = pa;
  a.pb = pb;
  a.axes = int(axes);
  a.inv_freq = inv_freq;
  a.qw = qw;
  a.kw = kw;
  a.w_f32 = wdtype == VA_F32;
  a.eps = eps;
  a.scaling = scaling;
  a.adjacent = adjacent != 0;
  return VA_OK;
}

// Sizes of rows that a launch counts in 31 bits.
bool fits(int64_t a, int64_t b, int64_t most) { return a <= most / (b > 0 ? b : 1); }

}  // namespace

extern "C" {

int64_t va_paged_plan_workspace_size(int64_t N) { return N < 0 ? -1 : va::plan_workspace_bytes(N); }

int va_paged_plan(const int32_t* kv_lens, const int32_t* new_lens, int64_t N,
                  int32_t* block_tables, int64_t stn, int64_t M, const int32_t* free_pages,
                  int64_t num_free, const int32_t* free_head, int64_t page_size,
                  int64_t num_tokens, int32_t* kv_lens_out, int32_t* qo_indptr,
                  int64_t* slot_mapping, int64_t* positions, int32_t* request_ids,
                  int64_t* pages_taken, void* workspace, int64_t workspace_bytes, void* stream) {
  if (N < 0 || M < 0 || num_free < 0 || num_tokens < 0)
    return api_error(VA_ERR_ARG, "negative size");
  if (N >= kInt31 || M >= kInt31 || num_free >= kInt31 || num_tokens >= kInt31)
    return api_error(VA_ERR_UNSUPPORTED, "sizes of 2^31 or more");
  if (page_size <= 0 || page_size >= kInt31)
    return api_error(VA_ERR_ARG, "page_size %lld", (long long)page_size);
  if (!qo_indptr || !pages_taken || (N && (!kv_lens || !new_lens || !kv_lens_out)) ||
      (N && M && !block_tables) || (num_free && !free_pages) ||
      (num_tokens && (!slot_mapping || !positions || !request_ids)))
    return api_error(VA_ERR_ARG, "null pointer");
  if (N > 1 && stn < M) return api_error(VA_ERR_ARG, "rows of block_tables overlap");
  const int64_t need = va::plan_workspace_bytes(N);
  if (need && (!workspace || workspace_bytes < need))
    return api_error(VA_ERR_WORKSPACE, "the plan needs %lld workspace bytes", (long long)need);
  if (need && reinterpret_cast<uintptr_t>(workspace) % 16)
    return api_error(VA_ERR_ARG, "workspace must be 16-byte aligned");
  return launched(
      va::launch_paged_plan(kv_lens, new_lens, N, block_tables, stn, M, free_pages, num_free,
                            free_head, page_size, num_tokens, kv_lens_out, qo_indptr, slot_mapping,
                            positions, request_ids, pages_taken,
                            static_cast<uint32_t*>(workspace), static_cast<hipStream_t>(stream)),
      "plan launch");
}

int va_qk_norm_rope(int dtype, const void* q, int64_t sqb, int64_t sqh, int64_t sqs, const void* k,
                    int64_t skb, int64_t skh, int64_t sks, void* q_out, int64_t sqob,
                    int64_t sqoh, int64_t sqos, void* k_out, int64_t skob, int64_t skoh,
                    int64_t skos, int64_t B, int64_t Hq, int64_t Hk, int64_t S, int64_t D,
                    const int64_t* positions, int64_t spa, int64_t spb, int64_t axes,
                    const int64_t* sections, const float* inv_freq, int64_t rotary_dim,
                    const void* q_weight, const void* k_weight, int weight_dtype, float eps,
                    float scaling, int interleaved, void* stream) {
  if (!dtype_ok(dtype)) return api_error(VA_ERR_ARG, "unknown dtype %d", dtype);
  if (!q || !k || !q_out || !k_out) return api_error(VA_ERR_ARG, "null tensor pointer");
  if (B <= 0 || Hq <= 0 || Hk <= 0 || S <= 0 || D <= 0)
    return api_error(VA_ERR_ARG, "non-positive size");
  if (!fits(B, S, kInt31) || !fits(B * S, Hq + Hk, (int64_t(1) << 26) - 1))
    return api_error(VA_ERR_UNSUPPORTED, "2^26 rows or more in a call");
  va::RopeArgs a{};
  const int rc = set_rotation(a, D, rotary_dim, positions, spa, spb, axes, sections, inv_freq,
                              q_weight, k_weight, dtype, weight_dtype, eps, scaling, interleaved);
  if (rc) return rc;
  a.q = {q, sqb, sqh, sqs, q_out, sqob, sqoh, sqos};
  a.k = {k, skb, skh, sks, k_out, skob, skoh, skos};
  a.B = B;
  a.S = S;
  a.Hq = int(Hq);
  a.Hk = int(Hk);
  return launched(va::launch_rope(dtype, a, static_cast<hipStream_t>(stream)), "rotation launch");
}

int va_qk_norm_rope_to_cache(
    int dtype, const void* q, int64_t sqt, int64_t sqh, const void* k, int64_t skt, int64_t skh,
    const void* v, int64_t svt, int64_t svh, void* q_out, int64_t sqot, int64_t sqoh,
    void* k_cache, int64_t skcp, int64_t skcn, int64_t skch, void* v_cache, int64_t svcp,
    int64_t svcn, int64_t svch, int64_t num_pages, int64_t page_size, const int64_t* slot_mapping,
    int64_t T, int64_t Hq, int64_t Hk, int64_t D, const int64_t* positions, int64_t spa,
    int64_t axes, const int64_t* sections, const float* inv_freq, int64_t rotary_dim,
    const void* q_weight, const void* k_weight, int weight_dtype, float eps, float scaling,
    int interleaved, void* stream) {
  if (!dtype_ok(dtype)) return api_error(VA_ERR_ARG, "unknown dtype %d", dtype);
  if (!q || !k || !v || !q_out || !k_cache || !v_cache || !slot_mapping)
    return api_error(VA_ERR_ARG, "null tensor pointer");
  if (T <= 0 || Hq <= 0 || Hk <= 0 || D <= 0) return api_error(VA_ERR_ARG, "non-positive size");
  if (!fits(T, Hq + 2 * Hk, (int64_t(1) << 26) - 1))
    return api_error(VA_ERR_UNSUPPORTED, "2^26 rows or more in a call");
  if (const int rc = check_pages(num_pages, page_size)) return rc;
  va::RopeArgs a{};
  const int rc = set_rotation(a, D, rotary_dim, positions, spa, 0, axes, sections, inv_freq,
                              q_weight, k_weight, dtype, weight_dtype, eps, scaling, interleaved);
  if (rc) return rc;
  a.q = {q, 0, sqh, sqt, q_out, 0, sqoh, sqot};
  a.k = {k, 0, skh, skt, nullptr, 0, 0, 0};
  a.v = v;
  a.vh = svh;
  a.vs = svt;
  a.kc = k_cache;
  a.vc = v_cache;
  a.kp = skcp;
  a.kn = skcn;
  a.kh = skch;
  a.vp = svcp;
  a.vn = svcn;
  a.vch = svch;
  a.slots = slot_mapping;
  a.num_slots = num_pages * page_size;
  a.page = uint32_t(page_size);
  a.B = 1;
  a.S = T;
  a.Hq = int(Hq);
  a.Hk = int(Hk);
  return launched(va::launch_rope(dtype, a, static_cast<hipStream_t>(stream)),
                  "rotation-to-cache launch");
}

int va_write_paged_kv(int dtype, const void* k, int64_t skt, int64_t skh, const void* v,
                      int64_t svt, int64_t svh, void* k_cache, int64_t skcp, int64_t skcn,
                      int64_t skch, void* v_cache, int64_t svcp, int64_t svcn, int64_t svch,
                      int64_t num_pages, int64_t page_size, const int64_t* slot_mapping, int64_t T,
                      int64_t Hk, int64_t D, void* stream) {
  if (!dtype_ok(dtype)) return api_error(VA_ERR_ARG, "unknown dtype %d", dtype);
  if (!k || !v || !k_cache || !v_cache || !slot_mapping)
    return api_error(VA_ERR_ARG, "null tensor pointer");
  if (T <= 0 || Hk <= 0 || D <= 0) return api_error(VA_ERR_ARG, "non-positive size");
  if (T >= int64_t(1) << 24 || !fits(Hk, D, int64_t(1) << 30))
    return api_error(VA_ERR_UNSUPPORTED, "2^24 tokens or 2^30 values of a token in a call");
  if (const int rc = check_pages(num_pages, page_size)) return rc;
  const va::WriteArgs a{k,    v,    skt,          skh,  svt,
                        svh,  k_cache, v_cache,   skcp, skcn,
                        skch, svcp, svcn,         svch, slot_mapping,
                        num_pages * page_size, uint32_t(page_size), T, int(Hk), int(D)};
  return launched(va::launch_write_kv(dtype, a, static_cast<hipStream_t>(stream)), "write launch");
}

int64_t va_paged_decode_workspace_size(int dtype, int64_t N, int64_t Hq, int64_t Hk, int64_t D,
                                       int64_t M, int64_t page_size) {
  if (!dtype_ok(dtype) || N <= 0 || Hq <= 0 || Hk <= 0 || Hq % Hk || D <= 0 || M < 0 ||
      page_size <= 0 || page_size >= kInt31 || M >= kInt31 || !fits(N, Hq, int64_t(1) << 23))
    return -1;
  va::PagedArgs a{};
  a.N = N;
  a.Hk = Hk;
  a.G = Hq / Hk;
  a.D = D;
  a.M = M;
  a.page = page_size;
  return va::paged_attn_workspace(dtype, a);
}

int va_paged_decode_attn(int dtype, const void* q, int64_t sqn, int64_t sqh, const void* k_cache,
                         int64_t skp, int64_t skn, int64_t skh, const void* v_cache, int64_t svp,
                         int64_t svn, int64_t svh, void* out, int64_t son, int64_t soh,
                         const int32_t* block_tables, int64_t stn, int64_t M,
                         const int32_t* kv_lens, int64_t N, int64_t Hq, int64_t Hk, int64_t D,
                         int64_t page_size, int64_t num_pages, float softmax_scale,
                         void* workspace, int64_t workspace_bytes, void* stream) {
  if (!dtype_ok(dtype)) return api_error(VA_ERR_ARG, "unknown dtype %d", dtype);
  if (!q || !k_cache || !v_cache || !out || !kv_lens || (M && !block_tables))
    return api_error(VA_ERR_ARG, "null tensor pointer");
  if (N <= 0 || Hq <= 0 || Hk <= 0 || D <= 0 || M < 0)
    return api_error(VA_ERR_ARG, "non-positive size");
  if (Hq % Hk) return api_error(VA_ERR_ARG, "num q heads not a multiple of kv heads");
  if (D > 256) return api_error(VA_ERR_UNSUPPORTED, "head_dim %lld > 256", (long long)D);
  if (const int rc = check_pages(num_pages, page_size)) return rc;
  const int64_t need = va_paged_decode_workspace_size(dtype, N, Hq, Hk, D, M, page_size);
  if (need < 0)
    return api_error(VA_ERR_UNSUPPORTED, "2^23 query rows, or 2^31 work units, in a call");
  if (!workspace || workspace_bytes < need)
    return api_error(VA_ERR_WORKSPACE, "paged decode needs %lld workspace bytes", (long long)need);
  if (reinterpret_cast<uintptr_t>(workspace) % 16)
    return api_error(VA_ERR_ARG, "workspace must be 16-byte aligned");
  va::PagedArgs a{};
  a.q = q;
  a.k = k_cache;
  a.v = v_cache;
  a.out = out;
  a.qn = sqn;
  a.qh = sqh;
  a.kp = skp;
  a.kn = skn;
  a.kh = skh;
  a.vp = svp;
  a.vn = svn;
  a.vh = svh;
  a.on = son;
  a.oh = soh;
  a.table = block_tables;
  a.table_stride = stn;
  a.M = M;
  a.lens = kv_lens;
  a.N = N;
  a.Hk = Hk;
  a.G = Hq / Hk;
  a.D = D;
  a.page = page_size;
  a.num_pages = num_pages;
  a.scale_log2 = softmax_scale * 1.4426950408889634f;
  return launched(va::launch_paged_attn(dtype, a, workspace, static_cast<hipStream_t>(stream)),
                  "paged decode launch");
}

}  // extern "C"
