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

static int64_t decode_workspace(int dtype, int64_t N, int64_t Hq, int64_t Hk, int64_t D, int64_t M,
                                int64_t page_size, bool prefix) {
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
  return prefix ? va::prefix_attn_workspace(dtype, a) : va::paged_attn_workspace(dtype, a);
}

int64_t va_paged_decode_workspace_size(int dtype, int64_t N, int64_t Hq, int64_t Hk, int64_t D,
                                       int64_t M, int64_t page_size) {
  return decode_workspace(dtype, N, Hq, Hk, D, M, page_size, false);
}

// Both decode attentions: without prefix_lens and group_rows, the plain one.
static int decode_attn(int dtype, const void* q, int64_t sqn, int64_t sqh, const void* k_cache,
                       int64_t skp, int64_t skn, int64_t skh, const void* v_cache, int64_t svp,
                       int64_t svn, int64_t svh, void* out, int64_t son, int64_t soh,
                       const int32_t* block_tables, int64_t stn, int64_t M,
                       const int32_t* kv_lens, const int32_t* prefix_lens,
                       const int32_t* group_rows, int64_t N, int64_t Hq, int64_t Hk, int64_t D,
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
  const int64_t need =
      decode_workspace(dtype, N, Hq, Hk, D, M, page_size, prefix_lens != nullptr);
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
  a.prefix_lens = prefix_lens;
  a.group_rows = group_rows;
  const auto on = static_cast<hipStream_t>(stream);
  return launched(prefix_lens ? va::launch_prefix_attn(dtype, a, workspace, on)
                              : va::launch_paged_attn(dtype, a, workspace, on),
                  "paged decode launch");
}

int va_paged_decode_attn(int dtype, const void* q, int64_t sqn, int64_t sqh, const void* k_cache,
                         int64_t skp, int64_t skn, int64_t skh, const void* v_cache, int64_t svp,
                         int64_t svn, int64_t svh, void* out, int64_t son, int64_t soh,
                         const int32_t* block_tables, int64_t stn, int64_t M,
                         const int32_t* kv_lens, int64_t N, int64_t Hq, int64_t Hk, int64_t D,
                         int64_t page_size, int64_t num_pages, float softmax_scale,
                         void* workspace, int64_t workspace_bytes, void* stream) {
  return decode_attn(dtype, q, sqn, sqh, k_cache, skp, skn, skh, v_cache, svp, svn, svh, out, son,
                     soh, block_tables, stn, M, kv_lens, nullptr, nullptr, N, Hq, Hk, D,
                     page_size, num_pages, softmax_scale, workspace, workspace_bytes, stream);
}

constexpr int64_t kMostGroups = int64_t(1) << 23;

// Sizes of tables, lists and counts that the kernels take.
static int check_share(int64_t N, int64_t R, int64_t M, int64_t P, int64_t F, int64_t page_size,
                       int64_t stn, int64_t most) {
  if (N < 0 || R < 0 || M < 0 || P < 0 || F < 0) return api_error(VA_ERR_ARG, "negative size");
  if (page_size <= 0 || page_size >= kInt31)
    return api_error(VA_ERR_ARG, "page_size %lld", (long long)page_size);
  if (N > most || R > most)
    return api_error(VA_ERR_UNSUPPORTED, "more than %lld rows", (long long)most);
  if (M >= kInt31 || P >= kInt31 || F >= kInt31)
    return api_error(VA_ERR_UNSUPPORTED, "sizes of 2^31 or more");
  // A work-group for every 1024 entries of a row: a launch takes fewer than 2^32 threads.
  if (!fits(N + R, M / 1024 + 1, kMostGroups))
    return api_error(VA_ERR_UNSUPPORTED, "tables of 2^33 entries or more");
  if (stn < 0) return api_error(VA_ERR_ARG, "negative stride");
  return VA_OK;
}
static int check_workspace(const char* what, const void* workspace, int64_t bytes, int64_t need) {
  if (need && (!workspace || bytes < need))
    return api_error(VA_ERR_WORKSPACE, "%s needs %lld workspace bytes", what, (long long)need);
  if (need && reinterpret_cast<uintptr_t>(workspace) % 16)
    return api_error(VA_ERR_ARG, "workspace must be 16-byte aligned");
  return VA_OK;
}

int64_t va_paged_fork_workspace_size(int64_t R, int64_t num_pages) {
  return R < 0 || num_pages < 0 ? -1 : va::fork_workspace_bytes(R, num_pages);
}

int va_paged_fork(const int32_t* kv_lens, const int32_t* keep_lens, const int32_t* parents,
                  int64_t N, int64_t R, const int32_t* block_tables, int64_t stn, int64_t M,
                  const int32_t* page_shares, int64_t num_pages, const int32_t* free_pages,
                  int64_t num_free, const int32_t* free_head, int64_t page_size,
                  int32_t* kv_lens_out, int32_t* block_tables_out, int32_t* page_shares_out,
                  int32_t* free_pages_out, int32_t* free_head_out, int32_t* copy_src,
                  int32_t* copy_dst, int32_t* copy_rows, void* workspace, int64_t workspace_bytes,
                  void* stream) {
  if (const int rc =
          check_share(N, R, M, num_pages, num_free, page_size, stn, va::kForkMostRows))
    return rc;
  if (!free_head_out || (N && !kv_lens) || (N && M && !block_tables) ||
      (R && (!parents || !kv_lens_out || !copy_src || !copy_dst || !copy_rows)) ||
      (R && M && !block_tables_out) || (num_pages && (!page_shares || !page_shares_out)) ||
      (num_free && (!free_pages || !free_pages_out)))
    return api_error(VA_ERR_ARG, "null pointer");
  const int64_t need = va::fork_workspace_bytes(R, num_pages);
  if (const int rc = check_workspace("the fork", workspace, workspace_bytes, need)) return rc;
  const va::ForkArgs a{kv_lens,          keep_lens,       parents,        block_tables,
                       stn,              N,               R,              M,
                       page_shares,      num_pages,       free_pages,     num_free,
                       free_head,        uint32_t(page_size), kv_lens_out, block_tables_out,
                       page_shares_out,  free_pages_out,  free_head_out,  copy_src,
                       copy_dst,         copy_rows};
  return launched(va::launch_paged_fork(a, workspace, static_cast<hipStream_t>(stream)),
                  "fork launch");
}

int64_t va_paged_compact_workspace_size(int64_t num_pages) {
  return num_pages < 0 ? -1 : va::compact_workspace_bytes(num_pages);
}

int va_paged_compact(const int32_t* kv_lens, int64_t N, const int32_t* block_tables, int64_t stn,
                     int64_t M, const int32_t* page_shares, int64_t num_pages,
                     const int32_t* free_pages, int64_t num_free, const int32_t* free_head,
                     int64_t page_size, int32_t* block_tables_out, int32_t* page_shares_out,
                     int32_t* free_pages_out, int32_t* free_head_out, int32_t* copy_src,
                     int32_t* copy_dst, int32_t* num_moves, void* workspace,
                     int64_t workspace_bytes, void* stream) {
  if (const int rc = check_share(N, 0, M, num_pages, num_free, page_size, stn, kMostGroups))
    return rc;
  if (!free_head_out || !num_moves || (N && !kv_lens) ||
      (N && M && (!block_tables || !block_tables_out)) ||
      (num_pages && (!page_shares || !page_shares_out)) ||
      (num_pages > 1 && (!copy_src || !copy_dst)) ||
      (num_free && (!free_pages || !free_pages_out)))
    return api_error(VA_ERR_ARG, "null pointer");
  const int64_t need = va::compact_workspace_bytes(num_pages);
  if (const int rc = check_workspace("the compaction", workspace, workspace_bytes, need))
    return rc;
  const va::CompactArgs a{kv_lens,    block_tables,  stn,        N,
                          M,          page_shares,   num_pages,  free_pages,
                          num_free,   free_head,     uint32_t(page_size), block_tables_out,
                          page_shares_out, free_pages_out, free_head_out, copy_src,
                          copy_dst,   num_moves};
  return launched(va::launch_paged_compact(a, workspace, static_cast<hipStream_t>(stream)),
                  "compaction launch");
}

int64_t va_paged_prefix_workspace_size(int64_t N) {
  return N < 0 ? -1 : va::prefix_workspace_bytes(N);
}

int va_paged_prefix(const int32_t* kv_lens, int64_t N, const int32_t* block_tables, int64_t stn,
                    int64_t M, const int32_t* group_ids, int64_t page_size, int32_t* prefix_lens,
                    int32_t* group_rows, void* workspace, int64_t workspace_bytes, void* stream) {
  if (const int rc = check_share(N, 0, M, 0, 0, page_size, stn, va::kPrefixMostRows)) return rc;
  if (N == 0) return VA_OK;
  if (!kv_lens || (M && !block_tables) || !prefix_lens || !group_rows)
    return api_error(VA_ERR_ARG, "null pointer");
  const int64_t need = va::prefix_workspace_bytes(N);
  if (const int rc = check_workspace("the prefix", workspace, workspace_bytes, need)) return rc;
  const va::PrefixArgs a{kv_lens, block_tables,        stn,         N,         M,
                         group_ids, uint32_t(page_size), prefix_lens, group_rows};
  return launched(va::launch_paged_prefix(a, workspace, static_cast<hipStream_t>(stream)),
                  "prefix launch");
}

int va_copy_paged_kv(int dtype, void* const* k_caches, void* const* v_caches, int64_t layers,
                     int64_t skp, int64_t skn, int64_t skh, int64_t svp, int64_t svn, int64_t svh,
                     int64_t num_pages, int64_t page_size, int64_t Hk, int64_t D,
                     const int32_t* src_pages, const int32_t* dst_pages, const int32_t* rows,
                     int64_t C, void* stream) {
  if (!dtype_ok(dtype)) return api_error(VA_ERR_ARG, "unknown dtype %d", dtype);
  if (layers < 0 || C < 0 || Hk <= 0 || D <= 0)
    return api_error(VA_ERR_ARG, "non-positive size");
  if (const int rc = check_pages(num_pages, page_size)) return rc;
  for (int64_t s : {skp, skn, skh, svp, svn, svh})
    if (s < 0) return api_error(VA_ERR_ARG, "negative stride");
  if (!fits(Hk, D, kInt31 - 1) || !fits(page_size, Hk * D, kInt31 - 1) || C >= kInt31 ||
      !fits(C, page_size * Hk * D / 2048 + 1, kInt31 - 1))
    return api_error(VA_ERR_UNSUPPORTED, "2^31 values of a page, or pieces, in a call");
  if (layers == 0 || C == 0) return VA_OK;
  if (!k_caches || !v_caches || !src_pages || !dst_pages)
    return api_error(VA_ERR_ARG, "null pointer");
  for (int64_t i = 0; i < layers; ++i)
    if (!k_caches[i] || !v_caches[i]) return api_error(VA_ERR_ARG, "null cache pointer");
  constexpr int64_t kMost = va::kCopyCaches / 2;
  for (int64_t at = 0; at < layers; at += kMost) {
    const int64_t n = layers - at < kMost ? layers - at : kMost;
    va::CopyArgs a{};
    for (int64_t i = 0; i < n; ++i) {
      a.cache[i] = k_caches[at + i];
      a.cache[n + i] = v_caches[at + i];
    }
    a.caches = int32_t(2 * n);
    a.sp[0] = skp, a.sn[0] = skn, a.sh[0] = skh;
    a.sp[1] = svp, a.sn[1] = svn, a.sh[1] = svh;
    a.src = src_pages;
    a.dst = dst_pages;
    a.rows = rows;
    a.C = C;
    a.num_pages = num_pages;
    a.page = int32_t(page_size);
    a.heads = int32_t(Hk);
    a.D = int32_t(D);
    const int rc = launched(va::launch_copy_kv(dtype, a, static_cast<hipStream_t>(stream)),
                            "page copy launch");
    if (rc) return rc;
  }
  return VA_OK;
}

int64_t va_paged_prefix_decode_workspace_size(int dtype, int64_t N, int64_t Hq, int64_t Hk,
                                              int64_t D, int64_t M, int64_t page_size) {
  return decode_workspace(dtype, N, Hq, Hk, D, M, page_size, true);
}

int va_paged_prefix_decode_attn(int dtype, const void* q, int64_t sqn, int64_t sqh,
                                const void* k_cache, int64_t skp, int64_t skn, int64_t skh,
                                const void* v_cache, int64_t svp, int64_t svn, int64_t svh,
                                void* out, int64_t son, int64_t soh, const int32_t* block_tables,
                                int64_t stn, int64_t M, const int32_t* kv_lens,
                                const int32_t* prefix_lens, const int32_t* group_rows, int64_t N,
                                int64_t Hq, int64_t Hk, int64_t D, int64_t page_size,
                                int64_t num_pages, float softmax_scale, void* workspace,
                                int64_t workspace_bytes, void* stream) {
  if (!prefix_lens || !group_rows) return api_error(VA_ERR_ARG, "null pointer");
  return decode_attn(dtype, q, sqn, sqh, k_cache, skp, skn, skh, v_cache, svp, svn, svh, out, son,
                     soh, block_tables, stn, M, kv_lens, prefix_lens, group_rows, N, Hq, Hk, D,
                     page_size, num_pages, softmax_scale, workspace, workspace_bytes, stream);
}

}  // extern "C"
