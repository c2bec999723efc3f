// Attention of a step's new tokens over a paged cache (cdml_paged_attn, cdml_paged_attn_q8):
// the launches and the join of a request's chunks.  The kernels are in paged_attn.inc.h and
// paged_attn_q8.inc.h, the choice between them in paged_plan.h.
#include <algorithm>

#include "paged_plan.h"

namespace cdml {
namespace {

// New token i of request b, head h, where the request has few rows.
__device__ __forceinline__ void join_few(const PagedArgs &a, int b, int i, int h) {
  const PagedSeq s = paged_seq(a, b);
  if (i >= s.n || s.n * a.group > a.few_rows || s.len <= a.few_chunk) return;
  const int hk = a.by_group.div(h), rr = i * a.group + h - hk * a.group;
  const float *part = a.few_part + (((size_t)b * a.kv_heads + hk) * a.few_rows + rr) * a.few_splits * (a.hd + 2);
  const Chunks chunks[1] = {{part, part + a.hd, chunks_seen(s.len - s.n + i + 1, a.few_chunk), a.hd + 2, a.hd + 2}};
  join_chunks(a.hd, chunks, a.o + (size_t)(s.first + i) * a.ldo + (size_t)h * a.hd);
}

// Row `row`, head h, of a request that ran in tiles.
__device__ __forceinline__ void join_tile(const PagedArgs &a, int row, int h) {
  const int b = request_of_row(a, row);
  if (b >= a.batch) return;
  const PagedSeq s = paged_seq(a, b);
  const int i = row - s.first;
  if (i < 0 || i >= s.n || s.n * a.group <= a.few_rows || s.len <= a.tile_chunk) return;
  const float *part = a.tile_part + ((size_t)row * a.heads + h) * a.tile_splits * (a.hd + 2);
  const Chunks chunks[1] = {{part, part + a.hd, chunks_seen(s.len - s.n + i + 1, a.tile_chunk), a.hd + 2, a.hd + 2}};
  join_chunks(a.hd, chunks, a.o + (size_t)row * a.ldo + (size_t)h * a.hd);
}

// A wave per (new token, head): the first few_tokens * batch workgroups for the requests of few
// rows, the others, one a row, for those that ran in tiles.  One launch for both: 30 tokens over
// 4000 keys, 16 heads over 2 of 40, fp16 take 21.2 us, 1.7 more with two.
__global__ void __launch_bounds__(256) paged_join_kernel(const PagedArgs a, int few_tokens) {
  const int h = blockIdx.y * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if (h >= a.heads) return;
  const unsigned few = (unsigned)few_tokens * a.batch;
  if (blockIdx.x < few) join_few(a, blockIdx.x / few_tokens, blockIdx.x % few_tokens, h);
  else join_tile(a, (int)(blockIdx.x - few), h);
}

int workspace_size(const char *what, bool q8, int rows, int batch, int max_new, int max_len, int num_heads,
                   int num_kv_heads, int head_dim, size_t *bytes) {
  if (!bytes) return fail(CDML_E_INVALID, "%s: bytes is NULL", what);
  int rc = check_sizes(what, rows, batch, max_new, max_len, num_heads, num_kv_heads, head_dim);
  if (rc) return rc;
  size_t most = 0;
  for (int size = q8 ? 1 : 2; size <= (q8 ? 1 : 4); size *= 2) {  // of any size of cached values
    const Plan p = make_plan(size, rows, batch, max_new, max_len, num_heads, num_kv_heads, head_dim);
    most = std::max(most, p.few_floats + p.tile_floats);
  }
  *bytes = sizeof(float) * most;
  return CDML_OK;
}

}  // namespace

int paged_attention(const char *what, bool q8, bool shared, const float *q, int ldq, const void *kcache, const void *vcache,
              const float *kscale, const float *vscale, int cache_type, int n_pages, int page_size,
              const int *block_table, int max_blocks, const int *kv_len, const int *cu_new, float *o, int ldo, int rows,
              int batch, int max_new, int max_len, int num_heads, int num_kv_heads, int head_dim, float scale, int *bad,
              void *workspace, size_t workspace_bytes, cdml_stream stream) {
  PagedArgs a{};
  int rc = check_pool(what, n_pages, page_size, max_blocks, batch, &a.page_shift);
  if (rc) return rc;
  rc = check_sizes(what, rows, batch, max_new, max_len, num_heads, num_kv_heads, head_dim);
  if (rc) return rc;
  const int size = q8 ? (int)q8_cache_type(cache_type) : cache_type_bytes(cache_type);
  if (!size) return fail(CDML_E_INVALID, "%s: unknown cache type %d", what, cache_type);
  const long long table = (long long)max_blocks * page_size;
  if (!shared && max_len > table)
    return fail(CDML_E_INVALID, "%s: max_len %d above the table's %lld tokens", what, max_len, table);
  const long long dim = (long long)num_heads * head_dim;
  if (ldq < dim || ldo < dim) return fail(CDML_E_INVALID, "%s: row stride smaller than the heads", what);
  if (rows == 0 || batch == 0 || max_new == 0) return CDML_OK;
  if (!q || !kcache || !vcache || !block_table || !kv_len || !cu_new || !o)
    return fail(CDML_E_INVALID, "%s: NULL pointer", what);
  if (q8) {
    rc = check_q8(what, kcache, vcache, kscale, vscale);
    if (rc) return rc;
  }
  const Plan p = make_plan(size, rows, batch, max_new, max_len, num_heads, num_kv_heads, head_dim);
  // (shared: that entry's size covers the plans of the types that run plain, and has been checked)
  size_t need = sizeof(float) * (p.few_floats + p.tile_floats);
  if (!shared) rc = workspace_size(what, q8, rows, batch, max_new, max_len, num_heads, num_kv_heads, head_dim, &need);
  if (rc) return rc;
  if (need && (!workspace || workspace_bytes < need || !aligned16(workspace)))
    return fail(CDML_E_INVALID, "%s: %zu bytes of 16-byte aligned workspace needed, %zu given", what, need,
                workspace_bytes);
  rc = ensure_device();
  if (rc) return rc;
  a.q = q;
  a.kc = kcache;
  a.vc = vcache;
  a.ks = kscale;
  a.vs = vscale;
  a.width = q8_width(head_dim);
  a.table = block_table;
  a.kv_len = kv_len;
  a.cu_new = cu_new;
  a.o = o;
  a.bad = bad;
  a.ldq = ldq;
  a.ldo = ldo;
  a.n_pages = n_pages;
  a.max_blocks = max_blocks;
  a.rows = rows;
  a.batch = batch;
  a.max_new = max_new;
  a.max_len = (int)std::min<long long>(max_len, table);
  a.heads = num_heads;
  a.kv_heads = num_kv_heads;
  a.group = num_heads / num_kv_heads;
  a.hd = head_dim;
  a.scale_log2 = scale * kLog2e;
  a.by_group = UDiv::make((uint32_t)a.group);
  a.few_rows = a.most_rows = p.few_rows;
  a.few_chunk = p.few_chunk;
  a.few_splits = p.few_splits;
  a.tile_chunk = p.tile_chunk;
  a.tile_splits = p.tile_splits;
  a.few_part = static_cast<float *>(workspace);
  a.tile_part = a.few_part + p.few_floats;
  const bool wide = head_dim % 8 == 0 && ldq % 4 == 0 && ldo % 4 == 0 && aligned16(q) && aligned16(o) &&
                    aligned16(kcache) && aligned16(vcache);
  const hipStream_t st = as_hip(stream);
  switch (cache_type) {
    case CDML_CACHE_F32: rc = paged_attn_f32(a, p.kernels, wide, st); break;
    case CDML_CACHE_F16: rc = paged_attn_f16(a, p.kernels, wide, st); break;
    case CDML_CACHE_BF16: rc = paged_attn_bf16(a, p.kernels, wide, st); break;
    case CDML_CACHE_I8: rc = paged_attn_i8(a, p.kernels, wide, st); break;
    default: rc = paged_attn_f8(a, p.kernels, wide, st);
  }
  if (rc) return rc;
  if (!p.few_floats && !p.tile_floats) return CDML_OK;
  const int few_tokens = p.few_floats ? p.few_rows / a.group : 0;  // of a request of few rows, at most
  const unsigned joins = (unsigned)batch * few_tokens + (p.tile_floats ? (unsigned)rows : 0u);
  paged_join_kernel<<<dim3(joins, (unsigned)(num_heads + 3) / 4), 256, 0, st>>>(a, few_tokens);
  return check_launch("paged_join_kernel");
}

}  // namespace cdml

using namespace cdml;

extern "C" int cdml_paged_attn_workspace_size(int rows, int batch, int max_new, int max_len, int num_heads,
                                              int num_kv_heads, int head_dim, size_t *bytes) {
  return workspace_size("cdml_paged_attn_workspace_size", false, rows, batch, max_new, max_len, num_heads, num_kv_heads,
                        head_dim, bytes);
}

extern "C" int cdml_paged_attn_q8_workspace_size(int rows, int batch, int max_new, int max_len, int num_heads,
                                                 int num_kv_heads, int head_dim, size_t *bytes) {
  return workspace_size("cdml_paged_attn_q8_workspace_size", true, rows, batch, max_new, max_len, num_heads,
                        num_kv_heads, head_dim, bytes);
}

extern "C" int cdml_paged_attn(const float *q, int ldq, const void *kcache, const void *vcache, int cache_type,
                               int n_pages, int page_size, const int *block_table, int max_blocks, const int *kv_len,
                               const int *cu_new, float *o, int ldo, int rows, int batch, int max_new, int max_len,
                               int num_heads, int num_kv_heads, int head_dim, float scale, int *bad, void *workspace,
                               size_t workspace_bytes, cdml_stream stream) {
  return paged_attention("cdml_paged_attn", false, false, q, ldq, kcache, vcache, nullptr, nullptr, cache_type, n_pages, page_size,
                   block_table, max_blocks, kv_len, cu_new, o, ldo, rows, batch, max_new, max_len, num_heads,
                   num_kv_heads, head_dim, scale, bad, workspace, workspace_bytes, stream);
}

extern "C" int cdml_paged_attn_q8(const float *q, int ldq, const void *kcache, const void *vcache, const float *kscale,
                                  const float *vscale, int cache_type, int n_pages, int page_size,
                                  const int *block_table, int max_blocks, const int *kv_len, const int *cu_new,
                                  float *o, int ldo, int rows, int batch, int max_new, int max_len, int num_heads,
                                  int num_kv_heads, int head_dim, float scale, int *bad, void *workspace,
                                  size_t workspace_bytes, cdml_stream stream) {
  return paged_attention("cdml_paged_attn_q8", true, false, q, ldq, kcache, vcache, kscale, vscale, cache_type, n_pages, page_size,
                   block_table, max_blocks, kv_len, cu_new, o, ldo, rows, batch, max_new, max_len, num_heads,
                   num_kv_heads, head_dim, scale, bad, workspace, workspace_bytes, stream);
}
