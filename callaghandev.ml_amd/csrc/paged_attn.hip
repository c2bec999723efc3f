// Attention of a step's new tokens over a paged cache (cdml_paged_attn): the choice of
// kernels and splits, and the join of a request's chunks.  The kernels are in
// paged_attn.inc.h.
#include <algorithm>

#include "paged.h"

namespace cdml {
namespace {

// o = sum_s w_s o_s / sum_s w_s l_s with w_s = 2^(m_s - M) over n chunks, one wave; the
// chunks' statistics lie one to a lane, 64 chunks at a time.
__device__ __forceinline__ void join_chunks(const PagedArgs &a, const float *part, int n, float *o) {
  const int lane = threadIdx.x & 63, stride = a.hd + 2;
  float M = kNoKey;
  for (int c = lane; c < n; c += 64) M = fmaxf(M, part[(size_t)c * stride + a.hd]);
  M = wave_max(M);
  float L = 0.f, acc[4] = {};
  for (int c0 = 0; c0 < n; c0 += 64) {
    const float *p = part + (size_t)c0 * stride;
    const int m = min(n - c0, 64);
    const float w = lane < m ? fast_exp2(p[(size_t)lane * stride + a.hd] - M) : 0.f;
    L += lane < m ? p[(size_t)lane * stride + a.hd + 1] * w : 0.f;
    constexpr int U = 8;  // chunks in flight; past the last one it is read again and left out
    for (int c = 0; c < m; c += U) {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if (lane + 64 * j >= a.hd) continue;
        float x[U];
#pragma unroll
        for (int u = 0; u < U; ++u) x[u] = p[(size_t)min(c + u, m - 1) * stride + lane + 64 * j];
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const float wc = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(w), min(c + u, m - 1)));
          acc[j] = c + u < m ? fmaf(x[u], wc, acc[j]) : acc[j];
        }
      }
    }
  }
  L = wave_sum(L);
#pragma unroll
  for (int j = 0; j < 4; ++j)
    if (lane + 64 * j < a.hd) o[lane + 64 * j] = L == 0.f ? 0.f : acc[j] / L;
}

__device__ __forceinline__ int chunks_seen(int seen, int chunk) { return seen <= 0 ? 0 : (seen - 1) / chunk + 1; }

// New token i of request b, head h, where the request has few rows.
__device__ __forceinline__ void join_few(const PagedArgs &a, int b, int i, int h) {
  const PagedSeq s = paged_seq(a, b);
  if (i >= s.n || s.n * a.group > a.few_rows || s.len <= a.few_chunk) return;
  const int hk = a.by_group.div(h), rr = i * a.group + h - hk * a.group;
  join_chunks(a, a.few_part + (((size_t)b * a.kv_heads + hk) * a.few_rows + rr) * a.few_splits * (a.hd + 2),
              chunks_seen(s.len - s.n + i + 1, a.few_chunk),
              a.o + (size_t)(s.first + i) * a.ldo + (size_t)h * a.hd);
}

// Row `row`, head h, of a request that ran in tiles.
__device__ __forceinline__ void join_tile(const PagedArgs &a, int row, int h) {
  const int lane = threadIdx.x & 63;
  int b = 0;  // requests that end at or before the row
  for (int b0 = 0; b0 < a.batch; b0 += 64) {
    const bool before = b0 + lane < a.batch && a.cu_new[b0 + lane + 1] <= row;
    const int n = __popcll(__builtin_amdgcn_ballot_w64(before));
    b += n;
    if (n < 64) break;
  }
  if (b >= a.batch) return;
  const PagedSeq s = paged_seq(a, b);
  const int i = row - s.first;
  if (i < 0 || i >= s.n || s.n * a.group <= a.few_rows || s.len <= a.tile_chunk) return;
  join_chunks(a, a.tile_part + ((size_t)row * a.heads + h) * a.tile_splits * (a.hd + 2),
              chunks_seen(s.len - s.n + i + 1, a.tile_chunk), a.o + (size_t)row * a.ldo + (size_t)h * a.hd);
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

// Which kernels run and how keys are split, from the sizes alone.
struct Plan {
  PagedKernels kernels;
  int few_rows, few_chunk, few_splits, tile_chunk, tile_splits;
  size_t few_floats, tile_floats;
};

// Most rows a K/V head on the vector units: there a cached value is multiplied once for
// every row, which 16-bit caches outrun first.  64 x 4096 keys, 4 rows, fp32 687 us against
// 795 by paged_span_kernel, fp16 447 against 429; 2 rows, bf16 183 against 216.
constexpr int kVecRows = 4, kVecRows16 = 2;
constexpr int kSpanRows = 16;  // most rows a K/V head of an MFMA operand
constexpr int kComputeUnits = 256;

int check_sizes(const char *what, int rows, int batch, int max_new, int max_len, int heads, int kv_heads, int hd) {
  if (rows < 0 || batch < 0 || batch > kPagedMaxBatch || max_new < 0 || max_len < 0)
    return fail(CDML_E_INVALID, "%s: bad size (rows %d, batch %d of at most %d, max_new %d, max_len %d)", what, rows,
                batch, kPagedMaxBatch, max_new, max_len);
  if (heads <= 0 || kv_heads <= 0 || heads % kv_heads || hd <= 0 || hd > 256)
    return fail(CDML_E_INVALID, "%s: bad heads (%d over %d K/V heads, head_dim %d of at most 256)", what, heads,
                kv_heads, hd);
  const long long group = heads / kv_heads;
  // the grids' limits (a launch has less than 2^32 threads along x, 2^24 workgroups of tiles),
  // and room for key numbers past the last tile
  const long long most = max_new * group;
  const long long groups = hd <= 128 ? 1 : (most + kVecRows - 1) / kVecRows;
  if (most > INT_MAX / 2 || max_len > INT_MAX / 2 || heads > 65535 || groups * kv_heads > 65535 ||
      (long long)kv_heads * hd > INT_MAX / 4 ||
      (hd <= 128 && most > kSpanRows && ((long long)rows * group / kPagedTileRows + batch) * kv_heads >= 1 << 24))
    return fail(CDML_E_INVALID, "%s: problem too large", what);
  return CDML_OK;
}

int round_up(int n, int m) { return (int)(((long long)n + m - 1) / m * m); }

Plan make_plan(int size, int rows, int batch, int max_new, int max_len, int heads, int kv_heads, int hd) {
  Plan p{};
  const int group = heads / kv_heads, most = max_new * group, len = max_len < 1 ? 1 : max_len;
  PagedKernels &k = p.kernels;
  k.tile = hd <= 128 && most > kSpanRows;
  k.rows = size > 1 && (hd > 128 || most <= (size == 4 ? kVecRows : kVecRows16));
  k.span = !k.rows && (!k.tile || group <= kSpanRows);
  p.few_rows = most < 1 ? 1 : k.tile ? kSpanRows : most;
  const long long pairs = (long long)(batch < 1 ? 1 : batch) * kv_heads;
  const long long groups = k.rows ? (p.few_rows + kVecRows - 1) / kVecRows : (p.few_rows + kSpanRows - 1) / kSpanRows;
  if (k.span) {
    // a whole request to a workgroup where these fill the CUs (16 x 16 pairs of 4096 bf16 keys:
    // 48.5 us, 55.3 in two chunks, 96 in chunks of 512), else two workgroups for every CU
    const long long many = pairs * groups;
    long long splits = many >= kComputeUnits ? 1 : (2 * kComputeUnits + many - 1) / many;
    if (splits > (len + 255) / 256) splits = (len + 255) / 256;
    p.few_chunk = round_up((int)((len + splits - 1) / splits), 128);
  } else if (groups > 2) {
    p.few_chunk = round_up(len, kPagedSub);  // rows without number (head dims above 128) are not split
  } else {
    // One chunk, which needs no join, up to 512 keys, or up to 1024 where requests and heads
    // fill the CUs: 16 heads of 64, bf16, 64 x 500 keys 25.7 us, 30.4 in chunks of 256; 4 x
    // 1000 keys 13.8 in one, 9.6 in 256s; 64 x 1000 keys 49.8 in one, 55.0.  Else 256 keys, or
    // 512 of fp32 where that leaves four workgroups for every CU: 16 heads of 128, fp32, 64 x
    // 8000 keys 1248 us, 1286 in 256s, but 1 x 2000 keys 15.8, 12.8 in 256s; 16 heads of 64,
    // bf16, 64 x 2000 keys 103.6, 91.5 in 256s.
    const long long wide = (long long)((len - 1) / 512 + 1) * pairs * groups;
    const bool one = len <= 512 || (len <= 1024 && pairs * groups >= kComputeUnits);
    p.few_chunk = one ? round_up(len, 256) : size == 4 && wide >= 4 * kComputeUnits ? 512 : 256;
  }
  p.few_splits = (len - 1) / p.few_chunk + 1;
  if ((k.rows || k.span) && p.few_splits > 1)
    p.few_floats = (size_t)batch * kv_heads * p.few_rows * p.few_splits * (hd + 2);
  // Matrix cores: keys are split where the tiles alone leave CUs without work, to two
  // workgroups for every CU.  16 heads of 64, bf16: 256 tokens over 8192 keys 59 us, 62
  // with twice the splits, 260 with none; 4 x 512 over 4096 152, 159, 160.
  // Pieces of 256 keys at least, or of 128 where those leave half the CUs without work: 5
  // heads of 96, fp32, 30 tokens over 500 keys 36.9 us, 26.2 so; 7 heads over 1 of 128 over 4000
  // 44.7, 36.9; but 16 over 2 of 40, fp16, 120 tokens over 4000 (256 workgroups) 29.2, 32.7.
  p.tile_chunk = INT_MAX;
  p.tile_splits = 1;
  if (k.tile) {
    const long long tiles = ((long long)rows * group / kPagedTileRows + batch) * kv_heads;
    long long splits = (2 * kComputeUnits + tiles - 1) / (tiles < 1 ? 1 : tiles);
    long long pieces = (len + 255) / 256;
    if (pieces > 1 && tiles * pieces < kComputeUnits / 2) pieces = (len + 127) / 128;
    if (splits > pieces) splits = pieces;
    if (splits > 1) {
      p.tile_chunk = round_up((int)((len + splits - 1) / splits), 64);
      p.tile_splits = (len - 1) / p.tile_chunk + 1;
      if (p.tile_splits > 1) p.tile_floats = (size_t)rows * heads * p.tile_splits * (hd + 2);
    }
  }
  return p;
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

int attention(const char *what, bool q8, const float *q, int ldq, const void *kcache, const void *vcache,
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
  if ((long long)max_len > (long long)max_blocks * page_size)
    return fail(CDML_E_INVALID, "%s: max_len %d above the table's %lld tokens", what, max_len,
                (long long)max_blocks * page_size);
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
  size_t need = 0;
  rc = workspace_size(what, q8, rows, batch, max_new, max_len, num_heads, num_kv_heads, head_dim, &need);
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
  a.max_len = max_len;
  a.heads = num_heads;
  a.kv_heads = num_kv_heads;
  a.group = num_heads / num_kv_heads;
  a.hd = head_dim;
  a.scale_log2 = scale * kLog2e;
  a.by_group = UDiv::make((uint32_t)a.group);
  a.few_rows = p.few_rows;
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

}  // namespace
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
  return attention("cdml_paged_attn", false, q, ldq, kcache, vcache, nullptr, nullptr, cache_type, n_pages, page_size,
                   block_table, max_blocks, kv_len, cu_new, o, ldo, rows, batch, max_new, max_len, num_heads,
                   num_kv_heads, head_dim, scale, bad, workspace, workspace_bytes, stream);
}

extern "C" int cdml_paged_attn_q8(const float *q, int ldq, const void *kcache, const void *vcache, const float *kscale,
                                  const float *vscale, int cache_type, int n_pages, int page_size,
                                  const int *block_table, int max_blocks, const int *kv_len, const int *cu_new,
                                  float *o, int ldo, int rows, int batch, int max_new, int max_len, int num_heads,
                                  int num_kv_heads, int head_dim, float scale, int *bad, void *workspace,
                                  size_t workspace_bytes, cdml_stream stream) {
  return attention("cdml_paged_attn_q8", true, q, ldq, kcache, vcache, kscale, vscale, cache_type, n_pages, page_size,
                   block_table, max_blocks, kv_len, cu_new, o, ldo, rows, batch, max_new, max_len, num_heads,
                   num_kv_heads, head_dim, scale, bad, workspace, workspace_bytes, stream);
}
