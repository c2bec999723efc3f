// Attention for requests that share their first pages (include/cdml.h): what a group shares is
// found in its tables, read once for all its rows, and joined with each request's own tokens.
#include <algorithm>

#include "paged_plan.h"

namespace cdml {
namespace {

constexpr int kFindThreads = 1024;

struct FindArgs {
  const int *table;
  int max_blocks;
  const int *kv_len, *cu, *group_start;
  int groups, batch, n_pages, page_shift;
  int *shared;
};

__device__ __forceinline__ int clamped(int x, int most) { return min(max(x, 0), most); }

// One workgroup a group: the least number of full old pages of a member, and the first column
// of the tables in which a member's page differs from the first member's.  A wave takes every
// sixteenth member, a lane every 64th column; the first 512 columns are read before it is known
// how many count, so that both answers come in one wait.  The last workgroup clears the
// requests of no group.
__global__ void __launch_bounds__(kFindThreads) paged_shared_kernel(const FindArgs a) {
  __shared__ int least;
  const int g = blockIdx.x, t = threadIdx.x, lane = t & 63, wave = __builtin_amdgcn_readfirstlane(t >> 6);
  if (g == a.groups) {
    const int from = a.groups ? clamped(a.group_start[0], a.batch) : a.batch;
    const int behind = a.groups ? clamped(a.group_start[a.groups], a.batch) : 0;
    for (int b = t; b < a.batch; b += kFindThreads)
      if (b < from || b >= behind) a.shared[b] = 0;
    return;
  }
  const int first = clamped(a.group_start[g], a.batch);
  const int members = min(max(a.group_start[g + 1], first), a.batch) - first;
  if (members < 2) {
    if (members == 1 && t == 0) a.shared[first] = 0;
    return;
  }
  const int *lead = a.table + (size_t)first * a.max_blocks;
  constexpr int WAVES = kFindThreads / 64, K = 8, U = 4;  // columns of a lane, members of a wave at a time
  // the first of columns [c0, c0 + 512) below `columns` that differs, of this lane's
  auto compare = [&](int c0, int columns) {
    int x[K], differs = INT_MAX;
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int c = c0 + 64 * k + lane;
      x[k] = c < columns ? lead[c] : 0;
    }
    for (int m = wave; m < members; m += WAVES * U) {
      int y[U][K];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int *row = lead + (size_t)min(m + WAVES * u, members - 1) * a.max_blocks;
#pragma unroll
        for (int k = 0; k < K; ++k) {
          const int c = c0 + 64 * k + lane;
          y[u][k] = c < columns ? row[c] : 0;
        }
      }
#pragma unroll
      for (int k = K - 1; k >= 0; --k) {
        bool same = (unsigned)x[k] < (unsigned)a.n_pages;
#pragma unroll
        for (int u = 0; u < U; ++u) same &= x[k] == y[u][k];
        const int c = c0 + 64 * k + lane;
        if (!same && c < columns) differs = min(differs, c);
      }
    }
    return differs;
  };
  if (t == 0) least = a.max_blocks;
  int pages = a.max_blocks;
  for (int b = first + t; b < first + members; b += kFindThreads) {
    const long long old = (long long)a.kv_len[b] - max(a.cu[b + 1] - a.cu[b], 0);
    pages = min(pages, (int)min(max(old, 0LL) >> a.page_shift, (long long)a.max_blocks));
  }
  pages = wave_min(min(pages, compare(0, a.max_blocks)));
  __syncthreads();
  if (lane == 0) atomicMin(&least, pages);
  __syncthreads();
  for (int c0 = 64 * K; c0 < least; c0 += 64 * K) {
    const int differs = wave_min(compare(c0, least));
    __syncthreads();
    if (lane == 0) atomicMin(&least, differs);
    __syncthreads();
  }
  const int tokens = least << a.page_shift;  // (at most a table's tokens)
  for (int b = first + t; b < first + members; b += kFindThreads) a.shared[b] = tokens;
}

// A wave per (row, head); not for rows that the fused kernel wrote.
__global__ void __launch_bounds__(256) paged_shared_join_kernel(const PagedArgs a) {
  const int row = blockIdx.x, h = blockIdx.y * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if (h >= a.heads) return;
  const int b = request_of_row(a, row);
  if (b >= a.batch) return;
  const PagedSeq s = paged_seq<true>(a, b);
  const int i = row - s.first;
  const bool few = s.n * a.group <= a.few_rows;
  if (i < 0 || i >= s.n || (few && a.fused)) return;
  const size_t at = ((size_t)row * a.heads + h) * a.part_splits, own = at + a.prefix_splits;
  const Chunks chunks[2] = {
      {a.part + at * a.part_width, a.part_stats + at * 2,
       min(chunks_seen(s.start, a.prefix_chunk), a.prefix_splits), a.part_width, 2},
      {a.part + own * a.part_width, a.part_stats + own * 2,
       min(chunks_seen(s.len - s.n + i + 1 - s.start, few ? a.few_chunk : a.tile_chunk),
           few ? a.few_splits : a.tile_splits),
       a.part_width, 2}};
  join_chunks(a.hd, chunks, a.o + (size_t)row * a.ldo + (size_t)h * a.hd);
}

struct SharedPlan {
  bool plain;          // every request reads its own pages
  bool prefix_tile;
  int prefix_rows;     // of a group, at most
  int prefix_chunk, prefix_splits;
  Plan own;
  int own_splits;
  bool fused;          // of the requests of few rows
  bool lone_waves;     // of them, too: a wave to a K/V head
  size_t parts, floats;
};

// Whether reading what the groups share once, in a launch of its own whose sums have to be joined,
// takes less time than every request's reading of its own pages, from the sizes alone (us):
//   requests of few rows read at 6 TB/s, in tiles a CU takes `tile` us for 32 keys of 128 rows,
//   0.6 of that where a wave or two have rows;
//   the launch and the joins take 12 us.
// 64 requests behind 8192 tokens, 32 heads over 8 of 128, bf16: 70 us, 199 by cdml_paged_attn;
// 105 requests in 5 groups behind 4102, 27 new tokens, 8 heads of 64, bf16: 115, 193; but 264 in 6
// behind 109, 27 new, one head of 96: 50 and 25; 26 in 2 behind 881, 7 heads over 1 of 128, fp32:
// 49 and 25.
bool worth_sharing(int size, int batch, int groups, int max_members, int max_new, int max_prefix, int group,
                   int kv_heads, int hd) {
  const double tile = (hd <= 32 ? 0.5 : hd <= 64 ? 0.85 : 1.5) * (size == 4 ? 1.8 : 1);
  auto us = [&](double readers, double rows) {
    const double keys = readers * kv_heads * max_prefix;
    if (rows <= kSpanRows) return keys * 2 * hd * size / 6e6;
    const double tiles = (double)(long long)((rows + kPagedTileRows - 1) / kPagedTileRows);
    return keys / 32 * tiles * tile * (rows <= kPagedTileRows / 2 ? 0.6 : 1) / kComputeUnits;
  };
  const double rows = (double)max_new * group;
  return us(batch, rows) - us(groups, rows * max_members) > 12;
}

SharedPlan plan_shared(int size, int rows, int batch, int groups, int max_members, int max_new, int max_prefix,
                       int max_tail, int heads, int kv_heads, int hd) {
  SharedPlan p{};
  p.plain = hd > 128 || groups == 0 || max_members < 2 || max_prefix == 0 ||
            !worth_sharing(size, batch, groups, max_members, max_new, max_prefix, heads / kv_heads, kv_heads, hd);
  if (p.plain) {
    p.own = make_plan(size, rows, batch, max_new, max_prefix + max_tail, heads, kv_heads, hd);
    p.floats = p.own.few_floats + p.own.tile_floats;
    return p;
  }
  const int group = heads / kv_heads;
  const long long most = std::min((long long)max_members * max_new, (long long)rows) * group;
  p.prefix_tile = most > kSpanRows;
  p.prefix_rows = (int)std::min<long long>(most, INT_MAX);
  // The split of the shared tokens that takes the least time: `unit` keys take as long as any
  // others, `start` of them a workgroup's beginning and end; a turn of `slots` workgroups more
  // takes 0.7 of the first.  64 requests behind 8192 tokens, 32 heads over 8 of 128, bf16 (16 tiles): 16
  // splits 40 us, 22 (two workgroups on some CUs, one on the others) 45, 32 37, but with
  // twice the parts to join; 16 x 8 beams behind 2048, i8 (256 spans): one split 37.9 us with
  // the joins, two 36.3, four 41.5.
  const long long all = (long long)rows * group;
  const long long tiles = groups * std::max<long long>(1, (all / groups + kPagedTileRows / 2) / kPagedTileRows);
  const long long work = (p.prefix_tile ? tiles : groups) * kv_heads;
  const int unit = p.prefix_tile ? 32 : 128, start = p.prefix_tile ? 6 : 4;
  const int slots = p.prefix_tile ? kComputeUnits : 2 * kComputeUnits;
  long long splits = 1, least = LLONG_MAX;
  for (long long n = 1; n <= (max_prefix + 255) / 256 && n * work <= 4 * slots + work; ++n) {
    const long long turns = (n * work + slots - 1) / slots;
    const long long cost = (3 + 7 * turns) * ((max_prefix + n * unit - 1) / (n * unit) + start);
    if (cost < least) {
      least = cost;
      splits = n;
    }
  }
  p.prefix_chunk = round_up((int)((max_prefix + splits - 1) / splits), 128);
  p.prefix_splits = (max_prefix - 1) / p.prefix_chunk + 1;
  p.own = make_plan(size, rows, batch, max_new, max_tail, heads, kv_heads, hd, true);
  p.own_splits = std::max(p.own.kernels.span ? p.own.few_splits : 1, p.own.kernels.tile ? p.own.tile_splits : 1);
  p.fused = p.own.kernels.span && p.own.few_splits == 1;
  // Where requests and heads fill the SIMDs without a split, four waves on a few keys wait for each
  // other longer than they read: 16 x 8 beams of 16 heads, up to 100 tokens of their own, i8, 51.3
  // us with four, 38.1 with one; but 64 requests of 8 heads, up to 500, bf16, 78.3 and 96.5.  Over 144
  // calls (i8 and bf16, head dims 64 and 128, 256 to 8192 pairs, tails of up to 8 to 500 tokens
  // behind 2048) the 88 that have one wave take 3 to 49% less so; of the others, tails of up to
  // 500 of 1024 pairs would take 2 to 9% less with one, all else longer.
  const long long pairs = (long long)batch * kv_heads;
  p.lone_waves = p.fused && pairs >= 4 * kComputeUnits && 4LL * max_tail <= pairs;
  p.parts = (size_t)rows * heads * (p.prefix_splits + p.own_splits);
  p.floats = p.parts * (round_up(hd, 4) + 2);
  return p;
}

int check_shared(const char *what, int rows, int batch, int groups, int max_members, int max_new, int max_prefix,
                 int max_tail, int heads, int kv_heads, int hd) {
  if (groups < 0 || groups > batch || max_members < 0 || max_prefix < 0 || max_tail < 0 ||
      (long long)max_prefix + max_tail > INT_MAX / 2)
    return fail(CDML_E_INVALID, "%s: bad size (batch %d, groups %d, max_members %d, max_prefix %d, max_tail %d)", what,
                batch, groups, max_members, max_prefix, max_tail);
  const int rc = check_sizes(what, rows, batch, max_new, max_prefix + max_tail, heads, kv_heads, hd);
  if (rc) return rc;
  // (a group's rows run in tiles where a request's do not; a workgroup of the join to a row)
  if (((long long)rows * (heads / kv_heads) / kPagedTileRows + batch) * kv_heads >= 1 << 24 ||
      rows >= 1 << 24 ||
      (long long)rows * (heads / kv_heads) > INT_MAX / 2)
    return fail(CDML_E_INVALID, "%s: problem too large", what);
  return CDML_OK;
}

}  // namespace
}  // namespace cdml

using namespace cdml;

extern "C" int cdml_paged_shared(const int *block_table, int max_blocks, const int *kv_len, const int *cu_new,
                                 const int *group_start, int groups, int batch, int n_pages, int page_size, int *shared,
                                 cdml_stream stream) {
  FindArgs a{};
  int rc = check_pool("cdml_paged_shared", n_pages, page_size, max_blocks, batch, &a.page_shift);
  if (rc) return rc;
  if (groups < 0 || groups > batch)
    return fail(CDML_E_INVALID, "cdml_paged_shared: %d groups of %d requests", groups, batch);
  if (batch == 0) return CDML_OK;
  if (!block_table || !kv_len || !cu_new || !group_start || !shared)
    return fail(CDML_E_INVALID, "cdml_paged_shared: NULL pointer");
  rc = ensure_device();
  if (rc) return rc;
  a.table = block_table;
  a.max_blocks = max_blocks;
  a.kv_len = kv_len;
  a.cu = cu_new;
  a.group_start = group_start;
  a.groups = groups;
  a.batch = batch;
  a.n_pages = n_pages;
  a.shared = shared;
  paged_shared_kernel<<<groups + 1, kFindThreads, 0, as_hip(stream)>>>(a);
  return check_launch("paged_shared_kernel");
}

extern "C" int cdml_paged_attn_shared_workspace_size(int rows, int batch, int groups, int max_members, int max_new,
                                                     int max_prefix, int max_tail, int num_heads, int num_kv_heads,
                                                     int head_dim, size_t *bytes) {
  const char *what = "cdml_paged_attn_shared_workspace_size";
  if (!bytes) return fail(CDML_E_INVALID, "%s: bytes is NULL", what);
  const int rc = check_shared(what, rows, batch, groups, max_members, max_new, max_prefix, max_tail, num_heads,
                              num_kv_heads, head_dim);
  if (rc) return rc;
  size_t most = 0;
  for (int size = 1; size <= 4; size *= 2)  // of any size of cached values
    most = std::max(most, plan_shared(size, rows, batch, groups, max_members, max_new, max_prefix, max_tail, num_heads,
                                      num_kv_heads, head_dim)
                              .floats);
  *bytes = sizeof(float) * most;
  return CDML_OK;
}

extern "C" int cdml_paged_attn_shared(const float *q, int ldq, const void *kcache, const void *vcache,
                                      const float *kscale, const float *vscale, int cache_type, int n_pages,
                                      int page_size, const int *block_table, int max_blocks, const int *kv_len,
                                      const int *cu_new, const int *group_start, const int *shared, float *o, int ldo,
                                      int rows, int batch, int groups, int max_members, int max_new, int max_prefix,
                                      int max_tail, int num_heads, int num_kv_heads, int head_dim, float scale, int *bad,
                                      void *workspace, size_t workspace_bytes, cdml_stream stream) {
  const char *what = "cdml_paged_attn_shared";
  PagedArgs a{};
  int rc = check_pool(what, n_pages, page_size, max_blocks, batch, &a.page_shift);
  if (rc) return rc;
  rc = check_shared(what, rows, batch, groups, max_members, max_new, max_prefix, max_tail, num_heads, num_kv_heads,
                    head_dim);
  if (rc) return rc;
  const bool q8 = q8_cache_type(cache_type);
  const int size = q8 ? 1 : cache_type_bytes(cache_type), max_len = max_prefix + max_tail;
  if (!size) return fail(CDML_E_INVALID, "%s: unknown cache type %d", what, cache_type);
  const long long table = (long long)max_blocks * page_size;
  if (max_prefix > table || max_tail > table)
    return fail(CDML_E_INVALID, "%s: max_prefix %d or max_tail %d above the table's %lld tokens", what, max_prefix,
                max_tail, table);
  const long long dim = (long long)num_heads * head_dim;
  if (ldq < dim || ldo < dim) return fail(CDML_E_INVALID, "%s: row stride smaller than the heads", what);
  if (rows == 0 || batch == 0 || max_new == 0) return CDML_OK;
  if (!q || !kcache || !vcache || !block_table || !kv_len || !cu_new || !group_start || !shared || !o)
    return fail(CDML_E_INVALID, "%s: NULL pointer", what);
  if (q8) {
    rc = check_q8(what, kcache, vcache, kscale, vscale);
    if (rc) return rc;
  }
  size_t need = 0;
  rc = cdml_paged_attn_shared_workspace_size(rows, batch, groups, max_members, max_new, max_prefix, max_tail, num_heads,
                                             num_kv_heads, head_dim, &need);
  if (rc) return rc;
  if (need && (!workspace || workspace_bytes < need || !aligned16(workspace)))
    return fail(CDML_E_INVALID, "%s: %zu bytes of 16-byte aligned workspace needed, %zu given", what, need,
                workspace_bytes);
  const SharedPlan p = plan_shared(size, rows, batch, groups, max_members, max_new, max_prefix, max_tail, num_heads,
                                   num_kv_heads, head_dim);
  if (p.plain)
    return paged_attention(what, q8, true, q, ldq, kcache, vcache, kscale, vscale, cache_type, n_pages, page_size,
                           block_table, max_blocks, kv_len, cu_new, o, ldo, rows, batch, max_new, max_len, num_heads,
                           num_kv_heads, head_dim, scale, bad, workspace, workspace_bytes, stream);
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
  a.group_start = group_start;
  a.shared = shared;
  a.groups = groups;
  a.part = static_cast<float *>(workspace);
  a.part_width = round_up(head_dim, 4);
  a.part_stats = a.part + p.parts * a.part_width;
  a.part_splits = p.prefix_splits + p.own_splits;
  a.prefix_chunk = p.prefix_chunk;
  a.prefix_splits = p.prefix_splits;
  a.fused = p.fused;
  const bool wide = head_dim % 8 == 0 && ldq % 4 == 0 && ldo % 4 == 0 && aligned16(q) && aligned16(o) &&
                    aligned16(kcache) && aligned16(vcache);
  const hipStream_t st = as_hip(stream);
  auto run = [&](const PagedKernels &k) {
    switch (cache_type) {
      case CDML_CACHE_F32: return paged_shared_f32(a, k, wide, st);
      case CDML_CACHE_F16: return paged_shared_f16(a, k, wide, st);
      case CDML_CACHE_BF16: return paged_shared_bf16(a, k, wide, st);
      case CDML_CACHE_I8: return paged_shared_i8(a, k, wide, st);
      default: return paged_shared_f8(a, k, wide, st);
    }
  };
  // what the groups share, all of a group's rows in the same kernel
  a.prefix = true;
  a.few_rows = p.prefix_tile ? 0 : INT_MAX;
  a.most_rows = p.prefix_rows;
  a.few_chunk = a.tile_chunk = p.prefix_chunk;
  a.few_splits = a.tile_splits = p.prefix_splits;
  rc = run({false, !p.prefix_tile, p.prefix_tile});
  if (rc) return rc;
  // the tokens behind
  a.prefix = false;
  a.few_rows = a.most_rows = p.own.few_rows;
  a.few_chunk = p.own.few_chunk;
  a.few_splits = p.own.few_splits;
  a.tile_chunk = p.own.tile_chunk;
  a.tile_splits = p.own.tile_splits;
  a.first_split = p.prefix_splits;
  a.lone_waves = p.lone_waves;
  rc = run(p.own.kernels);
  if (rc) return rc;
  if (p.fused && !p.own.kernels.tile) return CDML_OK;
  paged_shared_join_kernel<<<dim3((unsigned)rows, (unsigned)(num_heads + 3) / 4), 256, 0, st>>>(a);
  return check_launch("paged_shared_join_kernel");
}
