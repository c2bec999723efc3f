// What the entries of attention over a paged cache share on the host, and the join of chunks.
#pragma once

#include "paged.h"

namespace cdml {

// cdml_paged_attn and cdml_paged_attn_q8 for an entry of its own name.  shared: for
// cdml_paged_attn_shared, whose max_len may be above the table's tokens and is cut to them, and
// whose workspace holds what this cache type needs, not what any type would.
int paged_attention(const char *what, bool q8, bool shared, const float *q, int ldq, const void *kcache,
                    const void *vcache, const float *kscale, const float *vscale, int cache_type, int n_pages,
                    int page_size, const int *block_table, int max_blocks, const int *kv_len, const int *cu_new,
                    float *o, int ldo, int rows, int batch, int max_new, int max_len, int num_heads, int num_kv_heads,
                    int head_dim, float scale, int *bad, void *workspace, size_t workspace_bytes, cdml_stream stream);

namespace {

// Chunks' sums: n of them, `stride` floats apart, each of a maximum (log2) and a sum in stats,
// `stats_stride` apart.
struct Chunks {
  const float *o, *stats;
  int n, stride, stats_stride;
};
struct Join {
  float M, L, acc[4];
};
__device__ __forceinline__ float join_most(const Chunks &p, float M) {
  for (int c = threadIdx.x & 63; c < p.n; c += 64) M = fmaxf(M, p.stats[(size_t)c * p.stats_stride]);
  return M;
}
__device__ __forceinline__ void join_add(int hd, const Chunks &part, Join &t) {
  const int lane = threadIdx.x & 63;
  for (int c0 = 0; c0 < part.n; c0 += 64) {
    const float *p = part.o + (size_t)c0 * part.stride, *st = part.stats + (size_t)c0 * part.stats_stride;
    const int m = min(part.n - c0, 64);
    const float w = lane < m ? fast_exp2(st[(size_t)lane * part.stats_stride] - t.M) : 0.f;
    t.L += lane < m ? st[(size_t)lane * part.stats_stride + 1] * w : 0.f;
    constexpr int U = 8;  // chunks in flight; past the last one it is read again and left out
    for (int c = 0; c < m; c += U) {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if (lane + 64 * j >= hd) continue;
        float x[U];
#pragma unroll
        for (int u = 0; u < U; ++u) x[u] = p[(size_t)min(c + u, m - 1) * part.stride + lane + 64 * j];
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const float wc = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(w), min(c + u, m - 1)));
          t.acc[j] = c + u < m ? fmaf(x[u], wc, t.acc[j]) : t.acc[j];
        }
      }
    }
  }
}
// o = sum_s w_s o_s / sum_s w_s l_s with w_s = 2^(m_s - M) over the chunks of N places, one wave;
// the chunks' statistics lie one to a lane, 64 chunks at a time.
template <int N>
__device__ __forceinline__ void join_chunks(int hd, const Chunks (&part)[N], float *o) {
  const int lane = threadIdx.x & 63;
  Join t{};
  t.M = kNoKey;
#pragma unroll
  for (int i = 0; i < N; ++i) t.M = join_most(part[i], t.M);
  t.M = wave_max(t.M);
#pragma unroll
  for (int i = 0; i < N; ++i) join_add(hd, part[i], t);
  t.L = wave_sum(t.L);
#pragma unroll
  for (int j = 0; j < 4; ++j)
    if (lane + 64 * j < hd) o[lane + 64 * j] = t.L == 0.f ? 0.f : t.acc[j] / t.L;
}

// The request that row `row` is of (a wave's question), batch if of none: requests that end at
// or before the row.
__device__ __forceinline__ int request_of_row(const PagedArgs &a, int row) {
  const int lane = threadIdx.x & 63;
  int b = 0;
  for (int b0 = 0; b0 < a.batch; b0 += 64) {
    const bool before = b0 + lane < a.batch && a.cu_new[b0 + lane + 1] <= row;
    const int n = __popcll(__builtin_amdgcn_ballot_w64(before));
    b += n;
    if (n < 64) break;
  }
  return b;
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

inline int check_sizes(const char *what, int rows, int batch, int max_new, int max_len, int heads, int kv_heads, int hd) {
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

inline int round_up(int n, int m) { return (int)(((long long)n + m - 1) / m * m); }

// size: bytes of a cached value.  shared: for kernels that know shared prefixes, of which there
// are none on the vector units.
inline Plan make_plan(int size, int rows, int batch, int max_new, int max_len, int heads, int kv_heads, int hd,
                      bool shared = false) {
  Plan p{};
  const int group = heads / kv_heads, most = max_new * group, len = max_len < 1 ? 1 : max_len;
  PagedKernels &k = p.kernels;
  k.tile = hd <= 128 && most > kSpanRows;
  k.rows = size > 1 && !shared && (hd > 128 || most <= (size == 4 ? kVecRows : kVecRows16));
  k.span = !k.rows && (!k.tile || group <= kSpanRows);
  p.few_rows = most < 1 ? 1 : k.tile ? kSpanRows : most;
  const long long pairs = (long long)(batch < 1 ? 1 : batch) * kv_heads;
  const long long groups = k.rows ? (p.few_rows + kVecRows - 1) / kVecRows : (p.few_rows + kSpanRows - 1) / kSpanRows;
  if (k.span && shared && len <= 1024) {
    p.few_chunk = round_up(len, 128);  // one chunk, in whose kernel the join is
  } else if (k.span) {
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

}  // namespace
}  // namespace cdml
