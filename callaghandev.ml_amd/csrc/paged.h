// What the entries over the paged K/V cache share: argument checks and the arguments of
// the attention kernels, whose cache types are built in files of their own.
#pragma once

#include <cfloat>
#include <climits>

#include "attn_common.h"

namespace cdml {
namespace {

constexpr int kPagedMaxBatch = 4096;

inline int cache_type_bytes(int cache_type) {
  return cache_type == CDML_CACHE_F32 ? 4 : cache_type == CDML_CACHE_F16 || cache_type == CDML_CACHE_BF16 ? 2 : 0;
}

// The checks of a pool and its tables; the page size's log2 in *shift.
inline int check_pool(const char *what, int n_pages, int page_size, int max_blocks, int batch, int *shift) {
  if (page_size < 1 || page_size > 4096 || (page_size & (page_size - 1)))
    return fail(CDML_E_INVALID, "%s: page_size %d is no power of two up to 4096", what, page_size);
  // (scans of page_refs step past the last page by less than 2^30)
  if (n_pages < 1 || n_pages > (1 << 30) || (long long)n_pages * page_size > INT_MAX)
    return fail(CDML_E_INVALID, "%s: n_pages %d out of range", what, n_pages);
  if (max_blocks < 1 || (long long)max_blocks * page_size > INT_MAX)
    return fail(CDML_E_INVALID, "%s: max_blocks %d out of range", what, max_blocks);
  if (batch < 0 || batch > kPagedMaxBatch)
    return fail(CDML_E_INVALID, "%s: batch %d outside [0, %d]", what, batch, kPagedMaxBatch);
  *shift = __builtin_ctz((unsigned)page_size);
  return CDML_OK;
}

}  // namespace

// Inclusive sum over the lanes of a wave: within rows of 16 lanes by shifts, then each row's
// last lane to the rows after it.
template <int CTRL, int ROWS>
__device__ __forceinline__ uint32_t shifted(uint32_t x) {
  return __builtin_amdgcn_update_dpp(0, x, CTRL, ROWS, 0xf, false);
}
__device__ __forceinline__ uint32_t wave_scan(uint32_t x) {
  x += shifted<0x111, 0xf>(x);
  x += shifted<0x112, 0xf>(x);
  x += shifted<0x114, 0xf>(x);
  x += shifted<0x118, 0xf>(x);
  x += shifted<0x142, 0xa>(x);
  x += shifted<0x143, 0xc>(x);
  return x;
}

// A request's rows are numbered token-major: row rr of K/V head hk is head hk * group +
// rr % group of its new token rr / group.  Requests with at most few_rows rows a K/V head
// split their keys into chunks of few_chunk, those with more run in tiles of 128 rows and
// chunks of tile_chunk.  A request of one chunk is written to o, the chunks of others
// leave [head_dim] sums, a maximum (log2) and a sum in *_part.
struct PagedArgs {
  const float *q;
  const void *kc, *vc;
  const int *table, *kv_len, *cu_new;
  float *o;
  int *bad;
  int ldq, ldo, n_pages, page_shift, max_blocks, rows, batch, max_new, max_len;
  int heads, kv_heads, group, hd;
  float scale_log2;
  int few_rows, few_chunk, few_splits, tile_chunk, tile_splits;
  float *few_part;   // [batch][kv_heads][few_rows][few_splits][hd + 2]
  float *tile_part;  // [rows][heads][tile_splits][hd + 2]
  UDiv by_group;
};

struct PagedSeq {
  int first, n, len;  // first row, new tokens, tokens in the cache
};

__device__ __forceinline__ PagedSeq paged_seq(const PagedArgs &a, int b) {
  PagedSeq s;
  s.first = min(max(a.cu_new[b], 0), a.rows);
  const int end = min(max(a.cu_new[b + 1], s.first), a.rows);
  s.n = min(end - s.first, a.max_new);
  s.len = min(max(a.kv_len[b], 0), a.max_len);
  return s;
}

// The kernels of a call: for the requests of few rows either the vector units or a wave's
// matrix operand, and tiles for the others.
struct PagedKernels {
  bool rows, span, tile;
};

// Enqueue the kernels of one cache type (the arguments are validated).
int paged_attn_f32(const PagedArgs &a, const PagedKernels &k, bool wide, hipStream_t st);
int paged_attn_f16(const PagedArgs &a, const PagedKernels &k, bool wide, hipStream_t st);
int paged_attn_bf16(const PagedArgs &a, const PagedKernels &k, bool wide, hipStream_t st);

// The maximum (log2) of no key at all: no finite score lies below it, and beside any other its
// weight, with the sum 0 that it comes with, changes nothing.
constexpr float kNoKey = -FLT_MAX;
constexpr int kPagedTileRows = 128;  // rows of a tile workgroup
constexpr int kPagedSub = 512;       // keys whose pages a vector workgroup holds at a time

}  // namespace cdml
