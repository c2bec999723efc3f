// What the entries over the paged K/V cache share: argument checks and the arguments of
// the attention kernels, whose cache types are built in files of their own.
#pragma once

#include <cfloat>
#include <climits>
#include <type_traits>

#include "attn_common.h"

namespace cdml {
namespace {

constexpr int kPagedMaxBatch = 4096;

inline int cache_type_bytes(int cache_type) {
  return cache_type == CDML_CACHE_F32 ? 4 : cache_type == CDML_CACHE_F16 || cache_type == CDML_CACHE_BF16 ? 2 : 0;
}

inline bool q8_cache_type(int cache_type) { return cache_type == CDML_CACHE_I8 || cache_type == CDML_CACHE_F8; }

// Bytes of a K/V head's row of an 8-bit cache.
__host__ __device__ constexpr int q8_width(int hd) { return (hd + 15) & ~15; }

// The checks of an 8-bit cache's arrays.
inline int check_q8(const char *what, const void *kcache, const void *vcache, const float *kscale,
                    const float *vscale) {
  if (!kcache || !vcache || !kscale || !vscale) return fail(CDML_E_INVALID, "%s: NULL pointer", what);
  if (!aligned16(kcache) || !aligned16(vcache))
    return fail(CDML_E_INVALID, "%s: the cache is not 16-byte aligned", what);
  return CDML_OK;
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
  const float *ks, *vs;  // scales and bytes of a head's row of an 8-bit cache
  int width;
  const int *table, *kv_len, *cu_new;
  float *o;
  int *bad;
  int ldq, ldo, n_pages, page_shift, max_blocks, rows, batch, max_new, max_len;
  int heads, kv_heads, group, hd;
  float scale_log2;
  int few_rows, few_chunk, few_splits, tile_chunk, tile_splits;
  int most_rows;     // of a request of few rows, at most (a hint)
  bool wide;         // 16-byte aligned rows of Q, of whole vectors
  bool lone_waves;   // SHARED: requests have so few keys that a wave takes all of a K/V head
  float *few_part;   // [batch][kv_heads][few_rows][few_splits][hd + 2]
  float *tile_part;  // [rows][heads][tile_splits][hd + 2]
  UDiv by_group;
  // Requests that share their first tokens (SHARED): a launch for what the groups share, in
  // which a group is one request whose rows are those of all its members, and one for the
  // tokens behind.  Their chunks leave sums in part [rows][heads][part_splits][part_width] and
  // their maxima (log2) and sums in part_stats [rows][heads][part_splits][2], the shared
  // tokens' first.  fused: requests of few rows have one chunk of their own, which adds the
  // shared tokens' and writes o.
  const int *group_start, *shared;
  int groups;
  bool prefix, fused;  // prefix: which of the two launches
  float *part, *part_stats;
  int part_splits, part_width, first_split, prefix_chunk, prefix_splits;
};

// The kernel's arguments, read again: what a kernel's end needs is not held in scalar registers
// throughout (a kernel whose one argument is a PagedArgs).
__device__ __forceinline__ const PagedArgs &args_again() {
  auto p = (const __attribute__((address_space(4))) PagedArgs *)__builtin_amdgcn_kernarg_segment_ptr();
  asm volatile("" : "+s"(p));
  return *(const PagedArgs *)p;
}

// Chunks in which `seen` tokens lie.
__device__ __forceinline__ int chunks_seen(int seen, int chunk) { return seen <= 0 ? 0 : (seen - 1) / chunk + 1; }

struct PagedSeq {
  int first, n, len;  // first row, new tokens, tokens in the cache (past the last that counts)
  int start, table;   // first token that counts, row of the block table
  bool causal;        // new token i sees those up to len - n + i, else all
};

// Tokens that request b shares with its group, whole pages.
__device__ __forceinline__ int shared_tokens(const PagedArgs &a, int b) {
  return min(max(a.shared[b], 0), a.max_len) & ~((1 << a.page_shift) - 1);
}

// Request b; of a launch over what groups share, group b.
template <bool SHARED = false>
__device__ __forceinline__ PagedSeq paged_seq(const PagedArgs &a, int b) {
  PagedSeq s{};
  if (SHARED && a.prefix) {
    s.table = min(max(a.group_start[b], 0), a.batch);
    const int behind = min(max(a.group_start[b + 1], s.table), a.batch);
    if (behind - s.table < 2) return s;
    s.first = min(max(a.cu_new[s.table], 0), a.rows);
    s.len = shared_tokens(a, s.table);
    s.n = s.len ? min(max(a.cu_new[behind], s.first), a.rows) - s.first : 0;
    return s;
  }
  s.first = min(max(a.cu_new[b], 0), a.rows);
  const int end = min(max(a.cu_new[b + 1], s.first), a.rows);
  s.n = min(end - s.first, a.max_new);
  s.len = min(max(a.kv_len[b], 0), a.max_len);
  s.table = b;
  s.causal = true;
  if constexpr (SHARED) s.start = shared_tokens(a, b);
  return s;
}

// Keys [from, to) of split `split` of `splits`: a chunk from the first on, and the last takes the rest.
template <bool SHARED>
__device__ __forceinline__ int split_from(const PagedSeq &s, int split, int chunk) {
  return (SHARED ? s.start : 0) + split * chunk;
}
template <bool SHARED>
__device__ __forceinline__ int split_to(int from, int split, int splits, int chunk, int kend) {
  return SHARED && split == splits - 1 ? kend : min(from + chunk, kend);
}

// A cached value of 8 bits, without its scale.
struct I8 {
  uint8_t c;
};
struct F8 {
  uint8_t c;
};
template <typename T>
constexpr bool kQ8 = std::is_same<T, I8>::value || std::is_same<T, F8>::value;

// The kernels of a call: for the requests of few rows either the vector units or a wave's
// matrix operand, and tiles for the others.
struct PagedKernels {
  bool rows, span, tile;
};

// Enqueue the kernels of one cache type (the arguments are validated).
int paged_attn_f32(const PagedArgs &a, const PagedKernels &k, bool wide, hipStream_t st);
int paged_attn_f16(const PagedArgs &a, const PagedKernels &k, bool wide, hipStream_t st);
int paged_attn_bf16(const PagedArgs &a, const PagedKernels &k, bool wide, hipStream_t st);
int paged_attn_i8(const PagedArgs &a, const PagedKernels &k, bool wide, hipStream_t st);
int paged_attn_f8(const PagedArgs &a, const PagedKernels &k, bool wide, hipStream_t st);

// The same over what groups share, or over the tokens behind it.
int paged_shared_f32(const PagedArgs &a, const PagedKernels &k, bool wide, hipStream_t st);
int paged_shared_f16(const PagedArgs &a, const PagedKernels &k, bool wide, hipStream_t st);
int paged_shared_bf16(const PagedArgs &a, const PagedKernels &k, bool wide, hipStream_t st);
int paged_shared_i8(const PagedArgs &a, const PagedKernels &k, bool wide, hipStream_t st);
int paged_shared_f8(const PagedArgs &a, const PagedKernels &k, bool wide, hipStream_t st);

// The maximum (log2) of no key at all: no finite score lies below it, and beside any other its
// weight, with the sum 0 that it comes with, changes nothing.
constexpr float kNoKey = -FLT_MAX;
constexpr int kPagedTileRows = 128;  // rows of a tile workgroup
constexpr int kPagedSub = 512;       // keys whose pages a vector workgroup holds at a time

}  // namespace cdml
