// Bookkeeping and data movement of the paged K/V cache (include/cdml.h): the plan of
// a step's new tokens, their append, and the reordering of a beam search's tables.
//
// Page counts are small next to the cache (4 bytes a page), so free pages are found
// by a scan of page_refs and taken in increasing order: no free list to keep, and the
// same tables whatever the timing.  One workgroup does what needs the total first
// (all pages or none); what is wide (slots of many tokens, table rows, copies) has
// a grid of its own.
#include "paged.h"

namespace cdml {
namespace {

constexpr int PC_THREADS = 1024;
constexpr int PC_SCAN = 16;  // pages a thread looks at per round of a scan

struct PlanArgs {
  int *refs;
  int n_pages, page_shift;
  int *table;
  int max_blocks;
  int *kv_len;
  const int *new_len;
  int batch, rows;
  int *cu_new, *slots, *positions, *status;
  int fill;  // whether the planning workgroup writes slots and positions itself
};

// Inclusive sum over the workgroup's threads; *total receives the sum of all.
template <typename T>
__device__ __forceinline__ T block_scan(T x, T *wave_sums, T *total) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) {
    const T y = __shfl_up(x, off);
    if (lane >= off) x += y;
  }
  __syncthreads();  // wave_sums may still be read from the call before
  if (lane == 63) wave_sums[wave] = x;
  __syncthreads();
  T before = 0, all = 0;
#pragma unroll
  for (int w = 0; w < PC_THREADS / 64; ++w) {
    if (w < wave) before += wave_sums[w];
    all += wave_sums[w];
  }
  *total = all;
  return before + x;
}

// Largest i in [0, n] with v[i] <= x, for v that does not decrease and v[0] <= x.
__device__ __forceinline__ int last_not_above(const int *v, int n, int x) {
  int lo = 0, hi = n;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (v[mid] <= x) lo = mid;
    else hi = mid - 1;
  }
  return lo;
}

// Calls take(page, rank) for free pages in increasing order, ranks 0 .. want - 1
// (fewer if there are not as many), and returns how many free pages were seen, at
// least want if there are.  A thread looks at PC_SCAN pages in a row per round.
template <typename F>
__device__ __forceinline__ int scan_free(const int *refs, int n_pages, int want, int *wave_sums, F take) {
  int found = 0;
  for (int p0 = 0; p0 < n_pages && found < want; p0 += PC_THREADS * PC_SCAN) {
    const int mine = p0 + threadIdx.x * PC_SCAN;
    uint32_t free = 0;
#pragma unroll
    for (int i = 0; i < PC_SCAN; ++i)
      if (mine + i < n_pages && refs[mine + i] == 0) free |= 1u << i;
    int total = 0;
    int rank = found + block_scan<int>(__popc(free), wave_sums, &total) - (int)__popc(free);
    for (; free && rank < want; free &= free - 1) take(mine + __ffs(free) - 1, rank++);
    found += total;
  }
  return found;
}

__device__ __forceinline__ void write_row(const PlanArgs &a, int row, const int *cu) {
  int slot = -1, pos = 0;
  if (row < cu[a.batch]) {
    const int b = last_not_above(cu, a.batch, row), end = cu[b + 1];
    pos = a.kv_len[b] - end + row;  // kv_len holds the new tokens already
    const int page = a.table[(size_t)b * a.max_blocks + (pos >> a.page_shift)];
    slot = (page << a.page_shift) + (pos & ((1 << a.page_shift) - 1));
  }
  a.slots[row] = slot;
  a.positions[row] = pos;
}

// One workgroup: sums of pages and tokens over the requests, a first scan that only
// counts free pages up to the need, then the scan that takes them.
__global__ void __launch_bounds__(PC_THREADS) paged_plan_kernel(const PlanArgs a) {
  __shared__ int pages[kPagedMaxBatch + 1], cu[kPagedMaxBatch + 1];  // exclusive sums
  __shared__ long long sums64[PC_THREADS / 64];
  __shared__ int sums[PC_THREADS / 64];
  const int t = threadIdx.x, P1 = (1 << a.page_shift) - 1;
  const long long room = (long long)a.max_blocks << a.page_shift;
  long long n_need = 0, n_new = 0;
  int code = 0;
  for (int b0 = 0; b0 < a.batch; b0 += PC_THREADS) {
    const int b = b0 + t;
    int need = 0, fresh = 0;
    if (b < a.batch) {
      const int len = a.kv_len[b], add = a.new_len[b];
      if (len < 0 || add < 0 || (long long)len + add > room) {
        code = 2;
      } else {
        fresh = add;
        need = (int)(((long long)len + add + P1) >> a.page_shift) - (int)(((long long)len + P1) >> a.page_shift);
      }
    }
    long long all = 0;
    const long long p = n_need + block_scan<long long>(need, sums64, &all);
    n_need += all;
    const long long c = n_new + block_scan<long long>(fresh, sums64, &all);
    n_new += all;
    if (b < a.batch) {  // sums past 31 bits belong to a step that is refused below
      pages[b + 1] = (int)p;
      cu[b + 1] = (int)c;
    }
  }
  if (t == 0) pages[0] = cu[0] = 0;
  code = __syncthreads_or(code) ? 2 : 0;
  if (n_new > a.rows) code |= 4;
  if (n_need > a.n_pages) {
    code |= 1;
  } else if (n_need > 0) {
    if (scan_free(a.refs, a.n_pages, (int)n_need, sums, [](int, int) {}) < n_need) code |= 1;
  }
  if (t == 0) {
    a.status[0] = code;
    a.status[1] = (int)min(n_need, (long long)INT_MAX);
    a.status[2] = (int)min(n_new, (long long)INT_MAX);
  }
  __syncthreads();
  if (code) {  // (the same in every thread)
    for (int b = t; b <= a.batch; b += PC_THREADS) {
      a.cu_new[b] = 0;
      cu[b] = 0;
    }
  } else {
    // the i-th free page is block have(b) + i - pages[b] of the request it falls to
    scan_free(a.refs, a.n_pages, (int)n_need, sums, [&](int page, int rank) {
      const int b = last_not_above(pages, a.batch, rank);
      const int have = (int)(((long long)a.kv_len[b] + P1) >> a.page_shift);
      a.table[(size_t)b * a.max_blocks + have + rank - pages[b]] = page;
      a.refs[page] = 1;
    });
    __syncthreads();
    for (int b = t; b < a.batch; b += PC_THREADS) a.kv_len[b] += cu[b + 1] - cu[b];
    for (int b = t; b <= a.batch; b += PC_THREADS) a.cu_new[b] = cu[b];
  }
  if (!a.fill) return;
  __syncthreads();
  for (int row = t; row < a.rows; row += PC_THREADS) write_row(a, row, cu);
}

constexpr int SLOT_THREADS = 256, SLOT_ROWS = 4;  // rows per thread

__global__ void __launch_bounds__(SLOT_THREADS) paged_slots_kernel(const PlanArgs a) {
  __shared__ int cu[kPagedMaxBatch + 1];
  for (int b = threadIdx.x; b <= a.batch; b += SLOT_THREADS) cu[b] = a.cu_new[b];
  __syncthreads();
  const int row0 = blockIdx.x * SLOT_THREADS * SLOT_ROWS + threadIdx.x;
#pragma unroll
  for (int i = 0; i < SLOT_ROWS; ++i)
    if (row0 + i * SLOT_THREADS < a.rows) write_row(a, row0 + i * SLOT_THREADS, cu);
}

// ---- append -----------------------------------------------------------------

template <typename T>
__device__ __forceinline__ uint32_t bits16(float x);
template <>
__device__ __forceinline__ uint32_t bits16<_Float16>(float x) {
  return __builtin_bit_cast(uint16_t, (_Float16)x);
}
template <>
__device__ __forceinline__ uint32_t bits16<__bf16>(float x) {
  return __builtin_bit_cast(uint16_t, (__bf16)x);
}

// Eight values of a row, rounded to the cache's type, in 16-byte stores.
__device__ __forceinline__ void put8(float *dst, const vf4 &x, const vf4 &y) {
  *reinterpret_cast<vf4 *>(dst) = x;
  *reinterpret_cast<vf4 *>(dst + 4) = y;
}
template <typename T>
__device__ __forceinline__ void put8(T *dst, const vf4 &x, const vf4 &y) {
  vu4 w;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    w[i] = bits16<T>(x[2 * i]) | bits16<T>(x[2 * i + 1]) << 16;
    w[2 + i] = bits16<T>(y[2 * i]) | bits16<T>(y[2 * i + 1]) << 16;
  }
  *reinterpret_cast<vu4 *>(dst) = w;
}

// A thread moves eight columns (VEC) or one column of one row, of K and of V.
template <typename T, bool VEC>
__global__ void __launch_bounds__(256) paged_append_kernel(const float *__restrict__ k, int ldk,
                                                           const float *__restrict__ v, int ldv,
                                                           T *__restrict__ kc, T *__restrict__ vc,
                                                           const int *__restrict__ slots, int rows, int n_slots,
                                                           int dim, int units) {
  const size_t total = (size_t)rows * units;
  for (size_t i = (size_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (size_t)gridDim.x * 256) {
    const int row = (int)(i / (unsigned)units), u = (int)(i - (size_t)row * units);
    const int slot = slots[row];
    if ((unsigned)slot >= (unsigned)n_slots) continue;
    const size_t dst = (size_t)slot * dim;
    if constexpr (VEC) {
      const vf4 *pk = reinterpret_cast<const vf4 *>(k + (size_t)row * ldk + 8 * u);
      const vf4 *pv = reinterpret_cast<const vf4 *>(v + (size_t)row * ldv + 8 * u);
      const vf4 k0 = pk[0], k1 = pk[1], v0 = pv[0], v1 = pv[1];
      put8(kc + dst + 8 * u, k0, k1);
      put8(vc + dst + 8 * u, v0, v1);
    } else {
      kc[dst + u] = (T)k[(size_t)row * ldk + u];
      vc[dst + u] = (T)v[(size_t)row * ldv + u];
    }
  }
}

template <typename T>
void launch_append(const float *k, int ldk, const float *v, int ldv, void *kc, void *vc, const int *slots, int rows,
                   int n_slots, int dim, hipStream_t st) {
  const bool vec = dim % 8 == 0 && ldk % 4 == 0 && ldv % 4 == 0 && aligned16(k) && aligned16(v) && aligned16(kc) &&
                   aligned16(vc);
  const int units = vec ? dim / 8 : dim;
  const size_t blocks = ((size_t)rows * units + 255) / 256;
  const dim3 grid((unsigned)(blocks < 65536 ? blocks : 65536));
  if (vec)
    paged_append_kernel<T, true><<<grid, 256, 0, st>>>(k, ldk, v, ldv, (T *)kc, (T *)vc, slots, rows, n_slots, dim,
                                                       units);
  else
    paged_append_kernel<T, false><<<grid, 256, 0, st>>>(k, ldk, v, ldv, (T *)kc, (T *)vc, slots, rows, n_slots, dim,
                                                        units);
}

// ---- reorder ----------------------------------------------------------------

struct ReorderArgs {
  int *refs;
  int n_pages, page_shift;
  int *table;
  int max_blocks;
  int *kv_len;
  const int *parents;
  int batch;
  int *src, *dst, *status;
  int *old_len, *old_table;  // workspace: the state before the call
};

__device__ __forceinline__ int parent_of(const ReorderArgs &a, int r) {
  const int p = a.parents[r];
  return (unsigned)p < (unsigned)a.batch ? p : -1;
}
__device__ __forceinline__ void add_ref(const ReorderArgs &a, int page, int d) {
  if ((unsigned)page < (unsigned)a.n_pages) atomicAdd(a.refs + page, d);
}
// Whether a lower row takes the state of p too (all threads of the workgroup call it).
__device__ __forceinline__ bool taken_before(const ReorderArgs &a, int p, int r) {
  int hit = 0;
  for (int i = threadIdx.x; i < r; i += blockDim.x) hit |= a.parents[i] == p;
  return __syncthreads_or(hit) != 0;
}

// Row r's old table and length into the workspace; its old pages lose a reference,
// those it takes from its parent gain one (integer sums: any order gives the same).
__global__ void __launch_bounds__(256) paged_refs_kernel(const ReorderArgs a) {
  const int r = blockIdx.x, P1 = (1 << a.page_shift) - 1;
  const int room = (int)min((long long)a.max_blocks << a.page_shift, (long long)INT_MAX);
  const int len = min(max(a.kv_len[r], 0), room);
  const int used = (int)(((long long)len + P1) >> a.page_shift);
  const int p = parent_of(a, r);
  const bool second = p >= 0 && taken_before(a, p, r);
  const int *row = a.table + (size_t)r * a.max_blocks;
  if (threadIdx.x == 0) a.old_len[r] = len;
  for (int j = threadIdx.x; j < used; j += 256) {
    const int page = row[j];
    a.old_table[(size_t)r * a.max_blocks + j] = page;
    // a row that stays where it is keeps its full pages, and its open one unless a lower row has it
    if (p != r || (second && j == len >> a.page_shift)) add_ref(a, page, -1);
  }
  if (p < 0 || p == r) return;
  const int plen = min(max(a.kv_len[p], 0), room);
  const int take = (plen >> a.page_shift) + ((plen & P1) != 0 && !second);
  const int *from = a.table + (size_t)p * a.max_blocks;
  for (int j = threadIdx.x; j < take; j += 256) add_ref(a, from[j], 1);
}

// Workgroup 0 finds pages for the copies; workgroup r + 1 writes row r's other entries.
__global__ void __launch_bounds__(PC_THREADS) paged_tables_kernel(const ReorderArgs a) {
  __shared__ int first[kPagedMaxBatch];  // lowest row that takes each row's state; then the pages found
  __shared__ int sums[PC_THREADS / 64];
  const int t = threadIdx.x, P1 = (1 << a.page_shift) - 1;
  if (blockIdx.x > 0) {
    const int r = blockIdx.x - 1, p = parent_of(a, r);
    const int len = p < 0 ? 0 : a.old_len[p];
    const bool open = (len & P1) != 0, second = p >= 0 && taken_before(a, p, r);
    if (t == 0 && !(open && second)) a.kv_len[r] = len;
    if (p == r) return;
    const int n = (len >> a.page_shift) + (open && !second);
    for (int j = t; j < n; j += PC_THREADS)
      a.table[(size_t)r * a.max_blocks + j] = a.old_table[(size_t)p * a.max_blocks + j];
    return;
  }
  for (int r = t; r < a.batch; r += PC_THREADS) first[r] = INT_MAX;
  __syncthreads();
  int wrong = 0;
  for (int r = t; r < a.batch; r += PC_THREADS) {
    const int p = parent_of(a, r);
    if (p >= 0) atomicMin(first + p, r);
    else wrong += a.parents[r] != -1;
  }
  int bad = 0, copies = 0;
  block_scan(wrong, sums, &bad);
  // each thread's rows r = t + PC_THREADS * i, four of them at most: place among the copies, or -1
  constexpr int MINE = kPagedMaxBatch / PC_THREADS;
  int turn[MINE];
#pragma unroll
  for (int i = 0; i < MINE; ++i) {
    const int r = t + PC_THREADS * i, p = r < a.batch ? parent_of(a, r) : -1;
    const bool copy = p >= 0 && (a.old_len[p] & P1) != 0 && first[p] != r;
    int all = 0;
    const int at = copies + block_scan<int>(copy, sums, &all) - 1;
    turn[i] = copy ? at : -1;
    copies += all;
  }
  __syncthreads();  // the last read of `first` as such
  const int found = copies ? scan_free(a.refs, a.n_pages, copies, sums, [&](int page, int rank) { first[rank] = page; })
                           : 0;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < MINE; ++i) {
    const int r = t + PC_THREADS * i;
    if (r >= a.batch) break;
    int src = -1, dst = -1;
    if (turn[i] >= 0) {
      const int p = parent_of(a, r), len = a.old_len[p], full = len >> a.page_shift;
      if (turn[i] < found) {
        dst = first[turn[i]];
        src = a.old_table[(size_t)p * a.max_blocks + full];
        // the full pages of the row are another workgroup's
        a.table[(size_t)r * a.max_blocks + full] = dst;
        a.refs[dst] = 1;
      }
      a.kv_len[r] = turn[i] < found ? len : full << a.page_shift;
    }
    a.src[r] = src;
    a.dst[r] = dst;
  }
  if (t == 0) {
    a.status[0] = max(copies - found, 0);
    a.status[1] = min(copies, found);
    a.status[2] = bad;
  }
}

// Workgroup (row, 2 * layer + which): the open page's tokens, one contiguous run.
template <int UNIT>
__global__ void __launch_bounds__(256) paged_copy_kernel(char *kc, char *vc, size_t layer_bytes, int n_pages,
                                                         size_t page_bytes, int token_bytes, int page_mask,
                                                         const int *__restrict__ src, const int *__restrict__ dst,
                                                         const int *__restrict__ kv_len) {
  const int r = blockIdx.x, from = src[r], to = dst[r];
  if ((unsigned)from >= (unsigned)n_pages || (unsigned)to >= (unsigned)n_pages) return;
  const size_t bytes = (size_t)(kv_len[r] & page_mask) * token_bytes;
  char *base = ((blockIdx.y & 1) ? vc : kc) + (blockIdx.y >> 1) * layer_bytes;
  const char *s = base + from * page_bytes;
  char *d = base + to * page_bytes;
  for (size_t i = ((size_t)blockIdx.z * 256 + threadIdx.x) * UNIT; i < bytes; i += (size_t)gridDim.z * 256 * UNIT) {
    if constexpr (UNIT == 16) *reinterpret_cast<vu4 *>(d + i) = *reinterpret_cast<const vu4 *>(s + i);
    else *reinterpret_cast<uint16_t *>(d + i) = *reinterpret_cast<const uint16_t *>(s + i);
  }
}

}  // namespace
}  // namespace cdml

using namespace cdml;

extern "C" int cdml_paged_plan(int *page_refs, int n_pages, int page_size, int *block_table, int max_blocks,
                               int *kv_len, const int *new_len, int batch, int rows, int *cu_new, int *slots,
                               int *positions, int *status, cdml_stream stream) {
  PlanArgs a{};
  int rc = check_pool("cdml_paged_plan", n_pages, page_size, max_blocks, batch, &a.page_shift);
  if (rc) return rc;
  if (rows < 0) return fail(CDML_E_INVALID, "cdml_paged_plan: rows %d is negative", rows);
  if (!cu_new || !status || (rows && (!slots || !positions)) ||
      (batch && (!page_refs || !block_table || !kv_len || !new_len)))
    return fail(CDML_E_INVALID, "cdml_paged_plan: NULL pointer");
  rc = ensure_device();
  if (rc) return rc;
  a.refs = page_refs;
  a.n_pages = n_pages;
  a.table = block_table;
  a.max_blocks = max_blocks;
  a.kv_len = kv_len;
  a.new_len = new_len;
  a.batch = batch;
  a.rows = rows;
  a.cu_new = cu_new;
  a.slots = slots;
  a.positions = positions;
  a.status = status;
  a.fill = rows <= 4 * PC_THREADS;
  paged_plan_kernel<<<1, PC_THREADS, 0, as_hip(stream)>>>(a);
  rc = check_launch("paged_plan_kernel");
  if (rc || a.fill) return rc;
  const int per = SLOT_THREADS * SLOT_ROWS;
  paged_slots_kernel<<<(unsigned)((rows - 1) / per + 1), SLOT_THREADS, 0, as_hip(stream)>>>(a);
  return check_launch("paged_slots_kernel");
}

extern "C" int cdml_paged_append(const float *k_new, int ldk, const float *v_new, int ldv, void *kcache, void *vcache,
                                 int cache_type, const int *slots, int rows, int n_pages, int page_size, int kv_dim,
                                 cdml_stream stream) {
  int shift = 0;
  int rc = check_pool("cdml_paged_append", n_pages, page_size, 1, 0, &shift);
  if (rc) return rc;
  if (!cache_type_bytes(cache_type)) return fail(CDML_E_INVALID, "cdml_paged_append: unknown cache type %d", cache_type);
  if (rows < 0 || kv_dim <= 0 || ldk < kv_dim || ldv < kv_dim)
    return fail(CDML_E_INVALID, "cdml_paged_append: bad size (rows %d, kv_dim %d, ldk %d, ldv %d)", rows, kv_dim, ldk,
                ldv);
  if (rows == 0) return CDML_OK;
  if (!k_new || !v_new || !kcache || !vcache || !slots)
    return fail(CDML_E_INVALID, "cdml_paged_append: NULL pointer");
  rc = ensure_device();
  if (rc) return rc;
  const int n_slots = n_pages * page_size;
  const hipStream_t st = as_hip(stream);
  if (cache_type == CDML_CACHE_F32)
    launch_append<float>(k_new, ldk, v_new, ldv, kcache, vcache, slots, rows, n_slots, kv_dim, st);
  else if (cache_type == CDML_CACHE_F16)
    launch_append<_Float16>(k_new, ldk, v_new, ldv, kcache, vcache, slots, rows, n_slots, kv_dim, st);
  else
    launch_append<__bf16>(k_new, ldk, v_new, ldv, kcache, vcache, slots, rows, n_slots, kv_dim, st);
  return check_launch("paged_append_kernel");
}

extern "C" int cdml_paged_reorder_workspace_size(int batch, int max_blocks, size_t *bytes) {
  if (!bytes) return fail(CDML_E_INVALID, "cdml_paged_reorder_workspace_size: bytes is NULL");
  if (batch < 0 || batch > kPagedMaxBatch || max_blocks < 1)
    return fail(CDML_E_INVALID, "cdml_paged_reorder_workspace_size: bad size");
  *bytes = sizeof(int) * (size_t)batch * (1 + (size_t)max_blocks);
  return CDML_OK;
}

extern "C" int cdml_paged_reorder(int *page_refs, int n_pages, int page_size, int *block_table, int max_blocks,
                                  int *kv_len, const int *parents, int batch, int *copy_src, int *copy_dst,
                                  int *status, void *workspace, size_t workspace_bytes, cdml_stream stream) {
  ReorderArgs a{};
  int rc = check_pool("cdml_paged_reorder", n_pages, page_size, max_blocks, batch, &a.page_shift);
  if (rc) return rc;
  if (!status || (batch && (!page_refs || !block_table || !kv_len || !parents || !copy_src || !copy_dst)))
    return fail(CDML_E_INVALID, "cdml_paged_reorder: NULL pointer");
  size_t need = 0;
  rc = cdml_paged_reorder_workspace_size(batch, max_blocks, &need);
  if (rc) return rc;
  if (need && (!workspace || workspace_bytes < need || (reinterpret_cast<uintptr_t>(workspace) & 3)))
    return fail(CDML_E_INVALID, "cdml_paged_reorder: %zu bytes of 4-byte aligned workspace needed, %zu given", need,
                workspace_bytes);
  rc = ensure_device();
  if (rc) return rc;
  a.refs = page_refs;
  a.n_pages = n_pages;
  a.table = block_table;
  a.max_blocks = max_blocks;
  a.kv_len = kv_len;
  a.parents = parents;
  a.batch = batch;
  a.src = copy_src;
  a.dst = copy_dst;
  a.status = status;
  a.old_len = static_cast<int *>(workspace);
  a.old_table = a.old_len + batch;
  if (batch) {
    paged_refs_kernel<<<batch, 256, 0, as_hip(stream)>>>(a);
    rc = check_launch("paged_refs_kernel");
    if (rc) return rc;
  }
  paged_tables_kernel<<<batch + 1, PC_THREADS, 0, as_hip(stream)>>>(a);
  return check_launch("paged_tables_kernel");
}

extern "C" int cdml_paged_copy(void *kcache, void *vcache, int cache_type, int layers, size_t layer_stride,
                               int n_pages, int page_size, int kv_dim, const int *copy_src, const int *copy_dst,
                               const int *kv_len, int batch, cdml_stream stream) {
  int shift = 0;
  int rc = check_pool("cdml_paged_copy", n_pages, page_size, 1, batch, &shift);
  if (rc) return rc;
  const int size = cache_type_bytes(cache_type);
  if (!size) return fail(CDML_E_INVALID, "cdml_paged_copy: unknown cache type %d", cache_type);
  if (layers < 0 || layers > 32767 || kv_dim <= 0 || (long long)kv_dim * size > INT_MAX)
    return fail(CDML_E_INVALID, "cdml_paged_copy: bad size (layers %d, kv_dim %d)", layers, kv_dim);
  if (layers > 1 && layer_stride < (size_t)n_pages * page_size * kv_dim)
    return fail(CDML_E_INVALID, "cdml_paged_copy: layer_stride smaller than a layer's cache");
  if (batch == 0 || layers == 0) return CDML_OK;
  if (!kcache || !vcache || !copy_src || !copy_dst || !kv_len)
    return fail(CDML_E_INVALID, "cdml_paged_copy: NULL pointer");
  rc = ensure_device();
  if (rc) return rc;
  const int token = kv_dim * size;
  const size_t page = (size_t)page_size * token, layer = layer_stride * size;
  const bool vec = token % 16 == 0 && layer % 16 == 0 && aligned16(kcache) && aligned16(vcache);
  // a workgroup moves 16 KiB of a page at a time (4 16-byte units a thread)
  size_t parts = (page + 16383) / 16384;
  if (parts > 64) parts = 64;
  const dim3 grid(batch, 2 * layers, (unsigned)parts);
  if (vec)
    paged_copy_kernel<16><<<grid, 256, 0, as_hip(stream)>>>((char *)kcache, (char *)vcache, layer, n_pages, page, token,
                                                            page_size - 1, copy_src, copy_dst, kv_len);
  else
    paged_copy_kernel<2><<<grid, 256, 0, as_hip(stream)>>>((char *)kcache, (char *)vcache, layer, n_pages, page, token,
                                                           page_size - 1, copy_src, copy_dst, kv_len);
  return check_launch("paged_copy_kernel");
}
