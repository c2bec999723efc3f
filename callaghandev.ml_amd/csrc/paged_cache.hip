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
constexpr int PC_WAVES = PC_THREADS / 64;
constexpr int PC_ROUNDS = 16;  // 256 pages a wave, of a span
constexpr int PC_SPAN = PC_ROUNDS * 256 * PC_WAVES;

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

// Inclusive sums of x and y (below 2^31) over the workgroup's threads, and their totals.
// They are summed as halves of 16 bits, which 4096 terms cannot overflow.
struct ScanScratch {
  vu4 sums[PC_WAVES];
};
__device__ __forceinline__ void block_scan(int x, int y, ScanScratch &sc, long long *sum_x, long long *sum_y,
                                           long long *all_x, long long *all_y) {
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  vu4 v = {wave_scan(x & 0xffff), wave_scan((uint32_t)x >> 16), wave_scan(y & 0xffff), wave_scan((uint32_t)y >> 16)};
  __syncthreads();  // the scratch may still be read from the call before
  if (lane == 63) sc.sums[wave] = v;
  __syncthreads();
  vu4 all = {};
#pragma unroll
  for (int w = 0; w < PC_WAVES; ++w) {
    const vu4 s = sc.sums[w];
    if (w < wave) v += s;
    all += s;
  }
  auto whole = [](uint32_t lo, uint32_t hi) { return (long long)lo + ((long long)hi << 16); };
  *sum_x = whole(v[0], v[1]);
  *sum_y = whole(v[2], v[3]);
  *all_x = whole(all[0], all[1]);
  *all_y = whole(all[2], all[3]);
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

// The free pages among a wave's next 256, four to a lane: bit j for page p + 4 lane + j.
// COUNTED: the references were counted by this kernel's atomics, which add in L2; loads of
// the device's scope read there, whatever the CU's cache holds of their lines (tables and
// lengths may lie next to the references, and were read before).
template <bool COUNTED>
__device__ __forceinline__ uint32_t free_of(const int *refs, int p, int n_pages) {
  const int mine = p + 4 * (int)(threadIdx.x & 63);
  if (mine + 4 <= n_pages) {
    int r[4];
    if constexpr (COUNTED) {
      const uint64_t *two = reinterpret_cast<const uint64_t *>(refs + mine);
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const uint64_t w = __hip_atomic_load(two + i, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        r[2 * i] = (int)(uint32_t)w;
        r[2 * i + 1] = (int)(w >> 32);
      }
    } else {
      const int4 w = *reinterpret_cast<const int4 *>(refs + mine);
      r[0] = w.x, r[1] = w.y, r[2] = w.z, r[3] = w.w;
    }
    return (r[0] == 0) | (r[1] == 0) << 1 | (r[2] == 0) << 2 | (r[3] == 0) << 3;
  }
  uint32_t f = 0;
#pragma unroll
  for (int j = 0; j < 3; ++j) {
    if (mine + j >= n_pages) continue;
    const int r = COUNTED ? __hip_atomic_load(refs + mine + j, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT)
                          : refs[mine + j];
    if (r == 0) f |= 1u << j;
  }
  return f;
}

// Free pages in increasing order, by one workgroup, a span of the pool at a time, of which
// each wave has a run of its own and each lane, once counted, four bits for every 256 pages
// of it.
template <bool COUNTED>
struct FreePages {
  int *counts;    // LDS, [PC_WAVES]: free pages of a span's runs
  uint64_t mask;  // this lane's of the span counted last
  int span;       // its first page, or -1
  int before, all;  // free pages of the runs before this wave's, and of the span

  __device__ __forceinline__ explicit FreePages(int *lds) : counts(lds), mask(0), span(-1), before(0), all(0) {}
  __device__ __forceinline__ int run(int n_pages, int *end) const {
    const int len = min(n_pages - span, PC_SPAN), per = (len + PC_WAVES * 256 - 1) / (PC_WAVES * 256) * 256;
    const int begin = span + (int)(threadIdx.x >> 6) * per;
    *end = min(begin + per, span + len);
    return begin;
  }
  // Counts the span from page s on (all threads), unless it is the one counted last.
  __device__ __forceinline__ void count(const int *refs, int n_pages, int s) {
    if (s == span) return;
    span = s;
    int end;
    const int begin = run(n_pages, &end);
    mask = 0;
#pragma unroll 4
    for (int i = 0; i < PC_ROUNDS; ++i)
      if (begin + 256 * i < end) mask |= (uint64_t)free_of<COUNTED>(refs, begin + 256 * i, end) << (4 * i);
    const int c = wave_reduce((int)__popcll(mask), [](int a, int b) { return a + b; });
    __syncthreads();  // counts may still be read
    if ((threadIdx.x & 63) == 0) counts[threadIdx.x >> 6] = c;
    __syncthreads();
    before = all = 0;
#pragma unroll
    for (int w = 0; w < PC_WAVES; ++w) {
      if (w < (int)(threadIdx.x >> 6)) before += counts[w];
      all += counts[w];
    }
  }
  // list[r - from] = page for the span's free pages r = from .. upto - 1, counted from
  // `first` on (what the spans before it held).
  __device__ __forceinline__ void list_pages(int n_pages, int first, int from, int upto, int *list) const {
    int end, rank = first + before;
    int p = run(n_pages, &end);
    for (uint64_t m = mask; p < end && rank < upto; p += 256, m >>= 4) {
      int at = rank;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const uint64_t who = __builtin_amdgcn_ballot_w64(m >> j & 1);
        at += __builtin_amdgcn_mbcnt_hi((uint32_t)(who >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)who, 0));
        rank += __popcll(who);
      }
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (m >> j & 1) {
          if (at >= from && at < upto) list[at - from] = p + 4 * (int)(threadIdx.x & 63) + j;
          ++at;
        }
    }
  }
};

// Slot and position of row `row`, which starts after `first` rows of its request, whose
// cache held `len` tokens; or of a row of no request.
__device__ __forceinline__ void write_row(const PlanArgs &a, int row, int b, int first, int len) {
  int slot = -1, pos = 0;
  if (b >= 0) {
    pos = len + row - first;
    const int page = a.table[(size_t)b * a.max_blocks + (pos >> a.page_shift)];
    // (an entry that is no page, shifted, could pass 32 bits into another page's slots)
    if ((unsigned)page < (unsigned)a.n_pages) slot = (page << a.page_shift) + (pos & ((1 << a.page_shift) - 1));
  }
  a.slots[row] = slot;
  a.positions[row] = pos;
}

constexpr int PLAN_LIST = 8192;  // pages that are handed out at a time

// One workgroup: sums of pages and tokens over the requests, a count of free pages up to
// the need, then the scan that takes them.  A chain of memory round trips bounds it: 64
// requests over 40000 pages take 10.8 us.
__global__ void __launch_bounds__(PC_THREADS) paged_plan_kernel(const PlanArgs a) {
  __shared__ int pages[kPagedMaxBatch + 1], cu[kPagedMaxBatch + 1];  // exclusive sums
  __shared__ int old[kPagedMaxBatch];                                // kv_len before
  __shared__ ScanScratch scratch;
  __shared__ int counts[PC_WAVES], list[PLAN_LIST];
  FreePages<false> pool(counts);
  const int t = threadIdx.x, P1 = (1 << a.page_shift) - 1;
  const long long room = (long long)a.max_blocks << a.page_shift;
  long long n_need = 0, n_new = 0;
  int code = 0;
  for (int b0 = 0; b0 < a.batch; b0 += PC_THREADS) {
    const int b = b0 + t;
    int need = 0, fresh = 0;
    if (b < a.batch) {
      const int len = a.kv_len[b], add = a.new_len[b];
      old[b] = len;
      if (len < 0 || add < 0 || (long long)len + add > room) {
        code = 2;
      } else {
        fresh = add;
        need = (int)((((long long)len + add + P1) >> a.page_shift) - (((long long)len + P1) >> a.page_shift));
      }
    }
    long long sum_need, sum_new, all_need, all_new;
    block_scan(need, fresh, scratch, &sum_need, &sum_new, &all_need, &all_new);
    if (b < a.batch) {  // sums past 31 bits belong to a step that is refused below
      pages[b + 1] = (int)(n_need + sum_need);
      cu[b + 1] = (int)(n_new + sum_new);
    }
    n_need += all_need;
    n_new += all_new;
  }
  if (t == 0) pages[0] = cu[0] = 0;
  code = __syncthreads_or(code) ? 2 : 0;
  if (n_new > a.rows) code |= 4;
  long long n_free = 0;
  for (int span = 0; span < a.n_pages && n_free < n_need; span += PC_SPAN) {
    pool.count(a.refs, a.n_pages, span);
    n_free += pool.all;
  }
  if (n_free < n_need) code |= 1;
  if (t == 0) {
    a.status[0] = code;
    a.status[1] = (int)min(n_need, (long long)INT_MAX);
    a.status[2] = (int)min(n_new, (long long)INT_MAX);
  }
  if (code) {  // (the same in every thread)
    for (int b = t; b <= a.batch; b += PC_THREADS) a.cu_new[b] = 0;
    if (a.fill)
      for (int row = t; row < a.rows; row += PC_THREADS) write_row(a, row, -1, 0, 0);
    return;
  }
  // a span's free pages by rank, then the rank's place: block have(b) + rank - pages[b] of
  // the request that it falls to
  const int want = (int)n_need;
  for (int span = 0, first = 0; first < want; span += PC_SPAN) {
    pool.count(a.refs, a.n_pages, span);
    const int last = min(want, first + pool.all);
    for (int from = first; from < last; from += PLAN_LIST) {
      const int upto = min(last, from + PLAN_LIST);
      pool.list_pages(a.n_pages, first, from, upto, list);
      __syncthreads();
      for (int rank = from + t; rank < upto; rank += PC_THREADS) {
        const int b = last_not_above(pages, a.batch, rank), page = list[rank - from];
        const int have = (int)(((long long)old[b] + P1) >> a.page_shift);
        a.table[(size_t)b * a.max_blocks + have + rank - pages[b]] = page;
        a.refs[page] = 1;
      }
      __syncthreads();
    }
    first += pool.all;
  }
  for (int b = t; b <= a.batch; b += PC_THREADS) {
    a.cu_new[b] = cu[b];
    if (b < a.batch) a.kv_len[b] = old[b] + cu[b + 1] - cu[b];
  }
  if (!a.fill) return;
  __syncthreads();
  for (int row = t; row < a.rows; row += PC_THREADS) {
    const int b = row < cu[a.batch] ? last_not_above(cu, a.batch, row) : -1;
    write_row(a, row, b, b < 0 ? 0 : cu[b], b < 0 ? 0 : old[b]);
  }
}

constexpr int SLOT_THREADS = 256, SLOT_ROWS = 4;  // rows per thread

__global__ void __launch_bounds__(SLOT_THREADS) paged_slots_kernel(const PlanArgs a) {
  __shared__ int cu[kPagedMaxBatch + 1];
  for (int b = threadIdx.x; b <= a.batch; b += SLOT_THREADS) cu[b] = a.cu_new[b];
  __syncthreads();
  const int row0 = blockIdx.x * SLOT_THREADS * SLOT_ROWS + threadIdx.x;
#pragma unroll
  for (int i = 0; i < SLOT_ROWS; ++i) {
    const int row = row0 + i * SLOT_THREADS;
    if (row >= a.rows) break;
    const int b = row < cu[a.batch] ? last_not_above(cu, a.batch, row) : -1;
    // (kv_len holds the new tokens already)
    write_row(a, row, b, b < 0 ? 0 : cu[b], b < 0 ? 0 : a.kv_len[b] - (cu[b + 1] - cu[b]));
  }
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

// A thread moves eight columns (VEC) or one column of one row, of K and of V.  HBM bounds it:
// 16384 rows of 1024 into bf16 (201 MB) take 39 us, 5.2 TB/s.
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
// Whether a lower row takes the state of p too (a wave's question).
__device__ __forceinline__ bool taken_before(const ReorderArgs &a, int p, int r) {
  for (int i = threadIdx.x & 63; i - (int)(threadIdx.x & 63) < r; i += 64)
    if (__builtin_amdgcn_ballot_w64(i < r && a.parents[i] == p)) return true;
  return false;
}
__device__ __forceinline__ int length_of(const ReorderArgs &a, int r) {
  return (int)min((long long)max(a.kv_len[r], 0), min((long long)a.max_blocks << a.page_shift, (long long)INT_MAX));
}

// A wave per row: its old table and length into the workspace; its old pages lose a
// reference, those it takes from its parent gain one (integer sums: any order gives the
// same).
__device__ __forceinline__ void count_refs(const ReorderArgs &a, int r) {
  const int lane = threadIdx.x & 63, P1 = (1 << a.page_shift) - 1;
  const int len = length_of(a, r), used = (int)(((long long)len + P1) >> a.page_shift), p = parent_of(a, r);
  const bool second = p >= 0 && taken_before(a, p, r);
  const int *row = a.table + (size_t)r * a.max_blocks;
  if (lane == 0) a.old_len[r] = len;
  const int plen = p < 0 ? 0 : length_of(a, p), take = (plen >> a.page_shift) + ((plen & P1) != 0 && !second);
  const int *from = a.table + (size_t)max(p, 0) * a.max_blocks;
  // beams share most pages: one that the row has and takes again at the same place (all of
  // them, if it stays where it is) is left alone
  for (int j = lane; j < max(used, take); j += 64) {
    const int had = j < used ? row[j] : -1, gets = j < take ? from[j] : -1;
    if (j < used) a.old_table[(size_t)r * a.max_blocks + j] = had;
    if (had == gets) continue;
    add_ref(a, had, -1);
    add_ref(a, gets, 1);
  }
}

// A wave per row: its length and entries but those of a copy.
__device__ __forceinline__ void write_table(const ReorderArgs &a, int r) {
  const int lane = threadIdx.x & 63, P1 = (1 << a.page_shift) - 1, p = parent_of(a, r);
  const int len = p < 0 ? 0 : a.old_len[p];
  const bool open = (len & P1) != 0, second = p >= 0 && taken_before(a, p, r);
  if (lane == 0 && !(open && second)) a.kv_len[r] = len;
  if (p == r) return;
  const int n = (len >> a.page_shift) + (open && !second);
  for (int j = lane; j < n; j += 64)
    a.table[(size_t)r * a.max_blocks + j] = a.old_table[(size_t)p * a.max_blocks + j];
}

struct CopyScratch {
  int first[kPagedMaxBatch];  // lowest row that takes each row's state; then the pages found
  ScanScratch scan;
  int counts[PC_WAVES];
};

// One workgroup: pages for the copies, and their rows' entries and lengths.
template <bool COUNTED>
__device__ __forceinline__ void place_copies(const ReorderArgs &a, CopyScratch &sc) {
  const int t = threadIdx.x, P1 = (1 << a.page_shift) - 1;
  int *first = sc.first;
  for (int r = t; r < a.batch; r += PC_THREADS) first[r] = INT_MAX;
  __syncthreads();
  for (int r = t; r < a.batch; r += PC_THREADS) {
    const int p = parent_of(a, r);
    if (p >= 0) atomicMin(first + p, r);
  }
  __syncthreads();
  // each thread's rows r = t + PC_THREADS * i, four of them at most: place among the copies, or -1
  constexpr int MINE = kPagedMaxBatch / PC_THREADS;
  int turn[MINE], copies = 0, wrong = 0;
#pragma unroll
  for (int i = 0; i < MINE; ++i) {
    turn[i] = -1;
    if (i * PC_THREADS >= a.batch) continue;
    const int r = t + PC_THREADS * i, p = r < a.batch ? parent_of(a, r) : -1;
    const bool copy = p >= 0 && (a.old_len[p] & P1) != 0 && first[p] != r;
    long long at, bad, all_copies, all_bad;
    block_scan(copy, r < a.batch && p < 0 && a.parents[r] != -1, sc.scan, &at, &bad, &all_copies, &all_bad);
    if (copy) turn[i] = copies + (int)at - 1;
    copies += (int)all_copies;
    wrong += (int)all_bad;
  }
  __syncthreads();  // the last read of `first` as such
  FreePages<COUNTED> pool(sc.counts);
  int found = 0;
  for (int span = 0; span < a.n_pages && found < copies; span += PC_SPAN) {
    pool.count(a.refs, a.n_pages, span);
    pool.list_pages(a.n_pages, found, 0, copies, first);
    found += pool.all;
  }
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
    a.status[2] = wrong;
  }
}

constexpr int REFS_THREADS = 256;
// Rows up to which one workgroup does all, a wave each: 16 rows of two layers, copies
// included, 11.7 us in one launch, 12.2 in two; 32 rows 13.9, 12.4.
constexpr int REORDER_ONE = PC_WAVES;

__global__ void __launch_bounds__(REFS_THREADS) paged_refs_kernel(const ReorderArgs a) {
  const int r = blockIdx.x * (REFS_THREADS / 64) + (threadIdx.x >> 6);
  if (r < a.batch) count_refs(a, r);
}

// Workgroup 0 places the copies, the others write 16 rows each: two launches, since the pages
// that no row holds any more must be known first.  Round trips bound both: 512 rows of 128
// blocks 5.2 + 8.6 us.
__global__ void __launch_bounds__(PC_THREADS) paged_tables_kernel(const ReorderArgs a) {
  __shared__ CopyScratch sc;
  if (blockIdx.x == 0) {
    place_copies<false>(a, sc);
    return;
  }
  const int r = (blockIdx.x - 1) * PC_WAVES + (threadIdx.x >> 6);
  if (r < a.batch) write_table(a, r);
}

// All of it in one workgroup, for few rows (16 of 4 blocks: 6.2 us).
__global__ void __launch_bounds__(PC_THREADS) paged_reorder_kernel(const ReorderArgs a) {
  __shared__ CopyScratch sc;
  const int r = threadIdx.x >> 6;
  if (r < a.batch) count_refs(a, r);
  // Once the sums are done in L2 (this wait; a fence for the whole device takes 2.6 us),
  // place_copies reads them there.
  __builtin_amdgcn_s_waitcnt(0);
  __syncthreads();
  if (r < a.batch) write_table(a, r);
  place_copies<true>(a, sc);
}

// Workgroup (row, 2 * layer + which): the open page's tokens, one contiguous run (512 rows,
// two layers of 512 in bf16: 6.1 us).
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
  // (row numbers step past the last row by less than 2^30)
  if (rows < 0 || rows > (1 << 30))
    return fail(CDML_E_INVALID, "cdml_paged_plan: rows %d outside [0, 2^30]", rows);
  if (!cu_new || !status || (rows && (!slots || !positions)) ||
      (batch && (!page_refs || !block_table || !kv_len || !new_len)))
    return fail(CDML_E_INVALID, "cdml_paged_plan: NULL pointer");
  if (!aligned16(page_refs)) return fail(CDML_E_INVALID, "cdml_paged_plan: page_refs is not 16-byte aligned");
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
  // (8 x 256 rows 10.0 us so, 13.0 with a launch of their own; 8 x 1021 10.4, 12.9; 32 x 1021
  // 19.7 so, 14.6)
  a.fill = rows <= 8 * PC_THREADS;
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
  if (!aligned16(page_refs)) return fail(CDML_E_INVALID, "cdml_paged_reorder: page_refs is not 16-byte aligned");
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
  const hipStream_t st = as_hip(stream);
  if (batch <= REORDER_ONE) {
    paged_reorder_kernel<<<1, PC_THREADS, 0, st>>>(a);
    return check_launch("paged_reorder_kernel");
  }
  paged_refs_kernel<<<(batch + 3) / 4, REFS_THREADS, 0, st>>>(a);
  rc = check_launch("paged_refs_kernel");
  if (rc) return rc;
  paged_tables_kernel<<<1 + (batch + PC_WAVES - 1) / PC_WAVES, PC_THREADS, 0, st>>>(a);
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
