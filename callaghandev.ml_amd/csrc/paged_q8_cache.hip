// Data movement of 8-bit paged caches (include/cdml.h): rows quantised as they are written,
// the copies of a reordering, and cached rows of any type read back as fp32.
#include <algorithm>

#include "paged.h"

namespace cdml {
namespace {

// ---- append -----------------------------------------------------------------

struct Append8Args {
  const float *k, *v;
  int ldk, ldv;
  uint8_t *kc, *vc;
  float *ks, *vs;
  const int *slots;
  int units, n_slots, page_shift, heads, hd, width;  // units: rows * heads
  UDiv by_heads;
};

// The largest x over groups of L neighbouring lanes, in each of them.
template <int L>
__device__ __forceinline__ uint32_t lanes_most(uint32_t x) {
  x = max(x, dpp<0xB1>(x));
  x = max(x, dpp<0x4E>(x));
  if constexpr (L >= 8) x = max(x, dpp<0x141>(x));
  if constexpr (L >= 16) x = max(x, dpp<0x140>(x));
  if constexpr (L >= 32) {
    auto r = __builtin_amdgcn_permlane16_swap(x, x, false, false);
    x = max(r[0], r[1]);
  }
  if constexpr (L >= 64) {
    auto r = __builtin_amdgcn_permlane32_swap(x, x, false, false);
    x = max(r[0], r[1]);
  }
  return x;
}

// The whole number nearest to x / s, ties to even: the product with 1 / s is off by one at
// most, and what it leaves of x is exact (a multiple of half of s's last bit, below s).
__device__ __forceinline__ int nearest(float x, float s, float inverse) {
  float k = rintf(x * inverse);
  const float rest = fmaf(-k, s, x), half = 0.5f * s;
  const bool odd = (int)k & 1;
  if (rest > half || (rest == half && odd)) k += 1.f;
  if (rest < -half || (rest == -half && odd)) k -= 1.f;
  return (int)k;
}

// L lanes take a row of a K/V head, four values each.  The maximum is one of bit patterns,
// in which infinities and NaNs lie above all numbers: such a row gets the scale NaN.
// 4 x 4096 tokens, 16 heads of 64, f8: 37 us, 4.6 TB/s of reads and writes (a 2 GiB copy of torch's
// 4.9) where the rows come from memory, 31 where they are the last call's again; two rows of a
// thread on the way take as long, four longer.
template <bool F8, int L, bool VEC>
__global__ void __launch_bounds__(256) paged_append8_kernel(const Append8Args a) {
  const bool second = blockIdx.y != 0;
  const float *src = second ? a.v : a.k;
  const int ld = second ? a.ldv : a.ldk, d = 4 * (threadIdx.x % L);
  const int step = gridDim.x * (256 / L);
  for (int u = blockIdx.x * (256 / L) + threadIdx.x / L; u < a.units; u += step) {
    const int row = a.by_heads.div(u), h = u - row * a.heads;
    const int slot = a.slots[row];
    const float *p = src + (size_t)row * ld + (size_t)h * a.hd + d;
    float x[4];
    if constexpr (VEC) {
      const vf4 t = d < a.hd ? *reinterpret_cast<const vf4 *>(p) : vf4{};
#pragma unroll
      for (int c = 0; c < 4; ++c) x[c] = t[c];
    } else {
#pragma unroll
      for (int c = 0; c < 4; ++c) x[c] = d + c < a.hd ? p[c] : 0.f;
    }
    uint32_t most = 0;
#pragma unroll
    for (int c = 0; c < 4; ++c) most = max(most, __float_as_uint(x[c]) & 0x7fffffffu);
    most = lanes_most<L>(most);
    uint32_t codes = 0;
    float scale = 0.f;
    if (most >= 0x7f800000u) {
      scale = __uint_as_float(0x7fc00000u);
    } else if (most != 0) {
      if constexpr (F8) {
        // the least power of two that brings 1.m 2^e to 448 = 1.75 2^8 or less, 2^-126 at least
        const int e = max((int)(most >> 23) - 8 + ((most & 0x7fffffu) > 0x600000u), 1);
        const float inverse = __uint_as_float((uint32_t)(254 - e) << 23);
        scale = __uint_as_float((uint32_t)e << 23);
        codes = __builtin_amdgcn_cvt_pk_fp8_f32(x[0] * inverse, x[1] * inverse, codes, false);
        codes = __builtin_amdgcn_cvt_pk_fp8_f32(x[2] * inverse, x[3] * inverse, codes, true);
      } else {
        scale = fmaxf(__uint_as_float(most) / 127.f, 0x1p-126f);
        const float inverse = 1.f / scale;
#pragma unroll
        for (int c = 0; c < 4; ++c) codes |= (uint32_t)(nearest(x[c], scale, inverse) & 0xff) << 8 * c;
      }
    }
    if ((unsigned)slot >= (unsigned)a.n_slots) continue;
    const int at = slot & ((1 << a.page_shift) - 1);
    const size_t to = ((size_t)((slot >> a.page_shift) * (long long)a.heads + h) << a.page_shift) + at;
    if (d < a.width) *reinterpret_cast<uint32_t *>((second ? a.vc : a.kc) + to * a.width + d) = codes;
    if (d == 0) (second ? a.vs : a.ks)[to] = scale;
  }
}

template <bool F8, int L>
void launch_append8(const Append8Args &a, hipStream_t st) {
  const bool vec = a.hd % 4 == 0 && a.ldk % 4 == 0 && a.ldv % 4 == 0 && aligned16(a.k) && aligned16(a.v);
  const int blocks = (int)(((long long)a.units * L + 255) / 256);
  const dim3 grid(blocks < 65536 ? blocks : 65536, 2);
  if (vec) paged_append8_kernel<F8, L, true><<<grid, 256, 0, st>>>(a);
  else paged_append8_kernel<F8, L, false><<<grid, 256, 0, st>>>(a);
}

template <bool F8>
void launch_append8(const Append8Args &a, hipStream_t st) {
  if (a.width <= 16) launch_append8<F8, 4>(a, st);
  else if (a.width <= 32) launch_append8<F8, 8>(a, st);
  else if (a.width <= 64) launch_append8<F8, 16>(a, st);
  else if (a.width <= 128) launch_append8<F8, 32>(a, st);
  else launch_append8<F8, 64>(a, st);
}

// ---- copy -------------------------------------------------------------------

// Workgroups (row, 2 * layer + which): of every head the open page's codes, 16 bytes a
// thread, and its scales.
__global__ void __launch_bounds__(256) paged_copy8_kernel(uint8_t *kc, uint8_t *vc, float *ks, float *vs,
                                                          size_t layer_rows, int n_pages, int page_shift, int heads,
                                                          int width, const int *__restrict__ src,
                                                          const int *__restrict__ dst,
                                                          const int *__restrict__ kv_len) {
  const int r = blockIdx.x, from = src[r], to = dst[r];
  if ((unsigned)from >= (unsigned)n_pages || (unsigned)to >= (unsigned)n_pages) return;
  const int n = kv_len[r] & ((1 << page_shift) - 1);
  if (n == 0) return;
  const size_t layer = (blockIdx.y >> 1) * layer_rows;
  const size_t s = layer + ((size_t)from * heads << page_shift), d = layer + ((size_t)to * heads << page_shift);
  uint8_t *codes = (blockIdx.y & 1) ? vc : kc;
  float *scales = (blockIdx.y & 1) ? vs : ks;
  const unsigned t = blockIdx.z * 256 + threadIdx.x, all = gridDim.z * 256;
  const unsigned per = (unsigned)(n * (width >> 4)), total = per * heads;  // (below 2^32: see the entry)
  for (unsigned i = t; i < total; i += all) {
    const unsigned h = i / per;
    const size_t at = ((size_t)h << page_shift) * width + 16 * (size_t)(i - h * per);
    *reinterpret_cast<vu4 *>(codes + d * width + at) = *reinterpret_cast<const vu4 *>(codes + s * width + at);
  }
  for (unsigned i = t; i < (unsigned)(n * heads); i += all) {
    const unsigned h = i / n;
    const size_t at = ((size_t)h << page_shift) + (i - h * n);
    scales[d + at] = scales[s + at];
  }
}

// ---- read -------------------------------------------------------------------

struct ReadArgs {
  const void *kc, *vc;
  const float *ks, *vs;
  int n_pages, page_shift;
  const int *table;
  int max_blocks;
  const int *kv_len, *cu;
  float *k, *v;
  int ldk, ldv, rows, batch, heads, hd, width;
  int per_head, per_row, block_rows;  // stores of a head and of a row, rows of a workgroup
  int *bad;
  UDiv by_head, by_row;
};

constexpr int kReadRows = 64;  // most rows of a workgroup
enum : int { kNoRow = -2, kNoToken = -1 };

// The slot of a row's token (a wave's question): kNoRow where no request has the row, kNoToken
// where its request has no such token or the token's page is none.
__device__ __forceinline__ int slot_of_row(const ReadArgs &a, int row) {
  const int lane = threadIdx.x & 63;
  // the requests that end at or before the row: of every `step`-th, then between two of them
  const int step = (a.batch + 63) / 64;
  const int coarse = min((lane + 1) * step, a.batch);
  const int n = __popcll(__builtin_amdgcn_ballot_w64((lane + 1) * step <= a.batch && a.cu[coarse] <= row));
  int b = n * step;
  const int fine = min(b + lane + 1, a.batch);
  b += __popcll(__builtin_amdgcn_ballot_w64(lane < step && b + lane < a.batch && a.cu[fine] <= row));
  if (b >= a.batch) return kNoRow;
  const int first = max(a.cu[b], 0), end = a.cu[b + 1];
  if (row < first || row >= end) return kNoRow;
  const long long most = (long long)a.max_blocks << a.page_shift;
  const int len = (int)min((long long)max(a.kv_len[b], 0), most);
  const int t = len - (end - row);
  if (t < 0) return kNoToken;
  const int page = a.table[(size_t)b * a.max_blocks + (t >> a.page_shift)];
  if ((unsigned)page >= (unsigned)a.n_pages) {
    if (a.bad && lane == 0) *a.bad = 1;
    return kNoToken;
  }
  return (page << a.page_shift) + (t & ((1 << a.page_shift) - 1));
}

// W cached values as they are loaded, and as fp32.
template <int TYPE, int W>
struct Cached {
  static constexpr bool Q8 = TYPE == CDML_CACHE_I8 || TYPE == CDML_CACHE_F8;
  typedef typename std::conditional<
      TYPE == CDML_CACHE_F32, float,
      typename std::conditional<TYPE == CDML_CACHE_F16, _Float16,
                                typename std::conditional<Q8, uint8_t, __bf16>::type>::type>::type T;
  typedef T Values __attribute__((ext_vector_type(W)));
  Values x;
  float scale;

  __device__ __forceinline__ void load(const void *cache, size_t at) {
    const T *p = static_cast<const T *>(cache) + at;
    if constexpr (W == 1) x = *p;
    else x = *reinterpret_cast<const Values *>(p);
  }
  __device__ __forceinline__ void values(float (&y)[W]) const {
    if constexpr (Q8) {
      uint32_t w;
      if constexpr (W == 1) w = x[0];
      else w = __builtin_bit_cast(uint32_t, x);
      if constexpr (TYPE == CDML_CACHE_F8) {
        const auto lo = __builtin_amdgcn_cvt_pk_f32_fp8(w, false);
        y[0] = lo[0] * scale;
        if constexpr (W == 4) {
          const auto hi = __builtin_amdgcn_cvt_pk_f32_fp8(w, true);
          y[1] = lo[1] * scale;
          y[2] = hi[0] * scale;
          y[3] = hi[1] * scale;
        }
      } else {
#pragma unroll
        for (int c = 0; c < W; ++c) y[c] = (float)(int8_t)(w >> 8 * c) * scale;
      }
    } else {
#pragma unroll
      for (int c = 0; c < W; ++c) y[c] = (float)x[c];
    }
  }
};

// A workgroup finds its rows' slots, then streams them: W values a thread and store, four of
// those on the way.  Outputs beyond the L2s are stored past them (24 ragged requests, 8 heads of
// 128, i8, 670 MB: 169 us, 4.9 TB/s of reads and writes; stored as usual 214, a store at a time 192).
template <int TYPE, bool VEC, bool STREAM>
__global__ void __launch_bounds__(256) paged_read_kernel(const ReadArgs a) {
  constexpr int W = VEC ? 4 : 1, U = 4;
  typedef Cached<TYPE, W> Item;
  __shared__ int slots[kReadRows];
  const long long block = (long long)blockIdx.z * gridDim.x + blockIdx.x;
  if (block * a.block_rows >= a.rows) return;
  const int row0 = (int)block * a.block_rows, n_rows = min(a.block_rows, a.rows - row0);
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  for (int i = wave; i < n_rows; i += 4) {
    const int s = slot_of_row(a, row0 + i);
    if ((threadIdx.x & 63) == 0) slots[i] = s;
  }
  __syncthreads();
  const bool second = blockIdx.y != 0;
  const void *cache = second ? a.vc : a.kc;
  float *out = second ? a.v : a.k;
  const int ld = second ? a.ldv : a.ldk;
  const int total = n_rows * a.per_row;
  for (int i0 = threadIdx.x; i0 < total; i0 += 256 * U) {
    Item item[U];
    float *to[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int i = min(i0 + 256 * u, total - 1);
      const int r = a.by_row.div(i), j = i - r * a.per_row, h = a.by_head.div(j), d = W * (j - h * a.per_head);
      const int slot = slots[r];
      to[u] = i0 + 256 * u < total && slot != kNoRow ? out + (size_t)(row0 + r) * ld + (size_t)h * a.hd + d : nullptr;
      item[u].x = typename Item::Values{};
      item[u].scale = 0.f;
      if (slot < 0) continue;
      if constexpr (Item::Q8) {
        const int at = slot & ((1 << a.page_shift) - 1);
        const size_t row = ((size_t)((slot >> a.page_shift) * (long long)a.heads + h) << a.page_shift) + at;
        item[u].scale = (second ? a.vs : a.ks)[row];
        item[u].load(cache, row * a.width + d);
      } else {
        item[u].load(cache, (size_t)slot * ((size_t)a.heads * a.hd) + (size_t)h * a.hd + d);
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (!to[u]) continue;
      float y[W];
      item[u].values(y);
      if constexpr (VEC) {
        const vf4 z = {y[0], y[1], y[2], y[3]};
        if constexpr (STREAM) __builtin_nontemporal_store(z, reinterpret_cast<vf4 *>(to[u]));
        else *reinterpret_cast<vf4 *>(to[u]) = z;
      } else {
        *to[u] = y[0];
      }
    }
  }
}

template <int TYPE>
void launch_read(const ReadArgs &a, bool vec, bool stream, dim3 grid, hipStream_t st) {
  if (vec && stream) paged_read_kernel<TYPE, true, true><<<grid, 256, 0, st>>>(a);
  else if (vec) paged_read_kernel<TYPE, true, false><<<grid, 256, 0, st>>>(a);
  else paged_read_kernel<TYPE, false, false><<<grid, 256, 0, st>>>(a);
}

// The checks of heads that an 8-bit cache, or a reader, has.
int check_heads(const char *what, int heads, int hd) {
  if (heads <= 0 || hd <= 0 || hd > 256 || (long long)heads * hd > INT_MAX / 4)
    return fail(CDML_E_INVALID, "%s: bad heads (%d of %d, of at most 256)", what, heads, hd);
  return CDML_OK;
}

}  // namespace
}  // namespace cdml

using namespace cdml;

extern "C" int cdml_paged_append_q8(const float *k_new, int ldk, const float *v_new, int ldv, void *kcache,
                                    void *vcache, float *kscale, float *vscale, int cache_type, const int *slots,
                                    int rows, int n_pages, int page_size, int num_kv_heads, int head_dim,
                                    cdml_stream stream) {
  Append8Args a{};
  int rc = check_pool("cdml_paged_append_q8", n_pages, page_size, 1, 0, &a.page_shift);
  if (rc) return rc;
  if (!q8_cache_type(cache_type))
    return fail(CDML_E_INVALID, "cdml_paged_append_q8: cache type %d is none of 8 bits", cache_type);
  rc = check_heads("cdml_paged_append_q8", num_kv_heads, head_dim);
  if (rc) return rc;
  const int dim = num_kv_heads * head_dim;
  if (rows < 0 || ldk < dim || ldv < dim || (long long)rows * num_kv_heads > INT_MAX / 2)
    return fail(CDML_E_INVALID, "cdml_paged_append_q8: bad size (rows %d, %d heads of %d, ldk %d, ldv %d)", rows,
                num_kv_heads, head_dim, ldk, ldv);
  if (rows == 0) return CDML_OK;
  if (!k_new || !v_new || !slots) return fail(CDML_E_INVALID, "cdml_paged_append_q8: NULL pointer");
  rc = check_q8("cdml_paged_append_q8", kcache, vcache, kscale, vscale);
  if (rc) return rc;
  rc = ensure_device();
  if (rc) return rc;
  a.k = k_new;
  a.v = v_new;
  a.ldk = ldk;
  a.ldv = ldv;
  a.kc = static_cast<uint8_t *>(kcache);
  a.vc = static_cast<uint8_t *>(vcache);
  a.ks = kscale;
  a.vs = vscale;
  a.slots = slots;
  a.units = rows * num_kv_heads;
  a.n_slots = n_pages * page_size;
  a.heads = num_kv_heads;
  a.hd = head_dim;
  a.width = q8_width(head_dim);
  a.by_heads = UDiv::make((uint32_t)num_kv_heads);
  if (cache_type == CDML_CACHE_F8) launch_append8<true>(a, as_hip(stream));
  else launch_append8<false>(a, as_hip(stream));
  return check_launch("paged_append8_kernel");
}

extern "C" int cdml_paged_copy_q8(void *kcache, void *vcache, float *kscale, float *vscale, int layers,
                                  size_t layer_stride, int n_pages, int page_size, int num_kv_heads, int head_dim,
                                  const int *copy_src, const int *copy_dst, const int *kv_len, int batch,
                                  cdml_stream stream) {
  int shift = 0;
  int rc = check_pool("cdml_paged_copy_q8", n_pages, page_size, 1, batch, &shift);
  if (rc) return rc;
  rc = check_heads("cdml_paged_copy_q8", num_kv_heads, head_dim);
  if (rc) return rc;
  const size_t page = (size_t)page_size * num_kv_heads * q8_width(head_dim);
  if (layers < 0 || layers > 32767 || page > INT_MAX)
    return fail(CDML_E_INVALID, "cdml_paged_copy_q8: bad size (layers %d, pages of %zu bytes)", layers, page);
  if (layers > 1 && layer_stride < (size_t)n_pages * page_size)
    return fail(CDML_E_INVALID, "cdml_paged_copy_q8: layer_stride smaller than a layer's cache");
  if (batch == 0 || layers == 0) return CDML_OK;
  if (!copy_src || !copy_dst || !kv_len) return fail(CDML_E_INVALID, "cdml_paged_copy_q8: NULL pointer");
  rc = check_q8("cdml_paged_copy_q8", kcache, vcache, kscale, vscale);
  if (rc) return rc;
  rc = ensure_device();
  if (rc) return rc;
  size_t parts = (page + 16383) / 16384;  // (4 16-byte units a thread)
  if (parts > 64) parts = 64;
  paged_copy8_kernel<<<dim3(batch, 2 * layers, (unsigned)parts), 256, 0, as_hip(stream)>>>(
      static_cast<uint8_t *>(kcache), static_cast<uint8_t *>(vcache), kscale, vscale, layer_stride * num_kv_heads,
      n_pages, shift, num_kv_heads, q8_width(head_dim), copy_src, copy_dst, kv_len);
  return check_launch("paged_copy8_kernel");
}

extern "C" int cdml_paged_read(const void *kcache, const void *vcache, const float *kscale, const float *vscale,
                               int cache_type, int n_pages, int page_size, const int *block_table, int max_blocks,
                               const int *kv_len, const int *cu_rows, float *k_out, int ldk, float *v_out, int ldv,
                               int rows, int batch, int num_kv_heads, int head_dim, int *bad, cdml_stream stream) {
  ReadArgs a{};
  int rc = check_pool("cdml_paged_read", n_pages, page_size, max_blocks, batch, &a.page_shift);
  if (rc) return rc;
  const int size = cache_type_bytes(cache_type);
  if (!size && !q8_cache_type(cache_type))
    return fail(CDML_E_INVALID, "cdml_paged_read: unknown cache type %d", cache_type);
  rc = check_heads("cdml_paged_read", num_kv_heads, head_dim);
  if (rc) return rc;
  const int dim = num_kv_heads * head_dim;
  if (rows < 0 || ldk < dim || ldv < dim)
    return fail(CDML_E_INVALID, "cdml_paged_read: bad size (rows %d, %d heads of %d, ldk %d, ldv %d)", rows,
                num_kv_heads, head_dim, ldk, ldv);
  if (rows == 0 || batch == 0) return CDML_OK;
  if (!kcache || !vcache || !block_table || !kv_len || !cu_rows || !k_out || !v_out)
    return fail(CDML_E_INVALID, "cdml_paged_read: NULL pointer");
  if (!size) {
    rc = check_q8("cdml_paged_read", kcache, vcache, kscale, vscale);
    if (rc) return rc;
  }
  rc = ensure_device();
  if (rc) return rc;
  // (an 8-bit cache is aligned, its rows too)
  const bool vec = head_dim % 4 == 0 && ldk % 4 == 0 && ldv % 4 == 0 && aligned16(k_out) && aligned16(v_out) &&
                   aligned16(kcache) && aligned16(vcache);
  a.kc = kcache;
  a.vc = vcache;
  a.ks = kscale;
  a.vs = vscale;
  a.n_pages = n_pages;
  a.table = block_table;
  a.max_blocks = max_blocks;
  a.kv_len = kv_len;
  a.cu = cu_rows;
  a.k = k_out;
  a.v = v_out;
  a.ldk = ldk;
  a.ldv = ldv;
  a.rows = rows;
  a.batch = batch;
  a.heads = num_kv_heads;
  a.hd = head_dim;
  a.width = q8_width(head_dim);
  a.bad = bad;
  a.per_head = vec ? head_dim / 4 : head_dim;
  a.per_row = a.per_head * num_kv_heads;
  // about eight stores a thread
  const int block_rows = 2048 / a.per_row;
  a.block_rows = block_rows < 1 ? 1 : block_rows > kReadRows ? kReadRows : block_rows;
  const bool past = (size_t)rows * dim * 8 > (32u << 20);
  a.by_head = UDiv::make((uint32_t)a.per_head);
  a.by_row = UDiv::make((uint32_t)a.per_row);
  // an axis of a launch holds less than 2^32 threads, and one of more runs short without an error:
  // from 2^23 workgroups on, the third axis counts the turns of the first
  const unsigned blocks = (unsigned)((rows - 1) / a.block_rows) + 1, along = std::min(blocks, 1u << 23);
  const dim3 grid(along, 2, (blocks - 1) / along + 1);
  const hipStream_t st = as_hip(stream);
  switch (cache_type) {
    case CDML_CACHE_F32: launch_read<CDML_CACHE_F32>(a, vec, past, grid, st); break;
    case CDML_CACHE_F16: launch_read<CDML_CACHE_F16>(a, vec, past, grid, st); break;
    case CDML_CACHE_BF16: launch_read<CDML_CACHE_BF16>(a, vec, past, grid, st); break;
    case CDML_CACHE_I8: launch_read<CDML_CACHE_I8>(a, vec, past, grid, st); break;
    default: launch_read<CDML_CACHE_F8>(a, vec, past, grid, st);
  }
  return check_launch("paged_read_kernel");
}
