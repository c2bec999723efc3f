// The attention kernels over a paged cache, for one cache type T (float, _Float16 or
// __bf16; included by a file each).
#pragma once

#include "paged.h"

namespace cdml {
namespace {

// Four cached values as they are loaded.
template <typename T>
struct Raw4 {
  typedef vu2 type;
};
template <>
struct Raw4<float> {
  typedef vf4 type;
};

__device__ __forceinline__ float half_value(uint32_t w, int i, _Float16) {
  return (float)__builtin_bit_cast(_Float16, (uint16_t)(i ? w >> 16 : w & 0xffffu));
}
__device__ __forceinline__ float half_value(uint32_t w, int i, __bf16) {
  return __uint_as_float(i ? w & 0xffff0000u : w << 16);
}

// ---- one to four rows: vector units -------------------------------------------

constexpr int PR_THREADS = 256;

// Sum over groups of LPK (8 or 16) neighbouring lanes, in each of them.
template <int LPK>
__device__ __forceinline__ float lanes_sum(float x) {
  x += dpp<0xB1>(x);
  x += dpp<0x4E>(x);
  x += dpp<0x141>(x);
  if constexpr (LPK == 16) x += dpp<0x140>(x);
  return x;
}

// How rows are read: value by value (any head dim, any alignment), in 16-byte aligned
// vectors, or in vectors of which a lane's past the head dim (a multiple of 8) are zeros.
enum { kScalar = 0, kVector = 1, kVectorCut = 2 };

// A lane's EPL values of one cached row: NV loads of VW values, LPK * VW apart.
template <typename T, int VW, int NV, int LPK, int MODE>
struct RowSlice {
  static constexpr int WORDS = VW * NV * (int)sizeof(T) / 4;
  static_assert(VW * sizeof(T) % 4 == 0, "whole words");
  uint32_t w[WORDS];

  __device__ __forceinline__ void load(const T *p, int d0, int hd, bool zero) {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      constexpr int LW = WORDS / NV;  // words per load
      if constexpr (MODE != kScalar) {
        typedef uint32_t V __attribute__((ext_vector_type(LW)));
        if (MODE == kVectorCut && d0 + LPK * VW * i >= hd) {
#pragma unroll
          for (int c = 0; c < LW; ++c) w[i * LW + c] = 0;
        } else if constexpr (LW == 1) {
          w[i] = __builtin_nontemporal_load(reinterpret_cast<const uint32_t *>(p + LPK * VW * i));
        } else {
          const V t = __builtin_nontemporal_load(reinterpret_cast<const V *>(p + LPK * VW * i));
#pragma unroll
          for (int c = 0; c < LW; ++c) w[i * LW + c] = t[c];
        }
      } else {
#pragma unroll
        for (int c = 0; c < LW; ++c) w[i * LW + c] = 0;
#pragma unroll
        for (int c = 0; c < VW; ++c) {
          if (d0 + LPK * VW * i + c >= hd) continue;
          if constexpr (sizeof(T) == 4) w[i * LW + c] = __builtin_bit_cast(uint32_t, p[LPK * VW * i + c]);
          else w[i * LW + c / 2] |= (uint32_t)__builtin_bit_cast(uint16_t, p[LPK * VW * i + c]) << 16 * (c & 1);
        }
      }
    }
    if (zero) {
#pragma unroll
      for (int c = 0; c < WORDS; ++c) w[c] = 0;
    }
  }
  __device__ __forceinline__ float value(int e) const {
    if constexpr (sizeof(T) == 4) return __uint_as_float(w[e]);
    else return half_value(w[e / 2], e & 1, T{});
  }
};

// One workgroup: R rows of a (request, K/V head) against one chunk of its keys; a cached
// row goes through LPK lanes, its score through their sum, and every group of LPK lanes
// keeps an online softmax of its own keys.  The four waves take 64 / LPK keys in turn.
// U sets of rows go round, so that the loads of U - 1 steps are in flight while one is
// consumed: four where 64 registers hold them (8 x 2048 keys of bf16, 16 heads of 64: 15.0
// -> 14.4 us).  HBM bounds it: 64 x 8192 keys, 16 heads of 128, fp32 1248 us, 6.9 TB/s.
template <typename T, int HD, int R, int MODE>
__global__ void __launch_bounds__(PR_THREADS) paged_rows_kernel(const PagedArgs a) {
  constexpr int LPK = HD >= 64 && R > 2 ? 16 : 8;
  constexpr int EPL = HD / LPK;                                              // values per lane
  constexpr int VW = EPL * sizeof(T) >= 16 ? 16 / (int)sizeof(T) : EPL;      // per load
  constexpr int NV = EPL / VW, KPS = 64 / LPK;
  typedef RowSlice<T, VW, NV, LPK, MODE> Slice;
  constexpr int U = Slice::WORDS <= 8 ? 4 : 2;
  __shared__ int pages[kPagedSub + 1];
  __shared__ float red_m[4][R], red_l[4][R];
  __shared__ float red_o[4][R][HD];

  const int b = blockIdx.z;
  const PagedSeq s = paged_seq(a, b);
  const int nr = s.n * a.group;
  if (nr == 0 || nr > a.few_rows) return;
  const int hk = blockIdx.y % a.kv_heads, r0 = blockIdx.y / a.kv_heads * R;
  if (r0 >= nr) return;
  const int split = blockIdx.x, base = s.len - s.n;  // token i sees keys up to base + i
  const bool single = s.len <= a.few_chunk;
  const int kend = base + a.by_group.div(min(r0 + R, nr) - 1) + 1;  // past the last visible key
  const int c0 = split * a.few_chunk, c1 = min(c0 + a.few_chunk, kend);
  if (c0 >= c1 && !(single && split == 0)) return;

  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int g = lane / LPK, d0 = VW * (lane % LPK);
  const int P1 = (1 << a.page_shift) - 1, kv_dim = a.kv_heads * a.hd;

  float q[R][EPL], o[R][EPL], m[R], l[R];
  int lim[R];
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const int rr = min(r0 + r, nr - 1), i = a.by_group.div(rr);
    lim[r] = base + i;
    const float *qr = a.q + (size_t)(s.first + i) * a.ldq + (size_t)(hk * a.group + rr - i * a.group) * a.hd;
#pragma unroll
    for (int e = 0; e < EPL; ++e) {
      const int d = d0 + LPK * VW * (e / VW) + e % VW;
      q[r][e] = MODE == kVector || d < a.hd ? qr[d] * a.scale_log2 : 0.f;
      o[r][e] = 0.f;
    }
    m[r] = kNoKey;
    l[r] = 0.f;
  }

  const T *kb = static_cast<const T *>(a.kc) + (size_t)hk * a.hd + d0;
  const T *vb = static_cast<const T *>(a.vc) + (size_t)hk * a.hd + d0;
  for (int sub = c0; sub < c1; sub += kPagedSub) {
    const int end = min(sub + kPagedSub, c1), block0 = sub >> a.page_shift;
    const int n_blocks = ((end - 1) >> a.page_shift) - block0 + 1;
    if (sub > c0) __syncthreads();
    int wrong = 0;
    for (int i = threadIdx.x; i < n_blocks; i += PR_THREADS) {
      const int page = a.table[(size_t)b * a.max_blocks + block0 + i];
      const bool ok = (unsigned)page < (unsigned)a.n_pages;
      pages[i] = ok ? page : -1;
      wrong |= !ok;
    }
    const bool any_wrong = __syncthreads_or(wrong) != 0;
    if (any_wrong && a.bad && threadIdx.x == 0) *a.bad = 1;

    // keys past the end read the last one and are left out below
    auto fetch = [&](int key, Slice &kr, Slice &vr) {
      key = min(key, end - 1);
      const int page = pages[(key >> a.page_shift) - block0];
      const size_t at = ((size_t)(max(page, 0) << a.page_shift) + (key & P1)) * kv_dim;
      kr.load(kb + at, d0, a.hd, any_wrong && page < 0);
      vr.load(vb + at, d0, a.hd, any_wrong && page < 0);
    };
    auto step = [&](int key, const Slice &kr, const Slice &vr) {
      float sc[R];
#pragma unroll
      for (int r = 0; r < R; ++r) sc[r] = 0.f;
#pragma unroll
      for (int e = 0; e < EPL; ++e) {
        const float x = kr.value(e);
#pragma unroll
        for (int r = 0; r < R; ++r) sc[r] = fmaf(q[r][e], x, sc[r]);
      }
#pragma unroll
      for (int r = 0; r < R; ++r) sc[r] = lanes_sum<LPK>(sc[r]);
#pragma unroll
      for (int r = 0; r < R; ++r) {
        if (key <= lim[r] && key < end) {
          const float mn = fmaxf(m[r], sc[r]);
          const float alpha = fast_exp2(m[r] - mn), p = fast_exp2(sc[r] - mn);
          l[r] = fmaf(l[r], alpha, p);
#pragma unroll
          for (int e = 0; e < EPL; ++e) o[r][e] = fmaf(p, vr.value(e), o[r][e] * alpha);
          m[r] = mn;
        }
      }
    };
    Slice k[U], v[U];
    const int key0 = sub + wave * KPS + g, steps = (end - sub + 4 * KPS - 1) / (4 * KPS);
#pragma unroll
    for (int u = 0; u < U - 1; ++u) fetch(key0 + u * 4 * KPS, k[u], v[u]);
    for (int it = 0; it < steps; it += U) {
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int key = key0 + (it + u) * 4 * KPS;
        fetch(key + (U - 1) * 4 * KPS, k[(u + U - 1) % U], v[(u + U - 1) % U]);
        step(key, k[u], v[u]);
      }
    }
  }

  // the groups of a wave, then the waves
#pragma unroll
  for (int r = 0; r < R; ++r) {
#pragma unroll
    for (int off = LPK; off < 64; off <<= 1) {
      const float m2 = __shfl_xor(m[r], off), l2 = __shfl_xor(l[r], off);
      const float mn = fmaxf(m[r], m2), w1 = fast_exp2(m[r] - mn), w2 = fast_exp2(m2 - mn);
      l[r] = l[r] * w1 + l2 * w2;
#pragma unroll
      for (int e = 0; e < EPL; ++e) o[r][e] = o[r][e] * w1 + __shfl_xor(o[r][e], off) * w2;
      m[r] = mn;
    }
    if (lane == 0) {
      red_m[wave][r] = m[r];
      red_l[wave][r] = l[r];
    }
  }
  __syncthreads();
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const float M = fmaxf(fmaxf(red_m[0][r], red_m[1][r]), fmaxf(red_m[2][r], red_m[3][r]));
    const float w = fast_exp2(m[r] - M);
    if (g == 0) {
#pragma unroll
      for (int e = 0; e < EPL; ++e) red_o[wave][r][d0 + LPK * VW * (e / VW) + e % VW] = o[r][e] * w;
    }
  }
  __syncthreads();
  for (int t = threadIdx.x; t < R * HD; t += PR_THREADS) {
    const int r = t / HD, d = t % HD, rr = r0 + r;
    if (rr >= nr || d >= a.hd) continue;
    const float M = fmaxf(fmaxf(red_m[0][r], red_m[1][r]), fmaxf(red_m[2][r], red_m[3][r]));
    float L = 0.f;
#pragma unroll
    for (int w = 0; w < 4; ++w) L += red_l[w][r] * fast_exp2(red_m[w][r] - M);
    const float x = red_o[0][r][d] + red_o[1][r][d] + red_o[2][r][d] + red_o[3][r][d];
    if (single) {
      const int i = a.by_group.div(rr), h = hk * a.group + rr - i * a.group;
      a.o[(size_t)(s.first + i) * a.ldo + (size_t)h * a.hd + d] = L == 0.f ? 0.f : x / L;
    } else {
      float *part = a.few_part + ((((size_t)b * a.kv_heads + hk) * a.few_rows + rr) * a.few_splits + split) * (a.hd + 2);
      part[d] = x;
      if (d == 0) {
        part[a.hd] = M;
        part[a.hd + 1] = L;
      }
    }
  }
}

// ---- many rows: matrix cores --------------------------------------------------

constexpr int PT_THREADS = 256;

// Pieces of a cached value (common.h): fp32 has three, fp16's eleven bits lie in two,
// bf16 is one; and the products of their pieces with the three of Q or of the
// probabilities that reach fp32's accuracy, the main one last.
template <typename T>
struct Pieces;
template <>
struct Pieces<float> {
  static constexpr int N = 3, PRODUCTS = 6;
  static constexpr int A[6] = {2, 0, 1, 1, 0, 0}, B[6] = {0, 2, 1, 0, 1, 0};
};
template <>
struct Pieces<_Float16> {
  static constexpr int N = 2, PRODUCTS = 5;
  static constexpr int A[5] = {1, 0, 1, 0, 0}, B[5] = {1, 2, 0, 1, 0};
};
template <>
struct Pieces<__bf16> {
  static constexpr int N = 1, PRODUCTS = 3;
  static constexpr int A[3] = {0, 0, 0}, B[3] = {2, 1, 0};
};

// Where a key's row lies in the cache, and whether its page is a page.
struct Slot {
  uint32_t at;
  bool ok;
};
__device__ __forceinline__ Slot slot_in(const PagedArgs &a, int page, int key) {
  const bool ok = (unsigned)page < (unsigned)a.n_pages;
  return {((uint32_t)(ok ? page : 0) << a.page_shift) + (uint32_t)(key & ((1 << a.page_shift) - 1)), ok};
}

// Puts dim c of two neighbouring keys of V (a's the lower one) at place d of its row in
// every piece's plane.
template <typename T>
__device__ __forceinline__ void put_v(char *d, int plane, const typename Raw4<T>::type &a,
                                      const typename Raw4<T>::type &b, int c) {
  constexpr int NP = Pieces<T>::N;
  if constexpr (NP == 1) {
    *reinterpret_cast<uint32_t *>(d) = __builtin_amdgcn_perm(b[c / 2], a[c / 2], c & 1 ? 0x07060302u : 0x05040100u);
  } else {
    uint32_t h, m, l;
    if constexpr (NP == 3) split_bf16x3(a[c] * kSplitScale, b[c] * kSplitScale, h, m, l);
    else split_bf16x3(half_value(a[c / 2], c & 1, T{}), half_value(b[c / 2], c & 1, T{}), h, m, l);
    *reinterpret_cast<uint32_t *>(d) = h;
    *reinterpret_cast<uint32_t *>(d + plane) = m;
    if constexpr (NP == 3) *reinterpret_cast<uint32_t *>(d + 2 * plane) = l;
  }
}

// Four values of a row's columns d .. d + 3 at p, those past the head dim as zeros.
template <typename T>
__device__ __forceinline__ typename Raw4<T>::type load4_cut(const T *p, int d, int hd) {
  typename Raw4<T>::type r;
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int c = 0; c < 4; ++c) r[c] = d + c < hd ? (float)p[c] : 0.f;
  } else {
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      const uint32_t lo = d + 2 * c < hd ? __builtin_bit_cast(uint16_t, p[2 * c]) : 0;
      const uint32_t hi = d + 2 * c + 1 < hd ? __builtin_bit_cast(uint16_t, p[2 * c + 1]) : 0;
      r[c] = lo | hi << 16;
    }
  }
  return r;
}

// Stages one tile of BN keys: K rows and V transposed, of one K/V head, from their pages
// into registers and then, as bf16 pieces, into LDS (one plane per piece, rows of 16
// values = 32 bytes).  The upper half of the workgroup's waves stages K, the lower half V,
// four dims of a key per load.
//   K: slab s holds dims 16 s .. 16 s + 15 of every key: rows are keys, even and odd ones
//      in two clusters.
//   V: slab s holds keys 16 s .. 16 s + 15 of every dim: rows are dims, in four clusters
//      by d % 4.  A unit is four dims of two keys; key k of a slab sits at place
//      8 (k / 4 % 2) + 4 (k / 8) + k % 4, the order the P.V product reads.
// The pages of a tile are looked up a tile ahead of its rows.  What masked keys hold never
// matters to the scores; V's rows past the request's last key are staged as zeros, for the
// probabilities that they meet are exactly 0.
//   UNI (16-byte aligned rows, pages of 16 keys or more): the 16 keys of a block lie in one
//      page and a wave's load touches one block, so a load's address is a scalar base plus
//      an offset that the lane keeps throughout.  Lane l holds the base of block l of 64
//      (1024 keys); a tile reads its blocks' from there.  Looking every row's page up
//      instead costs some 50 vector instructions a tile, every block's a chain of 40 scalar
//      ones ahead of the tile's loads.
template <typename T, int HD, int BN, bool VEC, bool UNI>
struct PagedStage {
  typedef typename Raw4<T>::type Raw;
  // Global memory, said so: a load through a pointer made of numbers would be a flat one, and
  // every wait for LDS a wait for it too.
  typedef const __attribute__((address_space(1))) char *GlobalBytes;
  static constexpr int NP = Pieces<T>::N;
  static constexpr int HALF = PT_THREADS / 2;
  static constexpr int KROWB = BN / 2 * 32, VROWB = HD / 4 * 32;  // bytes of one row cluster
  static constexpr int KSLAB = 2 * KROWB + 128, VSLAB = 4 * VROWB + 256;
  static constexpr int KPLANE = HD / 16 * KSLAB, VPLANE = BN / 16 * VSLAB;
  static constexpr int BYTES = NP * (KPLANE + VPLANE);   // K planes, then V planes
  static constexpr int VU = (HD / 4) * (BN / 2) / HALF;  // V units per thread; twice as many K units
  static constexpr int NV = 2 * VU;                      // loads of either
  static constexpr int NB = BN / 16;                     // blocks of 16 keys
  static_assert(VU >= 1 && (HD / 4) * (BN / 2) % HALF == 0, "tile units");
  static __device__ __forceinline__ constexpr int kcluster(int c) { return c * (KROWB + 16); }
  static __device__ __forceinline__ constexpr int vcluster(int c) {
    return c * VROWB + (c & 1) * 16 + (c >> 1) * 128;
  }
  static constexpr int CH = HD / 4, KSTEP = HALF / CH;
  static_assert(16 % KSTEP == 0, "a K load stays in a block of 16 keys");
  static __device__ __forceinline__ constexpr int vgroups(int i) { return HALF / 8 * i % CH; }
  static __device__ __forceinline__ constexpr int vslabs(int i) { return HALF / 8 * i / CH; }
  Raw r[NV];
  int page[UNI ? 1 : NV];  // UNI: lane's block in the next 64, else of the next tile's rows
  uint32_t base_lo, base_hi;  // UNI: the lane's block in these 64
  uint64_t none;              // UNI: those whose page is none
  int group;                  // UNI: first key of these 64 blocks
  uint32_t zero;              // bit i: load i's page is none
  const T *base;            // the head's columns (UNI), this thread's columns
  const int *table;
  int col, row, dst;  // first column, first row in a tile, LDS byte offset of the first unit
  int slab;           // V: the first unit's block (wave-uniform)
  int loaded;         // first key of the tile in r
  int kv_dim, last;   // the request's last key
  bool kside;

  __device__ __forceinline__ void init(const PagedArgs &a, int b, int hk, int last_key) {
    const int t0 = __builtin_amdgcn_readfirstlane(threadIdx.x);
    kside = t0 >= HALF;
    const int t = threadIdx.x & (HALF - 1);
    // K: the P keys of one load instruction share a cluster
    constexpr int P = 64 / CH;
    const int c = t % CH, j = t / CH, kkey = (j & ~(2 * P - 1)) | ((j & (P - 1)) << 1) | ((j / P) & 1);
    const int sb = t & 7, g = (t >> 3) % CH;
    slab = ((t0 & (HALF - 1)) >> 3) / CH;
    const int place = ((sb >> 1) & 1) * 4 + (sb >> 2) * 2 + (sb & 1);  // of V's key pair
    col = kside ? 4 * c : 4 * g;
    row = kside ? kkey : 2 * sb + (UNI ? 0 : 16 * slab);
    dst = kside ? (c >> 2) * KSLAB + kcluster(kkey & 1) + (kkey >> 1) * 32 + (c & 3) * 8
                : NP * KPLANE + slab * VSLAB + g * 32 + place * 4;
    base = static_cast<const T *>(kside ? a.kc : a.vc) + (size_t)hk * a.hd + (UNI ? 0 : col);
    table = a.table + (size_t)b * a.max_blocks;
    kv_dim = a.kv_heads * a.hd;
    last = last_key;
  }
  // Load i's row in the tile, without the lane's part
  __device__ __forceinline__ int row_of(int i) const {
    return kside ? KSTEP * i : 16 * vslabs(i / 2) + (i & 1);
  }
  // UNI: the block of a tile that load i lies in
  __device__ __forceinline__ int block_of(int i) const {
    return kside ? KSTEP * i / 16 : slab + vslabs(i / 2);
  }
  __device__ __forceinline__ int key(int k0, int i) const { return min(k0 + row + row_of(i), last); }
  // UNI: pages of the 64 blocks from key k0 on, one to a lane
  __device__ __forceinline__ int page_of_block(const PagedArgs &a, int k0) const {
    return table[min(k0 + 16 * (int)(threadIdx.x & 63), last) >> a.page_shift];
  }
  __device__ __forceinline__ void start_group(const PagedArgs &a, int k0) {
    const int mine = k0 + 16 * (int)(threadIdx.x & 63);
    const Slot s = slot_in(a, page[0], mine);
    const uint64_t at = reinterpret_cast<uint64_t>(base + (size_t)s.at * kv_dim);
    base_lo = (uint32_t)at;
    base_hi = (uint32_t)(at >> 32);
    none = __builtin_amdgcn_ballot_w64(!s.ok);
    group = k0;
    page[0] = page_of_block(a, k0 + 1024);
  }
  // What load() of the first tile needs; then, after each load, of the next.
  __device__ __forceinline__ void lookup_first(const PagedArgs &a, int k0) {
    if constexpr (UNI) {
      page[0] = page_of_block(a, k0);
      start_group(a, k0);
    } else {
      lookup(a, k0);
    }
  }
  __device__ __forceinline__ void lookup(const PagedArgs &a, int k0) {
    if constexpr (!UNI) {
#pragma unroll
      for (int i = 0; i < NV; ++i) page[i] = table[key(k0, i) >> a.page_shift];
    }
  }

  __device__ __forceinline__ void load(const PagedArgs &a, int k0) {
    loaded = k0;
    if constexpr (UNI) {
      if (k0 - group >= 1024) start_group(a, k0);
      const int first = (k0 - group) >> 4;
      zero = (uint32_t)(none >> first) & ((1u << NB) - 1);  // (a tile's blocks lie in one group)
      GlobalBytes block[NB];
#pragma unroll
      for (int i = 0; i < NB; ++i)
        block[i] = (GlobalBytes)((uint64_t)(uint32_t)__builtin_amdgcn_readlane(base_hi, first + i) << 32 |
                                 (uint32_t)__builtin_amdgcn_readlane(base_lo, first + i));
      // (columns past the head dim read its last four again: Q is 0 there, and what they
      // give O is not stored)
      static_assert(vgroups(1) == 0 || vgroups(2) == 0, "two column offsets");
      uint32_t off[2];
#pragma unroll
      for (int i = 0; i < 2; ++i)
        off[i] = (uint32_t)(row * kv_dim + min(col + 4 * vgroups(i), a.hd - 4)) * (uint32_t)sizeof(T);
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        GlobalBytes p = nullptr;
        const int at = block_of(i);
#pragma unroll
        for (int c = 0; c < NB; ++c) p = at == c ? block[c] : p;
        p += (size_t)(kside ? KSTEP * i % 16 : (i & 1)) * kv_dim * sizeof(T);
        r[i] = *(const __attribute__((address_space(1))) Raw *)(p + off[kside ? 0 : vgroups(i / 2) != 0]);
      }
    } else {
      zero = 0;
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const Slot s = slot_in(a, page[i], key(k0, i));
        if (!s.ok) zero |= 1u << i;
        const int dc = kside ? 0 : 4 * vgroups(i / 2);
        const T *p = base + (size_t)s.at * kv_dim + dc;
        if constexpr (VEC) {
          r[i] = *reinterpret_cast<const Raw *>(p + min(0, a.hd - 4 - col - dc));
        } else {
          r[i] = load4_cut<T>(p, col + dc, a.hd);
        }
      }
    }
  }

  __device__ __forceinline__ void store(char *lds, int *bad) {
    if constexpr (UNI) {
      if (zero || loaded + BN - 1 > last) {  // (wave-uniform)
        if (zero && bad) *bad = 1;
#pragma unroll
        for (int i = 0; i < NV; ++i)
          if ((zero >> block_of(i) & 1) || (!kside && loaded + 16 * slab + row + row_of(i) > last)) r[i] = Raw{};
      }
    } else if (__builtin_amdgcn_ballot_w64(zero != 0)) {
      if (zero && bad) *bad = 1;
#pragma unroll
      for (int i = 0; i < NV; ++i)
        if (zero >> i & 1) r[i] = Raw{};
    }
    if (kside) {
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        char *d = lds + dst + KSTEP / 2 * 32 * i;
        if constexpr (NP == 1) {
          *reinterpret_cast<vu2 *>(d) = r[i];
        } else {
          float x[4];
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            if constexpr (NP == 3) x[c] = r[i][c];
            else x[c] = half_value(r[i][c / 2], c & 1, T{});
          }
          uint32_t h0, m0, l0, h1, m1, l1;
          split_bf16x3(x[0], x[1], h0, m0, l0);
          split_bf16x3(x[2], x[3], h1, m1, l1);
          *reinterpret_cast<vu2 *>(d) = vu2{h0, h1};
          *reinterpret_cast<vu2 *>(d + KPLANE) = vu2{m0, m1};
          if constexpr (NP == 3) *reinterpret_cast<vu2 *>(d + 2 * KPLANE) = vu2{l0, l1};
        }
      }
    } else {
#pragma unroll
      for (int i = 0; i < VU; ++i)
#pragma unroll
        for (int c = 0; c < 4; ++c)
          put_v<T>(lds + dst + vslabs(i) * VSLAB + vgroups(i) * 32 + vcluster(c), VPLANE, r[2 * i], r[2 * i + 1], c);
    }
  }

  // Byte offsets of a lane's operands in a plane: dims 16 s + 8 hf + 0..7 of key
  // row0 + li (row0 a multiple of 32), and eight keys of slab s for dim 32 db + li.
  static __device__ __forceinline__ int koperand(int li, int hf) {
    return kcluster(li & 1) + (li >> 1) * 32 + hf * 16;
  }
  static __device__ __forceinline__ int voperand(int li, int hf) {
    return NP * KPLANE + vcluster(li & 3) + (li >> 2) * 32 + hf * 16;
  }
};

// Q^T operand of a wave: the three bf16 pieces of this lane's row times scale_log2, eight
// values of every `step` (16 or 32, by the MFMA) from 8 * part on.
// Neither Q nor K takes the split's scale, so that scores come out as they are: what a
// component below 2^-110 loses (2^-134) reaches a score only through a component of
// 2^100 and more on the other side.  Returns whether Q holds one or the other
// (wave-uniform); such rows are recomputed on the fp32 MFMA.
template <int N, bool VEC>
__device__ __forceinline__ bool load_q_pieces(bf16x8 (&q)[N][3], const float *qrow, int hd, float scale, int step,
                                              int part) {
  uint32_t most = 0, least = ~0u;  // of |x|, and of 2 |x| - 1 as integers, which leaves zeros out
#pragma unroll
  for (int s = 0; s < N; ++s) {
    float x[8];
#pragma unroll
    for (int e = 0; e < 8; e += 4) {
      const int d = step * s + 8 * part + e;
      if constexpr (VEC) {
        const vf4 t = d < hd ? *reinterpret_cast<const vf4 *>(qrow + d) : vf4{};
#pragma unroll
        for (int c = 0; c < 4; ++c) x[e + c] = t[c] * scale;
      } else {
#pragma unroll
        for (int c = 0; c < 4; ++c) x[e + c] = d + c < hd ? qrow[d + c] * scale : 0.f;
      }
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      most = max(most, __float_as_uint(x[e]) & 0x7fffffffu);
      least = min(least, (__float_as_uint(x[e]) << 1) - 1u);
    }
    split_operand(x, 1.f, q[s]);
  }
  return __builtin_amdgcn_ballot_w64(most >= (100u + 127u) << 23 || least < (17u << 24) - 1u) != 0;  // 2^100, 2^-110
}

// The online softmax of one wave's 32 rows (one per lane % 32) over 32-key sub-blocks:
// S^T = K Q^T puts one row per lane, O^T += V^T P^T consumes the probabilities in place.
// Each sum has one accumulator, the corrections before the main product: a sum of 16
// products is rounded 12 times (fp16 10, bf16 6), where the fp32 MFMA rounds it 16 times.
template <typename T, int HD, int BN, bool VEC, bool UNI>
struct PagedRows {
  typedef PagedStage<T, HD, BN, VEC, UNI> Tile;
  typedef Pieces<T> PC;
  static constexpr int NP = PC::N;
  static constexpr int NDB = HD / 32;  // 32-wide head-dim blocks of O^T
  static constexpr int NS = HD / 16;   // MFMA k-steps of Q.K
  static constexpr int kAhead = NP == 1 ? (HD <= 64 ? 4 : 2) : NP == 3 && HD <= 64 ? 2 : 1;
  floatx16 oacc[NDB];
  float m_run, thr;  // the reference (log2), and the score from which it moves: any until it is set
  float l_sum;       // running sum over this half-wave's keys
  bool warm;         // every lane of the wave has its reference (wave-uniform)

  __device__ __forceinline__ void init() {
#pragma unroll
    for (int db = 0; db < NDB; ++db)
#pragma unroll
      for (int r = 0; r < 16; ++r) oacc[db][r] = 0.f;
    m_run = thr = -INFINITY;
    l_sum = 0.f;
    warm = false;
  }

  // -inf for the keys past this lane's last one (as an offset in its half's sub-block)
  __device__ __forceinline__ void apply_mask(floatx16 &sacc, int last_vis) const {
#pragma unroll
    for (int r = 0; r < 16; ++r) sacc[r] = acc_key(r) <= last_vis ? sacc[r] : -INFINITY;
  }

  // Operands are read AHEAD steps before their products, and kept there: left to itself, the
  // compiler reads each right before its use and waits (ragged chunks over bf16 857 us, 837 so;
  // 4 x 2048 of 4096 tokens, 16 heads of 64, fp32 620, 598).  As far ahead as the registers go.
  static __device__ __forceinline__ void hold() { __builtin_amdgcn_sched_barrier(0x6); }  // (vector and scalar units may pass)
  typedef bf16x8 Operand[NP];

  static __device__ __forceinline__ void read_v(Operand &v, const char *vt, int j) {
#pragma unroll
    for (int i = 0; i < NP; ++i)
      v[i] = *reinterpret_cast<const bf16x8 *>(vt + i * Tile::VPLANE + j / NDB * Tile::VSLAB + j % NDB * 256);
  }
  static __device__ __forceinline__ void read_k(Operand &k, const char *kt, int s) {
#pragma unroll
    for (int i = 0; i < NP; ++i) k[i] = *reinterpret_cast<const bf16x8 *>(kt + i * Tile::KPLANE + s * Tile::KSLAB);
  }

  __device__ __forceinline__ void accumulate_pv(const floatx16 &p, const char *vt) {
    constexpr int N = 2 * NDB, AHEAD = N < kAhead ? N : kAhead;
    Operand v[AHEAD];
    bf16x8 pp[3];
#pragma unroll
    for (int j = 0; j < AHEAD; ++j) read_v(v[j], vt, j);
    hold();
#pragma unroll
    for (int j = 0; j < N; ++j) {
      const int s = j / NDB, db = j % NDB;
      if (db == 0) {
        float x[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = p[8 * s + e];
        split_operand(x, 1.f, pp);
      }
#pragma unroll
      for (int i = 0; i < PC::PRODUCTS; ++i) oacc[db] = mfma32x32x16(v[j % AHEAD][PC::A[i]], pp[PC::B[i]], oacc[db]);
      hold();
      if (j + AHEAD < N) {
        read_v(v[j % AHEAD], vt, j + AHEAD);
        hold();
      }
    }
  }

  // Scores in log2 units, relative to the reference (absolute until there is one).
  __device__ __forceinline__ floatx16 scores(const char *kt, const bf16x8 (&q)[NS][3]) const {
    constexpr int AHEAD = NS < kAhead ? NS : kAhead;
    floatx16 sacc = {};
    Operand k[AHEAD];
#pragma unroll
    for (int s = 0; s < AHEAD; ++s) read_k(k[s], kt, s);
    hold();
#pragma unroll
    for (int s = 0; s < NS; ++s) {
#pragma unroll
      for (int i = 0; i < PC::PRODUCTS; ++i) sacc = mfma32x32x16(k[s % AHEAD][PC::A[i]], q[s][PC::B[i]], sacc);
      hold();
      if (s + AHEAD < NS) {
        read_k(k[s % AHEAD], kt, s + AHEAD);
        hold();
      }
    }
    const float ref = m_run == -INFINITY ? 0.f : m_run;
#pragma unroll
    for (int r = 0; r < 16; ++r) sacc[r] -= ref;
    return sacc;
  }

  // The common sub-block once every row has its reference: probabilities and their
  // per-lane sum first; false (nothing changed but sacc) if some lane's sum is above 2^32 or
  // NaN, and the caller takes softmax() on recomputed scores.
  __device__ __forceinline__ bool try_fast(floatx16 &sacc, const char *vt, bool masked, int last_vis) {
    if (masked) apply_mask(sacc, last_vis);
#pragma unroll
    for (int r = 0; r < 16; ++r) sacc[r] = fast_exp2(sacc[r]);
    float s8[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) s8[i] = sacc[2 * i] + sacc[2 * i + 1];
    const float ps = ((s8[0] + s8[1]) + (s8[2] + s8[3])) + ((s8[4] + s8[5]) + (s8[6] + s8[7]));
    if (__builtin_amdgcn_ballot_w64(!(ps <= kFastSumLimit))) return false;
    l_sum += ps;
    accumulate_pv(sacc, vt);
    return true;
  }

  __device__ __forceinline__ void softmax(floatx16 &sacc, bool masked, int last_vis) {
    if (masked) apply_mask(sacc, last_vis);
    const float m0 = max3_scores(sacc[0], sacc[1], sacc[2]);
    const float m1 = max3_scores(sacc[3], sacc[4], sacc[5]);
    const float m2 = max3_scores(sacc[6], sacc[7], sacc[8]);
    const float m3 = max3_scores(sacc[9], sacc[10], sacc[11]);
    const float m4 = max3_scores(sacc[12], sacc[13], sacc[14]);
    float smax = max3_scores(max3_scores(m0, m1, m2), max3_scores(m3, m4, sacc[15]), -INFINITY);
    smax = halves_max(smax);
    // Lazy rescale: the first visible key sets the reference, later only a rise of more
    // than the threshold moves it (the scores shift with it).
    const bool need = smax > thr;
    if (__builtin_amdgcn_ballot_w64(need)) {
      const bool first = m_run == -INFINITY;
      const float shift = need ? smax : 0.f;
      const float alpha = (need && !first) ? fast_exp2(-shift) : 1.0f;  // o and l are 0 before the first key
      m_run = need ? (first ? shift : m_run + shift) : m_run;
      thr = m_run == -INFINITY ? -INFINITY : kRescaleThreshold;
#pragma unroll
      for (int r = 0; r < 16; ++r) sacc[r] -= shift;
      if (__builtin_amdgcn_ballot_w64(need && !first)) {
        l_sum *= alpha;
#pragma unroll
        for (int db = 0; db < NDB; ++db)
#pragma unroll
          for (int r = 0; r < 16; ++r) oacc[db][r] *= alpha;
      }
    }
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      sacc[r] = fast_exp2(sacc[r]);
      l_sum += sacc[r];
    }
    warm = !__builtin_amdgcn_ballot_w64(m_run == -INFINITY);
  }

  // Undoes V's scale; whether some row came out non-finite (wave-uniform).
  __device__ __forceinline__ bool finish() {
    constexpr float unscale = NP == 3 ? kSplitUnscale : 1.f;
    float wrong = l_sum * 0.f;
#pragma unroll
    for (int db = 0; db < NDB; ++db) {
#pragma unroll
      for (int r = 0; r < 16; ++r) oacc[db][r] *= unscale;
      wrong = nonfinite_sum(oacc[db], wrong);
    }
    return any_nonfinite(wrong);
  }

  // The wave's rows over keys [c0, c1) on the fp32 MFMA straight from the pages: only for
  // rows that came out non-finite (common.h) or whose Q is out of the split's range (one NaN in
  // V of one head of 4 x 4096 tokens, fp32, 16 heads of 64: 798 -> 2980 us).
  // Where some row does not see all of a sub-block, V is summed per lane, without the keys
  // that the lane's row does not see: a product with their probability 0 would let their
  // infinities and NaNs through.
  __device__ __forceinline__ void recompute(const PagedArgs &a, const float *qrow, const int *table, int hk, int li,
                                            int hf, int c0, int c1, int lim, int lim_lo, int last) {
    init();
    const int kv_dim = a.kv_heads * a.hd;
    const T *kb = static_cast<const T *>(a.kc) + (size_t)hk * a.hd, *vb = static_cast<const T *>(a.vc) + (size_t)hk * a.hd;
#pragma unroll 1
    for (int kb0 = c0; kb0 < c1; kb0 += 32) {
      const int key = min(kb0 + li, last);
      const Slot ks = slot_in(a, table[key >> a.page_shift], key);
      const T *krow = kb + (size_t)ks.at * kv_dim;
      floatx16 sacc;
#pragma unroll
      for (int r = 0; r < 16; ++r) sacc[r] = m_run == -INFINITY ? 0.f : -m_run;
#pragma unroll 1
      for (int d = 0; d < HD; d += 2) {
        const bool in = d + hf < a.hd;
        sacc = mfma32x32x2(in && ks.ok ? (float)krow[d + hf] : 0.f, in ? qrow[d + hf] * a.scale_log2 : 0.f, sacc);
      }
      softmax(sacc, true, lim - kb0 - 4 * hf);
      const bool whole = kb0 + 31 <= lim_lo;  // (wave-uniform)
#pragma unroll 1
      for (int i = 0; i < (whole ? 16 : 32); ++i) {
        // whole: register i, whose key differs between the half-waves; else key i of the sub-block
        const int r = whole ? i : (i >> 3) * 4 + (i & 3);
        const int vk = kb0 + (whole ? acc_key(i) + 4 * hf : i), vkey = min(vk, last);
        const Slot vs = slot_in(a, table[vkey >> a.page_shift], vkey);
        const T *vrow = vb + (size_t)vs.at * kv_dim;
        float p = 0.f;
#pragma unroll
        for (int c = 0; c < 16; ++c) p = c == r ? sacc[c] : p;
        if (whole) {
#pragma unroll
          for (int db = 0; db < NDB; ++db)
            oacc[db] = mfma32x32x2(db * 32 + li < a.hd && vs.ok ? (float)vrow[db * 32 + li] : 0.f, p, oacc[db]);
        } else {
          p = __shfl(p, li + 32 * (i >> 2 & 1));
          if (vk <= lim) {
#pragma unroll
            for (int db = 0; db < NDB; ++db)
#pragma unroll
              for (int c = 0; c < 16; ++c) {
                const int d = db * 32 + acc_key(c) + 4 * hf;
                oacc[db][c] = fmaf(p, d < a.hd && vs.ok ? (float)vrow[d] : 0.f, oacc[db][c]);
              }
          }
        }
      }
    }
  }
};

// One workgroup: 128 rows of a (request, K/V head) against one chunk of its keys, each
// wave 32 rows.  Tiles of BN keys are double-buffered in LDS; the next tile's rows are in
// flight while the current one is consumed.  Workgroup ids: the K/V head runs fastest, so
// that tiles of one head meet on an XCD where the heads are a multiple of 8.  Then, of every
// 64 requests, the tiles that see the most keys come first, so that short ones fill the end:
// by classes, eighths of the most keys, within which a request's tiles follow each other and
// share its keys in L2.  One request after the other, 64 x 512 tokens (fp32, 8 heads of 32)
// 110 us, 81 so; 4 x 4096 tokens and ragged chunks the same within 1%, as with 16 classes.
//   Every value is held in bf16 pieces, which together have fp32's bits and its range: no
// scale, so no key, dim or probability is too small beside others.  Two fp16 pieces, three
// products for fp32 and two for 16-bit caches, would be 1.1 (bf16) to 1.8 times as fast, but
// they need a scale: a probability then loses what lies below 2^-35 of its row's largest, and
// a value what lies below 2^-40 of the largest beside it, while its part in the sum, the
// product of the two, may be as large as any.
//   What bounds it: 4 x 4096 tokens (fp32, 16 heads of 64) take 745 to 840 us by card, 1.0
// PFLOP/s of bf16 products where the library's largest plain ones reach 1.13; ragged chunks
// (bf16, 32 heads over 8 of 128) 765 to 840 us, as much.  The matrix cores are busy 51% of the
// cycles (46% at head dim 128) beside six (four) vector instructions for each of theirs; and
// cycles are long: the clock falls to 1.9 GHz (2.0) under their power.
constexpr int kTileClasses = 8;
// Waves a SIMD that registers are kept for; LDS holds as many.  16-bit caches, 16 heads of 64,
// 4 x 2048 of 4096 tokens: three 331 us (bf16) and 506 (fp16), two 348 and 530.
template <typename T>
constexpr int tile_waves(int hd) {
  if (hd <= 32 || (hd <= 64 && sizeof(T) == 2)) return 3;
  return hd <= 64 || sizeof(T) == 2 ? 2 : 1;
}
template <typename T, int HD, int BN, bool VEC, bool UNI>
__global__ void __launch_bounds__(PT_THREADS, tile_waves<T>(HD)) paged_tile_kernel(const PagedArgs a) {
  constexpr int NKB = BN / 32;  // 32-key sub-blocks per tile
  typedef PagedStage<T, HD, BN, VEC, UNI> Stage;
  __shared__ __attribute__((aligned(16))) char lds[2][Stage::BYTES];

  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int li = lane & 31, hf = lane >> 5;
  const int hk = blockIdx.x % a.kv_heads, flat = blockIdx.x / a.kv_heads, split = blockIdx.y;
  // the flat-th tile in that order
  int b = -1, tile = 0;
  for (int b0 = 0, before = 0; b0 < a.batch && b < 0; b0 += 64) {
    const PagedSeq s = paged_seq(a, min(b0 + lane, a.batch - 1));
    const int nr = b0 + lane < a.batch ? s.n * a.group : 0;
    const int tiles = nr > a.few_rows ? (nr + kPagedTileRows - 1) / kPagedTileRows : 0;
    int mine = tiles, later = 0, at = flat - before;
    int upto = (int)wave_scan(mine);
    const int all = __builtin_amdgcn_readlane(upto, 63);
    if (at >= all) {
      before += all;
      continue;
    }
    const uint64_t some = __builtin_amdgcn_ballot_w64(tiles != 0);
    if (some & (some - 1)) {
      // this lane's tiles of class c and above
      const int step = wave_reduce(tiles ? s.len : 0, [](int x, int y) { return max(x, y); }) / kTileClasses + 1;
      auto reach = [&](int c) {
        const long long row = ((long long)c * step - s.len + s.n) * a.group;  // the first that does
        return row <= 0 ? tiles : row < nr && tiles ? tiles - (int)row / kPagedTileRows : 0;
      };
      auto sum = [](int x) { return (int)__builtin_amdgcn_readlane(wave_scan(x), 63); };
      int c = 0;  // the last class for which that is more than `at`, of all lanes
#pragma unroll
      for (int bit = kTileClasses / 2; bit; bit >>= 1)
        if (sum(reach(c + bit)) > at) c += bit;
      later = reach(c + 1);
      mine = (c ? reach(c) : tiles) - later;  // (tiles that see no key are of the lowest)
      at -= sum(later);
      upto = (int)wave_scan(mine);
    }
    const int w = __builtin_ctzll(__builtin_amdgcn_ballot_w64(upto > at));
    b = b0 + w;
    tile = __builtin_amdgcn_readlane(tiles - 1 - later + upto - mine, w) - at;
  }
  if (b < 0) return;
  b = __builtin_amdgcn_readfirstlane(b);
  const PagedSeq s = paged_seq(a, b);
  const int nr = s.n * a.group, base = s.len - s.n;
  const int r0 = tile * kPagedTileRows, rw0 = r0 + wave * 32;
  const int kend = base + a.by_group.div(min(r0 + kPagedTileRows, nr) - 1) + 1;
  const bool single = s.len <= a.tile_chunk;
  const int c0 = split * a.tile_chunk, c1 = min(c0 + a.tile_chunk, kend);
  if (c0 >= c1 && !(single && split == 0)) return;

  const int rr = min(rw0 + li, nr - 1), tok = a.by_group.div(rr), head = hk * a.group + rr - tok * a.group;
  const int lim = base + tok;  // the last key this lane's row sees
  const int lim_lo = base + a.by_group.div(min(rw0, nr - 1)), lim_hi = base + a.by_group.div(min(rw0 + 31, nr - 1));
  const float *qrow = a.q + (size_t)(s.first + tok) * a.ldq + (size_t)head * a.hd;
  PagedRows<T, HD, BN, VEC, UNI> rows;
  rows.init();
  if (c0 < c1) {
    Stage st;
    st.init(a, b, hk, s.len - 1);
    st.lookup_first(a, c0);
    st.load(a, c0);
    st.lookup(a, c0 + BN);
    bf16x8 q[HD / 16][3];
    const bool wide = load_q_pieces<HD / 16, VEC>(q, qrow, a.hd, a.scale_log2, 16, hf);
    st.store(lds[0], a.bad);
    __syncthreads();
    const int ko = Stage::koperand(li, hf), vo = Stage::voperand(li, hf);
    int cur = 0;
    for (int k0 = c0; k0 < c1; k0 += BN, cur ^= 1) {
      // (past the last tile the request's last rows are loaded once more, and left there)
      st.load(a, k0 + BN);
      st.lookup(a, k0 + 2 * BN);
#pragma unroll
      for (int kb = 0; kb < NKB; ++kb) {
        const int kb0 = k0 + kb * 32;
        if (kb0 >= c1 || kb0 > lim_hi || rw0 >= nr) continue;
        const char *kop = lds[cur] + ko + kb * 512, *vop = lds[cur] + vo + 2 * kb * Stage::VSLAB;
        floatx16 sacc = rows.scores(kop, q);
        const bool masked = kb0 + 31 > lim_lo;
        const int last_vis = lim - kb0 - 4 * hf;
        bool done = false;
        if (rows.warm) {
          done = rows.try_fast(sacc, vop, masked, last_vis);
          if (!done) {
            // K is read from LDS again (the compiler may not keep the first scores)
            asm volatile("" ::: "memory");
            sacc = rows.scores(kop, q);
          }
        }
        if (!done) {
          rows.softmax(sacc, masked, last_vis);
          rows.accumulate_pv(sacc, vop);
        }
      }
      if (k0 + BN < c1) st.store(lds[cur ^ 1], a.bad);
      __syncthreads();
    }
    if ((rows.finish() || wide) && rw0 < nr)
      rows.recompute(a, qrow, a.table + (size_t)b * a.max_blocks, hk, li, hf, c0, min(c1, lim_hi + 1), lim, lim_lo,
                     s.len - 1);
  }
  if (rw0 + li >= nr) return;
  const float l = halves_sum(rows.l_sum);
  float *out, f = 1.f;
  if (single) {
    out = a.o + (size_t)(s.first + tok) * a.ldo + (size_t)head * a.hd;
    f = l == 0.f ? 0.f : 1.0f / l;
  } else {
    out = a.tile_part + (((size_t)(s.first + tok) * a.heads + head) * a.tile_splits + split) * (a.hd + 2);
    if (hf == 0) {
      out[a.hd] = fmaxf(rows.m_run, kNoKey);
      out[a.hd + 1] = l;
    }
  }
#pragma unroll
  for (int db = 0; db < HD / 32; ++db)
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const int d = db * 32 + 8 * g + 4 * hf;
      const vf4 x = {rows.oacc[db][4 * g] * f, rows.oacc[db][4 * g + 1] * f, rows.oacc[db][4 * g + 2] * f,
                     rows.oacc[db][4 * g + 3] * f};
      if (VEC && single) {
        if (d < a.hd) *reinterpret_cast<vf4 *>(out + d) = x;
      } else {
#pragma unroll
        for (int r = 0; r < 4; ++r)
          if (d + r < a.hd) out[d + r] = x[r];
      }
    }
}

// ---- few rows: matrix cores, a wave's own keys -----------------------------------

typedef float floatx4 __attribute__((ext_vector_type(4)));

// bf16 MFMA 16x16x32: D = A(16x32) * B(32x16) + C.  Lane l holds eight consecutive k,
// 8 * (l / 16) + 0..7, of row (A) or column (B) l % 16; D: column l % 16, rows
// 4 * (l / 16) + 0..3.
__device__ __forceinline__ floatx4 mfma16x16x32(bf16x8 a, bf16x8 b, floatx4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}

// The keys of a block of 32 as one wave stages it: whole rows in 16-byte loads, CPR of them
// a row.  K lies in LDS as it is, a row's chunks exchanged (chunk ^ turn(row)) so that the
// 16 rows whose same chunk an operand read takes together lie in different banks.  fp32's V
// lies as it is too, four floats between rows; V of a 16-bit type lies transposed, a dim's 32
// keys in the order that the P.V product reads them (key k at 8 (k / 4 % 4) + 4 (k / 16) +
// k % 4), as pairs put together on the way.
template <typename T, int HD, bool VEC>
struct SpanBlock {
  static constexpr int NP = Pieces<T>::N, PER = 16 / (int)sizeof(T);  // values of a 16-byte load
  static constexpr int CPR = HD / PER, NL = 32 * CPR / 64;            // loads a lane, of K and of V
  static constexpr int ROWS = CPR >= 16 ? 1 : 16 / CPR;               // rows in 256 bytes
  static constexpr int K_BYTES = 32 * HD * (int)sizeof(T);
  static constexpr int V_STRIDE = HD + 4;                  // fp32: floats
  static constexpr int V_ROW = 80;                         // 16-bit: bytes
  static constexpr int BYTES = K_BYTES + (NP == 3 ? 32 * V_STRIDE * 4 : HD * V_ROW);
  vu4 k[NL], v[NL];
  uint32_t slot;  // of this lane's key (lane % 32) in the loaded block; ~0: no page

  static __device__ __forceinline__ int turn(int row) { return row / ROWS & (CPR < 16 ? CPR - 1 : 15); }
  // K: load i of a lane is chunk k_chunk of row k_row
  static __device__ __forceinline__ int k_row(int i) { return ((threadIdx.x & 63) + 64 * i) / CPR; }
  static __device__ __forceinline__ int k_chunk(int i) { return ((threadIdx.x & 63) + 64 * i) % CPR; }
  // V: loads 2 u and 2 u + 1 are one chunk of two neighbouring rows (16-bit), or as K's (fp32)
  static __device__ __forceinline__ int v_row(int i) {
    if constexpr (NP == 3) return k_row(i);
    const int x = (threadIdx.x & 63) + 64 * (i / 2);
    return x / 8 / CPR * 16 + x % 8 * 2 + i % 2;
  }
  static __device__ __forceinline__ int v_chunk(int i) {
    if constexpr (NP == 3) return k_chunk(i);
    return ((threadIdx.x & 63) + 64 * (i / 2)) / 8 % CPR;
  }
  static __device__ __forceinline__ vu4 load16(const T *row, int chunk, int hd) {
    if constexpr (VEC) return chunk * PER < hd ? *reinterpret_cast<const vu4 *>(row + chunk * PER) : vu4{};
    vu4 w = {};
#pragma unroll
    for (int c = 0; c < PER; ++c)
      if (chunk * PER + c < hd) {
        if constexpr (NP == 3) w[c] = __builtin_bit_cast(uint32_t, (float)row[chunk * PER + c]);
        else w[c / 2] |= (uint32_t)__builtin_bit_cast(uint16_t, row[chunk * PER + c]) << 16 * (c & 1);
      }
    return w;
  }
  // Rows of a block, from the page and the number of this lane's key
  __device__ __forceinline__ void load(const PagedArgs &a, const T *kc, const T *vc, int kv_dim, int page, int key) {
    const Slot t = slot_in(a, page, key);
    slot = t.ok ? t.at : ~0u;
    const uint32_t at = t.at;  // (a page that is none reads page 0, and is zeroed below)
#pragma unroll
    for (int i = 0; i < NL; ++i) k[i] = load16(kc + (size_t)__shfl(at, k_row(i)) * kv_dim, k_chunk(i), a.hd);
#pragma unroll
    for (int i = 0; i < NL; ++i) v[i] = load16(vc + (size_t)__shfl(at, v_row(i)) * kv_dim, v_chunk(i), a.hd);
  }
  // Rows of no page, and V's past the request's last key, become zeros
  __device__ __forceinline__ void clean(int k0, int last, int *bad) {
    const uint64_t none = __builtin_amdgcn_ballot_w64(slot == ~0u);
    if (none == 0 && k0 + 31 <= last) return;
    if (none && bad) *bad = 1;
#pragma unroll
    for (int i = 0; i < NL; ++i) {
      if (none >> k_row(i) & 1) k[i] = vu4{};
      if ((none >> v_row(i) & 1) || k0 + v_row(i) > last) v[i] = vu4{};
    }
  }
  __device__ __forceinline__ void store(char *lds) const {
#pragma unroll
    for (int i = 0; i < NL; ++i)
      *reinterpret_cast<vu4 *>(lds + (k_row(i) * CPR + (k_chunk(i) ^ turn(k_row(i)))) * 16) = k[i];
    lds += K_BYTES;
    if constexpr (NP == 3) {
#pragma unroll
      for (int i = 0; i < NL; ++i) *reinterpret_cast<vu4 *>(lds + v_row(i) * V_STRIDE * 4 + v_chunk(i) * 16) = v[i];
    } else {
#pragma unroll
      for (int u = 0; u < NL / 2; ++u) {
        const int row = v_row(2 * u);
        char *d = lds + v_chunk(2 * u) * PER * V_ROW + (8 * (row / 4 % 4) + 4 * (row / 16) + row % 4) * 2;
#pragma unroll
        for (int c = 0; c < PER; ++c)
          *reinterpret_cast<uint32_t *>(d + c * V_ROW) =
              __builtin_amdgcn_perm(v[2 * u + 1][c / 2], v[2 * u][c / 2], c & 1 ? 0x07060302u : 0x05040100u);
      }
    }
  }
  // The pieces of dims 32 s + 8 q + 0..7 of a key
  static __device__ __forceinline__ void k_operand(const char *lds, int s, int key, int q, bf16x8 (&p)[3]) {
    auto chunk = [&](int c) { return *reinterpret_cast<const vu4 *>(lds + (key * CPR + (c ^ turn(key))) * 16); };
    if constexpr (NP == 1) {
      p[0] = __builtin_bit_cast(bf16x8, chunk(4 * s + q));
    } else {
      float x[8];
      if constexpr (NP == 3) {
        const vu4 a = chunk(8 * s + 2 * q), b = chunk(8 * s + 2 * q + 1);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          x[e] = __uint_as_float(a[e]);
          x[4 + e] = __uint_as_float(b[e]);
        }
      } else {
        const vu4 a = chunk(4 * s + q);
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = half_value(a[e / 2], e & 1, T{});
      }
      split_operand(x, 1.f, p);
    }
  }
  // The pieces of a dim for the keys of quarter q: 4 q + 0..3 and 16 + 4 q + 0..3
  static __device__ __forceinline__ void v_operand(const char *lds, int dim, int q, bf16x8 (&p)[3]) {
    lds += K_BYTES;
    if constexpr (NP == 3) {
      float x[8];
#pragma unroll
      for (int e = 0; e < 8; ++e)
        x[e] = reinterpret_cast<const float *>(lds)[(16 * (e / 4) + 4 * q + e % 4) * V_STRIDE + dim];
      split_operand(x, kSplitScale, p);
    } else {
      const vu4 w = *reinterpret_cast<const vu4 *>(lds + dim * V_ROW + q * 16);
      if constexpr (NP == 1) {
        p[0] = __builtin_bit_cast(bf16x8, w);
      } else {
        float x[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = half_value(w[e / 2], e & 1, T{});
        split_operand(x, 1.f, p);
      }
    }
  }
};

// f over the four lanes of a row (l, l ^ 16, l ^ 32, l ^ 48), in each of them.
template <typename F>
__device__ __forceinline__ float quarters(float x, F f) {
  auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  x = f(__uint_as_float(r[0]), __uint_as_float(r[1]));
  r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return f(__uint_as_float(r[0]), __uint_as_float(r[1]));
}

// The online softmax of up to 16 rows, one per lane % 16, over blocks of 32 keys: S^T = K Q^T
// gives quarter q = lane / 16 of the wave the keys 4 q + 0..3 and 16 + 4 q + 0..3, the order
// in which O^T += V^T P^T takes them.  Every sum has one accumulator, the corrections added
// before the main product.
template <typename T, int HD, bool VEC>
struct SpanRows {
  typedef SpanBlock<T, HD, VEC> Block;
  typedef Pieces<T> PC;
  static constexpr int NS = HD / 32, NDB = HD / 16;
  floatx4 o[NDB];  // dims 16 db + 4 q + 0..3
  float m, l;      // the reference (log2 units) and this quarter's sum

  __device__ __forceinline__ void init() {
#pragma unroll
    for (int db = 0; db < NDB; ++db) o[db] = floatx4{};
    m = -INFINITY;
    l = 0.f;
  }
  // Probabilities of the keys up to last_vis (counted from the quarter's first) in place of
  // the scores; o and l follow a reference that rises.
  __device__ __forceinline__ void softmax(float (&p)[8], int last_vis) {
    float top = -INFINITY;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      p[e] = 16 * (e / 4) + e % 4 <= last_vis ? p[e] : -INFINITY;
      top = fmaxf(top, p[e]);
    }
    top = quarters(top, [](float a, float b) { return fmaxf(a, b); });
    if (__builtin_amdgcn_ballot_w64(top > m)) {
      const float to = fmaxf(m, top), w = m == -INFINITY ? 0.f : fast_exp2(m - to);
      m = to;
      l *= w;
#pragma unroll
      for (int db = 0; db < NDB; ++db) o[db] *= w;
    }
    const float ref = m == -INFINITY ? 0.f : m;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      p[e] = fast_exp2(p[e] - ref);
      l += p[e];
    }
  }
  __device__ __forceinline__ void add(const char *lds, const bf16x8 (&q)[NS][3], int row, int quarter, int last_vis) {
    float p[8];
#pragma unroll
    for (int h = 0; h < 2; ++h) {  // keys 16 h .. 16 h + 15
      floatx4 s = {};
#pragma unroll
      for (int i = 0; i < NS; ++i) {
        bf16x8 k[3];
        Block::k_operand(lds, i, 16 * h + row, quarter, k);
#pragma unroll
        for (int c = 0; c < PC::PRODUCTS; ++c) s = mfma16x16x32(k[PC::A[c]], q[i][PC::B[c]], s);
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) p[4 * h + e] = s[e];
    }
    softmax(p, last_vis);
    bf16x8 pp[3];
    split_operand(p, 1.f, pp);
#pragma unroll
    for (int db = 0; db < NDB; ++db) {
      bf16x8 v[3];
      Block::v_operand(lds, 16 * db + row, quarter, v);
#pragma unroll
      for (int c = 0; c < PC::PRODUCTS; ++c) o[db] = mfma16x16x32(v[PC::A[c]], pp[PC::B[c]], o[db]);
    }
  }
  // Undoes V's scale; whether some row came out non-finite (wave-uniform)
  __device__ __forceinline__ bool finish() {
    constexpr float unscale = PC::N == 3 ? kSplitUnscale : 1.f;
    float wrong = l * 0.f;
#pragma unroll
    for (int db = 0; db < NDB; ++db) {
      o[db] *= unscale;
#pragma unroll
      for (int e = 0; e < 4; ++e) wrong = fmaf(o[db][e], 0.f, wrong);
    }
    return any_nonfinite(wrong);
  }
  // The rows over the wave's blocks in fp32 straight from the pages, without the keys that
  // a row does not see: for rows that came out non-finite or whose Q is out of the split's
  // range.
  __device__ __forceinline__ void recompute(const PagedArgs &a, const float *qrow, const int *table, const T *kc,
                                            const T *vc, int quarter, int first, int c1, int lim, int last) {
    init();
    const int kv_dim = a.kv_heads * a.hd;
    auto row_of = [&](const T *cache, int key) -> const T * {
      const Slot s = slot_in(a, table[key >> a.page_shift], key);
      return s.ok ? cache + (size_t)s.at * kv_dim : nullptr;
    };
#pragma unroll 1
    for (int k0 = first; k0 < c1; k0 += 128) {
      float p[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const T *k = row_of(kc, min(k0 + 16 * (e / 4) + 4 * quarter + e % 4, last));
        p[e] = 0.f;
#pragma unroll 1
        for (int d = 0; d < a.hd; ++d) p[e] = fmaf(k ? (float)k[d] : 0.f, qrow[d] * a.scale_log2, p[e]);
      }
      softmax(p, lim - k0 - 4 * quarter);
#pragma unroll
      for (int e = 0; e < 8; ++e)
#pragma unroll 1
        for (int q = 0; q < 4; ++q) {
          const float w = __shfl(p[e], (threadIdx.x & 15) + 16 * q);
          const int key = k0 + 16 * (e / 4) + 4 * q + e % 4;
          if (key > lim) continue;
          const T *v = row_of(vc, key);
#pragma unroll
          for (int db = 0; db < NDB; ++db)
#pragma unroll
            for (int c = 0; c < 4; ++c) {
              const int d = 16 * db + 4 * quarter + c;
              if (v && d < a.hd) o[db][c] = fmaf(w, (float)v[d], o[db][c]);
            }
        }
    }
  }
};

// One workgroup: the up to 16 rows of a (request, K/V head) against one chunk of its keys.
// Reading the cache bounds this, and rows fill one small MFMA operand at most, so the four
// waves split the keys: each walks blocks of 32 through LDS of its own, with no barrier until
// the waves' sums are joined.  The next block is loaded into registers while one is
// multiplied; two workgroups a CU keep 128 KB on the way at head dim 128.  64 x 8192 keys of
// bf16, 64 heads over 8 of 128: 373 us, 5.8 TB/s.
template <typename T, int HD, bool VEC>
__global__ void __launch_bounds__(PT_THREADS, sizeof(T) == 2 || HD <= 64 ? 2 : 1) paged_span_kernel(const PagedArgs a) {
  typedef SpanRows<T, HD, VEC> Rows;
  typedef SpanBlock<T, HD, VEC> Block;
  constexpr int NS = HD / 32, NDB = HD / 16, ROW = HD + 4;  // floats between rows of the join
  constexpr int WAVE_O = 16 * ROW * 4, WAVE = Block::BYTES > WAVE_O ? Block::BYTES : WAVE_O;
  __shared__ __attribute__((aligned(16))) char lds[4][WAVE];
  __shared__ float red_m[4][16], red_l[4][16];

  const int b = blockIdx.z, hk = blockIdx.y, split = blockIdx.x;
  const PagedSeq s = paged_seq(a, b);
  const int nr = s.n * a.group;
  if (nr == 0 || nr > a.few_rows) return;
  const int base = s.len - s.n;
  const bool single = s.len <= a.few_chunk;
  const int c0 = split * a.few_chunk, c1 = min(c0 + a.few_chunk, s.len);  // the last row sees all keys
  if (c0 >= c1 && !(single && split == 0)) return;

  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int row = lane & 15, quarter = lane >> 4;
  const int rr = min(row, nr - 1), tok = a.by_group.div(rr), head = hk * a.group + rr - tok * a.group;
  const int lim = base + tok, last = s.len - 1;
  const float *qrow = a.q + (size_t)(s.first + tok) * a.ldq + (size_t)head * a.hd;
  const int *table = a.table + (size_t)b * a.max_blocks;
  const int kv_dim = a.kv_heads * a.hd;
  const T *kc = static_cast<const T *>(a.kc) + (size_t)hk * a.hd, *vc = static_cast<const T *>(a.vc) + (size_t)hk * a.hd;

  Rows rows;
  rows.init();
  const int first = c0 + wave * 32;
  if (first < c1) {
    char *mine = lds[wave];
    // this lane's key (lane % 32 of the block) and its page, a block ahead of its rows
    auto key_at = [&](int k0) { return min(k0 + (lane & 31), last); };
    auto page_at = [&](int k0) { return table[key_at(k0) >> a.page_shift]; };
    Block blk;
    blk.load(a, kc, vc, kv_dim, page_at(first), key_at(first));
    int page = page_at(first + 128);
    bf16x8 q[NS][3];
    const bool wide = load_q_pieces<NS, VEC>(q, qrow, a.hd, a.scale_log2, 32, quarter);
#pragma unroll 1
    for (int k0 = first; k0 < c1; k0 += 128) {
      blk.clean(k0, last, a.bad);
      blk.store(mine);
      blk.load(a, kc, vc, kv_dim, page, key_at(k0 + 128));
      page = page_at(k0 + 256);
      // the LDS writes above are this wave's own: in order, but not for the compiler
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      rows.add(mine, q, row, quarter, lim - k0 - 4 * quarter);
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    }
    if (rows.finish() || wide) rows.recompute(a, qrow, table, kc, vc, quarter, first, c1, lim, last);
  }
  // the waves' sums: rows' statistics, then each wave's O scaled to the common maximum
  const float m = fmaxf(rows.m, kNoKey), l = quarters(rows.l, [](float x, float y) { return x + y; });
  if (quarter == 0) {
    red_m[wave][row] = m;
    red_l[wave][row] = l;
  }
  __syncthreads();
  const float w = fast_exp2(m - fmaxf(fmaxf(red_m[0][row], red_m[1][row]), fmaxf(red_m[2][row], red_m[3][row])));
  float *part_o = reinterpret_cast<float *>(lds[wave]) + row * ROW;
#pragma unroll
  for (int db = 0; db < NDB; ++db) *reinterpret_cast<floatx4 *>(part_o + db * 16 + 4 * quarter) = rows.o[db] * w;
  __syncthreads();
  for (int t = threadIdx.x; t < nr * HD; t += PT_THREADS) {
    const int r = t / HD, d = t % HD;
    if (d >= a.hd) continue;
    float x = 0.f, L = 0.f;
    const float M = fmaxf(fmaxf(red_m[0][r], red_m[1][r]), fmaxf(red_m[2][r], red_m[3][r]));
#pragma unroll
    for (int v = 0; v < 4; ++v) {
      x += reinterpret_cast<const float *>(lds[v])[r * ROW + d];
      L += red_l[v][r] * fast_exp2(red_m[v][r] - M);
    }
    if (single) {
      const int i = a.by_group.div(r), h = hk * a.group + r - i * a.group;
      a.o[(size_t)(s.first + i) * a.ldo + (size_t)h * a.hd + d] = L == 0.f ? 0.f : x / L;
    } else {
      float *part = a.few_part + ((((size_t)b * a.kv_heads + hk) * a.few_rows + r) * a.few_splits + split) * (a.hd + 2);
      part[d] = x;
      if (d == 0) {
        part[a.hd] = M;
        part[a.hd + 1] = L;
      }
    }
  }
}

template <typename T, int HD, int MODE>
void launch_rows(const PagedArgs &a, hipStream_t st) {
  const int most = a.few_rows;
  auto grid = [&](int r) { return dim3(a.few_splits, a.kv_heads * ((most + r - 1) / r), a.batch); };
  if (most <= 1) paged_rows_kernel<T, HD, 1, MODE><<<grid(1), PR_THREADS, 0, st>>>(a);
  else if (most <= 2) paged_rows_kernel<T, HD, 2, MODE><<<grid(2), PR_THREADS, 0, st>>>(a);
  else paged_rows_kernel<T, HD, 4, MODE><<<grid(4), PR_THREADS, 0, st>>>(a);
}

template <typename T, int HD>
void launch_rows(const PagedArgs &a, bool wide, hipStream_t st) {
  if (!wide) launch_rows<T, HD, kScalar>(a, st);
  else if (a.hd == HD) launch_rows<T, HD, kVector>(a, st);
  else launch_rows<T, HD, kVectorCut>(a, st);
}

template <typename T, int HD, int BN>
void launch_tile(const PagedArgs &a, bool wide, hipStream_t st) {
  const long long tiles = (long long)a.rows * a.group / kPagedTileRows + a.batch;
  const dim3 grid((unsigned)(tiles * a.kv_heads), a.tile_splits);
  // offsets inside 16 rows of a page fit 32 bits
  const bool uni = a.page_shift >= 4 && (long long)a.kv_heads * a.hd < (1 << 24);
  if (wide && uni) paged_tile_kernel<T, HD, BN, true, true><<<grid, PT_THREADS, 0, st>>>(a);
  else if (wide) paged_tile_kernel<T, HD, BN, true, false><<<grid, PT_THREADS, 0, st>>>(a);
  else paged_tile_kernel<T, HD, BN, false, false><<<grid, PT_THREADS, 0, st>>>(a);
}

template <typename T, int HD>
void launch_span(const PagedArgs &a, bool wide, hipStream_t st) {
  const dim3 grid(a.few_splits, a.kv_heads, a.batch);
  if (wide) paged_span_kernel<T, HD, true><<<grid, PT_THREADS, 0, st>>>(a);
  else paged_span_kernel<T, HD, false><<<grid, PT_THREADS, 0, st>>>(a);
}

// wide: head dims that are multiples of 8, and 16-byte aligned rows.
template <typename T>
int paged_attn(const PagedArgs &a, const PagedKernels &k, bool wide, hipStream_t st) {
  if (k.rows) {
    if (a.hd <= 32) launch_rows<T, 32>(a, wide, st);
    else if (a.hd <= 64) launch_rows<T, 64>(a, wide, st);
    else if (a.hd <= 128) launch_rows<T, 128>(a, wide, st);
    else launch_rows<T, 256>(a, wide, st);
    const int rc = check_launch("paged_rows_kernel");
    if (rc) return rc;
  }
  if (k.span) {
    if (a.hd <= 32) launch_span<T, 32>(a, wide, st);
    else if (a.hd <= 64) launch_span<T, 64>(a, wide, st);
    else launch_span<T, 128>(a, wide, st);
    const int rc = check_launch("paged_span_kernel");
    if (rc) return rc;
  }
  if (k.tile) {
    if (a.hd <= 32) launch_tile<T, 32, 32>(a, wide, st);
    else if (a.hd <= 64) launch_tile<T, 64, 32>(a, wide, st);
    else launch_tile<T, 128, 32>(a, wide, st);
    return check_launch("paged_tile_kernel");
  }
  return CDML_OK;
}

}  // namespace
}  // namespace cdml
