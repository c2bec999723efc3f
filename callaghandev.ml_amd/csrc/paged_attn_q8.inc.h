// Attention of few rows a K/V head over an 8-bit paged cache, for one of its types T (I8 or
// F8; included by a file each), and the choice between it and the tiles of paged_attn.inc.h.
#pragma once

#include "paged_attn.inc.h"

namespace cdml {
namespace {

// How a head's rows go through the lanes of a wave (row = lane % 16, quarter = lane / 16), 32
// keys at a time, straight from the cache into the operands of the 16x16x32 MFMA:
//   K: lane (row, quarter) has dims KD * quarter .. + KD - 1 of keys row and 16 + row.  A dot
//      product's order is free, so product s takes the lane's s-th eight dims, of Q too.
//   V: lane (row, quarter) has dims VD * row .. + VD - 1 of the keys 4 quarter + 0..3 and
//      16 + 4 quarter + 0..3, those whose probabilities it holds; product d takes its d-th
//      dim, so V is transposed as the codes of two keys become a pair of bf16.
// No byte passes LDS, and a load's address is a base plus an offset that the lane keeps.
template <typename T, int HD>
struct CodeBlock {
  static constexpr int KD = HD / 4, VD = HD / 16;              // dims a lane, of K and of V
  static constexpr int KW = KD / 4, VW = VD >= 4 ? VD / 4 : 1;  // words of a row
  uint32_t k[2][KW], v[8][VW];
  vf4 ks[2], vs[2];

  static constexpr int KL = KW >= 4 ? KW / 4 : 1;  // loads of K's row, 16 bytes each where it has as many

  template <int N>
  static __device__ __forceinline__ void words(uint32_t *w, const T *p) {
    if constexpr (N == 1) {
      w[0] = __builtin_nontemporal_load(reinterpret_cast<const uint32_t *>(p));
    } else {
      typedef uint32_t V __attribute__((ext_vector_type(N)));
      const V t = __builtin_nontemporal_load(reinterpret_cast<const V *>(p));
#pragma unroll
      for (int c = 0; c < N; ++c) w[c] = t[c];
    }
  }
  static __device__ __forceinline__ void k_words(uint32_t (&w)[KW], const T *p, const uint32_t (&off)[KL]) {
#pragma unroll
    for (int i = 0; i < KL; ++i) words<KW / KL>(w + KW / KL * i, p + off[i]);
  }
  static __device__ __forceinline__ void v_words(uint32_t (&w)[VW], const T *p) {
    if constexpr (VD >= 4) words<VW>(w, p);
    else w[0] = *reinterpret_cast<const uint16_t *>(p);
  }

  // The operand of product s over keys 16 h + row
  __device__ __forceinline__ bf16x8 k_operand(int h, int s) const {
    vu4 w;
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = code_pair(k[h][2 * s + i / 2], i & 1, T{});
    return __builtin_bit_cast(bf16x8, w);
  }
  // The operand of dim d of the lane's VD
  __device__ __forceinline__ bf16x8 v_operand(int d) const {
    vu4 w;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t a = v[2 * i][d / 4], b = v[2 * i + 1][d / 4];
      if constexpr (std::is_same<T, I8>::value) {
        const float x = code_value(I8{(uint8_t)(a >> 8 * (d % 4))}), y = code_value(I8{(uint8_t)(b >> 8 * (d % 4))});
        w[i] = __builtin_amdgcn_perm(__float_as_uint(y), __float_as_uint(x), 0x07060302u);
      } else {
        w[i] = __builtin_amdgcn_perm(code_pair(b, d / 2 % 2, T{}), code_pair(a, d / 2 % 2, T{}),
                                     d & 1 ? 0x07060302u : 0x05040100u);
      }
    }
    return __builtin_bit_cast(bf16x8, w);
  }
};

// Four scales in a row (aligned to their size alone).
__device__ __forceinline__ vf4 four_scales(const float *p) {
  struct __attribute__((packed, aligned(4))) Four {
    vf4 x;
  };
  return reinterpret_cast<const Four *>(p)->x;
}

// Where a wave's rows of 32 keys lie.  RUN keys, beginning at a multiple of RUN, lie in one page.
//   RUN 16: a half's page is the same for all lanes.  Lane l holds where half l % 2 of the
//      wave's block l / 2 lies, of 32 blocks; a block's two are read from there.
//   RUN 4, 1: every lane looks its rows' pages up, a block ahead.
template <typename T, int HD, int RUN>
struct CodeLoader {
  typedef CodeBlock<T, HD> Block;
  static constexpr int NV = RUN == 1 ? 8 : 2;  // pages that a lane's keys of V lie in
  static constexpr int STRIDE = 128;           // keys from one of a wave's blocks to its next
  const int *table;
  const T *kc, *vc;        // the head's
  const float *ks, *vs;
  uint32_t k_off[Block::KL], v_off;  // of the lane's dims, in bytes; RUN 16: and of its row in a half
  int row, quarter, width, last, first;
  int page[RUN == 16 ? 1 : 2 + NV];
  uint32_t at_lo, at_hi;   // RUN 16: rows before the lane's half
  uint64_t none;           // RUN 16: halves whose page is none; else lane's rows, as bits

  __device__ __forceinline__ void init(const PagedArgs &a, int trow, int hk, int first_key, int last_key) {
    const int lane = threadIdx.x & 63;
    row = lane & 15;
    quarter = lane >> 4;
    width = a.width;
    last = last_key;
    first = first_key;
    table = a.table + (size_t)trow * a.max_blocks;
    kc = head_of<T>(a, a.kc, hk);
    vc = head_of<T>(a, a.vc, hk);
    ks = a.ks + ((size_t)hk << a.page_shift);
    vs = a.vs + ((size_t)hk << a.page_shift);
    // Dims past a row's end read its beginning instead: Q is 0 there, and what they give O is
    // not stored.  (Rows are multiples of 16 bytes, so a load lies in a row or past it.)
#pragma unroll
    for (int i = 0; i < Block::KL; ++i) {
      const int d = Block::KD * quarter + 16 * i;
      k_off[i] = (RUN == 16 ? row * width : 0) + (d < width ? d : 0);
    }
    v_off = (RUN == 16 ? 4 * quarter * width : 0) + (Block::VD * row < width ? Block::VD * row : 0);
  }
  __device__ __forceinline__ int page_of(const PagedArgs &a, int key) const { return table[min(key, last) >> a.page_shift]; }
  // RUN 16: the key at which lane's half of the blocks from k0 on begins
  static __device__ __forceinline__ int half_key(int k0) {
    const int lane = threadIdx.x & 63;
    return k0 + STRIDE * (lane >> 1) + 16 * (lane & 1);
  }
  // Keys of the lane: of K, half h; of V, place e
  __device__ __forceinline__ int k_key(int k0, int h) const { return k0 + 16 * h + row; }
  __device__ __forceinline__ int v_key(int k0, int e) const { return k0 + 16 * (e / 4) + 4 * quarter + e % 4; }
  // The pages that load() of the block at k0 needs
  __device__ __forceinline__ void lookup(const PagedArgs &a, int k0) {
    if constexpr (RUN == 16) {
      page[0] = page_of(a, half_key(k0));
    } else {
#pragma unroll
      for (int h = 0; h < 2; ++h) page[h] = page_of(a, k_key(k0, h));
#pragma unroll
      for (int i = 0; i < NV; ++i) page[2 + i] = page_of(a, v_key(k0, 8 / NV * i));
    }
  }
  __device__ __forceinline__ void start_group(const PagedArgs &a, int k0) {
    // (a half past the last key reads the page of that, its rows from the same place)
    const Slot s = slot_in(a, page[0], half_key(k0));
    const size_t at = row_at<T>(a, s.at);
    at_lo = (uint32_t)at;
    at_hi = (uint32_t)(at >> 32);
    none = __builtin_amdgcn_ballot_w64(!s.ok);
    first = k0;
    lookup(a, k0 + 32 * STRIDE);
  }
  __device__ __forceinline__ void lookup_first(const PagedArgs &a) {
    lookup(a, first);
    if constexpr (RUN == 16) start_group(a, first);
  }

  // Loads the block at k0 and looks the next one's pages up.  Rows of no page come as zeros.
  __device__ __forceinline__ void load(const PagedArgs &a, Block &b, int k0) {
    if constexpr (RUN == 16) {
      if (k0 - first >= 32 * STRIDE) start_group(a, k0);
      const int i = (k0 - first) / STRIDE * 2;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const size_t at = (size_t)(uint32_t)__builtin_amdgcn_readlane(at_hi, i + h) << 32 |
                          (uint32_t)__builtin_amdgcn_readlane(at_lo, i + h);
        const T *kp = kc + at * width, *vp = vc + at * width;
        Block::k_words(b.k[h], kp, k_off);
#pragma unroll
        for (int e = 0; e < 4; ++e) Block::v_words(b.v[4 * h + e], vp + e * width + v_off);
        b.ks[h] = four_scales(ks + at + 4 * quarter);
        b.vs[h] = four_scales(vs + at + 4 * quarter);
      }
    } else {
      none = 0;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const Slot s = slot_in(a, page[h], k_key(k0, h));
        none |= (uint64_t)!s.ok << h;
        Block::k_words(b.k[h], kc + row_at<T>(a, s.at) * width, k_off);
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const Slot s = slot_in(a, page[2 + e * NV / 8], v_key(k0, e));
        none |= (uint64_t)!s.ok << (2 + e);
        const size_t at = row_at<T>(a, s.at);
        Block::v_words(b.v[e], vc + at * width + v_off);
        if constexpr (RUN == 1) {
          b.ks[e / 4][e % 4] = ks[at];
          b.vs[e / 4][e % 4] = vs[at];
        } else if (e % 4 == 0) {
          b.ks[e / 4] = four_scales(ks + at);
          b.vs[e / 4] = four_scales(vs + at);
        }
      }
      lookup(a, k0 + STRIDE);
    }
  }
  // Rows of no page, and V's past the request's last key, become zeros (the block at k0, the
  // last that was loaded).
  __device__ __forceinline__ void clean(Block &b, int k0, int *bad) const {
    if constexpr (RUN == 16) {
      const uint32_t wrong = (uint32_t)(none >> (k0 - first) / STRIDE * 2) & 3u;
      if (wrong == 0 && k0 + 31 <= last) return;
      if (wrong && bad) *bad = 1;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        if (wrong >> h & 1) {
          zero(b.k[h]);
          b.ks[h] = vf4{};
        }
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if ((wrong >> h & 1) || v_key(k0, 4 * h + e) > last) {
            zero(b.v[4 * h + e]);
            b.vs[h][e] = 0.f;
          }
      }
    } else {
      if (__builtin_amdgcn_ballot_w64(none != 0) == 0 && k0 + 31 <= last) return;
      if (none && bad) *bad = 1;
#pragma unroll
      for (int h = 0; h < 2; ++h)
        if (none >> h & 1) zero(b.k[h]);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const bool wrong = none >> (2 + e) & 1;
        if (wrong) b.ks[e / 4][e % 4] = 0.f;
        if (wrong || v_key(k0, e) > last) {
          zero(b.v[e]);
          b.vs[e / 4][e % 4] = 0.f;
        }
      }
    }
  }
  template <int W>
  static __device__ __forceinline__ void zero(uint32_t (&w)[W]) {
#pragma unroll
    for (int i = 0; i < W; ++i) w[i] = 0;
  }
};

// The online softmax of up to 16 rows, one per lane % 16, over blocks of 32 keys, as in SpanRows.
template <typename T, int HD>
struct CodeRows {
  typedef CodeBlock<T, HD> Block;
  static constexpr int NS = HD / 32, NDB = HD / 16;
  floatx4 o[NDB];  // register c of o[d]: dim VD * (4 quarter + c) + d
  float m, l;      // the reference (log2 units) and this quarter's sum

  __device__ __forceinline__ void init() {
#pragma unroll
    for (int d = 0; d < NDB; ++d) o[d] = floatx4{};
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
      for (int d = 0; d < NDB; ++d) o[d] *= w;
    }
    const float ref = m == -INFINITY ? 0.f : m;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      p[e] = fast_exp2(p[e] - ref);
      l += p[e];
    }
  }
  __device__ __forceinline__ void add(const Block &b, const bf16x8 (&q)[NS][3], int last_vis) {
    float p[8];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      floatx4 s = {};
#pragma unroll
      for (int i = 0; i < NS; ++i) {
        const bf16x8 k = b.k_operand(h, i);
#pragma unroll
        for (int c = 2; c >= 0; --c) s = mfma16x16x32(k, q[i][c], s);
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) p[4 * h + e] = s[e] * b.ks[h][e];
    }
    softmax(p, last_vis);
#pragma unroll
    for (int e = 0; e < 8; ++e) p[e] *= b.vs[e / 4][e % 4];
    bf16x8 pp[3];
    split_operand(p, kCodeScale, pp);
#pragma unroll
    for (int d = 0; d < NDB; ++d) {
      const bf16x8 v = b.v_operand(d);
#pragma unroll
      for (int c = 2; c >= 0; --c) o[d] = mfma16x16x32(v, pp[c], o[d]);
    }
  }
  // Undoes the scale of V's scales; whether some row came out non-finite (wave-uniform)
  __device__ __forceinline__ bool finish() {
    float wrong = l * 0.f;
#pragma unroll
    for (int d = 0; d < NDB; ++d) {
      o[d] *= kCodeUnscale;
#pragma unroll
      for (int c = 0; c < 4; ++c) wrong = fmaf(o[d][c], 0.f, wrong);
    }
    return any_nonfinite(wrong);
  }
  // The rows over the wave's blocks in fp32, value by value and without the keys that a row
  // does not see: for rows that came out non-finite or whose Q is out of the pieces' range.
  __device__ __forceinline__ void recompute(const PagedArgs &a, const float *qrow, const int *table, int hk, int quarter,
                                            int first, int c1, int lim, int last) {
    init();
    const T *kc = head_of<T>(a, a.kc, hk), *vc = head_of<T>(a, a.vc, hk);
    const size_t head = (size_t)hk << a.page_shift;
    auto row_of = [&](int key, size_t &at) {
      const Slot s = slot_in(a, table[key >> a.page_shift], key);
      at = row_at<T>(a, s.at);
      return s.ok;
    };
#pragma unroll 1
    for (int k0 = first; k0 < c1; k0 += 128) {
      float p[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        size_t at;
        const bool ok = row_of(min(k0 + 16 * (e / 4) + 4 * quarter + e % 4, last), at);
        p[e] = 0.f;
        if (!ok) continue;
        const float s = a.ks[head + at];
#pragma unroll 1
        for (int d = 0; d < a.hd; ++d) p[e] = fmaf(cached(kc[at * a.width + d], s), qrow[d] * a.scale_log2, p[e]);
      }
      softmax(p, lim - k0 - 4 * quarter);
#pragma unroll
      for (int e = 0; e < 8; ++e)
#pragma unroll 1
        for (int q = 0; q < 4; ++q) {
          const float w = __shfl(p[e], (threadIdx.x & 15) + 16 * q);
          const int key = k0 + 16 * (e / 4) + 4 * q + e % 4;
          if (key > lim) continue;
          size_t at;
          if (!row_of(key, at)) continue;
          const float s = a.vs[head + at];
#pragma unroll
          for (int i = 0; i < NDB; ++i)
#pragma unroll
            for (int c = 0; c < 4; ++c) {
              const int d = NDB * (4 * quarter + c) + i;
              if (d < a.hd) o[i][c] = fmaf(w, cached(vc[at * a.width + d], s), o[i][c]);
            }
        }
    }
  }
};

// One workgroup: up to 16 rows of a (request, K/V head) against one chunk of its keys.  The
// four waves take blocks of 32 keys in turn and join their sums at the end; a wave's next
// block is on the way while one is multiplied.
template <typename T, int HD, int RUN, bool VEC, bool SHARED>
__device__ __forceinline__ void code_rows(const PagedArgs &a, const PagedSeq &s, int b, int r0, int nr,
                                          float (&lds)[4][16 * (HD + 4)], float (&red_m)[4][16], float (&red_l)[4][16]) {
  typedef CodeRows<T, HD> Rows;
  typedef CodeBlock<T, HD> Block;
  constexpr int NS = HD / 32, NDB = HD / 16, ROW = HD + 4;  // floats between rows of the join
  const int hk = blockIdx.y % a.kv_heads, split = blockIdx.x, base = s.len - s.n;
  const int kend = s.causal ? base + a.by_group.div(min(r0 + 16, nr) - 1) + 1 : s.len;  // past the last visible key
  const bool single = !SHARED && s.len <= a.few_chunk;
  const int c0 = split_from<SHARED>(s, split, a.few_chunk);
  const int c1 = split_to<SHARED>(c0, split, a.few_splits, a.few_chunk, kend);
  if (c0 >= c1 && !(single && split == 0)) return;

  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int row = lane & 15, quarter = lane >> 4;
  const int rr = min(r0 + row, nr - 1), tok = a.by_group.div(rr), head = hk * a.group + rr - tok * a.group;
  const int last = s.len - 1, lim = s.causal ? base + tok : last;
  const float *qrow = a.q + (size_t)(s.first + tok) * a.ldq + (size_t)head * a.hd;

  Rows rows;
  rows.init();
  const int first = c0 + wave * 32;
  if (first < c1) {
    CodeLoader<T, HD, RUN> from;
    from.init(a, s.table, hk, first, last);
    from.lookup_first(a);
    Block x, y;
    from.load(a, x, first);
    bf16x8 q[NS][3];
    const bool wide = load_q_pieces<NS, VEC>(q, qrow, a.hd, a.scale_log2, 8, HD / 4 * quarter);
    // (past the wave's last block the request's last rows are loaded once more, and left there)
#pragma unroll 1
    for (int k0 = first; k0 < c1; k0 += 256) {
      from.clean(x, k0, a.bad);
      from.load(a, y, k0 + 128);
      rows.add(x, q, lim - k0 - 4 * quarter);
      if (k0 + 128 >= c1) break;
      from.clean(y, k0 + 128, a.bad);
      from.load(a, x, k0 + 256);
      rows.add(y, q, lim - k0 - 128 - 4 * quarter);
    }
    if (rows.finish() || wide)
      rows.recompute(a, qrow, a.table + (size_t)s.table * a.max_blocks, hk, quarter, first, c1, lim, last);
  }
  // the waves' sums: rows' statistics, then each wave's O scaled to the common maximum
  const float m = fmaxf(rows.m, kNoKey), l = quarters(rows.l, [](float x, float y) { return x + y; });
  if (quarter == 0) {
    red_m[wave][row] = m;
    red_l[wave][row] = l;
  }
  __syncthreads();
  const float w = fast_exp2(m - fmaxf(fmaxf(red_m[0][row], red_m[1][row]), fmaxf(red_m[2][row], red_m[3][row])));
#pragma unroll
  for (int c = 0; c < 4; ++c)
#pragma unroll
    for (int d = 0; d < NDB; ++d) lds[wave][row * ROW + NDB * (4 * quarter + c) + d] = rows.o[d][c] * w;
  __syncthreads();
  for (int t = threadIdx.x; t < min(nr - r0, 16) * HD; t += PT_THREADS) {
    const int r = t / HD, d = t % HD;
    if (d >= a.hd) continue;
    float x = 0.f, L = 0.f;
    const float M = fmaxf(fmaxf(red_m[0][r], red_m[1][r]), fmaxf(red_m[2][r], red_m[3][r]));
#pragma unroll
    for (int v = 0; v < 4; ++v) {
      x += lds[v][r * ROW + d];
      L += red_l[v][r] * fast_exp2(red_m[v][r] - M);
    }
    const int i = a.by_group.div(r0 + r), h = hk * a.group + r0 + r - i * a.group;
    if (single) {
      a.o[(size_t)(s.first + i) * a.ldo + (size_t)h * a.hd + d] = L == 0.f ? 0.f : x / L;
    } else {
      float *part;
      if constexpr (SHARED)
        part = a.part + (((size_t)(s.first + i) * a.heads + h) * a.part_splits + a.first_split + split) * (a.hd + 2);
      else
        part = a.few_part + ((((size_t)b * a.kv_heads + hk) * a.few_rows + r0 + r) * a.few_splits + split) * (a.hd + 2);
      part[d] = x;
      if (d == 0) {
        part[a.hd] = M;
        part[a.hd + 1] = L;
      }
    }
  }
}

template <typename T, int HD, int RUN, bool VEC, bool SHARED>
__global__ void __launch_bounds__(PT_THREADS, HD <= 128 ? 2 : 1) paged_code_kernel(const PagedArgs a) {
  __shared__ __attribute__((aligned(16))) float lds[4][16 * (HD + 4)];
  __shared__ float red_m[4][16], red_l[4][16];
  const int b = blockIdx.z;
  const PagedSeq s = paged_seq<SHARED>(a, b);
  const int nr = s.n * a.group;
  int r0 = blockIdx.y / a.kv_heads * 16;
  if (nr > a.few_rows || r0 >= nr) return;
  if constexpr (SHARED) {
    // (a group of more rows than the launch was told of takes its time)
    for (; r0 < nr; r0 += gridDim.y / a.kv_heads * 16) {
      code_rows<T, HD, RUN, VEC, true>(a, s, b, r0, nr, lds, red_m, red_l);
      __syncthreads();
    }
  } else {
    code_rows<T, HD, RUN, VEC, false>(a, s, b, r0, nr, lds, red_m, red_l);
  }
}

template <typename T, int HD, bool VEC, bool SHARED>
void launch_code(const PagedArgs &a, hipStream_t st) {
  const int row_groups = SHARED && a.prefix ? 1 : (a.few_rows + 15) / 16;
  const dim3 grid(a.few_splits, a.kv_heads * row_groups, SHARED && a.prefix ? a.groups : a.batch);
  if (a.page_shift >= 4) paged_code_kernel<T, HD, 16, VEC, SHARED><<<grid, PT_THREADS, 0, st>>>(a);
  else if (a.page_shift >= 2) paged_code_kernel<T, HD, 4, VEC, SHARED><<<grid, PT_THREADS, 0, st>>>(a);
  else paged_code_kernel<T, HD, 1, VEC, SHARED><<<grid, PT_THREADS, 0, st>>>(a);
}

template <typename T, int HD, bool SHARED>
void launch_code(const PagedArgs &a, bool wide, hipStream_t st) {
  if (wide) launch_code<T, HD, true, SHARED>(a, st);
  else launch_code<T, HD, false, SHARED>(a, st);
}

// wide: head dims that are multiples of 8, and 16-byte aligned rows of Q and O.
template <typename T, bool SHARED>
int paged_attn_q8(const PagedArgs &a, const PagedKernels &k, bool wide, hipStream_t st) {
  if (k.span) {
    if (a.hd <= 32) launch_code<T, 32, SHARED>(a, wide, st);
    else if (a.hd <= 64) launch_code<T, 64, SHARED>(a, wide, st);
    else if (SHARED || a.hd <= 128) launch_code<T, 128, SHARED>(a, wide, st);
    else if constexpr (!SHARED) launch_code<T, 256, SHARED>(a, wide, st);
    const int rc = check_launch("paged_code_kernel");
    if (rc) return rc;
  }
  return k.tile ? launch_tiles<T, SHARED>(a, wide, st) : CDML_OK;
}

}  // namespace
}  // namespace cdml
