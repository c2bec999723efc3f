// Attention of few rows a K/V head over a paged cache of one piece (I8, F8 and, for up to four
// rows, __bf16; included by a file each), and the choice between it and the tiles of
// paged_attn.inc.h.
#pragma once

#include "paged_attn.inc.h"

namespace cdml {
namespace {

// How a head's rows go through the lanes of a wave (row = lane % 16, quarter = lane / 16), 32
// keys at a time, straight from the cache into the operands of the 16x16x32 MFMA:
//   K: lane (row, quarter) has 16 bytes of every 64 of keys row and 16 + row, the quarters side by
//      side.  A dot product's order is free, so product s takes the lane's s-th eight dims, of
//      Q too.  (A quarter of a row to a lane, whose loads touch four times the segments: 64
//      requests behind 8192 bf16 tokens 74.4 us, 68.1 so.)
//   V: lane (row, quarter) has dims VD * row .. + VD - 1 of the keys 4 quarter + 0..3 and
//      16 + 4 quarter + 0..3, those whose probabilities it holds; product d takes its d-th
//      dim, so V is transposed as the codes of two keys become a pair of bf16.
// No code passes LDS, and a load's address is a base plus an offset that the lane keeps.
template <typename T, int HD>
struct CodeBlock {
  static constexpr int KD = HD / 4, VD = HD / 16;  // dims a lane, of K and of V
  static constexpr int B = sizeof(T), KW = KD * B / 4, VW = VD * B >= 4 ? VD * B / 4 : 1;  // words of a row
  uint32_t k[2][KW], v[8][VW];
  float scale;  // of key lane % 32: K's in the lower lanes, V's in the upper

  static constexpr int KL = KW >= 4 ? KW / 4 : 1;  // loads of K's row, 16 bytes each where it has as many
  // The dims of load i, and of product s, of a quarter
  static __device__ __forceinline__ constexpr int k_dim(int i, int quarter) { return KD / KL * (4 * i + quarter); }
  static __device__ __forceinline__ constexpr int q_dim(int s, int quarter) {
    constexpr int PER = KD / KL / 8;  // products of a load
    return k_dim(s / PER, quarter) + s % PER * 8;
  }

  // off stays a 32-bit register beside the base, for a load's own addition (the compiler would
  // widen it ahead of the loop, and add in vector instructions)
  template <int N>
  static __device__ __forceinline__ void words(uint32_t *w, const T *p, uint32_t off) {
    asm volatile("" : "+v"(off));
    p += off;
    if constexpr (N == 1) {
      w[0] = __builtin_nontemporal_load(reinterpret_cast<const uint32_t *>(p));
    } else {
      typedef uint32_t V __attribute__((ext_vector_type(N)));
      const V t = __builtin_nontemporal_load(reinterpret_cast<const V *>(p));
#pragma unroll
      for (int c = 0; c < N; ++c) w[c] = t[c];
    }
  }
  static __device__ __forceinline__ void k_words(uint32_t (&w)[KW], const T *p, const uint32_t (&off)[KL], uint32_t used) {
#pragma unroll
    for (int i = 0; i < KL; ++i) words<KW / KL>(w + KW / KL * i, p, off[i] & used);
  }
  static __device__ __forceinline__ void v_words(uint32_t (&w)[VW], const T *p, uint32_t off) {
    if constexpr (VD * B >= 4) words<VW>(w, p, off);
    else w[0] = *reinterpret_cast<const uint16_t *>(p + off);
  }

  // The operand of product s over keys 16 h + row
  __device__ __forceinline__ bf16x8 k_operand(int h, int s) const {
    vu4 w;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (kQ8<T>) w[i] = code_pair(k[h][2 * s + i / 2], i & 1, T{});
      else w[i] = k[h][4 * s + i];
    }
    return __builtin_bit_cast(bf16x8, w);
  }
  // The operand of dim d of the lane's VD
  __device__ __forceinline__ bf16x8 v_operand(int d) const {
    vu4 w;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t a = v[2 * i][d * B / 4], b = v[2 * i + 1][d * B / 4];
      if constexpr (!kQ8<T>) {
        w[i] = __builtin_amdgcn_perm(b, a, d & 1 ? 0x07060302u : 0x05040100u);
      } else if constexpr (std::is_same<T, I8>::value) {
        w[i] = byte_pair(a, b, d % 4);
      } else {
        w[i] = __builtin_amdgcn_perm(code_pair(b, d / 2 % 2, T{}), code_pair(a, d / 2 % 2, T{}),
                                     d & 1 ? 0x07060302u : 0x05040100u);
      }
    }
    return __builtin_bit_cast(bf16x8, w);
  }
};

// Where a wave's blocks of 32 keys, STRIDE keys apart, lie.  RUN keys, beginning at a multiple of
// RUN, lie in one page:
//   RUN 16, 8: a block's pages are looked up by scalar loads, a block ahead of its rows.
//   RUN 1: every lane looks its rows' pages up (pages of fewer tokens than 8).
template <typename T, int HD, int RUN, int STRIDE>
struct CodeLoader {
  typedef CodeBlock<T, HD> Block;
  typedef const __attribute__((address_space(4))) int *Table;  // nothing writes it in the meantime
  static constexpr int NP = RUN == 1 ? 1 : 32 / RUN, PER = 16 / RUN;  // pages of a block, and of half of one
  Table table;
  const T *kc, *vc;          // the head's
  const float *side;         // 8 bits: the scales of this lane, K's or V's
  uint32_t k_off[Block::KL], v_off[RUN == 1 ? 1 : 4];  // of the lane's dims, in elements; RUN > 1: and of its rows in a run
  int row, quarter, width, last;
  int page[NP];              // of the next block to be loaded
  int lane_page[RUN == 1 ? 11 : 1];  // RUN 1: of K's rows, V's, and the scale's

  __device__ __forceinline__ void init(const PagedArgs &a, int trow, int hk, int last_key) {
    const int lane = threadIdx.x & 63;
    row = lane & 15;
    quarter = lane >> 4;
    width = row_step<T>(a);
    const int dims = kQ8<T> ? a.width : a.hd;
    last = last_key;
    table = (Table)(uint64_t)(a.table + (size_t)trow * a.max_blocks);
    kc = head_of<T>(a, a.kc, hk);
    vc = head_of<T>(a, a.vc, hk);
    if constexpr (kQ8<T>) side = (lane < 32 ? a.ks : a.vs) + ((size_t)hk << a.page_shift) + (RUN == 1 ? 0 : lane % RUN);
    // Dims past a row's end read its beginning instead: Q is 0 there, and what they give O is
    // not stored.  (A head's rows are multiples of 16 bytes, so a load lies in one or past it.)
#pragma unroll
    for (int i = 0; i < Block::KL; ++i) {
      const int d = Block::k_dim(i, quarter);
      k_off[i] = (RUN == 1 ? 0 : row % RUN * width) + (d < dims ? d : 0);
    }
#pragma unroll
    for (int e = 0; e < (RUN == 1 ? 1 : 4); ++e)
      v_off[e] = (RUN == 1 ? 0 : (4 * quarter % RUN + e) * width) + (Block::VD * row < dims ? Block::VD * row : 0);
  }
  // Keys of the lane: of K, half h; of V, place e; of the scale
  __device__ __forceinline__ int k_key(int k0, int h) const { return k0 + 16 * h + row; }
  __device__ __forceinline__ int v_key(int k0, int e) const { return k0 + 16 * (e / 4) + 4 * quarter + e % 4; }
  __device__ __forceinline__ int scale_key(int k0) const { return k0 + (int)(threadIdx.x & 31); }
  __device__ __forceinline__ int page_of(const PagedArgs &a, int key) const { return table[min(key, last) >> a.page_shift]; }
  // The pages that load() of the block at k0 needs
  __device__ __forceinline__ void lookup(const PagedArgs &a, int k0) {
    if constexpr (RUN > 1) {
#pragma unroll
      for (int i = 0; i < NP; ++i) page[i] = page_of(a, k0 + RUN * i);
    } else {
#pragma unroll
      for (int h = 0; h < 2; ++h) lane_page[h] = page_of(a, k_key(k0, h));
#pragma unroll
      for (int e = 0; e < 8; ++e) lane_page[2 + e] = page_of(a, v_key(k0, e));
      lane_page[10] = page_of(a, scale_key(k0));
    }
  }

  // Elements before a row or run
  __device__ __forceinline__ size_t element(size_t at) const { return kQ8<T> ? at * width : at; }

  // Loads the block at k0 and looks the next one's pages up.  What comes from no page: bits of
  // runs, or of the lane's rows (0, 1: K's, 2 ..: V's, 10: the scale's).
  // A block from key `end` on is not used: its lanes read the same few bytes.
  __device__ __forceinline__ uint32_t load(const PagedArgs &a, Block &b, int k0, int end) {
    uint32_t none = 0;
    const uint32_t used = k0 < end ? ~0u : 0u;
    if constexpr (RUN > 1) {
      size_t at[NP];  // rows before the run
#pragma unroll
      for (int i = 0; i < NP; ++i) {
        // (a run past the last key lies in that one's page, its rows at the same places)
        const Slot s = slot_in(a, page[i], k0 + RUN * i);
        none |= (uint32_t)!s.ok << i;
        at[i] = row_at<T>(a, s.at);
      }
      lookup(a, k0 + STRIDE);
      if constexpr (kQ8<T>) {
        const int lane = threadIdx.x & 31;
        size_t mine = lane & 16 ? at[PER] : at[0];
        if constexpr (PER == 2) mine = lane & 8 ? lane & 16 ? at[3] : at[1] : mine;
        b.scale = side[mine];
      }
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const size_t run = PER == 1 ? at[h] : row & 8 ? at[PER * h + PER - 1] : at[PER * h];
        Block::k_words(b.k[h], kc + element(run), k_off, used);
      }
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const size_t run = PER == 1 ? at[h] : quarter & 2 ? at[PER * h + PER - 1] : at[PER * h];
#pragma unroll
        for (int e = 0; e < 4; ++e) Block::v_words(b.v[4 * h + e], vc + element(run), v_off[e] & used);
      }
    } else {
      auto place = [&](int i, int key) {
        const Slot s = slot_in(a, lane_page[i], key);
        none |= (uint32_t)!s.ok << i;
        return row_at<T>(a, s.at);
      };
      if constexpr (kQ8<T>) b.scale = side[place(10, scale_key(k0))];
#pragma unroll
      for (int h = 0; h < 2; ++h) Block::k_words(b.k[h], kc + element(place(h, k_key(k0, h))), k_off, used);
#pragma unroll
      for (int e = 0; e < 8; ++e) Block::v_words(b.v[e], vc + element(place(2 + e, v_key(k0, e))), v_off[0] & used);
      lookup(a, k0 + STRIDE);
    }
    return none;
  }
  // The scale of no page, and V's past the request's last key, become 0; so do the values where
  // they may be NaN (not I8).  none: what load() of the block returned.
  __device__ __forceinline__ void clean(Block &b, int k0, uint32_t none, int &bad) const {
    const bool past = k0 + 31 > last;
    if (RUN > 1 ? none == 0 : __builtin_amdgcn_ballot_w64(none != 0) == 0) {
      if (!past) return;
    } else if (none) {
      bad = 1;
    }
    const int i = RUN == 1 ? 10 : (int)(threadIdx.x & 31) / RUN;
    if (!kQ8<T> || (none >> i & 1) || ((threadIdx.x & 32) && scale_key(k0) > last)) b.scale = 0.f;
    if constexpr (!std::is_same<T, I8>::value) {
#pragma unroll
      for (int h = 0; h < 2; ++h)
        if (none >> (RUN == 1 ? h : PER * h + (PER == 2 ? row >> 3 : 0)) & 1) zero(b.k[h]);
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if ((none >> (RUN == 1 ? 2 + e : PER * (e / 4) + (PER == 2 ? quarter >> 1 : 0)) & 1) || v_key(k0, e) > last)
          zero(b.v[e]);
    }
  }
  template <int W>
  static __device__ __forceinline__ void zero(uint32_t (&w)[W]) {
#pragma unroll
    for (int i = 0; i < W; ++i) w[i] = 0;
  }
};

// x of the lane N places before (cyclically, of 16).
template <int N>
__device__ __forceinline__ float turned(float x) {
  return dpp<0x120 + N>(x);
}

// The online softmax of up to 16 rows, one per lane % 16, over blocks of 32 keys, as in SpanRows.
//   PACK: of up to four rows, one per lane % 4.  The operand's other columns hold the pieces: Q's
// and the probabilities' first, second and third in columns 0..3, 4..7 and 8..11, zeros in the
// last.  One product does for three, the parts of a score are added across the columns, those of
// O once at the end; and the pieces of Q take a third of the registers.
template <typename T, int HD, bool PACK>
struct CodeRows {
  typedef CodeBlock<T, HD> Block;
  static constexpr int NS = HD / 32, NDB = HD / 16, NP = PACK ? 1 : 3;
  static constexpr int ROWS = PACK ? 4 : 16;
  bf16x8 q[NS][NP];
  floatx4 o[NDB];  // register c of o[d]: dim VD * (4 quarter + c) + d
  float m, l;      // the reference (log2 units) and this quarter's sum
  bool warm;       // every lane has its reference (wave-uniform)
  uint32_t cut[2];  // PACK: what the lane's piece leaves out of a value, and of the rest

  __device__ __forceinline__ void init() {
#pragma unroll
    for (int d = 0; d < NDB; ++d) o[d] = floatx4{};
    m = -INFINITY;
    l = 0.f;
    warm = false;
    const int piece = threadIdx.x >> 2 & 3;
    cut[0] = piece == 0 ? 0u : piece == 3 ? ~0u : 0xffff0000u;
    cut[1] = piece < 2 ? 0u : piece == 3 ? ~0u : 0xffff0000u;
  }
  // Four values of a row from dim d on, zeros past the head dim
  template <bool VEC>
  static __device__ __forceinline__ vf4 q_values(const float *qrow, int d, int hd) {
    vf4 x;
    if constexpr (VEC) {
      x = *reinterpret_cast<const vf4 *>(qrow + min(d, hd - 4));
      if (d >= hd) x = vf4{};
    } else {
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        const float t = qrow[min(d + c, hd - 1)];
        x[c] = d + c < hd ? t : 0.f;
      }
    }
    return x;
  }
  // Q's pieces; whether Q is out of their range (wave-uniform, as in load_q_pieces).  PACK: a
  // value's top sixteen bits are its piece, what is left of it the next one's value.
  template <bool VEC>
  __device__ __forceinline__ bool load_q(const float *qrow, int hd, float scale, int quarter) {
    vf4 x[NS][2];
#pragma unroll
    for (int i = 0; i < NS; ++i)
#pragma unroll
      for (int h = 0; h < 2; ++h) x[i][h] = q_values<VEC>(qrow, Block::q_dim(i, quarter) + 4 * h, hd);
    uint32_t most = 0, least = ~0u;  // of 2 |x|, and of 2 |x| - 1 as integers, which leaves zeros out
#pragma unroll
    for (int i = 0; i < NS; ++i) {
      float y[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        y[e] = x[i][e / 4][e % 4] * scale;
        const uint32_t twice = __float_as_uint(y[e]) << 1;
        most = max(most, twice);
        least = min(least, twice - 1u);
      }
      if constexpr (PACK) {
        q[i][0] = piece_of(y);
      } else {
        bf16x8 all[3];
        split_operand(y, 1.f, all);
#pragma unroll
        for (int j = 0; j < 3; ++j) q[i][j] = all[2 - j];  // the corrections first
      }
    }
    return __builtin_amdgcn_ballot_w64(most >= (100u + 127u) << 24 || least < (17u << 24) - 1u) != 0;
  }
  // PACK: this lane's piece of eight values
  __device__ __forceinline__ bf16x8 piece_of(float (&x)[8]) const {
    vu4 w;
#pragma unroll
    for (int e = 0; e < 8; ++e)
#pragma unroll
      for (int c = 0; c < 2; ++c) x[e] -= __uint_as_float(__float_as_uint(x[e]) & cut[c]);
#pragma unroll
    for (int i = 0; i < 4; ++i)
      w[i] = __builtin_amdgcn_perm(__float_as_uint(x[2 * i + 1]), __float_as_uint(x[2 * i]), 0x07060302u);
    return __builtin_bit_cast(bf16x8, w);
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
    warm = !__builtin_amdgcn_ballot_w64(m == -INFINITY);
  }
  // The same without a look at the maximum, once every row has a reference: false, and nothing
  // changed, where a lane's probabilities sum up to more than 2^32, or to NaN.
  __device__ __forceinline__ bool try_fast(const float (&s)[8], const vf4 (&ks)[2], float (&p)[8]) {
    float sum[4];
#pragma unroll
    for (int e = 0; e < 8; ++e) p[e] = fast_exp2(fmaf(s[e], ks[e / 4][e % 4], -m));
#pragma unroll
    for (int e = 0; e < 4; ++e) sum[e] = p[e] + p[e + 4];
    const float all = (sum[0] + sum[1]) + (sum[2] + sum[3]);
    if (__builtin_amdgcn_ballot_w64(!(all <= kFastSumLimit))) return false;
    l += all;
    return true;
  }
  // scales: 64 floats of LDS for this wave.  masked: some row does not see all of the block
  // (wave-uniform).
  __device__ __forceinline__ void add(const Block &b, float *scales, int quarter, bool masked, int last_vis) {
    vf4 ks[2], vs[2];
    if constexpr (kQ8<T>) {
      scales[threadIdx.x & 63] = b.scale * (threadIdx.x & 32 ? kCodeScale : 1.f);
      // (LDS writes and reads of one wave are in order, but not for the compiler)
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        ks[h] = *reinterpret_cast<const vf4 *>(scales + 16 * h + 4 * quarter);
        vs[h] = *reinterpret_cast<const vf4 *>(scales + 32 + 16 * h + 4 * quarter);
      }
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    } else {
      ks[0] = ks[1] = vf4{1.f, 1.f, 1.f, 1.f};
    }
    float raw[8], p[8];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      floatx4 s = {};
#pragma unroll
      for (int i = 0; i < NS; ++i) {
        const bf16x8 k = b.k_operand(h, i);
#pragma unroll
        for (int c = 0; c < NP; ++c) s = mfma16x16x32(k, q[i][c], s);
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        if constexpr (PACK) {
          s[e] += turned<8>(s[e]);
          s[e] += turned<4>(s[e]);
        }
        raw[4 * h + e] = s[e];
      }
    }
    if (!warm || masked || !try_fast(raw, ks, p)) {
#pragma unroll
      for (int e = 0; e < 8; ++e) p[e] = raw[e] * ks[e / 4][e % 4];
      softmax(p, last_vis);
    }
    if constexpr (kQ8<T>) {
#pragma unroll
      for (int e = 0; e < 8; ++e) p[e] *= vs[e / 4][e % 4];
    }
    bf16x8 pp[3];
    if constexpr (PACK) {
      pp[0] = piece_of(p);
    } else {
      split_codes(p, pp);
    }
#pragma unroll
    for (int d = 0; d < NDB; ++d) {
      const bf16x8 v = b.v_operand(d);
#pragma unroll
      for (int c = NP - 1; c >= 0; --c) o[d] = mfma16x16x32(v, pp[c], o[d]);
    }
  }
  // Undoes the scale of V's scales; whether some row came out non-finite (wave-uniform)
  __device__ __forceinline__ bool finish() {
    float wrong = l * 0.f;
#pragma unroll
    for (int d = 0; d < NDB; ++d) {
      if constexpr (kQ8<T>) o[d] *= kCodeUnscale;
#pragma unroll
      for (int c = 0; c < 4; ++c) wrong = fmaf(o[d][c], 0.f, wrong);
    }
    return any_nonfinite(wrong);
  }
  // PACK: the pieces' sums of O (recompute's are whole in every lane)
  __device__ __forceinline__ void join_pieces(bool recomputed) {
    if (PACK && !recomputed) {
#pragma unroll
      for (int d = 0; d < NDB; ++d)
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          o[d][c] += turned<8>(o[d][c]);
          o[d][c] += turned<4>(o[d][c]);
        }
    }
  }
  // The rows over the wave's blocks in fp32, value by value and without the keys that a row
  // does not see: for rows that came out non-finite or whose Q is out of the pieces' range.
  __device__ __forceinline__ void recompute(const PagedArgs &a, const float *qrow, const int *table, int hk, int quarter,
                                            int first, int stride, int c1, int lim, int last) {
    init();
    const T *kc = head_of<T>(a, a.kc, hk), *vc = head_of<T>(a, a.vc, hk);
    auto row_of = [&](int key, size_t &at, const float *scales, float &scale) {
      const Slot s = slot_in(a, table[key >> a.page_shift], key);
      at = row_at<T>(a, s.at);
      if constexpr (kQ8<T>) {
        scale = scales[((size_t)hk << a.page_shift) + at];
        at *= a.width;
      }
      return s.ok;
    };
#pragma unroll 1
    for (int k0 = first; k0 < c1; k0 += stride) {
      float p[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        size_t at;
        float s = 1.f;
        const bool ok = row_of(min(k0 + 16 * (e / 4) + 4 * quarter + e % 4, last), at, a.ks, s);
        p[e] = 0.f;
        if (!ok) continue;
#pragma unroll 1
        for (int d = 0; d < a.hd; ++d) p[e] = fmaf(cached(kc[at + d], s), qrow[d] * a.scale_log2, p[e]);
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
          float s = 1.f;
          if (!row_of(key, at, a.vs, s)) continue;
#pragma unroll
          for (int i = 0; i < NDB; ++i)
#pragma unroll
            for (int c = 0; c < 4; ++c) {
              const int d = NDB * (4 * quarter + c) + i;
              if (d < a.hd) o[i][c] = fmaf(w, cached(vc[at + d], s), o[i][c]);
            }
        }
    }
  }
};

// One workgroup: up to 16 rows of a (request, K/V head) against one chunk of its keys.  The
// four waves take blocks of 32 keys in turn and join their sums at the end; a wave's next block
// is on the way while one is multiplied.  (Two on the way: 64 ragged requests, 32 heads over 8,
// f8, 131 us for 129; 8 x 2048 keys 15.7 for 14.6.)
//   What bounds it: HBM where requests are equal and long, 64 x 8192 keys, 16 heads of 128, i8: 329
// us, 6.7 TB/s of codes and scales.  Ragged requests (2048 to 8192 keys, 32 heads over 8, f8)
// take 126 us, 4.9 TB/s: workgroups end at different times (in chunks of 4096 keys 154).
constexpr int kCodeBlocks = 2;
template <typename T, int HD, int RUN, bool PACK, bool SHARED, int WAVES>
__device__ __forceinline__ void code_rows(const PagedArgs &a, const PagedSeq &s, int b, int hk, int r0, int nr,
                                          float (&lds)[4][CodeRows<T, HD, PACK>::ROWS * (HD + 4)], float (&red_m)[4][16], float (&red_l)[4][16],
                                          float (&scales)[4][64]) {
  typedef CodeRows<T, HD, PACK> Rows;
  typedef CodeBlock<T, HD> Block;
  constexpr int NDB = HD / 16, ROW = HD + 4, ROWS = Rows::ROWS;  // floats between rows of the join
  constexpr int STRIDE = 32 * WAVES;
  const int split = blockIdx.x, base = s.len - s.n;
  const int kend = s.causal ? base + a.by_group.div(min(r0 + ROWS, nr) - 1) + 1 : s.len;  // past the last visible key
  const bool single = SHARED ? a.fused && !a.prefix : s.len <= a.few_chunk;
  const int c0 = split_from<SHARED>(s, split, a.few_chunk);
  const int c1 = split_to<SHARED>(c0, split, a.few_splits, a.few_chunk, kend);
  if (c0 >= c1 && !(single && split == 0)) return;

  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int row = lane & (ROWS - 1), quarter = lane >> 4;
  const int rr = min(r0 + row, nr - 1), tok = a.by_group.div(rr), head = hk * a.group + rr - tok * a.group;
  const int last = s.len - 1, lim = s.causal ? base + tok : last;
  const int lim_lo = s.causal ? base + a.by_group.div(r0) : last;
  const float *qrow = a.q + (size_t)(s.first + tok) * a.ldq + (size_t)head * a.hd;

  Rows rows;
  rows.init();
  const int first = c0 + wave % WAVES * 32;
  if (first < c1) {
    CodeLoader<T, HD, RUN, STRIDE> from;
    from.init(a, s.table, hk, last);
    from.lookup(a, first);
    constexpr int U = kCodeBlocks;
    Block block[U];
    uint32_t none[U];
    int bad = 0;
#pragma unroll
    for (int u = 0; u < U - 1; ++u) none[u] = from.load(a, block[u], first + STRIDE * u, c1);
    const bool wide = a.wide ? rows.template load_q<true>(qrow, a.hd, a.scale_log2, quarter)
                             : rows.template load_q<false>(qrow, a.hd, a.scale_log2, quarter);
    // (left from its middle: a way back to its top with loads unused would make every turn wait for them)
#pragma unroll 1
    for (int k0 = first;; k0 += STRIDE * U) {
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int k = k0 + STRIDE * u, ahead = (u + U - 1) % U;
        if (k >= c1) goto summed;
        none[ahead] = from.load(a, block[ahead], k + STRIDE * (U - 1), c1);
        from.clean(block[u], k, none[u], bad);
        rows.add(block[u], scales[wave], quarter, k + 31 > lim_lo, lim - k - 4 * quarter);
      }
    }
  summed:
    const PagedArgs &z = args_again();
    if (bad && z.bad) *z.bad = 1;
    const bool again = rows.finish() || wide;
    if (again) {
      const float *row = z.q + (size_t)(s.first + tok) * z.ldq + (size_t)head * z.hd;
      rows.recompute(z, row, z.table + (size_t)s.table * z.max_blocks, hk, quarter, first, STRIDE, c1, lim, last);
    }
    rows.join_pieces(again);
  }
  // the waves' sums: rows' statistics, then each wave's O scaled to the common maximum
  const float m = fmaxf(rows.m, kNoKey), l = quarters(rows.l, [](float x, float y) { return x + y; });
  auto barrier = [] {
    if constexpr (WAVES == 1) __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    else __syncthreads();
  };
  if (lane < ROWS) {
    red_m[wave][row] = m;
    red_l[wave][row] = l;
  }
  barrier();
  float w = 1.f;
  if constexpr (WAVES > 1)
    w = fast_exp2(m - fmaxf(fmaxf(red_m[0][row], red_m[1][row]), fmaxf(red_m[2][row], red_m[3][row])));
  if (!PACK || (lane & 12) == 0) {
#pragma unroll
    for (int c = 0; c < 4; ++c)
#pragma unroll
      for (int d = 0; d < NDB; ++d) lds[wave][row * ROW + NDB * (4 * quarter + c) + d] = rows.o[d][c] * w;
  }
  barrier();
  const int v = WAVES == 1 ? wave : 0;
  write_rows<HD, ROWS, ROW, SHARED, WAVES>(args_again(), s, b, hk, r0, nr, split, single, lds[v], ROWS * ROW, red_m + v,
                                           red_l + v);
}

// WAVES 1: a wave to a (request, K/V head), which has few keys.
template <typename T, int HD, int RUN, bool PACK, bool SHARED, int WAVES>
__global__ void __launch_bounds__(PT_THREADS, HD <= 128 ? 2 : 1) paged_code_kernel(const PagedArgs a) {
  constexpr int ROWS = CodeRows<T, HD, PACK>::ROWS;
  __shared__ __attribute__((aligned(16))) float lds[4][ROWS * (HD + 4)];
  __shared__ float red_m[4][16], red_l[4][16];
  __shared__ __attribute__((aligned(16))) float scales[4][64];
  const int b = blockIdx.z;
  const PagedSeq s = paged_seq<SHARED>(a, b);
  const int nr = s.n * a.group;
  // K/V head and group of rows
  int y = blockIdx.y, groups = gridDim.y / a.kv_heads;
  if constexpr (WAVES == 1) {
    y = y * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    groups = 1;
    if (y >= a.kv_heads) return;
  }
  const int hk = y % a.kv_heads;
  int r0 = y / a.kv_heads * ROWS;
  if (nr > a.few_rows || r0 >= nr) return;
  if constexpr (SHARED) {
    // (a group of more rows than the launch was told of takes its time)
    for (; r0 < nr; r0 += groups * ROWS) {
      // (arguments read in every turn: held across turns, they would fill the registers)
      const PagedArgs &z = args_again();
      code_rows<T, HD, RUN, PACK, true, WAVES>(z, paged_seq<true>(z, b), b, hk, r0, nr, lds, red_m, red_l, scales);
      if constexpr (WAVES == 1) __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      else __syncthreads();
    }
  } else {
    code_rows<T, HD, RUN, PACK, false, WAVES>(a, s, b, hk, r0, nr, lds, red_m, red_l, scales);
  }
}

template <typename T, int HD, bool PACK, bool SHARED, int WAVES>
void launch_code(const PagedArgs &a, hipStream_t st) {
  constexpr int ROWS = CodeRows<T, HD, PACK>::ROWS;
  const int row_groups = SHARED && a.prefix ? 1 : (a.few_rows + ROWS - 1) / ROWS;
  const int y = WAVES == 1 ? (a.kv_heads + 3) / 4 : a.kv_heads * row_groups;
  const dim3 grid(a.few_splits, y, SHARED && a.prefix ? a.groups : a.batch);
  if (a.page_shift >= 4) paged_code_kernel<T, HD, 16, PACK, SHARED, WAVES><<<grid, PT_THREADS, 0, st>>>(a);
  else if (a.page_shift == 3) paged_code_kernel<T, HD, 8, PACK, SHARED, WAVES><<<grid, PT_THREADS, 0, st>>>(a);
  else paged_code_kernel<T, HD, 1, PACK, SHARED, WAVES><<<grid, PT_THREADS, 0, st>>>(a);
}

template <typename T, int HD, bool SHARED>
void launch_code(const PagedArgs &a, hipStream_t st) {
  if (a.most_rows <= 4) {
    if constexpr (SHARED)
      if (a.lone_waves) return launch_code<T, HD, true, SHARED, 1>(a, st);
    launch_code<T, HD, true, SHARED, 4>(a, st);
  } else if constexpr (kQ8<T>) {
    launch_code<T, HD, false, SHARED, 4>(a, st);
  }
}

// Requests of few rows
template <typename T, bool SHARED>
int launch_codes(const PagedArgs &a, hipStream_t st) {
  if (a.hd <= 32) launch_code<T, 32, SHARED>(a, st);
  else if (a.hd <= 64) launch_code<T, 64, SHARED>(a, st);
  else if (SHARED || a.hd <= 128) launch_code<T, 128, SHARED>(a, st);
  else if constexpr (!SHARED) launch_code<T, 256, SHARED>(a, st);
  return check_launch("paged_code_kernel");
}

// wide: head dims that are multiples of 8, and 16-byte aligned rows of Q and O.
template <typename T, bool SHARED>
int paged_attn_q8(const PagedArgs &args, const PagedKernels &k, bool wide, hipStream_t st) {
  PagedArgs a = args;
  a.wide = wide;
  if (k.span) {
    const int rc = launch_codes<T, SHARED>(a, st);
    if (rc) return rc;
  }
  return k.tile ? launch_tiles<T, SHARED>(a, wide, st) : CDML_OK;
}

}  // namespace
}  // namespace cdml
