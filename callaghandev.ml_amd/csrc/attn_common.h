// What the attention kernels share: the layout of MFMA accumulators, reductions over
// the half-waves and division by launch constants.
#pragma once

#include "common.h"

namespace cdml {
namespace {

constexpr float kLog2e = 1.4426950408889634f;

// Division by a launch-constant divisor d >= 1 for dividends 0 <= x < 2^31:
// x / d = (x * m) >> l with l = 31 + ceil(log2 d) and m = ceil(2^l / d) < 2^32
// (the error m * d - 2^l is below d, so x * error < 2^l for every such x).
// Block-uniform dividends keep the division on the scalar unit.
struct UDiv {
  uint32_t m;
  int l;
  static UDiv make(uint32_t d) {
    if (d == 0) d = 1;  // no launch divides by it
    int s = 0;
    while ((1ull << s) < d) ++s;
    const int l = 31 + s;
    return {(uint32_t)(((1ull << l) + d - 1) / d), l};
  }
  __device__ __forceinline__ int div(int x) const { return (int)(((uint64_t)(uint32_t)x * m) >> l); }
};

// max / sum of a value over the two half-waves (lanes l and l ^ 32) with
// v_permlane32_swap: both results hold the value of lane l % 32 and of lane
// l % 32 + 32.
__device__ __forceinline__ float halves_max(float x) {
#pragma float_control(precise, off)
  auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __builtin_fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));  // scores: no signalling NaN
}
__device__ __forceinline__ float halves_sum(float x) {
  auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

// A lane's neighbour by a DPP control, without a trip through LDS: quad_perm patterns
// exchange lane ^ 1 (0xB1) and lane ^ 2 (0x4E); mirrors of 8 (0x141) and 16 lanes (0x140)
// then pair the uniform quads and groups of 8.
template <int CTRL>
__device__ __forceinline__ uint32_t dpp(uint32_t x) {
  return __builtin_amdgcn_update_dpp(0, x, CTRL, 0xf, 0xf, true);
}
template <int CTRL>
__device__ __forceinline__ float dpp(float x) {
  return __uint_as_float(dpp<CTRL>(__float_as_uint(x)));
}
// f over all 64 lanes, in each of them (f commutative and associative; every lane active).
template <typename T, typename F>
__device__ __forceinline__ T wave_reduce(T x, F f) {
  static_assert(sizeof(T) == 4, "one register");
  uint32_t w = __builtin_bit_cast(uint32_t, x);
  auto with = [&](uint32_t o) {
    w = __builtin_bit_cast(uint32_t, f(__builtin_bit_cast(T, w), __builtin_bit_cast(T, o)));
  };
  with(dpp<0xB1>(w));
  with(dpp<0x4E>(w));
  with(dpp<0x141>(w));
  with(dpp<0x140>(w));
  auto r = __builtin_amdgcn_permlane16_swap(w, w, false, false);
  w = r[0];
  with(r[1]);
  r = __builtin_amdgcn_permlane32_swap(w, w, false, false);
  w = r[0];
  with(r[1]);
  return __builtin_bit_cast(T, w);
}
// The same for a double, whose words travel together.
template <typename F>
__device__ __forceinline__ double wave_reduce64(double x, F f) {
  auto with = [&](uint32_t lo, uint32_t hi) {
    x = f(x, __builtin_bit_cast(double, (uint64_t)hi << 32 | lo));
  };
  auto lo = [&] { return (uint32_t)__builtin_bit_cast(uint64_t, x); };
  auto hi = [&] { return (uint32_t)(__builtin_bit_cast(uint64_t, x) >> 32); };
  with(dpp<0xB1>(lo()), dpp<0xB1>(hi()));
  with(dpp<0x4E>(lo()), dpp<0x4E>(hi()));
  with(dpp<0x141>(lo()), dpp<0x141>(hi()));
  with(dpp<0x140>(lo()), dpp<0x140>(hi()));
  // both results of a swap hold the own value in one half of the lanes and the partner's
  // in the other: f of the two is the pair's
  auto swap = [&](auto a, auto b) {
    x = __builtin_bit_cast(double, (uint64_t)b[0] << 32 | a[0]);
    with(a[1], b[1]);
  };
  swap(__builtin_amdgcn_permlane16_swap(lo(), lo(), false, false),
       __builtin_amdgcn_permlane16_swap(hi(), hi(), false, false));
  swap(__builtin_amdgcn_permlane32_swap(lo(), lo(), false, false),
       __builtin_amdgcn_permlane32_swap(hi(), hi(), false, false));
  return x;
}
__device__ __forceinline__ float wave_max(float x) {
  return wave_reduce(x, [](float a, float b) { return fmaxf(a, b); });
}
__device__ __forceinline__ float wave_sum(float x) {
  return wave_reduce(x, [](float a, float b) { return a + b; });
}
__device__ __forceinline__ int wave_min(int x) {
  return wave_reduce(x, [](int a, int b) { return min(a, b); });
}

// max of three scores.  The scores come from MFMA accumulators and are
// never signalling NaNs, so the IEEE quieting that fmaxf otherwise adds to
// each operand is dropped (one v_max3_f32 instead of five instructions).
__device__ __forceinline__ float max3_scores(float a, float b, float c) {
#pragma float_control(precise, off)
  return __builtin_fmaxf(__builtin_fmaxf(a, b), c);
}

// Growth of the running max (log2 units) tolerated before the output is
// rescaled: probabilities stay <= 2^8, far from fp32 overflow.
constexpr float kRescaleThreshold = 8.0f;

// Offset of accumulator register r's key inside its 32-key sub-block for a
// lane of half-wave h: 8 * (r / 4) + 4 * h + r % 4 (the 32x32 MFMA D layout).
__device__ __forceinline__ constexpr int acc_key(int r) { return 8 * (r >> 2) + (r & 3); }

// A sub-block whose per-lane probability sum stays at or below this bound is
// accumulated without looking at its maximum: no probability exceeds it, so
// nothing overflows (the running sums stay below 2^32 times the key count).
constexpr float kFastSumLimit = 4294967296.0f;  // 2^32

}  // namespace
}  // namespace cdml
