// Selection of the next beams over beams and vocabulary (cdml_beam_select).
//
// Two launches.  beam_rows_kernel reads every live row's logits once: each wave holds a
// segment of BS_SEG of them in registers and leaves the segment's maximum, its sum of
// exponentials and its `beams` largest logits (no beam can give more to the result).
// beam_pick_kernel, one workgroup per request, joins a row's segments into its
// log-sum-exp and its `beams` best tokens, one wave per row, then merges the rows'
// sorted lists, one lane per beam.
//
// The sum decides between tokens of different beams, whose totals lie arbitrarily close,
// so it is kept in 64 bits, and so are totals and keys.  An exponential is 2^n 2^f with
// n = rint(x log2 e) and f = fma(x, log2 e, -n) (one rounding at 2^-25, whatever x), the
// product with log2 e's low part added: 2^f is off by one rounding of fp32, and these
// do not add up over a sum whose terms are independent.
#include "attn_common.h"

namespace cdml {
namespace {

constexpr int BS_THREADS = 256;
constexpr int BS_PER_LANE = 32;
constexpr int BS_SEG = 64 * BS_PER_LANE;  // logits a wave holds
constexpr int BS_MAX_BEAMS = 64;

struct BeamArgs {
  const float *x;
  const float *scores;
  const int *lengths;
  const uint8_t *finished;
  int ld, batch, beams, vocab, eos, n_seg;
  float penalty;
  float *new_scores;
  int *new_lengths;
  uint8_t *new_finished;
  int *parents, *tokens;
  // workspace, per row and segment
  double *sum;  // sum of exp(x - max)
  float *top;   // max
  float *val;   // [beams] largest logits, -infinity where there are fewer
  int *tok;     // their tokens
};

// exp(x - m) for m >= x, both finite: as 2^(n - n_m) 2^(f - f_m) while x log2 e has
// fraction bits, else from the (then exact or huge) difference.
struct ExpFrom {
  float n, f, m;
  bool small;
  static constexpr float kL = 1.44269502162933349609375f;  // log2 e rounded to fp32
  static constexpr float kLlo = 1.925963034e-08f;     // and the rest of it
  __device__ __forceinline__ static void parts(float x, float &n, float &f) {
    n = rintf(x * kL);
    f = fmaf(x, kLlo, fmaf(x, kL, -n));
  }
  __device__ __forceinline__ explicit ExpFrom(float max) : m(max) {
    parts(max, n, f);
    small = fabsf(max) < 65536.f;
  }
  __device__ __forceinline__ float operator()(float x) const {
    if (!small) return fast_exp2((x - m) * kL);
    x = fmaxf(x, m - 200.f);  // e^-200 is nothing next to e^0, and -infinity has no fraction
    float xn, xf;
    parts(x, xn, xf);
    return ldexpf(fast_exp2(xf - f), (int)(xn - n));
  }
};

__global__ void __launch_bounds__(BS_THREADS) beam_rows_kernel(const BeamArgs a, int vec) {
  const int row = blockIdx.y, lane = threadIdx.x & 63;
  const int seg = blockIdx.x * (BS_THREADS / 64) + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if (seg >= a.n_seg) return;
  // a finished beam's only candidate and a dead beam's none need no logits
  if (a.finished[row] != 0 || !isfinite(a.scores[row])) return;
  const float *x = a.x + (size_t)row * a.ld;
  const int t0 = seg * BS_SEG;
  // element 4 i + c of a lane is token t0 + 256 i + 4 lane + c
  float v[BS_PER_LANE];
#pragma unroll
  for (int i = 0; i < BS_PER_LANE / 4; ++i) {
    const int t = t0 + 256 * i + 4 * lane;
    if (vec && t + 4 <= a.vocab) {
      const vf4 w = *reinterpret_cast<const vf4 *>(x + t);
#pragma unroll
      for (int c = 0; c < 4; ++c) v[4 * i + c] = w[c];
    } else {
#pragma unroll
      for (int c = 0; c < 4; ++c) v[4 * i + c] = t + c < a.vocab ? x[t + c] : -INFINITY;
    }
  }
  float m = -INFINITY;
#pragma unroll
  for (int e = 0; e < BS_PER_LANE; ++e) {
    v[e] = v[e] == v[e] ? v[e] : -INFINITY;  // a NaN is no candidate
    m = fmaxf(m, v[e]);
  }
  const float best0 = m;
  m = wave_max(m);
  const size_t at = (size_t)row * a.n_seg + seg;
  double s = 0;
  if (isfinite(m)) {
    const ExpFrom e_of(m);
#pragma unroll
    for (int e = 0; e < BS_PER_LANE; ++e) s += (double)e_of(v[e]);
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) s += __shfl_xor(s, off);
  }
  if (lane == 0) {
    a.sum[at] = s;
    a.top[at] = m;
  }
  // `beams` times: the wave's largest, on ties the lowest token, leaves its lane
  float best = best0;
  for (int k = 0; k < a.beams; ++k) {
    const float w = k ? wave_max(best) : m;
    if (w == -INFINITY) {  // (the same in every lane)
      for (int r = k + lane; r < a.beams; r += 64) a.val[at * a.beams + r] = -INFINITY;
      break;
    }
    int e = BS_PER_LANE;
#pragma unroll
    for (int i = BS_PER_LANE - 1; i >= 0; --i) e = v[i] == w ? i : e;
    int tok = e < BS_PER_LANE ? t0 + 256 * (e >> 2) + 4 * lane + (e & 3) : INT32_MAX;
    int low = tok;
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) low = min(low, __shfl_xor(low, off));
    if (lane == 0) {
      a.val[at * a.beams + k] = w;
      a.tok[at * a.beams + k] = low;
    }
    if (tok == low) {
      best = -INFINITY;
#pragma unroll
      for (int i = 0; i < BS_PER_LANE; ++i) {
        v[i] = i == e ? -INFINITY : v[i];
        best = fmaxf(best, v[i]);
      }
    }
  }
}

// The order of a merge: the larger key, on ties the lower beam.
__device__ __forceinline__ bool ahead(double ka, int ba, double kb, int bb) {
  return ka > kb || (ka == kb && ba < bb);
}

__global__ void __launch_bounds__(BS_THREADS) beam_pick_kernel(const BeamArgs a) {
  extern __shared__ char smem[];  // per beam: [beams] logits, [beams] tokens; then the sums
  float *val = reinterpret_cast<float *>(smem);
  int *tok = reinterpret_cast<int *>(val + a.beams * a.beams);
  __shared__ double log_sum[BS_MAX_BEAMS];
  __shared__ float row_max[BS_MAX_BEAMS];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int K = a.beams, row0 = blockIdx.x * K;
  for (int k = wave; k < K; k += BS_THREADS / 64) {
    const int row = row0 + k;
    for (int r = lane; r < K; r += 64) val[k * K + r] = -INFINITY;
    if (a.finished[row] != 0 || !isfinite(a.scores[row])) continue;
    const size_t at = (size_t)row * a.n_seg;
    float m = -INFINITY;
    for (int s = lane; s < a.n_seg; s += 64) m = fmaxf(m, a.top[at + s]);
    m = wave_max(m);
    if (!isfinite(m)) continue;
    double sum = 0;
    for (int s = lane; s < a.n_seg; s += 64)
      if (a.top[at + s] > -INFINITY) sum += a.sum[at + s] * exp((double)a.top[at + s] - (double)m);
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) sum += __shfl_xor(sum, off);
    if (lane == 0) {
      row_max[k] = m;
      log_sum[k] = log(sum);
    }
    // the lists of the segments are sorted: lane l keeps a place in those of segments l, l + 64, ...;
    // of equal logits the lowest token comes first
    const int n_list = (a.n_seg + 63) / 64;
    uint32_t taken = 0;  // with n_list == 1, the place in the lane's one list
    for (int r = 0; r < K; ++r) {
      float best = -INFINITY;
      int low = INT32_MAX;
      if (n_list == 1) {
        if (lane < a.n_seg && (int)taken < K) {
          best = a.val[(at + lane) * K + taken];
          if (best > -INFINITY) low = a.tok[(at + lane) * K + taken];
        }
      } else {
        // many segments: everything after the last pick (value, token) in the lists' order
        const float lv = r ? val[k * K + r - 1] : INFINITY;
        const int lt = r ? tok[k * K + r - 1] : -1;
        for (int s = lane; s < a.n_seg; s += 64)
          for (int i = 0; i < K; ++i) {
            const float w = a.val[(at + s) * K + i];
            if (w == -INFINITY) break;
            const int t = a.tok[(at + s) * K + i];
            if (w < lv || (w == lv && t > lt)) {
              if (w > best || (w == best && t < low)) {
                best = w;
                low = t;
              }
              break;
            }
          }
      }
      const float w = wave_max(best);
      if (w == -INFINITY) break;
      const int mine = best == w ? low : INT32_MAX;
      int t = mine;
#pragma unroll
      for (int off = 32; off > 0; off >>= 1) t = min(t, __shfl_xor(t, off));
      if (mine == t) ++taken;
      if (lane == 0) {
        val[k * K + r] = w;
        tok[k * K + r] = t;
      }
      __builtin_amdgcn_wave_barrier();
      __threadfence_block();
    }
  }
  __syncthreads();
  if (wave) return;
  // lane k: beam k's list, its keys falling along it
  const int row = row0 + min(lane, K - 1);
  const double score = a.scores[row];
  const bool done = a.finished[row] != 0;
  const int len = a.lengths[row] + !done;
  const double div = pow((double)max(len, 1), (double)a.penalty);
  const bool live = lane < K && isfinite(a.scores[row]);
  int place = 0;
  double total = 0, key = -INFINITY;
  auto head = [&] {
    key = -INFINITY;
    if (!live) return;
    if (done) {
      if (place) return;
      total = score;
    } else {
      if (place >= K || val[lane * K + place] == -INFINITY) return;
      total = score + (((double)val[lane * K + place] - (double)row_max[lane]) - log_sum[lane]);
    }
    key = total / div;
  };
  head();
  const int pad = max(a.eos, 0);
  for (int r = 0; r < K; ++r) {
    double k = key;
    int b = lane;
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) {
      const double ok = __shfl_xor(k, off);
      const int ob = __shfl_xor(b, off);
      if (ahead(ok, ob, k, b)) {
        k = ok;
        b = ob;
      }
    }
    const int out = row0 + r;
    if (!(k > -INFINITY)) {  // no candidate is left for this place
      if (lane == r) {
        a.parents[out] = out;
        a.tokens[out] = pad;
        a.new_scores[out] = -INFINITY;
        a.new_finished[out] = 1;
        a.new_lengths[out] = len - !done;
      }
      continue;
    }
    if (lane == b) {
      const int t = done ? pad : tok[lane * K + place];
      a.parents[out] = row0 + b;
      a.tokens[out] = t;
      a.new_scores[out] = (float)total;
      a.new_finished[out] = done || t == a.eos;
      a.new_lengths[out] = len;
      ++place;
      head();
    }
  }
}

size_t align_up(size_t n) { return (n + 15) & ~(size_t)15; }

struct Layout {
  size_t sum, top, val, tok, bytes;
  int n_seg;
};
Layout layout(int batch, int beams, int vocab) {
  Layout l{};
  l.n_seg = (int)(((long long)vocab + BS_SEG - 1) / BS_SEG);
  const size_t n = (size_t)batch * beams * l.n_seg;
  l.sum = 0;
  l.top = l.sum + align_up(n * sizeof(double));
  l.val = l.top + align_up(n * sizeof(float));
  l.tok = l.val + align_up(n * beams * sizeof(float));
  l.bytes = l.tok + align_up(n * beams * sizeof(int));
  return l;
}

}  // namespace
}  // namespace cdml

using namespace cdml;

extern "C" int cdml_beam_select_workspace_size(int batch, int beams, int vocab, size_t *bytes) {
  if (!bytes) return fail(CDML_E_INVALID, "cdml_beam_select_workspace_size: bytes is NULL");
  if (batch < 0 || beams < 1 || beams > BS_MAX_BEAMS || vocab < 1 || (long long)batch * beams > 65535)
    return fail(CDML_E_INVALID,
                "cdml_beam_select: bad size (batch %d, beams %d of at most %d, vocab %d; at most 65535 rows)", batch,
                beams, BS_MAX_BEAMS, vocab);
  *bytes = layout(batch, beams, vocab).bytes;
  return CDML_OK;
}

extern "C" int cdml_beam_select(const float *logits, int ldl, const float *scores, const int *lengths,
                                const uint8_t *finished, int batch, int beams, int vocab, int eos_token,
                                float length_penalty, float *new_scores, int *new_lengths, uint8_t *new_finished,
                                int *parents, int *tokens, void *workspace, size_t workspace_bytes,
                                cdml_stream stream) {
  size_t need = 0;
  int rc = cdml_beam_select_workspace_size(batch, beams, vocab, &need);
  if (rc) return rc;
  if (ldl < vocab || eos_token >= vocab)
    return fail(CDML_E_INVALID, "cdml_beam_select: ldl %d below vocab, or eos_token %d outside it", ldl, eos_token);
  if (!(length_penalty >= -16.f && length_penalty <= 16.f))
    return fail(CDML_E_INVALID, "cdml_beam_select: length_penalty outside [-16, 16]");
  if (batch == 0) return CDML_OK;
  if (!logits || !scores || !lengths || !finished || !new_scores || !new_lengths || !new_finished || !parents ||
      !tokens)
    return fail(CDML_E_INVALID, "cdml_beam_select: NULL pointer");
  if (!workspace || workspace_bytes < need || !aligned16(workspace))
    return fail(CDML_E_INVALID, "cdml_beam_select: %zu bytes of 16-byte aligned workspace needed, %zu given", need,
                workspace_bytes);
  rc = ensure_device();
  if (rc) return rc;
  const Layout l = layout(batch, beams, vocab);
  char *ws = static_cast<char *>(workspace);
  BeamArgs a{};
  a.x = logits;
  a.scores = scores;
  a.lengths = lengths;
  a.finished = finished;
  a.ld = ldl;
  a.batch = batch;
  a.beams = beams;
  a.vocab = vocab;
  a.eos = eos_token;
  a.n_seg = l.n_seg;
  a.penalty = length_penalty;
  a.new_scores = new_scores;
  a.new_lengths = new_lengths;
  a.new_finished = new_finished;
  a.parents = parents;
  a.tokens = tokens;
  a.sum = reinterpret_cast<double *>(ws + l.sum);
  a.top = reinterpret_cast<float *>(ws + l.top);
  a.val = reinterpret_cast<float *>(ws + l.val);
  a.tok = reinterpret_cast<int *>(ws + l.tok);
  const int vec = ldl % 4 == 0 && aligned16(logits);
  const dim3 grid((unsigned)((l.n_seg + 3) / 4), (unsigned)(batch * beams));
  beam_rows_kernel<<<grid, BS_THREADS, 0, as_hip(stream)>>>(a, vec);
  rc = check_launch("beam_rows_kernel");
  if (rc) return rc;
  beam_pick_kernel<<<batch, BS_THREADS, 8 * beams * beams, as_hip(stream)>>>(a);
  return check_launch("beam_pick_kernel");
}
