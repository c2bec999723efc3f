// Selection of the next beams over beams and vocabulary (cdml_beam_select).
//
// Two launches, or one up to 512 logits, which the second kernel then reads itself.
// beam_rows_kernel reads every live row's logits once: each wave holds a segment of them in
// registers (64 * BS_LONG, or 64 * BS_SHORT) and leaves the segment's maximum, its sum of
// exponentials and its `beams` largest logits (no beam can give more to the result).
// beam_pick_kernel, one workgroup per request, joins a row's segments into its
// log-sum-exp and its `beams` best tokens, one wave per row, then merges the rows'
// sorted lists, one lane per beam.
//
// A wave finds its largest logits by a threshold: the `beams`-th largest of its 64 lanes'
// maxima, found without a look at the other values, is at most the `beams`-th largest of
// all; the few values that reach it are ranked against each other, one to a lane.  Where
// more than 64 do (equal logits), the largest is taken out `beams` times instead.
//
// The sum decides between tokens of different beams, whose totals lie arbitrarily close,
// so it is kept in 64 bits, and so are totals and keys.  With L the fp32 value next to
// log2 e and r = rint(m L) for a segment's maximum m, an exponential is 2^r 2^t with t =
// fma(x, L, -r): one rounding, small where the term is large.  What L leaves out, k =
// log2 e / L - 1, moves the whole sum: sum e^x = 2^r (s + k ln 2 (r s + sum t 2^t)) with s =
// sum 2^t, to the first order of k; and segments of any r join exactly.  From |m| = 1024 on
// the difference x - m is taken first: it is exact for every x whose term counts.
#include <cfloat>

#include "attn_common.h"

namespace cdml {
namespace {

constexpr int BS_THREADS = 256;
// Logits a lane holds, and a wave with it: a segment.
constexpr int BS_LONG = 32, BS_SHORT = 8;
constexpr int BS_PICK = 8;  // values a lane of the pick kernel holds, one for those picked before
constexpr int BS_MAX_BEAMS = 64;
// Short segments, while they leave a wave or so for every place on the card and a row's
// candidates to one pass of the pick kernel.  8 beams of 64 requests over 2048 logits (2048
// segments) 15.7 us in long ones, 14.4 in short, over 8192 (8192) 16.5, 19.2; of 4 requests
// over 16000 (252 candidates) 16.2, 14.6, over 50021 (784) 16.1, 19.7; 4 of 4 over 50021 (392)
// 12.1, 11.5.
constexpr int BS_SHORT_SEGMENTS = 4096, BS_SHORT_CANDIDATES = 64 * (BS_PICK - 1);

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
  double *sum;  // sum of exponentials, relative to what the maximum says
  float *top;   // max
  float *val;   // [beams] largest logits, -infinity where there are fewer
  int *tok;     // their tokens
};

constexpr float kL = 1.44269502162933349609375f;  // log2 e rounded to fp32
constexpr double kLeft = 1.3349758349838184e-8;   // log2 e / kL - 1
constexpr double kLn2 = 0.69314718055994531;

// The exponent of two that a segment's sum is taken relative to, from its maximum; and
// whether it is, or the maximum itself.
__device__ __forceinline__ float ref_exponent(float m) { return rintf(m * kL); }
__device__ __forceinline__ bool by_exponent(float m) { return fabsf(m) < 1024.f; }

// Sum over this lane's E values of e^x / 2^ref_exponent(m), or of e^(x - m).
template <int E>
__device__ __forceinline__ double sum_exp(const float (&x)[E], float m) {
  double s = 0;
  if (by_exponent(m)) {
    const float r = ref_exponent(m);
    float s1 = 0.f;
#pragma unroll
    for (int e = 0; e < E; e += 2) {
      const float t0 = fmaxf(fmaf(x[e], kL, -r), -200.f), t1 = fmaxf(fmaf(x[e + 1], kL, -r), -200.f);
      const float e0 = fast_exp2(t0), e1 = fast_exp2(t1);  // (2^-200 is 0)
      s1 = fmaf(t1, e1, fmaf(t0, e0, s1));
      s += (double)(e0 + e1);
    }
    return s + kLeft * kLn2 * ((double)r * s + (double)s1);
  }
#pragma unroll
  for (int e = 0; e < E; ++e) {
    const float d = fmaxf(x[e] - m, -200.f);
    s += (double)fast_exp2(fmaf(d, (float)(kLeft * kL), d * kL));
  }
  return s;
}

// A wave's list of candidates that reach its threshold.
struct TopList {
  float v[64];
  int t[64];
};

// The K largest of the wave's values (E to a lane; NaNs and -infinity are none; best: the
// lane's largest, m: the wave's), on ties the lowest token first, into val / tok in that
// order; -infinity where there are fewer.  token_of(e): the token of the lane's value e.
template <int E, typename F>
__device__ __forceinline__ void select_top(float (&v)[E], float best, float m, int K, TopList &list, float *val, int *tok,
                                           F token_of) {
  const int lane = threadIdx.x & 63;
  // the threshold: lanes' maxima leave one by one, equal ones together
  float least = m, mine = best;
  for (int out = 0;;) {
    out += __popcll(__builtin_amdgcn_ballot_w64(mine == least));
    if (least == -INFINITY || out >= K) break;
    mine = mine == least ? -INFINITY : mine;
    least = wave_max(mine);
  }
  // the values that reach it, in a list that lies one to a lane
  least = fmaxf(least, -FLT_MAX);
  int found = 0;
#pragma unroll
  for (int e = 0; e < E; ++e) {
    const bool reach = v[e] >= least;
    const uint64_t who = __builtin_amdgcn_ballot_w64(reach);
    if (who == 0) continue;
    const int place =
        found + __builtin_amdgcn_mbcnt_hi((uint32_t)(who >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)who, 0));
    if (reach && place < 64) {
      list.v[place] = v[e];
      list.t[place] = token_of(e);
    }
    found += __popcll(who);
  }
  if (found <= 64) {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");  // (the list is this wave's own)
    const float x0 = lane < found ? list.v[lane] : -INFINITY;
    const int x1 = lane < found ? list.t[lane] : INT32_MAX;
    int rank = 0;
    for (int i = 0; i < found; ++i) {
      const float y0 = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(x0), i));
      const int y1 = __builtin_amdgcn_readlane(x1, i);
      rank += y0 > x0 || (y0 == x0 && y1 < x1);
    }
    if (lane < found && rank < K) {
      val[rank] = x0;
      tok[rank] = x1;
    }
    for (int r = found + lane; r < K; r += 64) val[r] = -INFINITY;
    return;
  }
  // K times: the wave's largest, on ties the lowest token, leaves its lane
  for (int k = 0; k < K; ++k) {
    const float w = k ? wave_max(best) : m;
    if (w == -INFINITY) {  // (the same in every lane)
      for (int r = k + lane; r < K; r += 64) val[r] = -INFINITY;
      break;
    }
    int t = INT32_MAX;
#pragma unroll
    for (int e = 0; e < E; ++e) t = v[e] == w ? min(t, token_of(e)) : t;
    const int low = wave_min(t);
    if (lane == 0) {
      val[k] = w;
      tok[k] = low;
    }
    if (t == low) {
      best = -INFINITY;
#pragma unroll
      for (int e = 0; e < E; ++e) {
        v[e] = v[e] == w && token_of(e) == low ? -INFINITY : v[e];
        best = fmaxf(best, v[e]);
      }
    }
  }
}

// A wave's values of segment seg of a row's logits: element e of a lane is token
// 64 (E seg + e) + lane.  Those past the vocabulary are no candidates.
template <int E>
__device__ __forceinline__ void load_segment(float (&v)[E], const float *x, int seg, int vocab) {
  const int lane = threadIdx.x & 63, t0 = seg * 64 * E + lane;
  x += seg * 64 * E;
  if ((seg + 1) * 64 * E <= vocab) {
#pragma unroll
    for (int e = 0; e < E; ++e) v[e] = x[(uint32_t)(lane + 64 * e)];
  } else {
#pragma unroll
    for (int e = 0; e < E; ++e) v[e] = t0 + 64 * e < vocab ? x[(uint32_t)(lane + 64 * e)] : -INFINITY;
  }
}
template <int E>
__device__ __forceinline__ float largest(const float (&v)[E]) {
  float best = -INFINITY;
#pragma unroll
  for (int e = 0; e < E; ++e) best = fmaxf(best, v[e]);  // (of a NaN, the other)
  return best;
}

// Reading the logits and the instructions for each bound it alike: 512 rows of 50021 (102 MB)
// take 22 us, 4.6 TB/s.  (25 us while NaNs were taken out one by one; 28 and 30 with segments of
// half and twice the length; 16-byte loads change nothing.)
template <int E>
__global__ void __launch_bounds__(BS_THREADS) beam_rows_kernel(const BeamArgs a) {
  __shared__ TopList lists[BS_THREADS / 64];
  const int row = blockIdx.y, lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int seg = blockIdx.x * (BS_THREADS / 64) + wave;
  if (seg >= a.n_seg) return;
  float v[E];
  load_segment<E>(v, a.x + (size_t)row * a.ld, seg, a.vocab);
  // a finished beam's only candidate and a dead beam's none need no logits
  if (a.finished[row] != 0 || !isfinite(a.scores[row])) return;
  const float best = largest<E>(v);
  const float m = wave_max(best);
  const size_t at = (size_t)row * a.n_seg + seg;
  double s = 0;
  if (isfinite(m)) s = wave_reduce64(sum_exp<E>(v, m), [](double x, double y) { return x + y; });
  if (lane == 0) {
    a.sum[at] = s;
    a.top[at] = m;
  }
  select_top<E>(v, best, m, a.beams, lists[wave], a.val + at * a.beams, a.tok + at * a.beams,
                [&](int e) { return (seg * E + e) * 64 + lane; });
}

// ONE: the whole vocabulary is one short segment, and its row's wave reads the logits itself
// (8 beams of 64 requests, vocabulary 512: 9.6 us; 14.2 with a launch for the rows).  Chains of
// reductions over a wave bound it, the merge's one for each of the beams: 8 x 8 beams with 25
// segments 10 us.
template <bool ONE>
__global__ void __launch_bounds__(1024) beam_pick_kernel(const BeamArgs a) {
  extern __shared__ char smem[];  // per beam: [beams] logits, [beams] tokens
  float *val = reinterpret_cast<float *>(smem);
  int *tok = reinterpret_cast<int *>(val + a.beams * a.beams);
  __shared__ TopList lists[16];
  __shared__ double log_sum[BS_MAX_BEAMS], log_ref[BS_MAX_BEAMS];  // their sum is the row's log-sum-exp
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int K = a.beams, row0 = blockIdx.x * K;
  // what the merge needs of lane k's beam, read ahead of everything that waits
  const int row = row0 + min(lane, K - 1);
  const float score32 = a.scores[row];
  const bool done = a.finished[row] != 0;
  const int len = a.lengths[row] + !done;
  for (int k = wave; k < K; k += blockDim.x / 64) {
    const bool offers = a.finished[row0 + k] == 0 && isfinite(a.scores[row0 + k]);
    if constexpr (ONE) {
      float v[BS_SHORT];
      load_segment<BS_SHORT>(v, a.x + (size_t)(row0 + k) * a.ld, 0, a.vocab);
      const float best = largest<BS_SHORT>(v), m = wave_max(best);
      if (!offers || !isfinite(m)) {
        for (int r = lane; r < K; r += 64) val[k * K + r] = -INFINITY;
        continue;
      }
      const double sum = wave_reduce64(sum_exp<BS_SHORT>(v, m), [](double x, double y) { return x + y; });
      if (lane == 0) {
        log_ref[k] = by_exponent(m) ? kLn2 * (double)ref_exponent(m) : (double)m;
        log_sum[k] = log(sum);
      }
      select_top<BS_SHORT>(v, best, m, K, lists[wave], val + k * K, tok + k * K,
                           [&](int e) { return 64 * e + lane; });
      continue;
    }
    const size_t at = (size_t)(row0 + k) * a.n_seg;
    // the row's candidates, seven a lane and pass, beside the best K of the passes before
    constexpr int E = BS_PICK;
    const int n_cand = a.n_seg * K;
    float v[E];
    int t[E];
    auto load = [&](int from) {
#pragma unroll
      for (int e = 1; e < E; ++e) {
        const int i = from + 64 * (e - 1) + lane;
        v[e] = i < n_cand ? a.val[at * K + i] : -INFINITY;
        t[e] = i < n_cand ? a.tok[at * K + i] : 0;
      }
    };
    load(0);
    float m = -INFINITY;
    for (int s = lane; s < a.n_seg; s += 64) m = fmaxf(m, a.top[at + s]);
    m = wave_max(m);
    // (the lists and maxima of a row that offers nothing are whatever the workspace held)
    if (!offers || !isfinite(m)) {
      for (int r = lane; r < K; r += 64) val[k * K + r] = -INFINITY;
      continue;
    }
    // segments relative to the row's own exponent, or its maximum
    const bool pow2 = by_exponent(m);
    const double ref = pow2 ? kLn2 * (double)ref_exponent(m) : (double)m;
    double sum = 0;
    for (int s = lane; s < a.n_seg; s += 64) {
      const float top = a.top[at + s];
      const double part = a.sum[at + s];
      if (top == -INFINITY) continue;
      if (pow2 && by_exponent(top)) sum += ldexp(part, (int)(ref_exponent(top) - ref_exponent(m)));
      else sum += part * exp((by_exponent(top) ? kLn2 * (double)ref_exponent(top) : (double)top) - ref);
    }
    sum = wave_reduce64(sum, [](double x, double y) { return x + y; });
    if (lane == 0) {
      log_ref[k] = ref;
      log_sum[k] = log(sum);
    }
    v[0] = -INFINITY;
    t[0] = 0;
    for (int from = 0; from < n_cand; from += 64 * (E - 1)) {
      if (from) {
        load(from);
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");  // (val and tok: this wave's own)
        v[0] = lane < K ? val[k * K + lane] : -INFINITY;
        t[0] = lane < K ? tok[k * K + lane] : 0;
      }
      float best = v[0];
#pragma unroll
      for (int e = 1; e < E; ++e) best = fmaxf(best, v[e]);
      select_top<E>(v, best, wave_max(best), K, lists[wave], val + k * K, tok + k * K, [&](int e) { return t[e]; });
    }
  }
  __syncthreads();
  if (wave) return;
  // lane k: beam k's list, its keys falling along it; on equal keys the lowest lane wins
  const double score = score32;
  const double per = a.penalty == 0.f ? 1.0 : pow((double)max(len, 1), -(double)a.penalty);
  const bool live = lane < K && isfinite(score32);
  const int pad = max(a.eos, 0);
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
      total = score + (((double)val[lane * K + place] - log_ref[lane]) - log_sum[lane]);
    }
    key = total * per;
  };
  head();
  for (int r = 0; r < K; ++r) {
    const double k = wave_reduce64(key, [](double x, double y) { return y > x ? y : x; });
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
    const int b = __builtin_ctzll(__builtin_amdgcn_ballot_w64(key == k));
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
  int n_seg, per_lane;
};
Layout layout(int batch, int beams, int vocab) {
  Layout l{};
  const long long shorts = ((long long)vocab + 64 * BS_SHORT - 1) / (64 * BS_SHORT);
  const bool few = (long long)batch * beams * shorts <= BS_SHORT_SEGMENTS && beams * shorts <= BS_SHORT_CANDIDATES;
  l.per_lane = few ? BS_SHORT : BS_LONG;
  const int seg = 64 * l.per_lane;
  l.n_seg = (int)(((long long)vocab + seg - 1) / seg);
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
  if (batch < 0 || beams < 1 || beams > BS_MAX_BEAMS || vocab < 1 || vocab > (1 << 30) ||
      (long long)batch * beams > 65535)
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
  // a wave for every beam, up to 16
  const dim3 pick(64 * (beams < 16 ? beams : 16));
  const size_t smem = 8 * (size_t)beams * beams;
  if (vocab <= 64 * BS_SHORT) {
    beam_pick_kernel<true><<<batch, pick, smem, as_hip(stream)>>>(a);
    return check_launch("beam_pick_kernel");
  }
  const dim3 grid((unsigned)((l.n_seg + 3) / 4), (unsigned)(batch * beams));
  if (l.per_lane == BS_SHORT) beam_rows_kernel<BS_SHORT><<<grid, BS_THREADS, 0, as_hip(stream)>>>(a);
  else beam_rows_kernel<BS_LONG><<<grid, BS_THREADS, 0, as_hip(stream)>>>(a);
  rc = check_launch("beam_rows_kernel");
  if (rc) return rc;
  beam_pick_kernel<false><<<batch, pick, smem, as_hip(stream)>>>(a);
  return check_launch("beam_pick_kernel");
}
