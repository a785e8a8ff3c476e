// ugk_draft.hip - verification of drafted tokens against the target's probabilities, from given random numbers.
//
// Draft t of row i stays where u_i q_i(t) < p_i(t), which is with probability min(1, p_i(t) / q_i(t)); behind the first that
// does not, the token comes from max(p_i - q_i, 0), and behind all drafts from p_n: the tokens are then distributed as the
// target's own. The comparison and the cumulative sums are in 64 bits: the products of two floats are exact there, and a sum
// of a vocabulary of floats is off by 2^-35 of itself at most, so that the token hardly depends on the order of additions.
#include <climits>

#include "ugk_internal.h"

namespace ugk {
namespace {

constexpr int kDraftThreads = 1024, kDraftWaves = kDraftThreads / kWave, kSumThreads = 256;
constexpr int kStep = 4 * kDraftThreads;  // floats that a workgroup takes at a time
constexpr int kMaxSegs = 1024;            // segments of a row

// x, or 0 where it is no probability: neither a positive normal (class 8) nor a positive subnormal (7) number.
__device__ __forceinline__ float probability(float x) { return __builtin_amdgcn_classf(x, 1 << 7 | 1 << 8) ? x : 0.0f; }

// One sequence's row that its next token is drawn from: p, less the drafts' probabilities of the row (or null) or without the
// one token (or -1) whose draft was certain.
struct Row {
  const float *p, *less;
  int gone, a, n;  // accepted drafts, drafts
  bool bad;
  __device__ __forceinline__ double one(float x, float y, int v) const {
    return fmax((double)(v == gone ? 0.0f : probability(x)) - (double)probability(y), 0.0);
  }
  // N times four tokens, v0 .. v0 + 3, `step` apart, those from `end` on 0. whole: all of the wavefront's are before it. (All
  // loads before the first use: a branch around each would wait for it.)
  template <int N>
  __device__ __forceinline__ void quads(int v0, int step, int end, bool whole, double (&x)[N][4]) const {
    float4 f[N], g[N];
    if (whole && less) {
#pragma unroll
      for (int i = 0; i < N; i++) {
        f[i] = ld4(p + v0 + i * step);
        g[i] = ld4(less + v0 + i * step);
      }
    } else if (whole) {
#pragma unroll
      for (int i = 0; i < N; i++) {
        f[i] = ld4(p + v0 + i * step);
        g[i] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
      }
    } else {
      const int last = end - 1;
      const auto at = [&](const float *q, int v) {
        return make_float4(q[min(v, last)], q[min(v + 1, last)], q[min(v + 2, last)], q[min(v + 3, last)]);
      };
#pragma unroll
      for (int i = 0; i < N; i++) f[i] = at(p, v0 + i * step);
#pragma unroll
      for (int i = 0; i < N; i++) g[i] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
      if (less) {
#pragma unroll
        for (int i = 0; i < N; i++) g[i] = at(less, v0 + i * step);
      }
#pragma unroll
      for (int i = 0; i < N; i++) {
        const int v = v0 + i * step;
        f[i] = make_float4(v < end ? f[i].x : 0.0f, v + 1 < end ? f[i].y : 0.0f, v + 2 < end ? f[i].z : 0.0f, v + 3 < end ? f[i].w : 0.0f);
        g[i] = make_float4(v < end ? g[i].x : 0.0f, v + 1 < end ? g[i].y : 0.0f, v + 2 < end ? g[i].z : 0.0f, v + 3 < end ? g[i].w : 0.0f);
      }
    }
#pragma unroll
    for (int i = 0; i < N; i++) {
      const int v = v0 + i * step;
      x[i][0] = one(f[i].x, g[i].x, v);
      x[i][1] = one(f[i].y, g[i].y, v + 1);
      x[i][2] = one(f[i].z, g[i].z, v + 2);
      x[i][3] = one(f[i].w, g[i].w, v + 3);
    }
  }
};

// Sequence b's drafts, a lane of every wavefront to each, until one is not accepted; or, if `accepted`, as many as that says.
__device__ Row verify(const float *p, const float *q, const int *draft, const int *n_draft, const float *u, const int *accepted, int b,
                      int K, int V) {
  const int given = n_draft ? n_draft[b] : K, n = min(max(given, 0), K), lane = threadIdx.x & (kWave - 1);
  p += (size_t)b * (K + 1) * V;
  if (q) q += (size_t)b * K * V;
  draft += (size_t)b * K;
  u += (size_t)b * (K + 1);
  Row r;
  r.bad = given != n;
  r.n = n;
  int a = accepted ? accepted[b] : 0;
  for (; a < n && !accepted; a += kWave) {
    const int i = a + lane;
    bool no = i < n;
    if (no) {
      const int t = draft[i];
      if ((unsigned)t < (unsigned)V) {  // else no token: not accepted
        const double pt = probability(p[(size_t)i * V + t]), qt = q ? probability(q[(size_t)i * V + t]) : 1.0;
        no = !((double)u[i] * qt < pt);
      }
    }
    const unsigned long long first = __ballot(no);
    if (first) {
      a += __builtin_ctzll(first);
      break;
    }
  }
  r.a = min(a, n);
  const int t = r.a < n ? draft[r.a] : -1;
  r.bad = r.bad || (r.a < n && (unsigned)t >= (unsigned)V);
  r.p = p + (size_t)r.a * V;
  r.less = r.a < n && q ? q + (size_t)r.a * V : nullptr;
  r.gone = q ? -1 : t;
  return r;
}

// The sums of the segments of every sequence's row, one per workgroup, where one workgroup per sequence would leave most CUs
// idle; and the accepted drafts, for the launch behind this one.
__global__ __launch_bounds__(kSumThreads) void k_draft_sums(double *sums, int *accepted, const float *p, const float *q, const int *draft,
                                                           const int *n_draft, const float *u, int K, int V, int segs, int seg) {
  __shared__ double part[kSumThreads / kWave];
  const int b = blockIdx.x / segs, s = blockIdx.x % segs;
  const Row r = verify(p, q, draft, n_draft, u, nullptr, b, K, V);
  const int from = s * seg, to = min(from + seg, V);
  double t[4] = {0.0, 0.0, 0.0, 0.0};
#pragma unroll 1
  for (int v0 = from; v0 < to; v0 += kStep) {
    double x[kStep / (4 * kSumThreads)][4];
    r.quads(v0 + 4 * (int)threadIdx.x, 4 * kSumThreads, to, v0 + kStep <= to, x);
#pragma unroll
    for (int i = 0; i < kStep / (4 * kSumThreads); i++)
#pragma unroll
      for (int j = 0; j < 4; j++) t[j] += x[i][j];
  }
  const double sum = wave_scan((t[0] + t[1]) + (t[2] + t[3]));
  if ((threadIdx.x & (kWave - 1)) == kWave - 1) part[threadIdx.x / kWave] = sum;
  __syncthreads();
  if (threadIdx.x == 0) {
    sums[blockIdx.x] = (part[0] + part[1]) + (part[2] + part[3]);
    if (s == 0) accepted[b] = r.a;
  }
}

struct DrawLds {
  double seg[kMaxSegs], wave[kDraftWaves];
  int first, last;
};

// The token of row r at the fraction u of its cumulative sum, or -1 where that is 0. `sums`: the segments', or null; a
// wavefront sums a segment then. The segment in which the sum passes is walked with four tokens per thread.
__device__ int draw(const Row &r, int V, int segs, int seg, double u, const double *sums, DrawLds &lds) {
  const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x >> 6;
  int begin = 0;
  double target = 0.0, sofar = 0.0;
  bool any = true;
  if (segs > 1) {
    __syncthreads();  // what a draw before this one had there has been read
    if (sums) {
      for (int s = threadIdx.x; s < segs; s += kDraftThreads) lds.seg[s] = sums[s];
    } else {
#pragma unroll 1
      for (int s = wave; s < segs; s += kDraftWaves) {
        const int from = s * seg, to = min(from + seg, V);
        double t[4] = {0.0, 0.0, 0.0, 0.0};
#pragma unroll 1
        for (int v0 = from; v0 < to; v0 += 16 * kWave) {
          double x[4][4];
          r.quads(v0 + 4 * lane, 4 * kWave, to, v0 + 16 * kWave <= to, x);
#pragma unroll
          for (int i = 0; i < 4; i++)
#pragma unroll
            for (int j = 0; j < 4; j++) t[j] += x[i][j];
        }
        const double sum = wave_scan((t[0] + t[1]) + (t[2] + t[3]));
        if (lane == kWave - 1) lds.seg[s] = sum;
      }
    }
    __syncthreads();
    // by each wavefront alike, a run of segments per lane
    const int per = (segs + kWave - 1) / kWave, s0 = min(lane * per, segs), s1 = min(s0 + per, segs);
    double mine = 0.0;
    for (int s = s0; s < s1; s++) mine += lds.seg[s];
    const double to = wave_scan(mine), total = __shfl(to, kWave - 1);
    any = total > 0.0;
    target = u * total;
    // the first segment that the sum passes the target in, or else the last that has any mass
    const unsigned long long over = __ballot(mine > 0.0 && to > target), some = __ballot(mine > 0.0);
    const int x = over ? __builtin_ctzll(over) : some ? 63 - __builtin_clzll(some) : 0;
    double at = to - mine, held = at;
    int s = s0;
    for (int w = s0; w < s1; w++) {
      const double y = lds.seg[w];
      if (y > 0.0) {
        s = w;
        held = at;
      }
      at += y;
      if (y > 0.0 && at > target) break;
    }
    begin = __shfl(s, x) * seg;
    sofar = __shfl(held, x);
  }
  const int end = segs > 1 ? min(begin + seg, V) : V;
  int token = -1;
  for (int v0 = begin; v0 < end; v0 += kStep) {
    const int v = v0 + 4 * (int)threadIdx.x;
    double y[1][4];
    r.quads(v, 0, end, v0 + kStep <= end, y);
    const double (&x)[4] = y[0];
    const double mine = (x[0] + x[1]) + (x[2] + x[3]), up = wave_scan(mine);
    __syncthreads();  // the last step's have been read
    if (lane == kWave - 1) lds.wave[wave] = up;
    if (threadIdx.x == 0) {
      lds.first = INT_MAX;
      lds.last = -1;
    }
    __syncthreads();
    double before = 0.0, all = 0.0;
#pragma unroll
    for (int w = 0; w < kDraftWaves; w++) {
      before += w < wave ? lds.wave[w] : 0.0;
      all += lds.wave[w];
    }
    if (segs == 1 && v0 == begin) {  // V is at most kStep then: this is the whole row
      any = all > 0.0;
      target = u * all;
    }
    double sum = sofar + (before + (up - mine));
    int past = INT_MAX, last = -1;
#pragma unroll
    for (int i = 0; i < 4; i++) {
      sum += x[i];
      if (x[i] > 0.0) {
        last = v + i;
        if (past == INT_MAX && sum > target) past = v + i;
      }
    }
    const unsigned long long over = __ballot(past != INT_MAX), some = __ballot(last >= 0);
    if (over && lane == __builtin_ctzll(over)) atomicMin(&lds.first, past);
    if (some && lane == 63 - __builtin_clzll(some)) atomicMax(&lds.last, last);
    __syncthreads();
    if (lds.first != INT_MAX) {
      token = lds.first;
      break;
    }
    token = max(token, lds.last);
    sofar += all;
  }
  return any ? token : -1;
}

// One sequence per workgroup. Bound by the row (or two) of V floats that it reads without `sums`, at a CU's share of the
// memory's rate, and by the chain from the drafts to their probabilities, the row and the walk.
__global__ __launch_bounds__(kDraftThreads) void k_draft_verify(int *accepted, int *tokens, const float *p, const float *q, const int *draft,
                                                               const int *n_draft, const float *u, const double *sums, int K, int V,
                                                               int segs, int seg, int *word) {
  __shared__ DrawLds lds;
  const int b = blockIdx.x;
  Row r = verify(p, q, draft, n_draft, u, sums ? accepted : nullptr, b, K, V);
  const double x = u[(size_t)b * (K + 1) + K];
  int token = draw(r, V, segs, seg, x, sums ? sums + (size_t)b * segs : nullptr, lds);
  if (token < 0 && r.a < r.n) {  // p and q are the same
    r.less = nullptr;
    r.gone = -1;
    token = draw(r, V, segs, seg, x, nullptr, lds);
  }
  if (token < 0) {
    token = 0;
    r.bad = true;
  }
  if (r.bad && threadIdx.x == 0) *word = UGK_IDS_DRAFT_VERIFY;
  tokens += (size_t)b * (K + 1);
  draft += (size_t)b * K;
  for (int i = threadIdx.x; i <= K; i += kDraftThreads) tokens[i] = i < r.a ? draft[i] : i == r.a ? token : -1;
  if (threadIdx.x == 0) accepted[b] = r.a;
}

// Segments of a row: whole steps, at most kMaxSegs.
int seg_floats(int V) { return (int)(((long long)V + (long long)kMaxSegs * kStep - 1) / ((long long)kMaxSegs * kStep)) * kStep; }
// Sums in a launch of their own while one workgroup per sequence would leave CUs idle (64 x 50,257 tokens 6.1 + 5.9 us, in one
// launch 21.6); up to two steps are not worth it.
bool separate(int nseq, int V) { return V > 2 * kStep && nseq < 256; }
}  // namespace

size_t draft_verify_bytes(int nseq, int V) {
  return separate(nseq, V) ? (size_t)nseq * (((size_t)V + seg_floats(V) - 1) / seg_floats(V)) * sizeof(double) : 0;
}
// over all vocabularies of up to V
size_t draft_verify_bound(int V) {
  const size_t segs = ((size_t)V + kStep - 1) / kStep;
  return segs > 2 ? 255 * (segs < (size_t)kMaxSegs ? segs : (size_t)kMaxSegs) * sizeof(double) : 0;
}

int launch_draft_verify(int *accepted, int *tokens, const float *p, const float *q, const int *draft, const int *n_draft,
                        const float *u, double *sums, int nseq, int K, int V, int *word) {
  const int seg = seg_floats(V), segs = (int)(((long long)V + seg - 1) / seg);
  if (sums) {
    launch(k_draft_sums, dim3((unsigned)nseq * segs), dim3(kSumThreads), 0, sums, accepted, p, q, draft, n_draft, u, K, V, segs, seg);
    if (int e = check_launch("draft_verify")) return e;
  }
  launch(k_draft_verify, dim3(nseq), dim3(kDraftThreads), 0, accepted, tokens, p, q, draft, n_draft, u, sums, K, V, segs, seg, word);
  return check_launch("draft_verify");
}

}  // namespace ugk
