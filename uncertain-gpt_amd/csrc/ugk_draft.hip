// ugk_draft.hip - verification of drafted tokens against the target's
// probabilities, from given random numbers.
//
// Draft t of row i stays where u_i q_i(t) < p_i(t), which is with probability min(1, p_i(t) / q_i(t)); behind the first
// that does not, the token comes from max(p_i - q_i, 0), and behind all drafts from p_n: the tokens are then distributed as
// the target's own. The comparison and the cumulative sums are in 64 bits: the products of two floats are exact there, and a sum of a
// vocabulary of floats is off by 2^-35 of itself at most, so that the token hardly depends on the order of additions.
#include "ugk_internal.h"

namespace ugk {
namespace {

constexpr int kDraftThreads = 1024, kDraftWaves = kDraftThreads / kWave;

__device__ __forceinline__ double wave_sum64(double x) {
#pragma unroll
  for (int o = 32; o; o >>= 1) x += __shfl_xor(x, o);
  return x;
}

// What token v of a row may be drawn with. less: the drafts' probabilities of the row, or null; gone: the token that
// is not drawn (its draft was certain), or -1.
__device__ __forceinline__ double mass(const float *p, const float *less, int gone, int v) {
  const double x = less ? (double)p[v] - (double)less[v] : (double)p[v];
  return v != gone && x > 0.0 && x <= 3.402823466e38 ? x : 0.0;
}

// The token at the fraction u of the cumulative sum of [0, V), or -1 where the sum is 0: the sixteen wavefronts sum a
// sixteenth each, then a sixteenth of the one in which the sum passes, then one wavefront walks that 256th.
__device__ int draw(const float *p, const float *less, int gone, int V, double u, double *lds) {
  const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x >> 6;
  int begin = 0, end = V;
  double target = 0.0;
  bool any = true;
#pragma unroll 1
  for (int level = 0; level < 2; level++) {
    const int per = (end - begin + kDraftWaves - 1) / kDraftWaves;
    const int from = min(begin + wave * per, end), to = min(from + per, end);
    double s0 = 0.0, s1 = 0.0, s2 = 0.0, s3 = 0.0;
    int v = from + lane;
    for (; v + 3 * kWave < to; v += 4 * kWave) {
      s0 += mass(p, less, gone, v);
      s1 += mass(p, less, gone, v + kWave);
      s2 += mass(p, less, gone, v + 2 * kWave);
      s3 += mass(p, less, gone, v + 3 * kWave);
    }
    for (; v < to; v += kWave) s0 += mass(p, less, gone, v);
    const double sum = wave_sum64((s0 + s1) + (s2 + s3));
    __syncthreads();  // the last level's sums have been read
    if (lane == 0) lds[wave] = sum;
    __syncthreads();
    double total = 0.0;
    for (int w = 0; w < kDraftWaves; w++) total += lds[w];
    if (level == 0) {
      any = total > 0.0;
      target = u * total;
    }
    // the first part that the sum passes the target in, or else the last that has any mass
    double sofar = 0.0, at = 0.0;
    int part = 0;
    for (int w = 0; w < kDraftWaves; w++) {
      const double x = lds[w];
      if (x > 0.0) {
        part = w;
        at = sofar;
      }
      sofar += x;
      if (x > 0.0 && sofar > target) break;
    }
    target -= at;
    const int lo = min(begin + part * per, end);
    end = min(lo + per, end);
    begin = lo;
  }
  int token = -1;
  double sofar = 0.0;
  for (int v0 = begin; v0 < end; v0 += kWave) {  // by each wavefront alike
    const double x = v0 + lane < end ? mass(p, less, gone, v0 + lane) : 0.0;
    double y = x;
#pragma unroll
    for (int o = 1; o < kWave; o *= 2) {
      const double z = __shfl_up(y, o);
      if (lane >= o) y += z;
    }
    const unsigned long long some = __ballot(x > 0.0), past = __ballot(x > 0.0 && sofar + y > target);
    if (past) {
      token = v0 + __builtin_ctzll(past);
      break;
    }
    if (some) token = v0 + 63 - __builtin_clzll(some);
    sofar += __shfl(y, kWave - 1);
  }
  return any ? token : -1;
}

// One sequence per workgroup. Bound by the two rows of V floats that it reads (the second level reads a sixteenth of them
// again, from a cache), at a CU's share of the memory's rate.
__global__ __launch_bounds__(kDraftThreads) void k_draft_verify(int *accepted, int *tokens, const float *p, const float *q,
                                                               const int *draft, const int *n_draft, const float *u, int K, int V,
                                                               int *word) {
  __shared__ double lds[kDraftWaves];
  const int b = blockIdx.x, given = n_draft ? n_draft[b] : K, n = min(max(given, 0), K);
  p += (size_t)b * (K + 1) * V;
  if (q) q += (size_t)b * K * V;
  draft += (size_t)b * K;
  u += (size_t)b * (K + 1);
  int a = 0;
  bool bad = given != n;
  for (; a < n; a++) {
    const int t = draft[a];
    if ((unsigned)t >= (unsigned)V) {  // no token: not accepted
      bad = true;
      break;
    }
    const double pt = p[(size_t)a * V + t], qt = q ? q[(size_t)a * V + t] : 1.0;
    if (!((double)u[a] * qt < pt)) break;
  }
  const float *row = p + (size_t)a * V, *less = a < n && q ? q + (size_t)a * V : nullptr;
  int token = draw(row, less, a < n && !q ? draft[a] : -1, V, (double)u[K], lds);
  if (token < 0 && a < n) token = draw(row, nullptr, -1, V, (double)u[K], lds);  // p and q are the same
  if (token < 0) {
    token = 0;
    bad = true;
  }
  if (bad && threadIdx.x == 0) *word = UGK_IDS_DRAFT_VERIFY;
  tokens += (size_t)b * (K + 1);
  for (int i = threadIdx.x; i <= K; i += kDraftThreads) tokens[i] = i < a ? draft[i] : i == a ? token : -1;
  if (threadIdx.x == 0) accepted[b] = a;
}

}  // namespace

int launch_draft_verify(int *accepted, int *tokens, const float *p, const float *q, const int *draft, const int *n_draft,
                        const float *u, int nseq, int K, int V, int *word) {
  launch(k_draft_verify, dim3(nseq), dim3(kDraftThreads), 0, accepted, tokens, p, q, draft, n_draft, u, K, V, word);
  return check_launch("draft_verify");
}

}  // namespace ugk
