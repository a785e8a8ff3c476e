// ugk_attention.hip - causal attention over packed sequences with grouped
// heads, forward and backward (gpt2_kernels.cuh:416-619 computes the case of
// equal lengths, one key/value head per query head and head size 64).
//
// Per query row i and head, over its allowed keys: s_j = scale q.k_j, p =
// softmax(s), out = sum p_j v_j, lse = log sum exp s_j. Backward, with D =
// dout.out: p_j = exp(s_j - lse), dv_j += p_j dout, ds_j = p_j (dout.v_j - D)
// scale, dq += ds_j k_j, dk_j += ds_j q; dk and dv sum over the query heads of
// the group.
#include <math.h>

#include "ugk_internal.h"

namespace ugk {
namespace {

// One sequence: its first rows and its lengths.
struct Seq {
  int q0, k0, Lq, Lk;
  // the keys that query row i sees: [0, seen(i))
  __device__ __forceinline__ int seen(int i, int causal) const { return causal ? max(0, min(Lk, i + 1 + Lk - Lq)) : Lk; }
  // the first query row that sees key j
  __device__ __forceinline__ int first(int j, int causal) const { return causal ? max(0, j - (Lk - Lq)) : 0; }
};

// Rows [begin, end) of `rows`, at most `most` of them; *bad: the arrays say otherwise.
__device__ __forceinline__ int clamp_rows(const int *start, const int *end, int b, int rows, int most, int *begin,
                                          bool *bad) {
  if (!start) {
    *begin = b * most;
    return most;
  }
  const int s = start[b], e = end[b];
  *begin = min(max(s, 0), rows);
  const int stop = min(max(e, *begin), rows);
  const int n = min(stop - *begin, most);
  *bad = *bad || s != *begin || e != *begin + n;
  return n;
}

// Sequence b; a workgroup with `tell` reports offsets that were clamped.
__device__ __forceinline__ Seq sequence(const ugk_attention &a, int b, bool tell, int *word, int code) {
  Seq s;
  bool bad = false;
  s.Lq = clamp_rows(a.q_start, a.q_end, b, a.rows_q, a.max_q, &s.q0, &bad);
  s.Lk = clamp_rows(a.k_start, a.k_end, b, a.rows_k, a.max_k, &s.k0, &bad);
  if (bad && tell && threadIdx.x == 0) *word = code;
  return s;
}

__device__ __forceinline__ float wave_max(float v) {
#pragma unroll
  for (int o = 32; o; o >>= 1) {
    const float w = __shfl_xor(v, o);
    v = v > w ? v : w;
  }
  return v;
}

__device__ __forceinline__ float dot(const float *x, const float *y, int n) {
  float s = 0.0f;
  for (int d = 0; d < n; d++) s = fmaf(x[d], y[d], s);
  return s;
}

// One query row of one head by one wavefront: lanes over keys for the scores,
// over channels for the sum.
__device__ void row_forward(float *out, float *lse, const float *q, const float *k, const float *v, int n, int HS,
                            long long ldk, long long ldv, float scale) {
  const int lane = threadIdx.x & (kWave - 1);
  float m = -INFINITY;
  for (int j = lane; j < n; j += kWave) m = fmaxf(m, dot(q, k + j * ldk, HS) * scale);
  m = wave_max(m);
  float l = 0.0f, o0 = 0.0f, o1 = 0.0f;
  const int d0 = min(lane, HS - 1), d1 = min(lane + kWave, HS - 1);
  for (int j0 = 0; j0 < n; j0 += kWave) {
    const int j = j0 + lane;
    const float p = j < n ? expf(dot(q, k + j * ldk, HS) * scale - m) : 0.0f;
    l += wave_sum(p);
    for (int t = 0; t < min(kWave, n - j0); t++) {
      const float pt = __shfl(p, t);
      o0 = fmaf(pt, v[(j0 + t) * ldv + d0], o0);
      o1 = fmaf(pt, v[(j0 + t) * ldv + d1], o1);
    }
  }
  const float r = n ? l : 1.0f;
  if (lane < HS) out[lane] = o0 / r;
  if (lane + kWave < HS) out[lane + kWave] = o1 / r;
  if (lse && lane == 0) *lse = n ? m + logf(l) : -INFINITY;
}

__global__ __launch_bounds__(kBlock) void k_att_fwd_rows(float *out, float *lse, const float *q, const float *k,
                                                         const float *v, ugk_attention a, int *word) {
  const int per = (a.max_q + kBlock / kWave - 1) / (kBlock / kWave);
  const int b = blockIdx.x / (a.NH * per), h = blockIdx.x / per % a.NH, part = blockIdx.x % per;
  const Seq s = sequence(a, b, h == 0 && part == 0, word, UGK_IDS_ATTENTION_FORWARD);
  const int i = part * (kBlock / kWave) + (threadIdx.x >> 6);
  if (i >= s.Lq) return;
  const size_t row = s.q0 + i;
  const int hk = h / (a.NH / a.NKV);
  row_forward(out + row * a.ldo + h * a.HS, lse ? lse + row * a.NH + h : nullptr, q + row * a.ldq + h * a.HS,
              k + (size_t)s.k0 * a.ldk + hk * a.HS, v + (size_t)s.k0 * a.ldv + hk * a.HS, s.seen(i, a.causal), a.HS,
              a.ldk, a.ldv, a.scale);
}

__device__ __forceinline__ void put(float *p, float x, bool assign) { *p = assign ? x : *p + x; }

// dq of one query row of one head, and D.
__device__ void row_dq(float *dq, float *dsum, const float *dout, const float *q, const float *k, const float *v,
                       const float *out, float lse, int n, int HS, long long ldk, long long ldv, float scale,
                       bool assign) {
  const int lane = threadIdx.x & (kWave - 1);
  float D = 0.0f;
  if (lane < HS) D = dout[lane] * out[lane];
  if (lane + kWave < HS) D = fmaf(dout[lane + kWave], out[lane + kWave], D);
  D = wave_sum(D);
  if (lane == 0) *dsum = D;
  float a0 = 0.0f, a1 = 0.0f;
  const int d0 = min(lane, HS - 1), d1 = min(lane + kWave, HS - 1);
  for (int j0 = 0; j0 < n; j0 += kWave) {
    const int j = j0 + lane;
    float ds = 0.0f;
    if (j < n) ds = expf(dot(q, k + j * ldk, HS) * scale - lse) * (dot(dout, v + j * ldv, HS) - D) * scale;
    for (int t = 0; t < min(kWave, n - j0); t++) {
      const float x = __shfl(ds, t);
      a0 = fmaf(x, k[(j0 + t) * ldk + d0], a0);
      a1 = fmaf(x, k[(j0 + t) * ldk + d1], a1);
    }
  }
  if (lane < HS) put(dq + lane, a0, assign);
  if (lane + kWave < HS) put(dq + lane + kWave, a1, assign);
}

__global__ __launch_bounds__(kBlock) void k_att_dq_rows(float *dq, float *dsum, const float *dout, const float *q,
                                                        const float *k, const float *v, const float *out,
                                                        const float *lse, ugk_attention a, bool assign, int *word) {
  const int per = (a.max_q + kBlock / kWave - 1) / (kBlock / kWave);
  const int b = blockIdx.x / (a.NH * per), h = blockIdx.x / per % a.NH, part = blockIdx.x % per;
  const Seq s = sequence(a, b, h == 0 && part == 0, word, UGK_IDS_ATTENTION_BACKWARD);
  const int i = part * (kBlock / kWave) + (threadIdx.x >> 6);
  if (i >= s.Lq) return;
  const size_t row = s.q0 + i;
  const int hk = h / (a.NH / a.NKV);
  row_dq(dq + row * a.ldq + h * a.HS, dsum + row * a.NH + h, dout + row * a.ldo + h * a.HS, q + row * a.ldq + h * a.HS,
         k + (size_t)s.k0 * a.ldk + hk * a.HS, v + (size_t)s.k0 * a.ldv + hk * a.HS, out + row * a.ldo + h * a.HS,
         lse[row * a.NH + h], s.seen(i, a.causal), a.HS, a.ldk, a.ldv, a.scale, assign);
}

// dk and dv of key row j of key/value head hk.
__device__ void row_dkv(float *dk, float *dv, const float *dout, const float *q, const float *k, const float *v,
                        const float *lse, const float *dsum, const ugk_attention &a, const Seq &s, int j, int hk,
                        bool assign) {
  const int lane = threadIdx.x & (kWave - 1), HS = a.HS, G = a.NH / a.NKV;
  const int d0 = min(lane, HS - 1), d1 = min(lane + kWave, HS - 1);
  const size_t row = (size_t)s.k0 + j;
  const float *kj = k + row * a.ldk + hk * HS, *vj = v + row * a.ldv + hk * HS;
  float k0 = 0.0f, k1 = 0.0f, v0 = 0.0f, v1 = 0.0f;
  for (int h = hk * G; h < (hk + 1) * G; h++)
    for (int i0 = s.first(j, a.causal); i0 < s.Lq; i0 += kWave) {
      const int i = i0 + lane;
      float p = 0.0f, ds = 0.0f;
      if (i < s.Lq) {
        const size_t r = (size_t)s.q0 + i;
        p = expf(dot(q + r * a.ldq + h * HS, kj, HS) * a.scale - lse[r * a.NH + h]);
        ds = p * (dot(dout + r * a.ldo + h * HS, vj, HS) - dsum[r * a.NH + h]) * a.scale;
      }
      for (int t = 0; t < min(kWave, s.Lq - i0); t++) {
        const size_t r = (size_t)s.q0 + i0 + t;
        const float pt = __shfl(p, t), dt = __shfl(ds, t);
        const float *qr = q + r * a.ldq + h * HS, *gr = dout + r * a.ldo + h * HS;
        k0 = fmaf(dt, qr[d0], k0);
        k1 = fmaf(dt, qr[d1], k1);
        v0 = fmaf(pt, gr[d0], v0);
        v1 = fmaf(pt, gr[d1], v1);
      }
    }
  float *dkj = dk + row * a.ldk + hk * HS, *dvj = dv + row * a.ldv + hk * HS;
  if (lane < HS) {
    put(dkj + lane, k0, assign);
    put(dvj + lane, v0, assign);
  }
  if (lane + kWave < HS) {
    put(dkj + lane + kWave, k1, assign);
    put(dvj + lane + kWave, v1, assign);
  }
}

__global__ __launch_bounds__(kBlock) void k_att_dkv_rows(float *dk, float *dv, const float *dout, const float *q,
                                                         const float *k, const float *v, const float *lse,
                                                         const float *dsum, ugk_attention a, bool assign, int *word) {
  const int per = (a.max_k + kBlock / kWave - 1) / (kBlock / kWave);
  const int b = blockIdx.x / (a.NKV * per), hk = blockIdx.x / per % a.NKV, part = blockIdx.x % per;
  const Seq s = sequence(a, b, hk == 0 && part == 0, word, UGK_IDS_ATTENTION_BACKWARD);
  const int j = part * (kBlock / kWave) + (threadIdx.x >> 6);
  if (j >= s.Lk) return;
  row_dkv(dk, dv, dout, q, k, v, lse, dsum, a, s, j, hk, assign);
}

}  // namespace

size_t attention_parts_bytes(const ugk_attention &) { return 0; }
size_t attention_parts_bound() { return 0; }

int launch_attention_forward(float *out, float *lse, const float *q, const float *k, const float *v, float *,
                             const ugk_attention &a, int *word) {
  const unsigned per = grid_for((size_t)a.max_q, kBlock / kWave);
  launch(k_att_fwd_rows, dim3(per * a.NH * a.nseq), dim3(kBlock), 0, out, lse, q, k, v, a, word);
  return check_launch("attention_forward");
}

int launch_attention_backward(float *dq, float *dk, float *dv, const float *dout, const float *q, const float *k,
                              const float *v, const float *out, const float *lse, float *dsum, const ugk_attention &a,
                              bool assign, int *word) {
  if (a.max_q) {
    const unsigned per = grid_for((size_t)a.max_q, kBlock / kWave);
    launch(k_att_dq_rows, dim3(per * a.NH * a.nseq), dim3(kBlock), 0, dq, dsum, dout, q, k, v, out, lse, a, assign, word);
    if (int e = check_launch("attention_backward")) return e;
  }
  if (a.max_k) {
    const unsigned per = grid_for((size_t)a.max_k, kBlock / kWave);
    launch(k_att_dkv_rows, dim3(per * a.NKV * a.nseq), dim3(kBlock), 0, dk, dv, dout, q, k, v, lse, dsum, a, assign, word);
  }
  return check_launch("attention_backward");
}

}  // namespace ugk
