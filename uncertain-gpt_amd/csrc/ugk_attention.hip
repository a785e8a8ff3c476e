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

#include <type_traits>

#include "ugk_internal.h"
#include "ugk_split.h"

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

__device__ __forceinline__ void put(float *p, float x, bool assign) { *p = assign ? x : *p + x; }

// exp(s - m); a score of -infinity weighs nothing, whatever m is, and its key nothing in the gradients, whatever the infinite
// element that it came from would make of a product with 0.
__device__ __forceinline__ float weight(float s, float m) { return s == -INFINITY ? 0.0f : expf(s - m); }

// One query row of one head by one wavefront: lanes over keys for the scores,
// over channels for the sum. To lse, or the maximum and the sum behind it to ml (if not null) and ml[ml_step].
__device__ void row_forward(float *out, float *lse, float *ml, size_t ml_step, const float *q, const float *k,
                            const float *v, int n, int HS, long long ldk, long long ldv, float scale) {
  const int lane = threadIdx.x & (kWave - 1);
  float m = -INFINITY;
  for (int j = lane; j < n; j += kWave) m = fmaxf(m, dot(q, k + j * ldk, HS) * scale);
  m = wave_max(m);
  float l = 0.0f, o0 = 0.0f, o1 = 0.0f;
  const int d0 = min(lane, HS - 1), d1 = min(lane + kWave, HS - 1);
  for (int j0 = 0; j0 < n; j0 += kWave) {
    const int j = j0 + lane;
    const float p = j < n ? weight(dot(q, k + j * ldk, HS) * scale, m) : 0.0f;
    l += wave_sum(p);
    for (int t = 0; t < min(kWave, n - j0); t++) {
      const float pt = __shfl(p, t);
      o0 = fmaf(pt, v[(j0 + t) * ldv + d0], o0);
      o1 = fmaf(pt, v[(j0 + t) * ldv + d1], o1);
    }
  }
  const bool none = l == 0.0f;  // no key, or every score -infinity
  const float r = none ? 1.0f : l;
  if (lane < HS) out[lane] = none ? 0.0f : o0 / r;
  if (lane + kWave < HS) out[lane + kWave] = none ? 0.0f : o1 / r;
  if (lane == 0 && ml) {
    ml[0] = none ? -INFINITY : m;
    ml[ml_step] = l;
  } else if (lane == 0 && lse) {
    *lse = none ? -INFINITY : m + logf(l);
  }
}

// ---- forward, tiles on the matrix units -----------------------------------------
//
// The rows of a tile are (query row, head of the group) pairs, so that the heads
// of a group share the key and value tiles: row r of a sequence and key/value
// head is query row r / G, head r % G of the group. A wavefront holds one or two
// blocks of 32 rows; a workgroup of four goes over the keys BK at a time.
//
// S^T = K Q^T: a lane then holds one row's scores of half of the keys (the other half
// in lane ^ 32), so that the row's maximum, sum and factors are values of the
// lane, and its 16 registers of a 32 x 32 block are, rounded to halves, the
// operand of O^T += V^T P^T as they stand, with the keys in the order that
// frag_cols reads V's columns in. Nothing moves between lanes but one exchange of
// halves per block.
//
// Products are split (ugk_split.h). K and V are split while they are put into LDS, by the
// exponent of the tile's largest magnitude; that is taken over the registers that
// the tile was loaded into, one tile ahead, and goes through LDS with the barrier
// that the tile buffers need anyway: one barrier per tile. Where a tile's keys, or values, lie
// further apart than 2^kSpread, each is split by its own exponent (lift_rows), and the
// scores, or P, are taken that much lower: two passes over a lane's 16 registers more per block.
//
// A row's P go into the second product next to the largest contribution that the row
// has seen, that is P times the largest of V's row (of its tile, where the tile has one
// scale), not next to the largest P or the largest V: a large value of little weight
// leaves the others their digits, and what a row must not see moves nothing.
//
// A wavefront's rows are taken one by one instead (row_forward), where a masked key
// is not touched at all, if a tile that some of them see holds an infinity, or NaN that not
// all of the workgroup's see, or if scores leave the range of the above (2^22 in base 2).
//
// What bounds it: on gfx950 a wavefront's matrix instruction holds back the vector
// instructions of every wavefront on its SIMD (8 x (mfma, 4 fma): 20.2 ns per pair with one
// wavefront, 18.0 with two, of which the mfma alone takes 14.3), so the two
// add up. 16,384 rows of 12 heads of 64 take 1,313 us (1,268 to 1,345 from card to card): 314 TFLOP/s of products counted
// once, 942 of halves. That is 1.71 us for a SIMD's block of 32 rows and 64 keys, of which
// its 48 mfma take 0.69 (by counters 42% of the time, vector instructions 55%); the same products in single precision
// (v_mfma_f32_32x32x2_f32, 128 of 64 cycles) would take 3.7. An earlier state of this kernel
// took 1,530 us for 4 x 8,192 rows, and 1,122 without loading, splitting and storing the
// tiles. Tried without gain: K and V read ahead from LDS during the softmax (72.0
// against 71.2 us for 8 x 1,024 rows); workgroups of 8 wavefronts (1,445 against 1,528
// us for 4 x 8,192 rows, but two blocks per wavefront 1,352); a pair's tiles on one XCD
// (1,604 against 1,539); of those workgroups two per CU, with 128 registers a lane (spills:
// 562 against 470 us for 8,192 rows).
//
// A row's P are scaled to 2^kTop at the largest that they stand on, which moves
// (and the accumulators with it) only when one lies 2^7 above it: P then stays
// below 2^(kTop + 7), the halves' range.
//
// 8 x 1,024 rows of 12 heads of 64 whose values are of one size take 65 us, and 99 us where they are
// times 2^-8 to 2^8 from row to row; 13 packed sequences of 16/4 heads of 128 122 and 192. (Looking for such rows costs
// 1 to 2% where there are none; row by row the two took 25.9 and 54.5 ms.)
constexpr float kTop = 8.0f;
constexpr float kLog2e = 1.44269504088896340736f, kLn2 = 0.693147180559945309417f;

// Wavefronts of a workgroup. Four share the staging of a tile, also where a call has too few rows for all of
// them to hold any: the staging is then still four times as quick (one wavefront
// alone: 4 x 64 rows of 6 heads 12.4 against 10.7 us, 1,024 rows of 12 heads 44.6
// against 29.5, their backward 173 against 96).
constexpr int kTileWaves = 4, kTileThreads = kTileWaves * kWave, kTileRows = 32 * kTileWaves;

// One part of a split key axis: o normalised, its scores' maximum (or a number near it) m and the sum l of e^(s - m), per
// row. (m + log l in one number would lose l where m is large: a mask's lowest value.)
struct Parts {
  float *o, *m, *l;  // null: not split
  int splits, chunk; // keys per part
};

// How a kernel reads rows of HS floats, four at a time with nd of them left (0 or less
// behind the row): every slot is whole (HS is HSP), whole or behind the row (HS a multiple
// of 4), any.
enum Slots { kAny, kQuads, kWhole };

template <Slots kSlots>
__device__ __forceinline__ float4 load4(const float *p, int nd) {
  if (kSlots == kWhole || nd >= 4) return ld4(p);
  if (kSlots == kQuads) return make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  if (nd > 0) v.x = p[0];
  if (nd > 1) v.y = p[1];
  if (nd > 2) v.z = p[2];
  return v;
}
// Rows j, j + kStep, .. of [0, n): past it, zero (n > 0). tail: some of the tile's rows are.
template <int kStep, Slots kSlots>
__device__ __forceinline__ Rows4 load_rows(const float *base, long long ld, int j, int n, bool tail, int nd) {
  Rows4 t;
  if (tail) {
#pragma unroll
    for (int r = 0; r < 4; r++) {
      t.r[r] = load4<kSlots>(base + min(j + kStep * r, n - 1) * ld, nd);
      if (j + kStep * r >= n) t.r[r] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    }
  } else {
    const float *p = base + j * ld;
#pragma unroll
    for (int r = 0; r < 4; r++, p += kStep * ld) t.r[r] = load4<kSlots>(p, nd);
  }
  return t;
}
__device__ __forceinline__ float part4(const float4 &v, int d) { return d == 0 ? v.x : d == 1 ? v.y : d == 2 ? v.z : v.w; }

// The block's rows, scaled and split, to rows of halves kStep apart (h, l: the two parts' arrays, `stride` halves a row).
template <int kStep>
__device__ __forceinline__ void put_rows(const Rows4 &t, float scale, _Float16 *h, _Float16 *l, int stride) {
#pragma unroll
  for (int r = 0; r < 4; r++) {
    uint32_t h0, h1, l0, l1;
    split2(t.r[r].x, t.r[r].y, scale, h0, l0);
    split2(t.r[r].z, t.r[r].w, scale, h1, l1);
    *reinterpret_cast<v2u *>(h + kStep * r * stride) = v2u{h0, h1};
    *reinterpret_cast<v2u *>(l + kStep * r * stride) = v2u{l0, l1};
  }
}

// Eight floats from d on of a row, as operands.
template <Slots kSlots>
__device__ __forceinline__ void load8(const float *p, int d, int HS, bool live, float (&x)[8]) {
#pragma unroll
  for (int j = 0; j < 2; j++) {
    const float4 v = live ? load4<kSlots>(p + d + 4 * j, HS - d - 4 * j) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    x[4 * j] = v.x; x[4 * j + 1] = v.y; x[4 * j + 2] = v.z; x[4 * j + 3] = v.w;
  }
}

__device__ __forceinline__ void put4(float *p, float4 w, int nd, bool full, bool assign) {
  if (full || nd >= 4) {
    if (!assign) {
      const float4 u = ld4(p);
      w = make_float4(u.x + w.x, u.y + w.y, u.z + w.z, u.w + w.w);
    }
    st4(p, w);
  } else {
    if (nd > 0) put(p, w.x, assign);
    if (nd > 1) put(p + 1, w.y, assign);
    if (nd > 2) put(p + 2, w.z, assign);
  }
}
// An accumulator's column (this lane's row of the result) to memory, times f.
template <int DB, bool kFull>
__device__ __forceinline__ void put_row(float *p, const v16f (&acc)[DB], float f, int half, int HS, bool assign) {
#pragma unroll
  for (int x = 0; x < DB; x++)
#pragma unroll
    for (int y = 0; y < 4; y++) {
      const int d = 32 * x + 8 * y + 4 * half;
      put4(p + d, make_float4(acc[x][4 * y] * f, acc[x][4 * y + 1] * f, acc[x][4 * y + 2] * f, acc[x][4 * y + 3] * f),
           HS - d, kFull, assign);
    }
}

// The same times 2^e f, for any e; the factor stays far from the end of the range, where it would have few digits.
template <int DB, bool kFull>
__device__ __forceinline__ void put_scaled(float *p, v16f (&acc)[DB], int e, float f, int half, int HS, bool assign) {
  const int once = min(max(e, -80), 80), twice = min(max(e - once, -126), 127);
  if (__any(twice != 0)) {
#pragma unroll
    for (int x = 0; x < DB; x++)
#pragma unroll
      for (int y = 0; y < 16; y++) acc[x][y] *= pow2(twice);
  }
  put_row<DB, kFull>(p, acc, pow2(once) * f, half, HS, assign);
}

// The largest of a noted quantity over the workgroup's wavefronts.
template <int W>
__device__ __forceinline__ uint32_t noted(const uint32_t (&slot)[W]) {
  uint32_t m = slot[0];
#pragma unroll
  for (int w = 1; w < W; w++) m = max(m, slot[w]);
  return (uint32_t)__builtin_amdgcn_readfirstlane(m);
}

// Exponents that rows of the two tiles in LDS were lifted by (lift_rows), of two operands. All are zero but those of
// wavefronts whose byte of `by` is set, which take back what they set.
template <int kRows>
struct Lifts {
  static_assert(kTileWaves == 4, "one word of bytes");
  __attribute__((aligned(16))) int d[2][2][kRows];
  __attribute__((aligned(4))) uint8_t by[2][kTileWaves];
  __device__ __forceinline__ void clear() {
    for (int i = threadIdx.x; i < 4 * kRows; i += kTileThreads) d[i / (2 * kRows)][i / kRows % 2][i % kRows] = 0;
    if (threadIdx.x < 2 * kTileWaves) by[threadIdx.x / kTileWaves][threadIdx.x % kTileWaves] = 0;
  }
  __device__ __forceinline__ uint32_t any(int z) const { return *reinterpret_cast<const uint32_t *>(by[z]); }
  // those of rows 32 w + 8 x + 4 half .. + 3 of operand o
  __device__ __forceinline__ int4 four(int z, int o, int w, int x, int half) const {
    return *reinterpret_cast<const int4 *>(&d[z][o][32 * w + 8 * x + 4 * half]);
  }
};
__device__ __forceinline__ int part4(const int4 &v, int d) { return d == 0 ? v.x : d == 1 ? v.y : d == 2 ? v.z : v.w; }
// A block's scores (or what comes of them) times 2^d of their rows.
template <int kRows>
__device__ __forceinline__ void lower(v16f &c, const Lifts<kRows> &l, int z, int o, int w, int half, int more = 0) {
#pragma unroll
  for (int x = 0; x < 4; x++) {
    const int4 d = l.four(z, o, w, x, half);
#pragma unroll
    for (int y = 0; y < 4; y++) c[4 * x + y] = ldexpf(c[4 * x + y], part4(d, y) + more);
  }
}

// The rows of a wavefront's blocks lifted, and what they were lifted by noted for tile z, where one of them
// lies far below its tile's largest; bit z of *lifted: this was so. The tile has `rows` rows. operand(u), exponent(u)
// and first(u): a block's.
template <int DG, int kStep, int kPer, int kRows, typename Operand, typename Exponent, typename First>
__device__ __forceinline__ void lift_tile(Rows4 (&t)[kPer], Lifts<kRows> &l, int z, int rows, int lane, int wave, int *lifted,
                                          Operand operand, Exponent exponent, First first) {
  bool any = false;
#pragma unroll
  for (int u = 0; u < kPer; u++) {
    int d[4];
    any = lift_rows<DG, kStep>(t[u], exponent(u), rows - first(u), d) || any;
    if (lane % DG == 0) {
#pragma unroll
      for (int r = 0; r < 4; r++) l.d[z][operand(u)][first(u) + kStep * r] = d[r];
    }
  }
  if (lane == 0) l.by[z][wave] = any;
  *lifted = (*lifted & ~(1 << z)) | (int)any << z;
}

template <int HSP, int BK, int QB, bool kFull>
__global__ __launch_bounds__(kTileThreads, 2) void k_att_fwd(float *out, float *lse, const float *q, const float *k,
                                                             const float *v, ugk_attention a, Parts parts, unsigned pairs,
                                                             int *word) {
  constexpr int W = kTileWaves, kThreads = kTileThreads, KB = BK / 32, DC = HSP / 16, DB = HSP / 32, DG = HSP / 4, kTile = 32 * W * QB;
  constexpr int kBlocks = BK / 4 * DG, kPer = 2 * kBlocks / kThreads;  // 4 x 4 blocks: of K and of V, per thread
  static_assert(kPer >= 1 && kBlocks % kWave == 0, "whole wavefronts of K or V blocks");
  constexpr int kRs = HSP + 8, KG = BK / 4;  // halves a row: an odd multiple of 16 bytes, free of bank conflicts
  __shared__ __attribute__((aligned(16))) _Float16 lk[2][2][BK * kRs], lv[2][2][BK * kRs];
  __shared__ uint32_t slot[2][2][W];
  __shared__ Lifts<BK> lifts;
  const int tid = threadIdx.x, lane = tid & (kWave - 1), wave = __builtin_amdgcn_readfirstlane(tid >> 6), half = lane >> 5;
  const unsigned pair = blockIdx.x % pairs;
  const int tile = (int)(gridDim.x / pairs - 1 - blockIdx.x / pairs);  // the longest rows first
  const int b = pair / a.NKV, hk = pair % a.NKV, G = a.NH / a.NKV;
  const Seq s = sequence(a, b, hk == 0 && tile == 0 && blockIdx.y == 0, word, UGK_IDS_ATTENTION_FORWARD);
  const int rows = s.Lq * G, row0 = tile * kTile;
  if (row0 >= rows) return;
  const float *kb = k + (size_t)s.k0 * a.ldk + hk * a.HS, *vb = v + (size_t)s.k0 * a.ldv + hk * a.HS;
  // this part's keys, and those that the workgroup's last row sees
  const int first = parts.o ? min((int)blockIdx.y * parts.chunk, s.Lk) : 0;
  const int stop = parts.o ? min(first + parts.chunk, s.Lk) : s.Lk;
  const int n = max(first, min(stop, s.seen((min(row0 + kTile, rows) - 1) / G, a.causal)));
  const int least = s.seen(row0 / G, a.causal);  // what every row of the workgroup sees

  // this lane's rows
  bool bad = false;
  const int r0 = row0 + wave * (32 * QB) + (lane & 31);
  int lim[QB], lo = n, hi = first;  // what they see; least and most over the wavefront
  v8h qh[QB][DC], ql[QB][DC];
  int eq[QB];  // of q; the scores, to base 2, are products times 2^(eq + ek - 30) scale log2(e)
#pragma unroll
  for (int u = 0; u < QB; u++) {
    const int r = r0 + 32 * u;
    const bool live = r < rows;
    const int i = live ? r / G : 0, h = hk * G + (live ? r % G : 0);
    lim[u] = live ? min(n, s.seen(i, a.causal)) : 0;
    if (live) lo = min(lo, lim[u]);
    hi = max(hi, lim[u]);
    const float *qr = q + ((size_t)s.q0 + i) * a.ldq + h * a.HS;
    float x[DC][8];
    uint32_t m = 0;
#pragma unroll
    for (int c = 0; c < DC; c++) {
      load8<kFull ? kWhole : kAny>(qr, 16 * c + 8 * half, a.HS, live, x[c]);
#pragma unroll
      for (int j = 0; j < 8; j++) m = max(m, abs_bits(x[c][j]));
    }
    m = half_max_bits(m);
    bad = bad || m >= kInfBits;
    eq[u] = split_exp(m);
    const float f = a.scale < 0.0f ? -split_scale(eq[u]) : split_scale(eq[u]);
#pragma unroll
    for (int c = 0; c < DC; c++) split8(x[c], f, qh[u][c], ql[u][c]);
  }
#pragma unroll
  for (int o = 16; o; o >>= 1) {
    lo = min(lo, __shfl_xor(lo, o));
    hi = max(hi, __shfl_xor(hi, o));
  }
  lo = __builtin_amdgcn_readfirstlane(lo);
  hi = __builtin_amdgcn_readfirstlane(hi);

  Rows4 t[kPer];
  const auto is_v = [&](int u) { return kPer == 1 ? wave >= W / 2 : u >= kPer / 2; };
  const auto block = [&](int u) { return (tid + u * kThreads) % kBlocks; };
  const auto load = [&](int k0) {
    const bool tail = k0 + BK > n;
#pragma unroll
    for (int u = 0; u < kPer; u++) {
      const int d = block(u) % DG * 4, j = k0 + block(u) / DG;
      t[u] = load_rows<KG, kFull ? kWhole : kAny>((is_v(u) ? vb : kb) + d, is_v(u) ? a.ldv : a.ldk, j, n, tail, a.HS - d);
    }
  };
  // The tile's largest magnitudes, of K and V; where not all rows see all of it NaN counts as one.
  uint32_t small[kPer];
  const auto note = [&](int at, int k0) {
    uint32_t m[2] = {};
#pragma unroll
    for (int u = 0; u < kPer; u++) {
      const int w = is_v(u) ? 1 : 0;
      m[w] = max_abs(m[w], t[u], &small[u]);
      if (!kFull && a.HS <= block(u) % DG * 4) small[u] = kInfBits;  // behind the row
      if (k0 + BK > least) m[w] = max_abs<true>(m[w], t[u]);  // else a NaN is every row's result, as it comes
    }
    m[0] = wave_max_bits(m[0]);
    m[1] = wave_max_bits(m[1]);
    if (lane == 0) {
      slot[at][0][wave] = m[0];
      slot[at][1][wave] = m[1];
    }
  };
  int ek_next = 0, ev_next = 0;  // of the tile staged last
  int lifted = 0;                // bit z: this wavefront's rows of tile z are
  const auto stage = [&](int at, int k0) {
    const uint32_t mk = noted<W>(slot[at][0]), mv = noted<W>(slot[at][1]);
    bad = bad || (k0 < hi && (mk >= kInfBits || mv >= kInfBits));
    ek_next = split_exp(mk);
    ev_next = split_exp(mv);
    const float fk = split_scale(ek_next), fv = split_scale(ev_next);
    bool spread = false;
#pragma unroll
    for (int u = 0; u < kPer; u++) spread = spread || may_spread(small[u], is_v(u) ? mv : mk);
    if (__builtin_expect(__any(spread) || (lifted >> at & 1), 0))
      lift_tile<DG, KG>(t, lifts, at, n - k0, lane, wave, &lifted, [&](int u) { return is_v(u) ? 1 : 0; },
                        [&](int u) { return is_v(u) ? ev_next : ek_next; }, [&](int u) { return block(u) / DG; });
#pragma unroll
    for (int u = 0; u < kPer; u++) {
      const int p = block(u) / DG * kRs + block(u) % DG * 4;
      put_rows<KG>(t[u], is_v(u) ? fv : fk, (is_v(u) ? lv : lk)[at][0] + p, (is_v(u) ? lv : lk)[at][1] + p, kRs);
    }
  };

  // What the row's sums stand on, whole numbers: l on P 2^one, o on P V 2^all, V's scale included. Both are such that the
  // largest that the row has seen (of its P; of P times the largest of V's row or tile) comes to 2^kTop, or
  // up to 2^7 above. They only fall.
  v16f o[QB][DB] = {};
  float l[QB] = {}, one[QB], all[QB];
#pragma unroll
  for (int u = 0; u < QB; u++) one[u] = all[u] = 3.4028234663852886e38f;
  const int vcols = cols_at(lane, kRs);
  const auto compute = [&](int at, int k0, int ek, int ev_now) {
    const float ev = (float)ev_now;
    const uint32_t lifted_by = lifts.any(at);
    bool apart = false;
    float c2[QB], b0[QB];  // P is taken times 2^b0 to be an operand
    const auto stand = [&](int u) {
      b0[u] = apart ? one[u] : fmaxf(all[u] + ev, one[u] - 100.0f);
    };
#pragma unroll
    for (int u = 0; u < QB; u++) {
      c2[u] = fmaxf(ldexpf(fabsf(a.scale) * kLog2e, eq[u] + ek - 30), 0x1p-126f);
      bad = bad || c2[u] > 0x1p100f;
    }
#pragma unroll
    for (int w = 0; w < KB; w++) {  // 32 keys
      v16f sc[QB] = {};
#pragma unroll
      for (int c = 0; c < DC; c++) {
        const int p = (32 * w + (lane & 31)) * kRs + 16 * c + 8 * half;
        const v8h fh = frag(lk[at][0] + p), fl = frag(lk[at][1] + p);
#pragma unroll
        for (int u = 0; u < QB; u++) sc[u] = mfma3(fh, fl, qh[u][c], ql[u][c], sc[u]);
      }
      if (w == 0) {
        apart = __builtin_amdgcn_readfirstlane(lifted_by) != 0;
#pragma unroll
        for (int u = 0; u < QB; u++) stand(u);
      }
      if (apart) {
#pragma unroll
        for (int u = 0; u < QB; u++) lower(sc[u], lifts, at, 0, w, half);
      }
      if (k0 + 32 * w + 32 > lo) {  // some row does not see all of the keys
#pragma unroll
        for (int u = 0; u < QB; u++) {
          const int rel = lim[u] - k0 - 32 * w - 4 * half;
#pragma unroll
          for (int y = 0; y < 16; y++)
            if (8 * (y / 4) + y % 4 >= rel) sc[u][y] = -INFINITY;
        }
      }
      float m[QB];
      bool grown = apart;
#pragma unroll
      for (int u = 0; u < QB; u++) {
        m[u] = sc[u][0];
#pragma unroll
        for (int y = 1; y < 16; y++) m[u] = fmaxf(m[u], sc[u][y]);
        m[u] = half_max(m[u]) * c2[u];
        grown = grown || m[u] + fmaxf(one[u], b0[u]) > kTop + 7.0f;
      }
      if (__any(grown)) {
#pragma unroll
        for (int u = 0; u < QB; u++) {
          bad = bad || (fabsf(m[u]) >= 0x1p22f && m[u] != -INFINITY);
          float a = m[u];  // of P times V
          if (apart) {
            a = -INFINITY;
#pragma unroll
            for (int x = 0; x < 4; x++) {
              const int4 d = lifts.four(at, 1, w, x, half);
#pragma unroll
              for (int y = 0; y < 4; y++) a = fmaxf(a, fmaf(sc[u][4 * x + y], c2[u], (float)part4(d, y)));
            }
            a = half_max(a);
          }
          const float was = one[u], before = all[u];
          one[u] = fminf(was, kTop - ceilf(m[u]));
          all[u] = fminf(before, kTop - ceilf(a) - ev);
          stand(u);
          l[u] *= __builtin_amdgcn_exp2f(one[u] - was);
          const float f = __builtin_amdgcn_exp2f(all[u] - before);
#pragma unroll
          for (int x = 0; x < DB; x++)
#pragma unroll
            for (int y = 0; y < 16; y++) o[u][x][y] *= f;
        }
      }
#pragma unroll
      for (int u = 0; u < QB; u++) {
        float sum = 0.0f;
#pragma unroll
        for (int y = 0; y < 16; y++) {
          sc[u][y] = __builtin_amdgcn_exp2f(fmaf(sc[u][y], c2[u], b0[u]));
          sum += sc[u][y];
        }
        l[u] += ldexpf(sum, (int)(one[u] - b0[u]));
        if (apart) lower(sc[u], lifts, at, 1, w, half, (int)(all[u] + ev - one[u]));
      }
#pragma unroll
      for (int c = 0; c < 2; c++) {
        v8h ph[QB], pl[QB];
#pragma unroll
        for (int u = 0; u < QB; u++) {
          float p[8];
#pragma unroll
          for (int j = 0; j < 8; j++) p[j] = sc[u][8 * c + j];
          split8(p, ph[u], pl[u]);
        }
#pragma unroll
        for (int x = 0; x < DB; x++) {
          const int p = (32 * w + 16 * c) * kRs + 32 * x + vcols;
          const v8h fh = frag_cols(lv[at][0] + p, kRs), fl = frag_cols(lv[at][1] + p, kRs);
#pragma unroll
          for (int u = 0; u < QB; u++) o[u][x] = mfma3(fh, fl, ph[u], pl[u], o[u][x]);
        }
      }
    }
  };

  const int tiles = (n - first + BK - 1) / BK;
  lifts.clear();
  if (tiles > 0) {
    load(first);
    note(0, first);
    __syncthreads();
    stage(0, first);
    if (tiles > 1) {
      load(first + BK);
      note(1, first + BK);
    }
    __syncthreads();
    for (int at = 0; at < tiles; at++) {
      const int k0 = first + at * BK, ek = ek_next, ev_now = ev_next;
      // tile at + 1: its maxima are noted, its buffer was read two barriers ago
      if (at + 1 < tiles) stage((at + 1) & 1, k0 + BK);
      if (at + 2 < tiles) load(k0 + 2 * BK);
      if (k0 < hi) compute(at & 1, k0, ek, ev_now);
      if (at + 2 < tiles) note(at & 1, k0 + 2 * BK);
      __syncthreads();
    }
  }
  // a row all of whose scores passed the range downwards (none is NaN): what it stands on never moved
#pragma unroll
  for (int u = 0; u < QB; u++) bad = bad || (lim[u] > first && one[u] > 1e38f && l[u] == 0.0f);
  // trouble with a tile that the wavefront's rows see, or with their scores
  if (__any(bad)) {
    for (int x = 0; x < 32 * QB; x++) {
      const int rr = row0 + wave * (32 * QB) + x;
      if (rr >= rows) break;
      const int ii = rr / G, hh = hk * G + rr % G;
      const size_t g = (size_t)s.q0 + ii;
      const int upto = min(n, s.seen(ii, a.causal));
      const size_t prow = (((size_t)blockIdx.y * a.nseq + b) * a.max_q + ii) * a.NH + hh;
      row_forward(parts.o ? parts.o + prow * a.HS : out + g * a.ldo + hh * a.HS, lse ? lse + g * a.NH + hh : nullptr,
                  parts.o ? parts.m + prow : nullptr, parts.l - parts.m, q + g * a.ldq + hh * a.HS,
                  kb + first * a.ldk, vb + first * a.ldv, max(upto - first, 0), a.HS, a.ldk, a.ldv, a.scale);
    }
    return;
  }
#pragma unroll
  for (int u = 0; u < QB; u++) {
    const int r = r0 + 32 * u;
    if (r >= rows) break;
    const int i = r / G, h = hk * G + r % G;
    const size_t grow = (size_t)s.q0 + i, prow = (((size_t)blockIdx.y * a.nseq + b) * a.max_q + i) * a.NH + h;
    const float sum = half_sum(l[u]);
    const bool some = lim[u] > first;
    put_scaled<DB, kFull>(parts.o ? parts.o + prow * a.HS : out + grow * a.ldo + h * a.HS, o[u], (int)(one[u] - all[u]) - 15,
                          some ? 1.0f / sum : 0.0f, half, a.HS, true);
    if (half == 0 && (parts.o || lse)) {
      if (parts.o) {
        parts.m[prow] = some ? -one[u] * kLn2 : -INFINITY;
        parts.l[prow] = some ? sum : 0.0f;
      } else {
        lse[grow * a.NH + h] = some ? (__builtin_amdgcn_logf(sum) - one[u]) * kLn2 : -INFINITY;
      }
    }
  }
}

// ---- forward, few rows per key/value head ----------------------------------------
//
// With up to four (query row, head) pairs for a key/value head (a token's decode
// step), the work is to read K and V once: memory bounds it, and the products fit
// the vector units, whose 32-row counterpart would stay mostly empty. HSP / 4 lanes take
// a key, four floats each, so that a wavefront reads 64 / (HSP / 4) whole rows of
// K at a time, and then of V: U of them are in flight per lane before the first is
// used. A group of lanes has its own running maximum, sum and output (no exchange
// between groups until the end); its score sums go through DPP. The groups, then the
// workgroup's NW wavefronts, are joined at the end in their order, through LDS.
// Single precision throughout, and a key that a row must not see is left out by
// selects, so nothing of it reaches the row. A row whose scores all leave the range in base 2
// downwards, or one upwards, is computed by row_forward.
//
// 24 sequences of 8,192 keys, 8 key/value heads of 128: 271 us with one query head for
// each, 277 with four (1,611 MB, 5.8 to 6.0 TB/s); 64 of 2,048, 12 heads of 64, 144 us (805
// MB, 5.6 TB/s). On the 32-row tiles 24 of up to 16,384 keys took 993 us, here 413 and
// 283 with the key axis split. Five to eight rows go to the tiles (24 x 4,096 keys, eight
// query heads of 64 to each of 8: 102 us; four, here: 81), for here they would spill. The split
// (fwd_plan) costs 1% to 4% where the lengths are equal.
template <int kLanes>
__device__ __forceinline__ float lanes_sum(float v) {
  v += dpp_lane<kDppQuadSwap1>(v);
  v += dpp_lane<kDppQuadSwap2>(v);
  v += dpp_lane<kDppHalfMirror>(v);
  v += dpp_lane<kDppMirror>(v);
  if (kLanes == 32) v += __shfl_xor(v, 16);
  return v;
}

// Keys in flight per group of lanes, and wavefronts of a large workgroup: as many as the registers hold.
constexpr int few_loads(int R) { return R == 1 ? 8 : 4; }
constexpr int few_waves(int R) { return R <= 2 ? 16 : 8; }

template <int HSP, int R, int NW, bool kFull>
__global__ __launch_bounds__(NW * kWave) void k_att_few(float *out, float *lse, const float *q, const float *k,
                                                        const float *v, ugk_attention a, Parts parts, unsigned pairs,
                                                        int *word) {
  constexpr int kLanes = HSP / 4, kKeys = kWave / kLanes, U = few_loads(R), kStep = kKeys * U;
  __shared__ float4 lo[NW][R][kLanes];
  __shared__ float lm[NW][R], ll[NW][R];
  const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x >> 6;
  const int group = lane / kLanes, d = lane % kLanes * 4, nd = a.HS - d;
  const unsigned pair = blockIdx.x % pairs;
  const int part = blockIdx.x / pairs;
  const int b = pair / a.NKV, hk = pair % a.NKV, G = a.NH / a.NKV;
  const Seq s = sequence(a, b, hk == 0 && part == 0, word, UGK_IDS_ATTENTION_FORWARD);
  const int rows = s.Lq * G;
  if (rows <= 0) return;
  const float *kb = k + (size_t)s.k0 * a.ldk + hk * a.HS + (nd > 0 ? d : 0);
  const float *vb = v + (size_t)s.k0 * a.ldv + hk * a.HS + (nd > 0 ? d : 0);
  const int first = parts.o ? min(part * parts.chunk, s.Lk) : 0;
  const int stop = parts.o ? min(first + parts.chunk, s.Lk) : s.Lk;
  float4 qv[R], o[R];
  float m[R], l[R];
  int lim[R], least = stop, n = first;
#pragma unroll
  for (int r = 0; r < R; r++) {
    const int rr = min(r, rows - 1), i = rr / G, h = hk * G + rr % G;
    qv[r] = load4<kFull ? kWhole : kAny>(q + ((size_t)s.q0 + i) * a.ldq + h * a.HS + (nd > 0 ? d : 0), nd);
    const float f = a.scale * kLog2e;
    qv[r] = make_float4(qv[r].x * f, qv[r].y * f, qv[r].z * f, qv[r].w * f);
    lim[r] = r < rows ? min(stop, s.seen(i, a.causal)) : first;
    if (r < rows) least = min(least, lim[r]);
    n = max(n, lim[r]);
    o[r] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    m[r] = -INFINITY;
    l[r] = 0.0f;
  }
  for (int j0 = first + wave * kStep; j0 < n; j0 += NW * kStep) {
    float4 kv[U], vv[U];
#pragma unroll
    for (int u = 0; u < U; u++) kv[u] = load4<kFull ? kWhole : kAny>(kb + min(j0 + u * kKeys + group, n - 1) * a.ldk, nd);
#pragma unroll
    for (int u = 0; u < U; u++) vv[u] = load4<kFull ? kWhole : kAny>(vb + min(j0 + u * kKeys + group, n - 1) * a.ldv, nd);
    const auto take = [&](auto masked) {  // masked: not every row sees all of these keys
      constexpr bool kMasked = decltype(masked)::value;
#pragma unroll
      for (int r = 0; r < R; r++) {
        if (R > 1) __builtin_amdgcn_sched_barrier(0);  // row by row: the registers hold one row's scores
        float p[U], top = m[r];
#pragma unroll
        for (int u = 0; u < U; u++) {
          p[u] = lanes_sum<kLanes>(fmaf(qv[r].w, kv[u].w, fmaf(qv[r].z, kv[u].z, fmaf(qv[r].y, kv[u].y, qv[r].x * kv[u].x))));
          if (kMasked && j0 + u * kKeys + group >= lim[r]) p[u] = -INFINITY;
          top = fmaxf(top, p[u]);
        }
        const float base = top == -INFINITY ? 0.0f : top, keep = __builtin_amdgcn_exp2f(m[r] - base);
        float sum = 0.0f;
#pragma unroll
        for (int u = 0; u < U; u++) {
          p[u] = __builtin_amdgcn_exp2f(p[u] - base);
          sum += p[u];
        }
        m[r] = top;
        l[r] = fmaf(l[r], keep, sum);
        o[r] = make_float4(o[r].x * keep, o[r].y * keep, o[r].z * keep, o[r].w * keep);
#pragma unroll
        for (int u = 0; u < U; u++) {
          float4 w = vv[u];
          if (kMasked && j0 + u * kKeys + group >= lim[r]) w = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
          o[r].x = fmaf(p[u], w.x, o[r].x);
          o[r].y = fmaf(p[u], w.y, o[r].y);
          o[r].z = fmaf(p[u], w.z, o[r].z);
          o[r].w = fmaf(p[u], w.w, o[r].w);
        }
      }
    };
    if (j0 + kStep > least) take(std::true_type{});
    else take(std::false_type{});
  }
  // the wavefront's groups
#pragma unroll
  for (int r = 0; r < R; r++) {
#pragma unroll
    for (int x = kLanes; x < kWave; x *= 2) {
      __builtin_amdgcn_sched_barrier(0);
      const float m2 = __shfl_xor(m[r], x), l2 = __shfl_xor(l[r], x);
      const float4 o2 = make_float4(__shfl_xor(o[r].x, x), __shfl_xor(o[r].y, x), __shfl_xor(o[r].z, x), __shfl_xor(o[r].w, x));
      const float top = fmaxf(m[r], m2), base = top == -INFINITY ? 0.0f : top;
      const float f = __builtin_amdgcn_exp2f(m[r] - base), g = __builtin_amdgcn_exp2f(m2 - base);
      l[r] = l[r] * f + l2 * g;
      o[r] = make_float4(o[r].x * f + o2.x * g, o[r].y * f + o2.y * g, o[r].z * f + o2.z * g, o[r].w * f + o2.w * g);
      m[r] = top;
    }
    if (group == 0) lo[wave][r][lane] = o[r];
    if (lane == 0) {
      lm[wave][r] = m[r];
      ll[wave][r] = l[r];
    }
  }
  __syncthreads();
  // the wavefronts, kLanes threads per row
  static_assert(R * kLanes <= NW * kWave, "a thread has one row at most");
  bool lost = false;  // scores beyond the range in base 2
  const int r = threadIdx.x / kLanes, at = threadIdx.x % kLanes;
  const int i = r / G, h = hk * G + r % G;
  const size_t prow = ((size_t)part * a.nseq + b) * a.max_q + i, grow = (size_t)s.q0 + i;
  if (r < min(R, rows)) {
    float top = -INFINITY;
#pragma unroll
    for (int w = 0; w < NW; w++) top = fmaxf(top, lm[w][r]);
    const float base = top == -INFINITY ? 0.0f : top;
    float4 t = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    float sum = 0.0f;
#pragma unroll
    for (int w = 0; w < NW; w++) {
      const float f = __builtin_amdgcn_exp2f(lm[w][r] - base);
      const float4 y = lo[w][r][at];
      sum = fmaf(ll[w][r], f, sum);
      t = make_float4(fmaf(y.x, f, t.x), fmaf(y.y, f, t.y), fmaf(y.z, f, t.z), fmaf(y.w, f, t.w));
    }
    lost = (sum == 0.0f || top == INFINITY) && min(stop, s.seen(i, a.causal)) > first;
    const bool any = sum != 0.0f;  // else no key
    const float f = any ? 1.0f / sum : 0.0f;
    t = any ? make_float4(t.x * f, t.y * f, t.z * f, t.w * f) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    float *po = parts.o ? parts.o + prow * a.NH * a.HS + (size_t)h * a.HS : out + grow * a.ldo + h * a.HS;
    if (!lost) {
      put4(po + 4 * at, t, a.HS - 4 * at, kFull, true);
      if (at == 0 && parts.o) {
        parts.m[prow * a.NH + h] = top * kLn2;
        parts.l[prow * a.NH + h] = sum;
      } else if (at == 0 && lse) {
        lse[grow * a.NH + h] = any ? (top + __builtin_amdgcn_logf(sum)) * kLn2 : -INFINITY;
      }
    }
  }
  for (uint64_t rest = __ballot(lost && at == 0); rest; rest &= rest - 1) {
    const int x = __builtin_ctzll(rest), rr = __shfl(r, x), ii = rr / G, hh = hk * G + rr % G;
    const size_t p = (((size_t)part * a.nseq + b) * a.max_q + ii) * a.NH + hh, g = (size_t)s.q0 + ii;
    row_forward(parts.o ? parts.o + p * a.HS : out + g * a.ldo + hh * a.HS, lse ? lse + g * a.NH + hh : nullptr,
                parts.o ? parts.m + p : nullptr, parts.l - parts.m, q + g * a.ldq + hh * a.HS,
                k + ((size_t)s.k0 + first) * a.ldk + hk * a.HS, v + ((size_t)s.k0 + first) * a.ldv + hk * a.HS,
                min(stop, s.seen(ii, a.causal)) - first, a.HS, a.ldk, a.ldv, a.scale);
  }
}

// The parts of a split key axis joined, one wavefront per row and head: out =
// sum_x w_x o_x / sum_x w_x with w_x = l_x e^(m_x - max m), in the parts' order.
__global__ __launch_bounds__(kBlock) void k_att_join(float *out, float *lse, Parts parts, ugk_attention a) {
  const size_t at = (size_t)blockIdx.x * (kBlock / kWave) + (threadIdx.x >> 6), per = (size_t)a.nseq * a.max_q * a.NH;
  if (at >= per) return;
  const int lane = threadIdx.x & (kWave - 1), h = at % a.NH, i = at / a.NH % a.max_q, b = at / a.NH / a.max_q;
  const Seq s = sequence(a, b, false, nullptr, 0);
  if (i >= s.Lq) return;
  float m = -INFINITY;
  for (int x = lane; x < parts.splits; x += kWave) m = fmaxf(m, parts.m[x * per + at]);
  m = wave_max(m);
  float o0 = 0.0f, o1 = 0.0f, l = 0.0f;
  const int d0 = min(lane, a.HS - 1), d1 = min(lane + kWave, a.HS - 1);
  for (int x0 = 0; x0 < parts.splits; x0 += kWave) {
    const int x = x0 + lane, n = min(kWave, parts.splits - x0);
    const float lx = x < parts.splits ? parts.l[x * per + at] : 0.0f;
    const float w = lx == 0.0f ? 0.0f : lx * expf(parts.m[x * per + at] - m);  // 0: a part without a key of this row, its o is 0
    for (int t = 0; t < n; t++) {
      const float wt = __shfl(w, t), *o = parts.o + ((x0 + t) * per + at) * a.HS;
      l += wt;
      o0 = fmaf(wt, o[d0], o0);
      o1 = fmaf(wt, o[d1], o1);
    }
  }
  const bool none = l == 0.0f;
  const float r = none ? 1.0f : l;
  const size_t g = (size_t)s.q0 + i;
  float *po = out + g * a.ldo + h * a.HS;
  if (lane < a.HS) po[lane] = o0 / r;
  if (lane + kWave < a.HS) po[lane + kWave] = o1 / r;
  if (lse && lane == 0) lse[g * a.NH + h] = none ? -INFINITY : m + logf(l);
}


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
    bool gone = false;
    if (j < n) {
      const float z = dot(q, k + j * ldk, HS) * scale;
      gone = z == -INFINITY;
      ds = weight(z, lse) * (dot(dout, v + j * ldv, HS) - D) * scale;
    }
    const uint64_t skip = __ballot(gone);
    for (int t = 0; t < min(kWave, n - j0); t++) {
      if (skip >> t & 1) continue;
      const float x = __shfl(ds, t);
      a0 = fmaf(x, k[(j0 + t) * ldk + d0], a0);
      a1 = fmaf(x, k[(j0 + t) * ldk + d1], a1);
    }
  }
  if (lane < HS) put(dq + lane, a0, assign);
  if (lane + kWave < HS) put(dq + lane + kWave, a1, assign);
}

// dk and dv of key row j of key/value head hk from the (query row, head) pairs
// [ra, rb), to rows dkj and dvj.
__device__ void row_dkv(float *dkj, float *dvj, const float *dout, const float *q, const float *k, const float *v,
                        const float *lse, const float *dsum, const ugk_attention &a, const Seq &s, int j, int hk, int ra,
                        int rb, bool assign) {
  const int lane = threadIdx.x & (kWave - 1), HS = a.HS, G = a.NH / a.NKV;
  const int d0 = min(lane, HS - 1), d1 = min(lane + kWave, HS - 1);
  const size_t row = (size_t)s.k0 + j;
  const float *kj = k + row * a.ldk + hk * HS, *vj = v + row * a.ldv + hk * HS;
  float k0 = 0.0f, k1 = 0.0f, v0 = 0.0f, v1 = 0.0f;
  for (int g = 0; g < G; g++) {
    const int h = hk * G + g, end = min(s.Lq, (rb - g + G - 1) / G);
    for (int i0 = max(s.first(j, a.causal), (max(ra - g, 0) + G - 1) / G); i0 < end; i0 += kWave) {
      const int i = i0 + lane;
      float p = 0.0f, ds = 0.0f;
      bool gone = false;
      if (i < end) {
        const size_t r = (size_t)s.q0 + i;
        const float z = dot(q + r * a.ldq + h * HS, kj, HS) * a.scale;
        gone = z == -INFINITY;
        p = weight(z, lse[r * a.NH + h]);
        ds = p * (dot(dout + r * a.ldo + h * HS, vj, HS) - dsum[r * a.NH + h]) * a.scale;
      }
      const uint64_t skip = __ballot(gone);
      for (int t = 0; t < min(kWave, end - i0); t++) {
        if (skip >> t & 1) continue;
        const size_t r = (size_t)s.q0 + i0 + t;
        const float pt = __shfl(p, t), dt = __shfl(ds, t);
        const float *qr = q + r * a.ldq + h * HS, *gr = dout + r * a.ldo + h * HS;
        k0 = fmaf(dt, qr[d0], k0);
        k1 = fmaf(dt, qr[d1], k1);
        v0 = fmaf(pt, gr[d0], v0);
        v1 = fmaf(pt, gr[d1], v1);
      }
    }
  }
  if (lane < HS) {
    put(dkj + lane, k0, assign);
    put(dvj + lane, v0, assign);
  }
  if (lane + kWave < HS) {
    put(dkj + lane + kWave, k1, assign);
    put(dvj + lane + kWave, v1, assign);
  }
}

// ---- backward, tiles on the matrix units ----------------------------------------
//
// Two passes, each of which computes the scores again: dq over the rows as the
// forward holds them, then dk and dv over the keys, so that nothing is added by
// two workgroups and the results do not depend on their order (one pass with
// atomics would save the second S and dP, 4 of 14 HS operations per pair).
// P = exp(S - lse) needs no running maximum. A lane holds one row (dq) or one key (dk, dv)
// as it holds a row in the forward, the other side goes through LDS in tiles, and
// what its accumulators stand on follows what it has seen alone: the largest P of a
// key times the largest of dout's row, the largest dS times that of q's or k's. Rows that lie far
// below their tile's largest are lifted, and others taken one by one, as in the forward: 8 x 1,024 rows of 12 heads
// with dout's rows times 2^-8 to 2^8 take 253 us against 210, 4 x 2,048 of 16/4 heads of 128 1,460 against 1,150
// (row by row 26 and 123 ms).
//
// The same sum of matrix and vector instructions bounds them: of 858 (dk, dv) and 633 us
// (dq) at 4 x 4,096 rows of 12 heads, 612 and 465 were left without loading,
// splitting and storing the tiles. 8 x 1,024 rows of 12 heads: 137 and 103 us, 222
// as calls among others (145 TFLOP/s of 10 HS operations per pair). Workgroups of
// one wavefront were slower at every size tried.

// acc += A^T B for a 32-row block of B held in an accumulator's registers (C, scaled
// to halves by f): A's 32 rows in LDS, `cols` the lane's place in them (cols_at).
template <int DB>
__device__ __forceinline__ void mac_block(v16f (&acc)[DB], const v16f &c, float f, const _Float16 *ah, const _Float16 *al,
                                          int stride, int cols) {
#pragma unroll
  for (int y = 0; y < 2; y++) {
    float p[8];
#pragma unroll
    for (int j = 0; j < 8; j++) p[j] = c[8 * y + j];
    v8h bh, bl;
    split8(p, f, bh, bl);
#pragma unroll
    for (int x = 0; x < DB; x++) {
      const int at = 16 * y * stride + 32 * x + cols;
      acc[x] = mfma3(frag_cols(ah + at, stride), frag_cols(al + at, stride), bh, bl, acc[x]);
    }
  }
}
// A 32 x 32 block of products of rows in LDS with the operands in registers.
template <int DC>
__device__ __forceinline__ v16f dot_block(const _Float16 *ah, const _Float16 *al, int stride, const v8h (&bh)[DC],
                                          const v8h (&bl)[DC], int lane) {
  v16f c = {};
#pragma unroll
  for (int x = 0; x < DC; x++) {
    const int at = (lane & 31) * stride + 16 * x + 8 * (lane >> 5);
    c = mfma3(frag(ah + at), frag(al + at), bh[x], bl[x], c);
  }
  return c;
}

// Before a block of dS or P (16 per lane, the row's or key's other half in lane ^ 32) is
// accumulated with operands of exponent e: the accumulators stand on 2^ea, at least on the
// largest of the block times 2^e, so that dS 2^(15 + e - ea) is below 2^15. It moves
// in steps of 2^2 or more, for it costs a pass over the accumulators. (The block's own
// largest, not 1 for P or a bound from dout and v for dS: P is small where there are many keys or
// another has the weight, and the halves would lose its digits.) Returns whether the range does not do.
constexpr int kNoScale = -250;
template <int DB>
__device__ __forceinline__ bool raise(int &ea, v16f (&acc)[DB], const v16f &ds, int e) {
  float m = 0.0f;
#pragma unroll
  for (int y = 0; y < 16; y += 2) m = fmaxf(fmaxf(m, fabsf(ds[y])), fabsf(ds[y + 1]));
  m = half_max(m);
  const int need = max((int)(__float_as_uint(m) >> 23) - 126, -112), was = ea;
  if (m > 0.0f && need + e > ea) ea = need + e + 2;
  if (__any(ea != was)) {
    const float f = pow2(max(was - ea, -126));
#pragma unroll
    for (int x = 0; x < DB; x++)
#pragma unroll
      for (int y = 0; y < 16; y++) acc[x][y] *= f;
  }
  return m > 0x1p120f;
}

// A lane's row (HS floats at p) as operands; *e: its exponent. Returns the bits of its largest magnitude.
template <int DC, Slots kSlots>
__device__ __forceinline__ uint32_t load_operand(const float *p, int HS, bool live, int half, v8h (&h)[DC], v8h (&l)[DC],
                                                 int *e) {
  float x[DC][8];
  uint32_t m = 0;
#pragma unroll
  for (int c = 0; c < DC; c++) {
    load8<kSlots>(p, 16 * c + 8 * half, HS, live, x[c]);
#pragma unroll
    for (int j = 0; j < 8; j++) m = max(m, abs_bits(x[c][j]));
  }
  m = half_max_bits(m);
  *e = split_exp(m);
#pragma unroll
  for (int c = 0; c < DC; c++) split8(x[c], split_scale(*e), h[c], l[c]);
  return m;
}

template <int HSP, int BK, Slots kSlots>
__global__ __launch_bounds__(kTileThreads, HSP > 64 ? 1 : 2) void k_att_dq(
    float *dq, float *dsum, const float *dout, const float *q, const float *k, const float *v, const float *out,
    const float *lse, ugk_attention a, unsigned pairs, bool assign, int *word) {
  constexpr int W = kTileWaves, kThreads = kTileThreads, DC = HSP / 16, DB = HSP / 32, DG = HSP / 4;
  constexpr int kBlocks = BK / 4 * DG, kPer = 2 * kBlocks / kThreads;
  static_assert(kPer >= 1 && kBlocks % kWave == 0, "whole wavefronts of K or V blocks");
  constexpr int kRs = HSP + 8, KG = BK / 4;
  __shared__ __attribute__((aligned(16))) _Float16 lk[2][2][BK * kRs], lv[2][2][BK * kRs];
  __shared__ uint32_t slot[2][2][W];
  __shared__ Lifts<BK> lifts;
  const int tid = threadIdx.x, lane = tid & (kWave - 1), wave = tid >> 6, half = lane >> 5;
  const unsigned pair = blockIdx.x % pairs;
  const int tile = (int)(gridDim.x / pairs - 1 - blockIdx.x / pairs);
  const int b = pair / a.NKV, hk = pair % a.NKV, G = a.NH / a.NKV;
  const Seq s = sequence(a, b, hk == 0 && tile == 0, word, UGK_IDS_ATTENTION_BACKWARD);
  const int rows = s.Lq * G, row0 = tile * (32 * W);
  if (row0 >= rows) return;
  const float *kb = k + (size_t)s.k0 * a.ldk + hk * a.HS, *vb = v + (size_t)s.k0 * a.ldv + hk * a.HS;
  const int n = s.seen((min(row0 + 32 * W, rows) - 1) / G, a.causal), least = s.seen(row0 / G, a.causal);

  const int r = row0 + wave * 32 + (lane & 31);
  const bool live = r < rows;
  const int i = live ? r / G : 0, h = hk * G + (live ? r % G : 0);
  const int lim = live ? s.seen(i, a.causal) : 0;
  int lo = live ? lim : n, hi = lim;
#pragma unroll
  for (int o = 16; o; o >>= 1) {
    lo = min(lo, __shfl_xor(lo, o));
    hi = max(hi, __shfl_xor(hi, o));
  }
  lo = __builtin_amdgcn_readfirstlane(lo);
  hi = __builtin_amdgcn_readfirstlane(hi);
  const size_t grow = (size_t)s.q0 + i;
  v8h qh[DC], ql[DC], gh[DC], gl[DC];
  int eq, eg;
  const uint32_t qbits = load_operand<DC, kSlots>(q + grow * a.ldq + h * a.HS, a.HS, live, half, qh, ql, &eq);
  const float *gr = dout + grow * a.ldo + h * a.HS;
  const uint32_t gbits = load_operand<DC, kSlots>(gr, a.HS, live, half, gh, gl, &eg);
  float D = 0.0f;
#pragma unroll
  for (int c = 0; c < DC; c++) {
    float x[8], y[8];
    load8<kSlots>(gr, 16 * c + 8 * half, a.HS, live, x);
    load8<kSlots>(out + grow * a.ldo + h * a.HS, 16 * c + 8 * half, a.HS, live, y);
#pragma unroll
    for (int j = 0; j < 8; j++) D = fmaf(x[j], y[j], D);
  }
  D = half_sum(D);
  if (live && half == 0) dsum[grow * a.NH + h] = D;
  const float L2 = live ? lse[grow * a.NH + h] * kLog2e : 0.0f;
  const float cg = split_unscale(eg);
  bool bad = lim > 0 && (!(fabsf(L2) < 0x1p22f) || qbits >= kInfBits || gbits >= kInfBits);

  Rows4 t[kPer];
  const auto is_v = [&](int u) { return kPer == 1 ? wave >= W / 2 : u >= kPer / 2; };
  const auto block = [&](int u) { return (tid + u * kThreads) % kBlocks; };
  const auto load = [&](int at) {
    const int k0 = at * BK;
    const bool tail = k0 + BK > n;
#pragma unroll
    for (int u = 0; u < kPer; u++) {
      const int d = block(u) % DG * 4, j = k0 + block(u) / DG;
      const bool w = is_v(u);
      t[u] = load_rows<KG, kSlots>((w ? vb : kb) + d, w ? a.ldv : a.ldk, j, n, tail, a.HS - d);
    }
  };
  uint32_t small[kPer];
  const auto note = [&](int at) {
    uint32_t m[2] = {};
#pragma unroll
    for (int u = 0; u < kPer; u++) {
      const int w = is_v(u) ? 1 : 0;
      m[w] = max_abs(m[w], t[u], &small[u]);
      if (kSlots != kWhole && a.HS <= block(u) % DG * 4) small[u] = kInfBits;  // behind the row
      if ((at + 1) * BK > least) m[w] = max_abs<true>(m[w], t[u]);
    }
    m[0] = wave_max_bits(m[0]);
    m[1] = wave_max_bits(m[1]);
    if (lane == 0) {
      slot[at & 1][0][wave] = m[0];
      slot[at & 1][1][wave] = m[1];
    }
  };
  int ek = 0, ev = 0;  // of the tile staged last
  int lifted = 0;
  const auto stage = [&](int at) {
    const int z = at & 1;
    const uint32_t mk = noted<W>(slot[z][0]), mv = noted<W>(slot[z][1]);
    bad = bad || (at * BK < hi && (mk >= kInfBits || mv >= kInfBits));
    ek = split_exp(mk);
    ev = split_exp(mv);
    bool spread = false;
#pragma unroll
    for (int u = 0; u < kPer; u++) spread = spread || may_spread(small[u], is_v(u) ? mv : mk);
    if (__any(spread) || (lifted >> z & 1))
      lift_tile<DG, KG>(t, lifts, z, n - at * BK, lane, wave, &lifted, [&](int u) { return is_v(u) ? 1 : 0; },
                        [&](int u) { return is_v(u) ? ev : ek; }, [&](int u) { return block(u) / DG; });
    const float fk = split_scale(ek), fv = split_scale(ev);
#pragma unroll
    for (int u = 0; u < kPer; u++) {
      const int p = block(u) / DG * kRs + block(u) % DG * 4;
      const bool w = is_v(u);
      put_rows<KG>(t[u], w ? fv : fk, (w ? lv : lk)[z][0] + p, (w ? lv : lk)[z][1] + p, kRs);
    }
  };

  v16f acc[DB] = {};
  int ea = kNoScale;  // the exponent that the accumulators stand on
  const int cols = cols_at(lane, kRs);
  const auto compute = [&](int at, int ek_now, int ev_now) {
    const int z = at & 1, k0 = at * BK;
    const float c2 = ldexpf(a.scale * kLog2e, eq + ek_now - 30), cd = cg * split_unscale(ev_now);
    const uint32_t lifted_by = lifts.any(z);
    bool apart = false;
    bad = bad || (lim > k0 && (fabsf(c2) > 0x1p100f || cd > 0x1p100f));
#pragma unroll
    for (int w = 0; w < BK / 32; w++) {  // 32 keys
      const int o = 32 * w * kRs;
      v16f p = dot_block<DC>(lk[z][0] + o, lk[z][1] + o, kRs, qh, ql, lane);
      v16f dp = dot_block<DC>(lv[z][0] + o, lv[z][1] + o, kRs, gh, gl, lane);
      if (w == 0) apart = __builtin_amdgcn_readfirstlane(lifted_by) != 0;
      if (apart) {
        lower(p, lifts, z, 0, w, half);
        lower(dp, lifts, z, 1, w, half);
      }
#pragma unroll
      for (int y = 0; y < 16; y++) {
        const float x = __builtin_amdgcn_exp2f(fmaf(p[y], c2, -L2));
        p[y] = x * fmaf(dp[y], cd, -D);
      }
      if (k0 + 32 * w + 32 > lo) {
        const int rel = lim - k0 - 32 * w - 4 * half;
#pragma unroll
        for (int y = 0; y < 16; y++)
          if (8 * (y / 4) + y % 4 >= rel) p[y] = 0.0f;
      }
      if (apart) lower(p, lifts, z, 0, w, half);
      bad = raise(ea, acc, p, ek_now) || bad;
      mac_block<DB>(acc, p, pow2(max(min(15 + ek_now - ea, 127), -126)), lk[z][0] + o, lk[z][1] + o, kRs, cols);
    }
  };

  const int tiles = (n + BK - 1) / BK;
  lifts.clear();
  if (tiles > 0) {
    load(0);
    note(0);
    __syncthreads();
    stage(0);
    if (tiles > 1) {
      load(1);
      note(1);
    }
    __syncthreads();
    for (int at = 0; at < tiles; at++) {
      const int ek_now = ek, ev_now = ev;
      if (at + 1 < tiles) stage(at + 1);
      if (at + 2 < tiles) load(at + 2);
      if (at * BK < hi) compute(at, ek_now, ev_now);
      if (at + 2 < tiles) note(at + 2);
      __syncthreads();
    }
  }
  if (__any(bad)) {
    for (int x = 0; x < 32; x++) {
      const int rr = row0 + wave * 32 + x;
      if (rr >= rows) break;
      const int ii = rr / G, hh = hk * G + rr % G;
      const size_t g = (size_t)s.q0 + ii;
      row_dq(dq + g * a.ldq + hh * a.HS, dsum + g * a.NH + hh, dout + g * a.ldo + hh * a.HS, q + g * a.ldq + hh * a.HS, kb, vb,
             out + g * a.ldo + hh * a.HS, lse[g * a.NH + hh], s.seen(ii, a.causal), a.HS, a.ldk, a.ldv, a.scale, assign);
    }
    return;
  }
  if (live) put_scaled<DB, kSlots == kWhole>(dq + grow * a.ldq + h * a.HS, acc, ea - 30, a.scale, half, a.HS, assign);
}

// Rows r = (query row r / G, head r % G of the group) of q or dout in tiles of kTile,
// from `base`: rows `ld` floats apart, heads HS. A thread's four rows of a tile stand
// at the same places of every tile where G divides the tile (1, 2, 4, .. 32 heads), else
// each is divided out.
template <int kTile, int kStep>
struct GroupRows {
  const float *base;
  long long ld;
  int HS, G;
  __device__ __forceinline__ const float *at(int r) const {
    const int i = r / G;
    return base + i * ld + (r - i * G) * HS;
  }
  template <Slots kSlots>
  __device__ __forceinline__ Rows4 load(int r0, const long long (&off)[4], int x, int d, int n, int nd) const {
    Rows4 t;
    if (kTile % G == 0 && r0 + kTile <= n) {
      const float *p = base + r0 / G * ld + d;
#pragma unroll
      for (int y = 0; y < 4; y++) t.r[y] = load4<kSlots>(p + off[y], nd);
    } else {
#pragma unroll
      for (int y = 0; y < 4; y++) {
        const int r = r0 + x + kStep * y;
        t.r[y] = load4<kSlots>(at(min(r, n - 1)) + d, nd);
        if (r >= n) t.r[y] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
      }
    }
    return t;
  }
};

constexpr int kMaxSplits = 8;
// The rows' range split in parts, for few keys with many rows (grouped heads): each part's dk and dv, at [part][key row].
struct Halves {
  float *dk, *dv;  // null: not split
  int splits;
};

template <int HSP, Slots kSlots>
__global__ __launch_bounds__(kTileThreads, HSP > 64 ? 1 : 2) void k_att_dkv(
    float *dk, float *dv, const float *dout, const float *q, const float *k, const float *v, const float *lse,
    const float *dsum, ugk_attention a, Halves parts, unsigned pairs, bool assign, int *word) {
  constexpr int W = kTileWaves, kThreads = kTileThreads, BQ = 32, DC = HSP / 16, DB = HSP / 32, DG = HSP / 4;
  constexpr int kBlocks = BQ / 4 * DG, kPer = 2 * kBlocks / kThreads;
  static_assert(kPer >= 1 && kBlocks % kWave == 0, "whole wavefronts of Q or dout blocks");
  constexpr int kRs = HSP + 8, KG = BQ / 4;
  __shared__ __attribute__((aligned(16))) _Float16 lq[2][2][BQ * kRs], lg[2][2][BQ * kRs];
  __shared__ __attribute__((aligned(16))) float lL[2][BQ], lD[2][BQ];
  __shared__ uint32_t slot[2][3][W];
  __shared__ Lifts<BQ> lifts;
  const int tid = threadIdx.x, lane = tid & (kWave - 1), wave = tid >> 6, half = lane >> 5;
  const unsigned pair = blockIdx.x % pairs;
  // The keys that the most rows see first, their parts one after the other (with the parts
  // as the slower index the last part's long ones came last: packed 4,095 rows of 16/4
  // heads 205 us against 187, 4 x 2,048 600 against 548).
  const int splits = parts.dk ? parts.splits : 1, unit = (int)(blockIdx.x / pairs);
  const int tile = unit / splits, part_no = unit % splits;
  const int b = pair / a.NKV, hk = pair % a.NKV, G = a.NH / a.NKV;
  const Seq s = sequence(a, b, hk == 0 && unit == 0, word, UGK_IDS_ATTENTION_BACKWARD);
  const int key0 = tile * (32 * W);
  if (key0 >= s.Lk) return;
  // rows before `from` see none of the workgroup's keys, rows from `all` on all of them
  int from = min(s.first(key0, a.causal), s.Lq) * G / BQ * BQ, rows = s.Lq * G;
  if (parts.dk) {  // this part's rows
    const int per = ((rows - from + parts.splits - 1) / parts.splits + BQ - 1) / BQ * BQ;
    from = min(from + part_no * per, rows);
    rows = min(from + per, rows);
  }
  const int all = min(s.first(min(key0 + 32 * W, s.Lk) - 1, a.causal), s.Lq) * G;

  const int j = key0 + wave * 32 + (lane & 31);
  const bool live = j < s.Lk;
  const int lim = live ? min(s.first(j, a.causal), s.Lq) * G : rows;  // the first row that sees the key
  int lo = lim, hi = live ? lim : 0;
#pragma unroll
  for (int o = 16; o; o >>= 1) {
    lo = min(lo, __shfl_xor(lo, o));
    hi = max(hi, __shfl_xor(hi, o));
  }
  lo = __builtin_amdgcn_readfirstlane(lo);
  hi = __builtin_amdgcn_readfirstlane(hi);
  const size_t grow = (size_t)s.k0 + (live ? j : 0);
  v8h kh[DC], kl[DC], vh[DC], vl[DC];
  int ek, ev;
  const uint32_t kbits = load_operand<DC, kSlots>(k + grow * a.ldk + hk * a.HS, a.HS, live, half, kh, kl, &ek);
  const uint32_t vbits = load_operand<DC, kSlots>(v + grow * a.ldv + hk * a.HS, a.HS, live, half, vh, vl, &ev);
  const float cv = split_unscale(ev);
  bool bad = kbits >= kInfBits || vbits >= kInfBits;

  const GroupRows<BQ, KG> gq{q + (size_t)s.q0 * a.ldq + hk * G * a.HS, a.ldq, a.HS, G};
  const GroupRows<BQ, KG> gg{dout + (size_t)s.q0 * a.ldo + hk * G * a.HS, a.ldo, a.HS, G};
  const size_t stat = (size_t)s.q0 * a.NH + hk * G;
  Rows4 t[kPer];
  float tL = 0.0f, tD = 0.0f;
  bool past = false;  // this thread's row of the tile is behind the last one: its P are 0
  const auto is_g = [&](int u) { return kPer == 1 ? wave >= W / 2 : u >= kPer / 2; };
  const auto block = [&](int u) { return (tid + u * kThreads) % kBlocks; };
  long long off[kPer][4];  // a tile's rows from its first one
#pragma unroll
  for (int u = 0; u < kPer; u++)
#pragma unroll
    for (int x = 0; x < 4; x++) {
      const int r = block(u) / DG + KG * x, i = r / G;
      off[u][x] = i * (is_g(u) ? a.ldo : a.ldq) + (r - i * G) * a.HS;
    }
  const auto load = [&](int r0) {
#pragma unroll
    for (int u = 0; u < kPer; u++) {
      const int d = block(u) % DG * 4, x = block(u) / DG;
      t[u] = is_g(u) ? gg.template load<kSlots>(r0, off[u], x, d, rows, a.HS - d)
                     : gq.template load<kSlots>(r0, off[u], x, d, rows, a.HS - d);
    }
    if (tid < BQ) {
      const int r = r0 + tid, i = min(r, rows - 1) / G, x = min(r, rows - 1) - i * G;
      tL = lse[stat + (size_t)i * a.NH + x] * kLog2e;
      tD = dsum[stat + (size_t)i * a.NH + x];
      past = r >= rows;
      if (past) tL = tD = 0.0f;
      if (s.seen(i, a.causal) == 0) tL = 0.0f;  // a row without keys
    }
  };
  uint32_t small[kPer];
  const auto note = [&](int z, int r0) {
    uint32_t m[3] = {};
#pragma unroll
    for (int u = 0; u < kPer; u++) {
      const int w = is_g(u) ? 1 : 0;
      m[w] = max_abs(m[w], t[u], &small[u]);
      if (kSlots != kWhole && a.HS <= block(u) % DG * 4) small[u] = kInfBits;  // behind the row
      if (r0 < all) m[w] = max_abs<true>(m[w], t[u]);
    }
    if (tid < BQ) m[2] = abs_bits(tL);
    m[0] = wave_max_bits(m[0]);
    m[1] = wave_max_bits(m[1]);
    if (wave == 0) m[2] = wave_max_bits(m[2]);
    if (lane == 0) {
#pragma unroll
      for (int x = 0; x < 3; x++) slot[z][x][wave] = m[x];
    }
  };
  int eq = 0, eg = 0;  // of the tile staged last
  int lifted = 0;
  const auto stage = [&](int z, int r0) {
    const uint32_t mq = noted<W>(slot[z][0]), mg = noted<W>(slot[z][1]);
    bad = bad || (r0 + BQ > lo && (mq >= kInfBits || mg >= kInfBits || noted<W>(slot[z][2]) >= 0x4a800000u /* 2^22 */));
    eq = split_exp(mq);
    eg = split_exp(mg);
    bool spread = false;
#pragma unroll
    for (int u = 0; u < kPer; u++) spread = spread || may_spread(small[u], is_g(u) ? mg : mq);
    if (__any(spread) || (lifted >> z & 1))
      lift_tile<DG, KG>(t, lifts, z, rows - r0, lane, wave, &lifted, [&](int u) { return is_g(u) ? 1 : 0; },
                        [&](int u) { return is_g(u) ? eg : eq; }, [&](int u) { return block(u) / DG; });
    const float fq = split_scale(eq), fg = split_scale(eg);
#pragma unroll
    for (int u = 0; u < kPer; u++) {
      const int p = block(u) / DG * kRs + block(u) % DG * 4;
      const bool w = is_g(u);
      put_rows<KG>(t[u], w ? fg : fq, (w ? lg : lq)[z][0] + p, (w ? lg : lq)[z][1] + p, kRs);
    }
    if (tid < BQ) {
      lL[z][tid] = past ? -INFINITY : 15.0f - tL;
      lD[z][tid] = tD;
    }
  };

  v16f ak[DB] = {}, av[DB] = {};
  int ea = kNoScale, ev_acc = kNoScale;  // the exponents that dk's and dv's accumulators stand on
  const int cols = cols_at(lane, kRs);
  const auto compute = [&](int z, int r0, int eq_now, int eg_now) {
    const bool seen = live && lim < r0 + BQ;
    const float c2 = ldexpf(a.scale * kLog2e, ek + eq_now - 30), cd = cv * split_unscale(eg_now);
    bad = bad || (seen && (fabsf(c2) > 0x1p100f || cd > 0x1p100f));
    const uint32_t lifted_by = lifts.any(z);
    const int rel = r0 < hi || !live ? lim - r0 - 4 * half : 0;  // rows of the lane's half before rel do not see the key
    v16f p = dot_block<DC>(lq[z][0], lq[z][1], kRs, kh, kl, lane);
    const bool apart = __builtin_amdgcn_readfirstlane(lifted_by) != 0;
    if (apart) lower(p, lifts, z, 0, 0, half);
#pragma unroll
    for (int y = 0; y < 4; y++) {
      const float4 L = *reinterpret_cast<const float4 *>(&lL[z][8 * y + 4 * half]);
#pragma unroll
      for (int x = 0; x < 4; x++) p[4 * y + x] = __builtin_amdgcn_exp2f(fmaf(p[4 * y + x], c2, part4(L, x)));
    }
    if (r0 < hi || !live) {
#pragma unroll
      for (int y = 0; y < 16; y++)
        if (8 * (y / 4) + y % 4 < rel) p[y] = 0.0f;
    }
    if (apart) lower(p, lifts, z, 1, 0, half);
    bad = raise(ev_acc, av, p, eg_now) || bad;
    mac_block<DB>(av, p, pow2(max(min(15 + eg_now - ev_acc, 127), -126)), lg[z][0], lg[z][1], kRs, cols);
    // dP of dout's lifted rows, and with it D; P is that much lower
    v16f ds = dot_block<DC>(lg[z][0], lg[z][1], kRs, vh, vl, lane);
#pragma unroll
    for (int y = 0; y < 4; y++) {
      float4 D = *reinterpret_cast<const float4 *>(&lD[z][8 * y + 4 * half]);
      if (apart) {
        const int4 d = lifts.four(z, 1, 0, y, half);
        D = make_float4(ldexpf(D.x, -d.x), ldexpf(D.y, -d.y), ldexpf(D.z, -d.z), ldexpf(D.w, -d.w));
      }
#pragma unroll
      for (int x = 0; x < 4; x++) ds[4 * y + x] = p[4 * y + x] * fmaf(ds[4 * y + x], cd, -part4(D, x));
    }
    if (r0 < hi || !live) {
#pragma unroll
      for (int y = 0; y < 16; y++)
        if (8 * (y / 4) + y % 4 < rel) ds[y] = 0.0f;
    }
    if (apart) lower(ds, lifts, z, 0, 0, half);
    bad = raise(ea, ak, ds, eq_now) || bad;
    mac_block<DB>(ak, ds, pow2(max(min(15 + eq_now - ea, 127), -126)), lq[z][0], lq[z][1], kRs, cols);
  };

  const int tiles = rows > from ? (rows - from + BQ - 1) / BQ : 0;
  lifts.clear();
  if (tiles > 0) {
    load(from);
    note(0, from);
    __syncthreads();
    stage(0, from);
    if (tiles > 1) {
      load(from + BQ);
      note(1, from + BQ);
    }
    __syncthreads();
    for (int at = 0; at < tiles; at++) {
      const int r0 = from + at * BQ, eq_now = eq, eg_now = eg;
      if (at + 1 < tiles) stage((at + 1) & 1, r0 + BQ);
      if (at + 2 < tiles) load(r0 + 2 * BQ);
      if (r0 + BQ > lo) compute(at & 1, r0, eq_now, eg_now);
      if (at + 2 < tiles) note(at & 1, r0 + 2 * BQ);
      __syncthreads();
    }
  }
  const size_t wk = (size_t)a.NKV * a.HS, part = (size_t)part_no * a.rows_k * wk + hk * a.HS;
  float *ok = parts.dk ? parts.dk + part : dk + hk * a.HS, *ov = parts.dk ? parts.dv + part : dv + hk * a.HS;
  const size_t ldk = parts.dk ? wk : (size_t)a.ldk, ldv = parts.dk ? wk : (size_t)a.ldv;
  assign = assign || parts.dk;
  if (__any(bad)) {
    for (int x = 0; x < 32; x++) {
      const int jj = key0 + wave * 32 + x;
      if (jj >= s.Lk) break;
      const size_t g = (size_t)s.k0 + jj;
      row_dkv(ok + g * ldk, ov + g * ldv, dout, q, k, v, lse, dsum, a, s, jj, hk, from, rows, assign);
    }
    return;
  }
  if (!live) return;
  put_scaled<DB, kSlots == kWhole>(ok + grow * ldk, ak, ea - 45, a.scale, half, a.HS, assign);  // P, and so dS, was 2^15 up
  put_scaled<DB, kSlots == kWhole>(ov + grow * ldv, av, ev_acc - 45, 1.0f, half, a.HS, assign);
}

// The parts' dk and dv added, in the parts' order, a thread per element.
__global__ __launch_bounds__(kBlock) void k_att_dkv_join(float *dk, float *dv, Halves parts, ugk_attention a, bool assign) {
  const Seq s = sequence(a, blockIdx.z, false, nullptr, 0);
  const int j = blockIdx.x, c = blockIdx.y * kBlock + threadIdx.x, wk = a.NKV * a.HS;
  if (j >= s.Lk || c >= wk) return;
  const size_t row = (size_t)s.k0 + j, all = (size_t)a.rows_k * wk;
  float x[kMaxSplits], y[kMaxSplits];
#pragma unroll
  for (int p = 0; p < kMaxSplits; p++) {
    const size_t at = min(p, parts.splits - 1) * all + row * wk + c;
    x[p] = parts.dk[at];
    y[p] = parts.dv[at];
  }
#pragma unroll
  for (int p = 1; p < kMaxSplits; p++)
    if (p < parts.splits) {
      x[0] += x[p];
      y[0] += y[p];
    }
  put(dk + row * a.ldk + c, x[0], assign);
  put(dv + row * a.ldv + c, y[0], assign);
}

}  // namespace

namespace {
int cu_count() {
  static const int n = [] {
    int dev = 0, c = 0;
    if (hipGetDevice(&dev) != hipSuccess || hipDeviceGetAttribute(&c, hipDeviceAttributeMultiprocessorCount, dev) != hipSuccess) {
      (void)hipGetLastError();
      c = 0;
    }
    return c > 0 ? c : 256;
  }();
  return n;
}

// Workgroups of `tile` rows over all sequences of a call, about: packed sequences
// are mostly shorter than the longest.
long long filled(const ugk_attention &a, long long rows, long long most, int group, int tile) {
  const long long by_longest = (long long)a.nseq * ((most * group + tile - 1) / tile);
  const long long by_rows = (rows * group + tile - 1) / tile + a.nseq;
  return min(by_longest, by_rows) * a.NKV;
}
// dk and dv: parts of the rows' range where the keys make too few workgroups to fill
// the CUs, which hold two workgroups for heads up to 64 and one for larger ones,
// twice (the heads of a group share their keys: 4 x 2,048 rows of 16/4 heads 769 us
// whole, 370 in four parts and 13 to add them; up to 16 parts for four times as
// many workgroups took 203 against 187 us packed, 1,332 against 1,282 for 4 x 2,048 rows
// of 16/4 heads of 128). A part has four tiles or more, and the parts, which hold all
// key rows, stay below kSplitKeys keys per CU (attention_backward_bound): a cache of
// which the sequences are a small part has fewer.
constexpr long long kSplitKeys = 4 * kTileRows;  // per CU, over all parts and heads
int dkv_splits(const ugk_attention &a) {
  const long long rows = (long long)a.max_q * (a.NH / a.NKV);
  const long long want = (a.HS > 64 ? 2LL : 4LL) * cu_count() / max(filled(a, a.rows_k, a.max_k, 1, kTileRows), 1LL);
  const long long keys = kSplitKeys * cu_count() / max((long long)a.rows_k * a.NKV, 1LL);
  return (int)max(1LL, min(min(min(want, keys), (long long)kMaxSplits), rows / 128));
}

constexpr int kFewRows = 4, kFewChunk = 1024, kFewWide = 2048;  // rows of k_att_few; keys per part; keys of large workgroups
constexpr size_t kMaxParts = 1 << 15;  // rows of a head that the parts hold at most

// How the forward of `a` is cut: rows per key/value head where they are few and their
// workgroup's wavefronts (k_att_few), else blocks of 32 rows per wavefront; tiles of rows, parts of the key axis and keys per part.
struct FwdPlan {
  int few, W, QB, tiles, splits, chunk;
};
FwdPlan fwd_plan(const ugk_attention &a) {
  const long long pairs = (long long)a.nseq * a.NKV, rows = (long long)a.max_q * (a.NH / a.NKV);
  FwdPlan p{};
  int unit;  // keys that a workgroup takes at a time
  if (rows <= kFewRows) {
    p.few = rows <= 1 ? 1 : rows <= 2 ? 2 : 4;
    p.tiles = 1;
    // Large workgroups for short caches, which make few parts: 24 sequences, 32/8 heads of 128, of up to 512, 1,024,
    // 1,536 and 2,048 keys 17, 28, 28 and 36 us, 23, 40, 37 and 46 in workgroups of four wavefronts; 16 of 12
    // heads of 64 10, 13, 17 and 23, and 10, 14, 21 and 27. Of up to 4,096 49 and 44 (79 and 83 with 128).
    p.W = pairs < 4 * cu_count() && a.max_k <= kFewWide ? few_waves(p.few) : 4;
    unit = p.W * (a.HS <= 64 ? 4 : 2) * few_loads(p.few);
  } else {
    // Two 32-row blocks per wavefront halve the staging and the reads of K and V per
    // row, and pay while there are three workgroups per CU to balance the causal
    // rows' lengths (16,384 rows of 12 heads 1,335 us against 1,453, 4 x 4,096
    // 415 against 444; with one and a half 8 x 1,024 88 against 70).
    p.QB = a.HS <= 64 && filled(a, a.rows_q, a.max_q, a.NH / a.NKV, 2 * kTileRows) >= 3 * cu_count() ? 2 : 1;
    p.tiles = (int)((rows + kTileRows * p.QB - 1) / (kTileRows * p.QB));
    unit = a.HS <= 64 && p.QB == 1 ? 64 : 32;
  }
  p.splits = 1;
  const long long wgs = pairs * p.tiles, prow = (long long)a.nseq * a.max_q * a.NH;
  long long want = (p.few ? 1 : 2) * cu_count() / (wgs > 0 ? wgs : 1);
  // One tile of rows for all of a sequence's keys: parts of kFewChunk keys also where the
  // workgroups fill the CUs, for a cache's lengths differ and the longest would run alone.
  // On the 32-row tiles up to 8 of them (64/8 heads: 24 sequences of up to 16,384 keys of
  // 128 324 us, 525 without and 333 without the limit; 48 of them, of 64, 403, 561 and 411; 24
  // of 8,192 each 273, 309 and 273. Against it: 24 of 4,096 each, of 64, 102 and 92 without, 32
  // of up to 4,096 88 and 83).
  const long long chunks = (a.max_k + (long long)kFewChunk - 1) / kFewChunk;
  if (p.tiles == 1) want = max(want, p.few ? chunks : min((long long)a.max_k / kFewChunk, 8LL));
  want = min(want, (long long)a.max_k / (4 * unit));
  want = min(want, (long long)kMaxParts / (prow > 0 ? prow : 1));
  if (want > 1) {
    p.chunk = (int)((a.max_k + want - 1) / want + unit - 1) / unit * unit;
    p.splits = (a.max_k + p.chunk - 1) / p.chunk;
  }
  return p;
}
size_t parts_rows(const ugk_attention &a, const FwdPlan &p) { return (size_t)p.splits * a.nseq * a.max_q * a.NH; }
}  // namespace

size_t attention_parts_bytes(const ugk_attention &a) {
  const FwdPlan p = fwd_plan(a);
  return p.splits > 1 ? parts_rows(a, p) * (a.HS + 2) * sizeof(float) : 0;
}
size_t attention_parts_bound(size_t HS) { return kMaxParts * (HS + 2) * sizeof(float); }

int launch_attention_forward(float *out, float *lse, const float *q, const float *k, const float *v, float *mem,
                             const ugk_attention &a, int *word) {
  const FwdPlan p = fwd_plan(a);
  Parts parts{};
  if (p.splits > 1) {
    parts.m = mem;
    parts.l = parts.m + parts_rows(a, p);
    parts.o = parts.l + parts_rows(a, p);
    parts.splits = p.splits;
    parts.chunk = p.chunk;
  }
  const unsigned pairs = (unsigned)a.nseq * a.NKV;
  const auto go = [&](auto kernel) {
    launch(kernel, dim3(pairs * p.tiles, p.splits), dim3(kTileThreads), 0, out, lse, q, k, v, a, parts, pairs, word);
  };
  if (p.few) {
    const auto few = [&](auto kernel) {
      launch(kernel, dim3(pairs * p.splits), dim3(p.W * kWave), 0, out, lse, q, k, v, a, parts, pairs, word);
    };
#define UGK_FEW_HS(r, w)                                                             \
  if (a.HS == 64) few(k_att_few<64, r, w, true>);                                    \
  else if (a.HS < 64) few(k_att_few<64, r, w, false>);                               \
  else if (a.HS == 128) few(k_att_few<128, r, w, true>);                             \
  else few(k_att_few<128, r, w, false>);
#define UGK_FEW(r)                                                                   \
  case r:                                                                            \
    if (p.W == 4) { UGK_FEW_HS(r, 4) } else { UGK_FEW_HS(r, few_waves(r)) }          \
    break;
    switch (p.few) { UGK_FEW(1) UGK_FEW(2) UGK_FEW(4) }
#undef UGK_FEW
#undef UGK_FEW_HS
  } else if (a.HS <= 64) {
    const bool full = a.HS == 64;
    if (p.QB == 2) full ? go(k_att_fwd<64, 32, 2, true>) : go(k_att_fwd<64, 32, 2, false>);
    else full ? go(k_att_fwd<64, 64, 1, true>) : go(k_att_fwd<64, 64, 1, false>);
  } else {
    a.HS == 128 ? go(k_att_fwd<128, 32, 1, true>) : go(k_att_fwd<128, 32, 1, false>);
  }
  if (int e = check_launch("attention_forward")) return e;
  if (p.splits > 1) {
    launch(k_att_join, dim3(grid_for((size_t)a.nseq * a.max_q * a.NH, kBlock / kWave)), dim3(kBlock), 0, out, lse, parts, a);
    return check_launch("attention_forward");
  }
  return UGK_OK;
}

size_t attention_backward_bytes(const ugk_attention &a) {
  const size_t splits = dkv_splits(a), dsum = ((size_t)a.rows_q * a.NH + 63) / 64 * 64;
  return (dsum + (splits > 1 ? 2 * splits * a.rows_k * a.NKV * a.HS : 0)) * sizeof(float);
}
// dkv_splits: at most kMaxSplits, kSplitKeys keys per CU over all, and a part per 128 rows of q per key/value head, of
// which a group has more in proportion to its fewer key/value heads.
size_t attention_backward_bound(size_t rows, size_t NH, size_t HS) {
  const size_t splits = min((size_t)kMaxSplits, (rows + 127) / 128);
  const size_t split = min(splits * rows * NH, (size_t)kSplitKeys * cu_count()) * HS;
  return ((rows * NH + 63) / 64 * 64 + 2 * split) * sizeof(float);
}

int launch_attention_backward(float *dq, float *dk, float *dv, const float *dout, const float *q, const float *k,
                              const float *v, const float *out, const float *lse, float *mem, const ugk_attention &a,
                              bool assign, int *word) {
  float *dsum = mem;
  const unsigned pairs = (unsigned)a.nseq * a.NKV;
  // Head sizes of 65 to 127 that are multiples of 4 (80, 96, ..) have kernels of their own: reading
  // the rows' ends float by float costs dk and dv 288 bytes a lane of spills (4 x 2,048 rows of
  // 16/4 heads of 100: 1,225 us, 1,705 in the general form, which up to 64 spills nothing).
  const bool wide = a.HS > 64, full = a.HS == (wide ? 128 : 64), quads = a.HS % 4 == 0;
  if (const long long rows = (long long)a.max_q * (a.NH / a.NKV)) {
    const auto go = [&](auto kernel) {
      launch(kernel, dim3(pairs * grid_for((size_t)rows, kTileRows)), dim3(kTileThreads), 0, dq, dsum, dout, q, k, v, out, lse,
             a, pairs, assign, word);
    };
    if (wide) full ? go(k_att_dq<128, 32, kWhole>) : quads ? go(k_att_dq<128, 32, kQuads>) : go(k_att_dq<128, 32, kAny>);
    else full ? go(k_att_dq<64, 64, kWhole>) : go(k_att_dq<64, 64, kAny>);
    if (int e = check_launch("attention_backward")) return e;
  }
  if (a.max_k) {
    const int splits = dkv_splits(a);
    Halves parts{};
    if (splits > 1) {
      parts.dk = mem + ((size_t)a.rows_q * a.NH + 63) / 64 * 64;
      parts.dv = parts.dk + (size_t)splits * a.rows_k * a.NKV * a.HS;
      parts.splits = splits;
    }
    const auto go = [&](auto kernel) {
      launch(kernel, dim3(pairs * grid_for((size_t)a.max_k, kTileRows) * splits), dim3(kTileThreads), 0, dk, dv, dout, q, k, v,
             lse, dsum, a, parts, pairs, assign, word);
    };
    if (wide) full ? go(k_att_dkv<128, kWhole>) : quads ? go(k_att_dkv<128, kQuads>) : go(k_att_dkv<128, kAny>);
    else full ? go(k_att_dkv<64, kWhole>) : go(k_att_dkv<64, kAny>);
    if (splits > 1) {
      if (int e = check_launch("attention_backward")) return e;
      launch(k_att_dkv_join, dim3(a.max_k, grid_for((size_t)a.NKV * a.HS, kBlock), a.nseq), dim3(kBlock), 0, dk, dv, parts, a,
             assign);
    }
  }
  return check_launch("attention_backward");
}

}  // namespace ugk
