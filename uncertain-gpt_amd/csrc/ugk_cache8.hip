// ugk_cache8.hip - a cache of keys and values in 8 bits: store, load, attention
// over it, and the eviction of blocks that got little weight.
//
// A block of 64 tokens of one key/value head holds whole numbers c of up to 127
// times a scale s. s is a power of two: x / s and c s are then exact, a code is one
// rounding of one number (to half a step: 2^-7 to 2^-8 of the block's largest), and
// the codes of a block whose scale grows with a later token are rounded again from
// what they stand for, at most half a step of the new scale away. (A scale of
// max / 127 would have steps up to twice as fine, and would round all older
// codes again for every token that raises the maximum a little.)
//
// Keys lie as rows, values as columns: both are then the operands of
// v_mfma_i32_16x16x64_i8 as they come from memory, 16 codes per lane, without a
// conversion, a transposition or a trip through LDS. Rows are padded to a multiple
// of 16 codes with zeros. Key i of a block stands at place 4 (i % 16) + i / 16 of a
// column, the order in which the lanes hold the weights.
#include <math.h>

#include <type_traits>

#include "ugk_internal.h"
#include "ugk_split.h"

namespace ugk {
namespace {

constexpr int kKeys = kCacheBlock;  // 64: a lane holds four scores of a block and row
typedef int v4i __attribute__((ext_vector_type(4)));
constexpr float kLog2e8 = 1.44269504088896340736f, kLn28 = 0.69314718055994530942f;

// One sequence: its first row, its rows and its keys.
struct Seq8 {
  int q0, Lq, Lk;
  // the keys that row i sees: [0, seen(i))
  __device__ __forceinline__ int seen(int i, int causal) const { return causal ? max(0, min(Lk, i + 1 + Lk - Lq)) : Lk; }
};

// Sequence b; threads with `tell` report rows and lengths that were clamped.
__device__ __forceinline__ Seq8 sequence8(const ugk_cache8 &a, int b, bool tell, int *word, int code) {
  Seq8 s;
  bool bad = false;
  s.Lq = clamp_rows(a.q_start, a.q_end, b, a.rows_q, a.max_q, &s.q0, &bad);
  const int n = a.k_len ? a.k_len[b] : a.max_k;
  s.Lk = min(max(n, 0), a.max_k);
  bad = bad || s.Lk != n;
  if (bad && tell) *word = code;
  return s;
}

// What the table says of block j of sequence b, and the block, or -1 (reported) where that is none. (Two steps: a loop reads
// the table a turn before it needs the block.)
__device__ __forceinline__ int table_at(const ugk_cache8 &a, int b, int j) {
  const size_t at = (size_t)b * a.ld_table + j;
  return a.table ? a.table[at] : (int)at;
}
__device__ __forceinline__ int checked_block(const ugk_cache8 &a, int id, int *word, int code) {
  if ((unsigned)id < (unsigned)a.nblocks) return id;
  *word = code;
  return -1;
}
__device__ __forceinline__ int block_of(const ugk_cache8 &a, int b, int j, int *word, int code) {
  return checked_block(a, table_at(a, b, j), word, code);
}

__host__ __device__ __forceinline__ int padded(int HS) { return (HS + 15) & ~15; }

// ---- store and load -------------------------------------------------------------

// The scale for numbers up to the one with these bits: the least power of two s, 2^-126 to
// 2^121, with it <= 127 s (beyond 127 2^121 numbers are held as that); 0 for 0.
__device__ __forceinline__ float scale_for(uint32_t bits) {
  if (bits == 0) return 0.0f;
  // 1.f 2^(x - 127) <= 127 2^e, that is 1.f <= (127 / 64) 2^(e + 133 - x) with 127 / 64 = 1 + 0x7e0000 / 2^23
  const int e = (int)(bits >> 23) - 133 + ((bits & 0x7fffffu) > 0x7e0000u);
  return __uint_as_float((uint32_t)(min(max(e, -126), 121) + 127) << 23);
}
__device__ __forceinline__ int code_of(float x, float inv) { return (int)fminf(fmaxf(rintf(x * inv), -127.0f), 127.0f); }
__device__ __forceinline__ uint32_t pack4(int a, int b, int c, int d) {
  return (uint32_t)(a & 255) | (uint32_t)(b & 255) << 8 | (uint32_t)(c & 255) << 16 | (uint32_t)d << 24;
}
__device__ __forceinline__ int code_at(uint32_t w, int j) { return (int)(w << (24 - 8 * j)) >> 24; }
// Four codes of the scale `was` as codes of the scale `now` (ratio = was / now, a power of two below 1).
__device__ __forceinline__ uint32_t again4(uint32_t w, float ratio) {
  return pack4(code_of((float)code_at(w, 0), ratio), code_of((float)code_at(w, 1), ratio), code_of((float)code_at(w, 2), ratio),
               code_of((float)code_at(w, 3), ratio));
}

__device__ __forceinline__ int last_lane(int x) { return __builtin_amdgcn_readlane(x, kWave - 1); }

// What a workgroup of the store and the load has: block j of a sequence, of which rows [r0, r1) are
// the call's, those before r0 in the cache already.
struct Touched {
  int b, h, j, q, r0, r1;  // q: the buffer's row of r0
};
// Workgroups are of heads, and of `per` blocks of each sequence; or (per 0) of the `all` blocks that there are, a lane to a
// sequence finds which.
__device__ __forceinline__ bool touched(const ugk_cache8 &a, int per, int all, int *word, int code, Touched *t) {
  const bool first = blockIdx.x == 0 && blockIdx.y == 0;
  int nth = blockIdx.x / a.NKV;
  Seq8 s;
  t->h = blockIdx.x % a.NKV;
  if (per) {
    t->b = nth / per;
    nth %= per;
    const bool tell = t->h == 0 && nth == 0 && blockIdx.y == 0;
    s = sequence8(a, t->b, tell, word, code);
    if (s.Lq > s.Lk && tell && threadIdx.x == 0) *word = code;  // rows before the first key
  } else {
    const int lane = threadIdx.x & (kWave - 1);
    t->b = -1;
    for (int b0 = 0; b0 < a.nseq && (t->b < 0 || first); b0 += kWave) {
      Seq8 own{0, 0, 0};
      int n = 0;
      if (b0 + lane < a.nseq) {
        own = sequence8(a, b0 + lane, first, word, code);
        if (own.Lq > own.Lk && first) *word = code;
        if (own.Lq > 0) n = (own.Lk + kKeys - 1) / kKeys - max(own.Lk - own.Lq, 0) / kKeys;
      }
      const int to = wave_scan(n);
      const uint64_t over = __ballot(to > nth);
      if (over && t->b < 0) {
        const int l = __builtin_ctzll(over);
        t->b = b0 + l;
        s = Seq8{__builtin_amdgcn_readlane(own.q0, l), __builtin_amdgcn_readlane(own.Lq, l), __builtin_amdgcn_readlane(own.Lk, l)};
        nth -= __builtin_amdgcn_readlane(to - n, l);
      } else if (t->b < 0) {
        nth -= last_lane(to);
      }
      all -= last_lane(to);
    }
    if (first && all < 0 && threadIdx.x == 0) *word = code;  // rows in several sequences: there is no workgroup for some
    if (t->b < 0) return false;
  }
  const int begin = max(s.Lk - s.Lq, 0);
  t->j = begin / kKeys + nth;
  if (s.Lq == 0 || t->j * kKeys >= s.Lk) return false;
  t->r0 = max(begin - t->j * kKeys, 0);
  t->r1 = min(s.Lk - t->j * kKeys, kKeys);
  t->q = s.q0 + s.Lq - s.Lk + t->j * kKeys + t->r0;
  return true;
}

// One block of one head and of k or v (blockIdx.y) by a workgroup. A thread has four columns of the rows
// c, c + 16, c + 32, c + 48, whose codes are one word of each of the value's columns.
//
// Bound by memory: 4 bytes read and 1 written per number, 4.4 TB/s of 8 x 1,024 keys and values of 12 heads of 64 (14.2 us),
// 5.4 the way back (k_cache8_load, 11.7 us). A token behind others costs the launch and three loads that depend on
// each other: 4.4 us of 4 sequences, 6.4 of 24 with 8 heads of 128.
template <int CH>
__global__ __launch_bounds__(kBlock) void k_cache8_store(int8_t *k8, float *ks, int8_t *v8, float *vs, const float *k, const float *v,
                                                         ugk_cache8 a, int per, int all, int *word) {
  constexpr int HP = 16 * CH, G = HP / 4, kPer = (16 * G + kBlock - 1) / kBlock;
  __shared__ uint32_t tile[HP * 17];  // the values' words, 17 to a column of 16: banks that differ
  __shared__ uint32_t top[kBlock / kWave];
  Touched t;
  if (!touched(a, per, all, word, UGK_IDS_CACHE8_STORE, &t)) return;
  const bool values = blockIdx.y;
  const long long ld = values ? a.ldv : a.ldk;
  const float *src = (values ? v : k) + (long long)(t.q - t.r0) * ld + t.h * a.HS;
  const int id = block_of(a, t.b, t.j, word, UGK_IDS_CACHE8_STORE);  // on its way while the rows are
  // What lies outside the call's rows and the head is read from the nearest that does not, and taken as 0: a branch would wait
  // for each of these loads.
  float4 x[kPer][4];
  const auto mine = [&](int i, int r, auto &&take) {
    const int e = threadIdx.x + i * kBlock, d = e % G * 4, row = e / G + 16 * r;
    take(src + min(max(row, t.r0), t.r1 - 1) * ld, d, e / G < 16 && row >= t.r0 && row < t.r1, x[i][r]);
  };
  if (a.HS % 4 == 0) {
#pragma unroll
    for (int i = 0; i < kPer; i++)
#pragma unroll
      for (int r = 0; r < 4; r++)
        mine(i, r, [&](const float *p, int d, bool in, float4 &y) {
          const float4 z = ld4(p + min(d, a.HS - 4));
          in = in && d < a.HS;
          y = make_float4(in ? z.x : 0.0f, in ? z.y : 0.0f, in ? z.z : 0.0f, in ? z.w : 0.0f);
        });
  } else {
#pragma unroll
    for (int i = 0; i < kPer; i++)
#pragma unroll
      for (int r = 0; r < 4; r++)
        mine(i, r, [&](const float *p, int d, bool in, float4 &y) {
          const float z0 = p[min(d, a.HS - 1)], z1 = p[min(d + 1, a.HS - 1)], z2 = p[min(d + 2, a.HS - 1)], z3 = p[min(d + 3, a.HS - 1)];
          y = make_float4(in && d < a.HS ? z0 : 0.0f, in && d + 1 < a.HS ? z1 : 0.0f, in && d + 2 < a.HS ? z2 : 0.0f,
                          in && d + 3 < a.HS ? z3 : 0.0f);
        });
  }
  uint32_t most = 0;
  if (id < 0) return;
  const size_t at = (size_t)id * a.NKV + t.h;
  float *sp = (values ? vs : ks) + at;
  uint32_t *dst = reinterpret_cast<uint32_t *>((values ? v8 : k8) + at * kKeys * HP);
  // words of the values hold four keys: of a block that is not all new what they hold is on its way with the scale
  const bool whole = t.r0 == 0 && t.r1 == kKeys;
  uint32_t held[CH];
  if (values && !whole) {
#pragma unroll
    for (int i = 0; i < CH; i++) held[i] = dst[threadIdx.x + i * kBlock];
  }
  const float was = t.r0 > 0 ? *sp : 0.0f;
  bool finite = true;
  const auto look = [&](float &f) {
    const uint32_t u = abs_bits(f);
    finite = finite && u < kInfBits;
    if (u > kInfBits) f = 0.0f;  // NaN
    else most = max(most, u);
  };
#pragma unroll
  for (int i = 0; i < kPer; i++)
#pragma unroll
    for (int r = 0; r < 4; r++) {
      look(x[i][r].x);
      look(x[i][r].y);
      look(x[i][r].z);
      look(x[i][r].w);
    }
  if (!finite) *word = UGK_IDS_CACHE8_VALUES;
  most = wave_max_bits(most);
  if ((threadIdx.x & (kWave - 1)) == 0) top[threadIdx.x / kWave] = most;
  __syncthreads();
  static_assert(kBlock / kWave == 4, "four wavefronts");
  most = max(max(top[0], top[1]), max(top[2], top[3]));
  const float now = fmaxf(was, scale_for(most));
  const float inv = now > 0.0f ? 1.0f / now : 0.0f, ratio = was * inv;
  const bool grown = t.r0 > 0 && now > was && was > 0.0f;
  uint32_t w[kPer][4];
#pragma unroll
  for (int i = 0; i < kPer; i++)
#pragma unroll
    for (int r = 0; r < 4; r++)
      w[i][r] = pack4(code_of(x[i][r].x, inv), code_of(x[i][r].y, inv), code_of(x[i][r].z, inv), code_of(x[i][r].w, inv));
  if (!values) {
#pragma unroll
    for (int i = 0; i < kPer; i++) {
      const int e = threadIdx.x + i * kBlock, g = e % G, c = e / G;
#pragma unroll
      for (int r = 0; r < 4; r++) {
        const int row = c + 16 * r;
        if (c < 16 && row >= t.r0 && row < t.r1) dst[row * G + g] = w[i][r];
      }
    }
    if (grown)
      for (int e = threadIdx.x; e < t.r0 * G; e += kBlock) dst[e] = again4(dst[e], ratio);
  } else {
    // words of four keys of one column, from words of four columns of one key
#pragma unroll
    for (int i = 0; i < kPer; i++) {
      const int e = threadIdx.x + i * kBlock, g = e % G, c = e / G;
      if (c >= 16) continue;
#pragma unroll
      for (int d = 0; d < 4; d++)
        tile[(4 * g + d) * 17 + c] = pack4(code_at(w[i][0], d), code_at(w[i][1], d), code_at(w[i][2], d), code_at(w[i][3], d));
    }
    __syncthreads();
    static_assert(HP * 16 == CH * kBlock, "a word of each turn for every thread");
#pragma unroll
    for (int i = 0; i < CH; i++) {
      const int e = threadIdx.x + i * kBlock, d = e / 16, c = e % 16;
      uint32_t word4 = tile[d * 17 + c];
      if (!whole) {
        uint32_t fresh = 0, older = 0;  // the bytes of the call's rows, of the rows before
#pragma unroll
        for (int r = 0; r < 4; r++) {
          const int row = c + 16 * r;
          if (row < t.r0) older |= 0xffu << 8 * r;
          else if (row < t.r1) fresh |= 0xffu << 8 * r;
        }
        if (!fresh && !(older && grown)) continue;
        uint32_t old = held[i];
        if (grown) old = (again4(old, ratio) & older) | (old & ~older);
        word4 = (word4 & fresh) | (old & ~fresh);
      }
      dst[e] = word4;
    }
  }
  __syncthreads();  // every thread has read the scale that was
  if (threadIdx.x == 0 && (now != was || t.r0 == 0)) *sp = now;
}

// The store's rows, read back.
template <int CH>
__global__ __launch_bounds__(kBlock) void k_cache8_load(float *k, float *v, const int8_t *k8, const float *ks, const int8_t *v8,
                                                        const float *vs, ugk_cache8 a, int per, int all, int *word) {
  constexpr int HP = 16 * CH, G = HP / 4;
  __shared__ uint32_t tile[HP * 17];
  Touched t;
  if (!touched(a, per, all, word, UGK_IDS_CACHE8_LOAD, &t)) return;
  const bool values = blockIdx.y;
  const long long ld = values ? a.ldv : a.ldk;
  float *to = (values ? v : k) + (long long)(t.q - t.r0) * ld + t.h * a.HS;
  const int id = block_of(a, t.b, t.j, word, UGK_IDS_CACHE8_LOAD);
  if (id < 0) return;
  const size_t at = (size_t)id * a.NKV + t.h;
  const float s = (values ? vs : ks)[at];
  const uint32_t *src = reinterpret_cast<const uint32_t *>((values ? v8 : k8) + at * kKeys * HP);
  uint32_t w[CH];
#pragma unroll
  for (int i = 0; i < CH; i++) w[i] = src[threadIdx.x + i * kBlock];
  if (values) {
#pragma unroll
    for (int i = 0; i < CH; i++) {
      const int e = threadIdx.x + i * kBlock;
      tile[e / 16 * 17 + e % 16] = w[i];
    }
    __syncthreads();
  }
#pragma unroll
  for (int i = 0; i < CH; i++) {
    const int e = threadIdx.x + i * kBlock, row = e / G, g = e % G, nd = a.HS - 4 * g;
    if (row < t.r0 || row >= t.r1 || nd <= 0) continue;
    if (values) {
      const uint32_t *p = tile + 4 * g * 17 + (row & 15);
      const int r = row >> 4;
      w[i] = pack4(code_at(p[0], r), code_at(p[17], r), code_at(p[34], r), code_at(p[51], r));
    }
    float *p = to + row * ld + 4 * g;
    const float4 x = make_float4((float)code_at(w[i], 0) * s, (float)code_at(w[i], 1) * s, (float)code_at(w[i], 2) * s,
                                 (float)code_at(w[i], 3) * s);
    if (nd >= 4) {
      st4(p, x);
    } else {
      p[0] = x.x;
      if (nd > 1) p[1] = x.y;
      if (nd > 2) p[2] = x.z;
    }
  }
}

// ---- attention --------------------------------------------------------------------

// Parts of the key axis: o normalised, the maximum m of its scores in base 2 and the sum l of 2^(s - m), per slot and row of
// a group; `block`: the same m and l of each block of 64 keys, and `stat` of rows that have no parts (for the blocks'
// weights).
struct Parts8 {
  float *o;
  float2 *ml, *block, *stat;
  // What the launch behind has to know: the jobs that there are (one of every sequence, head and group where workgroups have
  // one), four words; eight words for each, in their order: the sequence's first row and its rows, the head, the group, the
  // slot of the first part, the parts (0: no such job); and, for the blocks' weights, of every sequence, head and group the
  // two last again where workgroups have many.
  int *told;
  int rows, step;      // of a slot; 1 where a job's parts lie in slots side by side, 2 where those behind the first are at 2 x workgroup
  int splits, least;   // most parts of a job where workgroups are of one, blocks per part at least
  int ld, most;        // blocks of max_k keys; jobs where they are counted
  int wgs, cus;        // workgroups that share all blocks (0: a workgroup has one job's part), CUs
  unsigned inverse;    // ceil(2^32 / heads of a group), 0 for one head
  float factor;        // |scale| log2(e) is this, 0 or 1/2 to 1, times 2^power: the product itself may leave a float's range
  int power;
};
__host__ __device__ __forceinline__ int part_floats(int HS) { return (HS + 3) & ~3; }
// Where a row of part p is, whose job's first part is in slot `first`.
__device__ __forceinline__ size_t part_row(const Parts8 &parts, int first, int p, int r) {
  const int slot = p ? (first & -parts.step) + parts.step * p : first;
  return (size_t)slot * parts.rows + r;
}

__device__ __forceinline__ float ex2(float x) { return __builtin_amdgcn_exp2f(x); }
__device__ __forceinline__ float or0(float m) { return m == -INFINITY ? 0.0f : m; }

// The exponent of a block's scale, a power of two; of 0 below all others.
__device__ __forceinline__ float exponent(float scale) { return scale == 0.0f ? -4096.0f : (float)(__builtin_amdgcn_frexp_expf(scale) - 1); }

// Running sums of a row. l stands on m, the largest score so far; the output's sum on the block whose weight times
// values was largest, 2^(mo + e): a block's values share a scale, so neither large values of little weight
// nor small ones of much cost the others their digits, and nothing leaves the range before the division.
struct Running {
  float m = -INFINITY, l = 0.0f, mo = -INFINITY, e = 0.0f;
  // A block's largest score, and its sum times 2^up on another score that is no larger than the largest so far.
  __device__ __forceinline__ void sum(float mb, float lb, float on, float up) {
    const float top = fmaxf(m, mb), base = or0(top);
    l = fmaf(l, ex2(m - base), lb * ex2((on - base) - up));
    m = top;
  }
  // A block with largest score mb and values of the scale 2^ve: the output's sum stands on it if it is the largest. Returns
  // the factor of the sum so far.
  __device__ __forceinline__ float stand(float mb, float ve) {
    const bool more = (mb - mo) + (ve - e) > 0.0f;  // (of scores that have no digits left for ve, equal ones too)
    const float mn = more ? mb : mo, en = more ? ve : e, f = ex2((mo - or0(mn)) + (e - en));
    mo = mn;
    e = en;
    return f;
  }
  // The factor of such a block's sum of values, of which its weights stand on mb; of a block of which the row sees nothing 0.
  __device__ __forceinline__ float factor(float mb, float ve) const { return mb == -INFINITY ? 0.0f : ex2((mb - or0(mo)) + (ve - e)); }
  // The factor that makes the output's sum the output, as a float and a power of two.
  __device__ __forceinline__ float last(float sum, int *p) const {
    const float x = (or0(mo) - or0(m)) + e, r = rintf(x);
    *p = (int)fminf(fmaxf(r, -4096.0f), 4096.0f);
    return sum != 0.0f ? ex2(x - r) / sum : 0.0f;
  }
};

// S times N floats of a row of q from `first` on, `step` apart, 0 behind its HS, with the sign of the scores' scale; and the
// largest magnitude's bits. (One branch for all: a branch for each N would wait for its loads.)
template <int S, int N>
__device__ __forceinline__ uint32_t load_q(const float *p, int first, int step, const ugk_cache8 &a, float (&x)[S][N]) {
  if (a.HS % 4 == 0) {
#pragma unroll
    for (int s = 0; s < S; s++)
#pragma unroll
      for (int d = 0; d < N; d += 4) {
        const int at = first + s * step + d;
        const float4 y = ld4(p + min(at, a.HS - 4));
        x[s][d] = at < a.HS ? y.x : 0.0f;
        x[s][d + 1] = at < a.HS ? y.y : 0.0f;
        x[s][d + 2] = at < a.HS ? y.z : 0.0f;
        x[s][d + 3] = at < a.HS ? y.w : 0.0f;
      }
  } else {
#pragma unroll
    for (int s = 0; s < S; s++)
#pragma unroll
      for (int d = 0; d < N; d++) {
        const int at = first + s * step + d;
        const float y = p[min(at, a.HS - 1)];
        x[s][d] = at < a.HS ? y : 0.0f;
      }
  }
  uint32_t most = 0;
#pragma unroll
  for (int s = 0; s < S; s++)
#pragma unroll
    for (int d = 0; d < N; d++) {
      most = max(most, abs_bits(x[s][d]));
      if (a.scale < 0.0f) x[s][d] = -x[s][d];
    }
  return most;
}

// |scale| log2(e) of the call, ks of a block and 2^x of a row's whole numbers, as one factor of its scores: a normal
// number, so that a score of 0 stays 0 and -infinity of a masked one itself.
__device__ __forceinline__ float score_factor(const Parts8 &parts, float ks, int x) {
  const float y = __builtin_amdgcn_ldexpf(parts.factor * __builtin_amdgcn_frexp_mantf(ks), parts.power + __builtin_amdgcn_frexp_expf(ks) + x);
  return fmaxf(fminf(y, 3.402823466e38f), 0x1p-126f);
}
// x is computed here, in this branch: the compiler otherwise moves what only the next step of a loop uses behind the branches
// in between, and holds all that it is computed from until there; and a choice between a number and NaN, made once, it makes
// again for all that is computed with it.
template <typename T>
__device__ __forceinline__ T here(T x) {
  asm volatile("" : "+v"(x));
  return x;
}

// The largest score of a block from the largest product, and what is added to a score times the factor so that 2^ of it is
// the weight times 2^up: a score beyond the range makes it NaN.
__device__ __forceinline__ float top_score(float product, float fac) { return product == -INFINITY ? product : product * fac; }
__device__ __forceinline__ float less_top(float top, float up) { return here(top == INFINITY ? NAN : up - or0(top)); }
// A score beyond 2^20 has too few digits behind the point for this: top is rounded, the fused product is not, and what is
// between them, 2^-5 below, would be the largest weight's exponent. The largest product is taken off before the factor then,
// which leaves exactly 0 of it (for whole wavefronts; of the rows that do not need it, 0 is taken off). Looking for it costs
// little: prompts of 8 x 1,024 and their store 57.9 to 58.3 us, 57.6 to 57.7 without; tokens and drafts the same.
__device__ __forceinline__ bool far_score(float top) { return fabsf(top) > 0x1p20f && fabsf(top) < INFINITY; }

// Sum and maximum over the 16 lanes of a row.
__device__ __forceinline__ float sum16(float v) {
  v += dpp_lane<kDppQuadSwap1>(v);
  v += dpp_lane<kDppQuadSwap2>(v);
  v += dpp_lane<kDppHalfMirror>(v);
  return v + dpp_lane<kDppMirror>(v);
}
__device__ __forceinline__ float max16(float v) {
  v = fmaxf(v, dpp_lane<kDppQuadSwap1>(v));
  v = fmaxf(v, dpp_lane<kDppQuadSwap2>(v));
  v = fmaxf(v, dpp_lane<kDppHalfMirror>(v));
  return fmaxf(v, dpp_lane<kDppMirror>(v));
}

// x 2^p, at most 2^30 but for infinities and NaN, as a whole number.
__device__ __forceinline__ int whole(float x, int p) {
  return (int)rintf(fminf(fmaxf(__builtin_amdgcn_ldexpf(x, p), -0x1p30f), 0x1p30f));
}
// A whole number of up to 2^30 as four digits of base 256 in [-128, 127], a byte each.
__device__ __forceinline__ uint32_t digits(int x) { return ((uint32_t)x + 0x00808080u) ^ 0x00808080u; }
// The number whose digits' sums of products are d (each below 2^21): exact but for the roundings to float.
__device__ __forceinline__ float undigits(v4i d) {
  return fmaf((float)(d[3] * 256 + d[2]), 65536.0f, (float)(d[1] * 256 + d[0]));
}

constexpr int kFewWaves = 4;

// The codes of a block as the operands of the 8-bit matrix units: 16 bytes a lane of 16 keys' rows (kf) and of 16 columns (vf),
// and the scales. A block that is not there is read as block 0, and its keys are masked.
template <int DT>
struct Codes {
  static constexpr int KS = (DT + 3) / 4;
  v4i kf[KS][4], vf[DT];
  int koff[KS], voff, HP;
  __device__ __forceinline__ Codes(int HP, int lane) : HP(HP) {
    const int col = lane & 15, quad = lane >> 4;
#pragma unroll
    for (int st = 0; st < KS; st++) koff[st] = col * HP + 16 * min(4 * st + quad, HP / 16 - 1);  // behind the row q's digits are 0
    voff = col * kKeys + 16 * quad;
  }
  __device__ __forceinline__ void keys(const int8_t *k8, size_t at) {
    const int8_t *p = k8 + at * kKeys * HP;
#pragma unroll
    for (int kt = 0; kt < 4; kt++)
#pragma unroll
      for (int st = 0; st < KS; st++) kf[st][kt] = *reinterpret_cast<const v4i *>(p + kt * 16 * HP + koff[st]);
  }
  // kOnce: no other wavefront loads them, and they pass the caches by (24 conversations of one token 62 us, else 70; of 32
  // rows, of which two wavefronts take each block, 32, and past the caches 33. Keys past the caches: 41, for a block's 64
  // bytes of a row are half of what a load brings).
  template <bool kOnce>
  __device__ __forceinline__ void values(const int8_t *v8, size_t at) {
    const int8_t *p = v8 + at * kKeys * HP;
#pragma unroll
    for (int t = 0; t < DT; t++) {
      const v4i *x = reinterpret_cast<const v4i *>(p + min(t, HP / 16 - 1) * 16 * kKeys + voff);
      vf[t] = kOnce ? __builtin_nontemporal_load(x) : *x;
    }
  }
};

// A 4 x 4 transposition of bytes: the words' bytes 0, then 1, 2 and 3.
__device__ __forceinline__ v4i turn4(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  const uint32_t t0 = __builtin_amdgcn_perm(b, a, 0x05010400u), t1 = __builtin_amdgcn_perm(b, a, 0x07030602u);
  const uint32_t t2 = __builtin_amdgcn_perm(d, c, 0x05010400u), t3 = __builtin_amdgcn_perm(d, c, 0x07030602u);
  return v4i{(int)__builtin_amdgcn_perm(t2, t0, 0x05040100u), (int)__builtin_amdgcn_perm(t2, t0, 0x07060302u),
             (int)__builtin_amdgcn_perm(t3, t1, 0x05040100u), (int)__builtin_amdgcn_perm(t3, t1, 0x07060302u)};
}

// The first n of four floats.
__device__ __forceinline__ void put4(float *p, float4 y, int n) {
  if (n >= 4) {
    st4(p, y);
  } else if (n > 0) {
    p[0] = y.x;
    if (n > 1) p[1] = y.y;
    if (n > 2) p[2] = y.z;
  }
}

// Where a row's results go: of this part of the key axis, or of the whole.
struct Place8 {
  float *o, *lse;
  float2 *ml, *stat;
  // whole: no other part has keys of the row, number r of the group
  __device__ __forceinline__ Place8(float *out, float *lse_, const Parts8 &parts, const ugk_cache8 &a, int slot, bool whole, int r,
                                    size_t row, int h) {
    const size_t at = row * a.NH + h, p = (size_t)slot * parts.rows + r;
    o = whole ? out + row * a.ldo + (size_t)h * a.HS : parts.o + p * part_floats(a.HS);
    ml = whole ? nullptr : parts.ml + p;
    lse = whole && lse_ ? lse_ + at : nullptr;
    stat = whole && parts.stat ? parts.stat + at : nullptr;
  }
  __device__ __forceinline__ void put(float top, float sum) const {
    if (ml) *ml = make_float2(top, sum);
    if (lse) *lse = sum == 0.0f ? -INFINITY : (top + __builtin_amdgcn_logf(sum)) * kLn28;
    if (stat) *stat = make_float2(top, sum);
  }
};

// A wavefront's blocks from the first, `by` apart, with what the next one needs on its way: the keys from where the
// scores are computed, the values from where the output is, the table a turn before.
struct Walk {
  int j, stop, by, id, next;  // next: what the table says of j + by
  __device__ __forceinline__ Walk(const ugk_cache8 &a, int b, int first, int stop, int by, int *word) : j(first), stop(stop), by(by) {
    id = next = 0;
    if (j < stop) {
      const int t = table_at(a, b, j);
      next = table_at(a, b, min(j + by, stop - 1));
      id = checked_block(a, t, word, UGK_IDS_CACHE8_ATTENTION);
    }
  }
  __device__ __forceinline__ bool there() const { return id >= 0; }
  __device__ __forceinline__ bool more() const { return j + by < stop; }
  // The next block, while this one is computed; the table's word on the one behind it is on its way then.
  __device__ __forceinline__ int ahead(const ugk_cache8 &a, int b, int *word) {
    const int i = checked_block(a, __builtin_amdgcn_readfirstlane(next), word, UGK_IDS_CACHE8_ATTENTION);
    next = table_at(a, b, min(j + 2 * by, stop - 1));
    return i;
  }
  __device__ __forceinline__ void step(int i) {
    j += by;
    id = i;
  }
};
__device__ __forceinline__ size_t block_head(int id, int NKV, int hk) { return (size_t)max(id, 0) * NKV + hk; }

// What a workgroup has at a time: of group `group` of R rows of a sequence and key/value head blocks [first, stop).
struct Job8 {
  Seq8 s;
  int b, hk, group, rows, first, stop, slot;
  bool whole;  // all blocks
};
// Blocks that a row at position i sees.
__device__ __forceinline__ int blocks_at(const Seq8 &s, const ugk_cache8 &a, int i) { return (s.seen(i, a.causal) + kKeys - 1) / kKeys; }
// The parts of nb blocks, of at most `chunk` each and as equal as they can be.
__device__ __forceinline__ int parts_for(int nb, int chunk) { return max(1, (nb + chunk - 1) / chunk); }

// The workgroup's jobs, one after another.
//
// Shared: the blocks of all sequences, groups (the last rows first) and key/value heads are one long row, from what the
// sequences really hold, of which every workgroup has the same share: it may begin and end within a job. Equal shares are
// what counts, for the CUs' time is their matrix and vector units' or their part of the memory's, and a CU that holds two
// workgroups is done no sooner than one that holds one of twice their blocks. (Parts of each job alone, about as many as the
// CUs hold: prompts behind long conversations, 16/4 heads of 128, 74 us, not 61; drafts 37, not 32.) A job's beginning (its
// rows, their results) counts as kBegin blocks: 6 of k_cache8_rows (4: 5% slower where a workgroup has some 20 blocks), 2 of
// tiles (1 and 3: 3%). Every wavefront finds its place alike, a lane to a sequence, then to a group, 2.7 us in all. Else
// workgroups are of pairs, groups (the longest first) and parts in turn.
template <int R, int kBegin, bool kShared>
struct Jobs {
  // the lane's sequence, its groups and their units: blocks, and kBegin of each (a group without a block has one: its rows'
  // results are written, too)
  struct Held {
    Seq8 s;
    int n, units;
  };
  const ugk_cache8 &a;
  const Parts8 &parts;
  const unsigned pairs, groups;
  const int G, lane;
  int *const word;
  int at, end, share, j;  // units; the number of the job
  bool whole;             // workgroups have whole groups

  __device__ __forceinline__ Jobs(const ugk_cache8 &a, const Parts8 &parts, unsigned pairs, unsigned groups, int *word)
      : a(a), parts(parts), pairs(pairs), groups(groups), G(a.NH / a.NKV), lane(threadIdx.x & (kWave - 1)), word(word), at(0), end(1), share(1),
        j(0), whole(false) {}
  __device__ __forceinline__ int blocks_of(const Seq8 &s, int t) const {  // its last row sees most
    const int row = min((t + 1) * R, s.Lq * G) - 1;
    return blocks_at(s, a, parts.inverse ? (int)__umulhi((unsigned)row, parts.inverse) : row);
  }
  __device__ __forceinline__ int units(int nb) const { return whole ? 1 : kBegin + max(nb, 1); }
  __device__ __forceinline__ Held held(int b, bool tell, int *longest) const {
    constexpr int kOwn = 64;  // groups that a lane adds up by itself; of sequences of more all lanes do
    Held h{{0, 0, 0}, 0, 0};
    if (b < a.nseq) {
      h.s = sequence8(a, b, tell, word, UGK_IDS_CACHE8_ATTENTION);
      h.n = (h.s.Lq * G + R - 1) / R;
    }
    if (whole) {
      h.units = h.n;
      return h;
    }
    for (int t = 0; t < h.n && h.n <= kOwn; t++) {
      const int nb = blocks_of(h.s, t);
      h.units += kBegin + max(nb, 1);
      *longest = max(*longest, nb);
    }
    for (uint64_t many = __ballot(h.n > kOwn); many; many &= many - 1) {
      const int l = __builtin_ctzll(many), n = __builtin_amdgcn_readlane(h.n, l);
      const Seq8 s{__builtin_amdgcn_readlane(h.s.q0, l), __builtin_amdgcn_readlane(h.s.Lq, l), __builtin_amdgcn_readlane(h.s.Lk, l)};
      int sum = 0;
      for (int t = lane; t < n; t += kWave) {
        const int nb = blocks_of(s, t);
        sum += kBegin + max(nb, 1);
        *longest = max(*longest, nb);
      }
      sum = last_lane(wave_scan(sum));
      if (lane == l) h.units = sum;
    }
    return h;
  }

  // The first job; false: none.
  __device__ __forceinline__ bool first(Job8 &w) {
    if (!kShared) return only(w);
    Held h{{0, 0, 0}, 0, 0}, one = h;  // the first 64 sequences', which are mostly all
    int all = 0, jobs = 0, longest = 0;
    for (int b0 = 0; b0 < a.nseq; b0 += kWave) {
      h = held(b0 + lane, blockIdx.x == 0, &longest);
      jobs += h.n;
      all += h.units;
      if (b0 == 0) one = h;
    }
    longest = (int)wave_max_bits((uint32_t)longest);
    jobs = last_lane(wave_scan(jobs)) * a.NKV;
    all = last_lane(wave_scan(all)) * a.NKV;
    // no group has much more than a CU's share: the parts' way through memory would cost more than they save
    whole = (long long)2 * longest * parts.cus <= 3LL * (all - kBegin * jobs);
    share = whole ? 1 : max(parts.least, (all + parts.wgs - 1) / parts.wgs);
    const bool over = jobs > parts.most;  // rows in more than one sequence: there is no place for so many
    if (blockIdx.x == 0 && threadIdx.x == 0) {
      *parts.told = over ? 0 : jobs;
      if (over) *word = UGK_IDS_CACHE8_ATTENTION;
    }
    all = __builtin_amdgcn_readfirstlane(over ? 0 : whole ? jobs : all);  // (or the job, and 25 more registers, are per lane)
    end = (int)min((long long)(blockIdx.x + 1) * share, (long long)all);
    at = (int)min((long long)blockIdx.x * share, (long long)all);
    if (at >= end) return false;
    if (whole) one.units = one.n;

    int x = at, n = 0;
    for (int b0 = 0; b0 < a.nseq; b0 += kWave) {
      h = b0 ? held(b0 + lane, false, &longest) : one;
      const int to = wave_scan(h.units) * a.NKV, before = wave_scan(h.n);
      const uint64_t over = __ballot(to > x);
      if (over) {
        const int l = __builtin_ctzll(over);
        n = __builtin_amdgcn_readlane(h.n, l);
        x -= __builtin_amdgcn_readlane(to - h.units * a.NKV, l);
        j += __builtin_amdgcn_readlane(before, l) - n;
        w.b = b0 + l;
        w.s.q0 = __builtin_amdgcn_readlane(h.s.q0, l);
        w.s.Lq = __builtin_amdgcn_readlane(h.s.Lq, l);
        w.s.Lk = __builtin_amdgcn_readlane(h.s.Lk, l);
        break;
      }
      x -= last_lane(to);
      j += last_lane(before);
    }
    w.group = 0;
    for (int t0 = 0; t0 < n; t0 += kWave) {
      const int t = n - 1 - t0 - lane, mine = t < 0 ? 0 : units(blocks_of(w.s, t)) * a.NKV, to = wave_scan(mine);
      const uint64_t over = __ballot(to > x);
      if (over) {
        const int l = __builtin_ctzll(over);
        x -= __builtin_amdgcn_readlane(to - mine, l);
        w.group = n - 1 - t0 - l;
        break;
      }
      x -= last_lane(to);
    }
    const int u = units(blocks_of(w.s, w.group));
    w.hk = x / u;
    j = (j + n - 1 - w.group) * a.NKV + w.hk;
    return take(w, x % u);
  }
  // The one behind w; false: none.
  __device__ __forceinline__ bool next(Job8 &w) {
    if (!kShared || at >= end) return false;
    j++;
    if (++w.hk == a.NKV) {
      w.hk = 0;
      if (--w.group < 0) {
        // the next sequence that has rows: a lane to each, for many may have none
        for (uint64_t some = 0; !some;) {
          if (++w.b >= a.nseq) return false;
          Seq8 s{0, 0, 0};
          if (w.b + lane < a.nseq) s = sequence8(a, w.b + lane, false, word, 0);
          some = __ballot(s.Lq > 0);
          const int l = some ? __builtin_ctzll(some) : kWave - 1;
          w.b += l;
          w.s.q0 = __builtin_amdgcn_readlane(s.q0, l);
          w.s.Lq = __builtin_amdgcn_readlane(s.Lq, l);
          w.s.Lk = __builtin_amdgcn_readlane(s.Lk, l);
        }
        w.group = (w.s.Lq * G + R - 1) / R - 1;
      }
    }
    return take(w, 0);
  }
  // This workgroup's blocks of job w, of which `at` is unit `off`; false: it has only of the job's beginning.
  __device__ __forceinline__ bool take(Job8 &w, int off) {
    const int nb = blocks_of(w.s, w.group), begin = whole ? 0 : kBegin, u = units(nb), stop = min(off + end - at, u) - begin;
    w.rows = w.s.Lq * G;
    w.first = max(off - begin, 0);
    if (stop <= w.first) return false;
    w.whole = w.first == 0 && stop == u - begin;
    w.slot = blockIdx.x + (parts.step == 1 ? j : (int)blockIdx.x + (at != (int)blockIdx.x * share));
    if (w.first == 0) tell(w, whole ? 1 : (at - off + u - 1) / share - (int)blockIdx.x + 1);
    w.stop = whole ? nb : min(stop, nb);
    at += u - off;
    return true;
  }
  __device__ __forceinline__ void tell(const Job8 &w, int n) const {
    if (!parts.told || threadIdx.x) return;
    const size_t at = ((size_t)w.b * a.NKV + w.hk) * groups + w.group;
    int4 *to = reinterpret_cast<int4 *>(parts.told + 4) + 2 * (kShared ? (size_t)j : at);
    to[0] = make_int4(w.s.q0, w.rows, w.hk, w.group);
    to[1] = make_int4(w.slot, n, 0, 0);
    if (kShared && parts.block) reinterpret_cast<int2 *>(parts.told + 4 + 8 * (size_t)parts.most)[at] = make_int2(w.slot, n);
  }
  __device__ __forceinline__ bool only(Job8 &w) {
    // Each CU gets one workgroup of every `cus`: of the first the longest, of the second the shortest first, and so on, so
    // that all have much the same to do (8 x 1,024 rows of 12 heads of 64: 46 us, and 49 with the longest first throughout).
    unsigned x = blockIdx.x;
    const unsigned cus = (unsigned)parts.cus, lap = x / cus;
    if (lap % 2 && (lap + 1) * cus <= gridDim.x) x = lap * cus + (cus - 1 - x % cus);
    const unsigned round = x / pairs, pair = (x % pairs + round) % pairs;
    w.b = pair / a.NKV;
    w.hk = pair % a.NKV;
    w.group = groups - 1 - round % groups;
    w.s = sequence8(a, w.b, w.hk == 0 && round == 0, word, UGK_IDS_CACHE8_ATTENTION);
    w.rows = w.s.Lq * G;
    const int part = round / groups;
    if (w.group * R >= w.rows) {
      if (part == 0) tell(w, 0);
      return false;
    }
    const int nb = blocks_at(w.s, a, (min((w.group + 1) * R, w.rows) - 1) / G);
    const int n = parts.o ? parts_for(nb, parts.least) : 1;
    if (part >= n) return false;
    const int each = nb / n, longer = nb - each * n;  // the first ones are one longer
    w.whole = n == 1;
    w.first = part * each + min(part, longer);
    w.stop = w.first + each + (part < longer);
    w.slot = (int)((pair * groups + w.group) * parts.splits) + part;
    if (part == 0) tell(w, n);
    return true;
  }
};

// ---- up to 32 rows (query rows times heads of the group) at a time ----
//
// A row of q is held as whole numbers of 31 bits next to its largest element, and those as four digits of base 256; its
// products with the codes are exact on the 8-bit matrix units, and so are the weights', 31 bits next to the block's
// largest, with the values' codes. So no code is converted, and a score is rounded where its digits' sums are added up.
// What all rows of a wavefront need of a call and a block.
struct Block8 {
  const ugk_cache8 &a;
  const Parts8 &parts;
  const Job8 &job;
  int lane, j;
  bool there;
  float kscale, vexp;
  // where the block's m and l of a row go
  __device__ __forceinline__ float2 *stat(int row) const {
    return parts.block + (((size_t)job.b * a.NKV + job.hk) * a.max_q * (a.NH / a.NKV) + row) * parts.ld + j;
  }
};

// Four rows: their four digits are one operand of 16 rows, so that a block's scores take two instructions per 16 keys at 128
// floats per head, and a lane finds the four digits of its score in its own four registers. A lane has a score of row lane /
// 16 for each 16 keys.
template <int DT>
struct Four {
  static constexpr int KS = (DT + 3) / 4, kStride = 20, kLds = 16 * kStride;  // kLds words of LDS per wavefront
  using Scores = float[4];
  using Weights = v4i;
  v4i aq[KS];
  int row, lim, ex;
  bool nan;
  Running run;
  float o[DT];

  // Rows from row0 on. Lane (4 row + digit, quad) holds dims 64 step + 16 quad + [0, 16) of q.
  __device__ __forceinline__ void load(const float *q, const ugk_cache8 &a, const Job8 &job, int row0, int lane) {
    const int col = lane & 15, quad = lane >> 4, G = a.NH / a.NKV, rr = min(row0 + (col >> 2), job.rows - 1);
    const float *p = q + ((size_t)job.s.q0 + rr / G) * a.ldq + (size_t)(job.hk * G + rr % G) * a.HS;
    float x[KS][16];
    uint32_t most = load_q(p, 16 * quad, 64, a, x);
    most = max(most, (uint32_t)__shfl_xor((int)most, 16));
    most = max(most, (uint32_t)__shfl_xor((int)most, 32));
    const int e = (int)(most >> 23) - 127;  // below 2^(e + 1)
#pragma unroll
    for (int st = 0; st < KS; st++) {
      aq[st] = v4i{0, 0, 0, 0};
#pragma unroll
      for (int d = 0; d < 16; d++) {
        const uint32_t y = digits(whole(x[st][d], 29 - e));
        aq[st][d / 4] |= (int)((y >> (8 * (lane & 3)) & 255u) << (8 * (d & 3)));
      }
    }
    // for the lanes that hold the row's scores: row quad
    ex = __shfl(e, 4 * quad) - 29;
    nan = (uint32_t)__shfl((int)most, 4 * quad) >= kInfBits;
    row = row0 + quad;
    lim = row < job.rows ? job.s.seen(row / G, a.causal) : 0;
#pragma unroll
    for (int t = 0; t < DT; t++) o[t] = 0.0f;
  }
  // The scores' products; the largest.
  __device__ __forceinline__ float products(const Codes<DT> &c, const Block8 &k, Scores &p) const {
    const int seen = k.there ? lim - k.j * kKeys : 0, col = k.lane & 15;  // of this block's keys
    float mb = -INFINITY;
#pragma unroll
    for (int kt = 0; kt < 4; kt++) {
      v4i acc = {0, 0, 0, 0};
#pragma unroll
      for (int st = 0; st < KS; st++) acc = __builtin_amdgcn_mfma_i32_16x16x64_i8(aq[st], c.kf[st][kt], acc, 0, 0, 0);
      p[kt] = kt * 16 + col < seen ? undigits(acc) : -INFINITY;
      mb = fmaxf(mb, p[kt]);
    }
    return mb;
  }
  // The weights as an operand.
  __device__ __forceinline__ void weights(Scores &p, float mb, const Block8 &k, uint32_t *lp, Weights &ap, float &fo, float &fb) {
    const int col = k.lane & 15, quad = k.lane >> 4;
    // a number where the row sees nothing: the result of one without any key is 0 whatever it holds
    const float most = max16(mb), fac = here(nan && most != -INFINITY ? NAN : score_factor(k.parts, k.kscale, ex));
    mb = top_score(most, fac);
    float less = less_top(mb, 0.0f);
    if (__any(far_score(mb))) {
      const float off = here(far_score(mb) ? most : 0.0f);
      less = here(far_score(mb) ? 0.0f : less);
#pragma unroll
      for (int kt = 0; kt < 4; kt++) p[kt] -= off;
    }
    uint32_t y[4];
    float lb = 0.0f;
#pragma unroll
    for (int kt = 0; kt < 4; kt++) {
      p[kt] = ex2(fmaf(p[kt], fac, less));
      lb += p[kt];
      y[kt] = digits((int)(p[kt] * 0x1p30f));  // (2^30 in the exponent would cost the weights four bits)
    }
    const v4i t = turn4(y[0], y[1], y[2], y[3]);  // the four keys' digits side by side: a word per digit
    uint32_t *w = lp + 4 * quad * kStride + col;
#pragma unroll
    for (int d = 0; d < 4; d++) w[d * kStride] = (uint32_t)t[d];
    __builtin_amdgcn_wave_barrier();
    ap = *reinterpret_cast<const v4i *>(lp + col * kStride + 4 * quad);
    __builtin_amdgcn_wave_barrier();
    if (k.parts.block) {
      const float sum = sum16(lb);
      if (col == 0 && row < k.job.rows) *k.stat(row) = make_float2(mb, sum);
    }
    run.sum(mb, lb, mb, 0.0f);
    fo = run.stand(mb, k.vexp);
    fb = run.factor(mb, k.vexp);
  }
  __device__ __forceinline__ void add(const Codes<DT> &c, const Weights &ap, float fo, float fb) {
#pragma unroll
    for (int t = 0; t < DT; t++) {
      const v4i acc = __builtin_amdgcn_mfma_i32_16x16x64_i8(ap, c.vf[t], v4i{0, 0, 0, 0}, 0, 0, 0);
      o[t] = here(fmaf(undigits(acc), fb, o[t] * fo));
    }
  }
  // Outputs, maxima and sums to LDS.
  __device__ __forceinline__ void put(float *lo, int stride, float *lm, float *ll, int lane) const {
    const int col = lane & 15, quad = lane >> 4;
    const float sum = sum16(run.l);
    int e;
    const float g = run.last(sum, &e);
    e -= 30;  // of the weights' whole numbers
#pragma unroll
    for (int t = 0; t < DT; t++) lo[quad * stride + 16 * t + col] = __builtin_amdgcn_ldexpf(o[t] * g, e);
    if (col == 0) {
      lm[quad] = run.m;
      ll[quad] = sum;
    }
  }
};

// x of the lanes that hold the same row in the four quarters of a wavefront, combined.
__device__ __forceinline__ float quarters_max(float x) {
  const auto s = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return half_max(fmaxf(__uint_as_float(s[0]), __uint_as_float(s[1])));
}
__device__ __forceinline__ float quarters_sum(float x) {
  const auto s = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return half_sum(__uint_as_float(s[0]) + __uint_as_float(s[1]));
}

// Sixteen rows: the same products transposed, with an operand per digit. A lane holds 16 scores of one row, lane % 16, and
// its weights are the second product's operand as they stand, for a column of the values' codes has its keys in the order in
// which the lanes hold them.
template <int DT>
struct Sixteen {
  static constexpr int KS = (DT + 3) / 4, kLds = 4;  // (none)
  using Scores = float[4][4];
  using Weights = v4i[4];
  v4i aq[KS][4];
  int row, lim, least, ex;  // least: what the first row sees
  bool nan;
  Running run;
  float o[DT][4];

  __device__ __forceinline__ void load(const float *q, const ugk_cache8 &a, const Job8 &job, int row0, int lane) {
    const int quad = lane >> 4, G = a.NH / a.NKV;
    row = row0 + (lane & 15);
    lim = row < job.rows ? job.s.seen(row / G, a.causal) : 0;
    least = job.s.seen(min(row0, job.rows - 1) / G, a.causal);
    const int rr = min(row, job.rows - 1);
    const float *p = q + ((size_t)job.s.q0 + rr / G) * a.ldq + (size_t)(job.hk * G + rr % G) * a.HS;
    float x[KS][16];
    uint32_t most = load_q(p, 16 * quad, 64, a, x);
    most = max(most, (uint32_t)__shfl_xor((int)most, 16));
    most = max(most, (uint32_t)__shfl_xor((int)most, 32));
    nan = most >= kInfBits;
    ex = (int)(most >> 23) - 127 - 29;
#pragma unroll
    for (int st = 0; st < KS; st++)
#pragma unroll
      for (int d = 0; d < 16; d += 4) {
        uint32_t y[4];
#pragma unroll
        for (int r = 0; r < 4; r++) y[r] = digits(whole(x[st][d + r], -ex));
        const v4i t = turn4(y[0], y[1], y[2], y[3]);
#pragma unroll
        for (int r = 0; r < 4; r++) aq[st][r][d / 4] = t[r];
      }
#pragma unroll
    for (int t = 0; t < DT; t++)
#pragma unroll
      for (int r = 0; r < 4; r++) o[t][r] = 0.0f;
  }
  __device__ __forceinline__ float products(const Codes<DT> &c, const Block8 &k, Scores &p) const {
    float mb = -INFINITY;
#pragma unroll
    for (int kt = 0; kt < 4; kt++) {
      __builtin_amdgcn_sched_barrier(0);  // tile by tile: the registers hold one tile's digits
      v4i acc[4];
#pragma unroll
      for (int d = 0; d < 4; d++) {
        acc[d] = v4i{0, 0, 0, 0};
#pragma unroll
        for (int st = 0; st < KS; st++) acc[d] = __builtin_amdgcn_mfma_i32_16x16x64_i8(c.kf[st][kt], aq[st][d], acc[d], 0, 0, 0);
      }
#pragma unroll
      for (int r = 0; r < 4; r++) p[kt][r] = here(undigits(v4i{acc[0][r], acc[1][r], acc[2][r], acc[3][r]}));
    }
    if (!k.there || (k.j + 1) * kKeys > least) {
      const int n = here(k.there ? lim - k.j * kKeys - 4 * (k.lane >> 4) : 0);  // seen of this block's keys from the lane's first on
#pragma unroll
      for (int kt = 0; kt < 4; kt++)
#pragma unroll
        for (int r = 0; r < 4; r++) p[kt][r] = kt * 16 + r < n ? p[kt][r] : -INFINITY;
    }
#pragma unroll
    for (int kt = 0; kt < 4; kt++)
#pragma unroll
      for (int r = 0; r < 4; r++) mb = fmaxf(mb, p[kt][r]);
    return mb;
  }
  __device__ __forceinline__ void weights(Scores &p, float mb, const Block8 &k, uint32_t *, Weights &bp, float &fo, float &fb) {
    const float most = quarters_max(mb), fac = here(nan && most != -INFINITY ? NAN : score_factor(k.parts, k.kscale, ex));
    mb = top_score(most, fac);
    float less = less_top(mb, 0.0f);
    if (__any(far_score(mb))) {
      const float off = here(far_score(mb) ? most : 0.0f);
      less = here(far_score(mb) ? 0.0f : less);
#pragma unroll
      for (int kt = 0; kt < 4; kt++)
#pragma unroll
        for (int r = 0; r < 4; r++) p[kt][r] -= off;
    }
    float lb = 0.0f;
#pragma unroll
    for (int r = 0; r < 4; r++) {
      uint32_t y[4];
#pragma unroll
      for (int kt = 0; kt < 4; kt++) {
        const float x = ex2(fmaf(p[kt][r], fac, less));
        lb += x;
        y[kt] = digits((int)(x * 0x1p30f));
      }
      const v4i t = turn4(y[0], y[1], y[2], y[3]);
#pragma unroll
      for (int d = 0; d < 4; d++) bp[d][r] = t[d];
    }
    if (k.parts.block) {
      const float sum = quarters_sum(lb);
      if (k.lane < 16 && row < k.job.rows) *k.stat(row) = make_float2(mb, sum);
    }
    run.sum(mb, lb, mb, 0.0f);
    fo = run.stand(mb, k.vexp);
    fb = run.factor(mb, k.vexp);
  }
  __device__ __forceinline__ void add(const Codes<DT> &c, const Weights &bp, float fo, float fb) {
#pragma unroll
    for (int t = 0; t < DT; t++) {
      if (t % 2 == 0) __builtin_amdgcn_sched_barrier(0);
      v4i acc[4];
#pragma unroll
      for (int d = 0; d < 4; d++) acc[d] = __builtin_amdgcn_mfma_i32_16x16x64_i8(c.vf[t], bp[d], v4i{0, 0, 0, 0}, 0, 0, 0);
#pragma unroll
      for (int r = 0; r < 4; r++) o[t][r] = here(fmaf(undigits(v4i{acc[0][r], acc[1][r], acc[2][r], acc[3][r]}), fb, o[t][r] * fo));
    }
  }
  __device__ __forceinline__ void put(float *lo, int stride, float *lm, float *ll, int lane) const {
    const int col = lane & 15, quad = lane >> 4;
    const float sum = quarters_sum(run.l);
    int e;
    const float g = run.last(sum, &e);
    e -= 30;  // of the weights' whole numbers
#pragma unroll
    for (int t = 0; t < DT; t++)
      *reinterpret_cast<float4 *>(&lo[col * stride + 16 * t + 4 * quad]) =
          make_float4(__builtin_amdgcn_ldexpf(o[t][0] * g, e), __builtin_amdgcn_ldexpf(o[t][1] * g, e),
                      __builtin_amdgcn_ldexpf(o[t][2] * g, e), __builtin_amdgcn_ldexpf(o[t][3] * g, e));
    if (quad == 0) {
      lm[col] = run.m;
      ll[col] = sum;
    }
  }
};

// Up to R rows: a token's, drafts, large groups, an observation window (in `groups` of them). The wavefronts share the blocks,
// and a wavefront has all rows, 4 or 16. Of 32 it has half, and two take the same blocks, the second from a cache. Keys are
// loaded into the registers that the scores have left, values into those that the output has, while the other half of the
// block is computed.
//
// Four rows are bound by memory: 346 MB of 24 conversations in 62 us, 5.5 TB/s, with three wavefronts on a SIMD (two:
// 70 us). Sixteen are bound by the digits' vector instructions, four of five of a block's, beside the loads: 86 MB of 16
// conversations, 20 rows each, 32 us. (20 rows as 16 and 4 of the same wavefront: 38 us, for it has all blocks' time in a
// row.) What is left of short calls is the way there: 16 x 12 heads of 64, up to 16 blocks each, 8.8 us, of which the
// blocks take 1.2.
template <int DT, int R>
__device__ __forceinline__ void rows_job(float *out, float *lse, const float *q, const int8_t *k8, const float *ks, const int8_t *v8,
                                         const float *vs, const ugk_cache8 &a, const Parts8 &parts, const Job8 &job, int *word) {
  using Rows = std::conditional_t<R == 4, Four<DT>, Sixteen<DT>>;
  constexpr int kRow = 16 * DT + 4, kRows = R == 4 ? 4 : 16, KW = R == 32 ? 2 : kFewWaves;
  __shared__ alignas(16) float lo[kFewWaves][kRows * kRow];
  __shared__ float lm[kFewWaves][kRows], ll[kFewWaves][kRows];
  __shared__ alignas(16) uint32_t lp[kFewWaves][Rows::kLds];
  const int thread = here((int)threadIdx.x);  // what is computed from it is not kept from job to job
  const int lane = thread & (kWave - 1), wave = __builtin_amdgcn_readfirstlane(thread >> 6);
  const int stop = job.stop, row0 = job.group * R, hk = job.hk;

  Codes<DT> c(padded(a.HS), lane);
  Walk walk(a, job.b, job.first + wave % KW, stop, KW, word);
  float kscale = 0.0f, vscale = 0.0f;
  if (walk.j < stop) {
    const size_t at = block_head(walk.id, a.NKV, hk);
    c.keys(k8, at);
    c.template values<R != 32>(v8, at);
    kscale = ks[at];
    vscale = vs[at];
  }
  Rows rows;
  rows.load(q, a, job, row0 + wave / KW * 16, lane);

  const auto block = [&](auto next) {  // next: another block follows
    constexpr bool kNext = decltype(next)::value;
    const int id = kNext ? walk.ahead(a, job.b, word) : 0;
    const size_t ahead = block_head(id, a.NKV, hk);
    const Block8 k{a, parts, job, lane, walk.j, walk.there(), kscale, exponent(vscale)};
    typename Rows::Scores p;
    typename Rows::Weights w;
    float fo, fb;
    const float mb = rows.products(c, k, p);
    __builtin_amdgcn_sched_barrier(0);  // into the registers that the products have read
    if (kNext) {
      c.keys(k8, ahead);
      kscale = ks[ahead];
      vscale = vs[ahead];
    }
    rows.weights(p, mb, k, lp[wave], w, fo, fb);
    rows.add(c, w, fo, fb);
    __builtin_amdgcn_sched_barrier(0);
    if (kNext) c.template values<R != 32>(v8, ahead);
    if (kNext) walk.step(id);
  };
  while (walk.more()) block(std::true_type{});
  if (walk.j < stop) block(std::false_type{});

  rows.put(lo[wave], kRow, lm[wave], ll[wave], lane);
  __syncthreads();
  // a row's sums of the wavefronts that have it; 16 lanes to a row, or a wavefront
  constexpr int kLanes = R == 4 ? kWave : 16, kAtOnce = kWave / kLanes;
  const int G = a.NH / a.NKV, d0 = 4 * (lane & (kLanes - 1));
  for (int n0 = kAtOnce * wave; n0 < R; n0 += kAtOnce * kFewWaves) {
    const int n = n0 + lane / kLanes, r = n % kRows, w0 = n / kRows * KW, row = row0 + n;
    if (row >= job.rows) break;
    float top = -INFINITY, total = 0.0f, wt[KW];
#pragma unroll
    for (int w = 0; w < KW; w++) top = fmaxf(top, lm[w0 + w][r]);
#pragma unroll
    for (int w = 0; w < KW; w++) {
      wt[w] = ll[w0 + w][r] == 0.0f ? 0.0f : ll[w0 + w][r] * ex2(lm[w0 + w][r] - or0(top));
      total += wt[w];
    }
    const int i = parts.inverse ? (int)__umulhi((unsigned)row, parts.inverse) : row;
    const Place8 to(out, lse, parts, a, job.slot, job.whole, n, (size_t)job.s.q0 + i, hk * G + row - i * G);
    const float inv = total == 0.0f ? 0.0f : 1.0f / total;
#pragma unroll
    for (int d = d0; d < 16 * DT; d += 4 * kLanes) {
      float4 y = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
      for (int w = 0; w < KW; w++) {
        const float4 z = ld4(&lo[w0 + w][r * kRow + d]);
        const float f = wt[w] * inv;
        y = make_float4(fmaf(f, z.x, y.x), fmaf(f, z.y, y.y), fmaf(f, z.z, y.z), fmaf(f, z.w, y.w));
      }
      put4(to.o + d, y, a.HS - d);
    }
    if (d0 == 0) to.put(top, total);
  }
}

template <int DT, int R, bool kShared>
__global__ __launch_bounds__(kFewWaves *kWave, R > 4 ? 2 : DT >= 6 ? 3 : 4) void k_cache8_rows(
    float *out, float *lse, const float *q, const int8_t *k8, const float *ks, const int8_t *v8, const float *vs, ugk_cache8 a, Parts8 parts,
    unsigned pairs, unsigned groups, int *word) {
  Jobs<R, 6, kShared> jobs(a, parts, pairs, groups, word);
  Job8 job;
  for (bool more = jobs.first(job); more; more = jobs.next(job)) {
    rows_job<DT, R>(out, lse, q, k8, ks, v8, vs, a, parts, job, word);
    __syncthreads();  // LDS is read until here
  }
}

// What m and l of the n parts of row r of a group say of the whole.
__device__ __forceinline__ float2 joined(const Parts8 &parts, int first, int n, int r) {
  float m = -INFINITY, l = 0.0f;
  for (int p0 = 0; p0 < n; p0 += 4) {
    float2 x[4];
    float top = m;
#pragma unroll
    for (int u = 0; u < 4; u++) {
      x[u] = parts.ml[part_row(parts, first, min(p0 + u, n - 1), r)];
      if (p0 + u >= n) x[u].y = 0.0f;
    }
#pragma unroll
    for (int u = 0; u < 4; u++) top = fmaxf(top, x[u].y == 0.0f ? -INFINITY : x[u].x);
    l *= ex2(m - or0(top));
    m = top;
#pragma unroll
    for (int u = 0; u < 4; u++) l += x[u].y == 0.0f ? 0.0f : x[u].y * ex2(x[u].x - or0(top));
  }
  return make_float2(m, l);
}

constexpr int kJoinRows8 = 2 * kBlock / kWave;  // rows that a workgroup joins

// Behind the attention, workgroups of two kinds. The first `joins` join the parts of a split key axis, half a wavefront per
// row and head, in the parts' order, where a group of `rows` rows had more than one. The others add up the weights of 16
// blocks of a sequence, 16 threads to each, which take every sixteenth row and head, in a fixed order:
// weight[b, j] += sum of l_j 2^(m_j - m) / l. Two launches in one: 4 to 6 us of rows that are a token's or drafts, a launch and
// three dependent loads; 9 us of prompts behind long conversations (35 MB of parts).
__global__ __launch_bounds__(kBlock) void k_cache8_finish(float *out, float *lse, float *weight, Parts8 parts, ugk_cache8 a, int rows,
                                                         int groups, int per_job, unsigned joins) {
  constexpr int kAtOnce = 4;  // of blocks
  const int G = a.NH / a.NKV;
  if (blockIdx.x >= joins) {
    __shared__ float part[16][17];
    __shared__ float2 whole[kBlock];
    __shared__ size_t from[kBlock];
    __shared__ int end[kBlock];
    const unsigned x = blockIdx.x - joins;
    const int of = (parts.ld + 15) / 16, b = x / of, j = x % of * 16 + (threadIdx.x & 15), slice = threadIdx.x >> 4;
    const Seq8 s = sequence8(a, b, false, nullptr, 0);
    const int nb = (s.Lk + kKeys - 1) / kKeys, n = s.Lq * G;
    if (x % of * 16 >= nb || (parts.wgs && *parts.told == 0)) return;
    float sum = 0.0f;
    for (int y0 = 0; y0 < n * a.NKV; y0 += kBlock) {  // a row and head per thread, then a block per thread
      const int mine = y0 + (int)threadIdx.x;
      if (mine < n * a.NKV) {
        const int hk = mine / n, rr = mine % n;
        int2 job = make_int2(0, 1);
        if (parts.told) {
          const size_t at = ((size_t)b * a.NKV + hk) * groups + rr / rows;
          const int *t = parts.told + 4 + (parts.wgs ? 8 * (size_t)parts.most + 2 * at : 8 * at + 4);
          job = make_int2(t[0], t[1]);
        }
        from[threadIdx.x] = (((size_t)b * a.NKV + hk) * a.max_q * G + rr) * parts.ld;
        end[threadIdx.x] = s.seen(rr / G, a.causal);
        whole[threadIdx.x] =
            job.y > 1 ? joined(parts, job.x, job.y, rr % rows) : parts.stat[((size_t)s.q0 + rr / G) * a.NH + hk * G + rr % G];
      }
      __syncthreads();
      const int stop = min(n * a.NKV - y0, kBlock);
      for (int y = slice; y < stop; y += 16 * kAtOnce) {
        float2 p[kAtOnce];
#pragma unroll
        for (int u = 0; u < kAtOnce; u++) {
          const int z = min(y + 16 * u, stop - 1);
          const bool sees = y + 16 * u < stop && j * kKeys < end[z];
          p[u] = sees ? parts.block[from[z] + j] : make_float2(0.0f, 0.0f);
        }
#pragma unroll
        for (int u = 0; u < kAtOnce; u++) {
          const float2 w = whole[min(y + 16 * u, stop - 1)];
          if (p[u].y != 0.0f) sum += p[u].y * ex2(p[u].x - w.x) / w.y;
        }
      }
      __syncthreads();
    }
    part[slice][threadIdx.x & 15] = sum;
    __syncthreads();
    if (slice || j >= nb) return;
    float t = 0.0f;
#pragma unroll
    for (int y = 0; y < 16; y++) t += part[y][threadIdx.x];
    weight[(size_t)b * a.ld_table + j] += t;
    return;
  }
  const unsigned x = blockIdx.x / per_job;
  const int r = blockIdx.x % per_job * kJoinRows8 + (threadIdx.x >> 5), d = 4 * (threadIdx.x & 31);
  const int4 *told = reinterpret_cast<const int4 *>(parts.told + 4) + 2 * (size_t)x;
  const int4 from = told[0], job = told[1];
  if (parts.wgs && x >= (unsigned)*parts.told) return;
  const int n = job.y, rr = from.w * rows + r;
  if (n < 2 || r >= rows || rr >= from.y) return;  // one workgroup had it whole; no row
  const int floats = part_floats(a.HS), h = from.z * G + rr % G;
  const size_t g = (size_t)from.x + rr / G;
  float m = -INFINITY, l = 0.0f;
  float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  // So many parts' loads are on their way together (four throughout: one conversation's 64 parts 6.6 us, not 6.1; twelve:
  // prompts behind long conversations 10.4, not 9.1).
  const auto join = [&](auto many, int t) {
    constexpr int kParts = decltype(many)::value;
    float4 y[kParts];
    float2 x[kParts];
    float top = m;
#pragma unroll
    for (int u = 0; u < kParts; u++) {
      const size_t p = part_row(parts, job.x, min(t + u, n - 1), r);
      y[u] = ld4(parts.o + p * floats + min(d, floats - 4));
      x[u] = parts.ml[p];
      if (t + u >= n) x[u].y = 0.0f;
    }
#pragma unroll
    for (int u = 0; u < kParts; u++) top = fmaxf(top, x[u].y == 0.0f ? -INFINITY : x[u].x);
    const float keep = ex2(m - or0(top));
    m = top;
    l *= keep;
    o = make_float4(o.x * keep, o.y * keep, o.z * keep, o.w * keep);
#pragma unroll
    for (int u = 0; u < kParts; u++) {
      const float w = x[u].y == 0.0f ? 0.0f : x[u].y * ex2(x[u].x - or0(top));  // 0: a part without a key of this row, its o is 0
      l += w;
      o = make_float4(fmaf(w, y[u].x, o.x), fmaf(w, y[u].y, o.y), fmaf(w, y[u].z, o.z), fmaf(w, y[u].w, o.w));
    }
  };
  int t = 0;
  for (; t + 4 < n; t += 8) join(std::integral_constant<int, 8>{}, t);
  if (t < n) join(std::integral_constant<int, 4>{}, t);
  const bool none = l == 0.0f;
  const float inv = none ? 1.0f : 1.0f / l;
  put4(out + g * a.ldo + (size_t)h * a.HS + d, make_float4(o.x * inv, o.y * inv, o.z * inv, o.w * inv), a.HS - d);
  if (lse && d == 0) lse[g * a.NH + h] = none ? -INFINITY : (m + __builtin_amdgcn_logf(l)) * kLn28;
}

// Many rows: a prompt's. 128 rows of a sequence and key/value head per workgroup, 32 to a wavefront, over blocks whose codes
// go through LDS as halves (which hold them exactly).
//
// The scores are computed transposed, so that a lane holds one row: its maximum and sum stay in the lane, and its weights are
// the second product's operand as they stand. q and the weights are two halves each (ugk_split.h), so a product is two of
// v_mfma_f32_32x32x16_f16, where fp32 keys and values need three.
//
// Bound by matrix and vector instructions, which add up on a SIMD: 64 of the first and some 540 of the others per block and
// wavefront at heads of 128. 8 x 1,024 rows of 12 heads of 64 42 to 44 us, 4 x 2,048 of them 72 to 75, of 16/4 heads of 128 160 to 178
// (of fp32 keys and values 67, 107 and 191). Products of one sum never follow one another, and their operands are two steps
// ahead (62 us, not 64, of prompts behind long conversations); wavefront priorities changed nothing.
constexpr int kTileWaves8 = 4, kTileRows8 = 32 * kTileWaves8, kTileThreads8 = kTileWaves8 * kWave;

// Four codes (bytes b0..b3 of w, with their signs turned over: c + 128) as halves.
__device__ __forceinline__ v2u halves4(uint32_t w) {
  const v2h off = {(_Float16)1152.0f, (_Float16)1152.0f};  // 0x6400 | byte is 1024 + byte
  const v2h lo = __builtin_bit_cast(v2h, __builtin_amdgcn_perm(0x64646464u, w, 0x04010400u)) - off;
  const v2h hi = __builtin_bit_cast(v2h, __builtin_amdgcn_perm(0x64646464u, w, 0x04030402u)) - off;
  return v2u{__builtin_bit_cast(uint32_t, lo), __builtin_bit_cast(uint32_t, hi)};
}

template <int DT>
__device__ __forceinline__ void tile_job(float *out, float *lse, const float *q, const int8_t *k8, const float *ks, const int8_t *v8,
                                         const float *vs, const ugk_cache8 &a, const Parts8 &parts, const Job8 &job, int *word) {
  constexpr int KSTR = 16 * DT + 8, VSTR = kKeys + 8, D32 = DT / 2, NL = (DT + 3) / 4;
  __shared__ alignas(16) _Float16 kl[2][kKeys * KSTR];
  __shared__ alignas(16) _Float16 vl[2][16 * DT * VSTR];
  const int thread = here((int)threadIdx.x);  // what is computed from it is not kept from job to job
  const int lane = thread & (kWave - 1), wave = __builtin_amdgcn_readfirstlane(thread >> 6);
  const int col = lane & 31, half = lane >> 5;
  const Seq8 &s = job.s;
  const int b = job.b, hk = job.hk, G = a.NH / a.NKV, HP = padded(a.HS), CH = HP / 16;
  const int rows = job.rows, row0 = job.group * kTileRows8, first = job.first, stop = job.stop;
  const int mine = row0 + 32 * wave + col, safe = min(mine, rows - 1), i = safe / G, h = hk * G + safe % G;
  const int lim = s.seen(i, a.causal);
  // what the wavefront's first and last rows see
  const int wave_first = min(row0 + 32 * wave, rows - 1), wave_last = min(row0 + 32 * wave + 31, rows - 1);
  const int least = s.seen(wave_first / G, a.causal), most_seen = s.seen(wave_last / G, a.causal);
  const bool idle = row0 + 32 * wave >= rows;

  // staging: thread t has words of 16 codes t, t + 256 of the block's keys and of its values
  int kdst[NL], vdst[NL];
#pragma unroll
  for (int n = 0; n < NL; n++) {
    const int w = thread + n * kTileThreads8, c = w & 3;
    kdst[n] = w / CH * KSTR + w % CH * 16;
    vdst[n] = (w >> 2) * VSTR + (c & 1) * 8 + (c >> 1) * 4;
  }
  v4u kr[NL], vr[NL];
  float kscale = 0.0f, vscale = 0.0f;
  bool there = true;
  int next = first < stop ? table_at(a, b, first) : 0;
  const auto fetch = [&](int j) {
    const int id = checked_block(a, __builtin_amdgcn_readfirstlane(next), word, UGK_IDS_CACHE8_ATTENTION);
    next = table_at(a, b, min(j + 1, stop - 1));
    there = id >= 0;
    const size_t at = block_head(id, a.NKV, hk);
#pragma unroll
    for (int n = 0; n < NL; n++) {
      const int w = thread + n * kTileThreads8;
      if (w < 4 * HP) {
        kr[n] = *reinterpret_cast<const v4u *>(k8 + at * kKeys * HP + 16 * w);
        vr[n] = *reinterpret_cast<const v4u *>(v8 + at * kKeys * HP + 16 * w);
      }
    }
    kscale = ks[at];
    vscale = vs[at];
  };
  if (first < stop) fetch(first);

  v8h qh[DT], ql[DT];
  int e;
  bool nan;
  {
    const float *p = q + ((size_t)s.q0 + i) * a.ldq + (size_t)h * a.HS;
    float x[DT][8];
    const uint32_t most = half_max_bits(load_q(p, 8 * half, 16, a, x));
    nan = most >= kInfBits;
    e = (int)(most >> 23) - 126 - 15;  // below 2^15 2^e
#pragma unroll
    for (int st = 0; st < DT; st++) {
#pragma unroll
      for (int d = 0; d < 8; d++) x[st][d] = nan ? 0.0f : __builtin_amdgcn_ldexpf(x[st][d], -e);
      split8(x[st], qh[st], ql[st]);
    }
  }

  Running run;
  v16f o[D32];
#pragma unroll
  for (int t = 0; t < D32; t++) o[t] = v16f{};

  if (CH < DT) {  // behind the keys' rows q is 0, and what is there has to be a number
    for (int x = thread; x < 2 * kKeys * KSTR / 2; x += kTileThreads8) reinterpret_cast<uint32_t *>(kl[0])[x] = 0u;
    __syncthreads();
  }
  for (int j = first; j < stop; j++) {
    _Float16 *kt = kl[(j - first) & 1], *vt = vl[(j - first) & 1];
#pragma unroll
    for (int n = 0; n < NL; n++) {
      if (thread + n * kTileThreads8 >= 4 * HP) continue;
      const v4u kw = kr[n] ^ 0x80808080u, vw = vr[n] ^ 0x80808080u;
      const v2u k0 = halves4(kw[0]), k1 = halves4(kw[1]), k2 = halves4(kw[2]), k3 = halves4(kw[3]);
      *reinterpret_cast<v4u *>(kt + kdst[n]) = v4u{k0[0], k0[1], k1[0], k1[1]};
      *reinterpret_cast<v4u *>(kt + kdst[n] + 8) = v4u{k2[0], k2[1], k3[0], k3[1]};
      // a word of the values: keys c, c + 16, c + 32, c + 48; the words are c = 4 x .. 4 x + 3
      const uint32_t t0 = __builtin_amdgcn_perm(vw[1], vw[0], 0x05010400u), t1 = __builtin_amdgcn_perm(vw[1], vw[0], 0x07030602u);
      const uint32_t t2 = __builtin_amdgcn_perm(vw[3], vw[2], 0x05010400u), t3 = __builtin_amdgcn_perm(vw[3], vw[2], 0x07030602u);
      *reinterpret_cast<v2u *>(vt + vdst[n]) = halves4(__builtin_amdgcn_perm(t2, t0, 0x05040100u));
      *reinterpret_cast<v2u *>(vt + vdst[n] + 16) = halves4(__builtin_amdgcn_perm(t2, t0, 0x07060302u));
      *reinterpret_cast<v2u *>(vt + vdst[n] + 32) = halves4(__builtin_amdgcn_perm(t3, t1, 0x05040100u));
      *reinterpret_cast<v2u *>(vt + vdst[n] + 48) = halves4(__builtin_amdgcn_perm(t3, t1, 0x07060302u));
    }
    const bool held = there;
    const float fac = here(score_factor(parts, kscale, e)), vnow = exponent(vscale);
    __syncthreads();
    if (j + 1 < stop) fetch(j + 1);
    if (idle || j * kKeys >= most_seen) continue;
    // The operands of two steps on their way, and of two products in a row no sum is the same.
    const _Float16 *kp = kt + col * KSTR + 8 * half, *vp = vt + col * VSTR + 8 * half;
    v8h kf[2][2], vf[D32];
    v16f sc[2] = {v16f{}, v16f{}};
#pragma unroll
    for (int st = 0; st < 2; st++)
#pragma unroll
      for (int x = 0; x < 2; x++) kf[st][x] = frag(kp + 32 * x * KSTR + 16 * st);
#pragma unroll
    for (int st = 0; st < DT; st++) {
      __builtin_amdgcn_sched_barrier(0);
      sc[0] = mfma(kf[st % 2][0], ql[st], sc[0]);
      sc[1] = mfma(kf[st % 2][1], ql[st], sc[1]);
      sc[0] = mfma(kf[st % 2][0], qh[st], sc[0]);
      sc[1] = mfma(kf[st % 2][1], qh[st], sc[1]);
      __builtin_amdgcn_sched_barrier(0);
      if (st + 2 < DT)
#pragma unroll
        for (int x = 0; x < 2; x++) kf[st % 2][x] = frag(kp + 32 * x * KSTR + 16 * (st + 2));
    }
#pragma unroll
    for (int t = 0; t < D32; t++) vf[t] = frag(vp + 32 * t * VSTR);
    __builtin_amdgcn_sched_barrier(0);
    float mb = -INFINITY;
    const bool masked = !held || (j + 1) * kKeys > least;
    const int seen = held ? lim - j * kKeys - 4 * half : 0;  // of this block's keys from the lane's first on
    if (masked) {
      const int n = here(seen);
#pragma unroll
      for (int x = 0; x < 2; x++)
#pragma unroll
        for (int r = 0; r < 16; r++) sc[x][r] = 32 * x + 8 * (r / 4) + r % 4 < n ? sc[x][r] : -INFINITY;
    }
#pragma unroll
    for (int x = 0; x < 2; x++)
#pragma unroll
      for (int r = 0; r < 16; r++) mb = fmaxf(mb, sc[x][r]);
    const float most = half_max(mb);
    mb = top_score(most, fac);
    const float fo = run.stand(mb, vnow);
    if (__any(fo != 1.0f)) {
      const float x = here(fo);
#pragma unroll
      for (int t = 0; t < D32; t++) o[t] *= x;
    }
    // The weights stand on what the output's sum stands on, times 2^14: the products add up in its registers.
    const float up = 14.0f + (vnow - run.e);
    float less = here(mb == INFINITY ? NAN : up - or0(run.mo)), lb = 0.0f;
    if (__any(far_score(mb))) {
      const float off = here(far_score(mb) ? most : 0.0f);
      less = here(far_score(mb) ? (mb - run.mo) + up : less);
#pragma unroll
      for (int x = 0; x < 2; x++)
#pragma unroll
        for (int r = 0; r < 16; r++) sc[x][r] -= off;
    }
    const bool apart = __any(run.e - vnow > 64.0f);  // weights that the row's sum needs may vanish next to another block's values
    if (apart) {
      const float own = here(far_score(mb) ? 0.0f : less_top(mb, 0.0f));  // on the block's own largest
#pragma unroll
      for (int x = 0; x < 2; x++)
#pragma unroll
        for (int r = 0; r < 16; r++) lb += ex2(fmaf(sc[x][r], fac, own));
      run.sum(mb, lb, mb, 0.0f);
    }
#pragma unroll
    for (int g = 0; g < 4; g++) {
      float p[8];
      v8h ph, pl;
#pragma unroll
      for (int r = 0; r < 8; r++) {
        p[r] = ex2(fmaf(sc[g / 2][8 * (g % 2) + r], fac, less));
        lb += p[r];
      }
      split8(p, ph, pl);
#pragma unroll
      for (int t = 0; t < D32; t++) o[t] = mfma(vf[t], pl, o[t]);
#pragma unroll
      for (int t = 0; t < D32; t++) {
        o[t] = mfma(vf[t], ph, o[t]);
        if (g < 3) vf[t] = frag(vp + 32 * t * VSTR + 16 * (g + 1));
      }
    }
    if (!apart) run.sum(mb, lb, run.mo, up);
  }
  if (mine >= rows) return;
  float sum = half_sum(run.l);
  if (nan && sum != 0.0f) sum = NAN;  // (its q is 0 here: all keys that it sees have the weight 1)
  int p;
  const float g = run.last(sum, &p);
  p -= 14;  // of the weights
  const Place8 to(out, lse, parts, a, job.slot, job.whole, mine - row0, (size_t)s.q0 + i, h);
#pragma unroll
  for (int t = 0; t < D32; t++)
#pragma unroll
    for (int r = 0; r < 16; r += 4) {
      const int d = 32 * t + 8 * (r / 4) + 4 * half;
      put4(to.o + d,
           make_float4(__builtin_amdgcn_ldexpf(o[t][r] * g, p), __builtin_amdgcn_ldexpf(o[t][r + 1] * g, p),
                       __builtin_amdgcn_ldexpf(o[t][r + 2] * g, p), __builtin_amdgcn_ldexpf(o[t][r + 3] * g, p)),
           a.HS - d);
    }
  if (half == 0) to.put(run.m, sum);
}

template <int DT, bool kShared>
__global__ __launch_bounds__(kTileThreads8, DT <= 4 ? 3 : 2) void k_cache8_tile(float *out, float *lse, const float *q, const int8_t *k8, const float *ks,
                               const int8_t *v8, const float *vs, ugk_cache8 a, Parts8 parts, unsigned pairs,
                               unsigned groups, int *word) {
  Jobs<kTileRows8, 2, kShared> jobs(a, parts, pairs, groups, word);
  Job8 job;
  for (bool more = jobs.first(job); more; more = jobs.next(job)) {
    tile_job<DT>(out, lse, q, k8, ks, v8, vs, a, parts, job, word);
    __syncthreads();  // LDS is read until here
  }
}

// ---- eviction ----------------------------------------------------------------------

constexpr int kEvictThreads = 1024, kBins = 2 * kEvictThreads;

// Sum over the workgroup's threads before this one, and in *all over all of them.
__device__ __forceinline__ int before(int x, int *lds, int *all) {
  const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x >> 6;
  const int y = wave_scan(x);
  __syncthreads();  // the last call's sums have been read
  if (lane == kWave - 1) lds[wave] = y;
  __syncthreads();
  int sum = 0, total = 0;
  for (int w = 0; w < kEvictThreads / kWave; w++) {
    const int z = lds[w];
    if (w < wave) sum += z;
    total += z;
  }
  *all = total;
  return sum + y - x;
}

// One sequence per workgroup, E entries of its table per thread, side by side in registers: the d lightest blocks by a search
// over the weights' bits, eleven at a time (counts in LDS: eight at a time took a turn more, and the exponents of many
// weights met in the same counter), ties by their index; then each entry's place from counts of those before it. Reading and
// writing 16 bytes per entry is nothing; what counts are the chain of barriers (three counts and two sums): 5.4 us of up to 16
// blocks of 16 sequences, 9.7 of up to 4,096 of 64.
template <int E>
__global__ __launch_bounds__(kEvictThreads) void k_cache8_evict(int *table_out, int *len_out, float *weight_out, int *dropped,
                                                               const int *table, const int *k_len, const float *weight, int ld,
                                                               int keep, int first, int recent, int *word) {
  __shared__ int count[kBins], lds[kEvictThreads / kWave];
  __shared__ int found, under;
  const int b = blockIdx.x, len = k_len[b];
  const int full = min(max(len, 0), (int)min((long long)ld * kKeys, (long long)0x7fffffff)), n = (full + kKeys - 1) / kKeys;
  if (full != len && threadIdx.x == 0) *word = UGK_IDS_CACHE8_EVICT;
  const int d = max(n - keep, 0), i0 = threadIdx.x * E;
  const size_t row = (size_t)b * ld;
  int id[E];
  float w[E];
  uint32_t key[E];
#pragma unroll
  for (int x = 0; x < E; x++) {
    const int i = i0 + x;
    id[x] = table[row + min(i, ld - 1)];  // without a branch, which would wait for each load
    w[x] = weight[row + min(i, ld - 1)];
    // ascending in the weight; NaN, whatever its sign, above all
    const uint32_t u = __float_as_uint(w[x] + 0.0f);
    key[x] = w[x] != w[x] ? 0xffffffffu : u >> 31 ? ~u : u | 0x80000000u;
  }
  // the value of the d-th lightest, eleven bits at a time (the last ten), and how many of its equals go
  uint32_t value = 0;
  int left = d, all;
  if (d > 0) {
#pragma unroll 1
    for (int turn = 0; turn < 3; turn++) {
      const int shift = turn == 0 ? 21 : turn == 1 ? 10 : 0, above = turn == 0 ? 31 : turn == 1 ? 21 : 10;  // the bits found so far
      for (int i = threadIdx.x; i < kBins; i += kEvictThreads) count[i] = 0;
      __syncthreads();
#pragma unroll
      for (int x = 0; x < E; x++) {
        const int i = i0 + x;
        const bool may = i >= first && i < n - recent;
        const bool same = turn == 0 || key[x] >> above == value >> above;
        if (may && same) atomicAdd(&count[key[x] >> shift & (turn == 2 ? 1023u : 2047u)], 1);
      }
      __syncthreads();
      const int c0 = count[2 * threadIdx.x], c1 = count[2 * threadIdx.x + 1];
      const int y = before(c0 + c1, lds, &all);
      if (y < left && y + c0 + c1 >= left) {
        const bool second = y + c0 < left;
        found = 2 * threadIdx.x + second;
        under = y + (second ? c0 : 0);
      }
      __syncthreads();
      value |= (uint32_t)found << shift;
      left -= under;
    }
  }
  int ties = 0;
#pragma unroll
  for (int x = 0; x < E; x++) ties += d > 0 && i0 + x >= first && i0 + x < n - recent && key[x] == value;
  int tie = before(ties, lds, &all), gone = 0;
  bool goes[E];
#pragma unroll
  for (int x = 0; x < E; x++) {
    const bool may = d > 0 && i0 + x >= first && i0 + x < n - recent, same = may && key[x] == value;
    goes[x] = may && (key[x] < value || (same && tie < left));
    tie += same;
    gone += goes[x];
  }
  int g = before(gone, lds, &all);  // behind its barriers everything has been read: the outputs may be the inputs
#pragma unroll
  for (int x = 0; x < E; x++) {
    const int i = i0 + x;
    if (i >= ld) break;
    const int to = goes[x] ? ld - d + g : i - g;
    g += goes[x];
    table_out[row + to] = id[x];
    weight_out[row + to] = goes[x] || i >= n ? 0.0f : w[x];
  }
  if (threadIdx.x == 0) {
    len_out[b] = full - d * kKeys;
    dropped[b] = d;
  }
}

int cu_count8() {
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

// How an attention call is cut: k_cache8_rows (4, 16, 32 rows) in so many groups, or k_cache8_tile (128) in so many
// tiles; `wgs` workgroups that share all blocks, or up to `splits` parts of `least` blocks or more of each; the rows of a
// slot of parts, the slots and jobs, and where a job's are.
//
// By rows (query rows times heads of the group; times in us, 24 sequences of up to 8,192 keys, heads of 128, by the
// smaller and the next larger form): 4 rows 36 and 39; 16 rows 27 and 33; 32 rows 37 and 49; 64 rows in two groups of 32
// or a tile 63 and 71. Where tiles fill the CUs, two groups are the slower (64 x 12 heads of 64, 64 rows each: 36
// and 31). Weights are added up by groups of 32 whatever the rows.
constexpr int kJobInts = 8;
struct Plan8 {
  int rows, groups, splits, least, wgs, grid, held, per_job, step;
  size_t slots, jobs;
};

Plan8 plan8(const ugk_cache8 &a, bool weigh) {
  Plan8 p{};
  const int cus = cu_count8();
  const long long pairs = (long long)a.nseq * a.NKV, G = a.NH / a.NKV, rows = a.max_q * G, blocks = (a.max_k + kKeys - 1) / kKeys;
  const bool groups = weigh || rows <= 32 || (rows <= 64 && pairs <= cus);
  p.rows = rows <= 4 ? 4 : rows <= 16 ? 16 : groups ? 32 : kTileRows8;
  p.groups = (int)((rows + p.rows - 1) / p.rows);
  p.held = (int)min((long long)p.rows, rows);
  p.per_job = (p.held + kJoinRows8 - 1) / kJoinRows8;
  p.step = 1;
  p.splits = 1;
  // Workgroups that the CUs hold at once. Fewer leave a SIMD's wavefront alone with its loads' and products' latency (heads
  // of 128, one to a CU: tiles 81 us, not 64, 32 rows 46, not 36); with more, some CUs have a second round (32 rows of heads
  // of 64, four: 29, not 24).
  const int at_once = cus * (a.HS > 64 ? (p.rows == 4 ? 3 : 2) : (p.rows == 4 ? 4 : 3));
  // at most so many jobs (a sequence that has one has a row), and the shares of so many blocks, were all sequences full
  const long long jobs = min(pairs * p.groups, (a.rows_q * G / p.rows + min(a.nseq, a.rows_q)) * a.NKV), share = blocks * jobs / at_once;
  // what a workspace of the same rows and heads has for the fp32 attention
  const size_t most = max(attention_parts_bound(a.HS), attention_backward_bound(a.rows_q, a.NH, a.HS)) / sizeof(float) - 4;
  const long long every = pairs * p.groups;
  const auto fit = [&](long long jobs, bool shared) {  // slots
    return ((long long)most - kJobInts * jobs - (shared && weigh ? 2 * every : 0)) / ((part_floats(a.HS) + 2) * (long long)p.held);
  };
  // Few blocks are not worth a look at all sequences and a second launch (16 x 12 heads of 64, one row, up to 1,024 keys 8.4
  // us, in shares 9.5 and 3.6; up to 4,096 keys 18.5, and 15 and 4; 24 x 8 heads of 128, up to 8,192 keys 50, and 36 and
  // 4.7), nor are many groups, which fill the CUs. But where most groups are not there, for max_q is a few sequences', the
  // workgroups that find none would take the time (64 sequences of 12 heads of 64, 2,048 rows of one and one of the others:
  // 78 and 9 us in shares, 101 else; where they are few it is nothing: a row of each of 10 of 400 sequences of up to 1,024
  // keys 12.6 and 3.8, 11.0 else).
  const bool few = blocks > 32 && jobs <= 4LL * at_once, empty = every > 4 * jobs && every > 8LL * at_once;
  if ((few || empty) && (blocks + 8) * jobs <= 1 << 30 && jobs * p.per_job < 1 << 23 && (rows + p.rows) * G >> 32 == 0) {
    // a job has one part more than workgroups' borders, and a workgroup two at most that are not whole
    const long long slots = fit(jobs, true);
    p.step = jobs <= at_once && slots >= 2 * jobs ? 1 : 2;
    p.wgs = (int)max(min((long long)at_once, p.step == 1 ? slots - jobs : slots / 2), 0LL);
  }
  if (p.wgs) {
    p.least = 4;
    p.slots = p.step == 1 ? p.wgs + jobs : 2LL * p.wgs;
    p.grid = max(p.wgs, (int)jobs);
    p.jobs = jobs;
  } else {
    // Whole where that fills two thirds of the CUs (192 workgroups of up to 16 blocks 8.4 us; in parts 8.1, and 4 to join
    // them); with weights to add up, the launch that joins parts is there anyway.
    const long long least = max(3 * jobs >= 2LL * cus && !weigh ? blocks : max(share, 4LL), 1LL);
    p.step = 1;
    p.splits = (int)max(min(min((blocks + least - 1) / least, fit(every, false) / every), ((1LL << 24) - 1) / every), 1LL);
    p.least = (int)max((blocks + p.splits - 1) / p.splits, 1LL);
    p.grid = (int)(every * p.splits);
    p.slots = p.splits > 1 ? p.grid : 0;
    p.jobs = every;
  }
  return p;
}
size_t slot_floats(const ugk_cache8 &a, const Plan8 &p) { return p.slots * p.held * part_floats(a.HS); }
size_t told_ints(const ugk_cache8 &a, const Plan8 &p, bool weigh) {
  return 4 + kJobInts * p.jobs + (p.wgs && weigh ? 2 * (size_t)a.nseq * a.NKV * p.groups : 0);
}
size_t parts_floats(const ugk_cache8 &a, const Plan8 &p, bool weigh) {
  return p.slots ? slot_floats(a, p) + told_ints(a, p, weigh) + 2 * p.slots * p.held : 0;
}
int blocks_of_keys(const ugk_cache8 &a) { return (a.max_k + kKeys - 1) / kKeys; }
}  // namespace

size_t cache8_attention_bytes(const ugk_cache8 &a, bool weigh) {
  const size_t stat = (size_t)a.rows_q * a.NH, block = (size_t)a.nseq * a.max_q * a.NH * blocks_of_keys(a);
  return (parts_floats(a, plan8(a, weigh), weigh) + (weigh ? 2 * (stat + block) : 0)) * sizeof(float);
}

int launch_cache8_attention(float *out, float *lse, const float *q, const void *k8, const float *ks, const void *v8,
                            const float *vs, float *weight, float *mem, const ugk_cache8 &a, int *word) {
  const Plan8 p = plan8(a, weight);
  const unsigned pairs = (unsigned)a.nseq * a.NKV, G = a.NH / a.NKV;
  Parts8 parts{};
  parts.rows = p.held;
  parts.step = p.step;
  parts.splits = p.splits;
  parts.least = p.least;
  parts.wgs = p.wgs;
  parts.cus = cu_count8();
  parts.ld = blocks_of_keys(a);
  parts.most = (int)p.jobs;
  int of_scale, of_product;  // the scale's sign goes with q
  parts.factor = frexpf(frexpf(fabsf(a.scale), &of_scale) * kLog2e8, &of_product);
  parts.power = of_scale + of_product;
  parts.inverse = G == 1 ? 0u : (unsigned)((1ULL << 32) / G + 1);
  if (p.slots) {
    parts.o = mem;
    parts.told = reinterpret_cast<int *>(mem + slot_floats(a, p));
    parts.ml = reinterpret_cast<float2 *>(mem + slot_floats(a, p) + told_ints(a, p, weight));
    mem += parts_floats(a, p, weight);
  }
  if (weight) {
    parts.stat = reinterpret_cast<float2 *>(mem);
    parts.block = parts.stat + (size_t)a.rows_q * a.NH;
  }
  const int8_t *kc = static_cast<const int8_t *>(k8), *vc = static_cast<const int8_t *>(v8);
  const auto go = [&](auto kernel) {
    launch(kernel, dim3(p.grid), dim3(kFewWaves * kWave), 0, out, lse, q, kc, ks, vc, vs, a, parts, pairs, (unsigned)p.groups, word);
  };
  const auto of = [&](auto shared) {
    constexpr bool kS = decltype(shared)::value;
    const int d = a.HS <= 32 ? 2 : a.HS <= 64 ? 4 : a.HS <= 96 ? 6 : 8;
    switch (p.rows) {
      case 4:
        d == 2   ? go(k_cache8_rows<2, 4, kS>)
        : d == 4 ? go(k_cache8_rows<4, 4, kS>)
        : d == 6 ? go(k_cache8_rows<6, 4, kS>)
                 : go(k_cache8_rows<8, 4, kS>);
        break;
      case 16:
        d == 2   ? go(k_cache8_rows<2, 16, kS>)
        : d == 4 ? go(k_cache8_rows<4, 16, kS>)
        : d == 6 ? go(k_cache8_rows<6, 16, kS>)
                 : go(k_cache8_rows<8, 16, kS>);
        break;
      case 32:
        d == 2   ? go(k_cache8_rows<2, 32, kS>)
        : d == 4 ? go(k_cache8_rows<4, 32, kS>)
        : d == 6 ? go(k_cache8_rows<6, 32, kS>)
                 : go(k_cache8_rows<8, 32, kS>);
        break;
      default:
        d == 2 ? go(k_cache8_tile<2, kS>) : d == 4 ? go(k_cache8_tile<4, kS>) : d == 6 ? go(k_cache8_tile<6, kS>) : go(k_cache8_tile<8, kS>);
    }
  };
  p.wgs ? of(std::true_type{}) : of(std::false_type{});
  if (int e = check_launch("cache8_attention")) return e;
  const unsigned joins = p.slots ? (unsigned)(p.jobs * p.per_job) : 0;
  const unsigned weighs = weight ? (unsigned)a.nseq * grid_for(parts.ld, 16) : 0;
  if (joins + weighs == 0) return UGK_OK;
  launch(k_cache8_finish, dim3(joins + weighs), dim3(kBlock), 0, out, lse, weight, parts, a, p.rows, p.groups, p.per_job, joins);
  return check_launch("cache8_attention");
}

// Blocks that max_q rows of a sequence touch at most, wherever they begin.
static int touched_blocks(const ugk_cache8 &a) {
  const int n = a.max_q < a.max_k ? a.max_q : a.max_k;
  const int by_rows = (int)(((long long)n + 2 * kKeys - 2) / kKeys), by_keys = (int)(((long long)a.max_k + kKeys - 1) / kKeys);
  return by_rows < by_keys ? by_rows : by_keys;
}
#define UGK_CH8(kernel)                                                        \
  switch (padded(a.HS) / 16) {                                                 \
    case 1: go(kernel<1>); break;                                              \
    case 2: go(kernel<2>); break;                                              \
    case 3: go(kernel<3>); break;                                              \
    case 4: go(kernel<4>); break;                                              \
    case 5: go(kernel<5>); break;                                              \
    case 6: go(kernel<6>); break;                                              \
    case 7: go(kernel<7>); break;                                              \
    default: go(kernel<8>);                                                    \
  }
// Workgroups of a head by blocks: `per` of each sequence, or, where that is more than twice as many as there can be (max_q is
// a few sequences'; 64 of 12 heads of 64, 2,048 rows of one and one of the others: 12 us, 41 else) and the CUs would have
// rounds of them, `all` that there can be. Rows of a sequence touch one block more than they fill, and another where they
// begin.
struct Store8 {
  int per, all;
};
static Store8 store8(const ugk_cache8 &a) {
  const long long per = touched_blocks(a), most = a.nseq * per, all = a.rows_q / kKeys + 2LL * min(a.nseq, a.rows_q);
  return most > 2 * all && 2 * most * a.NKV > 16LL * cu_count8() ? Store8{0, (int)all} : Store8{(int)per, (int)most};
}
long long cache8_store_workgroups(const ugk_cache8 &a) { return (long long)store8(a).all * a.NKV; }
int launch_cache8_store(void *k8, float *ks, void *v8, float *vs, const float *k, const float *v, const ugk_cache8 &a, int *word) {
  const Store8 n = store8(a);
  const auto go = [&](auto kernel) {
    launch(kernel, dim3((unsigned)n.all * a.NKV, 2), dim3(kBlock), 0, (int8_t *)k8, ks, (int8_t *)v8, vs, k, v, a, n.per, n.all, word);
  };
  UGK_CH8(k_cache8_store)
  return check_launch("cache8_store");
}
int launch_cache8_load(float *k, float *v, const void *k8, const float *ks, const void *v8, const float *vs, const ugk_cache8 &a,
                       int *word) {
  const Store8 n = store8(a);
  const auto go = [&](auto kernel) {
    launch(kernel, dim3((unsigned)n.all * a.NKV, 2), dim3(kBlock), 0, k, v, (const int8_t *)k8, ks, (const int8_t *)v8, vs, a, n.per, n.all,
           word);
  };
  UGK_CH8(k_cache8_load)
  return check_launch("cache8_load");
}
#undef UGK_CH8

int launch_cache8_evict(int *table_out, int *len_out, float *weight_out, int *dropped, const int *table, const int *k_len,
                        const float *weight, int nseq, int ld, int keep, int first, int recent, int *word) {
  const auto go = [&](auto kernel) {
    launch(kernel, dim3(nseq), dim3(kEvictThreads), 0, table_out, len_out, weight_out, dropped, table, k_len, weight, ld, keep, first, recent,
           word);
  };
  if (ld <= kEvictThreads) go(k_cache8_evict<1>);
  else if (ld <= 4 * kEvictThreads) go(k_cache8_evict<4>);
  else go(k_cache8_evict<16>);
  static_assert(kEvictBlocks == 16 * kEvictThreads, "the longest row of a table");
  return check_launch("cache8_evict");
}

}  // namespace ugk
