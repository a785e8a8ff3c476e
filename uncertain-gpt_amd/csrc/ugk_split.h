// ugk_split.h - products of single-precision matrices on the half-precision
// matrix units of gfx950.
//
// A float x, scaled by a power of two so that the largest of its row or tile
// lies in [2^14, 2^15), is held as h + l with h = half(x), l = half(x - h), both
// rounded to nearest (the splitting that Ootomo and Yokota, 2022, among others, use on such units). Each
// has 11 bits: |x - h| <= 2^-11 |x|, |x - h - l| <= 2^-23 |x| as long as l is a
// normal half (|x| >= 2^-2, or 2^-16 of the largest); below that the error stays
// under 2^-25, that is 2^-39 of the largest. A product x y is taken as xh yh + xl yh +
// xh yl in single-precision accumulators; the part left out, xl yl, is at most
// 2^-22 |x y|. So a product is off by 2^-21 of its size at most, eight roundings of single
// precision, and by a quarter of that in the mean, for three times the half-precision units' work: they
// do 16 times the operations of the single-precision ones (v_mfma_f32_32x32x16_f16
// takes 32 cycles, v_mfma_f32_32x32x2_f32 64 for an eighth of the products), so
// this has a ceiling of 5.3 times theirs. (Three bfloat16 parts would keep
// the exponent range without scaling, but need six products.) Against 64 bits the
// attention's results are as near as plain single precision's or nearer (8 x 1,024
// rows of 12 heads: 2.6e-7 and 3.2e-7 in the 2-norm, gradients 5.2e-7 and 7.0e-7).
#pragma once

#include "ugk_internal.h"

namespace ugk {
namespace {

typedef _Float16 v8h __attribute__((ext_vector_type(8)));
typedef _Float16 v2h __attribute__((ext_vector_type(2)));
typedef float v2f __attribute__((ext_vector_type(2)));
typedef float v16f __attribute__((ext_vector_type(16)));
typedef uint32_t v4u __attribute__((ext_vector_type(4)));
typedef uint32_t v2u __attribute__((ext_vector_type(2)));

// C += A B for a 32 x 32 tile over 16 products. Lane t holds row (of A) or column (of B)
// t % 32, products 8 (t / 32) .. + 7; of C column t % 32 and in register r row
// 8 (r / 4) + 4 (t / 32) + r % 4.
__device__ __forceinline__ v16f mfma(v8h a, v8h b, v16f c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0); }
// The same of two split operands.
__device__ __forceinline__ v16f mfma3(v8h ah, v8h al, v8h bh, v8h bl, v16f c) {
  return mfma(ah, bl, mfma(al, bh, mfma(ah, bh, c)));
}

// Two floats as halves: h, and l of what h leaves (x - h in one instruction, without a
// conversion of h; v_fma_mixlo_f16, which would round as well, takes 8 cycles, not 4).
__device__ __forceinline__ void split2(float x, float y, uint32_t &h, uint32_t &l) {
  const v2f v = {x, y};
  h = __builtin_bit_cast(uint32_t, __builtin_convertvector(v, v2h));
  float rx, ry;
  asm("v_fma_mix_f32 %0, %1, -1.0, %2 op_sel_hi:[1,0,0]" : "=v"(rx) : "v"(h), "v"(x));
  asm("v_fma_mix_f32 %0, %1, -1.0, %2 op_sel:[1,0,0] op_sel_hi:[1,0,0]" : "=v"(ry) : "v"(h), "v"(y));
  const v2f r = {rx, ry};
  l = __builtin_bit_cast(uint32_t, __builtin_convertvector(r, v2h));
}
__device__ __forceinline__ void split2(float x, float y, float f, uint32_t &h, uint32_t &l) { split2(x * f, y * f, h, l); }
// Eight of either kind, as an operand.
__device__ __forceinline__ void split8(const float (&x)[8], float f, v8h &h, v8h &l) {
  v4u a, b;
#pragma unroll
  for (int j = 0; j < 4; j++) {
    uint32_t hj, lj;
    split2(x[2 * j], x[2 * j + 1], f, hj, lj);
    a[j] = hj;
    b[j] = lj;
  }
  h = __builtin_bit_cast(v8h, a);
  l = __builtin_bit_cast(v8h, b);
}
__device__ __forceinline__ void split8(const float (&x)[8], v8h &h, v8h &l) {
  v4u a, b;
#pragma unroll
  for (int j = 0; j < 4; j++) {
    uint32_t hj, lj;
    split2(x[2 * j], x[2 * j + 1], hj, lj);
    a[j] = hj;
    b[j] = lj;
  }
  h = __builtin_bit_cast(v8h, a);
  l = __builtin_bit_cast(v8h, b);
}

// Operands from rows of halves in LDS, `stride` halves each. As rows: the lane's row t % 32, eight
// of its columns. As columns: column t % 32 of a 32-column block, of the eight
// rows 4 (t / 32) + j and 8 + 4 (t / 32) + j, j < 4, that lane t's accumulator registers 0..7 hold (8..15 of
// the rows from 16 on): two transposing reads of four rows of 16 columns per 16 lanes.
typedef _Float16 v4h __attribute__((ext_vector_type(4)));
typedef __fp16 v4f16 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) v4f16 lds_v4f16;
__device__ __forceinline__ v8h frag(const _Float16 *p) { return *reinterpret_cast<const v8h *>(p); }
__device__ __forceinline__ int cols_at(int lane, int stride) {
  return (4 * (lane >> 5) + (lane >> 2 & 3)) * stride + 16 * (lane >> 4 & 1) + 4 * (lane & 3);
}
__device__ __forceinline__ v8h frag_cols(const _Float16 *p, int stride) {
  const v4h a = __builtin_bit_cast(v4h, __builtin_amdgcn_ds_read_tr16_b64_v4f16((lds_v4f16 *)p));
  const v4h b = __builtin_bit_cast(v4h, __builtin_amdgcn_ds_read_tr16_b64_v4f16((lds_v4f16 *)(p + 8 * stride)));
  return __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
}

// The exponent that a largest magnitude (as its bits) is scaled by: x 2^(15 - e) is
// below 2^15. Below 2^-100 (and at 0) the scale stays; infinite and NaN give some
// exponent (the caller looks for them).
__device__ __forceinline__ int split_exp(uint32_t bits) { return max((int)(bits >> 23) - 126, -100); }
__device__ __forceinline__ float pow2(int e) { return __uint_as_float((uint32_t)(127 + e) << 23); }  // -126 <= e <= 127
__device__ __forceinline__ float split_scale(int e) { return pow2(15 - e); }    // e in [-100, 129]
__device__ __forceinline__ float split_unscale(int e) { return pow2(e - 15); }
constexpr uint32_t kInfBits = 0x7f800000u;

__device__ __forceinline__ uint32_t abs_bits(float x) { return __float_as_uint(x) & 0x7fffffffu; }
__device__ __forceinline__ uint32_t max_abs(uint32_t m, float4 v) {
  m = max(max(m, abs_bits(v.x)), abs_bits(v.y));
  return max(max(m, abs_bits(v.z)), abs_bits(v.w));
}

template <int kCtrl>
__device__ __forceinline__ uint32_t dpp_bits(uint32_t v) {
  return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, kCtrl, 0xf, 0xf, false);
}
// Largest of the wavefront's 64 lanes, in a scalar register.
__device__ __forceinline__ uint32_t wave_max_bits(uint32_t v) {
  v = max(v, dpp_bits<kDppQuadSwap1>(v));
  v = max(v, dpp_bits<kDppQuadSwap2>(v));
  v = max(v, dpp_bits<kDppHalfMirror>(v));
  v = max(v, dpp_bits<kDppMirror>(v));
  const uint32_t a = __builtin_amdgcn_readlane(v, 0), b = __builtin_amdgcn_readlane(v, 16);
  const uint32_t c = __builtin_amdgcn_readlane(v, 32), d = __builtin_amdgcn_readlane(v, 48);
  return max(max(a, b), max(c, d));
}
// Largest over the kLanes (16 or 32) lanes that share a row, in each of them.
template <int kLanes>
__device__ __forceinline__ uint32_t row_max_bits(uint32_t v) {
  v = max(v, dpp_bits<kDppQuadSwap1>(v));
  v = max(v, dpp_bits<kDppQuadSwap2>(v));
  v = max(v, dpp_bits<kDppHalfMirror>(v));
  v = max(v, dpp_bits<kDppMirror>(v));
  if (kLanes == 32) v = max(v, (uint32_t)__shfl_xor((int)v, 16));
  return v;
}
// x of this lane and of lane ^ 32, combined.
__device__ __forceinline__ float half_max(float x) {
  const auto s = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return fmaxf(__uint_as_float(s[0]), __uint_as_float(s[1]));
}
__device__ __forceinline__ uint32_t half_max_bits(uint32_t x) {
  const auto s = __builtin_amdgcn_permlane32_swap(x, x, false, false);
  return max(s[0], s[1]);
}
__device__ __forceinline__ float half_sum(float x) {
  const auto s = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __uint_as_float(s[0]) + __uint_as_float(s[1]);
}

// A tile of 4 x 4 blocks, from rows of `ld` floats to registers.
struct Rows4 {
  float4 r[4];
};
// The largest magnitude's bits. With kNan, NaN counts as the largest (of the
// non-negative floats the largest as signed integers, of the others as unsigned
// ones); without, it is passed over, for half of the instructions.
template <bool kNan>
__device__ __forceinline__ uint32_t max_abs(uint32_t m, const Rows4 &t) {
  if (kNan) {
    int pos = (int)m;
    uint32_t neg = 0;
#pragma unroll
    for (int r = 0; r < 4; r++) {
      const uint32_t x = __float_as_uint(t.r[r].x), y = __float_as_uint(t.r[r].y), z = __float_as_uint(t.r[r].z), w = __float_as_uint(t.r[r].w);
      pos = max(max(pos, (int)x), (int)y);
      pos = max(max(pos, (int)z), (int)w);
      neg = max(max(neg, x), y);
      neg = max(max(neg, z), w);
    }
    return max((uint32_t)pos, neg & 0x7fffffffu);
  }
  float f = __uint_as_float(m);
#pragma unroll
  for (int r = 0; r < 4; r++) {
    f = fmaxf(fmaxf(f, fabsf(t.r[r].x)), fabsf(t.r[r].y));
    f = fmaxf(fmaxf(f, fabsf(t.r[r].z)), fabsf(t.r[r].w));
  }
  return __float_as_uint(f);
}
// The largest magnitude's bits, NaN passed over, and in *least those of the smallest of the rows' four-element
// largest: a row that lies far below the tile's largest has such four elements (others may have them too).
__device__ __forceinline__ uint32_t max_abs(uint32_t m, const Rows4 &t, uint32_t *least) {
  float f = __uint_as_float(m), q[4];
#pragma unroll
  for (int r = 0; r < 4; r++) q[r] = fmaxf(fmaxf(fabsf(t.r[r].x), fabsf(t.r[r].y)), fmaxf(fabsf(t.r[r].z), fabsf(t.r[r].w)));
  f = fmaxf(fmaxf(f, q[0]), q[1]);
  *least = __float_as_uint(fminf(fminf(q[0], q[1]), fminf(q[2], q[3])));
  return __float_as_uint(fmaxf(fmaxf(f, q[2]), q[3]));
}
// A tile is held at the scale of its largest magnitude where its rows' largest are within 2^kSpread of that, else
// rows are taken times 2^-d, d <= 0, to the largest's binade, and d goes along with the tile. A row of zeros has a
// d below all others: what it is multiplied by counts for nothing, however large.
constexpr int kSpread = 6, kZeroRow = -(1 << 24);
__device__ __forceinline__ bool may_spread(uint32_t least, uint32_t largest) { return least + ((uint32_t)kSpread << 23) < largest; }
// The wavefront's rows, kLanes lanes to four of them kStep apart, in a tile of exponent e; whether one of them lies that
// far below. `rows`: the tile's rows from the first of the lane's four on (behind them are zeros that nothing reads).
template <int kLanes, int kStep>
__device__ __forceinline__ bool lift_rows(Rows4 &t, int e, int rows, int (&d)[4]) {
  bool below = false;
#pragma unroll
  for (int r = 0; r < 4; r++) {
    const uint32_t x = row_max_bits<kLanes>(max_abs(0u, t.r[r]));
    d[r] = x ? min(split_exp(x) - e, 0) : kStep * r < rows ? kZeroRow : 0;
    below = below || d[r] < -kSpread;
  }
  below = __any(below);
#pragma unroll
  for (int r = 0; r < 4; r++) {
    if (!below) d[r] = 0;
    t.r[r] = make_float4(ldexpf(t.r[r].x, -d[r]), ldexpf(t.r[r].y, -d[r]), ldexpf(t.r[r].z, -d[r]), ldexpf(t.r[r].w, -d[r]));
  }
  return below;
}

}  // namespace
}  // namespace ugk
