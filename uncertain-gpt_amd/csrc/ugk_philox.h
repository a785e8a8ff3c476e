// ugk_philox.h - counter-based normal draws, eps = f(seed, step, index).
//
// Philox4x32-10 (Salmon et al., "Parallel random numbers: as easy as 1, 2, 3",
// SC'11): four 32-bit counter words, a two-word key, ten rounds of two
// 32x32->64 multiplies (constants 0xD2511F53, 0xCD9E8D57) and a Weyl key
// schedule (0x9E3779B9, 0xBB67AE85). The stream is the one of
// gpt2_kernels.cuh:148-192 (philox4x32_10, u01, philox_normal): counter
// {index low, index high, step, 0}, key {seed low, seed high}, the first two
// output words mapped to (0,1) as ((float)x + 0.5f) * 2^-32, and one
// Box-Muller cosine branch per index.
//
// The integer part is exact on host and device. The float part, in the
// glibc-exact form, takes glibc's logf and cosf as ugk_libm.h restates them
// (equal to the host glibc on every input of their domains) and the correctly
// rounded square root, so that eps equals the host's bit for bit; in the ops'
// default (fast-math) form, the radius from the hardware log2 and square root
// and the device library's cosf sequence (ugk_dev_box_muller_fast).
#pragma once

#include <stdint.h>

#ifdef __HIPCC__
#include <hip/hip_runtime.h>

#include "ugk_libm_dev.h"
#define UGK_PHILOX_HD __host__ __device__ __forceinline__
#else
#define UGK_PHILOX_HD static inline
#endif

struct UgkPhilox4 {
  uint32_t w[4];
};

// Ten rounds; each 32x32 product is one 64-bit multiply (one v_mad_u64_u32).
UGK_PHILOX_HD UgkPhilox4 ugk_philox4x32_10(uint32_t c0, uint32_t c1, uint32_t c2, uint32_t c3,
                                           uint32_t k0, uint32_t k1) {
#pragma unroll
  for (int r = 0; r < 10; r++) {
    const uint64_t p0 = (uint64_t)0xD2511F53u * c0;
    const uint64_t p1 = (uint64_t)0xCD9E8D57u * c2;
    const uint32_t n0 = (uint32_t)(p1 >> 32) ^ c1 ^ k0;
    const uint32_t n2 = (uint32_t)(p0 >> 32) ^ c3 ^ k1;
    c1 = (uint32_t)p1;
    c3 = (uint32_t)p0;
    c0 = n0;
    c2 = n2;
    k0 += 0x9E3779B9u;
    k1 += 0xBB67AE85u;
  }
  return UgkPhilox4{{c0, c1, c2, c3}};
}

// uint32 -> (0, 1]: the conversion rounds to nearest, the add and the
// multiply by 2^-32 round separately (no contraction).
UGK_PHILOX_HD float ugk_u01(uint32_t x) { return ((float)x + 0.5f) * 2.3283064365386963e-10f; }

UGK_PHILOX_HD UgkPhilox4 ugk_philox_words(unsigned long long seed, int step, uint64_t index) {
  return ugk_philox4x32_10((uint32_t)index, (uint32_t)(index >> 32), (uint32_t)step, 0u,
                           (uint32_t)seed, (uint32_t)(seed >> 32));
}

#ifdef __HIPCC__
// Dropout's parameters. Element i stays where word i % 4 of the Philox block i / 4
// (counter {i / 4 low, high, step, stream}) is at least `below` = p 2^32, rounded;
// it is then multiplied by `scale` = 1 / (1 - p). The block serves four elements,
// so the draw costs a quarter of an eps draw's integer work per element, and the
// probability is exact to 2^-33.
struct UgkDrop {
  unsigned long long seed;
  int step;
  uint32_t stream, below;
  float scale;
};

// a ^ b ^ k in one v_bitop3_b32 (truth table 0x96), k in a scalar register.
// Only for a k that is the same in every lane of the wavefront.
__device__ __forceinline__ uint32_t ugk_xor3_uniform(uint32_t a, uint32_t b, uint32_t k) {
  uint32_t r;
  asm("v_bitop3_b32 %0, %1, %2, %3 bitop3:0x96" : "=v"(r) : "v"(a), "v"(b), "s"(k));
  return r;
}

// ugk_philox_words for a (seed, step) shared by the whole wavefront (the
// kernels draw eps(seed, step, i) for their own i): the same rounds, with each
// round's two three-way xors as one instruction each, the round key scalar.
// The fourth counter word (0 for eps) keeps streams of one seed and step apart.
__device__ __forceinline__ UgkPhilox4 ugk_dev_philox_words_uniform(unsigned long long seed, int step,
                                                                  uint64_t index, uint32_t stream = 0u) {
  uint32_t c0 = (uint32_t)index, c1 = (uint32_t)(index >> 32), c2 = (uint32_t)step, c3 = stream;
  uint32_t k0 = (uint32_t)seed, k1 = (uint32_t)(seed >> 32);
#pragma unroll
  for (int r = 0; r < 10; r++) {
    const uint64_t p0 = (uint64_t)0xD2511F53u * c0;
    const uint64_t p1 = (uint64_t)0xCD9E8D57u * c2;
    const uint32_t n0 = ugk_xor3_uniform((uint32_t)(p1 >> 32), c1, k0);
    const uint32_t n2 = ugk_xor3_uniform((uint32_t)(p0 >> 32), c3, k1);
    c1 = (uint32_t)p1;
    c3 = (uint32_t)p0;
    c0 = n0;
    c2 = n2;
    k0 += 0x9E3779B9u;
    k1 += 0xBB67AE85u;
  }
  return UgkPhilox4{{c0, c1, c2, c3}};
}

// Box-Muller, cosine branch, as gpt2_kernels.cuh:181-192 writes it and the
// host builds it: sqrtf(-2 logf(u1)) * cosf(2 pi u2), with 2 pi rounded to
// float and the product rounded before the cosine. u1 in [2^-33, 1] is a
// normal float and 2 pi u2 lies in (0, 2 pi], inside the domains of the
// restated logf and cosf (ugk_logf_normal, ugk_cosf_small); -2 ln u1 is -0 or
// in [1.1e-7, 46], inside the domain of the correctly rounded square root
// without rescaling. The same bits as the host's for every u1, u2.
__device__ __forceinline__ float ugk_dev_box_muller(uint32_t a, uint32_t b) {
  const float u1 = ugk_u01(a), u2 = ugk_u01(b);
  const float l = ugk_logf_normal(u1);
  const float x = 6.28318530717958647692f * u2;
  return ugk_dev_sqrtf_large(-2.0f * l) * ugk_cosf_small(x);
}

// The same transform with the radius from the hardware log2 and square root
// (v_log_f32, v_sqrt_f32), as a fast-math build computes it: -2 ln u1 as
// log2(u1) times -2 ln 2, rounded once, and a square root within 1 ulp; the
// cosine the device library's (ugk_dev_cosf_small, float arithmetic). The
// Philox ops' default form.
__device__ __forceinline__ float ugk_dev_bm_radius_fast(float u1) {
  return __builtin_amdgcn_sqrtf((-2.0f * __builtin_amdgcn_logf(u1)) * 0x1.62e43p-1f);
}

__device__ __forceinline__ float ugk_dev_box_muller_fast(uint32_t a, uint32_t b) {
  const float u1 = ugk_u01(a), u2 = ugk_u01(b);
  return ugk_dev_bm_radius_fast(u1) * ugk_dev_cosf_small(6.28318530717958647692f * u2);
}

// eps(seed, step, index); seed and step must be the same across the wavefront.
__device__ __forceinline__ float ugk_dev_philox_normal(unsigned long long seed, int step, uint64_t index) {
  const UgkPhilox4 o = ugk_dev_philox_words_uniform(seed, step, index);
  return ugk_dev_box_muller(o.w[0], o.w[1]);
}

__device__ __forceinline__ float ugk_dev_philox_normal_fast(unsigned long long seed, int step, uint64_t index) {
  const UgkPhilox4 o = ugk_dev_philox_words_uniform(seed, step, index);
  return ugk_dev_box_muller_fast(o.w[0], o.w[1]);
}

// Elements 4 block .. 4 block + 3 that stay: v[j] scaled, else +0 (whatever v[j]
// is, infinities and NaN too). The parameters must be the same across the wavefront.
__device__ __forceinline__ float4 ugk_drop4(float4 v, uint64_t block, const UgkDrop &d) {
  const UgkPhilox4 o = ugk_dev_philox_words_uniform(d.seed, d.step, block, d.stream);
  return make_float4(o.w[0] >= d.below ? v.x * d.scale : 0.0f, o.w[1] >= d.below ? v.y * d.scale : 0.0f,
                     o.w[2] >= d.below ? v.z * d.scale : 0.0f, o.w[3] >= d.below ? v.w * d.scale : 0.0f);
}

// The same for elements i .. i + 3, i any number: they lie in two blocks unless i is a multiple of 4.
__device__ __forceinline__ float4 ugk_drop4_at(float4 v, uint64_t i, const UgkDrop &d) {
  const unsigned sh = (unsigned)i & 3u;
  const UgkPhilox4 a = ugk_dev_philox_words_uniform(d.seed, d.step, i >> 2, d.stream);
  uint32_t w0 = a.w[0], w1 = a.w[1], w2 = a.w[2], w3 = a.w[3];
  if (sh) {
    const UgkPhilox4 b = ugk_dev_philox_words_uniform(d.seed, d.step, (i >> 2) + 1, d.stream);
    w0 = sh == 1 ? a.w[1] : sh == 2 ? a.w[2] : a.w[3];
    w1 = sh == 1 ? a.w[2] : sh == 2 ? a.w[3] : b.w[0];
    w2 = sh == 1 ? a.w[3] : sh == 2 ? b.w[0] : b.w[1];
    w3 = sh == 1 ? b.w[0] : sh == 2 ? b.w[1] : b.w[2];
  }
  return make_float4(w0 >= d.below ? v.x * d.scale : 0.0f, w1 >= d.below ? v.y * d.scale : 0.0f,
                     w2 >= d.below ? v.z * d.scale : 0.0f, w3 >= d.below ? v.w * d.scale : 0.0f);
}
#endif
