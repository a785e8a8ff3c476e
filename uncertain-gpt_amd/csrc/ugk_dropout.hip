// ugk_dropout.hip - dropout whose mask is drawn from Philox where it is used
// and never stored (ugk_philox.h: UgkDrop), flat and around the residual add.
//
// A thread takes four consecutive elements, the four words of one Philox block,
// at any alignment (gfx950 accepts a 16-byte access at a 4-byte address). All
// of a thread's loads are issued before the draw, which covers part of their
// latency.
#include "ugk_internal.h"
#include "ugk_philox.h"

namespace ugk {
namespace {

constexpr int kSlots = 2;  // blocks of four elements per thread

// a = result, and for kDropSplit b as well; x, y the inputs of DropForm.
template <DropForm kForm>
__device__ __forceinline__ void drop_apply(float4 &a, float4 &b, float4 x, float4 y, uint64_t block, bool same,
                                           const UgkDrop &d) {
  const float4 t = ugk_drop4(kForm == kDropAddTo ? y : x, block, d);
  const auto add = [](float4 u, float4 v) { return make_float4(u.x + v.x, u.y + v.y, u.z + v.z, u.w + v.w); };
  if constexpr (kForm == kDrop) a = t;
  if constexpr (kForm == kDropAcc) a = add(a, t);
  if constexpr (kForm == kDropAddTo) a = add(x, t);
  if constexpr (kForm == kDropSplit) {
    a = add(a, x);
    b = add(same ? a : b, t);
  }
}

template <DropForm kForm>
__global__ __launch_bounds__(kBlock) void k_dropout(float *a, float *b, const float *x, const float *y, size_t n,
                                                    UgkDrop d) {
  constexpr bool kReadA = kForm == kDropAcc || kForm == kDropSplit, kReadB = kForm == kDropSplit;
  const size_t n4 = n / 4, first = (size_t)blockIdx.x * (kBlock * kSlots) + threadIdx.x;
  const bool same = a == b;
  float4 xv[kSlots], yv[kSlots], av[kSlots], bv[kSlots];
#pragma unroll
  for (int u = 0; u < kSlots; u++) {
    const size_t i = first + (size_t)u * kBlock;
    if (i >= n4) continue;
    xv[u] = ld_nt4(x + 4 * i);
    if (kForm == kDropAddTo) yv[u] = ld_nt4(y + 4 * i);
    if (kReadA) av[u] = ld_nt4(a + 4 * i);
    if (kReadB) bv[u] = ld_nt4(b + 4 * i);
  }
#pragma unroll
  for (int u = 0; u < kSlots; u++) {
    const size_t i = first + (size_t)u * kBlock;
    if (i < n4) {
      drop_apply<kForm>(av[u], bv[u], xv[u], yv[u], i, same, d);
      if (!(kReadB && same)) st_nt4(a + 4 * i, av[u]);
      if (kReadB) st_nt4(b + 4 * i, bv[u]);
    } else if (i == n4 && 4 * n4 < n) {  // the last one to three elements
      float e[4][4] = {};
      for (int j = 0; j < (int)(n - 4 * n4); j++) {
        e[0][j] = x[4 * n4 + j];
        if (kForm == kDropAddTo) e[1][j] = y[4 * n4 + j];
        if (kReadA) e[2][j] = a[4 * n4 + j];
        if (kReadB) e[3][j] = b[4 * n4 + j];
      }
      const auto v = [&](int k) { return make_float4(e[k][0], e[k][1], e[k][2], e[k][3]); };
      float4 ra = v(2), rb = v(3);
      drop_apply<kForm>(ra, rb, v(0), v(1), n4, same, d);
      const float oa[4] = {ra.x, ra.y, ra.z, ra.w}, ob[4] = {rb.x, rb.y, rb.z, rb.w};
      for (int j = 0; j < (int)(n - 4 * n4); j++) {
        if (!(kReadB && same)) a[4 * n4 + j] = oa[j];
        if (kReadB) b[4 * n4 + j] = ob[j];
      }
    }
  }
}

}  // namespace

int launch_dropout(DropForm form, float *a, float *b, const float *x, const float *y, size_t n, const UgkDrop &drop) {
  if (n == 0) return 0;
  const dim3 grid(grid_for((n + 3) / 4, kBlock * kSlots)), block(kBlock);
  switch (form) {
    case kDrop: launch(k_dropout<kDrop>, grid, block, 0, a, b, x, y, n, drop); break;
    case kDropAcc: launch(k_dropout<kDropAcc>, grid, block, 0, a, b, x, y, n, drop); break;
    case kDropAddTo: launch(k_dropout<kDropAddTo>, grid, block, 0, a, b, x, y, n, drop); break;
    case kDropSplit: launch(k_dropout<kDropSplit>, grid, block, 0, a, b, x, y, n, drop); break;
  }
  return check_launch("dropout");
}

}  // namespace ugk
