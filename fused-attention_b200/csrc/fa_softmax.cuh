// Row-per-thread softmax pieces of the tcgen05 forward kernels: a thread holds one query row's
// scores of a K/V tile in registers and its running O in one TMEM lane.
#pragma once

#include "fa_sm100.cuh"

namespace fa {

// P = 2^(S * scale - m) for 32 columns of one row (masked entries, -inf, give 0; the polynomial
// pairs are only used on tiles without masked entries).  kPoly of the 16 pairs, spread over the
// chunk, take the polynomial; the rest go to MUFU ex2.
template <bool BF16, int kPoly>
__device__ __forceinline__ void softmax_chunk(const uint32_t (&r)[32], uint64_t scale2, uint64_t negm2,
                                              uint64_t (&sum2)[4], uint32_t (&pk)[16]) {
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const uint64_t x2 = ffma2(f2u(r[2 * i], r[2 * i + 1]), scale2, negm2);
    // polynomial pairs spread evenly over the chunk (i = 3, 7, 11, 15 for four of them)
    constexpr int kEvery = kPoly > 0 ? 16 / kPoly : 1;
    const bool poly = kPoly > 0 && i % kEvery == kEvery - 1;
    uint64_t p2;
    if (poly)
      p2 = exp2_poly2(x2);
    else
      p2 = f2(ex2_approx(f2lo(x2)), ex2_approx(f2hi(x2)));
    sum2[i & 3] = fadd2(sum2[i & 3], p2);
    pk[i] = pack2<BF16>(f2lo(p2), f2hi(p2));
  }
}

// Row max over NCH 32-column chunks: eight independent chains of the three-input max of sm_100
// (half the instructions of a two-input chain).
template <int NCH>
__device__ __forceinline__ float row_max(const uint32_t (&r)[NCH][32]) {
  float m8[8];
#pragma unroll
  for (int u = 0; u < 8; ++u) m8[u] = -INFINITY;
#pragma unroll
  for (int c = 0; c < NCH; ++c)
#pragma unroll
    for (int i = 0; i < 32; i += 2)
      m8[(c * 16 + i / 2) % 8] = fmax3(m8[(c * 16 + i / 2) % 8], __uint_as_float(r[c][i]), __uint_as_float(r[c][i + 1]));
  return fmaxf(fmax3(m8[0], m8[1], m8[2]), fmax3(m8[3], m8[4], fmax3(m8[5], m8[6], m8[7])));
}

// O row *= alpha in TMEM (D fp32 columns of this thread's lane).
template <int D>
__device__ __forceinline__ void rescale_o(uint32_t t_o, float alpha) {
#pragma unroll 1
  for (int c = 0; c < D / 32; ++c) {
    uint32_t o[32];
    tmem_ld32(t_o + c * 32, o);
    tmem_ld_wait(o);
#pragma unroll
    for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * alpha);
    tmem_st32(t_o + c * 32, o);
  }
}

}  // namespace fa
