// Shared by the kernels of attention over the paged cache.
#pragma once

#include "fa_internal.h"
#include "fa_sm100.cuh"

namespace fa {

// The bytes of w that are NaN in e4m3 (0x7f, 0xff), as a mask of whole bytes.
__device__ __forceinline__ uint32_t nan_bytes(uint32_t w) {
  return ((((w & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u) >> 7) * 0xffu;
}

// Output rows of tokens that no sequence has: o = 0, lse = -inf.  The grid's blocks share them; usually there are none.
template <int D>
__device__ __forceinline__ void clear_unowned_rows(const PagedParams& p) {
  if (!p.clear_unowned || p.offsets == nullptr) return;
  const int first = min(max(p.offsets[0], 0), p.T), end = min(max(p.offsets[p.B], 0), p.T);
  const int heads = p.H_kv * p.group;
  for (int i = blockIdx.x; i < first + p.T - end; i += gridDim.x) {
    const long long t = i < first ? i : end + (i - first);
    for (int j = threadIdx.x; j < heads * (D / 8); j += blockDim.x) {
      const int h = j / (D / 8), d = j % (D / 8) * 8;
      *reinterpret_cast<uint4*>(static_cast<uint16_t*>(p.out) + t * p.out_stride[0] + h * p.out_stride[1] + d) = make_uint4(0, 0, 0, 0);
      if (p.lse != nullptr && d == 0) p.lse[t * heads + h] = -INFINITY;
    }
  }
}

}  // namespace fa
