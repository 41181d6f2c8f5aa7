// Appending keys and values to a paged e4m3 cache, with the keys' RMS norm and rotary rotation on
// the way, for sm_100a.
//
// A page holds page_size tokens of one K/V head, [num_pages, H_kv, page_size, D] bytes, with one
// float32 scale per (page, head): a stored byte c stands for float(c) * scale.  The tokens of one
// call that fall into one page are rounded together:
//   need  = 2^e, the smallest e >= -126 with amax <= 448 * 2^e   (amax: finite magnitudes)
//   scale = need, or max(need, old scale) when the page holds older tokens of the sequence
//   c     = e4m3(x / scale), round to nearest even; +-inf saturates at +-448, NaN stays NaN
// Older tokens of a page whose scale grows are rounded again, c' = e4m3(c * old / scale).  Scales
// are powers of two because x / scale is then exact: e4m3 is a floating format, so a power of two
// costs no precision, and a grown scale changes older tokens only where they become subnormal.
//
// Keys are normed and rotated in float64 and rounded to float32 once before that: the value next to
// a rounding border decides a whole e4m3 step (2^-4 of the value), and with float64 the byte does
// not depend on the order of the sums.
//
// Bound: memory for prompts (2 bytes in, 1 out per element), latency for single tokens (the chain
// length -> page -> scale).  One block owns a (page, head, K or V) unit, the unit whose scale has to
// be agreed on: all its rows stay in registers between the maximum and the rounding, so the input
// is read once.  A unit is found from its first token: a block looks at a window of consecutive
// tokens and takes every unit that starts there.  Windows are one token for decoding and grow with
// the number of tokens.
#include "fa_internal.h"
#include "fa_sm100.cuh"

#include <cuda_fp8.h>

namespace fa {
namespace {

// 8 consecutive 16-bit elements -> float32.
template <bool BF16>
__device__ __forceinline__ void widen8(const uint4& v, float* f) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (BF16) {
      f[2 * i] = __uint_as_float(w[i] << 16);
      f[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    } else {
      const float2 t = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
      f[2 * i] = t.x;
      f[2 * i + 1] = t.y;
    }
  }
}

__device__ __forceinline__ uint32_t to_e4m3x4(float a, float b, float c, float d) {
  const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3);
  const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(c, d), __NV_SATFINITE, __NV_E4M3);
  return lo | (hi << 16);
}

__device__ __forceinline__ float2 from_e4m3x2(uint32_t v) {
  const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2(static_cast<__nv_fp8x2_storage_t>(v), __NV_E4M3);
  return __half22float2(__half2(h));
}

// 2^e, the smallest e >= -126 with amax <= 448 * 2^e = 0.875 * 2^(e + 9).
__device__ __forceinline__ float scale_for(float amax) {
  const uint32_t bits = __float_as_uint(amax);
  const int exponent = static_cast<int>(bits >> 23) - 126;  // amax = f * 2^exponent, f in [1/2, 1)
  int e = exponent - 9 + ((bits & 0x7fffffu) > 0x600000u ? 1 : 0);
  e = max(e, -126);
  return __uint_as_float(static_cast<uint32_t>(e + 127) << 23);
}

template <int LPR>
__device__ __forceinline__ double group_sum(double v) {
#pragma unroll
  for (int o = LPR / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

__device__ __forceinline__ int append_position(const AppendParams& p, int axis, int t, int at) {
  long long v = at;
  if (p.pos != nullptr) {
    const long long i = axis * p.pos_axis_stride + t;
    v = p.pos64 ? static_cast<const long long*>(p.pos)[i] : static_cast<const int*>(p.pos)[i];
  }
  if (v < 0 || v >= p.max_pos) {
    record_error(p.status, kDevBadIndex, t);
    v = 0;
  }
  return static_cast<int>(v);
}

// A key row's 16 elements of this lane (f: the elements at o0.., then at o1..), normed and rotated
// in float64.  Every lane of the warp calls it (row sums are shuffles).
template <int D, bool BF16, bool INTER>
__device__ __forceinline__ void key_row(const AppendParams& p, int t, int at, bool live, int l, int o0, int o1,
                                        float (&f)[16]) {
  double d[16];
#pragma unroll
  for (int i = 0; i < 16; ++i) d[i] = static_cast<double>(f[i]);
  if (p.k_weight != nullptr) {
    double sum = 0.0;
#pragma unroll
    for (int i = 0; i < 16; ++i) sum += d[i] * d[i];
    const double r = 1.0 / sqrt(group_sum<D / 16>(sum) / D + p.eps);
    float w[16];
    if (p.weight_f32) {
      const float* wf = static_cast<const float*>(p.k_weight);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        w[i] = wf[o0 + i];
        w[8 + i] = wf[o1 + i];
      }
    } else {
      const uint16_t* wh = static_cast<const uint16_t*>(p.k_weight);
      widen8<BF16>(*reinterpret_cast<const uint4*>(wh + o0), w);
      widen8<BF16>(*reinterpret_cast<const uint4*>(wh + o1), w + 8);
    }
#pragma unroll
    for (int i = 0; i < 16; ++i) d[i] = d[i] * r * static_cast<double>(w[i]);
  }
  if (p.cos != nullptr) {
    int row[kRopeMaxAxes];
#pragma unroll
    for (int a = 0; a < kRopeMaxAxes; ++a) row[a] = live && a < p.axes ? append_position(p, a, t, at) : 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int pair = 8 * l + i;
      int r = row[0];
#pragma unroll
      for (int a = 1; a < kRopeMaxAxes; ++a)
        if (a < p.axes && pair >= p.section_start[a]) r = row[a];
      const size_t where = static_cast<size_t>(r) * (D / 2) + pair;
      const double c = p.cos[where], s = p.sin[where];
      double& lo = INTER ? d[2 * i] : d[i];
      double& hi = INTER ? d[2 * i + 1] : d[8 + i];
      const double x = lo, y = hi;
      lo = x * c - y * s;
      hi = x * s + y * c;
    }
  }
#pragma unroll
  for (int i = 0; i < 16; ++i) f[i] = static_cast<float>(d[i]);
}

// grid: x = token windows, y = K/V heads, z = 0 keys, 1 values.
template <int D, bool BF16, bool INTER, int NPASS>
__global__ void __launch_bounds__(256) append_kernel(const AppendParams p) {
  constexpr int LPR = D / 16;
  __shared__ uint32_t warp_max[8];
  if (__syncthreads_or(ld_status(p.status)) != 0) return;
  const int h = blockIdx.y;
  const bool key = blockIdx.z == 0;
  const int rows = blockDim.x / LPR;  // rows of a pass
  const int l = threadIdx.x % LPR, group = threadIdx.x / LPR;
  const int o0 = INTER ? 16 * l : 8 * l, o1 = INTER ? 16 * l + 8 : D / 2 + 8 * l;
  const uint16_t* x = static_cast<const uint16_t*>(key ? p.k : p.v) + h * (key ? p.k_stride[1] : p.v_stride[1]);
  const long long x_token = key ? p.k_stride[0] : p.v_stride[0];
  uint8_t* pages = key ? p.k_pages : p.v_pages;
  float* scales = key ? p.k_scales : p.v_scales;
  const int P = p.page_size;

  int t = blockIdx.x * p.window;
  const int t_end = min(p.T, t + p.window);
  // the sequence of the window's first token: the last b with offsets[b] <= t
  int b = t;
  if (p.offsets != nullptr) {
    int lo = 0, hi = p.B;  // offsets[lo] <= t (offsets[0] = 0 is the caller's) < offsets[hi] or hi = B
    while (hi - lo > 1) {
      const int mid = (lo + hi) / 2;
      if (p.offsets[mid] <= t)
        lo = mid;
      else
        hi = mid;
    }
    b = lo;
  }
  while (t < t_end) {
    int first = t, end = t + 1;
    if (p.offsets != nullptr) {
      while (b < p.B && p.offsets[b + 1] <= t) ++b;
      if (b >= p.B) return;  // rows behind the last sequence
      first = p.offsets[b];
      end = p.offsets[b + 1];
      if (first < 0 || first > t || end > p.T) {
        if (threadIdx.x == 0) record_error(p.status, kDevBadIndex, b);
        return;
      }
    } else if (b >= p.B) {
      return;
    }
    const int at = p.seq_lens[b] - (end - t);  // the token's place in its sequence
    if (at < 0) {                              // a token before the sequence's start has no place
      t += min(-at, end - t);
      if (p.offsets == nullptr) b = t;
      continue;
    }
    const int slot = at % P;
    const int count = min(P - slot, end - t);
    if (t == first || slot == 0 || at == 0) {
      const int index = at / P;
      const int page = index < p.width ? p.block_table[b * p.table_stride + index] : -1;
      if (page < 0 || page >= p.num_pages) {
        if (threadIdx.x == 0) record_error(p.status, kDevBadIndex, b);
        return;
      }
      const size_t ph = static_cast<size_t>(page) * p.H_kv + h;
      uint8_t* out = pages + ph * P * D;
      const float old = slot > 0 ? scales[ph] : 0.f;
      float f[NPASS][16];
      uint32_t top = 0;
#pragma unroll
      for (int i = 0; i < NPASS; ++i) {
        const int r = i * rows + group;
        const bool live = r < count;
        uint4 a = make_uint4(0, 0, 0, 0), c = a;
        if (live) {
          const uint16_t* row = x + (t + r) * x_token;
          a = *reinterpret_cast<const uint4*>(row + o0);
          c = *reinterpret_cast<const uint4*>(row + o1);
        }
        widen8<BF16>(a, f[i]);
        widen8<BF16>(c, f[i] + 8);
        if (key && i * rows < count) key_row<D, BF16, INTER>(p, t + r, at + r, live, l, o0, o1, f[i]);
        if (live) {
#pragma unroll
          for (int j = 0; j < 16; ++j) {
            const uint32_t m = __float_as_uint(f[i][j]) & 0x7fffffffu;
            if (m < 0x7f800000u) top = max(top, m);  // magnitudes order like their bits
          }
        }
      }
      top = __reduce_max_sync(0xffffffffu, top);
      if (threadIdx.x % 32 == 0) warp_max[threadIdx.x / 32] = top;
      __syncthreads();
      for (int w = 0; w < static_cast<int>(blockDim.x) / 32; ++w) top = max(top, warp_max[w]);
      const float scale = fmaxf(scale_for(__uint_as_float(top)), old);
      const float inv = 1.f / scale;
      if (slot > 0 && scale > old) {  // the older tokens under the grown scale
        const float ratio = old * inv;
        for (int r = group; r < slot; r += rows) {
          uint4* row = reinterpret_cast<uint4*>(out + static_cast<size_t>(r) * D + 16 * l);
          const uint4 v = *row;
          uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const float2 lo = from_e4m3x2(w[j] & 0xffffu), hi = from_e4m3x2(w[j] >> 16);
            w[j] = to_e4m3x4(lo.x * ratio, lo.y * ratio, hi.x * ratio, hi.y * ratio);
          }
          *row = make_uint4(w[0], w[1], w[2], w[3]);
        }
      }
#pragma unroll
      for (int i = 0; i < NPASS; ++i) {
        const int r = i * rows + group;
        if (r < count) {
          uint8_t* row = out + static_cast<size_t>(slot + r) * D;
          uint32_t w[4];
#pragma unroll
          for (int j = 0; j < 4; ++j)
            w[j] = to_e4m3x4(f[i][4 * j] * inv, f[i][4 * j + 1] * inv, f[i][4 * j + 2] * inv, f[i][4 * j + 3] * inv);
          *reinterpret_cast<uint2*>(row + o0) = make_uint2(w[0], w[1]);
          *reinterpret_cast<uint2*>(row + o1) = make_uint2(w[2], w[3]);
        }
      }
      if (threadIdx.x == 0) scales[ph] = scale;
      __syncthreads();  // warp_max is free again
    }
    t += count;
    if (p.offsets == nullptr) b = t;
  }
}

template <int D, bool BF16, bool INTER>
void launch_append_t(const AppendParams& p, dim3 grid, int threads, int passes, cudaStream_t stream) {
  if (passes == 1)
    append_kernel<D, BF16, INTER, 1><<<grid, threads, 0, stream>>>(p);
  if constexpr (D >= 64)
    if (passes == 2) append_kernel<D, BF16, INTER, 2><<<grid, threads, 0, stream>>>(p);
  if constexpr (D >= 128)
    if (passes == 4) append_kernel<D, BF16, INTER, 4><<<grid, threads, 0, stream>>>(p);
}

}  // namespace

cudaError_t launch_append(AppendParams p, int D, bool bf16, bool interleaved, cudaStream_t stream) {
  // The rows of a unit: one token per sequence, or up to a page.
  const int unit = p.offsets == nullptr ? 1 : (p.page_size < p.T ? p.page_size : p.T);
  const int lanes = D / 16;
  int threads = 64, passes = 1;
  if (unit * lanes > threads) {
    threads = 256;
    while (passes * threads < unit * lanes) passes *= 2;
  }
  // Windows as short as the grid allows: a block takes its units one after another.
  const long long per_token = 2LL * p.H_kv;
  p.window = 1;
  while (p.window < p.page_size && (p.T + p.window - 1) / p.window * per_token > 148 * 32) p.window *= 2;
  const dim3 grid((p.T + p.window - 1) / p.window, p.H_kv, 2);
#define FA_APPEND_CASE(DD, BB, II)                                       \
  if (D == DD && bf16 == BB && interleaved == II) {                      \
    launch_append_t<DD, BB, II>(p, grid, threads, passes, stream);       \
    return cudaGetLastError();                                           \
  }
#define FA_APPEND_CASES(DD) \
  FA_APPEND_CASE(DD, false, false) FA_APPEND_CASE(DD, false, true) FA_APPEND_CASE(DD, true, false) FA_APPEND_CASE(DD, true, true)
  FA_APPEND_CASES(32)
  FA_APPEND_CASES(64)
  FA_APPEND_CASES(128)
#undef FA_APPEND_CASE
#undef FA_APPEND_CASES
  return cudaErrorInvalidValue;
}

}  // namespace fa
