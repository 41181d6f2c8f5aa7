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
// Keys are normed and rotated to about 2^-44 of |a| + |b|, for a pair (a, b), and rounded to float32 once
// before that: the value next to a rounding border decides a whole e4m3 step (2^-4 of the value), and so
// the byte is that of a float64 computation, whatever the order of its sums.  The row sums and the root are
// float64; the products and sums of the rotation carry their float32 rounding errors along (each product's
// by a fused multiply-add, each sum's by Knuth's two-sum), which costs ten float32 instructions per element,
// where float64 has to convert every operand on a pipe of 16 lanes.  (A float32 pass that checks a bound on
// its error and repeats what it leaves open was slower: one warp's pass in seven had an open byte, and the
// others of its page waited for it.)
//
// Bound: memory for prompts (2 bytes in, 1 out per element; in practice the instructions around them),
// latency for single tokens (the chain length -> page -> scale).  A (page, head, K or V) slice is what a scale
// has to be agreed on; a block takes one slice after another of the same tokens.  A thread keeps its one or
// two rows through all of them: 16 elements of a row, the row's 8 cosines and sines read once for all heads,
// the next slice's bytes in flight while this one is worked on, and nothing of a slice leaves the registers
// between the maximum and the rounding.  float32 arithmetic goes two values to an instruction.  The tokens of a
// page are found from the first one: a block looks at a window of consecutive tokens and takes every page
// that starts there.
#include "fa_internal.h"
#include "fa_sm100.cuh"

#include <cuda_fp8.h>

namespace fa {
namespace {

constexpr int kAppendThreads = 512;

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

template <int LPR, typename T>
__device__ __forceinline__ T group_sum(T v) {
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

// The table rows of a token, one for each axis (unused entries are the first's).
template <int D>
__device__ __forceinline__ void angle_rows(const AppendParams& p, int t, int at, bool live, size_t (&row)[kRopeMaxAxes]) {
#pragma unroll
  for (int x = 0; x < kRopeMaxAxes; ++x)
    row[x] = x == 0 || x < p.axes ? static_cast<size_t>(live ? append_position(p, x, t, at) : 0) * (D / 2) : row[0];
}
__device__ __forceinline__ size_t angle_place(const AppendParams& p, const size_t (&row)[kRopeMaxAxes], int pair) {
  size_t r = row[0];
#pragma unroll
  for (int x = 1; x < kRopeMaxAxes; ++x)
    if (x < p.axes && pair >= p.section_start[x]) r = row[x];
  return r + pair;
}

// cos and sin of a lane's 8 pairs, two to a register pair.
template <int D>
__device__ __forceinline__ void load_angles(const AppendParams& p, int t, int at, bool live, int l, uint64_t (&c)[4], uint64_t (&s)[4]) {
  size_t row[kRopeMaxAxes];
  angle_rows<D>(p, t, at, live, row);
  if (p.axes == 1) {
    const ulonglong2* pc = reinterpret_cast<const ulonglong2*>(p.cos + row[0] + 8 * l);
    const ulonglong2* ps = reinterpret_cast<const ulonglong2*>(p.sin + row[0] + 8 * l);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const ulonglong2 a = pc[i], b = ps[i];
      c[2 * i] = a.x;
      c[2 * i + 1] = a.y;
      s[2 * i] = b.x;
      s[2 * i + 1] = b.y;
    }
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const size_t a = angle_place(p, row, 8 * l + 2 * i), b = angle_place(p, row, 8 * l + 2 * i + 1);
      c[i] = f2(p.cos[a], p.cos[b]);
      s[i] = f2(p.sin[a], p.sin[b]);
    }
  }
}

template <int D, bool BF16, bool INTER>
__device__ __forceinline__ void load_weights(const AppendParams& p, int o0, int o1, float (&w)[16]) {
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
}

__device__ __forceinline__ uint64_t fneg2(uint64_t v) { return v ^ 0x8000000080000000ull; }

// A sum of float32 pairs and its rounding error (two-sum).
__device__ __forceinline__ void two_sum(uint64_t a, uint64_t b, uint64_t& sum, uint64_t& err) {
  sum = fadd2(a, b);
  const uint64_t bb = fsub2(sum, a);
  err = fadd2(fsub2(a, fsub2(sum, bb)), fsub2(b, bb));
}
// A product and its rounding error.
__device__ __forceinline__ void two_product(uint64_t a, uint64_t b, uint64_t& product, uint64_t& err) {
  product = fmul2(a, b);
  err = ffma2(a, b, fneg2(product));
}

// 1 / sqrt(mean square + eps) of the row whose piece x is, as a sum of two float32 (high, low), for the row times `by`:
// a power of two for rows far from 1, so that neither their products with weights nor the root's low part leave float32.
template <int D>
__device__ __forceinline__ float2 row_root(const uint64_t (&lo)[4], const uint64_t (&hi)[4], double eps, float& by) {
  double sum = 0.0;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const double a = f2lo(lo[j]), b = f2hi(lo[j]), c = f2lo(hi[j]), d = f2hi(hi[j]);
    sum = fma(a, a, fma(b, b, fma(c, c, fma(d, d, sum))));
  }
  const double mean = group_sum<D / 16>(sum) / D + eps;
  const double guess = rsqrtf(static_cast<float>(mean));
  double r = guess * (1.5 - 0.5 * mean * guess * guess);  // one Newton step: 2^-22 -> 2^-43
  by = 1.f;
  if (!(mean > 0x1p-100 && mean < 0x1p100)) {
    by = mean > 1.0 ? 0x1p-64f : 0x1p64f;
    r = 1.0 / sqrt(mean) / by;
  }
  const float high = static_cast<float>(r);
  return make_float2(high, static_cast<float>(r - high));
}

// The defined values of a key row's piece, in place.
template <int D>
__device__ __forceinline__ void define_row(uint64_t (&lo)[4], uint64_t (&hi)[4], bool normed, bool wide_weights,
                                           const uint64_t (&wl)[4], const uint64_t (&wh)[4], bool turned,
                                           const uint64_t (&c)[4], const uint64_t (&s)[4], double eps) {
  uint64_t root = 0, root_low = 0, by2 = 0;
  if (normed) {
    float by;
    const float2 r = row_root<D>(lo, hi, eps, by);
    by2 = f2(by, by);
    root = f2(r.x, r.x);
    root_low = f2(r.y, r.y);
  }
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    uint64_t a = lo[j], b = hi[j], a_low = 0, b_low = 0;
    if (normed) {  // exact with 16-bit weights
      a = fmul2(a, by2);
      b = fmul2(b, by2);
      if (wide_weights) {
        two_product(a, wl[j], a, a_low);
        two_product(b, wh[j], b, b_low);
      } else {
        a = fmul2(a, wl[j]);
        b = fmul2(b, wh[j]);
      }
    }
    uint64_t x = a, x_low = a_low, y = b, y_low = b_low;
    if (turned) {
      uint64_t p, p_low, q, q_low, e;
      const uint64_t ns = fneg2(s[j]);
      two_product(a, c[j], p, p_low);
      two_product(b, ns, q, q_low);
      two_sum(p, q, x, e);
      x_low = fadd2(e, fadd2(p_low, q_low));
      two_product(a, s[j], p, p_low);
      two_product(b, c[j], q, q_low);
      two_sum(p, q, y, e);
      y_low = fadd2(e, fadd2(p_low, q_low));
      if (wide_weights) {
        x_low = fadd2(x_low, ffma2(a_low, c[j], fmul2(b_low, ns)));
        y_low = fadd2(y_low, ffma2(a_low, s[j], fmul2(b_low, c[j])));
      }
    }
    if (normed) {
      uint64_t p, e;
      two_product(x, root, p, e);
      lo[j] = fadd2(p, ffma2(x_low, root, ffma2(x, root_low, e)));
      two_product(y, root, p, e);
      hi[j] = fadd2(p, ffma2(y_low, root, ffma2(y, root_low, e)));
    } else {
      lo[j] = fadd2(x, x_low);
      hi[j] = fadd2(y, y_low);
    }
  }
}

// A lane's 16 elements as 8 pairs, two to a register: lo[i] = first members of pairs 2i, 2i + 1, hi[i] = second.
template <bool BF16, bool INTER>
__device__ __forceinline__ void to_pairs(const uint4& v0, const uint4& v1, uint64_t (&lo)[4], uint64_t (&hi)[4]) {
  float a[8], b[8];
  widen8<BF16>(v0, a);
  widen8<BF16>(v1, b);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (INTER) {
      const float* x = i < 2 ? a + 4 * i : b + 4 * (i - 2);
      lo[i] = f2(x[0], x[2]);
      hi[i] = f2(x[1], x[3]);
    } else {
      lo[i] = f2(a[2 * i], a[2 * i + 1]);
      hi[i] = f2(b[2 * i], b[2 * i + 1]);
    }
  }
}

// Their bytes in memory order.
template <bool INTER>
__device__ __forceinline__ void to_bytes(const uint64_t (&lo)[4], const uint64_t (&hi)[4], uint32_t (&u)[4]) {
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    if constexpr (INTER) {
      u[2 * i] = to_e4m3x4(f2lo(lo[2 * i]), f2lo(hi[2 * i]), f2hi(lo[2 * i]), f2hi(hi[2 * i]));
      u[2 * i + 1] = to_e4m3x4(f2lo(lo[2 * i + 1]), f2lo(hi[2 * i + 1]), f2hi(lo[2 * i + 1]), f2hi(hi[2 * i + 1]));
    } else {
      u[i] = to_e4m3x4(f2lo(lo[2 * i]), f2hi(lo[2 * i]), f2lo(lo[2 * i + 1]), f2hi(lo[2 * i + 1]));
      u[2 + i] = to_e4m3x4(f2lo(hi[2 * i]), f2hi(hi[2 * i]), f2lo(hi[2 * i + 1]), f2hi(hi[2 * i + 1]));
    }
  }
}

// The largest finite magnitude of a lane's 16 values (NaN is passed over).
__device__ __forceinline__ float top_of(const uint64_t (&lo)[4], const uint64_t (&hi)[4]) {
  float top = 0.f;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    top = fmax3(top, fabsf(f2lo(lo[i])), fabsf(f2hi(lo[i])));
    top = fmax3(top, fabsf(f2lo(hi[i])), fabsf(f2hi(hi[i])));
  }
  if (top == INFINITY) {
    top = 0.f;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float v[4] = {fabsf(f2lo(lo[i])), fabsf(f2hi(lo[i])), fabsf(f2lo(hi[i])), fabsf(f2hi(hi[i]))};
#pragma unroll
      for (int j = 0; j < 4; ++j) top = fmaxf(top, v[j] < INFINITY ? v[j] : 0.f);
    }
  }
  return top;
}

// grid: x = token windows, y = ranges of slices (slice s: keys of head s / 2 if even, its values if odd).
template <int D, bool BF16, bool INTER, int NR>
__global__ void __launch_bounds__(kAppendThreads, 1) append_kernel(const __grid_constant__ AppendParams p) {
  constexpr int LPR = D / 16;
  __shared__ float warp_max[2][kAppendThreads / 32];
  const int status = ld_status(p.status);  // looked at before the first store
  const int rows = blockDim.x / LPR;       // rows of a pass
  const int l = threadIdx.x % LPR, group = threadIdx.x / LPR;
  const int o0 = INTER ? 16 * l : 8 * l, o1 = INTER ? 16 * l + 8 : D / 2 + 8 * l;
  const int s0 = blockIdx.y * p.slices, s1 = min(2 * p.H_kv, s0 + p.slices);
  const int P = 1 << p.page_shift;
  const bool normed = p.k_weight != nullptr, turned = p.cos != nullptr;
  uint64_t wl[4], wh[4];  // the norm's weights of this lane
  if (normed) {
    float w[16];
    load_weights<D, BF16, INTER>(p, o0, o1, w);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      wl[i] = INTER ? f2(w[4 * i], w[4 * i + 2]) : f2(w[2 * i], w[2 * i + 1]);
      wh[i] = INTER ? f2(w[4 * i + 1], w[4 * i + 3]) : f2(w[8 + 2 * i], w[8 + 2 * i + 1]);
    }
  }

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
    const int len = p.seq_lens[b];
    if (len < 0) {  // not a length; far below zero the place would wrap around
      if (threadIdx.x == 0) record_error(p.status, kDevBadIndex, b);
      return;
    }
    const int at = len - (end - t);            // the token's place in its sequence
    if (at < 0) {                              // a token before the sequence's start has no place
      t += min(-at, end - t);
      if (p.offsets == nullptr) b = t;
      continue;
    }
    const int slot = at & (P - 1);
    const int count = min(P - slot, end - t);
    if (t == first || slot == 0) {
      const int index = at >> p.page_shift;
      const int page = index < p.width ? p.block_table[b * p.table_stride + index] : -1;
      auto row_of = [&](int s, int r) {
        return (s & 1) == 0 ? static_cast<const uint16_t*>(p.k) + (t + r) * p.k_stride[0] + (s >> 1) * p.k_stride[1]
                            : static_cast<const uint16_t*>(p.v) + (t + r) * p.v_stride[0] + (s >> 1) * p.v_stride[1];
      };
      uint4 raw[NR][2];
      auto fetch = [&](int s) {
#pragma unroll
        for (int i = 0; i < NR; ++i) {
          raw[i][0] = raw[i][1] = make_uint4(0, 0, 0, 0);
          if (i * rows + group < count) {
            const uint16_t* row = row_of(s, i * rows + group);
            raw[i][0] = *reinterpret_cast<const uint4*>(row + o0);
            raw[i][1] = *reinterpret_cast<const uint4*>(row + o1);
          }
        }
      };
      fetch(s0);
      uint64_t cs[NR][4], sn[NR][4];
      if (turned) {
#pragma unroll
        for (int i = 0; i < NR; ++i) {
          const int r = i * rows + group;
          load_angles<D>(p, t + r, at + r, r < count, l, cs[i], sn[i]);
        }
      }
      if (page < 0 || page >= p.num_pages) {  // the same in every thread
        if (threadIdx.x == 0) record_error(p.status, kDevBadIndex, b);
        return;
      }
      if (__syncthreads_or(status) != 0) return;
#pragma unroll 1
      for (int s = s0; s < s1; ++s) {
        const bool key = (s & 1) == 0;
        const size_t ph = static_cast<size_t>(page) * p.H_kv + (s >> 1);
        uint8_t* out = (key ? p.k_pages : p.v_pages) + (ph << p.page_shift) * D;
        float* scales = key ? p.k_scales : p.v_scales;
        const float old = slot > 0 ? scales[ph] : 0.f;
        uint64_t lo[NR][4], hi[NR][4];
#pragma unroll
        for (int i = 0; i < NR; ++i) to_pairs<BF16, INTER>(raw[i][0], raw[i][1], lo[i], hi[i]);
        if (s + 1 < s1) fetch(s + 1);
        if (key && (normed || turned)) {
#pragma unroll
          for (int i = 0; i < NR; ++i) define_row<D>(lo[i], hi[i], normed, normed && p.weight_f32, wl, wh, turned, cs[i], sn[i], p.eps);
        }
        // The slice's largest magnitude over all rows (one barrier: two slices' words alternate).
        auto slice_top = [&](float top, float (&words)[kAppendThreads / 32]) {
          top = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(top)));  // magnitudes order like their bits
          if (blockDim.x == 32) return top;
          if (threadIdx.x % 32 == 0) words[threadIdx.x / 32] = top;
          __syncthreads();
          for (int i = 0; i < static_cast<int>(blockDim.x) / 32; ++i) top = fmaxf(top, words[i]);
          return top;
        };
        float mine = 0.f;
#pragma unroll
        for (int i = 0; i < NR; ++i)  // rows behind the last are zeros
          mine = fmaxf(mine, top_of(lo[i], hi[i]));
        const float top = slice_top(mine, warp_max[s & 1]);
        const float scale = fmaxf(scale_for(top), old);
        const float inv = 1.f / scale;
        if (slot > 0 && scale > old) {  // the older tokens under the grown scale
          const float ratio = old * inv;
          for (int r = group; r < slot; r += rows) {
            uint4* row = reinterpret_cast<uint4*>(out + static_cast<size_t>(r) * D + 16 * l);
            const uint4 v = *row;
            uint32_t u[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              const float2 a = from_e4m3x2(u[j] & 0xffffu), c = from_e4m3x2(u[j] >> 16);
              u[j] = to_e4m3x4(a.x * ratio, a.y * ratio, c.x * ratio, c.y * ratio);
            }
            *row = make_uint4(u[0], u[1], u[2], u[3]);
          }
        }
        const uint64_t inv2 = f2(inv, inv);
#pragma unroll
        for (int i = 0; i < NR; ++i) {
          if (i * rows >= count) continue;
          const int r = i * rows + group;
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            lo[i][j] = fmul2(lo[i][j], inv2);
            hi[i][j] = fmul2(hi[i][j], inv2);
          }
          uint32_t u[4];
          to_bytes<INTER>(lo[i], hi[i], u);
          if (r < count) {
            uint8_t* row = out + static_cast<size_t>(slot + r) * D;
            *reinterpret_cast<uint2*>(row + o0) = make_uint2(u[0], u[1]);
            *reinterpret_cast<uint2*>(row + o1) = make_uint2(u[2], u[3]);
          }
        }
        if (threadIdx.x == 0) scales[ph] = scale;
      }
      __syncthreads();  // the next page's slices use the same words
    }
    t += count;
    if (p.offsets == nullptr) b = t;
  }
}

template <int D, bool BF16, bool INTER>
cudaError_t launch_append_t(const AppendParams& p, dim3 grid, int threads, bool two, cudaStream_t stream) {
  if (two)
    append_kernel<D, BF16, INTER, 2><<<grid, threads, 0, stream>>>(p);
  else
    append_kernel<D, BF16, INTER, 1><<<grid, threads, 0, stream>>>(p);
  return cudaGetLastError();
}

}  // namespace

cudaError_t launch_append(AppendParams p, int D, bool bf16, bool interleaved, cudaStream_t stream) {
  // The rows of a unit: one token per sequence, or up to a page.
  const int unit = p.offsets == nullptr ? 1 : (1 << p.page_shift < p.T ? 1 << p.page_shift : p.T);
  const int lanes = D / 16;
  // Two rows a thread where there are two, one for single tokens.
  const bool two = unit * lanes > 32;
  int threads = 32;
  while ((two ? 2 : 1) * threads < unit * lanes) threads *= 2;
  // A window as long as the sequences' new tokens on average, up to a page: then about one page starts in it
  // (a block takes its pages one after another).
  const int per_sequence = p.T / p.B;
  p.window = 1;
  while (2 * p.window <= (1 << p.page_shift) && 2 * p.window <= per_sequence) p.window *= 2;
  // As many slices for a block as leave 32 warps to every SM.
  const long long windows = (p.T + p.window - 1) / p.window;
  p.slices = 1;
  while (p.slices < 2 * p.H_kv && windows * ((2 * p.H_kv + 2 * p.slices - 1) / (2 * p.slices)) * (threads / 32) >= 148 * 32) p.slices *= 2;
  const dim3 grid(static_cast<unsigned>(windows), (2 * p.H_kv + p.slices - 1) / p.slices);
#define FA_APPEND_CASE(DD, BB, II)                                       \
  if (D == DD && bf16 == BB && interleaved == II) return launch_append_t<DD, BB, II>(p, grid, threads, two, stream);
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
