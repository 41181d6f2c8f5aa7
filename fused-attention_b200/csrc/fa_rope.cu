// Per-head RMS norm of queries and keys with the rotary position rotation in the same pass,
// forward and backward, for sm_100a.
//
//   r = 1 / sqrt(mean(x^2) + eps),  y = x r w            (skipped where no weight is given)
//   pair (a, b) of y at position p:  z = (a c - b s, a s + b c),  c, s = cos/sin[p(axis of pair), pair]
//   backward, dz given:  dy = (da c + db s, db c - da s),  g = dy w,
//     dx = r (g - x r^2 mean(g x)),   dw = sum over rows of dy x r
// A pair is (i, i + D/2), or (2i, 2i + 1) when interleaved.  Sums and products are float32; each
// output is rounded once.
//
// Bound: memory.  Every element is read and written once (backward: x and dz read, dx written), so
// the layout is chosen for wide accesses and for reading the tables once per token instead of once
// per row: a group of D/16 lanes owns a token, keeps its 8 cosines and 8 sines per lane in
// registers and walks heads of that token, 16 elements (two 16-byte accesses) a lane and row.  The
// pairs a lane needs are all its own, so only the row sums cross lanes (log2(D/16) shuffles).
// kUnroll rows are loaded before the first is used.  Few tokens are spread out by giving each group
// fewer heads (the host picks heads per group).  Measured, bf16, D = 128, 32 + 8 heads: forward over 32768
// tokens 117 us, 5.9 TB/s or 90 % of the measured copy rate; over 8192 tokens forward 34 us, backward 56 us.
// The weight gradients are summed in registers over a block's rows, then over the block's groups,
// and written as one row per block; a second kernel adds those rows in a fixed order, so results do
// not depend on timing.
#include "fa_internal.h"
#include "fa_sm100.cuh"

namespace fa {
namespace {

constexpr int kRopeThreads = 256;

// 8 consecutive 16-bit elements -> float32.
template <bool BF16>
__device__ __forceinline__ void widen8(const uint4& v, float (&f)[8]) {
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

template <bool BF16>
__device__ __forceinline__ uint4 narrow8(const float (&f)[8]) {
  return make_uint4(pack2<BF16>(f[0], f[1]), pack2<BF16>(f[2], f[3]), pack2<BF16>(f[4], f[5]),
                    pack2<BF16>(f[6], f[7]));
}

// A lane's 16 elements as 8 pairs: lo = first members, hi = second members.  `v0` and `v1` are the
// lane's two 8-element vectors: [8l, +8) and [D/2 + 8l, +8), or [16l, +8) and [16l + 8, +8).
template <bool BF16, bool INTER>
__device__ __forceinline__ void to_pairs(const uint4& v0, const uint4& v1, float (&lo)[8], float (&hi)[8]) {
  if constexpr (INTER) {
    float a[8], b[8];
    widen8<BF16>(v0, a);
    widen8<BF16>(v1, b);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      lo[i] = a[2 * i];
      hi[i] = a[2 * i + 1];
      lo[4 + i] = b[2 * i];
      hi[4 + i] = b[2 * i + 1];
    }
  } else {
    widen8<BF16>(v0, lo);
    widen8<BF16>(v1, hi);
  }
}

template <bool BF16, bool INTER>
__device__ __forceinline__ void from_pairs(const float (&lo)[8], const float (&hi)[8], uint4& v0, uint4& v1) {
  if constexpr (INTER) {
    v0 = make_uint4(pack2<BF16>(lo[0], hi[0]), pack2<BF16>(lo[1], hi[1]), pack2<BF16>(lo[2], hi[2]),
                    pack2<BF16>(lo[3], hi[3]));
    v1 = make_uint4(pack2<BF16>(lo[4], hi[4]), pack2<BF16>(lo[5], hi[5]), pack2<BF16>(lo[6], hi[6]),
                    pack2<BF16>(lo[7], hi[7]));
  } else {
    v0 = narrow8<BF16>(lo);
    v1 = narrow8<BF16>(hi);
  }
}

template <int LPR>
__device__ __forceinline__ float group_sum(float v) {
#pragma unroll
  for (int o = LPR / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// bf16 rows whose squares leave float32's range (elements from about 2^57, or below 2^-48 with an eps next to 0): the row
// is multiplied by a power of two first, which is also returned.  Sets sum to the row's new sum of squares.
template <bool BF16>
__device__ __forceinline__ bool outside(float sum, float eps) {
  return BF16 && (!(sum < 0x1p120f) || (sum < 0x1p-90f && eps < 0x1p-90f));
}
template <int LPR>
__device__ __forceinline__ float bring_inside(float (&lo)[8], float (&hi)[8], float& sum) {
  const float by = sum < 0x1p-90f ? 0x1p80f : (sum < 0x1p120f ? 1.f : 0x1p-80f);  // 1: a row beside one that needs it
  float s = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    lo[i] *= by;
    hi[i] *= by;
    s = fmaf(lo[i], lo[i], fmaf(hi[i], hi[i], s));
  }
  sum = group_sum<LPR>(s);
  return by;
}

// One tensor of the call (queries or keys).
template <bool BWD>
struct RopeSide {
  const uint16_t* x;
  const uint16_t* dz;
  uint16_t* out;       // z forward, dx backward
  const void* w;
  long long xs[3];     // strides of x: batch, head, token
  long long os[3];     // strides of out
  int heads;
};

template <bool BWD>
__device__ __forceinline__ RopeSide<BWD> rope_side(const RopeParams& p, bool key) {
  RopeSide<BWD> s;
  s.x = static_cast<const uint16_t*>(key ? p.k : p.q);
  s.dz = static_cast<const uint16_t*>(key ? p.dk_out : p.dq_out);
  s.out = static_cast<uint16_t*>(BWD ? (key ? p.dk : p.dq) : (key ? p.k_out : p.q_out));
  s.w = key ? p.k_weight : p.q_weight;
  s.heads = key ? p.H_kv : p.H;
#pragma unroll
  for (int i = 0; i < 3; ++i) {
    s.xs[i] = key ? p.k_stride[i] : p.q_stride[i];
    s.os[i] = key ? p.dk_stride[i] : p.dq_stride[i];
  }
  return s;
}

// Element offsets of a lane's two vectors inside a row.
template <int D, bool INTER>
__device__ __forceinline__ void lane_offsets(int l, int& o0, int& o1) {
  o0 = INTER ? 16 * l : 8 * l;
  o1 = INTER ? 16 * l + 8 : D / 2 + 8 * l;
}

template <int D, bool BF16, bool INTER>
__device__ __forceinline__ void load_weight(const void* w, bool f32, int l, float (&wl)[8], float (&wh)[8]) {
  int o0, o1;
  lane_offsets<D, INTER>(l, o0, o1);
  if (w == nullptr) {
#pragma unroll
    for (int i = 0; i < 8; ++i) wl[i] = wh[i] = 1.f;
  } else if (f32) {
    const float* f = static_cast<const float*>(w);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      wl[i] = INTER ? f[o0 + 2 * i] : f[o0 + i];
      wh[i] = INTER ? f[o0 + 2 * i + 1] : f[o1 + i];
    }
  } else {
    const uint16_t* h = static_cast<const uint16_t*>(w);
    to_pairs<BF16, INTER>(*reinterpret_cast<const uint4*>(h + o0), *reinterpret_cast<const uint4*>(h + o1), wl, wh);
  }
}

// Position of token (b, n) on one axis, kept inside the table: an index outside it records
// kDevBadIndex and uses row 0.
__device__ __forceinline__ int rope_position(const RopeParams& p, int axis, int b, int n) {
  long long v;
  if (p.pos == nullptr) {
    v = n;
  } else {
    const long long at = axis * p.pos_axis_stride + b * p.pos_batch_stride + n;
    v = p.pos64 ? static_cast<const long long*>(p.pos)[at] : static_cast<const int*>(p.pos)[at];
  }
  if (v < 0 || v >= p.max_pos) {
    record_error(p.status, kDevBadIndex, n);
    v = 0;
  }
  return static_cast<int>(v);
}

// cos and sin of a lane's 8 pairs; four pairs of one axis are one access.
template <int D>
__device__ __forceinline__ void load_angles(const RopeParams& p, int b, int n, int l, float (&c)[8], float (&s)[8]) {
  int row[kRopeMaxAxes];
  row[0] = rope_position(p, 0, b, n);
#pragma unroll
  for (int a = 1; a < kRopeMaxAxes; ++a) row[a] = a < p.axes ? rope_position(p, a, b, n) : row[0];
  auto row_of = [&](int pair) {
    int r = row[0];
#pragma unroll
    for (int a = 1; a < kRopeMaxAxes; ++a)
      if (a < p.axes && pair >= p.section_start[a]) r = row[a];
    return static_cast<size_t>(r) * (D / 2);
  };
#pragma unroll
  for (int i = 0; i < 8; i += 4) {
    const int pair = 8 * l + i;
    const size_t first = row_of(pair);
    if (first == row_of(pair + 3)) {  // sections that end inside would have another row in between
      const size_t mid0 = row_of(pair + 1), mid1 = row_of(pair + 2);
      if (mid0 == first && mid1 == first) {
        const float4 x = *reinterpret_cast<const float4*>(p.cos + first + pair), y = *reinterpret_cast<const float4*>(p.sin + first + pair);
        c[i] = x.x; c[i + 1] = x.y; c[i + 2] = x.z; c[i + 3] = x.w;
        s[i] = y.x; s[i + 1] = y.y; s[i + 2] = y.z; s[i + 3] = y.w;
        continue;
      }
    }
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const size_t at = row_of(pair + k) + pair + k;
      c[i + k] = p.cos[at];
      s[i + k] = p.sin[at];
    }
  }
}

// ---------------------------------------------------------------------------------------- forward
// grid: x = token blocks, y = head ranges (first the queries', then the keys').
template <int D, bool BF16, bool INTER>
__global__ void __launch_bounds__(kRopeThreads, 3) rope_fwd_kernel(const RopeParams p) {
  constexpr int LPR = D / 16;
  constexpr int kGroups = kRopeThreads / LPR;
  constexpr int kUnroll = 2;
  const int status = ld_status(p.status);  // looked at before the first store
  const int l = threadIdx.x % LPR;
  const long long token = static_cast<long long>(blockIdx.x) * kGroups + threadIdx.x / LPR;
  const bool key = static_cast<int>(blockIdx.y) >= p.q_ranges;
  const int range = key ? blockIdx.y - p.q_ranges : blockIdx.y;
  const RopeSide<false> s = rope_side<false>(p, key);
  const int h0 = range * p.range_heads, h1 = min(s.heads, h0 + p.range_heads);
  const bool live = token < p.tokens;  // whole groups; the others stay for the shuffles
  const int b = live ? static_cast<int>(token / p.N) : 0;
  const int n = live ? static_cast<int>(token - static_cast<long long>(b) * p.N) : 0;
  int o0, o1;
  lane_offsets<D, INTER>(l, o0, o1);
  const uint16_t* x = s.x + b * s.xs[0] + n * s.xs[2];
  uint16_t* z = s.out + (static_cast<long long>(b) * s.heads * p.N + n) * D;
  float wl[8], wh[8], c[8], sn[8];
  load_weight<D, BF16, INTER>(s.w, p.weight_f32, l, wl, wh);
  load_angles<D>(p, b, n, l, c, sn);
  const bool norm = s.w != nullptr;
  for (int h = h0; h < h1; h += kUnroll) {
    uint4 v0[kUnroll], v1[kUnroll];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u)
      if (live && h + u < h1) {
        const uint16_t* row = x + (h + u) * s.xs[1];
        v0[u] = *reinterpret_cast<const uint4*>(row + o0);
        v1[u] = *reinterpret_cast<const uint4*>(row + o1);
      } else {
        v0[u] = v1[u] = make_uint4(0, 0, 0, 0);
      }
    if (status != 0) return;
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      float lo[8], hi[8];
      to_pairs<BF16, INTER>(v0[u], v1[u], lo, hi);
      if (norm) {
        float sum = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) sum = fmaf(lo[i], lo[i], fmaf(hi[i], hi[i], sum));
        sum = group_sum<LPR>(sum);
        float r = rsqrtf(sum * (1.f / D) + p.eps);
        if (__any_sync(0xffffffffu, outside<BF16>(sum, p.eps))) {
          const float by = bring_inside<LPR>(lo, hi, sum);
          r = rsqrtf(sum * (1.f / D) + p.eps * by * by);
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          lo[i] = lo[i] * r * wl[i];
          hi[i] = hi[i] * r * wh[i];
        }
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float a = lo[i], e = hi[i];
        lo[i] = a * c[i] - e * sn[i];
        hi[i] = a * sn[i] + e * c[i];
      }
      if (live && h + u < h1) {
        uint4 r0, r1;
        from_pairs<BF16, INTER>(lo, hi, r0, r1);
        uint16_t* row = z + static_cast<long long>(h + u) * p.N * D;
        *reinterpret_cast<uint4*>(row + o0) = r0;
        *reinterpret_cast<uint4*>(row + o1) = r1;
      }
    }
  }
}

// --------------------------------------------------------------------------------------- backward
// Blocks [0, q_blocks) walk the queries' units (token block, head range), the rest the keys'; each
// leaves its sum of dw (float32 [D]) in row blockIdx.x of the workspace.
template <int D, bool BF16, bool INTER>
__global__ void __launch_bounds__(kRopeThreads, 2) rope_bwd_kernel(const RopeParams p) {
  constexpr int LPR = D / 16;
  constexpr int kGroups = kRopeThreads / LPR;
  constexpr int kUnroll = 2;
  __shared__ float part[kRopeThreads / 32][D];
  if (__syncthreads_or(ld_status(p.status)) != 0) return;
  const bool key = static_cast<int>(blockIdx.x) >= p.q_blocks;
  const int block = key ? blockIdx.x - p.q_blocks : blockIdx.x;
  const int blocks = key ? gridDim.x - p.q_blocks : p.q_blocks;
  const RopeSide<true> s = rope_side<true>(p, key);
  const int ranges = (s.heads + p.range_heads - 1) / p.range_heads;
  const long long token_blocks = (p.tokens + kGroups - 1) / kGroups;
  const int l = threadIdx.x % LPR;
  int o0, o1;
  lane_offsets<D, INTER>(l, o0, o1);
  const bool norm = s.w != nullptr;
  float wl[8], wh[8], dl[8], dh[8];
  load_weight<D, BF16, INTER>(s.w, p.weight_f32, l, wl, wh);
#pragma unroll
  for (int i = 0; i < 8; ++i) dl[i] = dh[i] = 0.f;
  for (long long unit = block; unit < token_blocks * ranges; unit += blocks) {
    const int range = static_cast<int>(unit % ranges);
    const long long token = unit / ranges * kGroups + threadIdx.x / LPR;
    const bool live = token < p.tokens;
    const int b = live ? static_cast<int>(token / p.N) : 0;
    const int n = live ? static_cast<int>(token - static_cast<long long>(b) * p.N) : 0;
    const int h0 = range * p.range_heads, h1 = min(s.heads, h0 + p.range_heads);
    const uint16_t* x = s.x + b * s.xs[0] + n * s.xs[2];
    const uint16_t* dz = s.dz + (static_cast<long long>(b) * s.heads * p.N + n) * D;
    uint16_t* dx = s.out + b * s.os[0] + n * s.os[2];
    float c[8], sn[8];
    load_angles<D>(p, b, n, l, c, sn);
    for (int h = h0; h < h1; h += kUnroll) {
      uint4 x0[kUnroll], x1[kUnroll], z0[kUnroll], z1[kUnroll];
#pragma unroll
      for (int u = 0; u < kUnroll; ++u)
        if (live && h + u < h1) {
          const uint16_t* xr = x + (h + u) * s.xs[1];
          const uint16_t* zr = dz + static_cast<long long>(h + u) * p.N * D;
          x0[u] = *reinterpret_cast<const uint4*>(xr + o0);
          x1[u] = *reinterpret_cast<const uint4*>(xr + o1);
          z0[u] = *reinterpret_cast<const uint4*>(zr + o0);
          z1[u] = *reinterpret_cast<const uint4*>(zr + o1);
        } else {
          x0[u] = x1[u] = z0[u] = z1[u] = make_uint4(0, 0, 0, 0);
        }
      bool again = false;
#pragma unroll
      for (int u = 0; u < kUnroll; ++u) {
        float lo[8], hi[8];
        to_pairs<BF16, INTER>(z0[u], z1[u], lo, hi);
#pragma unroll
        for (int i = 0; i < 8; ++i) {  // dy: the rotation turned back
          const float a = lo[i], e = hi[i];
          lo[i] = a * c[i] + e * sn[i];
          hi[i] = e * c[i] - a * sn[i];
        }
        if (norm) {
          float xl[8], xh[8], sum = 0.f, dot = 0.f;
          to_pairs<BF16, INTER>(x0[u], x1[u], xl, xh);
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            sum = fmaf(xl[i], xl[i], fmaf(xh[i], xh[i], sum));
            dot = fmaf(lo[i] * wl[i], xl[i], fmaf(hi[i] * wh[i], xh[i], dot));
          }
          sum = group_sum<LPR>(sum);
          const float r = rsqrtf(sum * (1.f / D) + p.eps);
          const float t = group_sum<LPR>(dot) * (1.f / D) * r * r;
          const bool out = outside<BF16>(sum, p.eps);  // such a row is done again below
          again |= out;
          const float ra = live && h + u < h1 && !out ? r : 0.f;
          // rows outside the tensor add nothing to dw (they are zeros, and r is infinite where eps is 0)
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            dl[i] = fmaf(lo[i], xl[i] * ra, dl[i]);
            dh[i] = fmaf(hi[i], xh[i] * ra, dh[i]);
            lo[i] = r * (lo[i] * wl[i] - xl[i] * t);
            hi[i] = r * (hi[i] * wh[i] - xh[i] * t);
          }
        }
        if (live && h + u < h1) {
          uint4 r0, r1;
          from_pairs<BF16, INTER>(lo, hi, r0, r1);
          uint16_t* row = dx + (h + u) * s.os[1];
          *reinterpret_cast<uint4*>(row + o0) = r0;
          *reinterpret_cast<uint4*>(row + o1) = r1;
        }
      }
      if constexpr (BF16) {
        // Not inside the rows' own code: a branch there keeps the two rows from overlapping (8192 tokens: 72 us, now 56).
        if (__any_sync(0xffffffffu, again)) {
#pragma unroll 1
          for (int k = h; k < min(h1, h + kUnroll); ++k) {
            uint4 x0 = make_uint4(0, 0, 0, 0), x1 = x0, z0 = x0, z1 = x0;
            if (live) {
              const uint16_t* xr = x + k * s.xs[1];
              const uint16_t* zr = dz + static_cast<long long>(k) * p.N * D;
              x0 = *reinterpret_cast<const uint4*>(xr + o0);
              x1 = *reinterpret_cast<const uint4*>(xr + o1);
              z0 = *reinterpret_cast<const uint4*>(zr + o0);
              z1 = *reinterpret_cast<const uint4*>(zr + o1);
            }
            float xl[8], xh[8], lo[8], hi[8], sum = 0.f, dot = 0.f;
            to_pairs<BF16, INTER>(x0, x1, xl, xh);
            to_pairs<BF16, INTER>(z0, z1, lo, hi);
#pragma unroll
            for (int i = 0; i < 8; ++i) sum = fmaf(xl[i], xl[i], fmaf(xh[i], xh[i], sum));
            sum = group_sum<LPR>(sum);
            const bool mine = live && outside<BF16>(sum, p.eps);
            const float by = bring_inside<LPR>(xl, xh, sum), r = rsqrtf(sum * (1.f / D) + p.eps * by * by);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              const float a = lo[i], e = hi[i];
              lo[i] = a * c[i] + e * sn[i];
              hi[i] = e * c[i] - a * sn[i];
              dot = fmaf(lo[i] * wl[i], xl[i], fmaf(hi[i] * wh[i], xh[i], dot));
            }
            const float t = group_sum<LPR>(dot) * (1.f / D) * r * r;
            if (mine) {
#pragma unroll
              for (int i = 0; i < 8; ++i) {
                dl[i] = fmaf(lo[i], xl[i] * r, dl[i]);
                dh[i] = fmaf(hi[i], xh[i] * r, dh[i]);
                lo[i] = r * (lo[i] * wl[i] - xl[i] * t) * by;
                hi[i] = r * (hi[i] * wh[i] - xh[i] * t) * by;
              }
              uint4 r0, r1;
              from_pairs<BF16, INTER>(lo, hi, r0, r1);
              uint16_t* row = dx + k * s.os[1];
              *reinterpret_cast<uint4*>(row + o0) = r0;
              *reinterpret_cast<uint4*>(row + o1) = r1;
            }
          }
        }
      }
    }
  }
  if (!norm) return;  // uniform over the block
  // dw of the block: over the warp's groups, then over the warps
#pragma unroll
  for (int i = 0; i < 8; ++i)
#pragma unroll
    for (int o = LPR; o < 32; o <<= 1) {
      dl[i] += __shfl_xor_sync(0xffffffffu, dl[i], o);
      dh[i] += __shfl_xor_sync(0xffffffffu, dh[i], o);
    }
  const int warp = threadIdx.x / 32;
  if (threadIdx.x % 32 < LPR) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      part[warp][INTER ? o0 + 2 * i : o0 + i] = dl[i];
      part[warp][INTER ? o0 + 2 * i + 1 : o1 + i] = dh[i];
    }
  }
  __syncthreads();
  if (threadIdx.x < D) {
    float sum = 0.f;
#pragma unroll
    for (int w = 0; w < kRopeThreads / 32; ++w) sum += part[w][threadIdx.x];
    p.workspace[static_cast<size_t>(blockIdx.x) * D + threadIdx.x] = sum;
  }
}

// dw[d] = sum of the blocks' rows, in a fixed order.  grid: x = D / 32 column blocks, y = queries,
// keys; 32 threads of a column each add every 32nd row.
__global__ void __launch_bounds__(1024) rope_dw_kernel(const RopeParams p, int D, int blocks, bool bf16) {
  __shared__ float part[32][33];
  if (__syncthreads_or(ld_status(p.status)) != 0) return;
  const bool key = blockIdx.y != 0;
  void* out = key ? p.dk_weight : p.dq_weight;
  if (out == nullptr) return;
  const int col = blockIdx.x * 32 + threadIdx.x % 32, at = threadIdx.x / 32;
  const int first = key ? p.q_blocks : 0, last = key ? blocks : p.q_blocks;
  float sum = 0.f;
  for (int r = first + at; r < last; r += 32) sum += p.workspace[static_cast<size_t>(r) * D + col];
  part[at][threadIdx.x % 32] = sum;
  __syncthreads();
  if (at == 0) {
    sum = 0.f;
#pragma unroll
    for (int r = 0; r < 32; ++r) sum += part[r][threadIdx.x];
    if (p.weight_f32)
      static_cast<float*>(out)[col] = sum;
    else if (bf16)
      static_cast<__nv_bfloat16*>(out)[col] = __float2bfloat16_rn(sum);
    else
      static_cast<__half*>(out)[col] = __float2half_rn(sum);
  }
}

constexpr int groups_per_block(int D) { return kRopeThreads / (D / 16); }

}  // namespace

// Heads per group.  Where the tokens alone make several waves of blocks: all of them (each token is then read and
// written in one sweep; 32768 tokens forward take 117 us, in groups of 8 heads 130).  Else as many as the keys
// have, eight at least (equal blocks for queries and keys: 8192 tokens forward 34 us, in groups of 16 heads 36),
// and fewer where that leaves fewer than `blocks` blocks.
static int rope_range_heads(const RopeParams& p, int D, int blocks) {
  const long long token_blocks = (p.tokens + groups_per_block(D) - 1) / groups_per_block(D);
  if (token_blocks >= 6 * 148) return p.H > p.H_kv ? p.H : p.H_kv;
  int heads = p.H_kv > 8 ? p.H_kv : 8;
  while (heads > 1 && token_blocks * ((p.H + heads - 1) / heads + (p.H_kv + heads - 1) / heads) < blocks)
    heads = (heads + 1) / 2;
  return heads;
}

cudaError_t launch_rope_fwd(RopeParams p, int D, bool bf16, bool interleaved, cudaStream_t stream) {
  p.range_heads = rope_range_heads(p, D, 2 * 148);
  p.q_ranges = (p.H + p.range_heads - 1) / p.range_heads;
  const int k_ranges = (p.H_kv + p.range_heads - 1) / p.range_heads;
  const dim3 grid(static_cast<unsigned>((p.tokens + groups_per_block(D) - 1) / groups_per_block(D)), p.q_ranges + k_ranges);
#define FA_ROPE_CASE(DD, BB, II)                                  \
  if (D == DD && bf16 == BB && interleaved == II) {               \
    rope_fwd_kernel<DD, BB, II><<<grid, kRopeThreads, 0, stream>>>(p); \
    return cudaGetLastError();                                    \
  }
#define FA_ROPE_CASES(DD) \
  FA_ROPE_CASE(DD, false, false) FA_ROPE_CASE(DD, false, true) FA_ROPE_CASE(DD, true, false) FA_ROPE_CASE(DD, true, true)
  FA_ROPE_CASES(32)
  FA_ROPE_CASES(64)
  FA_ROPE_CASES(128)
#undef FA_ROPE_CASE
  return cudaErrorInvalidValue;
}

cudaError_t launch_rope_bwd(RopeParams p, int D, bool bf16, bool interleaved, cudaStream_t stream) {
  p.range_heads = rope_range_heads(p, D, 3 * kRopeBwdBlocks);
  const long long token_blocks = (p.tokens + groups_per_block(D) - 1) / groups_per_block(D);
  const long long q_units = token_blocks * ((p.H + p.range_heads - 1) / p.range_heads);
  const long long k_units = token_blocks * ((p.H_kv + p.range_heads - 1) / p.range_heads);
  // one wave of blocks, shared out by the number of heads
  const long long k_share = p.H_kv == 0 ? 0 : (kRopeBwdBlocks * static_cast<long long>(p.H_kv) + p.H + p.H_kv - 1) / (p.H + p.H_kv);
  const long long k_most = k_share < kRopeBwdBlocks ? k_share : kRopeBwdBlocks - 1;  // the queries keep one
  const long long q_share = kRopeBwdBlocks - k_most;
  p.q_blocks = static_cast<int>(q_units < q_share ? q_units : q_share);
  const int blocks = p.q_blocks + static_cast<int>(k_units < k_most ? k_units : k_most);
#define FA_ROPE_CASE(DD, BB, II)                                  \
  if (D == DD && bf16 == BB && interleaved == II)                 \
    rope_bwd_kernel<DD, BB, II><<<blocks, kRopeThreads, 0, stream>>>(p);
  FA_ROPE_CASES(32)
  FA_ROPE_CASES(64)
  FA_ROPE_CASES(128)
#undef FA_ROPE_CASE
#undef FA_ROPE_CASES
  cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess || (p.dq_weight == nullptr && p.dk_weight == nullptr)) return e;
  rope_dw_kernel<<<dim3(D / 32, 2), 1024, 0, stream>>>(p, D, blocks, bf16);
  return cudaGetLastError();
}

}  // namespace fa
