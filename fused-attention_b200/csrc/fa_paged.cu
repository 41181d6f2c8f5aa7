// Attention over a paged e4m3 cache with one scale per (page, K/V head), for sm_100a: the split
// kernel for few query rows (decoding, speculation, short chunks) and the kernel that joins splits.
//
//   s_j = (q . k8_j) * k_scale(page j) * scale,   o = sum_j softmax(s)_j * v_scale(page j) * v8_j
// Token i of a sequence's n new tokens, at sequence length L (new tokens included), sees keys
// j <= L - n + i.  A row that sees no key gives o = 0 and lse = -inf.
//
// Bound: HBM.  A decode step reads every cached byte once and does 4 G D operations on 2 D bytes
// (G query heads per K/V head), so what counts is bytes in flight and few instructions per byte.
//   * Units.  The rows of a (sequence, K/V head), n tokens x G heads, form tiles of 8 NT rows; the
//     tile's keys form units of kUnit keys, one 32-key tile for each warp.  All units
//     of the call, in order, are cut into equal contiguous shares, one per block of a single wave: no block has more than its share however
//     ragged the lengths are, and there is no atomic and no order that depends on timing.  A tile
//     that is cut is written as partial results and joined by the second kernel, in a fixed order.
//     Measured with D = 128: 128 sequences of 4096 keys and 8 K/V heads 174 us, 6.2 TB/s or 94 % of the
//     measured copy rate; 32 of up to 8192 65 us, 81 %; a fixed cost of about 9 us (two launches,
//     five dependent reads to the first key, the join) is what short histories pay.
//   * Warps.  The four warps of a block take 32-key tiles of a share in turn, each with its own
//     softmax state, and are joined in shared memory once per tile of rows.
//   * Matrix form.  S^T = K Q^T and O^T = V^T P^T on m16n8k16 (f16 in, f32 sums): keys (and for
//     O^T the head dim) are the 16-row side, query rows the 8-column side, so a group of 8 heads
//     wastes nothing.  The k index of S^T (the head dim) and the m index of O^T (again the head
//     dim) may be permuted freely, which lets a thread take 16-byte pieces of a cached row and turn
//     bytes into operands with one conversion per pair.  S^T leaves the instruction as an 8 x 8 tile
//     whose transpose is the second product's operand (movmatrix).  The e4m3 form of mma.sync needs no
//     conversions but was slower (74 us instead of 68 for 32 sequences of up to 8192).
//   * Types.  e4m3 is exact in f16, so K and V lose nothing; bf16 queries are brought into f16's
//     range by a power of two per row (exact).  A row has two references, float32: m of its scores, which
//     its sum l is relative to, and u of s - m + log2(v_scale).  P is f16, 2^(s - m + log2(v_scale) - u), so
//     the pages' scales ride in P's exponent and a page with a small scale loses no precision; u is kept apart
//     from m because beside a large score a scale's logarithm would be rounded away.  A reference moves
//     only when a score passes it by 2^kSlack: O and l are rescaled, and lanes compare notes, only then.
//   K of the next tile is loaded before the softmax of this one, V of this one before its S.
#include "fa_internal.h"
#include "fa_paged.cuh"
#include "fa_sm100.cuh"

#include <cuda_fp8.h>

namespace fa {
namespace {

constexpr int kPagedThreads = 128;
constexpr int kWarps = kPagedThreads / 32;
constexpr int kUnit = kPagedUnit;   // keys of a unit
constexpr int kTile = 32;           // keys of a warp's tile
constexpr float kSlack = 8.f;       // log2: weights stay below 2^8 of the reference, far inside f16
constexpr float kNoScale = -200.f;  // stands for log2 0: below every float32's

template <int D, int NT>
struct PagedCfg {  // resident blocks per SM, as the registers allow
  static constexpr int kPerSm = D == 128 ? (NT == 1 ? 3 : 2) : (NT == 1 ? 4 : 3);
};

// Two e4m3 bytes (the low 16 bits of v) -> two f16.
__device__ __forceinline__ uint32_t cvt2(uint32_t v) {
  uint32_t r;
  asm("{\n\t.reg .b16 a, b;\n\tmov.b32 {a, b}, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, a;\n\t}" : "=r"(r) : "r"(v));
  return r;
}
__device__ __forceinline__ uint32_t cvt2_hi(uint32_t v) {
  uint32_t r;
  asm("{\n\t.reg .b16 a, b;\n\tmov.b32 {a, b}, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, b;\n\t}" : "=r"(r) : "r"(v));
  return r;
}

__device__ __forceinline__ void mma16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                         uint32_t b0, uint32_t b1) {
  asm(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// Transpose of an 8 x 8 tile of 16-bit values held as the instruction's row fragments.
__device__ __forceinline__ uint32_t transpose8(uint32_t v) {
  uint32_t r;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}

// Read-once cache data: not kept in L1.
template <int N>
__device__ __forceinline__ void load_words(const uint8_t* p, uint32_t* w) {
  if constexpr (N == 4) {
    asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];"
                 : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]) : "l"(p));
  } else if constexpr (N == 2) {
    asm volatile("ld.global.nc.L1::no_allocate.v2.u32 {%0,%1}, [%2];" : "=r"(w[0]), "=r"(w[1]) : "l"(p));
  } else {
    asm volatile("ld.global.nc.L1::no_allocate.u32 %0, [%1];" : "=r"(w[0]) : "l"(p));
  }
}

// A thread's part of a 16-key block of K: rows g and g + 8, D / 4 bytes of each.
template <int D>
struct KBlock {
  uint32_t w[2][D / 16];
};
// ... and of V: keys 2t, 2t + 1, 2t + 8, 2t + 9, D / 8 bytes of each.
template <int D>
struct VBlock {
  uint32_t w[4][D / 32];
};

template <int D>
__device__ __forceinline__ void load_k(const uint8_t* block, int g, int t, KBlock<D>& k) {
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    const uint8_t* row = block + (g + 8 * r) * D;
    if constexpr (D == 128) {
      load_words<4>(row + 16 * t, k.w[r]);
      load_words<4>(row + 64 + 16 * t, k.w[r] + 4);
    } else if constexpr (D == 64) {
      load_words<4>(row + 16 * t, k.w[r]);
    } else {
      load_words<2>(row + 8 * t, k.w[r]);
    }
  }
}
// The head-dim index of byte `e` of word `s` of a thread's K row: the permutation S^T sums over.
template <int D>
__device__ __forceinline__ int k_column(int t, int s) {
  return D == 128 ? 16 * (s < 4 ? t : 4 + t) + 4 * (s & 3) : (D == 64 ? 16 * t + 4 * s : 8 * t + 4 * s);
}

template <int D>
__device__ __forceinline__ void load_v(const uint8_t* block, int g, int t, VBlock<D>& v) {
#pragma unroll
  for (int i = 0; i < 4; ++i) load_words<D / 32>(block + (2 * t + (i & 1) + 8 * (i >> 1)) * D + (D / 8) * g, v.w[i]);
}

// Where a block's share starts, found by one scan over the sequences.
struct Cursor {
  long long total;  // units of the call
  int b;            // sequence of the share's first unit
  long long skip;   // units of that sequence before it
  bool stop;        // the status word was set
};

__device__ __forceinline__ void sequence_shape(const PagedParams& p, int b, int& first, int& n, int& len) {
  if (p.offsets == nullptr) {
    first = b;
    n = 1;
  } else {
    first = p.offsets[b];
    n = p.offsets[b + 1] - first;
    if (first < 0 || n < 0 || first > p.T - n) {  // not inside q: no rows
      if (n != 0) record_error(p.status, kDevBadIndex, b);
      first = n = 0;
    }
  }
  len = p.seq_lens[b];
  if (len < 0 || len > p.capacity) {
    record_error(p.status, kDevBadIndex, b);
    len = 0;
  }
}

template <int RT>
__device__ __forceinline__ void sequence_units(const PagedParams& p, int n, int len, int& tiles, int& per_tile) {
  tiles = (n * p.group + RT - 1) / RT;
  per_tile = max(1, (len + kUnit - 1) / kUnit);
}

// Blocks that take part: none without a unit, so the shares are never empty.
__device__ __forceinline__ long long active_blocks(long long total) {
  return min(static_cast<long long>(gridDim.x), total);
}

template <int RT>
__device__ __forceinline__ Cursor find_share(const PagedParams& p, int status) {
  __shared__ long long warp_sum[kWarps];
  __shared__ long long found[2];
  const int chunk = (p.B + kPagedThreads - 1) / kPagedThreads;
  const int b0 = min(p.B, static_cast<int>(threadIdx.x) * chunk), b1 = min(p.B, b0 + chunk);
  long long mine = 0;
  int first, n, len, tiles, per_tile;
  for (int b = b0; b < b1; ++b) {
    sequence_shape(p, b, first, n, len);
    sequence_units<RT>(p, n, len, tiles, per_tile);
    mine += static_cast<long long>(tiles) * per_tile * p.H_kv;
  }
  long long incl = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long v = __shfl_up_sync(0xffffffffu, incl, o);
    if (static_cast<int>(threadIdx.x % 32) >= o) incl += v;
  }
  if (threadIdx.x % 32 == 31) warp_sum[threadIdx.x / 32] = incl;
  __syncthreads();
  long long total = 0;
#pragma unroll
  for (int w = 0; w < kWarps; ++w) {
    if (w == static_cast<int>(threadIdx.x / 32)) incl += total;
    total += warp_sum[w];
  }
  Cursor c;
  c.total = total;
  const long long blocks = active_blocks(total);
  if (static_cast<long long>(blockIdx.x) < blocks) {
    const long long start = total * blockIdx.x / blocks;
    long long before = incl - mine;
    if (start >= before && start < incl) {
      for (int b = b0; b < b1; ++b) {
        sequence_shape(p, b, first, n, len);
        sequence_units<RT>(p, n, len, tiles, per_tile);
        const long long units = static_cast<long long>(tiles) * per_tile * p.H_kv;
        if (start < before + units) {
          found[0] = b;
          found[1] = start - before;
          break;
        }
        before += units;
      }
    }
  }
  c.stop = __syncthreads_or(status) != 0;
  c.b = static_cast<int>(found[0]);
  c.skip = found[1];
  return c;
}

// A tile of rows: rows r0 .. of sequence b and K/V head h.
struct RowTile {
  int first;   // flat index of the sequence's first token
  int n;       // its new tokens
  int len;
  int h;       // K/V head
  int r0;      // first row: token r0 / group, head r0 % group of the group
};

// Adds the scores and values of keys [key0, key0 + 32) to a warp's state.
template <int D, int NT>
struct WarpState {
  float o[NT][D / 16][4];   // O^T: rows g, g + 8 of each 16-row tile, columns 2t, 2t + 1
  float m[NT][2];           // reference of s, all lanes of a column alike
  float u[NT][2];           // reference of s - m + log2(v_scale), likewise
  float l[NT][2];           // this thread's sum of 2^(s - m)
};

// EDGE: keys behind a row's last are masked, V's bytes behind the tile's last key are cleared, and so is NaN in V,
// which sets *saw_nan: the caller puts it back for the rows that see it.
template <int D, int NT, bool EDGE>
__device__ __forceinline__ void softmax_pv(WarpState<D, NT>& st, float (&s)[NT][2][4], const float (&qs)[NT][2],
                                           const float (&ks)[2], const float (&vs)[2], VBlock<D> (&v)[2],
                                           const int (&last)[NT][2], int key0, int keys, int g, int t,
                                           volatile int* saw_nan) {
  bool raise = false;
  float top[NT][2][2];  // per column: this thread's largest score of each block
#pragma unroll
  for (int nt = 0; nt < NT; ++nt)
#pragma unroll
    for (int c = 0; c < 2; ++c) {
#pragma unroll
      for (int blk = 0; blk < 2; ++blk) {
        const float f = qs[nt][c] * ks[blk];
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          float x = s[nt][blk][2 * r + c] * f;
          if (EDGE && key0 + 16 * blk + 8 * r + g > last[nt][c]) x = -INFINITY;
          s[nt][blk][2 * r + c] = x;
        }
        top[nt][c][blk] = fmaxf(s[nt][blk][c], s[nt][blk][2 + c]);
        // by the threshold above m, or with the scale above m + u (m = -inf: any score)
        raise |= top[nt][c][blk] - st.m[nt][c] > kSlack + fminf(0.f, st.u[nt][c] - vs[blk]);
      }
    }
  if (__any_sync(0xffffffffu, raise)) {  // new references, the same in all lanes of a column
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        float m = fmaxf(st.m[nt][c], fmaxf(top[nt][c][0], top[nt][c][1]));
#pragma unroll
        for (int o = 4; o < 32; o <<= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
        const float down = st.m[nt][c] - m;  // -inf for the first score, NaN (and no other lane's sum) before it
        const float before = st.u[nt][c] + down;
        float u = fmaxf((top[nt][c][0] - m) + vs[0], (top[nt][c][1] - m) + vs[1]);
#pragma unroll
        for (int o = 4; o < 32; o <<= 1) u = fmaxf(u, __shfl_xor_sync(0xffffffffu, u, o));
        u = fmaxf(fmaxf(before, u), kNoScale);
        const float alpha_l = st.m[nt][c] == -INFINITY ? 0.f : ex2_approx(down);
        const float alpha = st.m[nt][c] == -INFINITY ? 0.f : ex2_approx(before - u);
        st.m[nt][c] = m;
        st.u[nt][c] = u;
        st.l[nt][c] *= alpha_l;
#pragma unroll
        for (int mt = 0; mt < D / 16; ++mt) {
          st.o[nt][mt][c] *= alpha;
          st.o[nt][mt][2 + c] *= alpha;
        }
      }
  }
  uint32_t pb[NT][2][2];
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      const float m = st.m[nt][c] == -INFINITY ? 0.f : st.m[nt][c];  // no score yet: all terms below are 0
      float l = st.l[nt][c];
#pragma unroll
      for (int blk = 0; blk < 2; ++blk) {
        const float shift = vs[blk] - st.u[nt][c];
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          const float x = s[nt][blk][2 * r + c] - m;
          l += ex2_approx(x);
          s[nt][blk][2 * r + c] = ex2_approx(x + shift);
        }
      }
      st.l[nt][c] = l;
    }
#pragma unroll
    for (int blk = 0; blk < 2; ++blk)
#pragma unroll
      for (int r = 0; r < 2; ++r)
        pb[nt][blk][r] = transpose8(pack2<false>(s[nt][blk][2 * r], s[nt][blk][2 * r + 1]));
  }
#pragma unroll
  for (int blk = 0; blk < 2; ++blk) {
    if (EDGE) {  // bytes behind the last key may hold anything: 0 * NaN is not 0
      uint32_t nan = 0;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const bool behind = key0 + 16 * blk + 2 * t + (i & 1) + 8 * (i >> 1) >= keys;
#pragma unroll
        for (int w = 0; w < D / 32; ++w) {
          if (behind) v[blk].w[i][w] = 0;
          const uint32_t mask = nan_bytes(v[blk].w[i][w]);
          v[blk].w[i][w] &= ~mask;
          nan |= mask;
        }
      }
      if (nan != 0) *saw_nan = 1;
    }
#pragma unroll
    for (int w = 0; w < D / 32; ++w)
#pragma unroll
      for (int half = 0; half < 2; ++half) {  // bytes 0, 1 / 2, 3 of the word: head dims of one 16-row tile
        const uint32_t sel = half == 0 ? 0x5140u : 0x7362u;
        const uint32_t x = __byte_perm(v[blk].w[0][w], v[blk].w[1][w], sel);
        const uint32_t y = __byte_perm(v[blk].w[2][w], v[blk].w[3][w], sel);
        const uint32_t a0 = cvt2(x), a1 = cvt2_hi(x), a2 = cvt2(y), a3 = cvt2_hi(y);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
          mma16816(st.o[nt][2 * w + half], a0, a1, a2, a3, pb[nt][blk][0], pb[nt][blk][1]);
      }
  }
}

template <int D, int NT>
__global__ void __launch_bounds__(kPagedThreads, PagedCfg<D, NT>::kPerSm) paged_split_kernel(const PagedParams p) {
  constexpr int RT = 8 * NT;
  __shared__ float sh_o[kWarps][RT][D + 4];  // +4: rows start on different banks
  __shared__ float sh_m[kWarps][RT], sh_l[kWarps][RT];
  __shared__ volatile int sh_nan[kWarps];  // the warp met NaN in a value that some row does not see
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const int g = lane / 4, t = lane % 4;
  if (threadIdx.x == 0) p.joins[blockIdx.x].parts = 0;
  const Cursor cur = find_share<RT>(p, ld_status(p.status));
  if (cur.stop) return;
  clear_unowned_rows<D>(p);
  const long long blocks = active_blocks(cur.total);
  if (static_cast<long long>(blockIdx.x) >= blocks) return;
  long long unit = cur.total * blockIdx.x / blocks;
  const long long unit_end = cur.total * (blockIdx.x + 1) / blocks;
  const uint32_t kv_head_bytes = static_cast<uint32_t>(D) << p.page_shift;
  const int page_mask = (1 << p.page_shift) - 1;
  int b = cur.b;
  long long skip = cur.skip;
  bool first_segment = true;
  int first, n, len, tiles, per_tile;
  sequence_shape(p, b, first, n, len);
  sequence_units<RT>(p, n, len, tiles, per_tile);
  while (unit < unit_end) {
    while (skip >= static_cast<long long>(tiles) * per_tile * p.H_kv) {  // on to the next sequence that has rows
      skip = 0;
      ++b;
      if (b >= p.B) return;  // not reached: the units add up to `total`
      sequence_shape(p, b, first, n, len);
      sequence_units<RT>(p, n, len, tiles, per_tile);
    }
    const int item = static_cast<int>(skip / per_tile);
    const int u0 = static_cast<int>(skip - static_cast<long long>(item) * per_tile);
    const int u1 = static_cast<int>(min(static_cast<long long>(per_tile), u0 + (unit_end - unit)));
    // heads of a tile of rows next to each other: they read the same pages' table entries
    const int h = item % p.H_kv;
    const int r0 = item / p.H_kv * RT;
    const int rows = min(RT, n * p.group - r0);
    const int before = len - n;                                  // keys in front of the new tokens
    const int keys = max(0, min(len, before + (r0 + rows - 1) / p.group + 1));  // seen by the tile's last row
    const int seen_by_all = before + r0 / p.group + 1;           // keys that every row sees

    // ---- queries: the 8-column operand, k in the order of the cached row's pieces
    uint32_t qf[NT][D / 16][2];
    float qs[NT][2];
    int last[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const int r = r0 + 8 * nt + g;
      const bool live = 8 * nt + g < rows;
      const uint16_t* q = nullptr;
      if (live) q = static_cast<const uint16_t*>(p.q) + (first + r / p.group) * p.q_stride[0] + (h * p.group + r % p.group) * p.q_stride[1];
      uint2 raw[D / 16];
#pragma unroll
      for (int s = 0; s < D / 16; ++s)
        raw[s] = live ? *reinterpret_cast<const uint2*>(q + k_column<D>(t, s)) : make_uint2(0, 0);
      float row_scale = 1.f;
      if (p.bf16) {
        // the row's largest magnitude to [2^7, 2^8): a power of two, exact in f16 down to 2^-31 of it
        uint32_t top = 0;
#pragma unroll
        for (int s = 0; s < D / 16; ++s) {
          top = max(top, max(raw[s].x & 0x7fffu, (raw[s].x >> 16) & 0x7fffu));
          top = max(top, max(raw[s].y & 0x7fffu, (raw[s].y >> 16) & 0x7fffu));
        }
        top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
        const int e = min(254, max(8, static_cast<int>(top >> 7)));  // biased exponent
        const float down = __uint_as_float(static_cast<uint32_t>(min(254, 127 + 7 + 127 - e)) << 23);  // 2^(7 - (e - 127))
        row_scale = 1.f / down;
#pragma unroll
        for (int s = 0; s < D / 16; ++s) {
          qf[nt][s][0] = pack2<false>(__uint_as_float(raw[s].x << 16) * down, __uint_as_float(raw[s].x & 0xffff0000u) * down);
          qf[nt][s][1] = pack2<false>(__uint_as_float(raw[s].y << 16) * down, __uint_as_float(raw[s].y & 0xffff0000u) * down);
        }
      } else {
#pragma unroll
        for (int s = 0; s < D / 16; ++s) {
          qf[nt][s][0] = raw[s].x;
          qf[nt][s][1] = raw[s].y;
        }
      }
#pragma unroll
      for (int c = 0; c < 2; ++c) {  // columns 2t, 2t + 1 of S^T: the rows that lanes 4 (2t + c) hold
        qs[nt][c] = __shfl_sync(0xffffffffu, row_scale, 4 * (2 * t + c)) * p.scale_log2;
        last[nt][c] = before + (r0 + 8 * nt + 2 * t + c) / p.group;
      }
    }

    WarpState<D, NT> st;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
      for (int mt = 0; mt < D / 16; ++mt)
#pragma unroll
        for (int i = 0; i < 4; ++i) st.o[nt][mt][i] = 0.f;
      st.m[nt][0] = st.m[nt][1] = -INFINITY;
      st.u[nt][0] = st.u[nt][1] = kNoScale;
      st.l[nt][0] = st.l[nt][1] = 0.f;
    }

    // ---- this warp's 32-key tiles of keys [u0, u1) units
    const int key_end = min(keys, u1 * kUnit);
    const int* table = p.block_table + b * p.table_stride;
    const int last_index = keys > 0 ? (keys - 1) >> p.page_shift : 0;
    // The page of a 16-key block; blocks behind the last key stay on its page.
    auto page_of = [&](int key) -> int {
      const int page = table[min(key >> p.page_shift, last_index)];
      if (page < 0 || page >= p.num_pages) {
        record_error(p.status, kDevBadIndex, b);
        return 0;
      }
      return page;
    };
    int key0 = u0 * kUnit + warp * kTile;
    if (lane == 0) sh_nan[warp] = 0;
    __syncwarp();
    if (key0 < key_end) {
      KBlock<D> k[2];
      size_t at[2];     // (page, head) of the tile's two blocks
      int next_page[2];
#pragma unroll
      for (int blk = 0; blk < 2; ++blk) next_page[blk] = page_of(key0 + 16 * blk);
#pragma unroll
      for (int blk = 0; blk < 2; ++blk) {
        at[blk] = static_cast<size_t>(next_page[blk]) * p.H_kv + h;
        load_k<D>(p.k_pages + at[blk] * kv_head_bytes + ((key0 + 16 * blk) & page_mask) * D, g, t, k[blk]);
      }
      int key_next = key0 + kWarps * kTile;
      if (key_next < key_end)
#pragma unroll
        for (int blk = 0; blk < 2; ++blk) next_page[blk] = page_of(key_next + 16 * blk);
      auto one_tile = [&](auto edge) {
        VBlock<D> v[2];
        float ks[2], vs[2];
#pragma unroll
        for (int blk = 0; blk < 2; ++blk) {
          load_v<D>(p.v_pages + at[blk] * kv_head_bytes + ((key0 + 16 * blk) & page_mask) * D, g, t, v[blk]);
          ks[blk] = p.k_scales[at[blk]];
          vs[blk] = p.v_scales[at[blk]];
        }
        float s[NT][2][4];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int blk = 0; blk < 2; ++blk)
#pragma unroll
            for (int i = 0; i < 4; ++i) s[nt][blk][i] = 0.f;
#pragma unroll
        for (int blk = 0; blk < 2; ++blk)
#pragma unroll
          for (int w = 0; w < D / 16; ++w) {
            const uint32_t a0 = cvt2(k[blk].w[0][w]), a2 = cvt2_hi(k[blk].w[0][w]);
            const uint32_t a1 = cvt2(k[blk].w[1][w]), a3 = cvt2_hi(k[blk].w[1][w]);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) mma16816(s[nt][blk], a0, a1, a2, a3, qf[nt][w][0], qf[nt][w][1]);
          }
        const bool more = key_next < key_end;
        if (more) {
#pragma unroll
          for (int blk = 0; blk < 2; ++blk) {
            at[blk] = static_cast<size_t>(next_page[blk]) * p.H_kv + h;
            load_k<D>(p.k_pages + at[blk] * kv_head_bytes + ((key_next + 16 * blk) & page_mask) * D, g, t, k[blk]);
          }
          if (key_next + kWarps * kTile < key_end)
#pragma unroll
            for (int blk = 0; blk < 2; ++blk) next_page[blk] = page_of(key_next + kWarps * kTile + 16 * blk);
        }
        vs[0] = fmaxf(__log2f(vs[0]), kNoScale);
        vs[1] = fmaxf(__log2f(vs[1]), kNoScale);
        softmax_pv<D, NT, decltype(edge)::value>(st, s, qs, ks, vs, v, last, key0, keys, g, t, &sh_nan[warp]);
        key0 = key_next;
        key_next += kWarps * kTile;
      };
      // Two loops: the tiles that some row does not see to their end need masks and the clearing of NaN.
      while (key0 < key_end && key0 + kTile <= seen_by_all) one_tile(std::false_type{});
      while (key0 < key_end) one_tile(std::true_type{});
    }

    // ---- join the warps: l over the lanes of a column, then everything in shared memory
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        float l = st.l[nt][c];
#pragma unroll
        for (int o = 4; o < 32; o <<= 1) l += __shfl_xor_sync(0xffffffffu, l, o);
        if (g == 0) {
          sh_m[warp][8 * nt + 2 * t + c] = st.m[nt][c];
          sh_l[warp][8 * nt + 2 * t + c] = l;
        }
        // O relative to m: the pages' scales come back into it here
        const float f = exp2f(st.u[nt][c]);
#pragma unroll
        for (int mt = 0; mt < D / 16; ++mt) {
          st.o[nt][mt][c] *= f;
          st.o[nt][mt][2 + c] *= f;
        }
        // head dims D / 8 * g + 2 mt, + 1 of this row
        float* row = &sh_o[warp][8 * nt + 2 * t + c][D / 8 * g];
#pragma unroll
        for (int mt = 0; mt < D / 16; mt += 2)
          *reinterpret_cast<float4*>(row + 2 * mt) = make_float4(st.o[nt][mt][c], st.o[nt][mt][2 + c],
                                                                 st.o[nt][mt + 1][c], st.o[nt][mt + 1][2 + c]);
      }
    __syncwarp();
    if (sh_nan[warp] != 0) {  // rare: NaN among the values that some row does not see, for those that do
#pragma unroll 1
      for (int k0 = u0 * kUnit + warp * kTile; k0 < key_end; k0 += kWarps * kTile) {
        if (k0 + kTile <= seen_by_all) continue;
#pragma unroll 1
        for (int key = k0; key < min(k0 + kTile, keys); ++key) {
          const uint8_t* row = p.v_pages + (static_cast<size_t>(page_of(key)) * p.H_kv + h) * kv_head_bytes +
                               (key & page_mask) * D;
#pragma unroll 1
          for (int d = lane; d < D; d += 32)
            if ((row[d] & 0x7f) == 0x7f)
#pragma unroll 1
              for (int r = 0; r < RT; ++r)
                if (key <= before + (r0 + r) / p.group) sh_o[warp][r][d] = __int_as_float(0x7fffffff);
        }
      }
    }
    __syncthreads();
    const bool whole = u0 == 0 && u1 == per_tile;
    const int slot = 2 * blockIdx.x + (first_segment ? 0 : 1);
    constexpr int kPieces = D / 4;
    for (int i = threadIdx.x; i < RT * kPieces; i += kPagedThreads) {
      const int r = i / kPieces, d = i % kPieces * 4;
      float m = sh_m[0][r];
#pragma unroll
      for (int w = 1; w < kWarps; ++w) m = fmaxf(m, sh_m[w][r]);
      const float ref = m == -INFINITY ? 0.f : m;
      float l = 0.f;
      float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        const float f = ex2_approx(sh_m[w][r] - ref);
        l += sh_l[w][r] * f;
        const float4 o = *reinterpret_cast<const float4*>(&sh_o[w][r][d]);
        acc.x += o.x * f;
        acc.y += o.y * f;
        acc.z += o.z * f;
        acc.w += o.w * f;
      }
      if (whole) {
        if (r < rows) {
          const float inv = l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l);  // no key: 0; a NaN sum stays
          const int row = r0 + r;
          const long long token = first + row / p.group;
          const int head = h * p.group + row % p.group;
          uint16_t* out = static_cast<uint16_t*>(p.out) + token * p.out_stride[0] + head * p.out_stride[1] + d;
          const uint32_t lo = p.bf16 ? pack2<true>(acc.x * inv, acc.y * inv) : pack2<false>(acc.x * inv, acc.y * inv);
          const uint32_t hi = p.bf16 ? pack2<true>(acc.z * inv, acc.w * inv) : pack2<false>(acc.z * inv, acc.w * inv);
          *reinterpret_cast<uint2*>(out) = make_uint2(lo, hi);
          if (p.lse != nullptr && d == 0)
            p.lse[token * p.group * p.H_kv + head] = l == 0.f ? -INFINITY : m + log2f(l);
        }
      } else {
        *reinterpret_cast<float4*>(p.parts + (static_cast<size_t>(slot) * RT + r) * D + d) = acc;
        if (d == 0) p.part_ml[static_cast<size_t>(slot) * RT + r] = make_float2(m, l);
      }
    }
    if (!whole && u0 == 0 && threadIdx.x == 0) {
      // this block opens the cut tile: the blocks after it, up to the one that holds the tile's
      // last unit, have its other parts in their first slots
      const long long tile_end = unit - u0 + per_tile;
      const long long last_block = (tile_end * blocks - 1) / cur.total;
      PagedJoin j;
      j.parts = static_cast<int>(last_block - blockIdx.x) + 1;
      j.slot = slot;
      j.token = first;
      j.head = h;
      j.row = r0;
      j.rows = rows;
      p.joins[blockIdx.x] = j;
    }
    __syncthreads();
    unit += u1 - u0;
    skip += u1 - u0;
    first_segment = false;
  }
}

// Joins the parts of cut tiles.  grid: x = the block that opened the tile, y = groups of
// kJoinRows rows; the block's warps share a row's parts (kJoinSplit warps a row).
constexpr int kJoinThreads = 256;
constexpr int kJoinRows = 2;
constexpr int kJoinSplit = kJoinThreads / 32 / kJoinRows;

template <int D, int NT>
__global__ void __launch_bounds__(kJoinThreads) paged_join_kernel(const PagedParams p) {
  constexpr int RT = 8 * NT;
  constexpr int V = D / 32;  // consecutive values of a lane
  __shared__ float sh_o[kJoinRows][kJoinSplit][D];
  __shared__ float sh_l[kJoinRows][kJoinSplit];
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const PagedJoin j = p.joins[blockIdx.x];
  if (j.parts == 0) return;
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const int local = warp / kJoinSplit, split = warp % kJoinSplit;
  const int r = blockIdx.y * kJoinRows + local;
  const bool live = r < j.rows;
  auto slot_of = [&](int i) -> size_t { return i == 0 ? j.slot : 2 * (blockIdx.x + static_cast<size_t>(i)); };
  // the row's maximum over all parts first: the parts can then be loaded without waiting for each other
  float m = -INFINITY;
  if (live)
    for (int i = lane; i < j.parts; i += 32) m = fmaxf(m, p.part_ml[slot_of(i) * RT + r].x);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
  const float ref = m == -INFINITY ? 0.f : m;
  float l = 0.f, acc[V];
#pragma unroll
  for (int v = 0; v < V; ++v) acc[v] = 0.f;
  if (live) {
#pragma unroll 8
    for (int i = split; i < j.parts; i += kJoinSplit) {
      const size_t at = slot_of(i) * RT + r;
      const float2 ml = p.part_ml[at];
      const float* o = p.parts + at * D + V * lane;
      float x[V];
      if constexpr (V == 4) {
        const float4 q = *reinterpret_cast<const float4*>(o);
        x[0] = q.x;
        x[1] = q.y;
        x[2] = q.z;
        x[3] = q.w;
      } else {
#pragma unroll
        for (int v = 0; v < V; ++v) x[v] = o[v];
      }
      const float f = ex2_approx(ml.x - ref);
      l = fmaf(ml.y, f, l);
#pragma unroll
      for (int v = 0; v < V; ++v) acc[v] = fmaf(x[v], f, acc[v]);
    }
  }
#pragma unroll
  for (int v = 0; v < V; ++v) sh_o[local][split][V * lane + v] = acc[v];
  if (lane == 0) sh_l[local][split] = l;
  __syncthreads();
  if (split != 0 || !live) return;
  l = 0.f;
#pragma unroll
  for (int v = 0; v < V; ++v) acc[v] = 0.f;
#pragma unroll
  for (int s = 0; s < kJoinSplit; ++s) {
    l += sh_l[local][s];
#pragma unroll
    for (int v = 0; v < V; ++v) acc[v] += sh_o[local][s][V * lane + v];
  }
  const float inv = l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l);
  const int row = j.row + r;
  const long long token = j.token + row / p.group;
  const int head = j.head * p.group + row % p.group;
  const long long at = token * p.out_stride[0] + head * p.out_stride[1] + V * lane;
#pragma unroll
  for (int v = 0; v < V; ++v) {
    const float x = acc[v] * inv;
    if (p.bf16)
      static_cast<__nv_bfloat16*>(p.out)[at + v] = __float2bfloat16_rn(x);
    else
      static_cast<__half*>(p.out)[at + v] = __float2half_rn(x);
  }
  if (p.lse != nullptr && lane == 0)
    p.lse[token * p.group * p.H_kv + head] = l == 0.f ? -INFINITY : m + log2f(l);
}

template <int D, int NT>
cudaError_t launch_paged_t(const PagedParams& p, int blocks, bool join, cudaStream_t stream) {
  paged_split_kernel<D, NT><<<blocks, kPagedThreads, 0, stream>>>(p);
  cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess || !join) return e;
  // The join's blocks may start while the split kernel drains; they wait for its results.
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(blocks, (8 * NT + kJoinRows - 1) / kJoinRows);
  cfg.blockDim = dim3(kJoinThreads);
  cfg.stream = stream;
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, paged_join_kernel<D, NT>, p);
}

int resident_blocks(int D, int row_tile) {
  if (D == 128) return row_tile == 8 ? PagedCfg<128, 1>::kPerSm : PagedCfg<128, 2>::kPerSm;
  return row_tile == 8 ? PagedCfg<64, 1>::kPerSm : PagedCfg<64, 2>::kPerSm;
}

}  // namespace

int paged_row_tile(const PagedParams& p) {
  // Rows of a sequence and K/V head, on average: above 8, tiles of 16 rows read the cache half as often.
  const long long rows = static_cast<long long>(p.T) * p.group;
  return rows <= 8LL * p.B ? 8 : 16;
}

int paged_blocks(const PagedParams& p, int D) {
  const int row_tile = paged_row_tile(p);
  const int resident = resident_blocks(D, row_tile);  // blocks per SM
  const long long tiles = (static_cast<long long>(p.T) * p.group + row_tile - 1) / row_tile + p.B;
  const long long units = tiles * p.H_kv * ((p.capacity + kUnit - 1) / kUnit);
  return static_cast<int>(units < 148 * resident ? units : 148 * resident);
}

cudaError_t launch_paged(const PagedParams& p, int D, int blocks, cudaStream_t stream) {
  const bool join = p.capacity > kUnit;  // one unit per tile: nothing is ever cut
  const int row_tile = paged_row_tile(p);
#define FA_PAGED_CASE(DD)                                                       \
  if (D == DD) return row_tile == 8 ? launch_paged_t<DD, 1>(p, blocks, join, stream) \
                                    : launch_paged_t<DD, 2>(p, blocks, join, stream);
  FA_PAGED_CASE(32)
  FA_PAGED_CASE(64)
  FA_PAGED_CASE(128)
#undef FA_PAGED_CASE
  return cudaErrorInvalidValue;
}

}  // namespace fa
