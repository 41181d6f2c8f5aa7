// Attention over a paged e4m3 cache for many query rows (prompts in chunks behind what is cached), for
// sm_100a: tcgen05 UMMA on f16 tiles that a warpgroup makes from the cached bytes.
//
//   s_j = (q . k8_j) * k_scale(page j) * scale,   o = sum_j softmax(s)_j * v_scale(page j) * v8_j
// Token i of a sequence's n new tokens, at sequence length L, sees keys j <= L - n + i.
//
// Bound: the tensor cores and the exponentials, as in the dense forward (fa_fwd.cu), whose structure
// this is: a block owns two 128-row query tiles that read the same K/V head, one thread per row.  Here
//   * rows are (token, head of the group) pairs, so a tile of a group of G heads covers 128 / G tokens and
//     every cached byte a block reads serves 256 rows;
//   * K and V tiles are built by a warpgroup of their own: 16-byte pieces of a page, e4m3 -> f16 (exact),
//     into the swizzled layout that the tensor core reads.  The tiles hold the cached values themselves;
//   * pages' scales are float32 factors of the softmax, whatever their size.  A key's scale is part of the
//     factor that its score has anyway.  A value's scale w rides in the weights' exponents,
//       p' = 2^(s - m + log2 w - u),   O += p' v8,   l += 2^(u - log2 w) p',   o = 2^u O / l,
//     with m the largest s that the row has seen and m + u the largest s + log2 w.  So P stays inside f16 and
//     nothing that a row does not see has a part in it.  The factors are the same for kSeg keys of one page: per
//     row and kSeg keys one exponential, two products and some ten additions and maxima more;
//   * queries are brought to f16 by a power of two per row (exact down to 2^-31 of the row's largest
//     element) by the thread that owns the row; P is f16.
// Warp roles (512 threads):
//   warps 0-3, 4-7  softmax warpgroups of query tiles 0 and 1 (they load Q and write O)
//   warp 8          UMMA issuer: S_t = Q_t K_j^T, O_t += P_t V_j with P_t in TMEM
//   warps 9-11      V tiles: 16-key blocks, three, three and two of a tile's eight
//   warps 12-15     K tiles: two 16-key blocks each
// Registers: 128 a thread at launch; warps 8-15 drop to kRegsOther, the softmax warps rise to
// kRegsSoftmax, and 256 x kRegsOther + 256 x kRegsSoftmax = 512 x 128.
// TMEM (512 columns): S_0 | S_1 | O_0 | O_1, P_t over the first half of S_t; P is published in two halves.
#include "fa_internal.h"
#include "fa_paged.cuh"
#include "fa_sm100.cuh"
#include "fa_softmax.cuh"

#include <type_traits>

namespace fa {
namespace {

constexpr int kThreads = 512;
constexpr int kSoftmaxWarps = 8;
constexpr int kWarpMma = 8;
constexpr int kWarpV = 9;        // first of the three warps that build V tiles
constexpr int kWarpK = 12;       // first of the four warps that build K tiles
constexpr int kBM = 128;
constexpr int kBN = 128;
constexpr uint32_t kTmemCols = 512;
constexpr float kRescaleThreshold = 8.0f;  // log2 units
constexpr int kLaunchRegs = 128;
constexpr int kRegsSoftmax = 192;
constexpr int kRegsOther = 64;
static_assert(256 * kRegsOther + 256 * kRegsSoftmax <= kThreads * kLaunchRegs, "register split");
constexpr int kSoftmaxCopy = 1;  // the softmax warpgroups' own copy of the bounded-wait loop
// Of 16 exp2 pairs on interior tiles, those on the FMA pipe.  The conversions share that pipe's issue slots, so fewer
// pay than in the dense forward: chunks of 1024, 437 and 1024 tokens behind up to 8192 keys take 303 us with one, 307 with
// two; with pages of 16 keys 573 and 592 us for 4736 tokens behind 8192.
constexpr int kPolyPairs = 1;
// log2 of a value's scale is taken to be at least this far below the row's best weight: then p' of a score next to m is
// 2^-60, which f16 rounds to 0 as it would the smaller exact one, while float32 still holds what l needs of it.
constexpr float kScaleFloor = -60.f;
constexpr float kNoScale = -200.f;  // stands for log2 0: below every float32's
// The softmax subtracts the rounded reference from a product that is not rounded, which is off by up to half a step of the
// reference.  Up to here that is less than 1 and the same for all weights of a row; tiles that could hold larger scores
// (log2 units) go through large_tile.
constexpr float kLargeScore = 16777216.f;

template <int D>
struct ChunkCfg {
  static constexpr int kSwBytes = D >= 64 ? 128 : 64;  // a shared-memory row: one swizzle span
  static constexpr uint32_t kLayout = D >= 64 ? kLayoutSw128 : kLayoutSw64;
  static constexpr int kSbo = 8 * kSwBytes;
  static constexpr int kKStepsPerChunk = kSwBytes / 32;
  static constexpr int kChunkBytes = 128 * kSwBytes;   // Q, K and V tiles all have 128 rows
  static constexpr int kTileBytes = 128 * D * 2;
  static constexpr int kStages = D == 128 ? 2 : 4;     // K and V rings
  static constexpr int kOffQ = 0;
  static constexpr int kOffK = 2 * kTileBytes;
  static constexpr int kOffV = kOffK + kStages * kTileBytes;
  static constexpr int kOffRaw = kOffV + kStages * kTileBytes;  // the next K and V tiles' cached bytes
  static constexpr int kOffBar = kOffRaw + 2 * 128 * D;
  static constexpr int kOffFactors = kOffBar + 512;     // [softmax warp][parity of the tile][16]
  static constexpr int kSmemBytes = kOffFactors + kSoftmaxWarps * 2 * 16 * 4 + 1024;  // alignment slack
  // Byte offset of 16-byte piece c of row r of an f16 tile (pieces of D / 8 per row).
  static __device__ __forceinline__ uint32_t place(int r, int c) {
    if constexpr (D >= 64) return (c >> 3) * kChunkBytes + r * 128 + (((c & 7) ^ (r & 7)) << 4);
    return r * 64 + ((c ^ ((r >> 1) & 3)) << 4);
  }
};

enum : int {
  BAR_Q = 0,        // + tile (2)
  BAR_KFULL = 2,    // + stage (4)
  BAR_KEMPTY = 6,
  BAR_VFULL = 10,
  BAR_VEMPTY = 14,
  BAR_SFULL = 18,   // + tile (2)
  BAR_PFULLA = 20,
  BAR_PFULLB = 22,
  BAR_OFULL = 24,
  BAR_DRAIN = 26,
  BAR_NEVER = 27,   // never arrived at (the failure-detection test build waits on it)
  BAR_COUNT = 28
};

// One 16-byte piece of a cached row -> 16 f16 values.
__device__ __forceinline__ void to_f16(const uint4& raw, uint4& lo, uint4& hi) {
  const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
  uint32_t h[8];
#pragma unroll
  for (int i = 0; i < 4; ++i)
    asm("{\n\t.reg .b16 x, y;\n\tmov.b32 {x, y}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, x;\n\tcvt.rn.f16x2.e4m3x2 %1, y;\n\t}"
        : "=r"(h[2 * i]), "=r"(h[2 * i + 1]) : "r"(w[i]));
  lo = make_uint4(h[0], h[1], h[2], h[3]);
  hi = make_uint4(h[4], h[5], h[6], h[7]);
}

// The largest of N scores from `r` on.
template <int N>
__device__ __forceinline__ float top_of(const uint32_t* r) {
  constexpr int kChains = N / 8;
  float top[kChains];
#pragma unroll
  for (int u = 0; u < kChains; ++u) top[u] = fmaxf(__uint_as_float(r[2 * u]), __uint_as_float(r[2 * u + 1]));
#pragma unroll
  for (int i = kChains; i < N / 2; ++i)
    top[i % kChains] = fmax3(top[i % kChains], __uint_as_float(r[2 * i]), __uint_as_float(r[2 * i + 1]));
  if constexpr (kChains == 4) return fmaxf(fmax3(top[0], top[1], top[2]), top[3]);
  return fmaxf(top[0], top[1]);
}

// Weights p' = 2^(s factor + shift) of N scores as pairs of f16, added up in `sum`; the first pair is number kFirst of
// its 16.  kPolyPairs of those are a polynomial where `poly` (not on tiles with hidden keys, whose scores are -inf).
template <int N, int kFirst, bool poly>
__device__ __forceinline__ void weigh(const uint32_t* r, float factor, float shift, uint64_t (&sum)[4], uint32_t* pk) {
  const uint64_t factor2 = f2(factor, factor), shift2 = f2(shift, shift);
#pragma unroll
  for (int i = 0; i < N / 2; ++i) {
    const uint64_t x2 = ffma2(f2u(r[2 * i], r[2 * i + 1]), factor2, shift2);
    uint64_t p2;
    if (poly && (kFirst + i) % (16 / kPolyPairs) == 16 / kPolyPairs - 1) {
      // the polynomial is finite whatever x is: NaN reaches the row through the sum
      p2 = exp2_poly2(x2);
      sum[i & 3] = fadd2(sum[i & 3], ffma2(x2, 0ull, p2));
    } else {
      p2 = f2(ex2_approx(f2lo(x2)), ex2_approx(f2hi(x2)));
      sum[i & 3] = fadd2(sum[i & 3], p2);
    }
    pk[i] = pack2<false>(f2lo(p2), f2hi(p2));
  }
}

// S = Q K^T for one tile.
template <int D>
__device__ __forceinline__ void issue_qk(uint32_t d_tmem, uint64_t q_desc, uint64_t k_desc) {
  using C = ChunkCfg<D>;
  constexpr uint32_t IDESC = idesc_f16(false, kBM, kBN, false, false);
  constexpr int KS = C::kKStepsPerChunk;
#pragma unroll
  for (int k = 0; k < D / 16; ++k)
    umma_ss_w(d_tmem, desc_add(q_desc, (k / KS) * C::kChunkBytes + (k % KS) * 32),
              desc_add(k_desc, (k / KS) * C::kChunkBytes + (k % KS) * 32), IDESC, k > 0 ? 1u : 0u);
}

// O += P V over one half of the tile's keys.
template <int D>
__device__ __forceinline__ void issue_pv_half(uint32_t o_tmem, uint32_t p_tmem, uint64_t v_desc, uint32_t accumulate, int half) {
  constexpr uint32_t IDESC = idesc_f16(false, kBM, D, false, true);
  constexpr int kKeyStep = 16 * ChunkCfg<D>::kSwBytes;
  constexpr int kSteps = kBN / 32;
#pragma unroll
  for (int i = 0; i < kSteps; ++i) {
    const int k = half * kSteps + i;
    umma_ts_w(o_tmem, p_tmem + k * 8, desc_add(v_desc, k * kKeyStep), IDESC, (accumulate | k) ? 1u : 0u);
  }
}

constexpr int kNanWord = 6;  // words[kNanWord]: a value that some row may not see is NaN

struct ChunkWork {
  int b, h;       // sequence, K/V head; b < 0: nothing to do
  int first, n;   // flat index of the sequence's first new token, their number
  int before;     // keys in front of the new tokens
  int r0;         // first of the block's 256 rows
};

// blockIdx.x -> work: sequences in order, inside a sequence the last (longest) rows first, heads
// next to each other.  Every thread calls it.
__device__ __forceinline__ ChunkWork find_work(const PagedParams& p, int* words) {
  __shared__ long long warp_sum[kThreads / 32];
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const int chunk = (p.B + kThreads - 1) / kThreads;
  const int b0 = min(p.B, static_cast<int>(threadIdx.x) * chunk), b1 = min(p.B, b0 + chunk);
  if (threadIdx.x == 0) {
    words[0] = -1;
    words[kNanWord] = 0;
  }
  long long mine = 0;
  int first = 0, n = 0, len = 0;
  auto shape = [&](int b) {
    first = p.offsets == nullptr ? b : p.offsets[b];
    n = p.offsets == nullptr ? 1 : p.offsets[b + 1] - first;
    if (first < 0 || n < 0 || first > p.T - n) {  // not inside q: no rows
      if (n != 0) record_error(p.status, kDevBadIndex, b);
      first = n = 0;
    }
    len = p.seq_lens[b];
    if (len < 0 || len > p.capacity) {
      record_error(p.status, kDevBadIndex, b);
      len = 0;
    }
    return static_cast<long long>((n * p.group + 2 * kBM - 1) / (2 * kBM)) * p.H_kv;
  };
  for (int b = b0; b < b1; ++b) mine += shape(b);
  long long incl = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long v = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += v;
  }
  if (lane == 31) warp_sum[warp] = incl;
  __syncthreads();
  long long before = incl - mine;
  for (int w = 0; w < warp; ++w) before += warp_sum[w];
  const long long item = blockIdx.x;
  if (item >= before && item < before + mine) {
    for (int b = b0; b < b1; ++b) {
      const long long items = shape(b);
      if (item < before + items) {
        const int i = static_cast<int>(item - before);
        words[0] = b;
        words[1] = i % p.H_kv;
        words[2] = first;
        words[3] = n;
        words[4] = len - n;
        words[5] = (static_cast<int>(items / p.H_kv) - 1 - i / p.H_kv) * 2 * kBM;
        break;
      }
      before += items;
    }
  }
  __syncthreads();
  return {words[0], words[1], words[2], words[3], words[4], words[5]};
}

// One tile of a row's softmax with scores of any size, which are rounded before the reference is subtracted: the
// same sums as in the kernel's loop, through TMEM in pieces of 32 columns.  factors: the segments' key scales, then
// log2 of their value scales; keys from `hidden` on are not seen.  The row's m, u and l go in and come back by value: by
// reference the kernel's loop keeps them in memory (chunks of 1024 behind 8192 keys 312 us instead of 303).
template <int D, int kSeg>
__device__ __noinline__ float3 large_tile(uint32_t t_s, uint32_t t_o, const float* factors, float row_factor, int hidden,
                                          bool first, float m, float u, float l) {
  constexpr int kSegs = kBN / kSeg, kPiece = kSeg < 32 ? kSeg : 32;
  uint32_t x[32];
  float top = -INFINITY;
#pragma unroll 1
  for (int c = 0; c < kBN / 32; ++c) {
    tmem_ld32(t_s + c * 32, x);
    tmem_ld_wait(x);
#pragma unroll
    for (int i = 0; i < 32; ++i) {
      const float v = __fmul_rn(__uint_as_float(x[i]), factors[(c * 32 + i) / kSeg] * row_factor);
      x[i] = __float_as_uint(c * 32 + i < hidden ? v : -INFINITY);
    }
    top = fmaxf(top, top_of<32>(x));
    tmem_st32(t_s + c * 32, x);
  }
  tmem_st_wait();
  const bool up = top > m + kRescaleThreshold;
  const float m_new = up ? top : m, u_old = up ? u + (m - m_new) : u;
  float top_u = -INFINITY;
#pragma unroll 1
  for (int c = 0; c < kBN / 32; ++c) {
    tmem_ld32(t_s + c * 32, x);
    tmem_ld_wait(x);
#pragma unroll
    for (int i = 0; i < 32; i += kPiece)
      top_u = fmaxf(top_u, (top_of<kPiece>(&x[i]) - m_new) + factors[kSegs + (c * 32 + i) / kSeg]);
  }
  const bool up_u = top_u > u_old + kRescaleThreshold;
  const float u_new = up_u ? top_u : u_old;
  if (!first && __any_sync(0xffffffffu, up_u)) rescale_o<D>(t_o, up_u ? ex2_approx(u_old - u_new) : 1.f);
  float sum = 0.f;
#pragma unroll 1
  for (int c = 0; c < kBN / 32; ++c) {
    tmem_ld32(t_s + c * 32, x);
    tmem_ld_wait(x);
    uint32_t pk[16];
#pragma unroll
    for (int i = 0; i < 32; i += 2) {
      const float log_scale = fmaxf(factors[kSegs + (c * 32 + i) / kSeg], u_new + kScaleFloor) - u_new;
      const float a = ex2_approx(__fsub_rn(__uint_as_float(x[i]), m_new) + log_scale);
      const float b = ex2_approx(__fsub_rn(__uint_as_float(x[i + 1]), m_new) + log_scale);
      sum = fmaf(a + b, ex2_approx(-log_scale), sum);
      pk[i / 2] = pack2<false>(a, b);
    }
    tmem_st16(t_s + c * 16, pk);  // over columns that have been read
  }
  return make_float3(m_new, u_new, l * (up ? ex2_approx(m - m_new) : 1.f) + sum);
}

// kSeg: keys that share their factors for sure, the page size up to 64.
template <int D, int kSeg>
__global__ void __launch_bounds__(kThreads, 1) paged_chunk_kernel(const PagedParams p) {
  using C = ChunkCfg<D>;
  constexpr int ST = C::kStages;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw_base = smem_u32(smem_raw);
  const uint32_t base = (raw_base + 1023u) & ~1023u;
  uint8_t* smem = smem_raw + (base - raw_base);
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + C::kOffBar);
  volatile uint32_t* tmem_slot = reinterpret_cast<volatile uint32_t*>(smem + C::kOffBar + 8 * BAR_COUNT);
  int* words = reinterpret_cast<int*>(smem + C::kOffBar + 8 * BAR_COUNT + 16);
  const uint32_t bar0 = smem_u32(bars);
#define BAR(i) (bar0 + 8u * static_cast<uint32_t>(i))
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;

  if (__syncthreads_or(ld_status(p.status)) != 0) return;
  clear_unowned_rows<D>(p);
  const ChunkWork w = find_work(p, words);
  if (w.b < 0) return;
  const int rows = min(2 * kBM, w.n * p.group - w.r0);
  const int ntiles = rows > kBM ? 2 : 1;
  // keys that a tile's last row sees; a tile that sees none still runs over key 0 when the block has one
  auto keys_of = [&](int t) {
    const int last = w.r0 + min(rows, (t + 1) * kBM) - 1;
    return w.before + last / p.group + 1;
  };
  const int keys = max(0, keys_of(ntiles - 1));  // <= the sequence's length
  const int* table = p.block_table + w.b * p.table_stride;

  if (keys == 0) {  // no row sees a key
    for (int i = threadIdx.x; i < rows * (D / 8); i += kThreads) {
      const int r = w.r0 + i / (D / 8), head = w.h * p.group + r % p.group;
      const long long token = w.first + r / p.group;
      *reinterpret_cast<uint4*>(static_cast<uint16_t*>(p.out) + token * p.out_stride[0] + head * p.out_stride[1] + i % (D / 8) * 8) =
          make_uint4(0, 0, 0, 0);
      if (p.lse != nullptr && i % (D / 8) == 0) p.lse[token * p.group * p.H_kv + head] = -INFINITY;
    }
    return;
  }

  const int pages = ((keys - 1) >> p.page_shift) + 1;
  if (threadIdx.x == 0) {
    mbar_init(BAR(BAR_Q), 128);
    mbar_init(BAR(BAR_Q + 1), 128);
    for (int s = 0; s < 4; ++s) {
      mbar_init(BAR(BAR_KFULL + s), 128);
      mbar_init(BAR(BAR_KEMPTY + s), 1);
      mbar_init(BAR(BAR_VFULL + s), 96);
      mbar_init(BAR(BAR_VEMPTY + s), 1);
    }
    for (int t = 0; t < 2; ++t) {
      mbar_init(BAR(BAR_SFULL + t), 1);
      mbar_init(BAR(BAR_PFULLA + t), 128);
      mbar_init(BAR(BAR_PFULLB + t), 128);
      mbar_init(BAR(BAR_OFULL + t), 1);
    }
    mbar_init(BAR(BAR_DRAIN), 1);
    mbar_init(BAR(BAR_NEVER), 1);
    fence_barrier_init();
  }
  if (warp == 0) {
    tmem_alloc(smem_u32(const_cast<uint32_t*>(tmem_slot)), kTmemCols);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  const int nkv0 = (max(1, keys_of(0)) + kBN - 1) / kBN;
  const int nkv1 = ntiles == 2 ? (max(1, keys_of(1)) + kBN - 1) / kBN : 0;
  const int nmax = max(nkv0, nkv1);
  const uint32_t sK = base + C::kOffK, sV = base + C::kOffV;
  // the first key tile that some row of the block does not see to its end
  const int first_hidden = max(0, w.before + w.r0 / p.group + 1) / kBN;

  if (warp >= kSoftmaxWarps) {
    regs_decrease<kRegsOther>();
    if (warp == kWarpMma) {
      // ---------------------------------------------------------- UMMA issuer
      const uint64_t dq0 = sdesc_sw(base + C::kOffQ, 16, C::kSbo, C::kLayout);
      const uint64_t dq1 = sdesc_sw(base + C::kOffQ + C::kTileBytes, 16, C::kSbo, C::kLayout);
      const uint64_t dk0 = sdesc_sw(sK, 16, C::kSbo, C::kLayout);
      const uint64_t dv0 = sdesc_sw(sV, C::kChunkBytes, C::kSbo, C::kLayout);
      const uint32_t tS0 = tmem, tS1 = tmem + 128, tO0 = tmem + 256, tO1 = tmem + 384;
      bool ok = warp_all(mbar_wait(BAR(BAR_Q), 0, p.status, kDevTimeoutQ)) &&
                warp_all(mbar_wait(BAR(BAR_KFULL + 0), 0, p.status, kDevTimeoutKV));
      if (ok && nkv1 > 0) ok = warp_all(mbar_wait(BAR(BAR_Q + 1), 0, p.status, kDevTimeoutQ));
      if (ok) {
        tc_fence_after();
        issue_qk<D>(tS0, dq0, dk0);
        umma_commit_w(BAR(BAR_SFULL + 0));
        if (nkv1 > 0) {
          issue_qk<D>(tS1, dq1, dk0);
          umma_commit_w(BAR(BAR_SFULL + 1));
        }
        umma_commit_w(BAR(BAR_KEMPTY + 0));
      }
      for (int j = 0; ok && j < nmax; ++j) {
        const int vs = j % ST, ks1 = (j + 1) % ST;
        const uint64_t dvj = dv0 + static_cast<uint64_t>((vs * C::kTileBytes) >> 4);
        const uint64_t dkn = dk0 + static_cast<uint64_t>((ks1 * C::kTileBytes) >> 4);
        FA_STALL_HERE(j, BAR(BAR_NEVER), p.status, ok)
        if (!(ok = warp_all(mbar_wait(BAR(BAR_VFULL + vs), (j / ST) & 1, p.status, kDevTimeoutKV)))) break;
        bool k_ready = false, issued_s = false;
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          const int nt = t == 0 ? nkv0 : nkv1;
          const uint32_t tS = t == 0 ? tS0 : tS1, tO = t == 0 ? tO0 : tO1;
          if (j < nt) {
            if (!(ok = warp_all(mbar_wait(BAR(BAR_PFULLA + t), j & 1, p.status, kDevTimeoutP)))) break;
            tc_fence_after();
            issue_pv_half<D>(tO, tS, dvj, j > 0 ? 1u : 0u, 0);
            if (!(ok = warp_all(mbar_wait(BAR(BAR_PFULLB + t), j & 1, p.status, kDevTimeoutP)))) break;
            tc_fence_after();
            issue_pv_half<D>(tO, tS, dvj, 1u, 1);
            if (j + 1 == nt) {
              umma_commit_w(BAR(BAR_OFULL + t));
            } else {
              if (!k_ready) {
                if (!(ok = warp_all(mbar_wait(BAR(BAR_KFULL + ks1), ((j + 1) / ST) & 1, p.status, kDevTimeoutKV)))) break;
                tc_fence_after();
                k_ready = true;
              }
              issue_qk<D>(tS, t == 0 ? dq0 : dq1, dkn);
              umma_commit_w(BAR(BAR_SFULL + t));
              issued_s = true;
            }
          }
        }
        if (!ok) break;
        if (issued_s) umma_commit_w(BAR(BAR_KEMPTY + ks1));
        umma_commit_w(BAR(BAR_VEMPTY + vs));
      }
      umma_commit_w(BAR(BAR_DRAIN));
      drain_wait(BAR(BAR_DRAIN), 0, p.status);
      __syncwarp();
    } else {
      // ---------------------------------------------------------- K and V tiles, 16 keys at a time
      constexpr int kLanes = D / 16;             // lanes of a cached row
      constexpr int kRowsPerLoad = 32 / kLanes;
      constexpr int kLoads = 16 / kRowsPerLoad;  // a thread's pieces of a block
      const bool is_k = warp >= kWarpK;
      const int first_block = is_k ? 2 * (warp - kWarpK) : 3 * (warp - kWarpV);
      const int blocks = is_k ? 2 : (warp == kWarpV + 2 ? 2 : 3);
      constexpr int kMost = 3;                   // blocks of a warp, at most
      const int row_in_block = lane / kLanes, piece = lane % kLanes;
      const uint8_t* bytes = (is_k ? p.k_pages : p.v_pages) + piece * 16;
      uint8_t* ring = smem + (is_k ? C::kOffK : C::kOffV);
      // A block's bytes wait in shared memory (asynchronous copies, each thread its own pieces) from the
      // moment the block of the tile before has been converted: nearly a tile's time in flight.
      const uint8_t* raw = smem + C::kOffRaw + (is_k ? 0 : 128 * D) + first_block * 16 * D + lane * 16;
      const uint32_t full = BAR(is_k ? BAR_KFULL : BAR_VFULL), empty = BAR(is_k ? BAR_KEMPTY : BAR_VEMPTY);
      const uint32_t page_bytes = static_cast<uint32_t>(D) << p.page_shift;
      const int page_mask = (1 << p.page_shift) - 1;
      int page[kMost] = {};  // of the block's next copy, read a tile ahead
      auto page_of = [&](int j, int blk) {
        return table[min((j * kBN + (first_block + blk) * 16) >> p.page_shift, pages - 1)];
      };
      auto copy = [&](int j, int blk) {
        if (j < nmax) {
          const int key0 = j * kBN + (first_block + blk) * 16;
          const size_t at = static_cast<size_t>(page[blk] < 0 || page[blk] >= p.num_pages ? 0 : page[blk]) * p.H_kv + w.h;
          // rows behind the last key are inside the page: read, and cleared when they are converted
          const uint8_t* src = bytes + at * page_bytes + (key0 & page_mask) * D + row_in_block * D;
#pragma unroll
          for (int i = 0; i < kLoads; ++i)
            asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(raw + blk * 16 * D + i * 512)),
                         "l"(src + i * 512) : "memory");
          page[blk] = page_of(j + 1, blk);
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
      };
#pragma unroll
      for (int blk = 0; blk < kMost; ++blk) page[blk] = page_of(0, blk);
#pragma unroll
      for (int blk = 0; blk < kMost; ++blk)
        if (blk < blocks) copy(0, blk);
      bool ok = true;
      auto convert_tile = [&](int j, auto clean) {
        const int st = j % ST;
        uint8_t* tile = ring + st * C::kTileBytes;
        if (!(ok = mbar_wait(empty + 8 * st, ((j / ST) & 1) ^ 1, p.status, kDevTimeoutKVEmpty))) return;
#pragma unroll
        for (int blk = 0; blk < kMost; ++blk) {
          if (blk < blocks) {
            // the oldest of the warp's `blocks` copies in flight has landed
            if (blocks == 2)
              asm volatile("cp.async.wait_group 1;" ::: "memory");
            else
              asm volatile("cp.async.wait_group 2;" ::: "memory");
            const int row0 = (first_block + blk) * 16 + row_in_block;
#pragma unroll
            for (int i = 0; i < kLoads; ++i) {
              const int row = row0 + i * kRowsPerLoad;
              uint4 v = *reinterpret_cast<const uint4*>(raw + blk * 16 * D + i * 512);
              if (j * kBN + row >= keys) v = make_uint4(0, 0, 0, 0);  // behind the last key
              if constexpr (decltype(clean)::value) {
                const uint4 nan = make_uint4(nan_bytes(v.x), nan_bytes(v.y), nan_bytes(v.z), nan_bytes(v.w));
                if ((nan.x | nan.y | nan.z | nan.w) != 0) *const_cast<volatile int*>(&words[kNanWord]) = 1;
                v = make_uint4(v.x & ~nan.x, v.y & ~nan.y, v.z & ~nan.z, v.w & ~nan.w);
              }
              uint4 lo, hi;
              to_f16(v, lo, hi);
              // lanes of the two halves of a row store their two pieces in opposite order: the eight lanes
              // of a row then meet all banks
              const bool swap = D == 128 && piece >= 4;
              *reinterpret_cast<uint4*>(tile + C::place(row, 2 * piece + (swap ? 1 : 0))) = swap ? hi : lo;
              *reinterpret_cast<uint4*>(tile + C::place(row, 2 * piece + (swap ? 0 : 1))) = swap ? lo : hi;
            }
            copy(j + 1, blk);
          }
        }
        fence_async_shared();
        mbar_arrive(full + 8 * st);
      };
      // Values that some row does not see: NaN is taken out (0 * NaN is not 0) and put back at the end.  A loop of
      // its own: it costs 2 % of the kernel's time, in the common loop it cost 15 %.
      const int plain = is_k ? nmax : min(nmax, first_hidden);
      int j = 0;
      for (; ok && j < plain; ++j) convert_tile(j, std::false_type{});
      for (; ok && j < nmax; ++j) convert_tile(j, std::true_type{});
      asm volatile("cp.async.wait_all;" ::: "memory");
      __syncwarp();
    }
  } else {
    // ------------------------------------------------------------ softmax / epilogue, one thread per row
    regs_increase<kRegsSoftmax>();
    const int t = warp / 4;
    if (t < ntiles) {
      constexpr int NCH = kBN / 32;
      const int wq = warp % 4;
      const int row = wq * 32 + lane;
      const int r = w.r0 + t * kBM + row;
      const bool live = r < w.n * p.group;
      const int head = w.h * p.group + r % p.group;
      const long long token = w.first + r / p.group;
      // the row's last key; rows that see none run over key 0 and are written as such at the end
      const int own_last = live ? w.before + r / p.group : 0;
      const int last = max(0, own_last);
      const int full = max(0, w.before + (w.r0 + t * kBM) / p.group);  // every row of the tile sees keys <= full
      // The tile's factors: lane g loads the key scale of segment g, lane kSegs + g the value scale, a tile ahead
      // (and the page two ahead); the warp's lanes then read them in shared memory.
      constexpr int kSegs = kBN / kSeg;
      float* factors = reinterpret_cast<float*>(smem + C::kOffFactors) + warp * 32;
      const bool loads = lane < 2 * kSegs;
      const float* scales = lane < kSegs ? p.k_scales : p.v_scales;
      auto page_of = [&](int j) { return table[min((j * kBN + lane % kSegs * kSeg) >> p.page_shift, pages - 1)]; };
      auto scale_of = [&](int page) {
        if (page < 0 || page >= p.num_pages) {
          record_error(p.status, kDevBadIndex, w.b);
          page = 0;
        }
        return scales[static_cast<size_t>(page) * p.H_kv + w.h];
      };
      float next = 0.f;
      int next_page = 0;
      if (loads) {
        next = scale_of(page_of(0));
        next_page = page_of(1);
      }
      // Q row -> f16 by a power of two
      float row_factor, large_scale;  // a key scale from which the warp's scores could be large
      {
        uint8_t* tile = smem + C::kOffQ + t * C::kTileBytes;
        const uint16_t* q = static_cast<const uint16_t*>(p.q) + token * p.q_stride[0] + head * p.q_stride[1];
        uint32_t x[D / 8][4];
        uint32_t top = 0;
#pragma unroll
        for (int c = 0; c < D / 8; ++c) {
          const uint4 v = live ? *reinterpret_cast<const uint4*>(q + 8 * c) : make_uint4(0, 0, 0, 0);
          x[c][0] = v.x;
          x[c][1] = v.y;
          x[c][2] = v.z;
          x[c][3] = v.w;
#pragma unroll
          for (int i = 0; i < 4; ++i) top = max(top, max(x[c][i] & 0x7fffu, (x[c][i] >> 16) & 0x7fffu));
        }
        float down = 1.f;
        if (p.bf16) {
          const int e = min(254, max(8, static_cast<int>(top >> 7)));   // biased exponent
          down = __uint_as_float(static_cast<uint32_t>(261 - e) << 23); // largest element to [2^7, 2^8)
        }
#pragma unroll
        for (int c = 0; c < D / 8; ++c) {
          uint4 v = make_uint4(x[c][0], x[c][1], x[c][2], x[c][3]);
          if (p.bf16) {
#pragma unroll
            for (int i = 0; i < 4; ++i)
              x[c][i] = pack2<false>(__uint_as_float(x[c][i] << 16) * down, __uint_as_float(x[c][i] & 0xffff0000u) * down);
            v = make_uint4(x[c][0], x[c][1], x[c][2], x[c][3]);
          }
          *reinterpret_cast<uint4*>(tile + C::place(row, c)) = v;
        }
        row_factor = p.scale_log2 / down;
        float size = 0.f;
#pragma unroll
        for (int c = 0; c < D / 8; ++c)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float2 v = __half22float2(*reinterpret_cast<const __half2*>(&x[c][i]));
            size += fabsf(v.x) + fabsf(v.y);
          }
        size *= row_factor;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) size = fmaxf(size, __shfl_xor_sync(0xffffffffu, size, o));
        large_scale = kLargeScore / (448.f * size);
        fence_async_shared();
        mbar_arrive(BAR(BAR_Q + t));
      }
      const int nkv = t == 0 ? nkv0 : nkv1;
      const uint32_t lane_off = static_cast<uint32_t>(wq * 32) << 16;
      const uint32_t tS = tmem + t * 128 + lane_off;
      const uint32_t tO = tmem + 256 + t * 128 + lane_off;
      // References: m of the scores, m + u of the scores plus log2 of their value's scale (u by itself, small next to m).
      float m = -INFINITY, u = 0.f;
      float l = 0.f;
      bool ok = true;
      for (int j = 0; j < nkv; ++j) {
        float* tile_factors = factors + (j & 1) * 16;
        const bool large = __any_sync(0xffffffffu, lane < kSegs && next > large_scale);
        if (loads) {
          tile_factors[lane] = lane < kSegs ? next : (next > 0.f ? log2f(next) : kNoScale);
          next = scale_of(next_page);
          next_page = page_of(j + 2);
        }
        __syncwarp();
        if (!(ok = warp_all(mbar_wait<kSoftmaxCopy>(BAR(BAR_SFULL + t), j & 1, p.status, kDevTimeoutS)))) break;
        tc_fence_after();
        const int kbase = j * kBN;
        if (large) {
          const float3 state = large_tile<D, kSeg>(tS, tO, tile_factors, row_factor, last + 1 - kbase, j == 0, m, u, l);
          m = state.x;
          u = state.y;
          l = state.z;
          tmem_st_wait();
          tc_fence_before();
          mbar_arrive(BAR(BAR_PFULLA + t));
          mbar_arrive(BAR(BAR_PFULLB + t));
          continue;
        }
        uint32_t s[NCH][32];
#pragma unroll
        for (int c = 0; c < NCH; ++c) tmem_ld32(tS + c * 32, s[c]);
#pragma unroll
        for (int c = 0; c < NCH; ++c) tmem_ld_wait(s[c]);
        const bool masked = kbase + kBN - 1 > full;
        // On tiles with hidden keys not 0, which it is for a scale of zero and rounds to for tiny ones: hidden scores are
        // -inf before they are multiplied, and -inf * 0 is NaN.  2^-126 leaves every finite score within 2^-80 of the 0
        // that it stands for.
        auto score_factor = [&](int g, auto hides) {
          const float f = tile_factors[g] * row_factor;
          return decltype(hides)::value ? fmaxf(f, 0x1p-126f) : f;
        };
        uint64_t sum2 = 0ull;
        // The weights of half a tile, into TMEM and sum2.  hides: the tile has hidden keys, no polynomial.
        auto weigh_half = [&](int h, auto hides) {
          constexpr bool poly = !decltype(hides)::value;
          constexpr int kPiece = kSeg < 32 ? kSeg : 32;
          float factor, shift, log_scale;
          uint64_t sum[4];
#pragma unroll
          for (int c = h * NCH / 2; c < (h + 1) * NCH / 2; ++c) {
            uint32_t pk[16];
#pragma unroll
            for (int at = 0; at < 32; at += kPiece) {
              const int col = c * 32 + at, g = col / kSeg;
              if (col % kSeg == 0) {
                factor = score_factor(g, hides);
                log_scale = fmaxf(tile_factors[kSegs + g], u + kScaleFloor) - u;
                shift = log_scale - m;
                sum[0] = sum[1] = sum[2] = sum[3] = 0ull;
              }
              if (at == 0)
                weigh<kPiece, 0, poly>(&s[c][0], factor, shift, sum, pk);
              else
                weigh<kPiece, kPiece % 32 / 2, poly>(&s[c][kPiece % 32], factor, shift, sum, pk + kPiece % 32 / 2);
              if ((col + kPiece) % kSeg == 0) {
                const float back = ex2_approx(-log_scale);
                sum2 = ffma2(fadd2(fadd2(sum[0], sum[1]), fadd2(sum[2], sum[3])), f2(back, back), sum2);
              }
            }
            tmem_st16(tS + c * 16, pk);
          }
        };
        // Raises the references where the tile's maxima pass one by the threshold; l's and O's factors for that.
        float alpha = 1.f, alpha_o = 1.f;
        auto raise = [&](auto hides) {
          float top = -INFINITY, top_w = -INFINITY;
#pragma unroll
          for (int g = 0; g < kSegs; ++g) {
            float x = top_of<kSeg < 32 ? kSeg : 32>(&s[g * kSeg / 32][g * kSeg % 32]);
            if constexpr (kSeg == 64) x = fmaxf(x, top_of<32>(s[2 * g + 1]));
            x *= score_factor(g, hides);
            top = fmaxf(top, x);
            top_w = fmaxf(top_w, x + tile_factors[kSegs + g]);
          }
          const float mw = m + u;
          const bool up = top > m + kRescaleThreshold || top_w > mw + kRescaleThreshold;
          if (up) {
            const float m_new = fmaxf(m, top), u_new = fmaxf(mw, top_w) - m_new;
            alpha = ex2_approx(m - m_new);
            alpha_o = ex2_approx((m - m_new) + (u - u_new));
            m = m_new;
            u = u_new;
          }
          return __any_sync(0xffffffffu, up) != 0;
        };
        if (masked || j == 0) {
          if (masked) {
#pragma unroll
            for (int c = 0; c < NCH; ++c)
#pragma unroll
              for (int i = 0; i < 32; ++i)
                if (kbase + c * 32 + i > last) s[c][i] = __float_as_uint(-INFINITY);
          }
          const bool any = raise(std::true_type{});
          if (j > 0 && any) rescale_o<D>(tO, alpha_o);
          weigh_half(0, std::true_type{});
          weigh_half(1, std::true_type{});
          tmem_st_wait();
          tc_fence_before();
          mbar_arrive(BAR(BAR_PFULLA + t));
          mbar_arrive(BAR(BAR_PFULLB + t));
        } else {
          // the first half with the running references while the tile's maxima are computed beside it
          weigh_half(0, std::false_type{});
          if (raise(std::false_type{})) {
            sum2 = 0ull;
            weigh_half(0, std::false_type{});
            rescale_o<D>(tO, alpha_o);
          }
          tmem_st_wait();
          tc_fence_before();
          mbar_arrive(BAR(BAR_PFULLA + t));
          weigh_half(1, std::false_type{});
          tmem_st_wait();
          tc_fence_before();
          mbar_arrive(BAR(BAR_PFULLB + t));
        }
        l = l * alpha + (f2lo(sum2) + f2hi(sum2));
      }
      if (ok) ok = mbar_wait<kSoftmaxCopy>(BAR(BAR_OFULL + t), 0, p.status, kDevTimeoutO);
      ok = warp_all(ok);
      if (ok) {
        tc_fence_after();
        const bool seen = own_last >= 0;
        const float f = seen ? exp2f(u) / l : 0.f;
        uint16_t* out = static_cast<uint16_t*>(p.out) + token * p.out_stride[0] + head * p.out_stride[1];
#pragma unroll 1
        for (int c = 0; c < D / 32; ++c) {
          uint32_t o[32];
          tmem_ld32(tO + c * 32, o);
          tmem_ld_wait(o);
          if (live) {
#pragma unroll
            for (int v = 0; v < 4; ++v) {
              uint32_t pk[4];
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                const float a = seen ? __uint_as_float(o[8 * v + 2 * i]) * f : 0.f;
                const float b = seen ? __uint_as_float(o[8 * v + 2 * i + 1]) * f : 0.f;
                pk[i] = p.bf16 ? pack2<true>(a, b) : pack2<false>(a, b);
              }
              *reinterpret_cast<uint4*>(out + c * 32 + 8 * v) = make_uint4(pk[0], pk[1], pk[2], pk[3]);
            }
          }
        }
        if (p.lse != nullptr && live) p.lse[token * p.group * p.H_kv + head] = seen ? m + log2f(l) : -INFINITY;
        if (*const_cast<volatile int*>(&words[kNanWord]) != 0 && live) {  // rare: NaN among the values that the row sees
#pragma unroll 1
          for (int key = first_hidden * kBN; key <= own_last; ++key) {
            const int page = table[key >> p.page_shift];
            if (page < 0 || page >= p.num_pages) continue;
            const uint8_t* v = p.v_pages + (((static_cast<size_t>(page) * p.H_kv + w.h) << p.page_shift) +
                                            (key & ((1 << p.page_shift) - 1))) * D;
#pragma unroll 1
            for (int d = 0; d < D; d += 4) {
              const uint32_t nan = nan_bytes(*reinterpret_cast<const uint32_t*>(v + d));
              for (int i = 0; nan != 0 && i < 4; ++i)
                if ((nan >> (8 * i) & 1u) != 0) out[d + i] = 0x7fff;  // NaN in both types
            }
          }
        }
      }
    }
  }
#undef BAR

  tc_fence_before();
  __syncthreads();
  if (warp == 0) {
    tc_fence_after();
    tmem_dealloc(tmem, kTmemCols);
  }
}

template <int D, int kSeg>
cudaError_t launch_chunk_t(const PagedParams& p, int blocks, cudaStream_t stream) {
  static std::atomic<bool> smem_set[64];
  const cudaError_t e = opt_in_smem(paged_chunk_kernel<D, kSeg>, ChunkCfg<D>::kSmemBytes, smem_set, kLaunchRegs);
  if (e != cudaSuccess) return e;
  paged_chunk_kernel<D, kSeg><<<blocks, kThreads, ChunkCfg<D>::kSmemBytes, stream>>>(p);
  return cudaGetLastError();
}

}  // namespace

// Blocks of 256 rows, at most: per K/V head, the whole ones and a last one for each sequence.
static long long chunk_blocks(const PagedParams& p) {
  return (static_cast<long long>(p.T) * p.group / (2 * kBM) + p.B) * p.H_kv;
}

// Which kernel takes a call, by the two's times for its 128-key tiles.  The split kernel spends c1 = 7 ns of the whole GPU
// on 16 rows and 128 keys at D = 128 (4.2 ns at D = 64), the chunk kernel c2 of one SM on a block's rows: 2.1 us
// with up to 128 of them, 2.5 to 2.8 with more.  The border is c2 / c1 = 320 at D = 128 and 400 below.  Measured at
// D = 128, 8 K/V heads, groups of 4, 8192 keys, chunk / split in us: 16 x 16 tokens 147 / 226, 16 x 10 tokens 144 / 176,
// 1 x 256 tokens 167 / 194, 1 x 208 tokens 166 / 163, 1 x 160 tokens (the border) 167 / 131, 4 x 16 tokens 140 / 69, 1 x 64
// tokens 166 / 64: with one sequence the border is low, with many it is not.  Only averages are known here:
// sequences' lengths are on the device.
bool use_chunk(const PagedParams& p, int D) {
  if (chunk_blocks(p) > 0x7fffffffLL) return false;
#ifdef FA_CHUNK_ROWS  // a build that picks by rows alone, to time one kernel against the other
  return static_cast<long long>(p.T) * p.group >= static_cast<long long>(FA_CHUNK_ROWS) * p.B;
#else
  const long long rows = (static_cast<long long>(p.T) * p.group + p.B - 1) / p.B;  // of a sequence and K/V head
  const long long items = static_cast<long long>(p.B) * p.H_kv;
  const long long waves = (items * ((rows + 2 * kBM - 1) / (2 * kBM)) + 147) / 148;
  return items * ((rows + 15) / 16) >= (D == 128 ? 320 : 400) * waves;
#endif
}

cudaError_t launch_chunk(const PagedParams& p, int D, cudaStream_t stream) {
  const int blocks = static_cast<int>(chunk_blocks(p));
#define FA_CHUNK_CASE(DD) \
  if (D == DD)                                                                                                  \
    return p.page_shift == 4 ? launch_chunk_t<DD, 16>(p, blocks, stream)                                        \
                             : (p.page_shift == 5 ? launch_chunk_t<DD, 32>(p, blocks, stream) : launch_chunk_t<DD, 64>(p, blocks, stream));
  FA_CHUNK_CASE(32)
  FA_CHUNK_CASE(64)
  FA_CHUNK_CASE(128)
#undef FA_CHUNK_CASE
  return cudaErrorInvalidValue;
}

}  // namespace fa
