// C-ABI entry points around attention (declared in include/fa_sm100.h): norm + rotary positions,
// appends to the paged e4m3 cache, attention over it.  Argument checks that need no device come
// first, then the device check, then the launch on the caller's stream; nothing is allocated.
#include <cstdint>

#include "../../include/fa_sm100.h"
#include "fa_internal.h"

namespace {

bool aligned(const void* p, uintptr_t to) { return (reinterpret_cast<uintptr_t>(p) & (to - 1)) == 0; }

bool overlap(const void* a, const void* b, size_t bytes) {
  const uintptr_t x = reinterpret_cast<uintptr_t>(a), y = reinterpret_cast<uintptr_t>(b);
  return (x < y ? y - x : x - y) < bytes;
}

bool head_dim_ok(int D) { return D == 32 || D == 64 || D == 128; }

int page_shift(int page_size) { return page_size == 16 ? 4 : (page_size == 32 ? 5 : (page_size == 64 ? 6 : 7)); }

// Strides of 16-bit rows: multiples of 8 elements (16 bytes).
template <int N>
bool strides_ok(const long long (&s)[N]) {
  for (int i = 0; i < N; ++i)
    if (s[i] % 8 != 0) return false;
  return true;
}

// Axes of a rotation and the first pair of each; unused entries are set past the last pair.
int check_axes(int axes, const int (&start)[4], int D, int max_pos, int (&out)[fa::kRopeMaxAxes]) {
  if (axes < 1 || max_pos < 1) return FA_ERR_INVALID_ARG;
  if (axes > fa::kRopeMaxAxes) return FA_ERR_UNSUPPORTED;
  if (start[0] != 0) return FA_ERR_INVALID_ARG;
  for (int a = 0; a < fa::kRopeMaxAxes; ++a) {
    out[a] = a < axes ? start[a] : D / 2;
    if (a > 0 && a < axes && (start[a] < start[a - 1] || start[a] > D / 2)) return FA_ERR_INVALID_ARG;
  }
  return FA_OK;
}

int check_weight(const void* w, int weight_dtype, int dtype) {
  if (w == nullptr) return FA_OK;
  if (weight_dtype != FA_DTYPE_F32 && weight_dtype != dtype) return FA_ERR_UNSUPPORTED;
  return aligned(w, 16) ? FA_OK : FA_ERR_ALIGNMENT;
}

int check_cache(int B, int T, int width, int num_pages, int H_kv, int page_size, int D, const void* k_pages,
                const void* v_pages, const void* k_scales, const void* v_scales, const void* table,
                const void* seq_lens, const void* offsets, int dtype) {
  if (!k_pages || !v_pages || !k_scales || !v_scales || !table || !seq_lens) return FA_ERR_INVALID_ARG;
  if (B < 1 || T < 1 || width < 1 || num_pages < 1 || H_kv < 1) return FA_ERR_INVALID_ARG;
  if (offsets == nullptr && T != B) return FA_ERR_INVALID_ARG;
  if (!head_dim_ok(D) || (dtype != FA_DTYPE_F16 && dtype != FA_DTYPE_BF16)) return FA_ERR_UNSUPPORTED;
  if (page_size != 16 && page_size != 32 && page_size != 64 && page_size != 128) return FA_ERR_UNSUPPORTED;
  // lengths and row indexes are 32-bit inside the kernels, and 2 H_kv is a grid dimension
  if (static_cast<long long>(width) * page_size > (1LL << 30) || H_kv > 32767 || T > (1 << 28)) return FA_ERR_UNSUPPORTED;
  if (!aligned(k_pages, 16) || !aligned(v_pages, 16) || !aligned(k_scales, 4) || !aligned(v_scales, 4) ||
      !aligned(table, 4) || !aligned(seq_lens, 4) || !aligned(offsets, 4))
    return FA_ERR_ALIGNMENT;
  return FA_OK;
}

int norm_rope_params(const fa_norm_rope_args* a, int* dev_status, bool backward, fa::RopeParams* p) {
  if (a == nullptr || dev_status == nullptr || !a->q || !a->cos || !a->sin) return FA_ERR_INVALID_ARG;
  if (a->B < 1 || a->H < 1 || a->N < 1 || a->H_kv < 0 || (a->H_kv > 0) != (a->k != nullptr)) return FA_ERR_INVALID_ARG;
  if (!head_dim_ok(a->D) || (a->dtype != FA_DTYPE_F16 && a->dtype != FA_DTYPE_BF16)) return FA_ERR_UNSUPPORTED;
  const long long tokens = static_cast<long long>(a->B) * a->N;
  if (tokens > 0x7fffffffLL || a->H > 32767 || a->H_kv > 32767) return FA_ERR_UNSUPPORTED;
  int rc = check_axes(a->axes, a->section_start, a->D, a->max_pos, p->section_start);
  if (rc != FA_OK) return rc;
  if ((rc = check_weight(a->q_weight, a->weight_dtype, a->dtype)) != FA_OK) return rc;
  if ((rc = check_weight(a->k_weight, a->weight_dtype, a->dtype)) != FA_OK) return rc;
  if (!backward && (!a->q_out || (a->k && !a->k_out))) return FA_ERR_INVALID_ARG;
  if (backward) {
    if (!a->dq_out || !a->dq || (a->k && (!a->dk_out || !a->dk))) return FA_ERR_INVALID_ARG;
    if ((a->dq_weight && !a->q_weight) || (a->dk_weight && !a->k_weight)) return FA_ERR_INVALID_ARG;
    if ((a->q_weight || a->k_weight) && !a->workspace) return FA_ERR_INVALID_ARG;
  }
  if (!aligned(a->q, 16) || !aligned(a->k, 16) || !aligned(a->q_out, 16) || !aligned(a->k_out, 16) ||
      !aligned(a->dq_out, 16) || !aligned(a->dk_out, 16) || !aligned(a->dq, 16) || !aligned(a->dk, 16) ||
      !aligned(a->cos, 16) || !aligned(a->sin, 16) || !aligned(a->workspace, 16) || !aligned(a->pos, a->pos_is_int64 ? 8 : 4) ||
      !strides_ok(a->q_stride) || (a->k && !strides_ok(a->k_stride)) ||
      (backward && (!strides_ok(a->dq_stride) || (a->k && !strides_ok(a->dk_stride)))))
    return FA_ERR_ALIGNMENT;
  p->q = a->q;
  p->k = a->k;
  p->q_weight = a->q_weight;
  p->k_weight = a->k_weight;
  p->cos = a->cos;
  p->sin = a->sin;
  p->pos = a->pos;
  p->q_out = a->q_out;
  p->k_out = a->k_out;
  p->dq_out = a->dq_out;
  p->dk_out = a->dk_out;
  p->dq = a->dq;
  p->dk = a->dk;
  p->dq_weight = a->dq_weight;
  p->dk_weight = a->dk_weight;
  p->workspace = a->workspace;
  for (int i = 0; i < 3; ++i) {
    p->q_stride[i] = a->q_stride[i];
    p->k_stride[i] = a->k_stride[i];
    p->dq_stride[i] = a->dq_stride[i];
    p->dk_stride[i] = a->dk_stride[i];
  }
  p->pos_axis_stride = a->pos_stride[0];
  p->pos_batch_stride = a->pos_stride[1];
  p->tokens = tokens;
  p->status = dev_status;
  p->H = a->H;
  p->H_kv = a->H_kv;
  p->N = a->N;
  p->max_pos = a->max_pos;
  p->axes = a->axes;
  p->pos64 = a->pos_is_int64;
  p->weight_f32 = a->weight_dtype == FA_DTYPE_F32;
  p->eps = a->eps;
  return fa::check_device();
}

}  // namespace

extern "C" {

int fa_norm_rope_fwd(const fa_norm_rope_args* args, int* dev_status, void* stream) {
  fa::RopeParams p{};
  const int rc = norm_rope_params(args, dev_status, false, &p);
  if (rc != FA_OK) return rc;
  const cudaError_t e = fa::launch_rope_fwd(p, args->D, args->dtype == FA_DTYPE_BF16, args->interleaved != 0,
                                            static_cast<cudaStream_t>(stream));
  return e == cudaSuccess ? FA_OK : fa::cuda_fail(e);
}

int fa_norm_rope_bwd(const fa_norm_rope_args* args, int* dev_status, void* stream) {
  fa::RopeParams p{};
  const int rc = norm_rope_params(args, dev_status, true, &p);
  if (rc != FA_OK) return rc;
  const cudaError_t e = fa::launch_rope_bwd(p, args->D, args->dtype == FA_DTYPE_BF16, args->interleaved != 0,
                                            static_cast<cudaStream_t>(stream));
  return e == cudaSuccess ? FA_OK : fa::cuda_fail(e);
}

int fa_append_kv(const fa_append_args* a, int* dev_status, void* stream) {
  if (a == nullptr || dev_status == nullptr || !a->k || !a->v) return FA_ERR_INVALID_ARG;
  int rc = check_cache(a->B, a->T, a->width, a->num_pages, a->H_kv, a->page_size, a->D, a->k_pages, a->v_pages,
                       a->k_scales, a->v_scales, a->block_table, a->seq_lens, a->offsets, a->dtype);
  if (rc != FA_OK) return rc;
  if ((rc = check_weight(a->k_weight, a->weight_dtype, a->dtype)) != FA_OK) return rc;
  fa::AppendParams p{};
  if (a->cos != nullptr) {
    if (a->sin == nullptr) return FA_ERR_INVALID_ARG;
    if ((rc = check_axes(a->axes, a->section_start, a->D, a->max_pos, p.section_start)) != FA_OK) return rc;
    if (a->axes > 1 && a->pos == nullptr) return FA_ERR_INVALID_ARG;
  }
  if (!aligned(a->k, 16) || !aligned(a->v, 16) || !aligned(a->cos, 16) || !aligned(a->sin, 16) ||
      !aligned(a->pos, a->pos_is_int64 ? 8 : 4) || !strides_ok(a->k_stride) || !strides_ok(a->v_stride))
    return FA_ERR_ALIGNMENT;
  // keys and values are written at the same time
  const size_t slots = static_cast<size_t>(a->num_pages) * a->H_kv;
  if (overlap(a->k_pages, a->v_pages, slots * a->page_size * a->D) || overlap(a->k_scales, a->v_scales, slots * sizeof(float)))
    return FA_ERR_INVALID_ARG;
  if ((rc = fa::check_device()) != FA_OK) return rc;
  p.k = a->k;
  p.v = a->v;
  p.k_pages = static_cast<uint8_t*>(a->k_pages);
  p.v_pages = static_cast<uint8_t*>(a->v_pages);
  p.k_scales = a->k_scales;
  p.v_scales = a->v_scales;
  p.block_table = a->block_table;
  p.seq_lens = a->seq_lens;
  p.offsets = a->offsets;
  p.cos = a->cos;
  p.sin = a->sin;
  p.pos = a->pos;
  p.k_weight = a->k_weight;
  for (int i = 0; i < 2; ++i) {
    p.k_stride[i] = a->k_stride[i];
    p.v_stride[i] = a->v_stride[i];
  }
  p.table_stride = a->table_stride;
  p.pos_axis_stride = a->pos_axis_stride;
  p.eps = a->eps;
  p.status = dev_status;
  p.T = a->T;
  p.B = a->B;
  p.width = a->width;
  p.num_pages = a->num_pages;
  p.H_kv = a->H_kv;
  p.page_shift = page_shift(a->page_size);
  p.max_pos = a->max_pos;
  p.axes = a->axes;
  p.pos64 = a->pos_is_int64;
  p.weight_f32 = a->weight_dtype == FA_DTYPE_F32;
  const cudaError_t e = fa::launch_append(p, a->D, a->dtype == FA_DTYPE_BF16, a->interleaved != 0,
                                          static_cast<cudaStream_t>(stream));
  return e == cudaSuccess ? FA_OK : fa::cuda_fail(e);
}

int fa_paged_attention(const fa_paged_args* a, int* dev_status, void* stream) {
  if (a == nullptr || dev_status == nullptr || !a->q || !a->out || !a->workspace) return FA_ERR_INVALID_ARG;
  int rc = check_cache(a->B, a->T, a->width, a->num_pages, a->H_kv, a->page_size, a->D, a->k_pages, a->v_pages,
                       a->k_scales, a->v_scales, a->block_table, a->seq_lens, a->offsets, a->dtype);
  if (rc != FA_OK) return rc;
  if (a->H < 1 || a->H % a->H_kv != 0) return FA_ERR_INVALID_ARG;
  if (!(a->scale > 0.f) || !(a->scale * 1.4426950408889634f < INFINITY)) return FA_ERR_INVALID_ARG;
  if (static_cast<long long>(a->T) * a->H > (1LL << 30)) return FA_ERR_UNSUPPORTED;
  if (!aligned(a->q, 16) || !aligned(a->out, 16) || !aligned(a->lse, 4) || !aligned(a->workspace, 16) ||
      !strides_ok(a->q_stride) || !strides_ok(a->out_stride))
    return FA_ERR_ALIGNMENT;
  if ((rc = fa::check_device()) != FA_OK) return rc;
  fa::PagedParams p{};
  p.q = a->q;
  p.k_pages = static_cast<const uint8_t*>(a->k_pages);
  p.v_pages = static_cast<const uint8_t*>(a->v_pages);
  p.k_scales = a->k_scales;
  p.v_scales = a->v_scales;
  p.block_table = a->block_table;
  p.seq_lens = a->seq_lens;
  p.offsets = a->offsets;
  p.out = a->out;
  p.lse = a->lse;
  for (int i = 0; i < 2; ++i) {
    p.q_stride[i] = a->q_stride[i];
    p.out_stride[i] = a->out_stride[i];
  }
  p.table_stride = a->table_stride;
  p.status = dev_status;
  p.T = a->T;
  p.B = a->B;
  p.num_pages = a->num_pages;
  p.H_kv = a->H_kv;
  p.group = a->H / a->H_kv;
  p.page_shift = page_shift(a->page_size);
  p.capacity = a->width * a->page_size;
  p.bf16 = a->dtype == FA_DTYPE_BF16;
  p.clear_unowned = a->clear_unowned;
  p.scale_log2 = a->scale * 1.4426950408889634f;
  if (fa::use_chunk(p, a->D)) {
    const cudaError_t e = fa::launch_chunk(p, a->D, static_cast<cudaStream_t>(stream));
    return e == cudaSuccess ? FA_OK : fa::cuda_fail(e);
  }
  const int blocks = fa::paged_blocks(p, a->D);
  const size_t rows = 2 * static_cast<size_t>(blocks) * fa::paged_row_tile(p);
  p.joins = static_cast<fa::PagedJoin*>(a->workspace);  // 24 bytes each, then 16-byte aligned arrays
  uint8_t* at = static_cast<uint8_t*>(a->workspace) + (blocks * sizeof(fa::PagedJoin) + 15) / 16 * 16;
  p.part_ml = reinterpret_cast<float2*>(at);
  at += rows * sizeof(float2);
  p.parts = reinterpret_cast<float*>(at);
  at += rows * a->D * sizeof(float);
  if (at - static_cast<uint8_t*>(a->workspace) > FA_PAGED_WORKSPACE_BYTES(a->D)) return FA_ERR_UNSUPPORTED;
  const cudaError_t e = fa::launch_paged(p, a->D, blocks, static_cast<cudaStream_t>(stream));
  return e == cudaSuccess ? FA_OK : fa::cuda_fail(e);
}

}  // extern "C"
