// Python binding of the operators around attention: norm + rotary positions (with autograd), appends
// to the paged e4m3 cache, attention over it.  Checks the tensors, allocates outputs and workspaces
// with torch's allocator, and calls the C ABI (include/fa_sm100.h) on torch's current stream.
//
// These calls are short (a decode step's kernels take a few microseconds), so their host side is
// native: the same checks and packing in Python took 20 to 30 us a call, and a Python autograd
// function another 100 us a step, most of it handing the interpreter lock to the engine's thread.
#include <torch/extension.h>

#include <ATen/MemoryOverlap.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>

#include <cmath>
#include <limits>

#include "../../include/fa_sm100.h"

namespace py = pybind11;
using at::Tensor;
using OptTensor = std::optional<Tensor>;
using Sections = std::optional<std::vector<int64_t>>;

namespace {

// ---------------------------------------------------------------------------------- status words
// One int32[4] per device, owned by the Python binding (attention/_lib.py), which hands it over on
// first use.
constexpr int kMaxDevices = 64;
int* g_status[kMaxDevices] = {};
py::object* g_status_provider = nullptr;

int* status_word(const Tensor& t) {
  const int device = t.get_device();
  TORCH_CHECK(device >= 0 && device < kMaxDevices, "device index ", device, " is not supported");
  if (g_status[device] == nullptr) {
    py::gil_scoped_acquire gil;
    cudaStreamCaptureStatus capture = cudaStreamCaptureStatusNone;
    C10_CUDA_CHECK(cudaStreamIsCapturing(c10::cuda::getCurrentCUDAStream(device), &capture));
    TORCH_CHECK(capture == cudaStreamCaptureStatusNone || py::cast<bool>((*g_status_provider)(device, true)),
                "the first call on a device allocates its status word: make one before capturing a graph");
    g_status[device] = reinterpret_cast<int*>(py::cast<uintptr_t>((*g_status_provider)(device, false)));
  }
  return g_status[device];
}

// Runs one C entry point on t's device and current stream; its error codes become exceptions.
template <typename Args>
void call(int (*entry)(const Args*, int*, void*), const Args& args, const Tensor& t, const char* what) {
  int* status = status_word(t);
  c10::cuda::OptionalCUDAGuard guard;
  if (t.get_device() != c10::cuda::current_device()) guard.set_device(t.device());
  const int rc = entry(&args, status, c10::cuda::getCurrentCUDAStream(t.get_device()).stream());
  if (rc == FA_OK) return;
  TORCH_CHECK_VALUE(rc != FA_ERR_INVALID_ARG && rc != FA_ERR_UNSUPPORTED && rc != FA_ERR_ALIGNMENT, what, ": ", fa_strerror(rc));
  TORCH_CHECK(rc != FA_ERR_CUDA, what, ": ", fa_strerror(rc), ": ", fa_last_cuda_error());
  TORCH_CHECK(false, what, ": ", fa_strerror(rc));
}

// -------------------------------------------------------------------------------- shared helpers
bool on16(const Tensor& t) { return (reinterpret_cast<uintptr_t>(t.const_data_ptr()) & 15) == 0; }

const void* ptr(const Tensor& t) { return t.defined() ? t.const_data_ptr() : nullptr; }
void* out_ptr(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }

bool half_type(const Tensor& t) { return t.scalar_type() == at::kHalf || t.scalar_type() == at::kBFloat16; }
int type_code(const Tensor& t) {
  return t.scalar_type() == at::kHalf ? FA_DTYPE_F16 : (t.scalar_type() == at::kBFloat16 ? FA_DTYPE_BF16 : FA_DTYPE_F32);
}

// Strides of x in front of its last dimension (0 for dimensions of size 1); whether the kernels can
// read it as it is: contiguous in the last dimension, base and strides on 16-byte boundaries.
template <int N>
bool row_strides(const Tensor& x, long long (&s)[N]) {
  bool ok = x.stride(N) == 1 && on16(x);
  for (int i = 0; i < N; ++i) {
    s[i] = x.size(i) == 1 ? 0 : x.stride(i);
    ok = ok && s[i] % 8 == 0;
  }
  return ok;
}
// x, or a copy where the kernels cannot read x.
template <int N>
Tensor rows(const Tensor& x, long long (&s)[N]) {
  if (row_strides(x, s)) return x;
  Tensor c = x.clone(at::MemoryFormat::Contiguous);
  row_strides(c, s);
  return c;
}
Tensor aligned(const Tensor& x) {
  if (!x.defined()) return x;
  const Tensor c = x.contiguous();
  return on16(c) ? c : c.clone();
}

// A call writes into t: a backward pass that saved t before notices.  (Inference tensors have no version.)
void written(const Tensor& t) {
  if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}

// Dual tensors: the kernels give no tangents, and dropping one would be silent.
void check_no_tangent(const char* what, std::initializer_list<OptTensor> tensors) {
  for (const OptTensor& t : tensors)
    TORCH_CHECK(!t.has_value() || !t->defined() || !t->_fw_grad(/*level=*/0).defined(), what, " has no forward-mode derivative");
}

struct Turn {  // a rotation's checked arguments
  Tensor cos, sin, pos;
  int start[4] = {0, 0, 0, 0};
  int axes = 1;
  long long pos_stride[2] = {0, 0};  // axis, batch
};

// `lead`: the dimensions a position tensor has in front of its tokens, apart from the axes (a batch
// of `batch`, which may be left out, or none).
Turn check_turn(const Tensor& like, const Tensor& cos, const Tensor& sin, const OptTensor& pos, const Sections& sections,
                int64_t tokens, int64_t batch) {
  const int64_t D = like.size(-1);
  Turn t;
  TORCH_CHECK_TYPE(cos.scalar_type() == at::kFloat && sin.scalar_type() == at::kFloat, "cos and sin must be float32, got ",
                   cos.scalar_type(), " and ", sin.scalar_type());
  TORCH_CHECK_VALUE(cos.dim() == 2 && cos.sizes() == sin.sizes() && cos.size(1) * 2 == D && cos.size(0) >= 1 &&
                        cos.size(0) <= std::numeric_limits<int>::max(),
                    "cos and sin must both be (max_pos, ", D / 2, "); got ", cos.sizes(), ", ", sin.sizes());
  TORCH_CHECK_VALUE(cos.device() == like.device() && sin.device() == like.device(), "cos and sin must be on ", like.device(),
                    ", got ", cos.device(), " and ", sin.device());
  if (sections.has_value()) {
    const auto& s = *sections;
    int64_t sum = 0;
    bool ok = s.size() >= 1 && s.size() <= 4;
    for (size_t i = 0; ok && i < s.size(); ++i) {
      t.start[i] = static_cast<int>(sum);
      ok = s[i] >= 0 && s[i] <= D / 2;
      sum += s[i];
    }
    TORCH_CHECK_VALUE(ok && sum == D / 2, "sections must be 1 to 4 pair counts that add up to D/2=", D / 2, ", got ", s);
    t.axes = static_cast<int>(s.size());
    TORCH_CHECK_VALUE(pos.has_value(), "sections need positions, one row for each axis");
  }
  if (pos.has_value()) {
    Tensor p = *pos;
    TORCH_CHECK_TYPE(p.scalar_type() == at::kInt || p.scalar_type() == at::kLong, "positions must be int32 or int64, got ",
                     p.scalar_type());
    const int64_t lead = sections.has_value() ? 1 : 0, dims = p.dim() - lead;
    TORCH_CHECK_VALUE((dims == 1 || (dims == 2 && batch >= 0 && p.size(lead) == batch)) && p.size(-1) == tokens &&
                          (lead == 0 || p.size(0) == t.axes),
                      "positions must be ", lead ? "(axes, " : "(", batch >= 0 ? "[B,] " : "", "tokens=", tokens, "), got ", p.sizes());
    TORCH_CHECK_VALUE(p.device() == like.device(), "positions must be on ", like.device(), ", got ", p.device());
    if (p.size(-1) > 1 && p.stride(-1) != 1) p = p.contiguous();
    t.pos_stride[0] = lead ? p.stride(0) : 0;
    t.pos_stride[1] = dims == 2 ? p.stride(lead) : 0;
    t.pos = p;
  }
  t.cos = aligned(cos);
  t.sin = aligned(sin);
  return t;
}

void check_weight(const char* name, const Tensor& w, const Tensor& x) {
  TORCH_CHECK_TYPE(w.scalar_type() == at::kFloat || w.scalar_type() == x.scalar_type(), name, " must be float32 or ",
                   x.scalar_type(), ", got ", w.scalar_type());
  TORCH_CHECK_VALUE(w.dim() == 1 && w.size(0) == x.size(-1), name, " must be (", x.size(-1), ",), got ", w.sizes());
  TORCH_CHECK_VALUE(w.device() == x.device(), name, " must be on ", x.device(), ", got ", w.device());
}

// --------------------------------------------------------------------------------- norm + rotary
fa_norm_rope_args rope_args(const Tensor& q, const Tensor& k, const Tensor& qw, const Tensor& kw, const Turn& t, double eps,
                            bool interleaved) {
  fa_norm_rope_args a{};
  a.q = ptr(q);
  a.k = ptr(k);
  a.q_weight = ptr(qw);
  a.k_weight = ptr(kw);
  a.cos = t.cos.const_data_ptr<float>();
  a.sin = t.sin.const_data_ptr<float>();
  a.pos = ptr(t.pos);
  a.pos_stride[0] = t.pos_stride[0];
  a.pos_stride[1] = t.pos_stride[1];
  a.B = static_cast<int>(q.size(0));
  a.H = static_cast<int>(q.size(1));
  a.H_kv = k.defined() ? static_cast<int>(k.size(1)) : 0;
  a.N = static_cast<int>(q.size(2));
  a.D = static_cast<int>(q.size(3));
  a.dtype = type_code(q);
  a.weight_dtype = qw.defined() ? type_code(qw) : (kw.defined() ? type_code(kw) : a.dtype);
  a.max_pos = static_cast<int>(t.cos.size(0));
  a.axes = t.axes;
  for (int i = 0; i < 4; ++i) a.section_start[i] = t.start[i];
  a.pos_is_int64 = t.pos.defined() && t.pos.scalar_type() == at::kLong;
  a.interleaved = interleaved;
  a.eps = static_cast<float>(eps);
  return a;
}

std::pair<Tensor, Tensor> rope_forward(const Tensor& q, const Tensor& k, const Tensor& qw, const Tensor& kw, const Turn& t,
                                       double eps, bool interleaved) {
  Tensor q_out = at::empty(q.sizes(), q.options());
  Tensor k_out = k.defined() ? at::empty(k.sizes(), k.options()) : Tensor();
  if (q.numel() == 0) return {q_out, k_out};
  fa_norm_rope_args a{};
  long long qs[3], ks[3] = {0, 0, 0};
  const Tensor qr = rows(q, qs), kr = k.defined() ? rows(k, ks) : k;
  const Tensor qwa = aligned(qw), kwa = aligned(kw);
  a = rope_args(qr, kr, qwa, kwa, t, eps, interleaved);
  for (int i = 0; i < 3; ++i) {
    a.q_stride[i] = qs[i];
    a.k_stride[i] = ks[i];
  }
  a.q_out = q_out.data_ptr();
  a.k_out = out_ptr(k_out);
  call(fa_norm_rope_fwd, a, q, "qk_norm_rope");
  return {q_out, k_out};
}

// An uninitialised gradient of x: token-major in memory where x is, else head-major.
Tensor empty_like_rows(const Tensor& x) {
  if (x.stride(1) < x.stride(2))
    return at::empty({x.size(0), x.size(2), x.size(1), x.size(3)}, x.options()).transpose(1, 2);
  return at::empty(x.sizes(), x.options());
}

struct NormRope : torch::autograd::Function<NormRope> {
  static torch::autograd::variable_list forward(torch::autograd::AutogradContext* ctx, const Tensor& q, const OptTensor& k_opt,
                                                const OptTensor& qw_opt, const OptTensor& kw_opt, const Turn& t, double eps,
                                                bool interleaved) {
    const Tensor k = k_opt.value_or(Tensor()), qw = qw_opt.value_or(Tensor()), kw = kw_opt.value_or(Tensor());
    ctx->save_for_backward({q, k, qw, kw, t.cos, t.sin, t.pos});
    ctx->saved_data["turn"] = std::vector<int64_t>{t.start[0], t.start[1], t.start[2], t.start[3], t.axes, t.pos_stride[0],
                                                   t.pos_stride[1], interleaved};
    ctx->saved_data["eps"] = eps;
    const auto [q_out, k_out] = rope_forward(q, k, qw, kw, t, eps, interleaved);
    if (!k.defined()) return {q_out};
    return {q_out, k_out};
  }

  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx, torch::autograd::variable_list grads) {
    TORCH_CHECK(!at::GradMode::is_enabled(), "qk_norm_rope cannot be differentiated twice (create_graph=True)");
    const auto saved = ctx->get_saved_variables();
    const Tensor &q = saved[0], &k = saved[1], &qw = saved[2], &kw = saved[3];
    const auto v = ctx->saved_data["turn"].toIntVector();
    Turn t;
    t.cos = saved[4];
    t.sin = saved[5];
    t.pos = saved[6];
    for (int i = 0; i < 4; ++i) t.start[i] = static_cast<int>(v[i]);
    t.axes = static_cast<int>(v[4]);
    t.pos_stride[0] = v[5];
    t.pos_stride[1] = v[6];
    // gradients are asked for by the place among the tensors that were given
    const size_t at_qw = k.defined() ? 2 : 1, at_kw = at_qw + (qw.defined() ? 1 : 0);
    const bool want_qw = qw.defined() && ctx->needs_input_grad(at_qw), want_kw = kw.defined() && ctx->needs_input_grad(at_kw);
    if (q.numel() == 0)
      return {at::zeros_like(q), k.defined() ? at::zeros_like(k) : Tensor(), want_qw ? at::zeros_like(qw) : Tensor(),
              want_kw ? at::zeros_like(kw) : Tensor(), Tensor(), Tensor(), Tensor()};
    Tensor dq = empty_like_rows(q), dk = k.defined() ? empty_like_rows(k) : Tensor();
    Tensor dqw = want_qw ? at::empty(qw.sizes(), qw.options()) : Tensor();
    Tensor dkw = want_kw ? at::empty(kw.sizes(), kw.options()) : Tensor();
    Tensor workspace;
    if (qw.defined() || kw.defined()) workspace = at::empty({FA_ROPE_WORKSPACE_ROWS, q.size(3)}, q.options().dtype(at::kFloat));
    fa_norm_rope_args a{};
    long long qs[3], ks[3] = {0, 0, 0}, dqs[3], dks[3] = {0, 0, 0};
    const Tensor qr = rows(q, qs), kr = k.defined() ? rows(k, ks) : k;
    const Tensor qwa = aligned(qw), kwa = aligned(kw);
    const Tensor dzq = aligned(grads[0]), dzk = k.defined() ? aligned(grads[1]) : Tensor();
    row_strides(dq, dqs);
    if (k.defined()) row_strides(dk, dks);
    a = rope_args(qr, kr, qwa, kwa, t, ctx->saved_data["eps"].toDouble(), v[7] != 0);
    for (int i = 0; i < 3; ++i) {
      a.q_stride[i] = qs[i];
      a.k_stride[i] = ks[i];
      a.dq_stride[i] = dqs[i];
      a.dk_stride[i] = dks[i];
    }
    a.dq_out = ptr(dzq);
    a.dk_out = ptr(dzk);
    a.dq = dq.data_ptr();
    a.dk = out_ptr(dk);
    a.dq_weight = out_ptr(dqw);
    a.dk_weight = out_ptr(dkw);
    a.workspace = workspace.defined() ? workspace.data_ptr<float>() : nullptr;
    call(fa_norm_rope_bwd, a, q, "qk_norm_rope backward");
    return {dq, dk, dqw, dkw, Tensor(), Tensor(), Tensor()};
  }
};

std::pair<Tensor, OptTensor> qk_norm_rope(const Tensor& q, const OptTensor& k_opt, const Tensor& cos, const Tensor& sin,
                                          const OptTensor& positions, const OptTensor& q_weight, const OptTensor& k_weight,
                                          double eps, bool interleaved, const Sections& sections) {
  const Tensor k = k_opt.value_or(Tensor());
  check_no_tangent("qk_norm_rope", {q, k_opt, cos, sin, q_weight, k_weight});
  TORCH_CHECK_TYPE(half_type(q) && (!k.defined() || k.scalar_type() == q.scalar_type()), "q, k must be float16 (or both bfloat16)");
  TORCH_CHECK_VALUE(q.dim() == 4 && q.size(1) >= 1 &&
                        (!k.defined() || (k.dim() == 4 && k.size(1) >= 1 && k.size(0) == q.size(0) && k.size(2) == q.size(2) &&
                                          k.size(3) == q.size(3))),
                    "q, k must be (B, H, N, D) and (B, H_kv, N, D); got ", q.sizes(), k.defined() ? ", " : "",
                    k.defined() ? k.sizes() : at::IntArrayRef());
  const int64_t D = q.size(3);
  TORCH_CHECK_VALUE(D == 32 || D == 64 || D == 128, "head dim D=", D, " not supported; allowed (32, 64, 128)");
  const Turn t = check_turn(q, cos, sin, positions, sections, q.size(2), q.size(0));
  TORCH_CHECK_VALUE(k.defined() || !k_weight.has_value(), "k_weight is given without k");
  if (q_weight.has_value()) check_weight("q_weight", *q_weight, q);
  if (k_weight.has_value()) check_weight("k_weight", *k_weight, k);
  TORCH_CHECK_TYPE(!q_weight.has_value() || !k_weight.has_value() || q_weight->scalar_type() == k_weight->scalar_type(),
                   "q_weight and k_weight must share one dtype, got ", q_weight->scalar_type(), " and ", k_weight->scalar_type());
  TORCH_CHECK_VALUE(q.is_cuda() && (!k.defined() || k.device() == q.device()), "q, k must be on one CUDA device, got ", q.device(),
                    k.defined() ? ", " : "", k.defined() ? k.device().str() : "");
  TORCH_CHECK_VALUE(q.numel() == 0 || (q.size(0) * q.size(2) <= std::numeric_limits<int>::max() && q.size(1) < 32768 &&
                                       (!k.defined() || k.size(1) < 32768)),
                    "B * N must stay below 2^31 and the heads below 2^15, got ", q.sizes());
  const Tensor qw = q_weight.value_or(Tensor()), kw = k_weight.value_or(Tensor());
  const bool grad = at::GradMode::is_enabled() && (q.requires_grad() || (k.defined() && k.requires_grad()) ||
                                                   (qw.defined() && qw.requires_grad()) || (kw.defined() && kw.requires_grad()));
  if (grad) {
    const auto out = NormRope::apply(q, k_opt, q_weight, k_weight, t, eps, interleaved);
    return {out[0], k.defined() ? OptTensor(out[1]) : std::nullopt};
  }
  const auto [q_out, k_out] = rope_forward(q, k, qw, kw, t, eps, interleaved);
  return {q_out, k.defined() ? OptTensor(k_out) : std::nullopt};
}

// ----------------------------------------------------------------------------------------- cache
void check_cache(const Tensor& kp, const Tensor& vp, const Tensor& ks, const Tensor& vs) {
  TORCH_CHECK_TYPE(kp.scalar_type() == at::kFloat8_e4m3fn && vp.scalar_type() == at::kFloat8_e4m3fn,
                   "k_pages and v_pages must be float8_e4m3fn, got ", kp.scalar_type(), " and ", vp.scalar_type());
  TORCH_CHECK_TYPE(ks.scalar_type() == at::kFloat && vs.scalar_type() == at::kFloat, "k_scales and v_scales must be float32, got ",
                   ks.scalar_type(), " and ", vs.scalar_type());
  TORCH_CHECK_VALUE(kp.dim() == 4 && vp.sizes() == kp.sizes() && ks.sizes() == kp.sizes().slice(0, 2) && vs.sizes() == ks.sizes(),
                    "pages must be (num_pages, H_kv, page_size, D) and scales (num_pages, H_kv); got ", kp.sizes(), ", ", vp.sizes(),
                    ", ", ks.sizes(), ", ", vs.sizes());
  const int64_t P = kp.size(2), D = kp.size(3);
  TORCH_CHECK_VALUE((P == 16 || P == 32 || P == 64 || P == 128) && (D == 32 || D == 64 || D == 128) && kp.size(0) >= 1 &&
                        kp.size(1) >= 1 && kp.size(0) <= std::numeric_limits<int>::max(),
                    "page_size must be one of (16, 32, 64, 128) and D one of (32, 64, 128), got ", kp.sizes());
  for (const Tensor* x : {&kp, &vp, &ks, &vs})
    TORCH_CHECK_VALUE(x->device() == kp.device() && x->is_contiguous(), "pages and scales must be contiguous on one device (", kp.device(), ")");
  TORCH_CHECK_VALUE(on16(kp) && on16(vp), "pages must start on 16-byte boundaries");
}

// The batch's tables against the cache and T tokens on `device`.
void check_batch(const Tensor& kp, const Tensor& table, const Tensor& lens, const OptTensor& offsets, int64_t T, at::Device device) {
  TORCH_CHECK_TYPE(table.scalar_type() == at::kInt, "block_table must be int32, got ", table.scalar_type());
  TORCH_CHECK_TYPE(lens.scalar_type() == at::kInt, "seq_lens must be int32, got ", lens.scalar_type());
  TORCH_CHECK_TYPE(!offsets.has_value() || offsets->scalar_type() == at::kInt, "offsets must be int32, got ", offsets->scalar_type());
  TORCH_CHECK_VALUE(lens.dim() == 1 && (lens.size(0) <= 1 || lens.stride(0) == 1), "seq_lens must be (B,) and contiguous, got ", lens.sizes());
  const int64_t B = lens.size(0);
  TORCH_CHECK_VALUE(table.dim() == 2 && table.size(0) == B && table.size(1) >= 1 && (table.size(1) == 1 || table.stride(1) == 1),
                    "block_table must be (B=", B, ", pages) and contiguous in its last dimension, got ", table.sizes());
  TORCH_CHECK_VALUE(!offsets.has_value() || (offsets->dim() == 1 && offsets->size(0) == B + 1 && (B == 0 || offsets->stride(0) == 1)),
                    "offsets must be (B + 1 = ", B + 1, ",) and contiguous, got ", offsets->sizes());
  TORCH_CHECK_VALUE(offsets.has_value() || T == B, "without offsets there is one token per sequence: got ", T, " tokens, ", B, " sequences");
  TORCH_CHECK_VALUE(table.device() == device && lens.device() == device && (!offsets.has_value() || offsets->device() == device) &&
                        kp.device() == device,
                    "the tokens, the tables and the cache must be on one device, got ", device, ", ", table.device(), ", ", lens.device(),
                    ", ", kp.device());
  TORCH_CHECK_VALUE(device.is_cuda(), "the tokens and the cache must be on a CUDA device, got ", device);
  TORCH_CHECK_VALUE(B <= (1 << 24) && T <= (1 << 28) && table.size(1) * kp.size(2) <= (1 << 30),
                    "at most 2^24 sequences, 2^28 tokens and 2^30 tokens in a row of the block table; got ", B, ", ", T, ", ", table.sizes());
}

void append_kv(const Tensor& kp, const Tensor& vp, const Tensor& ks, const Tensor& vs, const Tensor& k, const Tensor& v,
               const Tensor& table, const Tensor& lens, const OptTensor& offsets, const OptTensor& cos, const OptTensor& sin,
               const OptTensor& positions, const OptTensor& k_weight, double eps, bool interleaved, const Sections& sections) {
  check_no_tangent("append_kv", {k, v, cos, sin, k_weight});
  TORCH_CHECK_TYPE(half_type(k) && v.scalar_type() == k.scalar_type(), "k, v must be float16 (or both bfloat16)");
  TORCH_CHECK(!at::GradMode::is_enabled() ||
                  !(k.requires_grad() || v.requires_grad() || (k_weight.has_value() && k_weight->requires_grad())),
              "append_kv has no backward: call it under torch.no_grad()");
  for (const Tensor* x : {&kp, &vp, &ks, &vs})
    TORCH_CHECK(!at::GradMode::is_enabled() || !x->requires_grad(), "append_kv writes into the cache, which must not require a gradient");
  check_cache(kp, vp, ks, vs);
  auto apart = [](const Tensor& x, const Tensor& y) {
    const uintptr_t i = reinterpret_cast<uintptr_t>(x.const_data_ptr()), j = reinterpret_cast<uintptr_t>(y.const_data_ptr());
    return (i < j ? j - i : i - j) >= x.nbytes();
  };
  TORCH_CHECK_VALUE(apart(kp, vp) && apart(ks, vs), "append_kv writes keys and values: their pages and scales must not share memory");
  const int64_t H_kv = kp.size(1), D = kp.size(3);
  TORCH_CHECK_VALUE(k.dim() == 3 && v.sizes() == k.sizes() && k.size(1) == H_kv && k.size(2) == D, "k, v must be (T, H_kv=", H_kv,
                    ", D=", D, "); got ", k.sizes(), ", ", v.sizes());
  TORCH_CHECK_VALUE(v.device() == k.device(), "k, v must be on one device, got ", k.device(), " and ", v.device());
  const int64_t T = k.size(0), B = lens.dim() == 1 ? lens.size(0) : 0;
  TORCH_CHECK_VALUE(cos.has_value() == sin.has_value() && (cos.has_value() || (!positions.has_value() && !sections.has_value())),
                    "a rotation needs cos and sin");
  Turn t;
  if (cos.has_value()) t = check_turn(k, *cos, *sin, positions, sections, T, -1);
  if (k_weight.has_value()) check_weight("k_weight", *k_weight, k);
  check_batch(kp, table, lens, offsets, T, k.device());
  if (T == 0 || B == 0) return;
  fa_append_args a{};
  const Tensor kr = rows(k, a.k_stride), vr = rows(v, a.v_stride);
  const Tensor w = k_weight.has_value() ? aligned(*k_weight) : Tensor();
  a.k = kr.const_data_ptr();
  a.v = vr.const_data_ptr();
  a.k_pages = kp.data_ptr();
  a.v_pages = vp.data_ptr();
  a.k_scales = ks.data_ptr<float>();
  a.v_scales = vs.data_ptr<float>();
  a.block_table = table.const_data_ptr<int>();
  a.seq_lens = lens.const_data_ptr<int>();
  a.offsets = offsets.has_value() ? offsets->const_data_ptr<int>() : nullptr;
  if (cos.has_value()) {
    a.cos = t.cos.const_data_ptr<float>();
    a.sin = t.sin.const_data_ptr<float>();
    a.pos = ptr(t.pos);
    a.pos_axis_stride = t.pos_stride[0];
    a.max_pos = static_cast<int>(t.cos.size(0));
    a.pos_is_int64 = t.pos.defined() && t.pos.scalar_type() == at::kLong;
  }
  a.k_weight = ptr(w);
  a.table_stride = table.stride(0);
  a.eps = eps;
  a.T = static_cast<int>(T);
  a.B = static_cast<int>(B);
  a.width = static_cast<int>(table.size(1));
  a.num_pages = static_cast<int>(kp.size(0));
  a.H_kv = static_cast<int>(H_kv);
  a.page_size = static_cast<int>(kp.size(2));
  a.D = static_cast<int>(D);
  a.dtype = type_code(k);
  a.weight_dtype = w.defined() ? type_code(w) : a.dtype;
  a.axes = t.axes;
  for (int i = 0; i < 4; ++i) a.section_start[i] = t.start[i];
  a.interleaved = interleaved;
  call(fa_append_kv, a, k, "append_kv");
  for (const Tensor* x : {&kp, &vp, &ks, &vs}) written(*x);
}

py::object paged_attention(const Tensor& q, const Tensor& kp, const Tensor& vp, const Tensor& ks, const Tensor& vs,
                           const Tensor& table, const Tensor& lens, const OptTensor& offsets, std::optional<double> scale_opt,
                           const OptTensor& out_opt, bool return_lse) {
  check_no_tangent("paged_attention", {q, kp, vp, ks, vs, out_opt});
  TORCH_CHECK_TYPE(half_type(q), "q must be float16 or bfloat16, got ", q.scalar_type());
  TORCH_CHECK(!at::GradMode::is_enabled() || !q.requires_grad(), "paged_attention has no backward: call it under torch.no_grad()");
  TORCH_CHECK(!at::GradMode::is_enabled() || !out_opt.has_value() || !out_opt->requires_grad(),
              "paged_attention writes into out, which must not require a gradient");
  check_cache(kp, vp, ks, vs);
  const int64_t H_kv = kp.size(1), D = kp.size(3);
  TORCH_CHECK_VALUE(q.dim() == 3 && q.size(2) == D && q.size(1) >= 1 && q.size(1) % H_kv == 0, "q must be (T, H, D=", D,
                    ") with H a multiple of H_kv=", H_kv, "; got ", q.sizes());
  const int64_t T = q.size(0), H = q.size(1), B = lens.dim() == 1 ? lens.size(0) : 0;
  const double scale = scale_opt.value_or(1.0 / std::sqrt(static_cast<double>(D)));
  // as float32, and times log2(e) in float32: what the kernel multiplies with
  TORCH_CHECK_VALUE(static_cast<float>(scale) > 0.f && std::isfinite(static_cast<float>(scale) * 1.4426950408889634f),
                    "scale must be positive and finite (below 2^127), got ", scale);
  TORCH_CHECK_VALUE(!out_opt.has_value() || (out_opt->sizes() == q.sizes() && out_opt->scalar_type() == q.scalar_type() && out_opt->device() == q.device()),
                    "out must be like q, ", q.sizes(), " ", q.scalar_type(), "; got ", out_opt->sizes(), " ", out_opt->scalar_type());
  // rows of o are written while others' q is read: o in q's place is fine, o beside it is not
  TORCH_CHECK_VALUE(!out_opt.has_value() || at::get_overlap_status(*out_opt, q) != at::MemOverlapStatus::Partial,
                    "out may be q itself but must not overlap it in part");
  check_batch(kp, table, lens, offsets, T, q.device());
  TORCH_CHECK_VALUE(T * H <= (1 << 30), "T * H must stay below 2^30, got ", q.sizes());
  Tensor out;
  if (out_opt.has_value())
    out = *out_opt;
  else
    out = B == 0 ? at::zeros(q.sizes(), q.options()) : at::empty(q.sizes(), q.options());
  Tensor lse;  // with the caller's out, rows that no sequence has are not written
  if (return_lse)
    lse = B == 0 || out_opt.has_value() ? at::full({T, H}, -std::numeric_limits<double>::infinity(), q.options().dtype(at::kFloat))
                                        : at::empty({T, H}, q.options().dtype(at::kFloat));
  if (T > 0 && B > 0) {
    fa_paged_args a{};
    const Tensor qr = rows(q, a.q_stride);
    TORCH_CHECK_VALUE(row_strides(out, a.out_stride) && (T == 1 || a.out_stride[0] != 0) && (H == 1 || a.out_stride[1] != 0),
                      "out must be contiguous in D, with its base and strides on 16-byte boundaries, and not expanded");
    const Tensor workspace = at::empty({FA_PAGED_WORKSPACE_BYTES(D)}, q.options().dtype(at::kByte));
    a.q = qr.const_data_ptr();
    a.k_pages = kp.const_data_ptr();
    a.v_pages = vp.const_data_ptr();
    a.k_scales = ks.const_data_ptr<float>();
    a.v_scales = vs.const_data_ptr<float>();
    a.block_table = table.const_data_ptr<int>();
    a.seq_lens = lens.const_data_ptr<int>();
    a.offsets = offsets.has_value() ? offsets->const_data_ptr<int>() : nullptr;
    a.out = out.data_ptr();
    a.lse = return_lse ? lse.data_ptr<float>() : nullptr;
    a.workspace = workspace.data_ptr();
    a.table_stride = table.stride(0);
    a.T = static_cast<int>(T);
    a.B = static_cast<int>(B);
    a.width = static_cast<int>(table.size(1));
    a.num_pages = static_cast<int>(kp.size(0));
    a.H = static_cast<int>(H);
    a.H_kv = static_cast<int>(H_kv);
    a.page_size = static_cast<int>(kp.size(2));
    a.D = static_cast<int>(D);
    a.dtype = type_code(q);
    a.clear_unowned = !out_opt.has_value();
    a.scale = static_cast<float>(scale);
    call(fa_paged_attention, a, q, "paged_attention");
    if (out_opt.has_value()) written(out);
  }
  if (return_lse) return py::make_tuple(out, lse);
  return py::cast(out);
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
  m.def("set_status_provider", [](py::object f) {
    delete g_status_provider;
    g_status_provider = new py::object(std::move(f));
  });
  m.def("qk_norm_rope", &qk_norm_rope);
  m.def("check_cache", &check_cache);
  m.def("append_kv", &append_kv);
  m.def("paged_attention", &paged_attention);
}
