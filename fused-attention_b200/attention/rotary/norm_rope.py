"""Per-head RMS norm of queries and keys with the rotary position rotation in the same pass, forward and
backward, on B200 (sm_100a): what a model does with q and k before fused_attention_autograd,
fused_gqa_attention or a paged cache.

    y = x * w / sqrt(mean(x^2) + eps)                (the identity where no weight is given)
    z = (a cos - b sin, a sin + b cos)               for each pair (a, b) of y

A pair is (i, i + D/2), or (2i, 2i + 1) with interleaved=True.  cos and sin are tables
[max_pos, D/2] in float32 (rope_tables makes them); the row is the token's position.  With `sections`
a token has a position on each of several axes (time, height, width): the first sections[0] pairs
turn by the first axis' position, the next sections[1] by the second's, and so on.

The kernel reads q and k as views of a fused projection ([B, N, H, D] in memory, transposed) and writes
contiguous [B, H, N, D], the attention kernels' layout: no copy in between.  The reference project has no
counterpart.
"""
import importlib.util
import os
import sys

import torch
from torch.autograd.function import once_differentiable

MAX_AXES = 4


def _native():
    """The ctypes binding (attention/_lib.py), loaded by path under one shared module name."""
    mod = sys.modules.get("_fa_b200_native")
    if mod is None:
        path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "_lib.py")
        spec = importlib.util.spec_from_file_location("_fa_b200_native", path)
        mod = importlib.util.module_from_spec(spec)
        sys.modules["_fa_b200_native"] = mod
        spec.loader.exec_module(mod)
    return mod


def rope_tables(max_pos, head_dim, base=10000.0, device=None):
    """(cos, sin), float32 [max_pos, head_dim / 2]: the angle of pair i at position p is
    p * base^(-2i / head_dim), computed in float64 and rounded once."""
    half = head_dim // 2
    inv = float(base) ** (-torch.arange(half, dtype=torch.float64, device=device) / half)
    angle = torch.arange(max_pos, dtype=torch.float64, device=device)[:, None] * inv
    return angle.cos().float(), angle.sin().float()


def check_tables(cos, sin, D, device):
    """Raise unless cos and sin are float32 [max_pos, D/2] tables on `device`; return them contiguous."""
    if cos.dtype != torch.float32 or sin.dtype != torch.float32:
        raise TypeError(f"cos and sin must be float32, got {cos.dtype} and {sin.dtype}")
    if cos.dim() != 2 or cos.shape != sin.shape or cos.shape[1] * 2 != D or cos.shape[0] < 1:
        raise ValueError(f"cos and sin must both be (max_pos, {D // 2}); got {tuple(cos.shape)}, {tuple(sin.shape)}")
    if cos.device != device or sin.device != device:
        raise ValueError(f"cos and sin must be on {device}, got {cos.device} and {sin.device}")
    nat = _native()
    return nat.aligned16(cos), nat.aligned16(sin)


def check_sections(sections, D):
    """The first pair of each axis (MAX_AXES entries) and the number of axes."""
    if sections is None:
        return (0, 0, 0, 0), 1
    sections = tuple(int(s) for s in sections)
    if not 1 <= len(sections) <= MAX_AXES or min(sections) < 0 or sum(sections) != D // 2:
        raise ValueError(f"sections must be 1 to {MAX_AXES} pair counts that add up to D/2={D // 2}, got {sections}")
    start = [0]
    for s in sections[:-1]:
        start.append(start[-1] + s)
    return tuple(start + [0] * (MAX_AXES - len(start))), len(sections)


def check_positions(positions, shape, device):
    """Raise unless positions is an int32 / int64 tensor on `device` of one of the given shapes; return it
    contiguous in its last dimension."""
    if positions.dtype not in (torch.int32, torch.int64):
        raise TypeError(f"positions must be int32 or int64, got {positions.dtype}")
    if tuple(positions.shape) not in shape:
        raise ValueError(f"positions must have shape {' or '.join(map(str, shape))}, got {tuple(positions.shape)}")
    if positions.device != device:
        raise ValueError(f"positions must be on {device}, got {positions.device}")
    if positions.stride(-1) != 1 and positions.shape[-1] > 1:
        positions = positions.contiguous()
    return positions


def check_weight(name, w, x):
    if w.dtype not in (torch.float32, x.dtype):
        raise TypeError(f"{name} must be float32 or {x.dtype}, got {w.dtype}")
    if tuple(w.shape) != (x.shape[-1],):
        raise ValueError(f"{name} must be ({x.shape[-1]},), got {tuple(w.shape)}")
    if w.device != x.device:
        raise ValueError(f"{name} must be on {x.device}, got {w.device}")
    return _native().aligned16(w)


def _check(q, k, cos, sin, positions, q_weight, k_weight, sections):
    """Arguments as the kernels take them; raises TypeError / ValueError for those they do not."""
    if q.dtype not in (torch.float16, torch.bfloat16) or (k is not None and k.dtype != q.dtype):
        raise TypeError("q, k must be float16 (or both bfloat16)")
    if q.dim() != 4 or (k is not None and (k.dim() != 4 or k.shape[1] < 1 or k.shape[0] != q.shape[0]
                                           or k.shape[2:] != q.shape[2:])):
        raise ValueError(f"q, k must be (B, H, N, D) and (B, H_kv, N, D); got {tuple(q.shape)}"
                         + ("" if k is None else f", {tuple(k.shape)}"))
    B, H, N, D = q.shape
    if D not in (32, 64, 128):
        raise ValueError(f"head dim D={D} not supported; allowed (32, 64, 128)")
    cos, sin = check_tables(cos, sin, D, q.device)
    start, axes = check_sections(sections, D)
    pos_stride = (0, 0)
    if positions is not None:
        lead = () if sections is None else (axes,)
        positions = check_positions(positions, (lead + (N,), lead + (B, N)), q.device)
        st = positions.stride()
        pos_stride = (st[0] if lead else 0, st[-2] if positions.dim() == len(lead) + 2 else 0)
    elif sections is not None:
        raise ValueError("sections need positions of shape (axes, N) or (axes, B, N)")
    if k is None and k_weight is not None:
        raise ValueError("k_weight is given without k")
    weights = []
    for name, w, x in (("q_weight", q_weight, q), ("k_weight", k_weight, k)):
        weights.append(None if w is None else check_weight(name, w, x))
    if q_weight is not None and k_weight is not None and q_weight.dtype != k_weight.dtype:
        raise TypeError(f"q_weight and k_weight must share one dtype, got {q_weight.dtype} and {k_weight.dtype}")
    if not q.is_cuda or (k is not None and k.device != q.device):
        raise ValueError(f"q, k must be on one CUDA device, got {q.device}" + ("" if k is None else f", {k.device}"))
    return cos, sin, positions, weights[0], weights[1], pos_stride, start, axes


def _ptr(t):
    return 0 if t is None else t.data_ptr()


_NO_STRIDE = (0, 0, 0)


def _pack(nat, q, k, q_stride, k_stride, checked, eps, interleaved, outs=(0,) * 9, dq_stride=_NO_STRIDE,
          dk_stride=_NO_STRIDE):
    """fa_norm_rope_args; `outs`: the nine pointers from q_out to workspace."""
    cos, sin, positions, qw, kw, pos_stride, start, axes = checked
    B, H, N, D = q.shape
    weight = kw if qw is None else qw
    code = nat._dtype_code(q)
    weight_code = nat.F32_CODE if weight is not None and weight.dtype == torch.float32 else code
    return nat.NORM_ROPE_ARGS.pack(
        q.data_ptr(), _ptr(k), _ptr(qw), _ptr(kw), cos.data_ptr(), sin.data_ptr(), _ptr(positions), *outs,
        *q_stride, *k_stride, *dq_stride, *dk_stride, *pos_stride,
        B, H, 0 if k is None else k.shape[1], N, D, code, weight_code, cos.shape[0], axes, *start,
        positions is not None and positions.dtype == torch.int64, interleaved, eps)


def _forward(q, k, checked, eps, interleaved):
    B, H, N, D = q.shape
    q_out = torch.empty((B, H, N, D), device=q.device, dtype=q.dtype)
    k_out = None if k is None else torch.empty(k.shape, device=k.device, dtype=k.dtype)
    if q.numel() == 0:
        return q_out, k_out
    nat = _native()
    q, q_stride = nat.rows16(q)
    k_stride = _NO_STRIDE
    if k is not None:
        k, k_stride = nat.rows16(k)
    nat.norm_rope_fwd(q, _pack(nat, q, k, q_stride, k_stride, checked, eps, interleaved,
                               (q_out.data_ptr(), _ptr(k_out), 0, 0, 0, 0, 0, 0, 0)))
    return q_out, k_out


def _empty_like_rows(x):
    """An uninitialised gradient of x: token-major memory where x is token-major, else head-major."""
    B, H, N, D = x.shape
    if x.stride(1) < x.stride(2):
        return torch.empty((B, N, H, D), device=x.device, dtype=x.dtype).transpose(1, 2)
    return torch.empty((B, H, N, D), device=x.device, dtype=x.dtype)


def _backward(q, k, checked, eps, interleaved, dq_out, dk_out, want_qw, want_kw):
    """(dq, dk, dq_weight, dk_weight); the weights' gradients where wanted, else None."""
    qw, kw = checked[3], checked[4]
    if q.numel() == 0:
        return (torch.zeros_like(q), None if k is None else torch.zeros_like(k),
                torch.zeros_like(qw) if want_qw else None, torch.zeros_like(kw) if want_kw else None)
    nat = _native()
    dq = _empty_like_rows(q)
    dk = None if k is None else _empty_like_rows(k)
    dqw = torch.empty_like(qw) if want_qw else None
    dkw = torch.empty_like(kw) if want_kw else None
    workspace = None
    if qw is not None or kw is not None:
        workspace = torch.empty((nat.ROPE_WORKSPACE_ROWS, q.shape[-1]), device=q.device, dtype=torch.float32)
    q, q_stride = nat.rows16(q)
    dq_out = nat.aligned16(dq_out)
    dq_stride = nat.rows16(dq)[1]
    k_stride = dk_stride = _NO_STRIDE
    if k is not None:
        k, k_stride = nat.rows16(k)
        dk_out = nat.aligned16(dk_out)
        dk_stride = nat.rows16(dk)[1]
    nat.norm_rope_bwd(q, _pack(nat, q, k, q_stride, k_stride, checked, eps, interleaved,
                               (0, 0, dq_out.data_ptr(), _ptr(dk_out) if k is not None else 0, dq.data_ptr(),
                                _ptr(dk), _ptr(dqw), _ptr(dkw), _ptr(workspace)), dq_stride, dk_stride))
    return dq, dk, dqw, dkw


class QKNormRopeFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, q_weight, k_weight, checked, eps, interleaved):
        ctx.save_for_backward(q, k, *checked[:5])
        ctx.rest = (checked[5:], eps, interleaved)
        return _forward(q, k, checked, eps, interleaved)

    @staticmethod
    @once_differentiable
    def backward(ctx, dq_out, dk_out=None):
        q, k, *tensors = ctx.saved_tensors
        rest, eps, interleaved = ctx.rest
        need = ctx.needs_input_grad
        dq, dk, dqw, dkw = _backward(q, k, (*tensors, *rest), eps, interleaved, dq_out, dk_out, need[2], need[3])
        return dq, dk, dqw, dkw, None, None, None


def qk_norm_rope(q, k, cos, sin, positions=None, q_weight=None, k_weight=None, eps=1e-6, interleaved=False,
                 sections=None):
    """(q_out, k_out): every row of q [B, H, N, D] and k [B, H_kv, N, D] (float16 / bfloat16, any strides
    with a contiguous last dimension; k may be None) normed and rotated, contiguous [B, H, N, D].

    q_weight, k_weight: [D], float32 or the dtype of q; None leaves that tensor's norm out.
    cos, sin:           float32 [max_pos, D/2]
    positions:          int32 / int64 [N] or [B, N], None: 0 .. N-1; with sections a leading dimension
                        of one row per axis
    Differentiable in q, k and the weights.  A position outside the tables is reported by check_status
    of the binding (attention/_lib.py).
    """
    checked = _check(q, k, cos, sin, positions, q_weight, k_weight, sections)
    if torch.is_grad_enabled() and (q.requires_grad or (k is not None and k.requires_grad)
                                    or (q_weight is not None and q_weight.requires_grad)
                                    or (k_weight is not None and k_weight.requires_grad)):
        return QKNormRopeFn.apply(q, k, q_weight, k_weight, checked, eps, interleaved)
    return _forward(q, k, checked, eps, interleaved)
