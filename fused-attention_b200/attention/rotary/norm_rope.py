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


_ops = None


def qk_norm_rope(q, k, cos, sin, positions=None, q_weight=None, k_weight=None, eps=1e-6, interleaved=False,
                 sections=None):
    """(q_out, k_out): every row of q [B, H, N, D] and k [B, H_kv, N, D] (float16 / bfloat16, any strides
    with a contiguous last dimension; k may be None) normed and rotated, contiguous [B, H, N, D].

    q_weight, k_weight: [D], float32 or the dtype of q; None leaves that tensor's norm out.
    cos, sin:           float32 [max_pos, D/2]
    positions:          int32 / int64 [N] or [B, N], None: 0 .. N-1; with sections a leading dimension
                        of one row per axis
    Differentiable (once, in reverse mode) in q, k and the weights; dual tensors are refused.  A position outside the tables is reported by check_status
    of the binding (attention/_lib.py).
    """
    global _ops
    if _ops is None:
        _ops = _native().load_ops()
    return _ops.qk_norm_rope(q, k, cos, sin, positions, q_weight, k_weight, eps, interleaved, sections)
