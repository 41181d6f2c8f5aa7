"""Attention over a paged e4m3 cache (attention.paged.cache) on B200 (sm_100a): one new token per sequence
(decoding) or several (speculation, prompts in chunks behind what is cached), MHA, GQA and MQA.

    o = softmax(scale * q k^T) v     with k, v = the cached values times their page's scale

Token i of a sequence's n new tokens sees the keys j <= seq_len - n + i: the cache holds the new tokens'
keys already (append_kv comes first).  The reference project has no counterpart.
"""
import math

import torch

if __package__:
    from .cache import _native, _rope, check_batch, check_cuda
else:  # imported by path
    import importlib.util
    import os
    import sys
    _name = "_fa_b200_paged_cache"
    _mod = sys.modules.get(_name)
    if _mod is None:
        _spec = importlib.util.spec_from_file_location(
            _name, os.path.join(os.path.dirname(os.path.abspath(__file__)), "cache.py"))
        _mod = importlib.util.module_from_spec(_spec)
        sys.modules[_name] = _mod
        _spec.loader.exec_module(_mod)
    _native, _rope, check_batch, check_cuda = _mod._native, _mod._rope, _mod.check_batch, _mod.check_cuda


def paged_attention(q, cache, block_table, seq_lens, offsets=None, scale=None, out=None, return_lse=False):
    """o [T, H, D] for the query tokens q [T, H, D] (float16 / bfloat16, any strides with a contiguous last
    dimension); H is a multiple of the cache's K/V heads, query head h reads K/V head h // (H // H_kv).

    block_table, seq_lens, offsets: as for append_kv; seq_lens counts the new tokens
    scale:       factor of q k^T, 1 / sqrt(D) unless given
    out:         where to write o; its rows behind offsets[B] are left as they are (without it they are 0)
    return_lse:  also return lse, float32 [T, H]: log2 of the sum of 2^(log2(e) scale q k) over the keys
    A token that sees no key gives o = 0 and lse = -inf.
    """
    if q.dtype not in (torch.float16, torch.bfloat16):
        raise TypeError(f"q must be float16 or bfloat16, got {q.dtype}")
    if torch.is_grad_enabled() and q.requires_grad:
        raise RuntimeError("paged_attention has no backward: call it under torch.no_grad()")
    H_kv, D = cache.num_kv_heads, cache.head_dim
    if q.dim() != 3 or q.shape[2] != D or q.shape[1] < 1 or q.shape[1] % H_kv:
        raise ValueError(f"q must be (T, H, D={D}) with H a multiple of H_kv={H_kv}; got {tuple(q.shape)}")
    T, H, _ = q.shape
    device = q.device
    B = check_batch(cache, block_table, seq_lens, offsets, T, device)
    scale = 1.0 / math.sqrt(D) if scale is None else float(scale)
    if not 0.0 < scale < math.inf:
        raise ValueError(f"scale must be positive and finite, got {scale}")
    if out is not None and (out.shape != q.shape or out.dtype != q.dtype or out.device != device):
        raise ValueError(f"out must be like q, {tuple(q.shape)} {q.dtype} on {device}; got {tuple(out.shape)} {out.dtype}")
    check_cuda(device)
    if out is None:
        make = torch.empty if offsets is None else torch.zeros
        out = make((T, H, D), device=device, dtype=q.dtype)
    lse = torch.full((T, H), -math.inf, device=device) if return_lse else None
    if T > 0 and B > 0:
        nat = _native()
        q, q_stride = nat.rows16(q)
        to, out_stride = nat.rows16(out)
        if to is not out:
            raise ValueError("out must be contiguous in D with its base and strides on 16-byte boundaries")
        workspace = torch.empty(nat.paged_workspace_bytes(D), dtype=torch.uint8, device=device)
        nat.paged_attention(q, nat.PAGED_ARGS.pack(
            q.data_ptr(), cache.k_pages.data_ptr(), cache.v_pages.data_ptr(), cache.k_scales.data_ptr(),
            cache.v_scales.data_ptr(), block_table.data_ptr(), seq_lens.data_ptr(), _rope._ptr(offsets), out.data_ptr(),
            _rope._ptr(lse), workspace.data_ptr(), *q_stride, *out_stride, block_table.stride(0),
            T, B, block_table.shape[1], cache.num_pages, H, H_kv, cache.page_size, D, nat._dtype_code(q), scale))
    return (out, lse) if return_lse else out
