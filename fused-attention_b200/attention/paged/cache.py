"""A paged key/value cache in 8 bits and the appending of new tokens to it, on B200 (sm_100a).

Pages are e4m3, [num_pages, H_kv, page_size, D], with one float32 scale for each (page, K/V head): a stored
value c stands for c * scale.  Token j of sequence b lies in page block_table[b, j // page_size].  One step of
serving appends each sequence's new keys and values (append_kv, which norms and rotates the keys on
the way) and then attends to the cache (attention.paged.paged_attention).

The reference project has no counterpart.
"""
import importlib.util
import os
import sys

import torch

if __package__:
    from ..rotary import norm_rope as _rope
else:  # imported by path
    _name = "_fa_b200_norm_rope"
    _rope = sys.modules.get(_name)
    if _rope is None:
        _spec = importlib.util.spec_from_file_location(
            _name, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "rotary", "norm_rope.py"))
        _rope = importlib.util.module_from_spec(_spec)
        sys.modules[_name] = _rope
        _spec.loader.exec_module(_rope)

PAGE_SIZES = (16, 32, 64, 128)
HEAD_DIMS = (32, 64, 128)
PAGE_DTYPE = torch.float8_e4m3fn
_native = _rope._native


class PagedKVCache:
    """The cache's four tensors: k_pages, v_pages (e4m3 [num_pages, H_kv, page_size, D]) and k_scales, v_scales
    (float32 [num_pages, H_kv]), all contiguous on one CUDA device."""

    __slots__ = ("k_pages", "v_pages", "k_scales", "v_scales")

    def __init__(self, k_pages, v_pages, k_scales, v_scales):
        if k_pages.dtype != PAGE_DTYPE or v_pages.dtype != PAGE_DTYPE:
            raise TypeError(f"k_pages and v_pages must be {PAGE_DTYPE}, got {k_pages.dtype} and {v_pages.dtype}")
        if k_scales.dtype != torch.float32 or v_scales.dtype != torch.float32:
            raise TypeError(f"k_scales and v_scales must be float32, got {k_scales.dtype} and {v_scales.dtype}")
        shape = k_pages.shape
        if len(shape) != 4 or v_pages.shape != shape or k_scales.shape != shape[:2] or v_scales.shape != shape[:2]:
            raise ValueError("pages must be (num_pages, H_kv, page_size, D) and scales (num_pages, H_kv); got "
                             f"{tuple(shape)}, {tuple(v_pages.shape)}, {tuple(k_scales.shape)}, {tuple(v_scales.shape)}")
        if shape[2] not in PAGE_SIZES or shape[3] not in HEAD_DIMS or shape[0] < 1 or shape[1] < 1:
            raise ValueError(f"page_size must be one of {PAGE_SIZES} and D one of {HEAD_DIMS}, got {tuple(shape)}")
        device = k_pages.device
        for name, x in (("k_pages", k_pages), ("v_pages", v_pages), ("k_scales", k_scales), ("v_scales", v_scales)):
            if x.device != device or not x.is_contiguous():
                raise ValueError(f"{name} must be contiguous on {device}")
        self.k_pages, self.v_pages, self.k_scales, self.v_scales = k_pages, v_pages, k_scales, v_scales

    @classmethod
    def empty(cls, num_pages, num_kv_heads, head_dim, page_size=64, device="cuda"):
        """A cache of num_pages free pages."""
        pages = [torch.zeros((num_pages, num_kv_heads, page_size, head_dim), dtype=torch.uint8, device=device)
                 .view(PAGE_DTYPE) for _ in range(2)]
        scales = [torch.zeros((num_pages, num_kv_heads), device=device) for _ in range(2)]
        return cls(*pages, *scales)

    num_pages = property(lambda self: self.k_pages.shape[0])
    num_kv_heads = property(lambda self: self.k_pages.shape[1])
    page_size = property(lambda self: self.k_pages.shape[2])
    head_dim = property(lambda self: self.k_pages.shape[3])

    def gather(self, block_table_row, length):
        """(K, V) of one sequence, float32 [length, H_kv, D]: what its cached tokens stand for."""
        pages = block_table_row[: -(-length // self.page_size)].long()
        out = []
        for p, s in ((self.k_pages, self.k_scales), (self.v_pages, self.v_scales)):
            x = p.view(torch.uint8)[pages].view(PAGE_DTYPE).float() * s[pages][:, :, None, None]
            out.append(x.transpose(1, 2).reshape(-1, self.num_kv_heads, self.head_dim)[:length])
        return tuple(out)


def check_batch(cache, block_table, seq_lens, offsets, T, device):
    """Raise unless the batch's tables fit the cache and T query tokens."""
    for name, x in (("block_table", block_table), ("seq_lens", seq_lens), ("offsets", offsets)):
        if x is None:
            continue
        if x.dtype != torch.int32:
            raise TypeError(f"{name} must be int32, got {x.dtype}")
        if x.device != device:
            raise ValueError(f"{name} must be on {device}, got {x.device}")
        if x.dim() != (2 if x is block_table else 1) or (x.shape[-1] > 1 and x.stride(-1) != 1):
            raise ValueError(f"{name} must be {'(B, pages)' if x is block_table else 'one-dimensional'} and "
                             f"contiguous in its last dimension, got {tuple(x.shape)}")
    B = seq_lens.shape[0]
    if block_table.shape[0] != B or block_table.shape[1] < 1:
        raise ValueError(f"block_table must be (B={B}, pages), got {tuple(block_table.shape)}")
    if offsets is None:
        if T != B:
            raise ValueError(f"without offsets there is one token per sequence: got {T} tokens, {B} sequences")
    elif offsets.shape[0] != B + 1:
        raise ValueError(f"offsets must be (B + 1 = {B + 1},), got {tuple(offsets.shape)}")
    if cache.k_pages.device != device:
        raise ValueError(f"the tokens and the cache must be on one device, got {device} and {cache.k_pages.device}")
    return B


def check_cuda(device):
    if device.type != "cuda":
        raise ValueError(f"the tokens and the cache must be on a CUDA device, got {device}")


def append_kv(cache, k, v, block_table, seq_lens, offsets=None, cos=None, sin=None, positions=None, k_weight=None,
              eps=1e-6, interleaved=False, sections=None):
    """Write the new tokens' keys and values into their pages.

    k, v:         [T, H_kv, D] float16 / bfloat16 (any strides with a contiguous last dimension)
    block_table:  int32 [B, pages], the pages of each sequence
    seq_lens:     int32 [B], lengths with the new tokens
    offsets:      int32 [B + 1], sequence b's new tokens are k[offsets[b]:offsets[b + 1]], the last ones of
                  its seq_lens[b]; None: one token per sequence
    cos, sin:     float32 [max_pos, D/2]: keys are rotated by their position, which is their place in the
                  sequence unless positions (int32 / int64 [T], with sections [axes, T]) says otherwise
    k_weight:     [D]: keys are normed first (see attention.rotary.norm_rope)

    The tokens of one call that lie in one page are rounded together, to the smallest power-of-two scale
    that holds them; a page that holds older tokens keeps its scale unless the new ones need a larger
    one, and then the older ones are rounded again.  Infinities are stored as the largest magnitude, NaN
    as NaN; neither changes a scale.  Tokens behind offsets[B], and tokens that would lie before their
    sequence's start, are not written.  A page that is written must belong to one sequence of the batch.
    """
    if k.dtype not in (torch.float16, torch.bfloat16) or v.dtype != k.dtype:
        raise TypeError("k, v must be float16 (or both bfloat16)")
    if torch.is_grad_enabled() and (k.requires_grad or v.requires_grad or (k_weight is not None and k_weight.requires_grad)):
        raise RuntimeError("append_kv has no backward: call it under torch.no_grad()")
    H_kv, D = cache.num_kv_heads, cache.head_dim
    if k.dim() != 3 or v.shape != k.shape or k.shape[1:] != (H_kv, D):
        raise ValueError(f"k, v must be (T, H_kv={H_kv}, D={D}); got {tuple(k.shape)}, {tuple(v.shape)}")
    if v.device != k.device:
        raise ValueError(f"k, v must be on one device, got {k.device} and {v.device}")
    T = k.shape[0]
    B = check_batch(cache, block_table, seq_lens, offsets, T, k.device)
    if (cos is None) != (sin is None) or (cos is None and (positions is not None or sections is not None)):
        raise ValueError("a rotation needs cos and sin")
    start, axes, max_pos, pos_stride = (0, 0, 0, 0), 1, 0, 0
    if cos is not None:
        cos, sin = _rope.check_tables(cos, sin, D, k.device)
        start, axes = _rope.check_sections(sections, D)
        max_pos = cos.shape[0]
        if positions is not None:
            positions = _rope.check_positions(positions, ((T,) if sections is None else (axes, T),), k.device)
            pos_stride = positions.stride(0) if sections is not None else 0
        elif sections is not None:
            raise ValueError("sections need positions of shape (axes, T)")
    if k_weight is not None:
        k_weight = _rope.check_weight("k_weight", k_weight, k)
    check_cuda(k.device)
    if T == 0 or B == 0:
        return
    nat = _native()
    k, k_stride = nat.rows16(k)
    v, v_stride = nat.rows16(v)
    code = nat._dtype_code(k)
    ptr = _rope._ptr
    nat.append_kv(k, nat.APPEND_ARGS.pack(
        k.data_ptr(), v.data_ptr(), cache.k_pages.data_ptr(), cache.v_pages.data_ptr(), cache.k_scales.data_ptr(),
        cache.v_scales.data_ptr(), block_table.data_ptr(), seq_lens.data_ptr(), ptr(offsets), ptr(cos), ptr(sin),
        ptr(positions), ptr(k_weight), *k_stride, *v_stride, block_table.stride(0), pos_stride, eps,
        T, B, block_table.shape[1], cache.num_pages, H_kv, cache.page_size, D, code,
        nat.F32_CODE if k_weight is not None and k_weight.dtype == torch.float32 else code, max_pos, axes, *start,
        positions is not None and positions.dtype == torch.int64, interleaved, 0))
