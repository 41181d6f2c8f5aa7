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

PAGE_DTYPE = torch.float8_e4m3fn
_ops = None


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


def _load_ops():
    global _ops
    _ops = _native().load_ops()
    return _ops


class PagedKVCache:
    """The cache's four tensors: k_pages, v_pages (torch.float8_e4m3fn [num_pages, H_kv, page_size, D], page_size 16,
    32, 64 or 128, D 32, 64 or 128; they start on 16-byte boundaries) and k_scales, v_scales (float32
    [num_pages, H_kv]), all contiguous on one device; appending needs keys and values that share no memory.  The
    operators write into these tensors."""

    __slots__ = ("k_pages", "v_pages", "k_scales", "v_scales")

    def __init__(self, k_pages, v_pages, k_scales, v_scales):
        (_ops or _load_ops()).check_cache(k_pages, v_pages, k_scales, v_scales)
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


def append_kv(cache, k, v, block_table, seq_lens, offsets=None, cos=None, sin=None, positions=None, k_weight=None,
              eps=1e-6, interleaved=False, sections=None):
    """Write the new tokens' keys and values into their pages.

    k, v:         [T, H_kv, D] float16 / bfloat16 (any strides with a contiguous last dimension)
    block_table:  int32 [B, pages], the pages of each sequence
    seq_lens:     int32 [B], lengths with the new tokens
    offsets:      int32 [B + 1] from 0, sequence b's new tokens are k[offsets[b]:offsets[b + 1]], the last ones of
                  its seq_lens[b]; None: one token per sequence
    cos, sin:     float32 [max_pos, D/2]: keys are rotated by their position, which is their place in the
                  sequence unless positions (int32 / int64 [T], with sections [axes, T]) says otherwise
    k_weight:     [D]: keys are normed first (see attention.rotary.norm_rope)

    The tokens of one call that lie in one page are rounded together, to the smallest power-of-two scale
    that holds them; a page that holds older tokens keeps its scale unless the new ones need a larger
    one, and then the older ones are rounded again.  Infinities in v, and in k where it is neither normed nor
    rotated, are stored as the largest magnitude, NaN as NaN; neither changes a scale.  Tokens behind
    offsets[B], and tokens that would lie before their sequence's start, are not written.  A page that is written
    must belong to one sequence of the batch.  A position, page, length or offset outside its table (a negative
    length too) is reported by check_status of the binding (attention/_lib.py).
    """
    (_ops or _load_ops()).append_kv(cache.k_pages, cache.v_pages, cache.k_scales, cache.v_scales, k, v, block_table, seq_lens,
                                    offsets, cos, sin, positions, k_weight, eps, interleaved, sections)
