"""Attention over a paged e4m3 cache (attention.paged.cache) on B200 (sm_100a): one new token per sequence
(decoding) or several (speculation, prompts in chunks behind what is cached), MHA, GQA and MQA.

    o = softmax(scale * q k^T) v     with k, v = the cached values times their page's scale

Token i of a sequence's n new tokens sees the keys j <= seq_len - n + i: the cache holds the new tokens'
keys already (append_kv comes first).  The reference project has no counterpart.
"""
import importlib.util
import os
import sys

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


def paged_attention(q, cache, block_table, seq_lens, offsets=None, scale=None, out=None, return_lse=False):
    """o [T, H, D] for the query tokens q [T, H, D] (float16 / bfloat16, any strides with a contiguous last
    dimension); H is a multiple of the cache's K/V heads, query head h reads K/V head h // (H // H_kv).

    block_table, seq_lens, offsets: as for append_kv; seq_lens counts the new tokens
    scale:       factor of q k^T, 1 / sqrt(D) unless given
    out:         where to write o (q itself is allowed, a part of its memory is not); its rows behind offsets[B] are left as
                 they are (without it they are 0)
    return_lse:  also return lse, float32 [T, H]: log2 of the sum of 2^(log2(e) scale q k) over the keys
    A token that sees no key gives o = 0 and lse = -inf.
    The cache's scales are finite and not negative, of any size.  A NaN in a cached key or value reaches the tokens that
    see it, no others.  Scores, their sums and o's are float32; a weight is rounded to float16 (2^-11 of it), relative
    to the token's own largest.
    A page, length or offset outside its table is reported by check_status of the binding (attention/_lib.py), like
    qk_norm_rope's positions.
    """
    global _ops
    if _ops is None:
        _ops = _native().load_ops()
    return _ops.paged_attention(q, cache.k_pages, cache.v_pages, cache.k_scales, cache.v_scales, block_table, seq_lens,
                                offsets, scale, out, return_lse)
