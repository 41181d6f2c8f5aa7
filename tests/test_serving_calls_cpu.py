"""Calls around attention that are refused, or no longer refused, without a GPU: beside test_serving_cpu.py."""
import pytest
import torch

from attention.paged.cache import PagedKVCache
from attention.paged.paged_attention import paged_attention
from tests.test_serving_cpu import PA, PAGED_ARGS, _packed, _rc, cache_tensors, half, step_args


def test_scales_may_start_anywhere():
    """Scales are read one by one: one layer's part of all layers' scales starts at any multiple of 4 bytes."""
    kp, vp, _, _ = cache_tensors(pages=3, H_kv=1)
    scales = torch.zeros(2, 5, 3, 1)
    for layer in range(5):
        PagedKVCache(kp, vp, scales[0, layer], scales[1, layer])


def test_pages_start_on_16_bytes():
    kp, vp, ks, vs = cache_tensors()
    odd = torch.zeros(kp.numel() + 8, dtype=torch.uint8)[8:].view(kp.dtype).view(kp.shape)
    for t in ((odd, vp, ks, vs), (kp, odd, ks, vs)):
        with pytest.raises(ValueError, match="16-byte"):
            PagedKVCache(*t)


def test_scales_of_scores_that_overflow_are_refused():
    """The kernels multiply with scale log2(e): above 2^127.47 that is infinite, and every row NaN."""
    with pytest.raises(ValueError, match="scale must be positive and finite"):
        paged_attention(**step_args(q=half(3, 4, 64), scale=3e38))
    assert _rc("fa_paged_attention", _packed(PAGED_ARGS, PA, scale=3e38)) == 1


def test_out_that_overlaps_part_of_q_is_refused():
    """Some blocks would read queries that others have overwritten with their rows."""
    both = half(5, 4, 64)
    with pytest.raises(ValueError, match="overlap it in part"):
        paged_attention(**step_args(q=both[:3], out=both[1:4]))
    for q, out in ((both[:3], both[:3]), (half(3, 8, 64)[:, :4], half(3, 8, 64)[:, 4:])):
        with pytest.raises(ValueError, match="CUDA device"):  # as far as a machine without one goes
            paged_attention(**step_args(q=q, out=out))
