"""Calls of append_kv and paged_attention that the documentation allows or rules out, beside those of test_paged_gpu.py."""
import pytest
import torch

from tests.serving_util import angles, append64, tables
from tests.test_paged_gpu import _append, _attend, _cache, _nat, batch, i32, make_cache, same_bytes, to_gpu

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("length", [-1, -(1 << 31) + 1, -(1 << 31)])
def test_negative_lengths_are_reported(length, cuda_device):
    """Also where the place of a token, its sequence's length less the tokens behind it, leaves 32 bits."""
    nat = _nat()
    P, H_kv, D = 16, 2, 64
    for news in ([1, 1, 1], [2, 1, 3]):
        table, starts, pages = batch([40, 20, 9], news, P)
        cache = make_cache(pages, H_kv, P, D)
        x = torch.randn(starts[-1], 4, D, device="cuda").half()
        for offsets in (i32(starts), None):
            if offsets is None and starts[-1] != 3:
                continue
            for b in range(3):
                lens = [40, 20, 9]
                lens[b] = length
                got = to_gpu(*cache)
                _append(_cache(*got), x[:, :H_kv], x[:, :H_kv], table.cuda(), i32(lens), offsets)
                with pytest.raises(nat.KernelError, match="outside its table"):
                    nat.check_status(cuda_device)
                own = [int(p) for p in table[b] if p < pages]  # nothing of that sequence is written
                assert all(same_bytes(t[own], r[own]) for t, r in zip(got, cache) if t.element_size() == 1)
                _attend(x, _cache(*got), table.cuda(), i32(lens), offsets)
                with pytest.raises(nat.KernelError, match="outside its table"):
                    nat.check_status(cuda_device)


def test_writes_are_seen_by_autograd(cuda_device):
    """The version of every tensor that a call writes moves, and of no other: a backward pass that saved `out` before
    raises instead of reading what was written over it."""
    P, H, H_kv, D = 16, 4, 2, 64
    table, starts, pages = batch([40, 20], [1, 1], P)
    tensors = to_gpu(*make_cache(pages, H_kv, P, D))
    cache, tg, lens = _cache(*tensors), table.cuda(), i32([40, 20])
    q, kv = torch.randn(2, H, D, device="cuda").half(), torch.randn(2, H_kv, D, device="cuda").half()

    def moved(call):
        watched = [*tensors, q, kv, tg, lens]
        before = [t._version for t in watched]
        call()
        return [t._version > v for t, v in zip(watched, before)]

    assert moved(lambda: _append(cache, kv, kv, tg, lens)) == [True] * 4 + [False] * 4
    assert moved(lambda: _attend(q, cache, tg, lens)) == [False] * 8
    assert moved(lambda: _attend(q, cache, tg, lens, out=q)) == [False] * 4 + [True] + [False] * 3
    x = torch.randn(2, H, D, device="cuda").half().requires_grad_(True)
    out = torch.ones(2, H, D, device="cuda").half()
    y = x * out
    _attend(q, cache, tg, lens, out=out)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()
    with torch.inference_mode():
        mine = torch.empty(2, H, D, device="cuda").half()
    _attend(q, cache, tg, lens, out=mine)  # tensors of inference mode have no version
    assert torch.equal(mine, out)
    _nat().check_status(cuda_device)


@pytest.mark.parametrize("eps", [1e-6, 0.0])
@pytest.mark.parametrize("rotated", [False, True], ids=["normed", "normed-rotated"])
@pytest.mark.parametrize("wtype", [torch.bfloat16, torch.float32], ids=["w16", "w32"])
def test_appended_rows_of_all_sizes_are_normed_exactly(eps, rotated, wtype, cuda_device):
    """bf16 key rows from 2^-120 to the type's largest number: the bytes are those of float64."""
    P, H_kv, D = 32, 2, 64
    lens = news = [100]
    table, starts, pages = batch(lens, news, P)
    g = torch.Generator().manual_seed(3)
    powers = torch.tensor([0, 40, 62, 90, 110, 122] + ([-20, -60, -90, -120] if eps == 0 else []))
    power = powers[torch.randint(0, len(powers), (100, H_kv, 1), generator=g)]
    k = (torch.randn(100, H_kv, D, generator=g, dtype=torch.float64) * torch.exp2(power.double())).bfloat16()
    k[7] = torch.finfo(torch.bfloat16).max
    v = torch.randn(100, H_kv, D, generator=g).bfloat16()
    w = (1 + 0.5 * torch.randn(D, generator=g)).to(wtype)
    cos, sin = tables(100, D, "cpu")
    c, s = angles(cos, sin, torch.arange(100), None) if rotated else (None, None)
    cache = make_cache(pages, H_kv, P, D)
    ref = append64(*cache, k, v, table, lens, starts, c, s, w, eps, False)
    got = to_gpu(*cache)
    kw = dict(cos=cos.cuda(), sin=sin.cuda()) if rotated else {}
    _append(_cache(*got), k.cuda(), v.cuda(), table.cuda(), i32(lens), i32(starts), k_weight=w.cuda(), eps=eps, **kw)
    _nat().check_status(cuda_device)
    for name, a, b in zip(("k_pages", "v_pages", "k_scales", "v_scales"), got, ref):
        assert same_bytes(a, b), (name, int((a.cpu().view(torch.uint8) != b.view(torch.uint8)).sum()))


def test_scales_of_a_layer_in_a_larger_tensor(cuda_device):
    """One layer's scales of all layers', which start at any multiple of 4 bytes."""
    P, H, H_kv, D = 16, 6, 3, 64
    lens, news = [70, 33, 20], [3, 2, 20]
    table, starts, pages = batch(lens, news, P, extra_pages=0 if (sum(-(-L // P) for L in lens)) % 2 else 1)
    assert pages * H_kv % 2 == 1
    kp, vp, ks, vs = make_cache(pages, H_kv, P, D)
    x = torch.randn(starts[-1], H, D, device="cuda").half()
    results = []
    for layer in range(3):
        scales = torch.full((2, 4, pages, H_kv), 7.0, device="cuda")
        scales[0, layer], scales[1, layer] = ks.cuda(), vs.cuda()
        before = scales.clone()
        pages_of = to_gpu(kp, vp)
        cache = _cache(*pages_of, scales[0, layer], scales[1, layer])
        _append(cache, x[:, :H_kv], x[:, H_kv:], table.cuda(), i32(lens), i32(starts))
        results.append((*(t.view(torch.uint8) for t in pages_of), scales[0, layer].clone(), scales[1, layer].clone(),
                        _attend(x, cache, table.cuda(), i32(lens), i32(starts))))
        for other in range(4):
            assert other == layer or torch.equal(scales[:, other], before[:, other])
    _nat().check_status(cuda_device)
    assert all(torch.equal(a, b) for r in results[1:] for a, b in zip(r, results[0]))
