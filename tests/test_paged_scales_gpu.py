"""Page scales of all sizes and NaN keys in attention over the paged cache, in both kernels.

Bounds are those of the split kernel (tests/serving_util.py, paged64) for every key that a row sees; keys that it
does not see have no part in them.  The chunk kernel computes some exponentials as a polynomial, off by less than 2^-13,
in the weights and in their sum: 2^-12 beside the 2^-11 that the bound has for a weight's rounding to f16, and 2^-16 for
the logarithms of scales that are no powers of two (an ulp of at most 126, 2^-18, twice over).  So the
bound is taken 1.6 times there, and lse may be off by 2^-12 + 2^-14 more, in natural units."""
import math

import pytest
import torch

from tests.serving_util import half_step, half_subnormal, paged64
from tests.test_paged_gpu import _append, _attend, _cache, _nat, batch, i32, make_cache, takes_chunk_kernel, to_gpu

pytestmark = pytest.mark.gpu

SPLIT = dict(lens=[300, 131], news=[3, 2], P=32, H=8, H_kv=4, D=128)
CHUNK = dict(lens=[300, 450], news=[260, 200], P=32, H=32, H_kv=16, D=128)
CHUNK64 = dict(lens=[700, 333], news=[300, 333], P=64, H=32, H_kv=16, D=64)
CHUNK16 = dict(lens=[517, 260], news=[400, 260], P=16, H=40, H_kv=20, D=32)
SHAPES = [SPLIT, CHUNK, CHUNK64, CHUNK16]
ids = ["split", "chunk", "chunk-64", "chunk-16"]


def is_chunk(s):
    return takes_chunk_kernel(sum(s["news"]), len(s["lens"]), s["H"], s["H_kv"], s["D"])


def test_shapes_take_the_kernels_they_are_named_after():
    assert [is_chunk(s) for s in SHAPES] == [False, True, True, True]


def check(o, lse, q, cache, table, lens, starts, scale, chunk):
    ref, ref_lse, bound, lse_bound = paged64(q, *cache, table, lens, starts, scale)
    if chunk:
        bound, lse_bound = 1.6 * bound, lse_bound + math.log2(math.e) * (2.0 ** -12 + 2.0 ** -14)
    o, lse = o.double().cpu(), lse.double().cpu()
    assert bool(o.isfinite().all())
    tol = half_step(q.dtype) * (ref.abs() + bound) + bound + half_subnormal(q.dtype)
    worst = float(((o - ref).abs() / tol).max())
    assert worst <= 1.0, worst
    seen = ref_lse.isfinite()
    assert bool((lse[~seen] == -math.inf).all())
    assert bool(((lse - ref_lse).abs() <= lse_bound)[seen].all())


def run(s, cache, q, scale=None):
    table, starts, _ = batch(s["lens"], s["news"], s["P"])
    scale = scale or s["D"] ** -0.5
    o, lse = _attend(q.cuda(), _cache(*to_gpu(*cache)), table.cuda(), i32(s["lens"]), i32(starts), scale=scale, return_lse=True)
    _nat().check_status(torch.device("cuda", torch.cuda.current_device()))
    check(o, lse, q, cache, table, s["lens"], starts, scale, is_chunk(s))


def queries(s, dtype, seed=5):
    return torch.randn(sum(s["news"]), s["H"], s["D"], generator=torch.Generator().manual_seed(seed)).to(dtype)


@pytest.mark.parametrize("s", SHAPES, ids=ids)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=["bf16", "fp16"])
def test_key_scales_of_zero(s, dtype, cuda_device):
    """Keys that stand for zero, whatever their bytes: every visible value counts alike."""
    _, _, pages = batch(s["lens"], s["news"], s["P"])
    kp, vp, ks, vs = make_cache(pages, s["H_kv"], s["P"], s["D"])
    ks[:, 0] = 0
    run(s, (kp, vp, ks, vs), queries(s, dtype))
    run(s, (kp, vp, torch.zeros_like(ks), vs), queries(s, dtype))


@pytest.mark.parametrize("s", SHAPES, ids=ids)
def test_tiny_queries_and_small_key_scales(s, cuda_device):
    """bf16 query rows of zeros and of subnormals, keys of about 2^-10, a small scale: scores next to zero."""
    _, _, pages = batch(s["lens"], s["news"], s["P"])
    kp, vp, ks, vs = make_cache(pages, s["H_kv"], s["P"], s["D"])
    q = queries(s, torch.bfloat16)
    q[::3] = 0
    q[1::3] *= 2.0 ** -125
    run(s, (kp, vp, torch.full_like(ks, 2.0 ** -16), vs), q)
    run(s, (kp, vp, ks, vs), q, scale=2.0 ** -30)


@pytest.mark.parametrize("s", SHAPES, ids=ids)
@pytest.mark.parametrize("zero", ["keys", "values", "both"])
def test_zero_tokens(s, zero, cuda_device):
    """Appended zeros, of one head or of all: their pages have the smallest scale there is, 2^-126."""
    table, starts, pages = batch(s["lens"], s["news"], s["P"])
    for heads in (slice(0, 1), slice(None)):
        cache = _cache(*to_gpu(*make_cache(pages, s["H_kv"], s["P"], s["D"], junk=True)))
        all_starts = [0]
        for L in s["lens"]:
            all_starts.append(all_starts[-1] + L)
        x = torch.randn(all_starts[-1], 2, s["H_kv"], s["D"], generator=torch.Generator().manual_seed(3)).half()
        if zero != "values":
            x[:, 0, heads] = 0
        if zero != "keys":
            x[:, 1, heads] = 0
        xg = x.cuda()
        _append(cache, xg[:, 0], xg[:, 1], table.cuda(), i32(s["lens"]), i32(all_starts))
        tensors = [t.view(torch.uint8).cpu().view(t.dtype) if t.element_size() == 1 else t.cpu()
                   for t in (cache.k_pages, cache.v_pages, cache.k_scales, cache.v_scales)]
        assert float((tensors[2] if zero != "values" else tensors[3])[int(table[0, 0]), 0]) == 2.0 ** -126
        run(s, tensors, queries(s, torch.float16))


@pytest.mark.parametrize("s", SHAPES, ids=ids)
@pytest.mark.parametrize("power", [30, 60, 100])
@pytest.mark.parametrize("which", ["keys", "values"])
def test_large_tokens_that_a_row_does_not_see(s, power, which, cuda_device):
    """The page of the last tokens is 2^power above the others (a bf16 outlier): the rows before them are as exact
    as without it, and so are those of pages far below, where the scores pick them."""
    table, _, pages = batch(s["lens"], s["news"], s["P"])
    kp, vp, ks, vs = make_cache(pages, s["H_kv"], s["P"], s["D"])
    for b, L in enumerate(s["lens"]):
        (ks if which == "keys" else vs)[int(table[b, (L - 1) // s["P"]])] *= 2.0 ** power
        if which == "values":
            vs[int(table[b, 1])] *= 2.0 ** -power
    run(s, (kp, vp, ks, vs), queries(s, torch.bfloat16) * 3)


@pytest.mark.parametrize("s", SHAPES, ids=ids)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=["bf16", "fp16"])
def test_scales_that_are_no_powers_of_two(s, dtype, cuda_device):
    """Any finite scale is used as it is, in float32: large scores (20 and more) keep their weights."""
    _, _, pages = batch(s["lens"], s["news"], s["P"])
    kp, vp, ks, vs = make_cache(pages, s["H_kv"], s["P"], s["D"])
    g = torch.Generator().manual_seed(8)
    ks = 2.0 ** -7 * (0.5 + torch.rand(ks.shape, generator=g))
    vs = vs * (0.5 + torch.rand(vs.shape, generator=g))
    run(s, (kp, vp, ks, vs), (queries(s, torch.float32) * 8).to(dtype))


def test_single_tokens_and_a_chunk_in_one_batch(cuda_device):
    """A serving batch: 31 sequences that decode and one prompt's chunk, lengths from 1 to 1500."""
    g = torch.Generator().manual_seed(2)
    lens = [1 + int(x) for x in torch.randint(0, 1500, (32,), generator=g)]
    news = [1] * 32
    lens[17], news[17], lens[3] = 1400, 512, 1
    s = dict(lens=lens, news=news, P=64, H=32, H_kv=8, D=128)
    _, _, pages = batch(lens, news, 64)
    assert is_chunk(s)
    run(s, make_cache(pages, 8, 64, 128), queries(s, torch.bfloat16))


@pytest.mark.parametrize("s", SHAPES, ids=ids)
def test_bad_pages_are_reported(s, cuda_device):
    """A page out of range, first and last of a sequence: code 111, and the next call works."""
    nat = _nat()
    table, starts, pages = batch(s["lens"], s["news"], s["P"])
    cache = make_cache(pages, s["H_kv"], s["P"], s["D"])
    gpu, q = _cache(*to_gpu(*cache)), queries(s, torch.float16).cuda()
    for at, page in ((0, pages), (0, -1), ((s["lens"][0] - 1) // s["P"], 1 << 30)):
        bad = table.clone()
        bad[0, at] = page
        _attend(q, gpu, bad.cuda(), i32(s["lens"]), i32(starts))
        with pytest.raises(nat.KernelError, match="outside its table"):
            nat.check_status(cuda_device)
    run(s, cache, queries(s, torch.float16))


@pytest.mark.parametrize("s", SHAPES, ids=ids)
def test_nan_keys_of_every_place_in_a_tile(s, cuda_device):
    """A NaN in a cached key makes NaN of the rows that see it, wherever in a tile of 32 or 128 keys it stands, and
    changes no other row."""
    table, starts, pages = batch(s["lens"], s["news"], s["P"])
    kp, vp, ks, vs = make_cache(pages, s["H_kv"], s["P"], s["D"])
    q = queries(s, torch.float16)
    args = (table.cuda(), i32(s["lens"]), i32(starts))
    ref = _attend(q.cuda(), _cache(*to_gpu(kp, vp, ks, vs)), *args).cpu()
    group = s["H"] // s["H_kv"]
    for key0 in (0, 128):
        for shift in range(0, 128, s["H_kv"]):  # another key for each head but the last
            bad = kp.clone()
            expected = torch.zeros(ref.shape[:2], dtype=torch.bool)
            for h in range(s["H_kv"] - 1):
                key = key0 + (shift + h) % 128
                bad.view(torch.uint8)[int(table[0, key // s["P"]]), h, key % s["P"], (7 * h) % s["D"]] = 0x7f | (h % 2 << 7)
                first = max(0, key - (s["lens"][0] - s["news"][0]))  # the first token that sees it
                expected[first:starts[1], h * group:(h + 1) * group] = True
            o, lse = _attend(q.cuda(), _cache(*to_gpu(bad, vp, ks, vs)), *args, return_lse=True)
            o = o.cpu()
            assert bool(o[expected].isnan().all()) and torch.equal(lse.cpu().isnan(), expected)
            assert torch.equal(o[~expected], ref[~expected])
    _nat().check_status(cuda_device)


@pytest.mark.parametrize("s", SHAPES, ids=ids)
@pytest.mark.parametrize("power", [6, 13, 20, 30, 60])
def test_large_scores_pick_one_value(s, power, cuda_device):
    """Scores of about 2^power: where one leads by more than 64 and more than all float32 sums can be off, o is its
    value, rounded as a weight (2^-11), a logarithm (2^-16) and an output, whatever the scales."""
    table, starts, pages = batch(s["lens"], s["news"], s["P"])
    kp, vp, ks, vs = make_cache(pages, s["H_kv"], s["P"], s["D"])
    vs = vs * (0.5 + torch.rand(vs.shape, generator=torch.Generator().manual_seed(8)))
    q = queries(s, torch.bfloat16) * 2.0 ** power
    o, lse = _attend(q.cuda(), _cache(*to_gpu(kp, vp, ks, vs)), table.cuda(), i32(s["lens"]), i32(starts), return_lse=True)
    _nat().check_status(cuda_device)
    o, lse, leading = o.double().cpu(), lse.double().cpu(), 0
    assert bool(o.isfinite().all())
    group, scale = s["H"] // s["H_kv"], s["D"] ** -0.5
    for b, L in enumerate(s["lens"]):
        own = [int(x) for x in table[b, :-(-L // s["P"])]]
        K, V = ((x[own].double() * y[own].double()[..., None, None]).transpose(1, 2).reshape(-1, s["H_kv"], s["D"])[:L]
                for x, y in ((kp, ks), (vp, vs)))
        n = s["news"][b]
        hidden = torch.arange(L)[None] >= torch.arange(L - n, L)[:, None] + 1
        for h in range(s["H"]):
            row = q[starts[b]:starts[b + 1], h].double()
            x = (row @ K[:, h // group].T * scale).masked_fill(hidden, -math.inf)
            off = (row.abs() @ K[:, h // group].abs().T * scale).masked_fill(hidden, 0).amax(1) * 2 * s["D"] * 2.0 ** -24
            best, at = x.topk(min(2, L), 1)
            ahead = best[:, 0] - best[:, 1] > 64 + 4 * off
            leading += int(ahead.sum())
            ref = V[at[:, 0], h // group]
            bound = (2.0 ** -11 + 2.0 ** -16) * ref.abs() + 2.0 ** -60 * V.abs().max()
            tol = half_step(q.dtype) * (ref.abs() + bound) + bound
            got = o[starts[b]:starts[b + 1], h]
            assert bool(((got - ref).abs() <= tol)[ahead].all()), float(((got - ref).abs() / tol)[ahead].max())
            wide = math.log2(math.e) * (off + 2.0 ** -11) + 2.0 ** -22 * best[:, 0].abs() * math.log2(math.e)
            assert bool(((lse[starts[b]:starts[b + 1], h] - math.log2(math.e) * best[:, 0]).abs() <= wide)[ahead].all())
    assert leading > 10 * (power > 6)
