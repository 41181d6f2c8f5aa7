"""The paged e4m3 cache on the GPU: append_kv against a page-by-page float64 form (every byte and scale equal),
paged_attention against float64 attention over the same bytes, and a serving run of all three operators.

Bounds of attention: tests/serving_util.py (paged64) plus half a step of the output's type."""
import math

import pytest
import torch

from tests.serving_util import (E4M3, angles, append64, half_step, half_subnormal, norm_rope64, paged64, tables)

pytestmark = pytest.mark.gpu
EPS = 1e-6


def _nat():
    from attention.fused.fused import _native
    return _native()


def _cache(*tensors):
    from attention.paged.cache import PagedKVCache
    return PagedKVCache(*tensors)


def _append(*a, **kw):
    from attention.paged.cache import append_kv
    return append_kv(*a, **kw)


def _attend(*a, **kw):
    from attention.paged.paged_attention import paged_attention
    return paged_attention(*a, **kw)


def make_cache(pages, H_kv, P, D, seed=0, junk=False):
    """A cache in use: e4m3 values of all sizes, power-of-two scales that differ between pages and heads.  With
    `junk`, every byte and scale is arbitrary (NaN among them)."""
    g = torch.Generator().manual_seed(seed)
    if junk:
        kp, vp = (torch.randint(0, 256, (pages, H_kv, P, D), generator=g, dtype=torch.uint8).view(E4M3) for _ in range(2))
        ks, vs = (torch.full((pages, H_kv), float("nan")) for _ in range(2))
    else:
        kp, vp = ((torch.randn(pages, H_kv, P, D, generator=g) * 90).clamp(-448, 448).to(E4M3) for _ in range(2))
        ks, vs = (torch.exp2(torch.randint(-10, -4, (pages, H_kv), generator=g).float()) for _ in range(2))
    return kp, vp, ks, vs


def batch(lens, news, P, extra_pages=2, seed=0, width=None):
    """(block table, lens, starts, pages): a shuffled table; entries behind a sequence's last page are out of range."""
    g = torch.Generator().manual_seed(seed + 1)
    width = width or max(1, max(-(-L // P) for L in lens))
    need = sum(-(-L // P) for L in lens)
    order = torch.randperm(need + extra_pages, generator=g)
    table = torch.full((len(lens), width), 1 << 29, dtype=torch.int32)
    at = 0
    for b, L in enumerate(lens):
        n = -(-L // P)
        table[b, :n] = order[at:at + n].int()
        at += n
    starts = [0]
    for n in news:
        starts.append(starts[-1] + n)
    return table, starts, need + extra_pages


def to_gpu(*tensors):
    return [t.cuda() if t.dtype != E4M3 else t.view(torch.uint8).cuda().view(E4M3) for t in tensors]


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def same_bytes(a, b):
    return torch.equal(a.cpu().view(torch.uint8), b.cpu().view(torch.uint8))


# ------------------------------------------------------------------------------------------ append
APPENDS = [
    # lens, new tokens, page, H_kv, D
    ([1], [1], 16, 1, 32),
    ([17, 16, 1, 33, 40], [1, 1, 1, 1, 1], 16, 2, 64),
    ([5, 64, 130], [5, 64, 3], 64, 3, 128),
    ([100, 0, 37, 64], [70, 0, 37, 0], 32, 2, 128),
    ([300, 129], [300, 2], 128, 1, 128),
    ([200, 90, 7], [137, 90, 1], 128, 2, 64),
    ([260], [259], 128, 2, 32),
    ([33, 65, 97], [17, 31, 64], 16, 5, 32),
]


@pytest.mark.parametrize("lens,news,P,H_kv,D", APPENDS, ids=str)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=["bf16", "fp16"])
@pytest.mark.parametrize("variant", ["plain", "rotated", "normed", "axes"])
def test_append_bytes(lens, news, P, H_kv, D, dtype, variant, cuda_device):
    table, starts, pages = batch(lens, news, P)
    cache = make_cache(pages, H_kv, P, D)
    T = starts[-1]
    g = torch.Generator().manual_seed(7)
    x = (torch.randn(T + 3, 2 * H_kv, D, generator=g) * (10.0 ** torch.randint(-2, 3, (T + 3, 1, 1), generator=g))).to(dtype)
    k, v = x[:, :H_kv], x[:, H_kv:]  # three rows behind the last sequence
    interleaved = variant in ("axes", "normed")
    cos, sin = tables(400, D, "cpu")
    w = (1 + 0.5 * torch.randn(D, generator=g)).to(torch.float32 if variant == "axes" else dtype) if variant in ("normed", "axes") else None
    sections = (D // 2 - 7, 4, 3) if variant == "axes" else None
    own = torch.cat([torch.arange(L - n, L) for L, n in zip(lens, news)] + [torch.zeros(3, dtype=torch.long)])
    pos = torch.randint(0, 400, (3, T + 3), generator=g) if variant == "axes" else None
    kw = {}
    c = s = None
    if variant != "plain":
        c, s = angles(cos, sin, own if pos is None else pos, sections)
        kw = dict(cos=cos.cuda(), sin=sin.cuda(), positions=None if pos is None else pos.cuda(),
                  k_weight=None if w is None else w.cuda(), eps=EPS, interleaved=interleaved, sections=sections)
    ref = append64(*cache, k, v, table, lens, starts, c, s, w, EPS, interleaved)
    got = to_gpu(*cache)
    xg = x.cuda()
    _append(_cache(*got), xg[:, :H_kv], xg[:, H_kv:], table.cuda(), i32(lens), i32(starts), **kw)
    _nat().check_status(cuda_device)
    for name, a, b in zip(("k_pages", "v_pages", "k_scales", "v_scales"), got, ref):
        assert same_bytes(a, b), (name, int((a.cpu().view(torch.uint8) != b.view(torch.uint8)).sum()))
    if all(n == 1 for n in news):  # the same without offsets
        got = to_gpu(*cache)
        kw = {n: (t[:, :T].contiguous() if n == "positions" and t is not None else t) for n, t in kw.items()}
        _append(_cache(*got), xg[:T, :H_kv], xg[:T, H_kv:], table.cuda(), i32(lens), **kw)
        assert all(same_bytes(a, b) for a, b in zip(got, ref))


def test_append_token_by_token_grows_scales(cuda_device):
    """Tokens of growing size, one call each: every call re-rounds the page under its new scale, like the plain form."""
    P, H_kv, D = 32, 2, 64
    table, _, pages = batch([40], [1], P)
    ref = make_cache(pages, H_kv, P, D, junk=True)
    got = to_gpu(*ref)
    g = torch.Generator().manual_seed(1)
    for j in range(40):
        x = (torch.randn(1, 2 * H_kv, D, generator=g) * 1.3 ** ((j * 7) % 29)).half()
        ref = append64(*ref, x[:, :H_kv], x[:, H_kv:], table, [j + 1], [0, 1], None, None, None, EPS, False)
        xg = x.cuda()
        _append(_cache(*got), xg[:, :H_kv], xg[:, H_kv:], table.cuda(), i32([j + 1]))
    used = [int(p) for p in table[0]]
    for a, b in zip(got[2:], ref[2:]):
        assert torch.equal(a.cpu()[used], b[used])
    for a, b in zip(got[:2], ref[:2]):  # bytes behind the last token are left alone
        assert same_bytes(a, b)


def test_append_extremes(cuda_device):
    """Zeros, infinities, NaN, subnormals and the largest values; they change no other token's bytes."""
    P, H_kv, D = 16, 1, 32
    for dtype in (torch.bfloat16, torch.float16):
        x = torch.randn(12, 2, D, generator=torch.Generator().manual_seed(2)).to(dtype)
        x[3] = 0
        x[4, 1, 5], x[4, 1, 6] = float("inf"), float("-inf")
        x[5, 1, 7] = float("nan")
        x[6] = torch.finfo(dtype).tiny / 4
        x[7, 1, 0] = 448.0
        lens, starts = [12, 3, 1], [0, 8, 11, 12]
        x[8:11] = 0           # a page of zeros
        x[11] = torch.finfo(dtype).max
        lens = [8, 3, 1]
        table, _, pages = batch(lens, [8, 3, 1], P)
        cache = make_cache(pages, H_kv, P, D, junk=True)
        ref = append64(*cache, x[:, :1], x[:, 1:], table, lens, starts, None, None, None, EPS, False)
        got = to_gpu(*cache)
        xg = x.cuda()
        _append(_cache(*got), xg[:, :1], xg[:, 1:], table.cuda(), i32(lens), i32(starts))
        _nat().check_status(cuda_device)
        for a, b in zip(got, ref):
            assert torch.equal(a.cpu().float().nan_to_num(-7), b.float().nan_to_num(-7))
        page = int(table[0, 0])
        row = got[1].cpu().float()[page, 0]
        assert row[4, 5] == 448 and row[4, 6] == -448 and bool(row[5, 7].isnan()) and float(got[3][page, 0]) == 1.0
        assert float(got[3][int(table[1, 0]), 0]) == 2.0 ** -126


def test_append_tokens_before_the_start_and_empty_calls(cuda_device):
    """A sequence shorter than its new tokens keeps the last ones; empty batches write nothing."""
    P, H_kv, D = 16, 2, 64
    lens, news = [3, 20, 0], [10, 25, 4]
    table, starts, pages = batch(lens, news, P)
    cache = make_cache(pages, H_kv, P, D)
    x = torch.randn(39, 2 * H_kv, D, generator=torch.Generator().manual_seed(3)).bfloat16()
    ref = append64(*cache, x[:, :H_kv], x[:, H_kv:], table, lens, starts, None, None, None, EPS, False)
    got = to_gpu(*cache)
    xg = x.cuda()
    _append(_cache(*got), xg[:, :H_kv], xg[:, H_kv:], table.cuda(), i32(lens), i32(starts))
    assert all(same_bytes(a, b) for a, b in zip(got, ref))
    before = [t.clone() for t in got]
    empty = torch.empty(0, H_kv, D, dtype=torch.bfloat16, device="cuda")
    _append(_cache(*got), empty, empty, table.cuda(), i32(lens), i32([0, 0, 0, 0]))
    _append(_cache(*got), xg[:, :H_kv], xg[:, H_kv:], table.cuda(), i32(lens), i32([0, 0, 0, 0]))
    _append(_cache(*got), empty, empty, table[:0].cuda(), i32([]))
    _nat().check_status(cuda_device)
    assert all(same_bytes(a, b) for a, b in zip(got, before))


def test_append_long_prompt(cuda_device):
    """Windows of several tokens per block (a long prompt), against the plain form."""
    P, H_kv, D = 64, 8, 128
    lens, news = [5000, 1234], [4990, 1000]
    table, starts, pages = batch(lens, news, P)
    cache = make_cache(pages, H_kv, P, D)
    x = torch.randn(starts[-1], 2 * H_kv, D, generator=torch.Generator().manual_seed(4)).bfloat16()
    ref = append64(*cache, x[:, :H_kv], x[:, H_kv:], table, lens, starts, None, None, None, EPS, False)
    got = to_gpu(*cache)
    xg = x.cuda()
    _append(_cache(*got), xg[:, :H_kv], xg[:, H_kv:], table.cuda(), i32(lens), i32(starts))
    _nat().check_status(cuda_device)
    assert all(same_bytes(a, b) for a, b in zip(got, ref))


# --------------------------------------------------------------------------------------- attention
def takes_chunk_kernel(T, B, H, H_kv, D):
    """The library's choice between its two kernels (csrc/fa_chunk.cu, use_chunk)."""
    rows = -(-T * (H // H_kv) // B)
    items = B * H_kv
    waves = -(-items * -(-rows // 256) // 148)
    return items * -(-rows // 16) >= (320 if D == 128 else 400) * waves


def check_attention(o, lse, q, cache, table, lens, starts, scale, T=None):
    """T: the call's query tokens, where q is only the ones that sequences have."""
    chunk = takes_chunk_kernel(T or q.shape[0], len(lens), q.shape[1], cache[0].shape[1], q.shape[2])
    ref, ref_lse, bound, lse_bound = paged64(q, *cache, table, lens, starts, scale, chunk)
    o = o.double().cpu()
    tol = half_step(q.dtype) * (ref.abs() + bound) + bound + half_subnormal(q.dtype)
    assert bool(o.isfinite().all())
    worst = float(((o - ref).abs() / tol).max())
    assert worst <= 1.0, worst
    if lse is not None:
        lse = lse.double().cpu()
        seen = ref_lse.isfinite()
        assert bool((lse[~seen] == -math.inf).all())
        assert bool(((lse - ref_lse).abs() <= lse_bound)[seen].all())


ATTENDS = [
    # lens, new tokens, page, H, H_kv, D
    ([1], [1], 16, 1, 1, 32),
    ([1, 2, 15, 16, 17], [1, 1, 1, 1, 1], 16, 8, 2, 64),
    ([64, 65, 63, 128, 129, 1000], [1] * 6, 64, 32, 8, 128),
    ([777, 1], [1, 1], 128, 4, 4, 128),
    ([500, 300], [1, 1], 32, 14, 2, 128),      # groups of 7
    ([200, 1500], [1, 1], 16, 64, 2, 64),      # groups of 32: several tiles of rows
    ([90, 4, 0, 33], [3, 4, 0, 1], 16, 8, 8, 64),
    ([130, 70], [65, 70], 32, 6, 2, 128),
    ([257, 1025], [2, 5], 64, 24, 8, 128),
    ([40, 7], [17, 7], 16, 5, 1, 32),
    ([3000], [1], 64, 16, 1, 128),
    ([300], [300], 128, 4, 1, 64),
]


@pytest.mark.parametrize("lens,news,P,H,H_kv,D", ATTENDS, ids=str)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=["bf16", "fp16"])
def test_attention(lens, news, P, H, H_kv, D, dtype, cuda_device):
    table, starts, pages = batch(lens, news, P)
    cache = make_cache(pages, H_kv, P, D)
    q = (3 * torch.randn(starts[-1], H, D, generator=torch.Generator().manual_seed(5))).to(dtype)
    gpu = _cache(*to_gpu(*cache))
    args = (q.cuda(), gpu, table.cuda(), i32(lens))
    o, lse = _attend(*args, i32(starts), return_lse=True)
    _nat().check_status(cuda_device)
    check_attention(o, lse, q, cache, table, lens, starts, D ** -0.5)
    assert torch.equal(o, _attend(*args, i32(starts)))  # the same bits every time
    if all(n == 1 for n in news):
        assert torch.equal(o, _attend(*args))


CHUNKS = [
    # lens, new tokens, page, H, H_kv, D: many rows, which the chunk kernel takes
    ([700, 129, 128, 1], [500, 129, 100, 1], 64, 64, 16, 128),
    ([5, 300, 0, 257], [50, 200, 0, 257], 16, 48, 16, 128),   # tokens in front of the first key, groups of 3
    ([400, 383], [384, 129], 128, 28, 4, 128),                # groups of 7
    ([333, 300], [333, 300], 32, 16, 16, 64),
    ([1000], [256], 16, 32, 8, 64),
    ([513, 640, 64], [300, 257, 64], 32, 40, 8, 32),
    ([2100], [700], 64, 8, 8, 128),
]


@pytest.mark.parametrize("lens,news,P,H,H_kv,D", CHUNKS, ids=str)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=["bf16", "fp16"])
def test_attention_of_many_rows(lens, news, P, H, H_kv, D, dtype, cuda_device):
    table, starts, pages = batch(lens, news, P)
    assert takes_chunk_kernel(starts[-1], len(lens), H, H_kv, D)
    cache = make_cache(pages, H_kv, P, D)
    q = (3 * torch.randn(starts[-1], H, D, generator=torch.Generator().manual_seed(5))).to(dtype)
    gpu = _cache(*to_gpu(*cache))
    args = (q.cuda(), gpu, table.cuda(), i32(lens), i32(starts))
    o, lse = _attend(*args, return_lse=True)
    _nat().check_status(cuda_device)
    check_attention(o, lse, q, cache, table, lens, starts, D ** -0.5)
    assert torch.equal(o, _attend(*args))


def test_many_rows_read_only_what_they_see(cuda_device):
    """The chunk kernel with NaN behind the last tokens, bad table entries behind the last pages, rows behind the last
    sequence, strided q and out, and page scales of all sizes."""
    P, H, H_kv, D = 32, 32, 16, 128
    lens, news = [290, 33, 470, 3], [200, 33, 150, 9]
    table, starts, pages = batch(lens, news, P, extra_pages=5)
    kp, vp, ks, vs = make_cache(pages, H_kv, P, D)
    vs *= torch.exp2(torch.randint(-30, 1, vs.shape, generator=torch.Generator().manual_seed(1)).float())
    used = set()
    for b, L in enumerate(lens):
        for j in range(-(-L // P)):
            page = int(table[b, j])
            used.add(page)
            for t in (kp, vp):
                t.view(torch.uint8)[page, :, min(P, L - j * P):] = 0x7f
    for page in set(range(pages)) - used:
        ks[page] = vs[page] = float("nan")
    T = starts[-1] + 5
    assert takes_chunk_kernel(T, len(lens), H, H_kv, D)
    q = torch.randn(T, H + 8, D, generator=torch.Generator().manual_seed(6)).bfloat16()
    out = torch.full((T, 2 * H, D), 9.0, dtype=torch.bfloat16, device="cuda")
    args = (q.cuda()[:, 8:], _cache(*to_gpu(kp, vp, ks, vs)), table.cuda(), i32(lens), i32(starts))
    o, lse = _attend(*args, out=out[:, H:], return_lse=True)
    _nat().check_status(cuda_device)
    clean = [t.clone() for t in (kp, vp, ks, vs)]
    for t in clean[:2]:
        t.copy_(t.float().nan_to_num(0).to(E4M3))
    n = starts[-1]
    check_attention(o[:n], lse[:n], q[:n, 8:], clean, table, lens, starts, D ** -0.5, T)
    assert bool((out[:, :H] == 9).all()) and bool((out[n:] == 9).all()) and bool((lse[n:] == -math.inf).all())
    o2, lse2 = _attend(*args, return_lse=True)
    assert torch.equal(o2[:n], o[:n]) and bool((o2[n:] == 0).all()) and torch.equal(lse2, lse)


def test_many_rows_with_unusual_queries(cuda_device):
    """bf16 queries far outside f16's range; NaN and infinity stay in their rows."""
    P, H, H_kv, D = 64, 16, 16, 128
    lens, news = [400, 380], [330, 360]
    table, starts, pages = batch(lens, news, P)
    cache = make_cache(pages, H_kv, P, D)
    gpu = _cache(*to_gpu(*cache))
    tables = (table.cuda(), i32(lens), i32(starts))
    assert takes_chunk_kernel(starts[-1], 2, H, H_kv, D)
    for power in (60, -60):
        q = (torch.randn(starts[-1], H, D, generator=torch.Generator().manual_seed(1)) * 2.0 ** power).bfloat16()
        o, lse = _attend(q.cuda(), gpu, *tables, scale=2.0 ** -power / 8, return_lse=True)
        check_attention(o, lse, q, cache, table, lens, starts, 2.0 ** -power / 8)
    q = torch.randn(starts[-1], H, D, generator=torch.Generator().manual_seed(1)).half()
    ref = _attend(q.cuda(), gpu, *tables)
    for bad in (float("nan"), float("inf")):
        q2 = q.clone()
        q2[5, 3, 7] = bad
        o = _attend(q2.cuda(), gpu, *tables)
        assert bool(o[5, 3].isnan().all())
        keep = torch.ones(q.shape[:2], dtype=torch.bool)
        keep[5, 3] = False
        assert torch.equal(o.cpu()[keep], ref.cpu()[keep])


def test_many_rows_failure_detection(cuda_device):
    """A status word that is set stops the chunk kernel before it writes; in the failure-detection build, whose issuer
    waits for something that never comes, it records a timeout and returns, and the product kernel works after that."""
    import ctypes
    import os
    from tests.test_failure_detection_gpu import PIPELINE_TIMEOUT_CODES, STALL_LIB
    from tests.test_serving_cpu import PAGED_ARGS
    P, H, H_kv, D = 64, 16, 16, 128
    lens, news = [400, 380], [330, 360]
    table, starts, pages = batch(lens, news, P)
    cache = make_cache(pages, H_kv, P, D)
    tensors = to_gpu(*cache)
    q = torch.randn(starts[-1], H, D, generator=torch.Generator().manual_seed(1)).half()
    qg, tg, lg, sg = q.cuda(), table.cuda(), i32(lens), i32(starts)
    nat = _nat()
    status = nat.status_tensor(cuda_device)
    out = torch.full_like(qg, 5.0)
    status.fill_(1)
    try:
        _attend(qg, _cache(*tensors), tg, lg, sg, out=out)
        torch.cuda.synchronize()
        assert bool((out == 5).all())
    finally:
        status.zero_()
    if not os.path.exists(STALL_LIB):
        pytest.skip("the failure-detection build is not there")
    lib = ctypes.CDLL(STALL_LIB)
    own = torch.zeros(4, dtype=torch.int32, device="cuda")
    workspace = torch.empty(16 << 20, dtype=torch.uint8, device="cuda")
    packed = PAGED_ARGS.pack(qg.data_ptr(), *(t.data_ptr() for t in tensors), tg.data_ptr(), lg.data_ptr(), sg.data_ptr(),
                             out.data_ptr(), 0, workspace.data_ptr(), H * D, D, H * D, D, tg.stride(0), starts[-1], 2, tg.shape[1],
                             pages, H, H_kv, P, D, 0, 0, D ** -0.5)
    lib.fa_paged_attention.argtypes = [ctypes.c_void_p] * 3
    assert lib.fa_paged_attention(packed, own.data_ptr(), torch.cuda.current_stream().cuda_stream) == 0
    torch.cuda.synchronize()
    assert own.tolist()[0] in PIPELINE_TIMEOUT_CODES
    o = _attend(qg, _cache(*tensors), tg, lg, sg)
    nat.check_status(cuda_device)
    check_attention(o, None, q, cache, table, lens, starts, D ** -0.5)


def test_attention_reads_only_what_it_sees(cuda_device):
    """Bytes and scales behind the last token are NaN, table entries behind the last page out of range."""
    P, H, H_kv, D = 32, 8, 2, 128
    lens, news = [1, 31, 32, 33, 70, 200], [1, 2, 1, 3, 1, 40]
    table, starts, pages = batch(lens, news, P, extra_pages=5)
    kp, vp, ks, vs = make_cache(pages, H_kv, P, D)
    used = set()
    for b, L in enumerate(lens):
        for j in range(-(-L // P)):
            page = int(table[b, j])
            used.add(page)
            end = min(P, L - j * P)
            for t in (kp, vp):
                t.view(torch.uint8)[page, :, end:] = 0x7f
    for page in set(range(pages)) - used:
        ks[page] = vs[page] = float("nan")
        kp.view(torch.uint8)[page] = vp.view(torch.uint8)[page] = 0xff
    q = torch.randn(starts[-1], H, D, generator=torch.Generator().manual_seed(6)).bfloat16()
    o, lse = _attend(q.cuda(), _cache(*to_gpu(kp, vp, ks, vs)), table.cuda(), i32(lens), i32(starts), return_lse=True)
    _nat().check_status(cuda_device)
    clean = [t.clone() for t in (kp, vp, ks, vs)]
    for t in clean[:2]:
        t.copy_(t.float().nan_to_num(0).to(E4M3))
    check_attention(o, lse, q, clean, table, lens, starts, D ** -0.5)


def test_rows_without_keys_and_rows_behind(cuda_device):
    """Empty sequences and tokens in front of the first key give 0 and -inf; rows behind the last sequence keep
    what `out` held, or are 0."""
    P, H, H_kv, D = 16, 4, 2, 64
    lens, news = [0, 2, 5], [1, 6, 0]
    table, starts, pages = batch(lens, news, P)
    cache = make_cache(pages, H_kv, P, D)
    gpu = _cache(*to_gpu(*cache))
    q = torch.randn(10, H, D, generator=torch.Generator().manual_seed(8)).half()
    args = (q.cuda(), gpu, table.cuda(), i32(lens), i32(starts))
    out = torch.full((10, H, D), 7.0, dtype=torch.float16, device="cuda")
    o, lse = _attend(*args, out=out, return_lse=True)
    assert o is out and bool((o[7:] == 7).all())
    assert bool((o[:5] == 0).all()) and bool((lse[:5] == -math.inf).all())
    check_attention(o[:7], lse[:7], q[:7], cache, table, lens, starts, D ** -0.5)
    assert bool((_attend(*args)[7:] == 0).all())
    assert _attend(q[:0].cuda(), gpu, table.cuda(), i32(lens), i32([0, 0, 0, 0])).shape == (0, H, D)
    assert bool((_attend(q.cuda(), gpu, table[:0].cuda(), i32([]), i32([0])) == 0).all())
    _nat().check_status(cuda_device)


def test_page_scales_far_apart(cuda_device):
    """Pages whose value scales differ by 2^40, and sharp scores that pick either: no page loses precision."""
    P, H, H_kv, D = 16, 2, 1, 32
    lens, news = [64], [1]
    table, starts, pages = batch(lens, news, P)
    kp, vp, ks, vs = make_cache(pages, H_kv, P, D)
    for i, page in enumerate(table[0].tolist()):
        vs[page] = 2.0 ** (-34 + 13 * i)
        ks[page] = 2.0 ** -6
    for sharp in (0.0, 4.0):
        q = torch.zeros(1, H, D).half()
        first = kp[int(table[0, 0]), 0, 3].float()
        q[0, 0] = (sharp * first / first.norm() * 8).half()
        q[0, 1] = torch.randn(D, generator=torch.Generator().manual_seed(1)).half()
        o, lse = _attend(q.cuda(), _cache(*to_gpu(kp, vp, ks, vs)), table.cuda(), i32(lens), return_lse=True)
        # scaled up, out of fp16's subnormals: compare where the output's type can hold it
        check_attention(o, lse, q, (kp, vp, ks, vs), table, lens, starts, D ** -0.5)
        qb = q.bfloat16()
        o, lse = _attend(qb.cuda(), _cache(*to_gpu(kp, vp, ks, vs)), table.cuda(), i32(lens), return_lse=True)
        check_attention(o, lse, qb, (kp, vp, ks, vs), table, lens, starts, D ** -0.5)


def test_large_and_small_queries(cuda_device):
    """bf16 queries far outside f16's range, with a scale that brings the scores back."""
    P, H, H_kv, D = 32, 4, 2, 64
    lens, news = [100], [1]
    table, starts, pages = batch(lens, news, P)
    cache = make_cache(pages, H_kv, P, D)
    for power in (60, -60):
        q = (torch.randn(1, H, D, generator=torch.Generator().manual_seed(1)) * 2.0 ** power).bfloat16()
        scale = 2.0 ** -power / 8
        o, lse = _attend(q.cuda(), _cache(*to_gpu(*cache)), table.cuda(), i32(lens), scale=scale, return_lse=True)
        check_attention(o, lse, q, cache, table, lens, starts, scale)


def test_nan_query_stays_in_its_row(cuda_device):
    P, H, H_kv, D = 16, 4, 1, 64
    lens, news = [50, 20], [2, 1]
    table, starts, pages = batch(lens, news, P)
    gpu = _cache(*to_gpu(*make_cache(pages, H_kv, P, D)))
    for dtype in (torch.float16, torch.bfloat16):
        q = torch.randn(3, H, D, generator=torch.Generator().manual_seed(1)).to(dtype)
        ref = _attend(q.cuda(), gpu, table.cuda(), i32(lens), i32(starts))
        for bad in (float("nan"), float("inf")):
            q2 = q.clone()
            q2[0, 2, 5] = bad
            o = _attend(q2.cuda(), gpu, table.cuda(), i32(lens), i32(starts))
            assert bool(o[0, 2].isnan().all())
            keep = torch.ones(3, H, dtype=torch.bool)
            keep[0, 2] = False
            assert torch.equal(o.cpu()[keep], ref.cpu()[keep])


def test_strides_and_shared_pages(cuda_device):
    """q and out as views, a block table that is a view of a wider one, the same page in two sequences (a shared
    prompt) and twice in one."""
    P, H, H_kv, D = 16, 8, 2, 64
    lens, news = [48, 33, 40], [1, 1, 1]
    table, starts, pages = batch(lens, news, P)
    table[1, :2] = table[0, :2]
    table[2, 1] = table[2, 0]
    cache = make_cache(pages, H_kv, P, D)
    q = torch.randn(3, H + 4, D, generator=torch.Generator().manual_seed(1)).half()
    qg = q.cuda()[:, 2:2 + H]
    wide = torch.zeros(3, 9, dtype=torch.int32, device="cuda")
    wide[:, :table.shape[1]] = table.cuda()
    out = torch.zeros(3, 2 * H, D, dtype=torch.float16, device="cuda")
    o, lse = _attend(qg, _cache(*to_gpu(*cache)), wide[:, :table.shape[1]], i32(lens), out=out[:, H:], return_lse=True)
    check_attention(o, lse, q[:, 2:2 + H], cache, table, lens, starts, D ** -0.5)
    assert bool((out[:, :H] == 0).all())
    odd = torch.empty(3 * H * D + 1, dtype=torch.float16, device="cuda")[1:].view(3, H, D).copy_(qg)
    assert torch.equal(_attend(odd, _cache(*to_gpu(*cache)), table.cuda(), i32(lens)), o)


@pytest.mark.parametrize("lens,news,P,H,H_kv,D", [ATTENDS[2], ATTENDS[8], CHUNKS[0], CHUNKS[3]], ids=str)
def test_out_may_be_q_and_keys_may_be_values(lens, news, P, H, H_kv, D, cuda_device):
    """Writing o over q, and a cache whose keys are its values: the same bits as apart."""
    table, starts, pages = batch(lens, news, P)
    kp, vp, ks, vs = make_cache(pages, H_kv, P, D)
    q = torch.randn(starts[-1], H, D, generator=torch.Generator().manual_seed(6)).bfloat16().cuda()
    args = (table.cuda(), i32(lens), i32(starts))
    apart = _attend(q, _cache(*to_gpu(kp, kp.clone(), ks, ks.clone())), *args)
    kg, sg = to_gpu(kp, vp, ks, vs)[::2]
    o = q.clone()
    assert _attend(o, _cache(kg, kg, sg, sg), *args, out=o) is o
    assert torch.equal(o, apart)


def test_many_sequences_and_long_tables(cuda_device):
    """More sequences than a block has threads, most of them short, one long; a table much wider than needed."""
    P, H, H_kv, D = 16, 4, 2, 32
    g = torch.Generator().manual_seed(11)
    lens = torch.randint(0, 40, (300,), generator=g).tolist()
    lens[123] = 2500
    news = [min(L, int(n)) if L else 1 for L, n in zip(lens, torch.randint(0, 4, (300,), generator=g))]
    table, starts, pages = batch(lens, news, P, width=4096)
    cache = make_cache(pages, H_kv, P, D)
    q = torch.randn(starts[-1], H, D, generator=g).bfloat16()
    o, lse = _attend(q.cuda(), _cache(*to_gpu(*cache)), table.cuda(), i32(lens), i32(starts), return_lse=True)
    _nat().check_status(cuda_device)
    check_attention(o, lse, q, cache, table, lens, starts, D ** -0.5)


def nan_case(lens, news, P, H, H_kv, D, dtype):
    """NaN values among the new tokens' keys, hidden from the tokens before them: (q, tensors, clean tensors, the
    entries of o that have to be NaN, table, starts)."""
    table, starts, pages = batch(lens, news, P)
    kp, vp, ks, vs = make_cache(pages, H_kv, P, D)
    g = torch.Generator().manual_seed(9)
    expected = torch.zeros(starts[-1], H, D, dtype=torch.bool)
    clean = vp.clone()
    for b, (L, n) in enumerate(zip(lens, news)):
        for _ in range(3):
            key = L - 1 - int(torch.randint(0, max(1, min(n, L)), (), generator=g))
            head, d = int(torch.randint(0, H_kv, (), generator=g)), int(torch.randint(0, D, (), generator=g))
            page = int(table[b, key // P])
            vp.view(torch.uint8)[page, head, key % P, d] = 0xff if d % 2 else 0x7f
            clean.view(torch.uint8)[page, head, key % P, d] = 0
            for i in range(n):
                if L - n + i >= key:
                    expected[starts[b] + i, head * (H // H_kv):(head + 1) * (H // H_kv), d] = True
    q = torch.randn(starts[-1], H, D, generator=g).to(dtype)
    return q, (kp, vp, ks, vs), (kp, clean, ks, vs), expected, table, starts


@pytest.mark.parametrize("lens,news,P,H,H_kv,D", [
    ([50, 133], [5, 40], 16, 8, 2, 64), ([300, 40], [20, 9], 64, 4, 4, 128), ([90], [60], 32, 6, 1, 32),
    ([700, 129, 128], [500, 129, 100], 64, 64, 16, 128), ([333, 300], [333, 300], 32, 16, 16, 64),
    ([513, 640, 64], [300, 257, 64], 32, 40, 8, 32)], ids=str)
def test_nan_values_reach_only_the_tokens_that_see_them(lens, news, P, H, H_kv, D, cuda_device):
    q, tensors, clean, expected, table, starts = nan_case(lens, news, P, H, H_kv, D, torch.float16)
    o = _attend(q.cuda(), _cache(*to_gpu(*tensors)), table.cuda(), i32(lens), i32(starts))
    _nat().check_status(cuda_device)
    o = o.cpu()
    assert torch.equal(o.isnan(), expected)
    ref = _attend(q.cuda(), _cache(*to_gpu(*clean)), table.cuda(), i32(lens), i32(starts)).cpu()
    assert torch.equal(o[~expected], ref[~expected])


def test_nan_keys_reach_only_the_tokens_that_see_them(cuda_device):
    for lens, news, P, H, H_kv, D in (([50, 133], [5, 40], 16, 8, 2, 64), ([700, 129, 128], [500, 129, 100], 64, 64, 16, 128)):
        table, starts, pages = batch(lens, news, P)
        kp, vp, ks, vs = make_cache(pages, H_kv, P, D)
        q = torch.randn(starts[-1], H, D, generator=torch.Generator().manual_seed(1)).half()
        args = (table.cuda(), i32(lens), i32(starts))
        ref = _attend(q.cuda(), _cache(*to_gpu(kp, vp, ks, vs)), *args).cpu()
        key = lens[0] - 3
        kp.view(torch.uint8)[int(table[0, key // P]), 1, key % P, 5] = 0x7f
        o = _attend(q.cuda(), _cache(*to_gpu(kp, vp, ks, vs)), *args).cpu()
        hit = torch.zeros(o.shape[:2], dtype=torch.bool)
        hit[starts[1] - 3:starts[1], H // H_kv:2 * (H // H_kv)] = True
        assert bool(o[hit].isnan().all()) and torch.equal(o[~hit], ref[~hit])


@pytest.mark.parametrize("D", [32, 64, 128])
@pytest.mark.parametrize("group,n", [(4, 1), (16, 1), (3, 7)])
def test_full_grids_fit_the_workspace(D, group, n, cuda_device):
    """Tables wide enough for a full grid of blocks, with both row tiles: every block has its part of the workspace."""
    P, H_kv = 16, 4
    lens = [900, 20, 333, 5, 700, 64]
    news = [min(n, L) for L in lens]
    table, starts, pages = batch(lens, news, P, width=2000)
    cache = make_cache(pages, H_kv, P, D)
    q = torch.randn(starts[-1], H_kv * group, D, generator=torch.Generator().manual_seed(3)).half()
    o, lse = _attend(q.cuda(), _cache(*to_gpu(*cache)), table.cuda(), i32(lens), i32(starts), return_lse=True)
    _nat().check_status(cuda_device)
    check_attention(o, lse, q, cache, table, lens, starts, D ** -0.5)


def test_out_that_overlaps_itself_is_refused(cuda_device):
    P, H, H_kv, D = 16, 4, 2, 64
    table, starts, pages = batch([40, 20], [1, 1], P)
    gpu = _cache(*to_gpu(*make_cache(pages, H_kv, P, D)))
    q = torch.randn(2, H, D, device="cuda").half()
    for out in (torch.empty(1, H, D, device="cuda").half().expand(2, H, D), torch.empty(2, 1, D, device="cuda").half().expand(2, H, D),
                torch.empty(2, D, H, device="cuda").half().transpose(1, 2)):
        with pytest.raises(ValueError, match="out must be contiguous"):
            _attend(q, gpu, table.cuda(), i32([40, 20]), out=out)


def test_cache_past_32_bit_offsets(cuda_device):
    """Pages whose byte offsets pass 2^32."""
    P, H, H_kv, D = 128, 8, 2, 128
    pages = (1 << 32) // (H_kv * P * D) + 40
    kp, vp = (torch.zeros(pages, H_kv, P, D, dtype=torch.uint8, device="cuda").view(E4M3) for _ in range(2))
    ks, vs = (torch.zeros(pages, H_kv, device="cuda") for _ in range(2))
    lens, news = [300, 130], [300, 130]
    table = torch.tensor([[pages - 1, 3, pages - 7], [pages - 20, pages - 30, 0]], dtype=torch.int32)
    starts = [0, 300, 430]
    x = torch.randn(430, 2 * H_kv, D, generator=torch.Generator().manual_seed(1)).bfloat16()
    xg = x.cuda()
    cache = _cache(kp, vp, ks, vs)
    _append(cache, xg[:, :H_kv], xg[:, H_kv:], table.cuda(), i32(lens), i32(starts))
    q = torch.randn(2, H, D, generator=torch.Generator().manual_seed(2)).bfloat16()
    o, lse = _attend(q.cuda(), cache, table.cuda(), i32(lens), return_lse=True)
    _nat().check_status(cuda_device)
    small = torch.tensor([[0, 1, 2], [3, 4, 5]], dtype=torch.int32)
    ref = append64(*make_cache(6, H_kv, P, D), x[:, :H_kv], x[:, H_kv:], small, lens, starts, None, None, None, EPS, False)
    rows = table.flatten().tolist()
    for i, (p, L) in enumerate(zip(rows, [128, 128, 44, 128, 2, 0])):
        for a, b in ((kp, ref[0]), (vp, ref[1])):
            assert same_bytes(a[p, :, :L], b[i, :, :L])
    check_attention(o, lse, q, ref, small, lens, [0, 1, 2], D ** -0.5)


def test_bad_tables_are_reported(cuda_device):
    """Pages, lengths and offsets out of range: code 111, no access outside the buffers, and the next call works."""
    nat = _nat()
    P, H, H_kv, D = 16, 4, 2, 64
    lens, news = [40, 20], [2, 1]
    table, starts, pages = batch(lens, news, P)
    cache = make_cache(pages, H_kv, P, D)
    gpu = _cache(*to_gpu(*cache))
    q = torch.randn(3, H, D, generator=torch.Generator().manual_seed(1)).half()
    kv = torch.randn(3, H_kv, D, device="cuda").half()

    def attend(table, lens, starts):
        return _attend(q.cuda(), gpu, table.cuda(), i32(lens), i32(starts))

    def append(table, lens, starts):
        scratch = _cache(*to_gpu(*cache))
        return _append(scratch, kv, kv, table.cuda(), i32(lens), i32(starts))

    bad_page, negative = table.clone(), table.clone()
    bad_page[0, 2] = pages
    negative[1, 1] = -1
    for call in (attend, append):
        for a in ((bad_page, lens, starts), (negative, lens, starts), (table, [40, 16 * table.shape[1] + 1], starts),
                  (table, lens, [0, 2, 4])):
            call(*a)
            with pytest.raises(nat.KernelError, match="outside its table"):
                nat.check_status(cuda_device)
    cos, sin = tables(30, D, "cuda")
    _append(_cache(*to_gpu(*cache)), kv, kv, table.cuda(), i32(lens), i32(starts), cos=cos, sin=sin)
    with pytest.raises(nat.KernelError, match="outside its table"):  # positions 38, 39 in a table of 30
        nat.check_status(cuda_device)
    o = attend(table, lens, starts)
    nat.check_status(cuda_device)
    check_attention(o, None, q, cache, table, lens, starts, D ** -0.5)


def test_nonzero_status_word_writes_nothing(cuda_device):
    nat = _nat()
    P, H, H_kv, D = 16, 4, 2, 64
    table, starts, pages = batch([40, 20], [2, 1], P)
    cache = to_gpu(*make_cache(pages, H_kv, P, D))
    before = [t.clone() for t in cache]
    q = torch.randn(3, H, D, device="cuda").half()
    out = torch.full_like(q, 5.0)
    status = nat.status_tensor(cuda_device)
    status.fill_(1)
    try:
        _append(_cache(*cache), q[:, :H_kv], q[:, :H_kv], table.cuda(), i32([40, 20]), i32(starts))
        _attend(q, _cache(*cache), table.cuda(), i32([40, 20]), i32(starts), out=out)
        torch.cuda.synchronize()
        assert bool((out == 5).all()) and all(same_bytes(a, b) for a, b in zip(cache, before))
    finally:
        status.zero_()


# ------------------------------------------------------------------------------------- serving run
def test_serving_run(cuda_device):
    """Prompts in chunks, then decoding with changing batches: norm + rotation of q, append, attention, through
    CUDA graphs for the decode steps, against float64 attention over unquantised keys and values.

    Each e4m3 value is off by at most 2^-4 of itself (half a step) or 2^-10 of its scale, 448 scales being
    less than twice the page's largest magnitude.  Rows of q and k have RMS 1.02 and D = 64: a score's error is
    at most 2^-4 sum|q k| / 8 <= 2^-4 |q| |k| / 8 = 0.52; weights then change by at most a factor e^(+-1.04), and
    o by less than (e^1.04 - 1 + 2^-4) < 2 times the largest |v|.  That bound is wide; the exact one is paged64's
    on the cached bytes, which is also checked."""
    from attention.rotary.norm_rope import qk_norm_rope
    P, H, H_kv, D, width = 16, 8, 2, 64, 12
    g = torch.Generator(device="cuda").manual_seed(21)
    cos, sin = tables(P * width, D, "cuda")
    qw, kw = ((1 + 0.2 * torch.randn(D, device="cuda", generator=g)).bfloat16() for _ in range(2))
    cache = _cache(*to_gpu(*make_cache(40, H_kv, P, D, junk=True)))
    table = torch.randperm(36, generator=torch.Generator().manual_seed(1))[:36].view(3, 12).int()
    tg = table.cuda()
    history = [[], [], []]

    def project(T):
        x = torch.randn(T, H + 2 * H_kv, D, device="cuda", generator=g).bfloat16()
        return x[:, :H], x[:, H:H + H_kv], x[:, H + H_kv:]

    def step(q, k, v, lens_t, offsets, positions):
        qr, _ = qk_norm_rope(q.transpose(0, 1)[None], None, cos, sin, positions[None], qw)
        qr = qr[0].transpose(0, 1)
        _append(cache, k, v, tg, lens_t, offsets, cos=cos, sin=sin, k_weight=kw)
        return qr, _attend(qr, cache, tg, lens_t, offsets)

    def remember(k, v, lens, starts):
        for b, L in enumerate(lens):
            for i in range(starts[b], starts[b + 1]):
                p = L - (starts[b + 1] - i)
                c, s = angles(cos, sin, torch.tensor([p], device="cuda"), None)
                history[b].append((norm_rope64(k[i:i + 1], kw, c[:, None], s[:, None], EPS, False)[0].cpu(), v[i].double().cpu()))

    def check(qr, o, lens, starts):
        host = [t.cpu() if t.dtype != E4M3 else t.view(torch.uint8).cpu().view(E4M3)
                for t in (cache.k_pages, cache.v_pages, cache.k_scales, cache.v_scales)]
        check_attention(o, None, qr.cpu(), host, table, lens, starts, D ** -0.5)
        for b, L in enumerate(lens):
            n = starts[b + 1] - starts[b]
            if n == 0:
                continue
            K = torch.stack([x[0] for x in history[b]])
            V = torch.stack([x[1] for x in history[b]])
            Kc, Vc = (x.double().cpu() for x in cache.gather(tg[b], L))
            for a, r in ((Kc, K), (Vc, V)):  # rounded, perhaps again under a grown scale
                top = r.abs().amax()
                assert bool(((a - r).abs() <= 2 * (2.0 ** -4 * r.abs() + 2.0 ** -10 * 2 * top / 448)).all())
            for h in range(H):
                x = K[:, h // 4] @ qr[starts[b + 1] - 1, h].double().cpu() / 8
                ref = torch.softmax(x, 0) @ V[:, h // 4]
                spread = V[:, h // 4].abs().amax(0)
                assert bool(((o[starts[b + 1] - 1, h].double().cpu() - ref).abs() <= 2 * spread).all())

    lens = [0, 0, 0]
    for news in ([37, 5, 16], [20, 0, 1], [3, 30, 40]):  # prompts, chunk by chunk
        starts = [0]
        for n in news:
            starts.append(starts[-1] + n)
        lens = [a + b for a, b in zip(lens, news)]
        positions = torch.cat([torch.arange(L - n, L) for L, n in zip(lens, news)]).cuda()
        q, k, v = project(starts[-1])
        qr, o = step(q, k, v, i32(lens), i32(starts), positions)
        remember(k, v, lens, starts)
        check(qr, o, lens, starts)

    # decoding: one captured step, replayed with new tokens and lengths
    q, k, v = (t.clone() for t in project(3))
    lens_t = i32(lens)
    positions = torch.zeros(3, dtype=torch.int32, device="cuda")
    saved = [t.clone() for t in (cache.k_pages.view(torch.uint8), cache.v_pages.view(torch.uint8), cache.k_scales, cache.v_scales)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(q, k, v, lens_t, None, positions)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        qr, o = step(q, k, v, lens_t, None, positions)
    for t, was in zip((cache.k_pages.view(torch.uint8), cache.v_pages.view(torch.uint8), cache.k_scales, cache.v_scales), saved):
        t.copy_(was)
    for _ in range(20):
        lens = [n + 1 for n in lens]
        for t, new in zip((q, k, v), project(3)):
            t.copy_(new)
        lens_t.copy_(torch.tensor(lens, dtype=torch.int32))
        positions.copy_(lens_t - 1)
        graph.replay()
        remember(k, v, lens, [0, 1, 2, 3])
        check(qr, o, lens, [0, 1, 2, 3])
    _nat().check_status(cuda_device)


def test_calls_on_two_streams(cuda_device):
    """Two attentions at once on two streams, each with its own workspace: the same bits as one after the other."""
    P, H, H_kv, D = 64, 16, 2, 128
    lens, news = [4000, 2000, 3000], [1, 1, 1]
    table, starts, pages = batch(lens, news, P)
    cache = _cache(*to_gpu(*make_cache(pages, H_kv, P, D)))
    qs = [torch.randn(3, H, D, device="cuda").half() for _ in range(2)]
    tg, lg = table.cuda(), i32(lens)
    ref = [_attend(q, cache, tg, lg) for q in qs]
    streams = [torch.cuda.Stream() for _ in qs]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    outs = [[], []]
    for _ in range(20):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                outs[i].append(_attend(qs[i], cache, tg, lg))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(o, ref[i]) for o in outs[i])
