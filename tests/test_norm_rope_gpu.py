"""qk_norm_rope on the GPU against its float64 form: forward, backward, strides, positions, streams, graphs.

Bounds: the output is rounded once (half a step of its type) after float32 arithmetic.  A forward value
is a c - b s with a, b = x r w: r is off by less than 12 float32 half steps (a sum of D/8 fused
terms and log2 D partial sums, halved by the root, rsqrt within 2 steps), x r w by 2 more, the rotation
by 3: 32 half steps of |a c| + |b s| hold with room.  Backward: the same factors once more through g and
the mean of g x (a float32 sum of at most D/8 + 7 terms, relative to the sum of magnitudes): 96 half
steps of r (|g| + |x| r^2 mean|g x|).  A weight gradient sums rows: n half steps of the sum of magnitudes
for n rows, plus those of its terms.
"""
import pytest
import torch

from tests.serving_util import (U32, angles, half_step, half_subnormal, norm_rope64, pairs, rotated_size, tables,
                                unpairs)

pytestmark = pytest.mark.gpu
EPS = 1e-6


def _op():
    from attention.rotary.norm_rope import qk_norm_rope
    return qk_norm_rope


def _nat():
    from attention.fused.fused import _native
    return _native()


def make(B, H, H_kv, N, D, dtype, wtype=None, axes=1, seed=0, max_pos=300, device="cuda", fused=True):
    g = torch.Generator(device=device).manual_seed(seed)
    x = (torch.randn(B, N, H + 2 * H_kv, D, device=device, generator=g)
         * (0.1 + 3 * torch.rand(H + 2 * H_kv, 1, device=device, generator=g))).to(dtype)
    q, k = x[:, :, :H].transpose(1, 2), x[:, :, H:H + H_kv].transpose(1, 2)
    if not fused:
        q, k = q.contiguous(), k.contiguous()
    w = [None, None] if wtype is None else [(1 + 0.5 * torch.randn(D, device=device, generator=g)).to(wtype) for _ in range(2)]
    cos, sin = tables(max_pos, D, device)
    sections = None
    if axes > 1:
        half = D // 2
        sections = (half - 3 * (axes - 1),) + (3,) * (axes - 1)
    shape = (B, N) if sections is None else (axes, B, N)
    pos = torch.randint(0, max_pos, shape, device=device, generator=g, dtype=torch.int32)
    dz = [torch.randn(B, h, N, D, device=device, generator=g).to(dtype) for h in (H, H_kv)]
    return q, k, cos, sin, pos, w, sections, dz


def check_forward(out, x, w, c, s, interleaved, what):
    ref = norm_rope64(x, w, c, s, EPS, interleaved)
    size = rotated_size(x, w, c, s, EPS, interleaved)
    tol = half_step(out.dtype) * (ref.abs() + 32 * U32 * size) + 32 * U32 * size + half_subnormal(out.dtype)
    worst = ((out.double() - ref).abs() / tol).max()
    assert float(worst) <= 1.0, (what, float(worst))


def check_backward(dx, dw, x, w, c, s, interleaved, dz, what):
    x64 = x.detach().double()
    a, b = pairs(dz.double(), interleaved)
    dy = unpairs(a * c + b * s, b * c - a * s, interleaved)
    dy_size = unpairs(a.abs() * c.abs() + b.abs() * s.abs(), b.abs() * c.abs() + a.abs() * s.abs(), interleaved)
    if w is None:
        ref, size = dy, dy_size
    else:
        w64 = w.detach().double()
        r = 1 / torch.sqrt((x64 * x64).mean(-1, keepdim=True) + EPS)
        g = dy * w64
        ref = r * (g - x64 * r * r * (g * x64).mean(-1, keepdim=True))
        g_size = dy_size * w64.abs()
        size = r * (g_size + x64.abs() * r * r * (g_size * x64.abs()).mean(-1, keepdim=True))
        rows = x[..., 0].numel()
        dw_ref = (dy * x64 * r).sum((0, 1, 2))
        dw_size = (dy_size * (x64 * r).abs()).sum((0, 1, 2))
        tol = half_step(dw.dtype) * dw_ref.abs() + (rows + 96) * U32 * dw_size * (1 + half_step(dw.dtype)) + half_subnormal(dw.dtype)
        assert dw.dtype == w.dtype
        worst = ((dw.double() - dw_ref).abs() / tol).max()
        assert float(worst) <= 1.0, (what, "dw", float(worst))
    tol = half_step(dx.dtype) * (ref.abs() + 96 * U32 * size) + 96 * U32 * size + half_subnormal(dx.dtype)
    worst = ((dx.double() - ref).abs() / tol).max()
    assert float(worst) <= 1.0, (what, "dx", float(worst))


CASES = [
    (1, 1, 1, 1, 32), (2, 3, 1, 5, 64), (1, 32, 8, 1, 128), (3, 5, 5, 67, 128), (2, 8, 2, 129, 64), (64, 4, 2, 1, 32),
    (1, 7, 7, 33, 32), (2, 32, 8, 200, 128),
]


@pytest.mark.parametrize("shape", CASES, ids=str)
@pytest.mark.parametrize("dtype,wtype", [(torch.bfloat16, torch.bfloat16), (torch.float16, torch.float32),
                                         (torch.bfloat16, None)], ids=["bf16", "fp16-w32", "bf16-rotation"])
@pytest.mark.parametrize("interleaved", [False, True], ids=["halves", "interleaved"])
def test_forward_and_backward(shape, dtype, wtype, interleaved, cuda_device):
    B, H, H_kv, N, D = shape
    for axes in (1, 3):
        q, k, cos, sin, pos, w, sections, dz = make(B, H, H_kv, N, D, dtype, wtype, axes)
        q, k = q.detach().requires_grad_(True), k.detach().requires_grad_(True)
        w = [None if x is None else x.requires_grad_(True) for x in w]
        qo, ko = _op()(q, k, cos, sin, pos, *w, eps=EPS, interleaved=interleaved, sections=sections)
        assert qo.is_contiguous() and ko.is_contiguous() and qo.shape == q.shape and ko.shape == k.shape
        c, s = (x.unsqueeze(1) for x in angles(cos, sin, pos, sections))
        with torch.no_grad():
            check_forward(qo, q, w[0], c, s, interleaved, "q")
            check_forward(ko, k, w[1], c, s, interleaved, "k")
        leaves = [x for x in (q, k, *w) if x is not None]
        grads = torch.autograd.grad((qo, ko), leaves, dz)
        dw = grads[2:] if wtype is not None else (None, None)
        with torch.no_grad():
            check_backward(grads[0], dw[0], q, w[0], c, s, interleaved, dz[0], "q")
            check_backward(grads[1], dw[1], k, w[1], c, s, interleaved, dz[1], "k")
    _nat().check_status(cuda_device)


def test_gradient_against_differences(cuda_device):
    """<dx, u> and <dw, u> of the kernel against central differences of the float64 form.  The step is 2^-13
    on values of size one: the third-order term is below 2^-22 of the terms; the kernel's own error is
    that of check_backward, summed over the entries."""
    q, k, cos, sin, pos, w, sections, dz = make(1, 2, 1, 3, 64, torch.float16, torch.float32, 3, seed=5)
    q = q.detach().requires_grad_(True)
    w0 = w[0].requires_grad_(True)
    qo, _ = _op()(q, None, cos, sin, pos, w0, sections=sections)
    dq, dw = torch.autograd.grad(qo, (q, w0), dz[0])
    c, s = (x.unsqueeze(1) for x in angles(cos, sin, pos, sections))
    g = torch.Generator(device="cuda").manual_seed(9)
    for x, grad, f in ((q, dq, lambda v: norm_rope64(v, w0, c, s, EPS, False)),
                       (w0, dw, lambda v: norm_rope64(q, v, c, s, EPS, False))):
        x64 = x.detach().double()
        for _ in range(4):
            u = torch.randn(x64.shape, device="cuda", generator=g, dtype=torch.float64)
            h = 2.0 ** -13
            with torch.no_grad():
                diff = ((f(x64 + h * u) - f(x64 - h * u)) * dz[0].double()).sum() / (2 * h)
            got = (grad.double() * u).sum()
            size = float((grad.double() * u).abs().sum())
            # half a step of each entry of the gradient (11 bits for dq), float32 sums, and the differences' own error
            tol = size * (2 * half_step(grad.dtype) + 2.0 ** -16) + 2.0 ** -16 * float(dz[0].double().abs().sum())
            assert abs(float(got - diff)) <= tol, (float(got), float(diff), tol)


def test_rows_of_zeros_and_extremes(cuda_device):
    """A row of zeros stays zero (eps keeps the root finite); NaN and infinities stay in their own rows."""
    q, k, cos, sin, pos, w, _, _ = make(1, 4, 2, 3, 64, torch.bfloat16, torch.bfloat16, fused=False)
    clean = _op()(q, k, cos, sin, pos, *w)
    q, k = q.clone(), k.clone()
    q[0, 0, 0] = 0
    q[0, 1, 1, 5] = float("nan")
    k[0, 1, 2, 3] = float("inf")
    qo, ko = _op()(q, k, cos, sin, pos, *w)
    assert bool((qo[0, 0, 0] == 0).all())
    assert bool(qo[0, 1, 1].isnan().all()) and bool(ko[0, 1, 2].isnan().any())
    for got, ref, bad in ((qo, clean[0], [(0, 0), (1, 1)]), (ko, clean[1], [(1, 2)])):
        keep = torch.ones(got.shape[1:3], dtype=torch.bool)
        for h, n in bad:
            keep[h, n] = False
        assert torch.equal(got[0, keep], ref[0, keep])


def test_far_more_key_heads_than_query_heads(cuda_device):
    """The backward blocks are shared out by heads: the queries keep some however few heads they have."""
    q, k, cos, sin, pos, w, _, dz = make(1, 1, 400, 3, 32, torch.float16, torch.float32)
    leaves = [x.detach().requires_grad_(True) for x in (q, k, *w)]
    out = _op()(leaves[0], leaves[1], cos, sin, pos, leaves[2], leaves[3])
    grads = torch.autograd.grad(out, leaves, dz)
    c, s = (x.unsqueeze(1) for x in angles(cos, sin, pos, None))
    with torch.no_grad():
        check_backward(grads[0], grads[2], q, w[0], c, s, False, dz[0], "q")
        check_backward(grads[1], grads[3], k, w[1], c, s, False, dz[1], "k")


@pytest.mark.parametrize("N", [0, 1])
def test_lengths_zero_and_one(N, cuda_device):
    q, k, cos, sin, pos, w, _, _ = make(2, 3, 1, N, 64, torch.float16, torch.float32)
    q, w0 = q.detach().requires_grad_(True), w[0].requires_grad_(True)
    qo, ko = _op()(q, k, cos, sin, pos, w0, w[1])
    assert qo.shape == (2, 3, N, 64) and ko.shape == (2, 1, N, 64)
    dq, dw = torch.autograd.grad(qo.sum(), (q, w0))
    assert dq.shape == q.shape and dw.shape == w0.shape
    if N == 0:
        assert bool((dw == 0).all())


def test_positions_strides_and_alignment(cuda_device):
    """Positions as [N], [B, N], expanded, int64 and None; q odd-aligned, expanded over heads, head-major."""
    B, H, H_kv, N, D = 3, 4, 2, 9, 64
    q, k, cos, sin, pos, w, _, _ = make(B, H, H_kv, N, D, torch.bfloat16, torch.bfloat16)
    ref = _op()(q, k, cos, sin, pos, *w)
    for p in (pos.long(), pos.t().contiguous().t(), torch.stack((pos, pos), -1)[..., 0]):
        got = _op()(q, k, cos, sin, p, *w)
        assert torch.equal(got[0], ref[0]) and torch.equal(got[1], ref[1])
    ar = torch.arange(N, device="cuda", dtype=torch.int32)
    base = _op()(q, k, cos, sin, None, *w)
    for p in (ar, ar.long(), ar.expand(B, N)):
        got = _op()(q, k, cos, sin, p, *w)
        assert torch.equal(got[0], base[0]) and torch.equal(got[1], base[1])
    for make_q in (lambda x: x.contiguous(),
                   lambda x: torch.empty(x.numel() + 3, dtype=x.dtype, device="cuda")[3:].view(x.shape).copy_(x),
                   lambda x: torch.empty(B, H, N, D + 4, dtype=x.dtype, device="cuda")[..., 2:D + 2].copy_(x),
                   lambda x: torch.empty(D, B, H, N, dtype=x.dtype, device="cuda").permute(1, 2, 3, 0).copy_(x)):
        got = _op()(make_q(q), k, cos, sin, pos, *w)
        assert torch.equal(got[0], ref[0])
    wide = q[:, :1].expand(B, H, N, D)
    got = _op()(wide, None, cos, sin, pos, w[0])
    assert got[1] is None and all(torch.equal(got[0][:, h], ref[0][:, 0]) for h in range(H))
    odd_w = torch.empty(D + 1, dtype=torch.bfloat16, device="cuda")[1:].copy_(w[0])
    assert torch.equal(_op()(q, k, cos, sin, pos, odd_w, w[1])[0], ref[0])


def test_broadcast_and_shared_inputs_get_summed_gradients(cuda_device):
    """k expanded over heads and one weight used for both q and k: autograd adds the parts up."""
    q, _, cos, sin, pos, w, _, dz = make(2, 4, 4, 6, 64, torch.float16, torch.float32)
    base = torch.randn(2, 1, 6, 64, device="cuda").half().requires_grad_(True)
    w0 = w[0].requires_grad_(True)
    qo, ko = _op()(q, base.expand(2, 4, 6, 64), cos, sin, pos, w0, w0)
    db, dw = torch.autograd.grad((qo, ko), (base, w0), (dz[0], dz[1]))
    c, s = (x.unsqueeze(1) for x in angles(cos, sin, pos, None))
    b64 = base.detach().double().requires_grad_(True)
    w64 = w0.detach().double().requires_grad_(True)
    f = (norm_rope64(q, w64, c, s, EPS, False) * dz[0].double()).sum() \
        + (norm_rope64(b64.expand(2, 4, 6, 64), w64, c, s, EPS, False) * dz[1].double()).sum()
    rb, rw = torch.autograd.grad(f, (b64, w64))
    # four heads' fp16 gradients are added in fp16 (expand's backward): three more roundings of partial sums
    assert float((db.double() - rb).abs().max()) <= 8 * half_step(torch.float16) * float(rb.abs().max()) * 4
    assert float((dw.double() - rw).abs().max()) <= 2.0 ** -16 * float(rw.abs().max()) * 8


def test_partial_gradients_and_unused_outputs(cuda_device):
    q, k, cos, sin, pos, w, _, dz = make(1, 2, 2, 5, 32, torch.float16, torch.float16)
    k1 = k.detach().requires_grad_(True)
    qo, ko = _op()(q, k1, cos, sin, pos, *w)
    both = torch.autograd.grad(ko, k1, dz[1], retain_graph=True)[0]
    assert torch.equal(both, torch.autograd.grad((qo, ko), k1, (dz[0], dz[1]))[0])
    w1 = w[1].requires_grad_(True)
    _, ko = _op()(q, k, cos, sin, pos, w[0], w1)
    assert torch.autograd.grad(ko, w1, dz[1])[0].shape == w1.shape


def test_same_bits_every_time_and_many_blocks(cuda_device):
    """A problem with more units than backward blocks; two runs give the same bits."""
    q, k, cos, sin, pos, w, _, dz = make(4, 32, 8, 700, 128, torch.bfloat16, torch.float32, max_pos=700)
    leaves = [x.detach().requires_grad_(True) for x in (q, k, *w)]
    runs = []
    for _ in range(2):
        out = _op()(leaves[0], leaves[1], cos, sin, pos, leaves[2], leaves[3])
        runs.append((*out, *torch.autograd.grad(out, leaves, dz)))
    assert all(torch.equal(a, b) for a, b in zip(*runs))
    c, s = (x.unsqueeze(1) for x in angles(cos, sin, pos, None))
    with torch.no_grad():
        check_forward(runs[0][0], q, w[0], c, s, False, "q")
        check_backward(runs[0][2], runs[0][4], q, w[0], c, s, False, dz[0], "q")
        check_backward(runs[0][3], runs[0][5], k, w[1], c, s, False, dz[1], "k")


def test_streams_and_graphs(cuda_device):
    """Another stream than the inputs', and a captured forward and backward replayed on new inputs."""
    q, k, cos, sin, pos, w, _, dz = make(2, 4, 2, 40, 64, torch.bfloat16, torch.bfloat16, fused=False)
    ref = _op()(q, k, cos, sin, pos, *w)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = _op()(q, k, cos, sin, pos, *w)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got[0], ref[0]) and torch.equal(got[1], ref[1])
    leaves = [x.detach().clone().requires_grad_(True) for x in (q, k, *w)]

    def step():
        out = _op()(leaves[0], leaves[1], cos, sin, pos, leaves[2], leaves[3])
        return (*out, *torch.autograd.grad(out, leaves, dz))

    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step()
    with torch.no_grad():
        leaves[0].mul_(-0.5)
        pos.copy_((pos + 7) % 300)
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(outs, step()))


def test_positions_outside_the_table_are_reported(cuda_device):
    """The kernel stays inside the tables, records code 111, and works again after the reset."""
    nat = _nat()
    q, k, cos, sin, pos, w, _, _ = make(1, 2, 1, 8, 64, torch.bfloat16, torch.bfloat16)
    for bad in (-1, 300, 1 << 30):
        p = pos.clone()
        p[0, 3] = bad
        _op()(q, k, cos, sin, p, *w)
        with pytest.raises(nat.KernelError, match="outside its table"):
            nat.check_status(cuda_device)
    ref = _op()(q, k, cos, sin, pos, *w)
    nat.check_status(cuda_device)
    c, s = (x.unsqueeze(1) for x in angles(cos, sin, pos, None))
    check_forward(ref[0], q, w[0], c, s, False, "q")


def test_into_causal_attention(cuda_device):
    """Norm + rotation, then fused_attention_autograd (GQA): outputs and all gradients against float64."""
    from attention.backward.fused_backward import fused_attention_autograd
    B, H, H_kv, N, D = 1, 4, 2, 128, 64
    q, k, cos, sin, pos, w, _, _ = make(B, H, H_kv, N, D, torch.float16, torch.float32, max_pos=N)
    g = torch.Generator(device="cuda").manual_seed(3)
    v = torch.randn(B, H_kv, N, D, device="cuda", generator=g).half()
    do = torch.randn(B, H, N, D, device="cuda", generator=g).half()
    leaves = [x.detach().requires_grad_(True) for x in (q, k, v, *w)]
    qo, ko = _op()(leaves[0], leaves[1], cos, sin, None, leaves[3], leaves[4])
    o = fused_attention_autograd(qo, ko, leaves[2])
    grads = torch.autograd.grad(o, leaves, do)
    l64 = [x.detach().double().requires_grad_(True) for x in leaves]
    c, s = angles(cos, sin, torch.arange(N, device="cuda"), None)
    q64, k64 = norm_rope64(l64[0], l64[3], c, s, EPS, False), norm_rope64(l64[1], l64[4], c, s, EPS, False)
    a = (q64 @ k64.repeat_interleave(2, 1).transpose(-1, -2)) / D ** 0.5
    a = a.masked_fill(torch.ones(N, N, dtype=torch.bool, device="cuda").triu(1), float("-inf"))
    o64 = torch.softmax(a, -1) @ l64[2].repeat_interleave(2, 1)
    ref = torch.autograd.grad(o64, l64, do.double())
    # the framework's rule for attention outputs and gradients (2e-2 absolute and relative)
    assert float(((o.double() - o64).abs() / (2e-2 + 2e-2 * o64.abs())).max()) <= 1
    for got, r in zip(grads[:3], ref[:3]):
        scale = max(1.0, float(r.abs().max()))  # q and k of some heads are small: their gradients are large
        assert float((got.double() - r).abs().max()) <= 2e-2 * scale
    for got, r in zip(grads[3:], ref[3:]):
        assert float((got.double() - r).abs().max()) <= 2e-2 * max(1.0, float(r.abs().max()))
