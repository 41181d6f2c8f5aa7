"""qk_norm_rope where eps or the size of the elements leaves the ordinary range, against its float64 form.

Bounds are those of test_norm_rope_gpu.py."""
import pytest
import torch

from tests.serving_util import U32, angles, half_step, half_subnormal, norm_rope64, pairs, rotated_size, unpairs
from tests.test_norm_rope_gpu import _nat, _op, make

pytestmark = pytest.mark.gpu


def forward_ok(out, x, w, c, s, eps, interleaved):
    ref = norm_rope64(x, w, c, s, eps, interleaved)
    size = rotated_size(x, w, c, s, eps, interleaved)
    tol = half_step(out.dtype) * (ref.abs() + 32 * U32 * size) + 32 * U32 * size + half_subnormal(out.dtype)
    worst = float(((out.double() - ref).abs() / tol).max())
    assert worst <= 1.0, worst


def backward_ok(dx, dw, x, w, c, s, eps, interleaved, dz):
    x64, w64 = x.detach().double(), w.detach().double()
    a, b = pairs(dz.double(), interleaved)
    dy = unpairs(a * c + b * s, b * c - a * s, interleaved)
    dy_size = unpairs(a.abs() * c.abs() + b.abs() * s.abs(), b.abs() * c.abs() + a.abs() * s.abs(), interleaved)
    r = 1 / torch.sqrt((x64 * x64).mean(-1, keepdim=True) + eps)
    xn = x64 * r
    g, g_size = dy * w64, dy_size * w64.abs()
    ref = r * (g - xn * (g * xn).mean(-1, keepdim=True))
    size = r * (g_size + xn.abs() * (g_size * xn.abs()).mean(-1, keepdim=True))
    rows = x[..., 0].numel()
    dw_ref, dw_size = (dy * xn).sum((0, 1, 2)), (dy_size * xn.abs()).sum((0, 1, 2))
    tol = half_step(dw.dtype) * dw_ref.abs() + (rows + 96) * U32 * dw_size * (1 + half_step(dw.dtype)) + half_subnormal(dw.dtype)
    worst = float(((dw.double() - dw_ref).abs() / tol).max())
    assert worst <= 1.0, ("dw", worst)
    most = torch.finfo(dx.dtype).max
    held = ref.abs() < most / 2  # a gradient of 1/|x| may be too large for the type
    tol = half_step(dx.dtype) * (ref.abs() + 96 * U32 * size) + 96 * U32 * size + half_subnormal(dx.dtype)
    worst = float(((dx.double() - ref).abs() / tol)[held].max())
    assert worst <= 1.0, ("dx", worst)


def both_ways(q, k, cos, sin, pos, w, sections, dz, eps, interleaved):
    q, k, *w = (x.detach().requires_grad_(True) for x in (q, k, *w))
    out = _op()(q, k, cos, sin, pos, *w, eps=eps, interleaved=interleaved, sections=sections)
    grads = torch.autograd.grad(out, (q, k, *w), dz)
    _nat().check_status(q.device)
    c, s = (x.unsqueeze(1) for x in angles(cos, sin, pos, sections))
    with torch.no_grad():
        for o, x, wt, dx, dw, z in zip(out, (q, k), w, grads[:2], grads[2:], dz):
            forward_ok(o, x, wt, c, s, eps, interleaved)
            backward_ok(dx, dw, x, wt, c, s, eps, interleaved, z)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=["bf16", "fp16"])
@pytest.mark.parametrize("shape", [(1, 1, 1, 1, 32), (2, 3, 1, 5, 64), (1, 7, 5, 33, 128)], ids=str)
def test_eps_of_zero(dtype, shape, cuda_device):
    """Odd numbers of heads and tokens: the places of a block that have no row have no part in dw."""
    case = make(*shape, dtype, torch.float32)
    both_ways(*case, 0.0, False)


@pytest.mark.parametrize("interleaved", [False, True], ids=["halves", "interleaved"])
@pytest.mark.parametrize("eps", [1e-6, 0.0])
@pytest.mark.parametrize("shape", [(2, 3, 1, 5, 64), (1, 7, 5, 33, 128), (3, 2, 2, 40, 32)], ids=str)
def test_rows_whose_squares_leave_float32(shape, eps, interleaved, cuda_device):
    """bf16 rows of all sizes from 2^-60 (eps 0) or 1 to 2^110, rows of ordinary size between them: as in float64, and the
    ordinary rows' bits do not depend on their neighbours.  (append_kv squares in float64: both norms agree.)"""
    q, k, cos, sin, pos, w, sections, dz = make(*shape, torch.bfloat16, torch.float32)
    plain = _op()(q, k, cos, sin, pos, *w, eps=eps, interleaved=interleaved)
    g = torch.Generator(device="cuda").manual_seed(4)
    powers = torch.tensor([0, 0, 0, 58, 61, 64, 90, 110] + ([-40, -50, -60] if eps == 0 else [0, 10, 20]), device="cuda")
    parts = []
    for x in (q, k):
        p = powers[torch.randint(0, len(powers), x.shape[:3], device="cuda", generator=g)]
        parts.append((p, (x.double() * torch.exp2(p.double())[..., None]).bfloat16()))
    (pq, q2), (pk, k2) = parts
    both_ways(q2, k2, cos, sin, pos, w, sections, dz, eps, interleaved)
    got = _op()(q2, k2, cos, sin, pos, *w, eps=eps, interleaved=interleaved)
    for a, b, p in ((got[0], plain[0], pq), (got[1], plain[1], pk)):
        assert torch.equal(a[p == 0], b[p == 0])
