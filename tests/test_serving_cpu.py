"""Refusals and host-side rules of qk_norm_rope, append_kv, paged_attention and PagedKVCache, without a GPU."""
import ctypes
import os
import re
import struct
import subprocess

import pytest
import torch

from attention.paged.cache import PAGE_DTYPE, PagedKVCache, append_kv
from attention.paged.paged_attention import paged_attention
from attention.rotary.norm_rope import qk_norm_rope, rope_tables

REPO = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def _nat():
    from attention.fused.fused import _native
    return _native()


# The structs of include/fa_sm100.h, field by field.
NORM_ROPE_ARGS = struct.Struct("@16P14q15if")
APPEND_ARGS = struct.Struct("@13P6qd18i")
PAGED_ARGS = struct.Struct("@11P5q10if4x")


def half(*shape, dtype=torch.float16):
    return torch.zeros(shape, dtype=dtype)


def rope_args(**kw):
    a = dict(q=half(2, 4, 8, 64), k=half(2, 2, 8, 64), cos=torch.zeros(32, 32), sin=torch.zeros(32, 32), positions=None,
             q_weight=None, k_weight=None, sections=None)
    a.update(kw)
    return a


@pytest.mark.parametrize("kw,error,match", [
    (dict(q=half(2, 4, 8, 64, dtype=torch.float32)), TypeError, "float16"),
    (dict(k=half(2, 2, 8, 64, dtype=torch.bfloat16)), TypeError, "float16"),
    (dict(q=half(4, 8, 64)), ValueError, "B, H, N, D"),
    (dict(k=half(2, 2, 9, 64)), ValueError, "B, H, N, D"),
    (dict(k=half(1, 2, 8, 64)), ValueError, "B, H, N, D"),
    (dict(k=half(2, 0, 8, 64)), ValueError, "B, H, N, D"),
    (dict(q=half(2, 4, 8, 48), k=None, cos=torch.zeros(32, 24), sin=torch.zeros(32, 24)), ValueError, "head dim"),
    (dict(cos=torch.zeros(32, 32, dtype=torch.float64)), TypeError, "float32"),
    (dict(cos=torch.zeros(32, 64)), ValueError, "max_pos"),
    (dict(cos=torch.zeros(31, 32)), ValueError, "max_pos"),
    (dict(cos=torch.zeros(0, 32), sin=torch.zeros(0, 32)), ValueError, "max_pos"),
    (dict(positions=torch.zeros(8)), TypeError, "int32 or int64"),
    (dict(positions=torch.zeros(9, dtype=torch.int32)), ValueError, "positions"),
    (dict(positions=torch.zeros(3, 2, 8, dtype=torch.int32)), ValueError, "positions"),
    (dict(sections=(16, 8, 8)), ValueError, "positions"),
    (dict(sections=(16, 8, 4), positions=torch.zeros(3, 8, dtype=torch.int32)), ValueError, "sections"),
    (dict(sections=(8, 8, 8, 4, 4), positions=torch.zeros(5, 8, dtype=torch.int32)), ValueError, "sections"),
    (dict(sections=(33, -1), positions=torch.zeros(2, 8, dtype=torch.int32)), ValueError, "sections"),
    (dict(sections=(16, 16), positions=torch.zeros(3, 8, dtype=torch.int32)), ValueError, "positions"),
    (dict(q_weight=torch.ones(64, dtype=torch.bfloat16)), TypeError, "q_weight"),
    (dict(q_weight=torch.ones(32)), ValueError, "q_weight"),
    (dict(q_weight=torch.ones(64), k_weight=half(64)), TypeError, "share"),
    (dict(k=None, k_weight=torch.ones(64)), ValueError, "without k"),
    (dict(), ValueError, "CUDA device"),
])
def test_norm_rope_refuses(kw, error, match):
    with pytest.raises(error, match=match):
        qk_norm_rope(**rope_args(**kw))


def cache_tensors(pages=4, H_kv=2, P=16, D=64):
    return [torch.zeros(pages, H_kv, P, D, dtype=torch.uint8).view(PAGE_DTYPE) for _ in range(2)] + \
        [torch.zeros(pages, H_kv) for _ in range(2)]


def test_cache_refuses():
    good = cache_tensors()
    c = PagedKVCache(*good)
    assert (c.num_pages, c.num_kv_heads, c.page_size, c.head_dim) == (4, 2, 16, 64)
    for i, bad, error in ((0, good[0].view(torch.uint8), TypeError), (2, good[2].half(), TypeError),
                          (1, good[1][:3], ValueError), (3, good[3][:, :1], ValueError),
                          (0, good[0].view(torch.uint8).transpose(1, 2).contiguous().view(PAGE_DTYPE).transpose(1, 2), ValueError)):
        t = list(good)
        t[i] = bad
        with pytest.raises(error):
            PagedKVCache(*t)
    for kw in (dict(P=8), dict(P=48), dict(D=96), dict(pages=0)):
        with pytest.raises(ValueError):
            PagedKVCache(*cache_tensors(**kw))
    e = PagedKVCache.empty(3, 2, 128, 32, device="cpu")
    assert e.k_pages.shape == (3, 2, 32, 128) and e.v_scales.shape == (3, 2)


def step_args(**kw):
    a = dict(cache=PagedKVCache(*cache_tensors()), block_table=torch.zeros(3, 2, dtype=torch.int32),
             seq_lens=torch.ones(3, dtype=torch.int32), offsets=None)
    a.update(kw)
    return a


BAD_TABLES = [
    (dict(block_table=torch.zeros(3, 2, dtype=torch.int64)), TypeError, "block_table"),
    (dict(block_table=torch.zeros(2, 2, dtype=torch.int32)), ValueError, "block_table"),
    (dict(block_table=torch.zeros(3, 0, dtype=torch.int32)), ValueError, "block_table"),
    (dict(block_table=torch.zeros(2, 3, dtype=torch.int32).t()), ValueError, "block_table"),
    (dict(seq_lens=torch.ones((), dtype=torch.int32)), ValueError, "seq_lens"),
    (dict(seq_lens=torch.ones(3)), TypeError, "seq_lens"),
    (dict(seq_lens=torch.ones(3, 1, dtype=torch.int32)), ValueError, "seq_lens"),
    (dict(seq_lens=torch.ones(6, dtype=torch.int32)[::2]), ValueError, "seq_lens"),
    (dict(offsets=torch.zeros(3, dtype=torch.int32)), ValueError, "offsets"),
    (dict(offsets=torch.zeros(4, dtype=torch.int64)), TypeError, "offsets"),
    (dict(seq_lens=torch.ones(2, dtype=torch.int32), block_table=torch.zeros(2, 2, dtype=torch.int32)), ValueError, "one token"),
    (dict(), ValueError, "CUDA device"),
]


@pytest.mark.parametrize("kw,error,match", BAD_TABLES + [
    (dict(k=half(3, 2, 64, dtype=torch.float32)), TypeError, "float16"),
    (dict(v=half(3, 2, 64, dtype=torch.bfloat16)), TypeError, "float16"),
    (dict(k=half(3, 4, 64), v=half(3, 4, 64)), ValueError, "H_kv"),
    (dict(v=half(2, 2, 64)), ValueError, "H_kv"),
    (dict(cos=torch.zeros(9, 32)), ValueError, "cos and sin"),
    (dict(positions=torch.zeros(3, dtype=torch.int32)), ValueError, "cos and sin"),
    (dict(cos=torch.zeros(9, 32), sin=torch.zeros(9, 32), positions=torch.zeros(4, dtype=torch.int32)), ValueError, "positions"),
    (dict(cos=torch.zeros(9, 32), sin=torch.zeros(9, 32), sections=(16, 16)), ValueError, "positions"),
    (dict(k_weight=torch.ones(32)), ValueError, "k_weight"),
    (dict(k_weight=torch.ones(64).requires_grad_(True)), RuntimeError, "no backward"),
    (dict(k=half(3, 2, 64).requires_grad_(True)), RuntimeError, "no backward"),
])
def test_append_refuses(kw, error, match):
    a = dict(k=half(3, 2, 64), v=half(3, 2, 64))
    a.update(kw)
    with pytest.raises(error, match=match):
        append_kv(**step_args(**a))


def test_append_refuses_keys_and_values_in_one_place():
    """Attention may read a cache whose keys are its values; an append would write both."""
    kp, vp, ks, vs = cache_tensors()
    both = torch.zeros(2 * kp.numel(), dtype=torch.uint8).view(kp.dtype)
    for t in ((kp, kp, ks, vs), (kp, vp, ks, ks),
              (both[:kp.numel()].view(kp.shape), both[kp.numel() - 64:-64].view(kp.shape), ks, vs)):
        with pytest.raises(ValueError, match="share memory"):
            append_kv(PagedKVCache(*t), half(3, 2, 64), half(3, 2, 64), torch.zeros(3, 2, dtype=torch.int32),
                      torch.ones(3, dtype=torch.int32))


@pytest.mark.parametrize("kw,error,match", BAD_TABLES + [
    (dict(q=half(3, 4, 64, dtype=torch.float32)), TypeError, "float16"),
    (dict(q=half(3, 3, 64)), ValueError, "multiple of H_kv"),
    (dict(q=half(3, 4, 32)), ValueError, "multiple of H_kv"),
    (dict(q=half(3, 64)), ValueError, "multiple of H_kv"),
    (dict(scale=0.0), ValueError, "scale"),
    (dict(scale=float("nan")), ValueError, "scale"),
    (dict(scale=float("inf")), ValueError, "scale"),
    (dict(out=half(3, 2, 64)), ValueError, "out must be like q"),
    (dict(out=half(3, 4, 64, dtype=torch.bfloat16)), ValueError, "out must be like q"),
    (dict(q=half(3, 4, 64).requires_grad_(True)), RuntimeError, "no backward"),
])
def test_attention_refuses(kw, error, match):
    a = dict(q=half(3, 4, 64))
    a.update(kw)
    with pytest.raises(error, match=match):
        paged_attention(**step_args(**a))


def test_rope_tables():
    cos, sin = rope_tables(50, 64)
    assert cos.shape == sin.shape == (50, 32) and cos.dtype == torch.float32
    a = 37 * 10000.0 ** (-2 * 5 / 64)
    assert abs(float(cos[37, 5]) - __import__("math").cos(a)) <= 2.0 ** -24


def test_packed_arguments_match_the_header(tmp_path):
    """The formats that these tests pack with have the size and offsets that a C compiler gives the header's structs."""
    fields = {"fa_norm_rope_args": (NORM_ROPE_ARGS, ["q_stride", "B", "eps"], [16 * 8, 16 * 8 + 14 * 8, 16 * 8 + 14 * 8 + 15 * 4]),
              "fa_append_args": (APPEND_ARGS, ["k_stride", "eps", "T"], [13 * 8, 19 * 8, 20 * 8]),
              "fa_paged_args": (PAGED_ARGS, ["q_stride", "T", "scale"], [11 * 8, 16 * 8, 16 * 8 + 10 * 4])}
    src = "#include <stdio.h>\n#include <stddef.h>\n#include \"fa_sm100.h\"\nint main(void) {\n"
    for name, (_, members, _) in fields.items():
        src += f'printf("%zu", sizeof(struct {name}));\n'
        src += "".join(f'printf(" %zu", offsetof(struct {name}, {m}));\n' for m in members) + 'printf("\\n");\n'
    src += "return 0; }\n"
    c = tmp_path / "sizes.c"
    c.write_text(src)
    exe = tmp_path / "sizes"
    subprocess.run(["gcc", "-I", os.path.join(REPO, "include"), str(c), "-o", str(exe)], check=True)
    lines = subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout.splitlines()
    for line, (packer, _, offsets) in zip(lines, fields.values()):
        assert [int(x) for x in line.split()] == [packer.size] + offsets
    text = open(os.path.join(REPO, "include", "fa_sm100.h")).read()
    assert set(re.findall(r"struct (fa_\w+_args) \{", text)) == set(fields)


def _rc(name, packed):
    return getattr(_nat().load(), name)(packed, 256, None)


NR = dict(q=256, k=512, qw=0, kw=0, cos=256, sin=256, pos=0, qo=256, ko=256, dqo=0, dko=0, dq=0, dk=0, dqw=0, dkw=0, ws=0,
          st=[64] * 14, B=1, H=4, H_kv=2, N=8, D=64, dtype=0, wdtype=0, max_pos=16, axes=1, s0=0, s1=0, s2=0, s3=0,
          pos64=0, inter=0, eps=1e-6)
AP = dict(k=256, v=256, kp=256, vp=1 << 20, ks=256, vs=1 << 20, table=256, lens=256, offsets=0, cos=0, sin=0, pos=0, kw=0,
          st=[64] * 6, eps=1e-6, T=3, B=3, width=2, pages=4, H_kv=2, P=16, D=64, dtype=0, wdtype=0, max_pos=0, axes=1,
          s0=0, s1=0, s2=0, s3=0, pos64=0, inter=0, reserved=0)
PA = dict(q=256, kp=256, vp=256, ks=256, vs=256, table=256, lens=256, offsets=0, out=256, lse=0, ws=256, st=[64] * 5,
          T=3, B=3, width=2, pages=4, H=4, H_kv=2, P=16, D=64, dtype=0, clear=0, scale=0.125)


def _packed(packer, base, **kw):
    values = []
    for v in {**base, **kw}.values():
        values += v if isinstance(v, list) else [v]
    return packer.pack(*values)


@pytest.mark.parametrize("kw,code", [
    (dict(q=0), 1), (dict(cos=0), 1), (dict(B=0), 1), (dict(N=0), 1), (dict(qo=0), 1), (dict(ko=0), 1), (dict(k=0), 1),
    (dict(H_kv=0), 1), (dict(max_pos=0), 1), (dict(axes=0), 1), (dict(s0=1), 1), (dict(axes=3, s1=9, s2=4), 1),
    (dict(axes=2, s1=33), 1), (dict(axes=5), 2), (dict(D=48), 2), (dict(dtype=2), 2), (dict(qw=256, wdtype=1), 2),
    (dict(B=1 << 20, N=1 << 12), 2), (dict(q=264), 3), (dict(ko=264), 3), (dict(qw=264), 3), (dict(cos=264), 3),
    (dict(pos=258), 3), (dict(pos=260, pos64=1), 3), (dict(st=[12] + [64] * 13), 3)])
def test_norm_rope_c_refusals(kw, code):
    assert _rc("fa_norm_rope_fwd", _packed(NORM_ROPE_ARGS, NR, **kw)) == code


@pytest.mark.parametrize("kw,code", [
    (dict(), 1), (dict(dqo=256, dq=256, dko=256), 1), (dict(dqo=256, dq=256, dko=256, dk=256, dqw=256), 1),
    (dict(dqo=256, dq=256, dko=256, dk=256, qw=256), 1), (dict(dqo=264, dq=256, dko=256, dk=256), 3)])
def test_norm_rope_backward_c_refusals(kw, code):
    assert _rc("fa_norm_rope_bwd", _packed(NORM_ROPE_ARGS, NR, **kw)) == code


CACHE_CODES = [
    (dict(kp=0), 1), (dict(vs=0), 1), (dict(table=0), 1), (dict(lens=0), 1), (dict(B=0), 1), (dict(T=0), 1),
    (dict(T=4), 1), (dict(width=0), 1), (dict(pages=0), 1), (dict(D=96), 2), (dict(P=8), 2), (dict(P=24), 2),
    (dict(dtype=2), 2), (dict(width=1 << 27), 2), (dict(kp=264), 3), (dict(table=258), 3), (dict(st=None), 3)]


@pytest.mark.parametrize("kw,code", CACHE_CODES + [
    (dict(k=0), 1), (dict(cos=256), 1), (dict(cos=256, sin=256), 1), (dict(cos=256, sin=256, max_pos=4, axes=2, s1=8), 1),
    (dict(kw=256, wdtype=1), 2), (dict(kw=264), 3), (dict(v=260), 3), (dict(cos=264, sin=256, max_pos=4), 3),
    (dict(H_kv=32768), 2), (dict(vp=256), 1), (dict(vp=256 + 4 * 2 * 16 * 64 - 16), 1), (dict(vs=256 + 4), 1)])
def test_append_c_refusals(kw, code):
    if kw.get("st", 0) is None:
        kw = dict(st=[4] + [64] * 5)
    assert _rc("fa_append_kv", _packed(APPEND_ARGS, AP, **kw)) == code


@pytest.mark.parametrize("kw,code", CACHE_CODES + [
    (dict(q=0), 1), (dict(out=0), 1), (dict(ws=0), 1), (dict(H=0), 1), (dict(H=3), 1), (dict(scale=0.0), 1),
    (dict(scale=float("inf")), 1), (dict(scale=float("nan")), 1), (dict(ws=264), 3), (dict(lse=258), 3)])
def test_attention_c_refusals(kw, code):
    if kw.get("st", 0) is None:
        kw = dict(st=[4] + [64] * 4)
    assert _rc("fa_paged_attention", _packed(PAGED_ARGS, PA, **kw)) == code


def test_null_arguments_and_no_device():
    lib = _nat().load()
    for name in ("fa_norm_rope_fwd", "fa_norm_rope_bwd", "fa_append_kv", "fa_paged_attention"):
        assert getattr(lib, name)(None, 256, None) == 1
    if not torch.cuda.is_available():
        for name, packed in (("fa_norm_rope_fwd", _packed(NORM_ROPE_ARGS, NR)), ("fa_append_kv", _packed(APPEND_ARGS, AP)),
                             ("fa_paged_attention", _packed(PAGED_ARGS, PA))):
            assert _rc(name, packed) in (4, 5, 6)
            assert getattr(lib, name)(packed, None, None) == 1


def test_modules_load_by_path():
    """The files can be imported by path, like the other kernel files."""
    import importlib.util
    base = os.path.join(REPO, "fused-attention_b200", "attention")
    for rel, name in (("rotary/norm_rope.py", "qk_norm_rope"), ("paged/cache.py", "append_kv"),
                      ("paged/paged_attention.py", "paged_attention")):
        spec = importlib.util.spec_from_file_location("by_path_" + name, os.path.join(base, rel))
        mod = importlib.util.module_from_spec(spec)
        spec.loader.exec_module(mod)
        assert callable(getattr(mod, name))
    assert ctypes.sizeof(ctypes.c_void_p) == 8
