"""Operators around attention, as they are measured: what a model does with queries and keys before
attention (per-head RMS norm and rotary positions, forward and backward), how new keys and values
enter a paged cache held in e4m3 with one scale for each page and K/V head, and attention over that
cache, from one token per sequence (decode) to chunks of tokens (prefill behind a prompt already there).

`own` false computes the operators with elementary torch operations in 32 bits (64 where the value next to
a rounding border is what comes out); `own` true calls this repository's kernels.
"""
import math
import random
import sys

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
E4M3 = torch.float8_e4m3fn
E4M3_MAX = 448.0
EPS = 1e-6


# ------------------------------------------------------------------------------------------- cases
def listed():
    return [
        # A decode step of 64 sequences: one new token each, 32 query and 8 K/V heads.
        dict(name="norm-rope decode 64", op="norm_rope", B=64, N=1, H=32, H_kv=8, D=128, dtype="bf16",
             wtype="bf16", axes=1, interleaved=False, max_pos=8192, backward=False),
        # A training step's q and k, forward and backward, at the framework's batch of 4.
        dict(name="norm-rope train 4x2048", op="norm_rope", B=4, N=2048, H=32, H_kv=8, D=128, dtype="bf16",
             wtype="bf16", axes=1, interleaved=False, max_pos=2048, backward=True),
        # Video tokens (time, height, width), an odd count of them, narrow heads, weights in 32 bits.
        dict(name="norm-rope video 2x1955", op="norm_rope", B=2, N=1955, H=16, H_kv=16, D=64, dtype="fp16",
             wtype="fp32", axes=3, interleaved=True, max_pos=128, backward=True),
        # The longest prompt that the framework's own limits allow, forward only.
        dict(name="norm-rope prefill 32768", op="norm_rope", B=1, N=32768, H=32, H_kv=8, D=128, dtype="bf16",
             wtype="bf16", axes=1, interleaved=False, max_pos=32768, backward=False),
        # The same decode step's keys and values into their pages.
        dict(name="append decode 64", op="append", B=64, n=1, L=8192, H_kv=8, D=128, page=64, dtype="bf16",
             norm=True, axes=1, interleaved=False, ragged=True),
        # Prompts of different lengths appended in one call, behind a few tokens that are there.
        dict(name="append ragged 5x2047", op="append", B=5, n=2047, L=4111, H_kv=8, D=128, page=64, dtype="bf16",
             norm=True, axes=1, interleaved=False, ragged=True),
        # One long prompt, small pages, narrow heads, rotation without a norm.
        dict(name="append prefill 32768", op="append", B=1, n=32768, L=32768, H_kv=8, D=64, page=16, dtype="fp16",
             norm=False, axes=1, interleaved=True, ragged=False),
        # One sequence with a short history: latency counts.
        dict(name="attend 1x1000", op="attend", B=1, n=1, L=1000, H=32, H_kv=8, D=128, page=64, dtype="bf16",
             ragged=False),
        # A serving batch of 32 with histories of all lengths up to 8192.
        dict(name="attend 32 ragged 8192", op="attend", B=32, n=1, L=8192, H=32, H_kv=8, D=128, page=64,
             dtype="bf16", ragged=True),
        # Few sequences with long histories, sixteen query heads to a K/V head.
        dict(name="attend 4x32768 group 16", op="attend", B=4, n=1, L=32768, H=32, H_kv=2, D=128, page=128,
             dtype="fp16", ragged=False),
        # As many K/V as query heads, narrow heads, small pages, two tokens per sequence (one guessed ahead).
        dict(name="attend 16x2049 mha", op="attend", B=16, n=2, L=2049, H=32, H_kv=32, D=64, page=16,
             dtype="fp16", ragged=True),
        # Chunks of prompts behind histories that are in the cache already.
        dict(name="attend chunk 3x1024", op="attend", B=3, n=1024, L=8192, H=32, H_kv=8, D=128, page=64,
             dtype="bf16", ragged=True),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def draw(rng):
    op = rng.choice(["norm_rope", "append", "attend"])
    D = rng.choice([32, 64, 128, 128])
    H_kv = rng.choice([1, 2, 4, 5, 8])
    H = H_kv * rng.choice([1, 2, 3, 4, 7, 8])
    dtype = rng.choice(["bf16", "fp16"])
    if op == "norm_rope":
        rows = _log_int(rng, 64, 1 << 20)  # head rows of q and k together
        tokens = max(1, rows // (H + H_kv))
        B = min(_log_int(rng, 1, 64), tokens)
        N = max(1, tokens // B)
        backward = rng.random() < 0.5 and B * N * (H + H_kv) <= 327680
        return dict(op=op, B=B, N=N, H=H, H_kv=H_kv, D=D, dtype=dtype, wtype=rng.choice(["bf16", "fp32"]) if dtype == "bf16" else "fp32",
                    axes=rng.choice([1, 1, 2, 3]), interleaved=rng.random() < 0.5, max_pos=N + rng.randrange(1, 4096),
                    backward=backward)
    page = rng.choice([16, 32, 64, 128])
    if op == "append":
        B = _log_int(rng, 1, 128)
        n = 1 if rng.random() < 0.4 else _log_int(rng, 1, max(2, 16384 // B))
        return dict(op=op, B=B, n=n, L=n + _log_int(rng, 1, 8192), H_kv=H_kv, D=D, page=page, dtype=dtype,
                    norm=rng.random() < 0.5, axes=rng.choice([1, 1, 3]), interleaved=rng.random() < 0.5,
                    ragged=rng.random() < 0.7)
    B = _log_int(rng, 1, 64)
    L = _log_int(rng, 17, min(32768, (1 << 18) // B))
    n = 1 if rng.random() < 0.6 else _log_int(rng, 1, min(L, 1024, max(1, 2048 // B)))
    while B * H * n * L > 1 << 29:  # no dearer than the largest listed chunk
        n = max(1, n // 2)
        L = max(17, L // 2)
        n = min(n, L)
    return dict(op=op, B=B, n=n, L=L, H=H, H_kv=H_kv, D=D, page=page, dtype=dtype, ragged=rng.random() < 0.7)


def _lengths(case):
    """(lengths with the new tokens, new tokens) of each sequence: a function of the case alone, spread
    over [1/4, 1] of the largest by the golden ratio."""
    B, L, n = case["B"], case["L"], case["n"]
    if not case["ragged"]:
        return [L] * B, [n] * B
    spread = [1.0 if i == 0 else 0.25 + 0.75 * ((i * 0.6180339887498949) % 1.0) for i in range(B)]
    news = [max(1, int(n * spread[(i + 1) % B])) if i else n for i in range(B)]
    lens = [max(news[i], int(L * spread[i])) for i in range(B)]
    return lens, news


def _sections(case):
    half, axes = case["D"] // 2, case["axes"]
    if axes == 1:
        return None
    first = [half // axes // 2 * 2 or 1] * (axes - 1)
    return (half - sum(first),) + tuple(first)


# ------------------------------------------------------------------------------------------ inputs
def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _tables(max_pos, D, device="cuda"):
    half = D // 2
    inv = 10000.0 ** (-torch.arange(half, dtype=torch.float64, device=device) / half)
    ang = torch.arange(max_pos, dtype=torch.float64, device=device)[:, None] * inv
    return ang.cos().float(), ang.sin().float()


def _cache(case, g, pages):
    """A cache in use: e4m3 values that fill most of their range, one power-of-two scale for each page and head."""
    shape = (pages, case["H_kv"], case["page"], case["D"])
    made = []
    for spread in (2.0, 1.0):
        scales = torch.exp2(torch.randint(-8, -5, shape[:2], device="cuda", generator=g).float())
        x = torch.randn(shape, device="cuda", generator=g, dtype=torch.float16).mul_(spread * 64.0)
        made += [x.clamp_(-E4M3_MAX, E4M3_MAX).to(E4M3), scales]
        del x
    return made


def prepare(case, seed):
    g = _gen(seed)
    dt = DTYPES[case["dtype"]]
    s = dict(case=case, op=case["op"], D=case["D"])
    if case["op"] == "norm_rope":
        B, N, H, H_kv, D = (case[k] for k in ("B", "N", "H", "H_kv", "D"))
        # q and k as they leave a fused projection: views of one [B, N, (H + 2 H_kv) D] tensor
        x = torch.randn(B, N, H + 2 * H_kv, D, device="cuda", generator=g, dtype=torch.float32)
        x *= torch.rand(H + 2 * H_kv, 1, device="cuda", generator=g) * 3 + 0.25  # each head has its own size
        x = x.to(dt)
        s["q"] = x[:, :, :H].transpose(1, 2)
        s["k"] = x[:, :, H:H + H_kv].transpose(1, 2)
        s["qw"] = (1 + 0.3 * torch.randn(D, device="cuda", generator=g)).to(DTYPES[case["wtype"]])
        s["kw"] = (1 + 0.3 * torch.randn(D, device="cuda", generator=g)).to(DTYPES[case["wtype"]])
        s["cos"], s["sin"] = _tables(case["max_pos"], D)
        s["sections"] = _sections(case)
        shape = (B, N) if s["sections"] is None else (case["axes"], B, N)
        if N == 1 or case["axes"] > 1:
            s["pos"] = torch.randint(0, case["max_pos"], shape, device="cuda", generator=g, dtype=torch.int32)
        else:  # packed sequences: every row of the batch starts somewhere in its own document
            start = torch.randint(0, case["max_pos"] - N + 1, (B, 1), device="cuda", generator=g, dtype=torch.int32)
            s["pos"] = start + torch.arange(N, device="cuda", dtype=torch.int32)
        s["interleaved"] = case["interleaved"]
        s["backward"] = case["backward"]
        if case["backward"]:
            s["dq"] = torch.randn(B, H, N, D, device="cuda", generator=g, dtype=torch.float32).to(dt)
            s["dk"] = torch.randn(B, H_kv, N, D, device="cuda", generator=g, dtype=torch.float32).to(dt)
            for name in ("q", "k", "qw", "kw"):
                s[name] = s[name].detach().requires_grad_(True)
        return s
    lens, news = _lengths(case)
    B, P, H_kv, D = case["B"], case["page"], case["H_kv"], case["D"]
    width = max(-(-v // P) for v in lens)
    pages = B * width + 3
    s["kp"], s["ks"], s["vp"], s["vs"] = _cache(case, g, pages)
    s["table"] = torch.randperm(pages, device="cuda", generator=g)[:B * width].view(B, width).to(torch.int32)
    s["lens"] = torch.tensor(lens, dtype=torch.int32, device="cuda")
    single = all(v == 1 for v in news)
    T = sum(news)
    starts = [0]
    for v in news:
        starts.append(starts[-1] + v)
    s["offsets"] = None if single else torch.tensor(starts, dtype=torch.int32, device="cuda")
    s["nmax"], s["lmax"] = max(news), max(lens)
    if case["op"] == "append":
        x = torch.randn(T, 2 * H_kv, D, device="cuda", generator=g, dtype=torch.float32)
        x *= torch.rand(2 * H_kv, 1, device="cuda", generator=g) * 3 + 0.25
        x = x.to(dt)
        s["k"], s["v"] = x[:, :H_kv], x[:, H_kv:]
        s["kw"] = (1 + 0.3 * torch.randn(D, device="cuda", generator=g)).to(dt) if case["norm"] else None
        s["cos"], s["sin"] = _tables(max(lens), D)
        s["sections"] = _sections(case)
        s["interleaved"] = case["interleaved"]
        s["pos"] = None if case["axes"] == 1 else torch.randint(0, max(lens), (case["axes"], T), device="cuda", generator=g, dtype=torch.int32)
    else:
        s["q"] = (2.0 * torch.randn(T, case["H"], D, device="cuda", generator=g, dtype=torch.float32)).to(dt)
    return s


# ------------------------------------------------------------------------------------- plain forms
def _pair_angles(cos, sin, pos, sections):
    """cos and sin of every pair at every token: pos [..., tokens], with a leading axis where sections are given."""
    if sections is None:
        return cos[pos], sin[pos]
    axis = torch.repeat_interleave(torch.arange(len(sections), device=pos.device),
                                   torch.tensor(sections, device=pos.device), output_size=sum(sections))
    p = pos[axis].movedim(0, -1).long()  # [..., tokens, pairs]
    pair = torch.arange(p.shape[-1], device=pos.device)
    return cos[p, pair], sin[p, pair]


def _split(x, interleaved):
    return (x[..., 0::2], x[..., 1::2]) if interleaved else x.chunk(2, dim=-1)


def _join(a, b, interleaved):
    return torch.stack((a, b), dim=-1).flatten(-2) if interleaved else torch.cat((a, b), dim=-1)


def _plain_norm_rope(x, w, c, s, interleaved):
    x32 = x.float()
    y = x32 * torch.rsqrt(x32.square().mean(-1, keepdim=True) + EPS) * w.float()
    a, b = _split(y, interleaved)
    return _join(a * c - b * s, a * s + b * c, interleaved).to(x.dtype)


def _plain_norm_rope_grad(x, w, c, s, interleaved, dz):
    x32, w32 = x.float(), w.float()
    r = torch.rsqrt(x32.square().mean(-1, keepdim=True) + EPS)
    a, b = _split(dz.float(), interleaved)
    dy = _join(a * c + b * s, b * c - a * s, interleaved)
    dw = (dy * x32 * r).double().sum((0, 1, 2)).to(w.dtype)
    g = dy * w32
    dx = r * (g - x32 * r.square() * (g * x32).mean(-1, keepdim=True))
    return dx.to(x.dtype), dw


def _run_norm_rope(st):
    with torch.no_grad():
        c, s = _pair_angles(st["cos"], st["sin"], st["pos"], st["sections"])
        c, s = c.unsqueeze(1), s.unsqueeze(1)  # over the heads
        i = st["interleaved"]
        out = [_plain_norm_rope(st["q"], st["qw"], c, s, i), _plain_norm_rope(st["k"], st["kw"], c, s, i)]
        if st["backward"]:
            dq, dqw = _plain_norm_rope_grad(st["q"], st["qw"], c, s, i, st["dq"])
            dk, dkw = _plain_norm_rope_grad(st["k"], st["kw"], c, s, i, st["dk"])
            out += [dq, dk, dqw, dkw]
        return out


def _token_places(st, T):
    """Sequence, index in its new tokens and new tokens of the sequence, of each of the T new tokens."""
    t = torch.arange(T, device="cuda")
    if st["offsets"] is None:
        return t, torch.zeros_like(t), torch.ones_like(t)
    o = st["offsets"].long()
    b = torch.searchsorted(o[1:], t, right=True)
    return b, t - o[b], (o[1:] - o[:-1])[b]


def _exponent(amax):
    """The smallest e with amax <= 448 * 2^e."""
    f, e = torch.frexp(amax)
    return (e - 9 + (f > 0.875).int()).clamp(min=-126)


def _plain_store(pages, scales, x, st, places):
    """Rounds x [T, H_kv, D] (32 bits) into its pages; the pages' scales grow where the new tokens need it."""
    P = pages.shape[2]
    b, i, n = places
    table, lens = st["table"].long(), st["lens"].long()
    pos = lens[b] - n + i
    page, slot = table[b, pos // P], pos % P
    amax = torch.zeros(pages.shape[:2], device="cuda").index_reduce_(0, page, x.abs().amax(-1), "amax")
    need = torch.ldexp(torch.ones_like(amax), _exponent(amax))
    # the first page of each sequence may hold older tokens, which keep their scale or are rounded again
    first_t = torch.arange(table.shape[0], device="cuda") if st["offsets"] is None else st["offsets"][:-1].long()
    fpage, fslot = page[first_t], slot[first_t]
    old = scales[fpage]
    fresh = need.clone()
    fresh[fpage] = torch.where((fslot > 0)[:, None], torch.maximum(old, need[fpage]), need[fpage])
    codes = pages.view(torch.uint8)
    there = codes[fpage].view(E4M3).float()
    behind = torch.arange(P, device="cuda")[None, None, :, None] >= fslot[:, None, None, None]
    there = torch.where(behind, there, there * (old / fresh[fpage])[:, :, None, None])
    codes[fpage] = there.to(E4M3).view(torch.uint8)
    scales[page] = fresh[page]
    codes[page, :, slot] = (x / fresh[page][:, :, None]).to(E4M3).view(torch.uint8)


def _run_append(st):
    k, v = st["k"], st["v"]
    places = _token_places(st, k.shape[0])
    b, i, n = places
    pos = st["lens"].long()[b] - n + i if st["pos"] is None else st["pos"]
    c, s = _pair_angles(st["cos"].double(), st["sin"].double(), pos, st["sections"])
    x = k.double()
    if st["kw"] is not None:
        x = x / torch.sqrt(x.square().mean(-1, keepdim=True) + EPS) * st["kw"].double()
    a, d = _split(x, st["interleaved"])
    c, s = c.unsqueeze(1), s.unsqueeze(1)
    x = _join(a * c - d * s, a * s + d * c, st["interleaved"]).float()
    _plain_store(st["kp"], st["ks"], x, st, places)
    _plain_store(st["vp"], st["vs"], v.float(), st, places)
    return [st["kp"], st["vp"], st["ks"], st["vs"]]


def _run_attend(st):
    q, table, lens = st["q"], st["table"].long(), st["lens"].long()
    T, H, D = q.shape
    B, H_kv, P = table.shape[0], st["kp"].shape[1], st["kp"].shape[2]
    G, nmax, L = H // H_kv, st["nmax"], st["lmax"]

    def dense(pages, scales):  # [B, H_kv, L, D] in 32 bits
        x = pages.view(torch.uint8)[table].view(E4M3).float() * scales[table][..., None, None]
        return x.transpose(1, 2).reshape(B, H_kv, -1, D)[:, :, :L]

    b, i, n = _token_places(st, T)
    qp = torch.zeros(B, nmax, H, D, device="cuda").index_put((b, i), q.float())
    qp = qp.view(B, nmax, H_kv, G, D).permute(0, 2, 3, 1, 4).reshape(B, H_kv, G * nmax, D)
    x = torch.matmul(qp, dense(st["kp"], st["ks"]).transpose(-1, -2)).view(B, H_kv, G, nmax, L)
    count = torch.ones_like(lens) if st["offsets"] is None else (st["offsets"][1:] - st["offsets"][:-1]).long()
    last = (lens - count)[:, None] + torch.arange(nmax, device="cuda")  # the last key of each token
    seen = torch.arange(L, device="cuda")[None, None] <= last[:, :, None]
    x.mul_(1.0 / math.sqrt(D)).masked_fill_(~seen[:, None, None], float("-inf"))
    x.sub_(x.amax(-1, keepdim=True)).exp_()
    total = x.sum(-1, keepdim=True)
    o = torch.matmul(x.view(B, H_kv, G * nmax, L), dense(st["vp"], st["vs"])).view(B, H_kv, G, nmax, D) / total
    return o.permute(0, 3, 1, 2, 4).reshape(B, nmax, H, D)[b, i].to(q.dtype)


def run(state):
    if own:
        return _run_own(state)
    return {"norm_rope": _run_norm_rope, "append": _run_append, "attend": _run_attend}[state["op"]](state)


# ----------------------------------------------------------------------------- the framework's calls
def _package():
    if "fused-attention_b200" not in sys.path:
        sys.path.insert(0, "fused-attention_b200")


def _run_own(st):
    _package()
    if st["op"] == "norm_rope":
        from attention.rotary.norm_rope import qk_norm_rope
        q, k = qk_norm_rope(st["q"], st["k"], st["cos"], st["sin"], positions=st["pos"], q_weight=st["qw"],
                            k_weight=st["kw"], eps=EPS, interleaved=st["interleaved"], sections=st["sections"])
        if not st["backward"]:
            return [q, k]
        return [q.detach(), k.detach(),
                *torch.autograd.grad((q, k), (st["q"], st["k"], st["qw"], st["kw"]), (st["dq"], st["dk"]))]
    from attention.paged.cache import PagedKVCache
    cache = PagedKVCache(st["kp"], st["vp"], st["ks"], st["vs"])
    if st["op"] == "append":
        from attention.paged.cache import append_kv
        append_kv(cache, st["k"], st["v"], st["table"], st["lens"], st["offsets"], cos=st["cos"], sin=st["sin"],
                  positions=st["pos"], k_weight=st["kw"], eps=EPS, interleaved=st["interleaved"], sections=st["sections"])
        return [cache.k_pages, cache.v_pages, cache.k_scales, cache.v_scales]
    from attention.paged.paged_attention import paged_attention
    return paged_attention(st["q"], cache, st["table"], st["lens"], st["offsets"])


# -------------------------------------------------------------------------------------------- work
def work(case):
    el, D = 2, case["D"]
    if case["op"] == "norm_rope":
        tokens = case["B"] * case["N"]
        rows = tokens * (case["H"] + case["H_kv"])
        seen = min(tokens, case["max_pos"]) * D * 4  # a cos and a sin for each pair of a position
        passes = 4 if case["backward"] else 2  # x and dz in, y and dx out
        return {"bytes": rows * D * el * passes + seen + tokens * 4 * case["axes"],
                "flops": rows * D * (14 if case["backward"] else 6)}
    lens, news = _lengths(case)
    T, H_kv, P = sum(news), case["H_kv"], case["page"]
    if case["op"] == "append":
        touched = sum((L - 1) // P - (L - n) // P + 1 for L, n in zip(lens, news))
        return {"bytes": 2 * T * H_kv * D * (el + 1) + 2 * touched * H_kv * 4 + min(T, max(lens)) * D * 4,
                "flops": T * H_kv * D * 10}
    H = case["H"]
    pairs = sum(n * L - n * (n - 1) // 2 for L, n in zip(lens, news))
    keys = sum(lens)
    return {"bytes": 2 * keys * H_kv * D + 2 * sum(-(-L // P) for L in lens) * H_kv * 4 + 2 * T * H * D * el,
            "flops": 4 * pairs * H * D}


# ------------------------------------------------------------------------------------------- exact
def exact(case, seed):
    st = prepare(case, seed)
    with torch.no_grad():
        if st["op"] == "append":
            return _exact_append(st)
        if st["op"] == "attend":
            return _exact_attend(st)
    return _exact_norm_rope(st)


def _turns(st, pos):
    """e^{i angle} of each pair at each token, complex128, from the tables."""
    z = torch.complex(st["cos"].double(), st["sin"].double())
    if st["sections"] is None:
        return z[pos.long()]
    out, lo = [], 0
    for axis, width in enumerate(st["sections"]):
        out.append(z[pos[axis].long()][..., lo:lo + width])
        lo += width
    return torch.cat(out, -1)


def _turned(x, turn, interleaved):
    D = x.shape[-1]
    z = torch.view_as_complex(x.unflatten(-1, (D // 2, 2) if interleaved else (2, D // 2))
                              .movedim(-1 if interleaved else -2, -1).contiguous()) * turn
    z = torch.view_as_real(z)
    return z.flatten(-2) if interleaved else z.movedim(-1, -2).flatten(-2)


def _exact_norm_rope(st):
    turn = _turns(st, st["pos"]).unsqueeze(1)
    outs, grads = [], []
    for x, w, dz in ((st["q"], st["qw"], st.get("dq")), (st["k"], st["kw"], st.get("dk"))):
        x64 = x.detach().double().requires_grad_(True)
        w64 = w.detach().double().requires_grad_(True)
        size = (x64 * x64).sum(-1, keepdim=True) / st["D"] + EPS
        z = _turned(x64 * w64 * size.pow(-0.5), turn, st["interleaved"])
        outs.append(z.detach())
        if st["backward"]:
            grads.append(torch.autograd.grad(z, (x64, w64), dz.double()))
        del z, x64
    if not grads:
        return outs
    return outs + [grads[0][0], grads[1][0], grads[0][1], grads[1][1]]


def _exact_append(st):
    kp, vp, ks, vs = (st[n].double() for n in ("kp", "vp", "ks", "vs"))
    P, H_kv = kp.shape[2], kp.shape[1]
    T = st["k"].shape[0]
    lens = st["lens"].tolist()
    starts = st["offsets"].tolist() if st["offsets"] is not None else list(range(T + 1))
    table = st["table"].tolist()
    k = st["k"].double()
    if st["kw"] is not None:
        k = k / ((k * k).sum(-1, keepdim=True) / st["D"] + EPS).sqrt() * st["kw"].double()
    if st["pos"] is None:
        own_pos = torch.cat([torch.arange(lens[b] - (starts[b + 1] - starts[b]), lens[b]) for b in range(len(lens))])
        turn = _turns(st, own_pos.cuda())
    else:
        turn = _turns(st, st["pos"])
    k = _turned(k, turn.unsqueeze(1), st["interleaved"]).float().double()  # the definition rounds to 32 bits here
    for x, pages, scales in ((k, kp, ks), (st["v"].double(), vp, vs)):
        for b, L in enumerate(lens):
            t, at = starts[b], L - (starts[b + 1] - starts[b])
            while at < L:
                page, slot = table[b][at // P], at % P
                count = min(P - slot, L - at)
                part = x[t:t + count].transpose(0, 1)  # [H_kv, count, D]
                top = part.abs().amax((1, 2)) / E4M3_MAX
                # values of 24 bits: one above a power of two is 8.6e-8 above it in log2, one at it is not
                scale = torch.exp2(torch.ceil(torch.log2(top.clamp(min=2.0 ** -126)) - 1e-9))
                if slot:
                    scale = torch.maximum(scale, scales[page])
                    pages[page][:, :slot] = (pages[page][:, :slot] * (scales[page] / scale)[:, None, None]).float().to(E4M3).double()
                pages[page][:, slot:slot + count] = (part / scale[:, None, None]).float().to(E4M3).double()
                scales[page] = scale
                t, at = t + count, at + count
    return [kp, vp, ks, vs]


def _exact_attend(st):
    q = st["q"].double()
    T, H, D = q.shape
    H_kv = st["kp"].shape[1]
    lens = st["lens"].tolist()
    starts = st["offsets"].tolist() if st["offsets"] is not None else list(range(T + 1))
    out = torch.empty_like(q)
    for b, L in enumerate(lens):
        n = starts[b + 1] - starts[b]
        pages = st["table"][b, :-(-L // st["kp"].shape[2])].long()
        for h in range(H_kv):
            K, V = ((st[p].view(torch.uint8)[pages, h].view(E4M3).double() * st[s][pages, h].double()[:, None, None]).reshape(-1, D)[:L]
                    for p, s in (("kp", "ks"), ("vp", "vs")))
            mask = torch.arange(L, device="cuda")[None] > torch.arange(L - n, L, device="cuda")[:, None]
            for head in range(h * (H // H_kv), (h + 1) * (H // H_kv)):
                a = (q[starts[b]:starts[b + 1], head] @ K.T) * D ** -0.5
                a = torch.softmax(a.masked_fill_(mask, -math.inf), -1)
                out[starts[b]:starts[b + 1], head] = a @ V
    return out


if __name__ == "__main__":
    for c in listed() + [draw(random.Random(i)) for i in range(40)]:
        print(c, work(c))
