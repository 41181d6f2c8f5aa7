"""Plain 64-bit forms of the operators around attention (norm + rotary positions, the paged e4m3 cache,
attention over it), for small cases, and the error bounds their kernels are held to."""
import math

import torch

E4M3 = torch.float8_e4m3fn
U32 = 2.0 ** -24  # half a step of float32, relative


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def half_subnormal(dtype):
    """Half the distance of the smallest numbers of a 16-bit type."""
    return torch.finfo(dtype).tiny * torch.finfo(dtype).eps / 2


def tables(max_pos, D, device, base=10000.0):
    i = torch.arange(D // 2, dtype=torch.float64)
    a = torch.arange(max_pos, dtype=torch.float64)[:, None] * base ** (-2 * i / D)
    return a.cos().float().to(device), a.sin().float().to(device)


def angles(cos, sin, positions, sections):
    """float64 cos, sin [..., tokens, pairs]; positions [..., tokens], with sections a leading axis."""
    if sections is None:
        return cos.double()[positions.long()], sin.double()[positions.long()]
    c, s, at = [], [], 0
    for axis, n in enumerate(sections):
        p = positions[axis].long()
        c.append(cos.double()[p][..., at:at + n])
        s.append(sin.double()[p][..., at:at + n])
        at += n
    return torch.cat(c, -1), torch.cat(s, -1)


def pairs(x, interleaved):
    D = x.shape[-1]
    return (x[..., 0::2], x[..., 1::2]) if interleaved else (x[..., :D // 2], x[..., D // 2:])


def unpairs(a, b, interleaved):
    return torch.stack((a, b), -1).flatten(-2) if interleaved else torch.cat((a, b), -1)


def norm_rope64(x, w, c, s, eps, interleaved):
    """float64 norm + rotation; c, s broadcast over the heads already."""
    y = x.double()
    if w is not None:
        y = y / torch.sqrt((y * y).mean(-1, keepdim=True) + eps) * w.double()
    a, b = pairs(y, interleaved)
    return unpairs(a * c - b * s, a * s + b * c, interleaved)


def rotated_size(x, w, c, s, eps, interleaved):
    """|a c| + |b s| and |a s| + |b c|: what the rotation's float32 errors are relative to."""
    y = x.double()
    if w is not None:
        y = y / torch.sqrt((y * y).mean(-1, keepdim=True) + eps) * w.double()
    a, b = (v.abs() for v in pairs(y, interleaved))
    return unpairs(a * c.abs() + b * s.abs(), a * s.abs() + b * c.abs(), interleaved)


def scale64(amax):
    """The smallest power of two, at least 2^-126, that holds amax in 448 steps of it."""
    if amax == 0:
        return 2.0 ** -126
    f, e = math.frexp(amax)
    return 2.0 ** max(-126, e - 9 + (f > 0.875))


def to_e4m3(x):
    """float32 -> e4m3 with saturation, NaN kept."""
    return torch.where(x.isnan(), x, x.clamp(-448.0, 448.0)).to(E4M3)


def append64(kp, vp, ks, vs, k, v, table, lens, starts, c, s, w, eps, interleaved):
    """The cache's four tensors (CPU) after an append: one page at a time.  c, s: float64 [T, pairs] or None."""
    kp, vp, ks, vs = kp.clone(), vp.clone(), ks.clone(), vs.clone()
    P = kp.shape[2]
    if w is not None or c is not None:
        one = torch.ones(1, dtype=torch.float64)
        k = norm_rope64(k, w, *((one, one * 0) if c is None else (c[:, None], s[:, None])), eps, interleaved)
    for x, pages, scales in ((k.float(), kp, ks), (v.float(), vp, vs)):
        for b, L in enumerate(lens):
            n = starts[b + 1] - starts[b]
            j = max(0, L - n)
            while j < L:
                page, slot = int(table[b, j // P]), j % P
                count = min(P - slot, L - j)
                t = starts[b] + j - (L - n)
                for h in range(pages.shape[1]):
                    part = x[t:t + count, h]
                    mag = part.abs()
                    amax = float(torch.where(mag.isfinite(), mag, torch.zeros(())).max())
                    scale = scale64(amax)
                    if slot and float(scales[page, h]) > scale:
                        scale = float(scales[page, h])
                    elif slot:
                        old = pages[page, h, :slot].float() * (float(scales[page, h]) / scale)
                        pages[page, h, :slot] = to_e4m3(old)
                    pages[page, h, slot:slot + count] = to_e4m3((part.double() / scale).float())
                    scales[page, h] = scale
                j += count
    return kp, vp, ks, vs


def paged64(q, kp, vp, ks, vs, table, lens, starts, scale, chunk=False):
    """(o, lse, bound, lse_bound) of paged attention in 64 bits; `bound` is what the kernels' arithmetic may add to
    half a step of the output's type, `lse_bound` how far lse may be off (all CPU tensors):
      * a score is a float32 sum of D exact products: off by at most 2 D 2^-24 of the sum of their magnitudes
        (in natural units; the products' sum may be truncated, hence 2), and so is its weight, relative;
        the same again, plus 2^-20 for the exponentials, holds for the softmax sum;
      * a weight is rounded to f16: 2^-11 of it, or 2^-25 of the largest weight times page scale;
      * the weighted sum over n keys is a float32 sum: 2 n 2^-24 of the sum of magnitudes;
      * lse: the scores' error, the softmax sum's (2^-20 and n 2^-24, relative) and two float32 roundings.
    The chunk kernel (chunk=True) adds:
      * a share of the exponentials as a polynomial, 7.5e-5 < 2^-13 of them, in the weights and in their sum;
      * weights relative to the largest weight alone: 2^-25 of it times the sum of |v|;
      * cached values as f16(64 value / largest page scale): 2^-25 of 1/64 of that scale, where f16 is subnormal."""
    T, H, D = q.shape
    P, H_kv = kp.shape[2], kp.shape[1]
    G = H // H_kv
    o = torch.zeros(T, H, D, dtype=torch.float64)
    lse = torch.full((T, H), -math.inf, dtype=torch.float64)
    bound = torch.zeros(T, H, D, dtype=torch.float64)
    lse_bound = torch.zeros(T, H, dtype=torch.float64)
    q = q.double()
    for b, L in enumerate(lens):
        n = starts[b + 1] - starts[b]
        pages = [int(table[b, i]) for i in range(-(-L // P))]
        skip = max(0, n - L)  # tokens in front of the first key
        if not pages or n <= skip:
            continue
        t = slice(starts[b] + skip, starts[b + 1])
        K = (kp[pages].double() * ks[pages].double()[..., None, None]).transpose(1, 2).reshape(-1, H_kv, D)[:L]
        code = vp[pages].double().transpose(1, 2).reshape(-1, H_kv, D)[:L]
        size = vs[pages].double()[:, None].expand(-1, P, -1).reshape(-1, H_kv)[:L]
        count = torch.arange(L - n + skip, L)[:, None] + 1.0  # keys that each token sees
        hidden = torch.arange(L)[None] >= count
        for h in range(H):
            g = h // G
            k, v, row = K[:, g], code[:, g] * size[:, g, None], q[t, h]
            x = (row @ k.T * scale).masked_fill(hidden, -math.inf)
            off = (row.abs() @ k.abs().T * scale).masked_fill(hidden, 0).amax(1, keepdim=True) * 2 * D * U32
            p = torch.softmax(x, 1)
            o[t, h] = p @ v
            lse[t, h] = torch.logsumexp(x, 1) * math.log2(math.e)
            weight = 2.0 ** -11 + 2.0 ** -19 + 4 * count * U32
            more = 0.0
            if chunk:
                off = off + row.abs().sum(1, keepdim=True) * scale * 2.0 ** -31 * float(ks[pages, g].max())
                weight = weight + 2.0 ** -12
                seen = torch.where(hidden, 0.0, 1.0).to(v.dtype)
                more = 2.0 ** -25 * p.amax(1, keepdim=True) * (seen @ v.abs()) + 2.0 ** -31 * float(vs[pages, g].max())
            most = (p * size[:, g]).amax(1, keepdim=True)
            seen_code = torch.where(hidden, 0.0, 1.0).to(v.dtype) @ code[:, g].abs()
            bound[t, h] = (p @ v.abs()) * (weight + 2 * off) + 2.0 ** -25 * most * seen_code + more
            lse_bound[t, h] = (math.log2(math.e) * (off + (2.0 ** -12 if chunk else 0) + 2.0 ** -20 + count * U32)).squeeze(1) \
                + 4 * U32 * (1 + lse[t, h].abs())
    return o, lse, bound, lse_bound
