"""The paged cache's operators from their definitions
(include/shaobo_fa3_cache.h), in fp64 and integers, sequence by sequence, with
how far a kernel may be off (attn_oracle.py says how roundings are counted).

A cache here is a dict: k, v (pages), bits, table [B, width], kv, new (lists),
page_size, D, dtype."""
import math

import torch

import attn_oracle as A

E = A.E
LEVELS = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def codes_of(x):
    """(codes, scales) of rows x [..., D] of 16-bit values, by comparing with
    every level: the nearest, of two equally near the even one."""
    x = x.double()
    top = x.abs().amax(-1, keepdim=True)
    level = torch.tensor(LEVELS, dtype=torch.float64, device=x.device)
    # |6 |x| - level a|, exact in fp64 (11 and 14 significant bits)
    far = (6 * x.abs()[..., None] - level * top[..., None]).abs()
    near = far.amin(-1, keepdim=True)
    even = torch.arange(8, device=x.device) % 2 == 0
    rank = torch.where(far == near, torch.where(even, 2, 1), 0)
    code = rank.argmax(-1)
    code = torch.where(top == 0, torch.zeros_like(code), code)
    sign = x < 0
    finite = torch.isfinite(top)
    # (a sixth of 8 or 11 bits never lies halfway between two fp32 numbers)
    scale = (top / 6.0).float().squeeze(-1)
    code = torch.where(finite, code + 8 * sign, torch.zeros_like(code))
    return code, torch.where(finite.squeeze(-1), scale, torch.full_like(scale, math.nan))


def parts(pages):
    """Codes [pages, H, page, D] and scales [pages, H, page] of 4-bit pages."""
    n, H, ps, row = pages.shape
    flat = pages.reshape(n, H, ps * row)
    c = flat[..., :ps * (row - 4)].reshape(n, H, ps, row - 4)
    c = torch.stack((c & 15, c >> 4), -1).flatten(-2)
    return c.int(), flat[..., ps * (row - 4):].contiguous().view(torch.float32)


def pack(code, scale):
    """4-bit pages of codes [pages, H, page, D] and scales."""
    n, H, ps, D = code.shape
    c = code.to(torch.uint8)
    c = (c[..., 0::2] | (c[..., 1::2] << 4)).reshape(n, H, ps * D // 2)
    s = scale.float().contiguous().view(torch.uint8).reshape(n, H, ps * 4)
    return torch.cat((c, s), 2).reshape(n, H, ps, D // 2 + 4)


def rows_of(pages, bits):
    """fp64 rows [pages, H, page, D] that pages stand for."""
    if bits == 16:
        return pages.double()
    code, scale = parts(pages)
    level = torch.tensor(LEVELS + tuple(-x for x in LEVELS), dtype=torch.float64,
                         device=pages.device)
    return level[code.long()] * scale.double()[..., None]


def there(cache, b):
    """[kv] truth values: the place has a page; [kv] page and row of it."""
    kv, ps = clipped(cache, b)[0], cache["page_size"]
    j = torch.arange(kv, device=cache["table"].device)
    page = cache["table"][b].long()[j // ps]
    ok = (page >= 0) & (page < cache["k"].shape[0])
    return ok, torch.where(ok, page, torch.zeros_like(page)), j % ps


def clipped(cache, b):
    """Tokens of sequence b and new ones, taken into their ranges."""
    most = cache["table"].shape[1] * cache["page_size"]
    return max(0, min(most, int(cache["kv"][b]))), int(cache["new"][b])


def sequence(cache, b):
    """k, v [H, kv, D] fp64 of sequence b (zeros where there is no page) and there()'s mask."""
    ok, page, row = there(cache, b)
    out = []
    for pages in (cache["k"], cache["v"]):
        if pages.shape[0] == 0:
            out.append(torch.zeros(pages.shape[1], ok.numel(), cache["D"], dtype=torch.float64,
                                   device=ok.device))
            continue
        used, inv = torch.unique(page, return_inverse=True)
        x = rows_of(pages[used], cache["bits"])[inv, :, row].transpose(0, 1)
        out.append(torch.where(ok[None, :, None], x, torch.zeros((), dtype=x.dtype, device=x.device)))
    return out[0], out[1], ok


def attend(q, cache, causal=True, scale=None, softcap=0.0, slopes=None, prefix=None,
           selected=None):
    """out, lse and their bounds, fp64."""
    B, Hq, S, D = q.shape
    Hkv, ps = cache["k"].shape[1], cache["page_size"]
    G = Hq // Hkv
    scale = D ** -0.5 if scale is None else scale
    u, dev = torch.finfo(q.dtype).eps / 2, q.device
    # (4 bits in fp16: P times a value's scale as two bf16 terms, the second off
    # by half a step of what the first leaves, 2^-8 of 2^-8; below 2^-126 it is
    # flushed, and with it nothing of fp16's size)
    up = u if cache["bits"] == 16 or q.dtype == torch.bfloat16 else (torch.finfo(torch.bfloat16).eps / 2) ** 2
    out = torch.zeros(B, Hq, S, D, dtype=torch.float64, device=dev)
    lse = torch.full((B, Hq, S), -math.inf, dtype=torch.float64, device=dev)
    out_off, lse_off = torch.zeros_like(out), torch.zeros_like(lse)
    slope = A.options(B, Hq, slopes)
    for b in range(B):
        kv, new = clipped(cache, b)
        k, v, ok = sequence(cache, b)
        i = torch.arange(S, device=dev)[:, None]
        j = torch.arange(kv, device=dev)[None, :]
        dist = (i + kv - new - j).double()
        seen = ok[None, :] & (i < new)
        if causal:
            seen = seen & ((dist >= 0) | (j < (int(prefix[b]) if prefix is not None else 0)))
        for h in range(Hq):
            mine, times = seen, None
            if selected is not None:
                n = selected[b, h // G].long()  # [S, count]
                times = (n[:, None, :] == (j[0] // ps)[None, :, None]).sum(-1)
                mine = seen & (times > 0)
            x = A.Head(q[b, h], k[h // G], scale, softcap, slope(b, h), mine, dist)
            if times is not None:
                x.s = x.s + torch.log(times.double().clamp(min=1))
            vd = A.clean(v[h // G], x.keys)
            p = x.probabilities()
            out[b, h] = p @ vd
            lse[b, h] = torch.logsumexp(x.s, 1)
            dx = x.dx.amax(1) if kv else torch.zeros(S, dtype=torch.float64, device=dev)
            off = dx + (mine.sum(1) + 64) * E
            lse_off[b, h] = torch.where(x.rows, off + 8 * E * lse[b, h].abs(),
                                        torch.zeros_like(off))
            size = p @ vd.abs()
            out_off[b, h] = size * (up + 2 * off[:, None]) * 1.01 + u * out[b, h].abs() * 1.01 + \
                A.smallest(q.dtype) * (vd.abs().sum(0)[None, :] + 2)
    return out, lse, out_off, lse_off


def select(q, bounds, cache, count):
    """[B, Hkv, S, count] page numbers."""
    B, Hq, S, D = q.shape
    Hkv, ps = bounds.shape[1], cache["page_size"]
    G = Hq // Hkv
    out = torch.full((B, Hkv, S, count), -1, dtype=torch.int32)
    for b in range(B):
        kv, new = clipped(cache, b)
        for i in range(new):
            place = kv - new + i
            if place < 0:
                continue
            own = place // ps
            page = cache["table"][b, :own + 1].long()
            ok = (page >= 0) & (page < bounds.shape[0])
            for h in range(Hkv):
                x = bounds[page.clamp(0, max(0, bounds.shape[0] - 1)), h].double()
                qs = q[b, h * G:(h + 1) * G, i].double()[:, None]
                s = torch.maximum(qs * x[None, :, 0], qs * x[None, :, 1]).sum(-1)
                # (a bound, or the score of any head, that is not finite)
                wild = (~torch.isfinite(s)).any(0) | (~torch.isfinite(x)).flatten(1).any(1)
                s = torch.where(wild, torch.full_like(s[0], math.inf), s.amax(0))
                order = [(0 if n == own else 1, -float(s[n]), n) for n in range(own + 1)
                         if bool(ok[n])]
                take = sorted(n for _, _, n in sorted(order)[:count])
                out[b, h, i, :len(take)] = torch.tensor(take, dtype=torch.int32)
    return out.to(q.device)


def turned(x, cache, freqs, positions, interleaved):
    """x turned, fp64 [B, H, S, D], and how far a kernel may be off: half a
    step of the type for its one rounding, by way of fp32 (2^-24), and angles
    off by 2^-48 of a radian's size."""
    B, _, S, _ = x.shape
    if freqs is None:
        return x.double(), torch.zeros_like(x, dtype=torch.float64)
    if positions is None:
        i = torch.arange(S, device=x.device)
        positions = torch.stack([clipped(cache, b)[0] - clipped(cache, b)[1] + i
                                 for b in range(B)])[None]
    P = freqs.shape[1]
    angle = (positions.double()[..., None] * freqs.double()[:, None, None, :]).sum(0)[:, None]
    cos, sin = torch.cos(angle), torch.sin(angle)
    loose = 2.0 ** -24 + angle.abs() * 2.0 ** -48
    y = x.double().clone()
    lo, hi = (slice(0, 2 * P, 2), slice(1, 2 * P, 2)) if interleaved else \
        (slice(0, P), slice(P, 2 * P))
    a, b = y[..., lo].clone(), y[..., hi].clone()
    y[..., lo], y[..., hi] = a * cos - b * sin, b * cos + a * sin
    off = torch.zeros_like(y)
    off[..., lo] = off[..., hi] = (a.abs() + b.abs()) * loose
    off[..., :2 * P] = off[..., :2 * P] + torch.finfo(x.dtype).eps / 2 * y[..., :2 * P].abs() + \
        A.smallest(x.dtype)
    return y, off
