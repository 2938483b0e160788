"""The attention layer's operators in fp64, from their definitions
(include/shaobo_fa3_attn.h), one head at a time, with how far a kernel may be
off: every bound below counts roundings.

u is half a step of the tensors' type (torch.finfo(t).eps / 2), e = 2^-24 half
a step of fp32.  A kernel rounds P (and dS) to the type before a product and
the output once more, so an output sum_j p_j v_j is off by at most
u sum_j p_j |v_j| + u |out|; fp16 has a smallest step, 2^-24, which p below
2^-14 is rounded to (half of it off).  The rest is fp32: a dot product of D
terms is off by D e sum |q_i k_i|, the exponent's argument by a few e of its
size, and a factor exp(x + dx) by dx relatively."""
import math

import torch

E = 2.0 ** -24


def visible(b, Sq, Sk, causal, documents, documents_k, prefix_lens, kv_lens, device="cpu"):
    """(mask [Sq, Sk], distance [Sq, Sk], keys in use) of batch entry b."""
    kv = Sk if kv_lens is None else max(0, min(Sk, int(kv_lens[b])))
    i = torch.arange(Sq, device=device)[:, None]
    j = torch.arange(Sk, device=device)[None, :]
    d = i + kv - Sq - j
    seen = (j < kv) & (i >= 0)
    if causal:
        prefix = 0 if prefix_lens is None else int(prefix_lens[b])
        seen = seen & ((d >= 0) | (j < prefix))
    if documents is not None:
        q = documents[b].to(device)
        k = (documents if documents_k is None else documents_k)[b].to(device)
        seen = seen & (q[:, None] == k[None, :]) & (q[:, None] >= 0)
    return seen, d.double(), kv


def clean(x, rows):
    """x with the rows that take no part as zeros (they may hold anything)."""
    return torch.where(rows[:, None], x, torch.zeros((), dtype=x.dtype, device=x.device))


class Head:
    """Scores and probabilities of one head, and the fp32 error of a score."""

    def __init__(self, q, k, scale, softcap, slope, seen, dist):
        D = q.shape[1]
        rows, keys = seen.any(1), seen.any(0)
        self.q, self.k = clean(q.double(), rows), clean(k.double(), keys)
        dot = self.q @ self.k.t().contiguous()
        s = dot * scale
        size = (self.q.abs() @ self.k.abs().t().contiguous()) * abs(scale)
        # the dot product, its scale, and a few operations on the score
        self.dx = (D + 8) * E * size
        self.slope = torch.ones_like(s)
        if softcap:
            t = torch.tanh(s / softcap)
            self.slope = 1.0 - t * t
            self.dx = self.dx + 8 * E * softcap
            s = softcap * t
        if slope is not None:
            bias = float(slope) * dist.abs()
            s = s - bias
            self.dx = self.dx + 8 * E * bias.abs()
        self.s = torch.where(seen, s, torch.full_like(s, -math.inf))
        self.seen, self.rows, self.keys = seen, rows, keys
        self.dx = torch.where(seen, self.dx + 8 * E * s.abs(), torch.zeros_like(s))

    def probabilities(self, lse=None):
        """exp(s - lse) (lse None: the scores' own)."""
        if lse is None:
            lse = torch.logsumexp(self.s, 1)
        x = self.s - torch.where(self.rows, lse, torch.zeros_like(lse))[:, None]
        return torch.where(self.seen, torch.exp(x), torch.zeros_like(x))


def options(B, Hq, slopes):
    def slope(b, h):
        if slopes is None:
            return None
        return slopes[b, h] if slopes.dim() == 2 else slopes[h]
    return slope


def smallest(dtype):
    """Off by this at most where a value is too small for the type's relative
    rounding: fp16's subnormals are 2^-24 apart; exp2 and the fp32 products of
    a P below 2^-126, the smallest normal number of fp32 and bf16, are flushed
    to zero, 2^-126 at most."""
    return 2.0 ** -25 if dtype == torch.float16 else 2.0 ** -126


def forward(q, k, v, causal, scale=None, softcap=0.0, slopes=None, documents=None,
            documents_k=None, prefix_lens=None, kv_lens=None):
    """out, lse and their bounds, fp64."""
    B, Hq, Sq, D = q.shape
    Hkv, Sk = k.shape[1], k.shape[2]
    scale = D ** -0.5 if scale is None else scale
    u, dev = torch.finfo(q.dtype).eps / 2, q.device
    out = torch.zeros(B, Hq, Sq, D, dtype=torch.float64, device=dev)
    lse = torch.full((B, Hq, Sq), -math.inf, dtype=torch.float64, device=dev)
    out_off, lse_off = torch.zeros_like(out), torch.zeros_like(lse)
    slope = options(B, Hq, slopes)
    for b in range(B):
        seen, dist, kv = visible(b, Sq, Sk, causal, documents, documents_k, prefix_lens, kv_lens,
                                 dev)
        for h in range(Hq):
            x = Head(q[b, h], k[b, h * Hkv // Hq], scale, softcap, slope(b, h), seen, dist)
            vd = clean(v[b, h * Hkv // Hq].double(), x.keys)
            p = x.probabilities()
            n = seen.sum(1)
            out[b, h] = p @ vd
            lse[b, h] = torch.logsumexp(x.s, 1)
            dx = x.dx.amax(1) if Sk else torch.zeros(Sq, dtype=torch.float64, device=dev)
            # (n + 64) e: the sum over keys, exp2, log2, the join of split parts
            off = dx + (n + 64) * E
            lse_off[b, h] = torch.where(x.rows, off + 8 * E * lse[b, h].abs(),
                                        torch.zeros_like(off))
            size = p @ vd.abs()
            out_off[b, h] = size * (u + 2 * off[:, None]) * 1.01 + u * out[b, h].abs() * 1.01 + \
                smallest(q.dtype) * (vd.abs().sum(0)[None, :] + 2)
    return out, lse, out_off, lse_off


def backward(dout, q, k, v, out, lse, causal, scale=None, softcap=0.0, slopes=None,
             documents=None, documents_k=None, prefix_lens=None, kv_lens=None):
    """{name: (gradient, bound)} from the given out and lse, fp64."""
    B, Hq, Sq, D = q.shape
    Hkv, Sk = k.shape[1], k.shape[2]
    scale = D ** -0.5 if scale is None else scale
    u, dev, low = torch.finfo(q.dtype).eps / 2, q.device, smallest(q.dtype)
    zeros = {n: torch.zeros(t.shape, dtype=torch.float64, device=dev)
             for n, t in (("dq", q), ("dk", k), ("dv", v), ("delta", lse))}
    got = {n: t.clone() for n, t in zeros.items()}
    off = {n: t.clone() for n, t in zeros.items()}
    slope = options(B, Hq, slopes)
    for b in range(B):
        seen, dist, kv = visible(b, Sq, Sk, causal, documents, documents_k, prefix_lens, kv_lens,
                                 dev)
        for h in range(Hq):
            c = h * Hkv // Hq
            x = Head(q[b, h], k[b, c], scale, softcap, slope(b, h), seen, dist)
            vd = clean(v[b, c].double(), x.keys)
            do, o = (clean(t[b, h].double(), x.rows) for t in (dout, out))
            p = x.probabilities(lse[b, h].double())
            delta = (do * o).sum(1)
            dsize = (do.abs() * o.abs()).sum(1)
            dp = do @ vd.t().contiguous()
            ds = p * (dp - delta[:, None]) * x.slope
            # fp32: p by dx and lse's own size, dP and delta as dot products,
            # 1 - tanh^2 by a few e
            dx = x.dx + 8 * E * torch.where(x.rows, lse[b, h].double(),
                                            torch.zeros_like(delta)).abs()[:, None] + 16 * E
            dpsize = do.abs() @ vd.abs().t().contiguous()
            ds_off = p * ((D + 8) * E * (dpsize + dsize[:, None]) * x.slope +
                          (dp - delta[:, None]).abs() * (2 * dx * x.slope + 8 * E))
            p_off = p * 2 * dx + u * p + low * seen
            # (a P flushed to zero, 2^-126 at most, takes dS = P (dP - delta)
            # with it; then dS's own flush in fp32 and in the type)
            ds_off = ds_off + u * ds.abs() + \
                (2.0 ** -126 * ((dp - delta[:, None]).abs() + 1) + low) * seen
            n = torch.tensor(float(max(Sq * Hq // Hkv, Sk) + 8), dtype=torch.float64, device=dev)
            got["delta"][b, h] = delta
            off["delta"][b, h] = (D + 8) * E * dsize
            got["dq"][b, h] = scale * (ds @ x.k)
            off["dq"][b, h] = abs(scale) * ((ds_off + n * E * ds.abs()) @ x.k.abs())
            got["dk"][b, c] += scale * (ds.t().contiguous() @ x.q)
            off["dk"][b, c] += abs(scale) * ((ds_off + n * E * ds.abs()).t().contiguous() @ x.q.abs())
            got["dv"][b, c] += p.t().contiguous() @ do
            off["dv"][b, c] += (p_off + n * E * p).t().contiguous() @ do.abs()
    for n in ("dq", "dk", "dv"):
        off[n] = (off[n] + u * got[n].abs() + low) * 1.01
    return {n: (got[n], off[n]) for n in got}


def rotary(x, positions, freqs, interleaved, inverse=False):
    """The rotated x and its bound, fp64: the angle is reduced exactly, its
    fp32 remainder and the sine are off by 2^-22 together, the products and
    their sum by 2 e each, the result by half a step."""
    P = freqs.shape[1]
    angle = (positions.double()[..., None] * freqs.double()[:, None, None, :]).sum(0)[:, None]
    # fp64 angles: 2^-52 of their size off themselves
    loose = 2.0 ** -21 + angle.abs() * 2.0 ** -50
    cos, sin = torch.cos(angle), torch.sin(-angle if inverse else angle)
    y = x.double().clone()
    if interleaved:
        a, b = y[..., 0:2 * P:2].clone(), y[..., 1:2 * P:2].clone()
    else:
        a, b = y[..., :P].clone(), y[..., P:2 * P].clone()
    lo, hi = a * cos - b * sin, b * cos + a * sin
    off = torch.zeros_like(y)
    r = (a.abs() + b.abs()) * loose
    u = torch.finfo(x.dtype).eps / 2
    if interleaved:
        y[..., 0:2 * P:2], y[..., 1:2 * P:2] = lo, hi
        off[..., 0:2 * P:2], off[..., 1:2 * P:2] = r, r
    else:
        y[..., :P], y[..., P:2 * P] = lo, hi
        off[..., :P], off[..., P:2 * P] = r, r
    turned = torch.zeros(x.shape[-1], dtype=torch.bool, device=x.device)
    turned[:2 * P] = True
    off = torch.where(turned, (off + u * y.abs()) * 1.01 + smallest(x.dtype),
                      torch.zeros_like(off))
    return y, off
