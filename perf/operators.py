"""What the attention layer's operators are measured on.

A case is one pass through one operator, as a program that trains or serves
an attention layer calls it:

* "fwd"    torch.ops.shaobo_fa3.attn_forward: softmax attention whose scores
           may be capped by a tanh, biased by distance and masked (causal,
           prefix, documents, key lengths); prompts and single tokens;
* "bwd"    torch.ops.shaobo_fa3.attn_backward: its gradient from the saved
           output and log-sum-exp;
* "rotary" torch.ops.shaobo_fa3.rotary: positions on several axes applied to
           q and k, or their gradient (the inverse rotation).

Tensors are [batch, heads, sequence, head_dim]; "bshd" cases hold them as
[batch, sequence, heads, head_dim] and pass transposed views.  Document
lengths, key lengths and prefixes come from the case alone, values from the
seed.
"""
import math
import os
import random
import sys

import torch

own = False

_PKG = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                    "flash-attention3_amd")
if _PKG not in sys.path:
    sys.path.insert(0, _PKG)


def _attn(op, batch, heads_q, heads_kv, seq_q, seq_k, head_dim, dtype="bf16", layout="bhsd",
          causal=True, softcap=0.0, slopes=False, doc_len=0, prefix=0, ragged=False, **name):
    return {"op": op, "batch": batch, "heads_q": heads_q, "heads_kv": heads_kv, "seq_q": seq_q,
            "seq_k": seq_k, "head_dim": head_dim, "dtype": dtype, "layout": layout,
            "causal": causal, "softcap": softcap, "slopes": slopes, "doc_len": doc_len,
            "prefix": prefix, "ragged": ragged, **name}


def _rotary(batch, heads_q, heads_kv, seq, head_dim, axes, rotary_dim, dtype="bf16",
            layout="bshd", interleaved=False, inverse=False, start=0, **name):
    return {"op": "rotary", "batch": batch, "heads_q": heads_q, "heads_kv": heads_kv,
            "seq": seq, "head_dim": head_dim, "axes": axes, "rotary_dim": rotary_dim,
            "dtype": dtype, "layout": layout, "interleaved": interleaved, "inverse": inverse,
            "start": start, **name}


def listed():
    return [
        # a single token of one short conversation: all latency
        _attn("fwd", 1, 8, 2, 1, 129, 64, "fp16", name="fwd_token_s129_d64"),
        # a batch of single tokens over caches filled to different lengths, capped scores
        _attn("fwd", 16, 32, 8, 1, 8192, 128, softcap=30.0, ragged=True,
              name="fwd_tokens_gqa_s8192_cap"),
        # a long prompt in an odd number of tokens behind a bidirectional prefix (image and text)
        _attn("fwd", 1, 16, 4, 2011, 2011, 128, layout="bshd", softcap=50.0, prefix=600,
              name="fwd_prefix_cap_s2011"),
        # training on samples packed into rows, grouped-query heads
        _attn("fwd", 2, 32, 8, 4096, 4096, 128, layout="bshd", doc_len=1500,
              name="fwd_docs_gqa_s4096"),
        # the largest: full attention with a distance bias over long rows (encoders)
        _attn("fwd", 2, 16, 16, 8192, 8192, 64, "fp16", causal=False, slopes=True,
              name="fwd_bias_full_s8192_d64"),
        # a short fine-tuning step's gradient, capped scores
        _attn("bwd", 2, 8, 8, 256, 256, 64, softcap=30.0, name="bwd_cap_s256_d64"),
        # an odd number of heads and tokens, distance bias, samples packed with a padded end
        _attn("bwd", 1, 7, 7, 1923, 1923, 128, "fp16", slopes=True, doc_len=700,
              name="bwd_bias_docs_s1923"),
        # prefix training with capped scores, grouped-query heads
        _attn("bwd", 4, 16, 4, 1024, 1024, 128, layout="bshd", softcap=50.0, prefix=300,
              name="bwd_prefix_cap_gqa_s1024"),
        # the largest gradient: packed samples, grouped-query heads
        _attn("bwd", 2, 32, 8, 4096, 4096, 128, layout="bshd", doc_len=1500,
              name="bwd_docs_gqa_s4096"),
        # the single tokens of a batch being served, far positions
        _rotary(16, 32, 8, 1, 128, 3, 128, start=1000000, name="rotary_token_b16"),
        # a vision encoder's odd-sized grid, two axes, neighbouring pairs, half of the dims
        _rotary(3, 12, 12, 1369, 64, 2, 32, "fp32", "bhsd", interleaved=True,
                name="rotary_grid_fp32_s1369"),
        # the gradient of a training batch's rotation, three axes
        _rotary(2, 32, 8, 8192, 128, 3, 128, inverse=True, name="rotary_grad_s8192"),
    ]


def draw(rng):
    """One case of the ranges above: tokens from 1 (gradients: 16) to 8192, batch x
    heads from 1 to 512 and cache lengths to 16384, over their logarithms; at most 2.2e9
    scores (half of that for gradients)."""
    def log_int(low, high):
        return max(low, min(high, round(math.exp(rng.uniform(math.log(low), math.log(high))))))

    while True:
        op = rng.choice(["fwd", "fwd", "token", "bwd", "bwd", "rotary"])
        batch = log_int(1, 16)
        group = rng.choice([1, 1, 2, 3, 4, 8])
        heads_kv = log_int(1, 16)
        heads_q = heads_kv * group
        if batch * heads_q > 512:
            continue
        dtype = rng.choice(["bf16", "bf16", "fp16"])
        layout = rng.choice(["bhsd", "bshd"])
        head_dim = rng.choice([64, 128])
        if op == "rotary":
            axes = rng.choice([1, 2, 3])
            case = _rotary(batch, heads_q, heads_kv, log_int(1, 8192), head_dim, axes,
                           rng.choice([head_dim, head_dim, head_dim // 2]),
                           rng.choice([dtype, dtype, "fp32"]), layout, rng.random() < 0.4,
                           rng.random() < 0.4, rng.choice([0, 1000000]))
            if work(case)["bytes"] <= 7e8:
                return case
            continue
        softcap = rng.choice([0.0, 0.0, 30.0, 50.0])
        slopes = rng.random() < 0.35
        if op == "token":
            seq_k = log_int(1, 16384)
            case = _attn("fwd", batch, heads_q, heads_kv, min(seq_k, rng.choice([1, 1, 1, 2, 5])),
                         seq_k, head_dim, dtype, layout, True, softcap, slopes,
                         ragged=rng.random() < 0.6)
        else:
            # (a row that sees one key alone has no gradient in q and k)
            least = 16 if op == "bwd" else 1
            seq = log_int(least, 8192)
            causal = rng.random() < 0.7
            doc_len = rng.choice([0, 0, max(least, seq // 3), max(least, seq // 12)])
            prefix = seq // 3 if causal and not doc_len and rng.random() < 0.4 else 0
            case = _attn(op, batch, heads_q, heads_kv, seq, seq, head_dim, dtype, layout, causal,
                         softcap, slopes, doc_len, prefix)
        scores = batch * heads_q * case["seq_q"] * case["seq_k"]
        cache = 4 * batch * heads_kv * case["seq_k"] * head_dim
        if scores <= (1.1e9 if op == "bwd" else 2.2e9) and cache <= 6e8:
            return case


# ---------------------------------------------------------------------------
# What a case's masks are: plain lists made from the case alone.
def _rng_of(case):
    return random.Random(repr([(k, case[k]) for k in sorted(case) if k != "name"]))


def _kv_lens(case):
    """Filled part of each row's keys: all of it, or ragged ones with at
    least as many keys as queries."""
    if not case["ragged"]:
        return [case["seq_k"]] * case["batch"]
    rng = _rng_of(case)
    low = min(case["seq_q"], case["seq_k"])
    return [rng.randint(max(low, case["seq_k"] // 4), case["seq_k"])
            for _ in range(case["batch"])]


def _prefixes(case):
    rng = _rng_of(case)
    return [rng.randint(case["prefix"] // 2, case["prefix"]) for _ in range(case["batch"])]


def _documents(case):
    """Lengths of the documents of each row; the rest of the row is padding."""
    rng = _rng_of(case)
    rows = []
    for _ in range(case["batch"]):
        left, lens = case["seq_q"], []
        while left > 0:
            n = max(1, min(left, round(case["doc_len"] * math.exp(rng.gauss(0.0, 0.7)))))
            if n == left and rng.random() < 0.5 and lens:
                break
            lens.append(n)
            left -= n
        rows.append(lens)
    return rows


def _pairs(case):
    """Visible (query, key) pairs of one head, over the batch."""
    total = 0
    for b, kv in enumerate(_kv_lens(case)):
        sq = case["seq_q"]
        if case["doc_len"]:
            spans, at = [], 0
            for n in _documents(case)[b]:
                spans.append((at, at + n))
                at += n
        else:
            spans = [(0, max(sq, kv))]
        prefix = _prefixes(case)[b] if case["prefix"] else 0
        off = kv - sq
        for first, last in spans:
            if not case["causal"]:
                rows = min(last, sq) - first
                total += max(0, rows) * max(0, min(last, kv) - first)
            else:  # row i sees keys first .. max(i + off + 1, prefix), inside its span
                for i in range(first, min(last, sq)):
                    total += max(0, min(max(i + off + 1, prefix), last, kv) - first)
    return total


def work(case):
    """bytes: each tensor read or written once (of the keys and values the
    filled part); flops: 4 D a visible pair forward, 10 D backward."""
    D, B, Hq, Hkv = (case[n] for n in ("head_dim", "batch", "heads_q", "heads_kv"))
    if case["op"] == "rotary":
        size = 4 if case["dtype"] == "fp32" else 2
        x = B * case["seq"] * (Hq + Hkv) * D
        return {"bytes": 2 * size * x + 4 * case["axes"] * B * case["seq"],
                "flops": 3.0 * B * case["seq"] * (Hq + Hkv) * case["rotary_dim"]}
    rows, keys = B * Hq * case["seq_q"], Hkv * sum(_kv_lens(case))
    pairs = float(Hq) * _pairs(case)
    if case["op"] == "fwd":
        return {"bytes": rows * (4 * D + 4) + keys * 4 * D, "flops": 4.0 * D * pairs}
    return {"bytes": rows * (8 * D + 8) + keys * 4 * D + B * Hkv * case["seq_k"] * 4 * D,
            "flops": 10.0 * D * pairs}


# ---------------------------------------------------------------------------
_TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


class _State:
    pass


def _randn(gen, case, heads, seq, std=1.0):
    B, D = case["batch"], case["head_dim"]
    shape = (B, seq, heads, D) if case["layout"] == "bshd" else (B, heads, seq, D)
    x = (torch.randn(shape, generator=gen, device="cuda") * std).to(_TYPES[case["dtype"]])
    return x.transpose(1, 2) if case["layout"] == "bshd" else x


def _inputs(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(1000003 * (seed + 1))
    st = _State()
    st.op = case["op"]
    if st.op == "rotary":
        B, S, axes, P = case["batch"], case["seq"], case["axes"], case["rotary_dim"] // 2
        st.q = _randn(gen, case, case["heads_q"], S)
        st.k = _randn(gen, case, case["heads_kv"], S)
        # a token's place: the slowest axis counts on, the others run over a grid
        at = torch.arange(S, device="cuda") + case["start"] + 17 * (seed % 5)
        side = max(1, math.isqrt(S))
        places = [at] if axes == 1 else [at // side, at % side] if axes == 2 else \
            [at // (side * 2), at // 7 % side, at % side]
        st.positions = torch.stack(places).to(torch.int32)[:, None, :].expand(
            axes, B, S).contiguous()
        # each axis owns a run of the pairs; pair p turns by theta^(-p / P) a step
        p = torch.arange(P, device="cuda")
        inv = (10000.0 ** (-p.double() / P)).float()
        st.freqs = torch.where((p * axes // P)[None] == torch.arange(axes, device="cuda")[:, None],
                               inv[None], torch.zeros((), device="cuda"))
        st.interleaved, st.inverse = case["interleaved"], case["inverse"]
        return st
    B, Hq, Hkv, Sq, Sk = (case[n] for n in ("batch", "heads_q", "heads_kv", "seq_q", "seq_k"))
    # (capped scores: queries large enough to reach the cap)
    st.q = _randn(gen, case, Hq, Sq, 4.0 if case["softcap"] else 1.0)
    st.k, st.v = _randn(gen, case, Hkv, Sk), _randn(gen, case, Hkv, Sk)
    st.causal, st.scale, st.softcap = case["causal"], case["head_dim"] ** -0.5, case["softcap"]
    st.slopes = st.documents = st.prefix_lens = st.kv_lens = None
    if case["slopes"]:
        h = torch.arange(1, Hq + 1, device="cuda", dtype=torch.float32)
        st.slopes = torch.exp2(-8.0 * h / Hq)
    if case["doc_len"]:
        ids = torch.full((B, Sq), -1, dtype=torch.int32)
        for b, lens in enumerate(_documents(case)):
            at = 0
            for n, length in enumerate(lens):
                ids[b, at:at + length] = n + seed % 3
                at += length
        st.documents = ids.cuda()
    if case["prefix"]:
        st.prefix_lens = torch.tensor(_prefixes(case), dtype=torch.int32, device="cuda")
    if case["ragged"]:
        st.kv_lens = torch.tensor(_kv_lens(case), dtype=torch.int32, device="cuda")
    if st.op == "bwd":
        st.dout = _randn(gen, case, Hq, Sq)
        out, st.lse = _forward(st)
        st.out = torch.empty_like(st.q).copy_(out)
    return st


def prepare(case, seed):
    return _inputs(case, seed)


# ---------------------------------------------------------------------------
# The plain forms.
def _visible(st):
    """[B, 1, Sq, Sk] truth values, and i + offset - j as fp32."""
    B, Sq, Sk = st.q.shape[0], st.q.shape[2], st.k.shape[2]
    i = torch.arange(Sq, device="cuda")[None, :, None]
    j = torch.arange(Sk, device="cuda")[None, None, :]
    kv = st.kv_lens.long()[:, None, None] if st.kv_lens is not None else \
        torch.full((B, 1, 1), Sk, device="cuda")
    far = i + kv - Sq - j
    seen = (j < kv).expand(B, Sq, Sk)
    if st.causal:
        back = far >= 0
        if st.prefix_lens is not None:
            back = back | (j < st.prefix_lens.long()[:, None, None])
        seen = seen & back
    if st.documents is not None:
        dq, dk = st.documents[:, :, None], st.documents[:, None, :Sk]
        seen = seen & (dq == dk) & (dq >= 0)
    return seen[:, None], far[:, None]


def _scores(st):
    """Masked fp32 scores [B, Hq, Sq, Sk], and the tanh where they are capped."""
    B, Hq, Sq, D = st.q.shape
    Hkv, Sk = st.k.shape[1], st.k.shape[2]
    q = st.q.float().reshape(B, Hkv, Hq // Hkv * Sq, D)
    s = torch.matmul(q, st.k.float().transpose(2, 3)).mul_(st.scale).view(B, Hq, Sq, Sk)
    t = None
    if st.softcap:
        t = torch.tanh(s / st.softcap)
        s = t * st.softcap
    seen, far = _visible(st)
    if st.slopes is not None:
        s = s - st.slopes[:, None, None] * far.abs()
    return s.masked_fill_(~seen, float("-inf")), t


def _forward(st):
    B, Hq, Sq, D = st.q.shape
    Hkv, Sk = st.k.shape[1], st.k.shape[2]
    s, _ = _scores(st)
    m = s.amax(-1, keepdim=True)
    m = torch.where(m == float("-inf"), torch.zeros_like(m), m)
    p = torch.exp(s - m)
    z = p.sum(-1, keepdim=True)
    o = torch.matmul(p.view(B, Hkv, Hq // Hkv * Sq, Sk), st.v.float()).view(B, Hq, Sq, D)
    o = o / torch.where(z == 0, torch.ones_like(z), z)
    return o.to(st.q.dtype), (m + torch.log(z)).squeeze(-1)


def _backward(st):
    B, Hq, Sq, D = st.q.shape
    Hkv, Sk = st.k.shape[1], st.k.shape[2]
    rows = Hq // Hkv * Sq
    s, t = _scores(st)
    lse = torch.where(st.lse == float("-inf"), torch.zeros_like(st.lse), st.lse)
    p = torch.exp(s - lse[..., None])
    del s
    do = st.dout.float()
    delta = (do * st.out.float()).sum(-1)
    do = do.reshape(B, Hkv, rows, D)
    dv = torch.matmul(p.view(B, Hkv, rows, Sk).transpose(2, 3), do)
    ds = torch.matmul(do, st.v.float().transpose(2, 3)).view(B, Hq, Sq, Sk)
    ds = ds.sub_(delta[..., None]).mul_(p).mul_(st.scale)
    if t is not None:
        ds = ds * (1.0 - t * t)
    ds = ds.view(B, Hkv, rows, Sk)
    dq = torch.matmul(ds, st.k.float()).view(B, Hq, Sq, D)
    dk = torch.matmul(ds.transpose(2, 3), st.q.float().reshape(B, Hkv, rows, D))
    return dq.to(st.q.dtype), dk.to(st.q.dtype), dv.to(st.q.dtype), delta


def _turn(st, x):
    angle = (st.positions.double()[..., None] * st.freqs.double()[:, None, None, :]).sum(0)
    cos, sin = torch.cos(angle).float()[:, None], torch.sin(angle).float()[:, None]
    if st.inverse:
        sin = -sin
    P = st.freqs.shape[1]
    f = x.float()
    r, rest = f[..., :2 * P], f[..., 2 * P:]
    if st.interleaved:
        a, b = r[..., 0::2], r[..., 1::2]
        y = torch.stack((a * cos - b * sin, b * cos + a * sin), -1).flatten(-2)
    else:
        a, b = r[..., :P], r[..., P:]
        y = torch.cat((a * cos - b * sin, b * cos + a * sin), -1)
    return torch.cat((y, rest), -1).to(x.dtype)


def run(st):
    if own:
        import shaobo_fa3_torch  # noqa: F401  (registers the operators)
        ops = torch.ops.shaobo_fa3
        if st.op == "rotary":
            q, k = ops.rotary([st.q, st.k], st.positions, st.freqs, st.interleaved, st.inverse)
            return {"q": q, "k": k}
        mask = (st.causal, st.scale, st.softcap, st.slopes, st.documents, None, st.prefix_lens,
                st.kv_lens)
        if st.op == "fwd":
            out, lse = ops.attn_forward(st.q, st.k, st.v, *mask)
            return {"out": out, "lse": lse}
        dq, dk, dv, delta = ops.attn_backward(st.dout, st.q, st.k, st.v, st.out, st.lse, *mask)
        return {"dq": dq, "dk": dk, "dv": dv, "delta": delta}
    if st.op == "rotary":
        return {"q": _turn(st, st.q), "k": _turn(st, st.k)}
    if st.op == "fwd":
        out, lse = _forward(st)
        return {"out": out, "lse": lse}
    dq, dk, dv, delta = _backward(st)
    return {"dq": dq, "dk": dk, "dv": dv, "delta": delta}


# ---------------------------------------------------------------------------
def exact(case, seed):
    """The operators' definitions in fp64, head by head."""
    st = _inputs(case, seed)
    if st.op == "rotary":
        return {"q": _exact_turn(case, st, st.q), "k": _exact_turn(case, st, st.k)}
    B, Hq, Sq, D = st.q.shape
    Hkv, Sk = st.k.shape[1], st.k.shape[2]
    group = Hq // Hkv
    kv_lens, docs = _kv_lens(case), st.documents
    prefixes = _prefixes(case) if case["prefix"] else [0] * B
    i = torch.arange(Sq, device="cuda").unsqueeze(1)
    j = torch.arange(Sk, device="cuda").unsqueeze(0)
    out = {n: torch.zeros(s, dtype=torch.float64, device="cuda") for n, s in (
        (("out", (B, Hq, Sq, D)), ("lse", (B, Hq, Sq))) if st.op == "fwd" else
        (("dq", (B, Hq, Sq, D)), ("dk", (B, Hkv, Sk, D)), ("dv", (B, Hkv, Sk, D)),
         ("delta", (B, Hq, Sq))))}
    for b in range(B):
        last = i + (kv_lens[b] - Sq)  # the row's own place among the keys
        hidden = (j >= kv_lens[b]).expand(Sq, Sk)
        if case["causal"]:
            hidden = hidden | ((j > last) & (j >= prefixes[b]))
        if docs is not None:
            hidden = hidden | (docs[b].unsqueeze(1) != docs[b].unsqueeze(0)) | \
                (docs[b].unsqueeze(1) < 0)
        for h in range(Hq):
            q, k, v = st.q[b, h].double(), st.k[b, h // group].double(), \
                st.v[b, h // group].double()
            x = (q @ k.t().contiguous()) / math.sqrt(D)
            slope = 1.0
            if case["softcap"]:
                x = torch.tanh(x / case["softcap"])
                slope = 1.0 - x ** 2
                x = x * case["softcap"]
            if st.slopes is not None:
                x -= float(st.slopes[h]) * (last - j).abs()
            x = torch.where(hidden, torch.full_like(x, -math.inf), x)
            if st.op == "fwd":
                out["lse"][b, h] = torch.logsumexp(x, 1)
                out["out"][b, h] = torch.nan_to_num(torch.softmax(x, 1), nan=0.0) @ v
                continue
            do = st.dout[b, h].double()
            p = torch.where(hidden, torch.zeros_like(x),
                            torch.exp(x - st.lse[b, h].double().unsqueeze(1)))
            delta = torch.sum(do * st.out[b, h].double(), 1)
            ds = p * (do @ v.t().contiguous() - delta.unsqueeze(1)) * slope / math.sqrt(D)
            out["delta"][b, h] = delta
            out["dq"][b, h] = ds @ k
            out["dk"][b, h // group] += ds.t().contiguous() @ q
            out["dv"][b, h // group] += p.t().contiguous() @ do
    return out


def _exact_turn(case, st, x):
    P = case["rotary_dim"] // 2
    turn = torch.zeros(st.positions.shape[1:] + (P,), dtype=torch.float64, device="cuda")
    for a in range(case["axes"]):
        turn += st.positions[a].double().unsqueeze(-1) * st.freqs[a].double()
    turn = torch.polar(torch.ones_like(turn), -turn if case["inverse"] else turn).unsqueeze(1)
    y = x.double().clone()
    low, high = (slice(0, 2 * P, 2), slice(1, 2 * P, 2)) if case["interleaved"] else \
        (slice(0, P), slice(P, 2 * P))
    z = torch.complex(y[..., low].contiguous(), y[..., high].contiguous()) * turn
    y[..., low], y[..., high] = z.real, z.imag
    return y
