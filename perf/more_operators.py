"""What the paged cache's operators are measured on.

A case is one pass through one operator, as a program that serves an attention
layer calls it:

* "append" torch.ops.shaobo_fa3.cache_append: new tokens' keys turned by their
           positions and written, with the values, into the pages of a cache;
           queries turned on the way.  A cache held in 4 bits is read back by
           torch.ops.shaobo_fa3.cache_read, as a program does that hands it on:
           what its codes stand for is the output;
* "attn"   torch.ops.shaobo_fa3.cache_attn: attention of the new tokens to the
           pages of their sequence, held in 16 bits or in 4;
* "sparse" torch.ops.shaobo_fa3.cache_select and cache_attn: the pages that a
           bound of their scores selects for each new token, and attention to
           those alone.

New tokens are [batch, heads, sequence, head_dim], the last of their sequence's
positions; "bshd" cases hold them as [batch, sequence, heads, head_dim] and pass
transposed views.  Lengths come from the case alone, the order of the pages and
all values from the seed.

A row of a 4-bit cache is head_dim codes (a sign and one of the levels 0, 1/2,
1, 3/2, 2, 3, 4, 6; two a byte, the first in the low half) and one fp32 scale;
of a page and head first all codes are held, then all scales.
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


def _case(op, batch, heads_q, heads_kv, head_dim, seq, cache, bits=16, page=64, dtype="bf16",
          layout="bshd", ragged=False, padded=False, bounds=False, rotary_dim=0, axes=1,
          interleaved=False, softcap=0.0, slopes=False, count=0, **name):
    return {"op": op, "batch": batch, "heads_q": heads_q, "heads_kv": heads_kv,
            "head_dim": head_dim, "seq": seq, "cache": cache, "bits": bits, "page": page,
            "dtype": dtype, "layout": layout, "ragged": ragged, "padded": padded,
            "bounds": bounds, "rotary_dim": rotary_dim, "axes": axes, "interleaved": interleaved,
            "softcap": softcap, "slopes": slopes, "count": count, **name}


def listed():
    return [
        # the next token of one conversation: all latency
        _case("append", 1, 32, 8, 128, 1, 1025, rotary_dim=128, name="append_token_b1"),
        # the next tokens of a batch being served, pages with bounds
        _case("append", 64, 32, 8, 128, 1, 1024, ragged=True, bounds=True, rotary_dim=128,
              name="append_tokens_b64_bounds"),
        # a long prompt
        _case("append", 1, 32, 8, 128, 8192, 8192, rotary_dim=128, name="append_prompt_s8192"),
        # a batch of short prompts of odd lengths into 4 bits, neighbouring pairs, two axes
        _case("append", 3, 16, 16, 64, 411, 411, bits=4, page=32, dtype="fp16", padded=True,
              rotary_dim=32, axes=2, interleaved=True, layout="bhsd", name="append4_prompts_s411_d64"),
        # a later part of a long prompt into 4 bits, pages with bounds
        _case("append", 2, 32, 8, 128, 2048, 4096, bits=4, bounds=True, rotary_dim=128,
              name="append4_part_s2048_bounds"),
        # a single token of one short conversation: all latency
        _case("attn", 1, 8, 2, 64, 1, 129, dtype="fp16", page=32, name="attn_token_s129_d64"),
        # a batch of single tokens over sequences of different lengths, capped scores
        _case("attn", 16, 32, 8, 128, 1, 8192, ragged=True, softcap=30.0,
              name="attn_tokens_b16_s8192_cap"),
        # the largest cache, in 4 bits
        _case("attn", 48, 32, 8, 128, 1, 16384, bits=4, ragged=True,
              name="attn4_tokens_b48_s16384"),
        # drafted tokens to be checked, distance bias, 4 bits
        _case("attn", 8, 16, 4, 128, 5, 6001, bits=4, page=32, dtype="fp16", ragged=True,
              slopes=True, layout="bhsd", name="attn4_drafts_s6001_bias"),
        # a later part of a long prompt over what is there, 4 bits
        _case("attn", 1, 32, 8, 128, 1531, 9211, bits=4, name="attn4_part_s1531"),
        # one very long sequence's next token, 64 of its 2048 pages
        _case("sparse", 1, 32, 8, 128, 1, 131072, bits=4, count=64, name="sparse4_token_s131072"),
        # a batch of them
        _case("sparse", 16, 32, 8, 128, 1, 32768, ragged=True, count=48,
              name="sparse_tokens_b16_s32768"),
    ]


def draw(rng):
    """One case of the ranges above: new tokens from 1 to 8192, sequences to 131072 tokens,
    batch x query heads from 1 to 2048, over their logarithms; caches up to 2.2e9 bytes in 16
    bits (appended ones up to 2e8) and at most 4e8 scores."""
    def log_int(low, high):
        return max(low, min(high, round(math.exp(rng.uniform(math.log(low), math.log(high))))))

    while True:
        op = rng.choice(["append", "append", "attn", "attn", "attn", "sparse"])
        kind = rng.choice(["token", "token", "draft", "part"])
        group = rng.choice([1, 2, 3, 4, 4, 8])
        heads_kv, head_dim = log_int(1, 16), rng.choice([64, 128, 128])
        batch = log_int(1, 64) if kind == "token" else log_int(1, 8)
        common = dict(bits=rng.choice([16, 4]), page=rng.choice([32, 64, 64, 128]),
                      dtype=rng.choice(["bf16", "bf16", "fp16"]),
                      layout=rng.choice(["bhsd", "bshd"]), ragged=rng.random() < 0.5)
        seq = 1 if kind == "token" else rng.randint(2, 8) if kind == "draft" else \
            log_int(9, 8192 if op == "append" else 2048)
        if op == "sparse":
            if kind == "part":
                continue
            cache = log_int(2048, 131072)
            case = _case(op, batch, heads_kv * group, heads_kv, head_dim, seq, cache,
                         count=rng.choice([8, 16, 33, 64]), **common)
        elif op == "append":
            cache = seq + (0 if rng.random() < 0.5 else log_int(1, 2048))
            case = _case(op, batch, heads_kv * group, heads_kv, head_dim, seq, cache,
                         padded=seq > 8 and rng.random() < 0.4, bounds=rng.random() < 0.5,
                         rotary_dim=rng.choice([head_dim, head_dim, head_dim // 2]),
                         axes=rng.choice([1, 1, 2, 3]), interleaved=rng.random() < 0.3, **common)
        else:
            cache = max(seq, log_int(1, 16384))
            case = _case(op, batch, heads_kv * group, heads_kv, head_dim, seq, cache,
                         softcap=rng.choice([0.0, 0.0, 30.0]), slopes=rng.random() < 0.3, **common)
        if case["ragged"] and cache < 8 * seq:
            case["ragged"] = False
        held = 4 * batch * heads_kv * cache * head_dim
        scores = batch * heads_kv * group * seq * cache
        if batch * heads_kv * group > 2048 or held > 2.2e9 or \
                (op == "append" and work(case)["bytes"] > 2e8) or (op == "attn" and scores > 4e8):
            continue
        return case


# ---------------------------------------------------------------------------
# What a case's lengths are: plain lists made from the case alone.
def _rng_of(case):
    return random.Random(repr([(k, case[k]) for k in sorted(case) if k != "name"]))


def _lens(case):
    """Tokens of each sequence with the new ones, and how many of them are new."""
    rng, new, kv = _rng_of(case), [], []
    for _ in range(case["batch"]):
        n = rng.randint(max(1, case["seq"] // 2), case["seq"]) if case["padded"] else case["seq"]
        old = case["cache"] - case["seq"]
        if case["ragged"]:
            old = rng.randint(old // 4, old)
        new.append(n)
        kv.append(old + n)
    return kv, new


def _pages_of(case):
    return [-(-kv // case["page"]) for kv in _lens(case)[0]]


def work(case):
    """bytes: each row that is needed read or written once; flops: 4 D a
    visible pair of attention, 4 a channel of a page's bound, 6 a turned pair."""
    B, Hq, Hkv, D, S, ps = (case[n] for n in ("batch", "heads_q", "heads_kv", "head_dim", "seq",
                                              "page"))
    kv, new = _lens(case)
    row = 2 * D if case["bits"] == 16 else D // 2 + 4
    if case["op"] == "append":
        tokens = sum(new)
        nbytes = B * S * Hq * 4 * D + tokens * Hkv * 2 * (2 * D + row)
        if case["bounds"]:
            nbytes += sum((k - 1) // ps - (k - n) // ps + 1 for k, n in zip(kv, new)) * Hkv * 4 * D
        if case["bits"] == 4:
            nbytes += 2 * Hkv * (sum(kv) * row + B * case["cache"] * 2 * D)
        return {"bytes": nbytes, "flops": 3.0 * B * S * (Hq + Hkv) * case["rotary_dim"]}
    rows = B * Hq * S
    nbytes, flops = rows * (4 * D + 4), 0.0
    if case["op"] == "attn":
        nbytes += 2 * Hkv * sum(kv) * row
        pairs = sum(n * (k - n) + n * (n + 1) // 2 for k, n in zip(kv, new))
        return {"bytes": nbytes, "flops": 4.0 * D * Hq * pairs}
    for k in kv:
        for i in range(S):
            last = k - S + i
            pages = min(case["count"], last // ps + 1)
            keys = (pages - 1) * ps + last % ps + 1
            # (pages may be shared by a sequence's new tokens: counted once)
            nbytes += (2 * Hkv * keys * row if i == S - 1 else 0) + 4 * Hkv * pages
            flops += 4.0 * D * Hq * (keys + last // ps)
        nbytes += Hkv * (k // ps) * 4 * D
    return {"bytes": nbytes, "flops": flops}


# ---------------------------------------------------------------------------
_TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


class _State:
    pass


def _new_rows(gen, case, heads, std=1.0):
    B, S, D = case["batch"], case["seq"], case["head_dim"]
    shape = (B, S, heads, D) if case["layout"] == "bshd" else (B, heads, S, D)
    x = (torch.randn(shape, generator=gen, device="cuda") * std).to(_TYPES[case["dtype"]])
    return x.transpose(1, 2) if case["layout"] == "bshd" else x


def _held_rows(gen, case, pages, keys):
    """Rows that the cache holds before the call; a few channels of keys are large."""
    H, D = case["heads_kv"], case["head_dim"]
    x = torch.randn(pages, H, case["page"], D, generator=gen, device="cuda")
    if keys:
        wide = torch.rand(H, 1, D, generator=gen, device="cuda")
        x.mul_(0.7 + 1.5 * (wide > 0.95)).add_(torch.randn(H, 1, D, generator=gen, device="cuda"),
                                               alpha=0.5)
    return x.to(_TYPES[case["dtype"]])


def _inputs(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(1000003 * (seed + 1))
    B, S, ps, Hq, Hkv = (case[n] for n in ("batch", "seq", "page", "heads_q", "heads_kv"))
    st = _State()
    st.op, st.bits, st.page = case["op"], case["bits"], ps
    st.type, st.head_dim = _TYPES[case["dtype"]], case["head_dim"]
    kv, new = _lens(case)
    used = _pages_of(case)
    pages = sum(used) + 2
    order = torch.randperm(pages, generator=gen, device="cuda").to(torch.int32)
    # pages of the sequences one after the other in the order; -1 behind them
    width = -(-case["cache"] // ps)
    u = torch.tensor(used, device="cuda")
    slot = torch.arange(width, device="cuda")[None, :]
    at = (torch.cumsum(u, 0) - u)[:, None] + slot
    st.page_table = torch.where(slot < u[:, None], order[at.clamp(max=pages - 1)],
                                torch.full((), -1, dtype=torch.int32, device="cuda"))
    st.kv_lens = torch.tensor(kv, dtype=torch.int32, device="cuda")
    st.new_lens = torch.tensor(new, dtype=torch.int32, device="cuda") if case["padded"] else None
    k = _held_rows(gen, case, pages, True)
    st.bounds = None
    if case["bounds"] or case["op"] == "sparse":
        # (of the page's rows that are there; the last page of a sequence may end early)
        there = torch.zeros(pages, dtype=torch.int64, device="cuda")
        held = st.kv_lens.long() - (torch.tensor(new, device="cuda") if st.op == "append" else 0)
        rows = (held[:, None] - slot * ps).clamp(0, ps)
        there[st.page_table[st.page_table >= 0].long()] = rows[st.page_table >= 0]
        seen = (torch.arange(ps, device="cuda") < there[:, None])[:, None, :, None]
        seen = seen | (there == 0)[:, None, None, None]
        inf = torch.full((), math.inf, dtype=k.dtype, device="cuda")
        st.bounds = torch.stack((torch.where(seen, k, inf).amin(2),
                                 torch.where(seen, k, -inf).amax(2)), 2)
    st.k_pages = _pack(k) if st.bits == 4 else k
    del k
    v = _held_rows(gen, case, pages, False)
    st.v_pages = _pack(v) if st.bits == 4 else v
    del v
    if st.op == "append":
        st.q, st.k, st.v = (_new_rows(gen, case, h) for h in (Hq, Hkv, Hkv))
        P, axes = case["rotary_dim"] // 2, case["axes"]
        st.interleaved = case["interleaved"]
        p = torch.arange(P, device="cuda")
        inv = (10000.0 ** (-p.double() / P)).float()
        # one axis: the token's place; more: a grid of them, each axis owning a run of the pairs
        st.positions = None
        if axes > 1:
            t = torch.arange(S, device="cuda") + 17 * (seed % 5)
            side = max(1, math.isqrt(S))
            places = [t // side, t % side, t // 7 % side][:axes]
            st.positions = torch.stack(places).to(torch.int32)[:, None, :].expand(
                axes, B, S).contiguous()
        owner = (p * axes // P)[None] == torch.arange(axes, device="cuda")[:, None]
        st.freqs = torch.where(owner, inv[None], torch.zeros((), device="cuda"))
        st.seqlen = case["cache"]
        return st
    st.q = _new_rows(gen, case, Hq, 4.0 if case["softcap"] else 1.0)
    st.scale, st.softcap, st.count = case["head_dim"] ** -0.5, case["softcap"], case["count"]
    st.slopes = None
    if case["slopes"]:
        st.slopes = torch.exp2(-8.0 * torch.arange(1, Hq + 1, device="cuda").float() / Hq)
    return st


def prepare(case, seed):
    return _inputs(case, seed)


# ---------------------------------------------------------------------------
# The plain forms.
_LEVELS = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def _pack(x):
    """[pages, H, page, D] rows as a 4-bit cache holds them."""
    pages, H, ps, D = x.shape
    x = x.float()
    top = x.abs().amax(-1, keepdim=True)
    # six times a magnitude against the midpoints of the levels (fp32 holds both
    # products exactly; on a midpoint the even code)
    y = 6.0 * x.abs()
    code = torch.zeros(x.shape, dtype=torch.uint8, device=x.device)
    for n, mid in enumerate((0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0)):
        edge = mid * top
        code += (y >= edge) if n % 2 else (y > edge)
    code = torch.where(top == 0, torch.zeros_like(code), code) | (8 * (x < 0)).to(torch.uint8)
    scale = torch.where(torch.isfinite(top), top / 6.0, torch.full_like(top, math.nan))
    codes = (code[..., 0::2] | (code[..., 1::2] << 4)).reshape(pages, H, ps * D // 2)
    scales = scale.reshape(pages, H, ps).view(torch.uint8)
    return torch.cat((codes, scales), 2).view(pages, H, ps, D // 2 + 4)


def _parts(pages):
    """Codes [pages, H, page, D / 2] and scales [pages, H, page] of a 4-bit cache, as views."""
    n, H, ps, row = pages.shape
    flat = pages.view(n, H, ps * row)
    codes = flat[..., :ps * (row - 4)].unflatten(2, (ps, row - 4))
    return codes, flat[..., ps * (row - 4):].view(torch.float32)


def _rows(st, pages, at):
    """fp32 rows [B, H, ..., page, D] of the pages `at`, [B, n] of all heads or [B, H, S, n]."""
    H = pages.shape[1]
    at = (at.unsqueeze(1) if at.dim() == 2 else at).clamp(min=0).long()
    heads = torch.arange(H, device="cuda").view(1, H, *([1] * (at.dim() - 2)))
    if st.bits == 16:
        return pages[at, heads].float()
    codes, scales = _parts(pages)
    c = codes[at, heads]
    c = torch.stack((c & 15, c >> 4), -1).flatten(-2).int()
    level = torch.tensor(_LEVELS + tuple(-x for x in _LEVELS), device="cuda")
    return level[c].mul_(scales[at, heads].unsqueeze(-1))


def _turned(st, x, place):
    """x turned by its positions, in fp64 (a row of 4-bit codes goes by its 16-bit values)."""
    pos = place[None] if st.positions is None else st.positions
    angle = (pos.double()[..., None] * st.freqs.double()[:, None, None, :]).sum(0)
    cos, sin = torch.cos(angle)[:, None], torch.sin(angle)[:, None]
    P = st.freqs.shape[1]
    f = x.double()
    r, rest = f[..., :2 * P], f[..., 2 * P:]
    if st.interleaved:
        a, b = r[..., 0::2], r[..., 1::2]
        y = torch.stack((a * cos - b * sin, b * cos + a * sin), -1).flatten(-2)
    else:
        a, b = r[..., :P], r[..., P:]
        y = torch.cat((a * cos - b * sin, b * cos + a * sin), -1)
    return torch.cat((y, rest), -1).to(x.dtype)


def _append(st):
    B, Hkv, S, D = st.k.shape
    i = torch.arange(S, device="cuda")[None, :]
    new = st.new_lens.long()[:, None] if st.new_lens is not None else \
        torch.full((B, 1), S, device="cuda")
    place = st.kv_lens.long()[:, None] - new + i
    q, k = _turned(st, st.q, place), _turned(st, st.k, place)
    ok = (i < new).flatten()
    page = torch.gather(st.page_table.long(), 1, place.clamp(0, st.page_table.shape[1] *
                                                             st.page - 1) // st.page).flatten()[ok]
    row = (place % st.page).flatten()[ok]
    k = k.transpose(1, 2).reshape(B * S, Hkv, D)[ok]
    v = st.v.transpose(1, 2).reshape(B * S, Hkv, D)[ok]
    for pages, x in ((st.k_pages, k), (st.v_pages, v)):
        if st.bits == 16:
            pages[page, :, row] = x
        else:
            codes, scales = _parts(pages)
            c, s = _parts(_pack(x[:, :, None]))
            codes[page, :, row] = c[:, :, 0]
            scales[page, :, row] = s[:, :, 0]
    if st.bounds is not None:
        # (pages whose first place is among the new rows start anew)
        first = page[row == 0]
        low, high = st.bounds[:, :, 0].float(), st.bounds[:, :, 1].float()
        low[first], high[first] = math.inf, -math.inf
        at = page[:, None, None].expand(-1, Hkv, D)
        low.scatter_reduce_(0, at, k.float(), "amin")
        high.scatter_reduce_(0, at, k.float(), "amax")
        st.bounds.copy_(torch.stack((low, high), 2))
    return q


def _read(st):
    """What the cache stands for, [B, H, S, D], zeros behind each sequence."""
    there = torch.arange(st.seqlen, device="cuda")[None, :] < st.kv_lens[:, None]
    out = []
    for pages in (st.k_pages, st.v_pages):
        x = _rows(st, pages, st.page_table).flatten(2, 3)[:, :, :st.seqlen]
        out.append(x.masked_fill_(~there[:, None, :, None], 0.0).to(st.type))
    return out


def _select(st):
    """Page numbers [B, H, S, count] of the sequence, ascending, -1 behind them."""
    B, Hq, S, D = st.q.shape
    Hkv, N = st.bounds.shape[1], st.page_table.shape[1]
    at = st.page_table.clamp(min=0).long()
    b = st.bounds.double()[at]  # [B, N, H, 2, D]
    low, high = (b[:, :, :, n].permute(0, 2, 3, 1).contiguous() for n in (0, 1))
    q = st.q.double().reshape(B, Hkv, Hq // Hkv * S, D)
    score = torch.matmul(q.clamp(min=0), high) + torch.matmul(q.clamp(max=0), low)
    score = score.view(B, Hkv, Hq // Hkv, S, N).amax(2)
    last = (st.kv_lens.long()[:, None] - S + torch.arange(S, device="cuda"))[:, None, :, None]
    n = torch.arange(N, device="cuda")
    score = score.masked_fill(n > last // st.page, -math.inf)
    score = score.masked_fill(n == last // st.page, math.inf)
    top, page = torch.sort(score, dim=-1, descending=True, stable=True)
    page = torch.where(top == -math.inf, N, page)[..., :st.count]
    if page.shape[-1] < st.count:
        page = torch.cat((page, torch.full((B, Hkv, S, st.count - page.shape[-1]), N,
                                           device="cuda")), -1)
    page = torch.sort(page, -1)[0]
    return torch.where(page == N, -1, page).to(torch.int32)


def _attend(st, selected=None):
    B, Hq, S, D = st.q.shape
    Hkv, ps = st.k_pages.shape[1], st.page
    G = Hq // Hkv
    q = st.q.float().view(B, Hkv, G, S, D)
    last = st.kv_lens.long()[:, None] - S + torch.arange(S, device="cuda")  # [B, S]
    inside = torch.arange(ps, device="cuda")
    if selected is None:  # rows [B, H, G S], keys [B, H, M]
        at = st.page_table
        place = (torch.arange(at.shape[1], device="cuda")[:, None] * ps + inside).flatten()
        place = place.view(1, 1, 1, 1, -1)
        q = q.reshape(B, Hkv, 1, G * S, D)
        last = last[:, None, None, None, :].expand(B, 1, 1, G, S).reshape(B, 1, 1, G * S, 1)
    else:  # rows [B, H, S, G], keys [B, H, S, M]
        at = torch.gather(st.page_table[:, None, None].expand(B, Hkv, S, -1), 3,
                          selected.clamp(min=0).long())
        place = (selected[..., None].long() * ps + inside).masked_fill(selected[..., None] < 0,
                                                                       2 ** 40)
        place = place.flatten(3)[:, :, :, None]
        q = q.transpose(2, 3)
        last = last[:, None, :, None, None]
    seen = place <= last
    keys = _rows(st, st.k_pages, at)
    keys = keys.view(*q.shape[:3], -1, D)
    s = torch.matmul(q, keys.transpose(3, 4)).mul_(st.scale)
    del keys
    if st.softcap:
        s = torch.tanh(s / st.softcap) * st.softcap
    if st.slopes is not None:
        m = st.slopes.view(1, Hkv, G, 1)
        m = m.expand(1, Hkv, G, S).reshape(1, Hkv, 1, G * S, 1) if selected is None else \
            m.view(1, Hkv, 1, G, 1)
        s = s - m * (last - place)
    s = s.masked_fill_(~seen, -math.inf)
    m = s.amax(-1, keepdim=True)
    p = torch.exp(s.sub_(torch.where(m == -math.inf, torch.zeros_like(m), m)))
    del s
    z = p.sum(-1, keepdim=True)
    values = _rows(st, st.v_pages, at).view(*q.shape[:3], -1, D)
    o = torch.matmul(p, values) / torch.where(z == 0, torch.ones_like(z), z)
    lse = (m + torch.log(z)).squeeze(-1)
    if selected is not None:
        o, lse = o.transpose(2, 3), lse.transpose(2, 3)
    return o.reshape(B, Hq, S, D).to(st.type), lse.reshape(B, Hq, S)


def _appended(st, q):
    """An append's outputs: the turned queries, what the cache holds then, its bounds."""
    out = {"q": q}
    if st.bounds is not None:
        out["bounds"] = st.bounds
    if st.bits == 16:
        out["k_pages"], out["v_pages"] = st.k_pages, st.v_pages
    return out


def run(st):
    if own:
        import shaobo_fa3_torch  # noqa: F401  (registers the operators)
        ops = torch.ops.shaobo_fa3
        if st.op == "append":
            q, = ops.cache_append(st.k, st.v, st.k_pages, st.v_pages, st.page_table, st.kv_lens,
                                  st.new_lens, st.q, st.positions, st.freqs, st.interleaved,
                                  st.bounds)
            out = _appended(st, q)
            if st.bits == 4:
                out["k"], out["v"] = ops.cache_read(st.k_pages, st.v_pages, st.page_table,
                                                    st.kv_lens, st.seqlen, st.type)
            return out
        selected = None
        if st.op == "sparse":
            selected = ops.cache_select(st.q, st.bounds, st.page_table, st.kv_lens, st.page,
                                        st.count)
        out, lse = ops.cache_attn(st.q, st.k_pages, st.v_pages, st.page_table, st.kv_lens, None,
                                  True, st.scale, st.softcap, st.slopes, None, selected)
        return {"out": out, "lse": lse} if selected is None else \
            {"out": out, "lse": lse, "selected": selected}
    if st.op == "append":
        out = _appended(st, _append(st))
        if st.bits == 4:
            out["k"], out["v"] = _read(st)
        return out
    selected = _select(st) if st.op == "sparse" else None
    out, lse = _attend(st, selected)
    return {"out": out, "lse": lse} if selected is None else \
        {"out": out, "lse": lse, "selected": selected}


# ---------------------------------------------------------------------------
# The operators' definitions in fp64, sequence by sequence.
def _exact_sequence(case, st, pages, b, length):
    """Rows [H, length, D] that the cache stands for."""
    ps, D = case["page"], case["head_dim"]
    at = st.page_table[b, :-(-length // ps)].long()
    x = pages[at].transpose(0, 1)  # [H, n, page, row]
    if case["bits"] == 16:
        return x.double().reshape(x.shape[0], -1, D)[:, :length]
    x = x.reshape(x.shape[0], x.shape[1], -1)
    codes, scales = x[..., :ps * D // 2], x[..., ps * D // 2:].contiguous().view(torch.float32)
    low, high = codes.int() % 16, codes.int() // 16
    c = torch.stack((low, high), -1).reshape(x.shape[0], -1, D)
    e, m = (c // 2) % 4, c % 2
    size = torch.where(e == 0, 0.5 * m, torch.exp2(e.double() - 1) * (1 + 0.5 * m))
    size = torch.where(c >= 8, -size, size)
    return (size * scales.double().reshape(x.shape[0], -1, 1))[:, :length]


def _exact_turn(case, st, x, places):
    P = case["rotary_dim"] // 2
    turn = torch.zeros(places.shape[1:] + (P,), dtype=torch.float64, device="cuda")
    for a in range(places.shape[0]):
        turn += places[a].double().unsqueeze(-1) * st.freqs[a].double()
    turn = torch.polar(torch.ones_like(turn), turn).unsqueeze(1)
    y = x.double().clone()
    low, high = (slice(0, 2 * P, 2), slice(1, 2 * P, 2)) if case["interleaved"] else \
        (slice(0, P), slice(P, 2 * P))
    z = torch.complex(y[..., low].contiguous(), y[..., high].contiguous()) * turn
    y[..., low], y[..., high] = z.real, z.imag
    return y


def _exact_four(x):
    """What 4 bits hold of rows [..., D]: the nearest level of a sixth of the largest magnitude."""
    top = x.abs().amax(-1, keepdim=True)
    t = 6 * x.abs() / torch.where(top == 0, torch.ones_like(top), top)
    step = torch.where(t < 2, 0.5, torch.where(t < 4, 1.0, 2.0)).double()
    return torch.sign(x) * torch.round(t / step) * step * top / 6  # (torch.round: ties to even)


def _exact_append(case, st):
    B, S, ps = case["batch"], case["seq"], case["page"]
    kv, new = _lens(case)
    i = torch.arange(S, device="cuda")
    places = st.positions if st.positions is not None else \
        torch.stack([kv[b] - new[b] + i for b in range(B)])[None]
    q, k = _exact_turn(case, st, st.q, places), _exact_turn(case, st, st.k, places)
    v = st.v.double()
    out = {"q": q}
    if case["bounds"]:
        bounds = st.bounds.double()
        for b in range(B):
            for n in range((kv[b] - new[b]) // ps, (kv[b] - 1) // ps + 1):
                lo, hi = max(n * ps, kv[b] - new[b]), min((n + 1) * ps, kv[b])
                rows = k[b, :, lo - kv[b] + new[b]:hi - kv[b] + new[b]]
                page = int(st.page_table[b, n])
                low, high = rows.amin(1), rows.amax(1)
                if lo > n * ps:
                    low, high = torch.minimum(low, bounds[page, :, 0]), \
                        torch.maximum(high, bounds[page, :, 1])
                bounds[page, :, 0], bounds[page, :, 1] = low, high
        out["bounds"] = bounds
    if case["bits"] == 16:
        for name, pages, x in (("k_pages", st.k_pages, k), ("v_pages", st.v_pages, v)):
            pool = pages.double()
            for b in range(B):
                t = torch.arange(kv[b] - new[b], kv[b], device="cuda")
                pool[st.page_table[b].long()[t // ps], :, t % ps] = x[b, :, :new[b]].transpose(0, 1)
            out[name] = pool
        return out
    # (a row of codes goes by its 16-bit values)
    for name, pages, x in (("k", st.k_pages, k.to(st.type).double()), ("v", st.v_pages, v)):
        y = torch.zeros(B, x.shape[1], case["cache"], x.shape[3], dtype=torch.float64,
                        device="cuda")
        for b in range(B):
            old = kv[b] - new[b]
            if old:
                y[b, :, :old] = _exact_sequence(case, st, pages, b, old)
            y[b, :, old:kv[b]] = _exact_four(x[b, :, :new[b]])
        out[name] = y
    return out


def exact(case, seed):
    st = _inputs(case, seed)
    if case["op"] == "append":
        return _exact_append(case, st)
    B, Hq, S, D = st.q.shape
    Hkv, ps, N = case["heads_kv"], case["page"], st.page_table.shape[1]
    G = Hq // Hkv
    kv, _ = _lens(case)
    out = torch.zeros(B, Hq, S, D, dtype=torch.float64, device="cuda")
    lse = torch.zeros(B, Hq, S, dtype=torch.float64, device="cuda")
    selected = torch.full((B, Hkv, S, case["count"]), -1, dtype=torch.int32, device="cuda")
    for b in range(B):
        keys = _exact_sequence(case, st, st.k_pages, b, kv[b])
        values = _exact_sequence(case, st, st.v_pages, b, kv[b])
        j = torch.arange(kv[b], device="cuda").unsqueeze(0)
        place = (kv[b] - S + torch.arange(S, device="cuda")).unsqueeze(1)
        for h in range(Hkv):
            hidden = j > place
            if case["op"] == "sparse":
                rows = st.bounds[st.page_table[b, :-(-kv[b] // ps)].long(), h].double()
                for i in range(S):
                    mine = (kv[b] - S + i) // ps
                    q = st.q[b, h * G:(h + 1) * G, i].double().unsqueeze(1)
                    best = torch.maximum(q * rows[:mine, 0], q * rows[:mine, 1]).sum(-1)
                    best = best.max(0)[0]  # of the group's heads
                    few = torch.argsort(-best, stable=True)[:case["count"] - 1]
                    few = torch.sort(torch.cat((few, torch.tensor([mine], device="cuda"))))[0]
                    selected[b, h, i, :few.numel()] = few.to(torch.int32)
                    hidden[i] |= ~torch.isin(j[0] // ps, few)
            for g in range(h * G, (h + 1) * G):
                x = st.q[b, g].double() @ keys[h].t().contiguous() / math.sqrt(D)
                if case["softcap"]:
                    x = torch.tanh(x / case["softcap"]) * case["softcap"]
                if st.slopes is not None:
                    x -= float(st.slopes[g]) * (place - j)
                x = torch.where(hidden, torch.full_like(x, -math.inf), x)
                lse[b, g] = torch.logsumexp(x, 1)
                out[b, g] = torch.softmax(x, 1) @ values[h]
    if case["op"] == "attn":
        return {"out": out, "lse": lse}
    return {"out": out, "lse": lse, "selected": selected}
