"""The paged cache where it can go wrong: what lies behind sequences and in
other pages, NaN that is seen and NaN that is not, strides and far offsets,
streams, graphs, a served sequence against the whole prompt, refusals."""
import ctypes
import math

import pytest

import attn_oracle as A
import cache_oracle as O
import shaobo_fa3 as F
from test_gpu_attn import i32, refused, within
from test_gpu_cache import append_case, attn_case, check_append, check_attn, gen_of, make_cache, rows, where

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

BF, HF = torch.bfloat16, torch.float16


@pytest.fixture(scope="module")
def T():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    F.load()
    import shaobo_fa3_torch
    assert shaobo_fa3_torch._ATTN, "lib/_fa3_torch_attn.so is not built"
    return shaobo_fa3_torch


def spoiled(cache):
    """The cache with NaN and infinities (4 bits: any bytes, NaN for scales)
    wherever no sequence has a row, and pages of others behind the sequences."""
    used = torch.zeros(cache["k"].shape[0], cache["page_size"], dtype=torch.bool, device="cuda")
    table, ps = cache["table"].clone(), cache["page_size"]
    for b in range(table.shape[0]):
        ok, page, row = O.there(cache, b)
        used[page[ok], row[ok]] = True
        n = -(-O.clipped(cache, b)[0] // ps)
        table[b, n:] = torch.arange(table.shape[1] - n, device="cuda", dtype=torch.int32) % used.shape[0]
    out = dict(cache, table=table)
    for n in ("k", "v"):
        x = cache[n].clone()
        if cache["bits"] == 16:
            junk = torch.tensor([math.nan, math.inf, -math.inf], device="cuda", dtype=x.dtype)
            x = torch.where(used[:, None, :, None], x, junk[torch.randint(0, 3, x.shape, device="cuda",
                                                                           generator=gen_of(2))])
        else:
            code, scale = O.parts(x)
            noise = torch.randint(0, 16, code.shape, device="cuda", generator=gen_of(3), dtype=torch.int32)
            code = torch.where(used[:, None, :, None], code, noise)
            scale = torch.where(used[:, None, :], scale, torch.full_like(scale, math.nan))
            x = O.pack(code, scale)
        out[n] = x
    return out


EDGE = [dict(kv=[1, 33, 70], Hq=4), dict(kv=[130, 257], Hq=8, D=128), dict(kv=[61, 3000], D=128, ps=128),
        dict(kv=[90, 200], S=70, D=128), dict(kv=[101, 333], S=130, Hq=4, ps=32), dict(kv=[45, 3], new=[9, 2], S=12),
        dict(kv=[200], S=3, holes=[1], Hq=4, D=128), dict(kv=[200, 90], slopes=1, S=2), dict(kv=[200, 90], S=80, softcap=5.0)]


@pytest.mark.parametrize("bits,dtype", [(16, BF), (4, BF), (16, HF), (4, HF)])
@pytest.mark.parametrize("case", EDGE, ids=str)
def test_other_rows_may_hold_anything(T, case, bits, dtype):
    """Behind the sequences and in pages of nobody: bit for bit the same.  Padding
    rows of q too."""
    cache, q, o = attn_case(case, bits, dtype)
    want = check_attn(T, cache, q, o)
    for b, n in enumerate(cache["new"]):
        q[b, :, n:] = math.nan
    bad = spoiled(cache)
    kw = dict(causal=o["causal"], softmax_scale=o["scale"], softcap=o["softcap"], slopes=o.get("slopes"), return_lse=True)
    got = T.cache_attention(q, bad["k"], bad["v"], **where(bad), **kw)
    torch.cuda.synchronize()
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    N = cache["table"].shape[1]
    every = torch.arange(N, device="cuda", dtype=torch.int32).expand(*q.shape[:1], cache["k"].shape[1], q.shape[2], N)
    a = T.cache_attention(q, cache["k"], cache["v"], selected=every.contiguous(), **where(cache), **kw)
    b = T.cache_attention(q, bad["k"], bad["v"], selected=every.contiguous(), **where(bad), **kw)
    torch.cuda.synchronize()
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    x = T.cache_read(cache["k"], cache["v"], page_table=cache["table"], kv_lens=i32(cache["kv"]), seqlen=400, dtype=dtype)
    y = T.cache_read(bad["k"], bad["v"], page_table=bad["table"], kv_lens=i32(cache["kv"]), seqlen=400, dtype=dtype)
    assert all(torch.equal(c, d) for c, d in zip(x, y))


@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("case", [dict(kv=[1]), dict(kv=[200], Hq=8, D=128), dict(kv=[3000], D=128), dict(kv=[300], S=150),
                                  dict(kv=[300], S=150, D=128, softcap=5.0), dict(kv=[100], S=5, slopes=1)], ids=str)
def test_visible_nan_shows(T, case, bits):
    """A row whose q is NaN, or that sees a key that is, has NaN for output and
    log-sum-exp; rows of other heads of another KV head do not."""
    cache, q, o = attn_case(case, bits, BF)
    kw = dict(causal=o["causal"], softcap=o["softcap"], slopes=o.get("slopes"), return_lse=True)
    q2 = q.clone()
    q2[0, 0, -1] = math.nan
    out, lse = T.cache_attention(q2, cache["k"], cache["v"], **where(cache), **kw)
    assert torch.isnan(out[0, 0, -1]).all() and torch.isnan(lse[0, 0, -1])
    assert torch.isfinite(out[0, q.shape[1] // 2:]).all()
    # a key, the last of the sequence: seen by the last row alone
    kv, ps = case["kv"][0], cache["page_size"]
    page, row = int(cache["table"][0, (kv - 1) // ps]), (kv - 1) % ps
    if bits == 16:
        cache["k"][page, 0, row, 3] = math.nan
    else:
        code, scale = O.parts(cache["k"])
        scale[page, 0, row] = math.nan
        cache["k"] = O.pack(code, scale)
    out, lse = T.cache_attention(q, cache["k"], cache["v"], **where(cache), **kw)
    G = q.shape[1] // cache["k"].shape[1]
    assert torch.isnan(out[0, :G, -1]).all() and torch.isnan(lse[0, :G, -1]).all()
    assert torch.isfinite(out[0, G:]).all() and torch.isfinite(lse[0, G:]).all()


def test_rows_that_see_nothing_beside_nan(T):
    """Non-causal rows without keys (every page is none) and padding rows are
    zeros whatever q holds."""
    for bits in (16, 4):
        for S in (3, 100):
            cache, q, o = attn_case(dict(kv=[150, 90], new=[S - 1, S], S=S, Hq=4, D=128, causal=False), bits, BF)
            cache["table"][1] = -1
            q[1], q[0, :, -1] = math.nan, math.inf
            out, lse = T.cache_attention(q, cache["k"], cache["v"], causal=False, return_lse=True, **where(cache))
            assert (out[1] == 0).all() and (lse[1] == -math.inf).all()
            assert (out[0, :, -1] == 0).all() and (lse[0, :, -1] == -math.inf).all()
            assert torch.isfinite(out[0, :, :-1]).all()


# ---------------------------------------------------------------------------
@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("S", [1, 5, 90])
def test_strides(T, bits, S):
    """Pages of k and v in one pool, 16-bit rows of all heads of a place side by
    side, a table that is part of a wider one, rows that are views."""
    cache, q, o = attn_case(dict(kv=[200, 77], S=S, Hq=8, Hkv=4, D=128, ps=32), bits, BF)
    want = check_attn(T, cache, q, o)
    n, H, ps, row = cache["k"].shape
    pool = torch.zeros(n, 2, H, ps, row, dtype=cache["k"].dtype, device="cuda")
    if bits == 16:
        pool = torch.zeros(n, ps, 2, H, row, dtype=BF, device="cuda").permute(0, 2, 3, 1, 4)
    views = dict(cache, k=pool[:, 0], v=pool[:, 1])
    views["k"].copy_(cache["k"])
    views["v"].copy_(cache["v"])
    wide = torch.full((2, cache["table"].shape[1] + 5), 12345, dtype=torch.int32, device="cuda")
    wide[:, 2:2 + cache["table"].shape[1]] = cache["table"]
    views["table"] = wide[:, 2:2 + cache["table"].shape[1]]
    big = torch.zeros(2, S + 3, 8 + 2, 128 + 8, dtype=BF, device="cuda")
    qv = big[:, 1:S + 1, 1:9, :128].transpose(1, 2)
    qv.copy_(q)
    out, lse = T.cache_attention(qv, views["k"], views["v"], return_lse=True, **where(views))
    assert torch.equal(out, want[0]) and torch.equal(lse, want[1])
    # the same rows appended through both
    gen = gen_of(5)
    k, v = (rows(gen, 2, 4, S, 128, BF, True) for _ in range(2))
    bounds = [torch.zeros(n, H, 2, 128, dtype=BF, device="cuda") for _ in range(2)]
    fr = T.rotary_freqs([64], device="cuda")
    got = [T.cache_append(k, v, c["k"], c["v"], q=x, freqs=fr, bounds=b, **where(c))
           for c, x, b in ((cache, q, bounds[0]), (views, qv, bounds[1]))]
    assert torch.equal(got[0], got[1]) and torch.equal(*bounds)
    assert torch.equal(cache["k"], views["k"].contiguous()) and torch.equal(cache["v"], views["v"].contiguous())


@pytest.mark.parametrize("bits", [16, 4])
def test_offsets_past_32_bits(T, bits):
    """Pages more than 2^32 bytes into their tensor."""
    H, ps, D = 8, 128, 128
    pages = 2 ** 32 // (H * ps * (2 * D if bits == 16 else D // 2 + 4)) + 40
    k, v, bounds = T.cache_pages(pages, H, ps, D, BF, bits=bits, bounds=True)
    table = i32([[pages - 1, pages - 7, pages - 3], [pages - 2, 5, pages - 20]])
    cache = dict(k=k, v=v, bits=bits, table=table, kv=[300, 270], new=[300, 200], page_size=ps, D=D, dtype=BF)
    gen = gen_of(4)
    x, y = (rows(gen, 2, H, 300, D, BF) for _ in range(2))
    q = rows(gen, 2, H, 300, D, BF)
    T.cache_append(x, y, k, v, bounds=bounds, **where(cache))
    got = T.cache_read(k, v, page_table=table, kv_lens=i32([300, 270]), seqlen=300, dtype=BF)
    if bits == 16:
        assert torch.equal(got[0][0], x[0]) and torch.equal(got[1][0], y[0])
        assert torch.equal(got[0][1, :, 70:270], x[1, :, :200])
    small = dict(cache, k=k[-40:].clone(), v=v[-40:].clone(), table=(table - (pages - 40)).clamp(min=-1))
    assert int(bounds[pages - 1].float().abs().sum()) > 0
    for S in (1, 100):
        c = dict(cache, new=[S, S])
        s = dict(small, new=[S, S])
        c["table"] = table.clone()
        c["table"][1, 1] = -1  # (page 5 is not among the small ones)
        a = T.cache_attention(q[:, :, :S].contiguous(), k, v, return_lse=True, **where(c))
        b = T.cache_attention(q[:, :, :S].contiguous(), s["k"], s["v"], return_lse=True, **where(s))
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
        check_attn(T, s, q[:, :, :S].contiguous(), dict(causal=True, softcap=0.0, scale=None))
    sel = T.cache_select(q[:, :, :1].contiguous(), bounds, page_table=table, kv_lens=i32([300, 270]), page_size=ps, count=2)
    assert torch.equal(sel, O.select(q[:, :, :1], bounds, dict(cache, new=[1, 1]), 2))


def test_turned_in_place_and_beside(T):
    """The C entry: q's output may be q, and nothing around its rows is written."""
    lib = F.load()
    B, Hq, Hkv, S, D, ps = 2, 6, 2, 21, 64, 32
    gen = gen_of(7)
    k, v = (rows(gen, B, Hkv, S, D, BF) for _ in range(2))
    room = torch.full((B, Hq, S + 2, D + 16), 7.0, dtype=BF, device="cuda")
    q = room[:, :, 1:S + 1, 8:8 + D]
    q.copy_(rows(gen, B, Hq, S, D, BF))
    cache = make_cache(gen, [40, 21], [S, S], Hkv, D, ps)
    fr = T.rotary_freqs([32], device="cuda")
    want = T.cache_append(k, v, cache["k"], cache["v"], q=q, freqs=fr, **where(cache))
    lens, new = i32([40, 21]), i32([S, S])
    p = F.CacheAppendParams()
    lib.shaobo_fa3_cache_append_params_init(ctypes.byref(p))
    p.seqlen, p.num_heads_q, p.pairs, p.freqs = S, Hq, 32, fr.data_ptr()
    c = p.cache
    c.batch, c.num_heads_kv, c.head_dim, c.dtype = B, Hkv, D, F.DTYPE_BF16
    c.pages, c.page_size, c.width = cache["k"].shape[0], ps, cache["table"].shape[1]
    for n in ("k", "v"):
        t = getattr(c, n)
        t.data, (t.page_stride, t.head_stride, t.row_stride, _) = cache[n].data_ptr(), cache[n].stride()
    c.page_table, c.page_table_stride = cache["table"].data_ptr(), cache["table"].stride(0)
    c.kv_lens, c.new_lens = lens.data_ptr(), new.data_ptr()
    for n, t in (("k", k), ("v", v), ("q", q), ("q_out", q)):
        x = getattr(p, n)
        x.data, (x.batch_stride, x.head_stride, x.row_stride, _) = t.data_ptr(), t.stride()
    before = cache["k"].clone()
    assert lib.shaobo_fa3_cache_append(ctypes.byref(p), torch.cuda.current_stream().cuda_stream) == F.SUCCESS
    torch.cuda.synchronize()
    assert torch.equal(q, want) and torch.equal(cache["k"], before)
    edge = room.clone()
    edge[:, :, 1:S + 1, 8:8 + D] = 7.0
    assert (edge == 7.0).all()


# ---------------------------------------------------------------------------
@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("D,ps", [(64, 32), (128, 64)])
def test_one_by_one_equals_at_once(T, bits, D, ps):
    """Tokens appended singly, in parts and together: the same pages and bounds."""
    gen = gen_of(3)
    k, v, q = (rows(gen, 2, h, 150, D, BF) for h in (2, 2, 4))
    table = torch.randperm(10, generator=gen, device="cuda").int().view(2, 5)
    fr = T.rotary_freqs([D // 2], device="cuda")
    results = []
    for cuts in ([150], [1] * 150, [70, 1, 1, 40, 38]):
        kp, vp, bounds = T.cache_pages(10, 2, ps, D, BF, bits=bits, bounds=True)
        at, qs = 0, []
        for n in cuts:
            at += n
            qs.append(T.cache_append(*(x[:, :, at - n:at].contiguous() for x in (k, v)), kp, vp,
                                     q=q[:, :, at - n:at].contiguous(), freqs=fr, bounds=bounds,
                                     page_table=table, kv_lens=i32([at, at])))
        results.append((kp, vp, bounds, torch.cat(qs, 2)))
    for r in results[1:]:
        for a, b in zip(results[0], r):
            assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))


@pytest.mark.parametrize("cap", [0.0, 8.0])
def test_serving_equals_the_prompt(T, cap):
    """rotary + score_attention over a whole sequence against a prompt appended
    in two parts and tokens one by one, with and without selection of all pages."""
    B, Hq, Hkv, S, D, ps = 2, 8, 2, 170, 128, 32
    gen = gen_of(11)
    q, k, v = (rows(gen, B, h, S, D, BF, True) for h in (Hq, Hkv, Hkv))
    fr = T.rotary_freqs([D // 2], device="cuda")
    pos = torch.arange(S, device="cuda").expand(1, B, S)
    kp, vp, bounds = T.cache_pages(20, Hkv, ps, D, BF, bounds=True)
    table = torch.randperm(20, generator=gen, device="cuda").int().view(B, 10)
    outs, cuts = [], [100, 58] + [1] * 12
    at, qs, lses = 0, [], []
    for n in cuts:
        at += n
        part = [x[:, :, at - n:at] for x in (q, k, v)]
        where_ = dict(page_table=table, kv_lens=i32([at, at]))
        qt = T.cache_append(part[1], part[2], kp, vp, q=part[0], freqs=fr, bounds=bounds, **where_)
        out, lse = T.cache_attention(qt, kp, vp, softcap=cap, return_lse=True, **where_)
        if n == 1:
            sel = T.cache_select(qt, bounds, page_size=ps, count=10, **where_)
            o2, l2 = T.cache_attention(qt, kp, vp, softcap=cap, selected=sel, return_lse=True, **where_)
            assert (out.double() - o2.double()).abs().max() <= 2.0 ** -7 * out.double().abs().max()
            assert (lse - l2).abs().max() <= 1e-4
        outs.append(out), qs.append(qt), lses.append(lse)
    kt, vt = T.cache_read(kp, vp, page_table=table, kv_lens=i32([S, S]), seqlen=S, dtype=BF)
    assert torch.equal(vt, v)
    # the layer's own rotation differs by fp32's rounding before the one to 16 bits
    qr, kr = T.rotary(q, k, positions=pos, freqs=fr)
    step = 2.0 ** -7
    assert ((kr - kt).abs() <= step * kr.abs() + 1e-6).all()
    want, wlse, off, lse_off = A.forward(torch.cat(qs, 2), kt, vt, True, softcap=cap)
    within("lse", torch.cat(lses, 2), wlse, lse_off)
    within("out", torch.cat(outs, 2), want, off)
    dense, dlse = T.score_attention(torch.cat(qs, 2), kt, vt, softcap=cap, return_lse=True)
    within("dense", dense, want, off)
    within("dense lse", dlse, wlse, lse_off)


DEALT = [
    # (the kernel for few rows cuts several sequences by their lengths)
    dict(kv=[9000] + [40] * 9, Hq=8), dict(kv=[1, 700, 0, 5000, 33], D=128, Hq=8),
    dict(kv=[200 + 37 * n for n in range(70)], Hq=4), dict(kv=[0] * 65 + [3000, 1], Hq=4, D=128),
    dict(kv=[300, 2500, 90], new=[3, 0, 2], S=4, Hq=8, D=128), dict(kv=[5000, 10], S=3, Hq=2, Hkv=1, softcap=9.0, std=3.0),
    dict(kv=[10] * 255 + [4000]), dict(kv=[4000] + [10] * 256), dict(kv=[600, 4100, 700], S=2, slopes=1, Hq=8, ps=32),
    dict(kv=[3000, 2900], holes=[0, 5, 20], Hq=4, D=128), dict(kv=[16000] + [100] * 90, Hq=16, Hkv=8, D=128),
    dict(kv=[2600, 700], D=128, Hq=32, Hkv=1), dict(kv=[400] * 40 + [9000], Hq=32, Hkv=16, D=64, prefix=[500] * 41, S=2),
]


@pytest.mark.parametrize("bits,dtype", [(16, BF), (4, HF)])
@pytest.mark.parametrize("case", DEALT, ids=lambda c: f"{len(c['kv'])}-{max(c['kv'])}-{c.get('S', 1)}")
def test_sequences_of_very_different_lengths(T, case, bits, dtype):
    check_attn(T, *attn_case(case, bits, dtype))


def step(T, s):
    """One decoding step of a state: append, select, attend twice."""
    w = dict(page_table=s["table"], kv_lens=s["lens"])
    qt = T.cache_append(s["k"], s["v"], s["kp"], s["vp"], q=s["q"], freqs=s["fr"], bounds=s["bounds"], **w)
    sel = T.cache_select(qt, s["bounds"], page_size=s["ps"], count=4, **w)
    return (qt, sel, *T.cache_attention(qt, s["kp"], s["vp"], return_lse=True, **w),
            *T.cache_attention(qt, s["kp"], s["vp"], selected=sel, return_lse=True, **w))


def step_state(T, bits, S=1, seed=1, old=900):
    gen = gen_of(seed)
    B, Hq, Hkv, D, ps = 3, 8, 2, 128, 64
    kp, vp, bounds = T.cache_pages(60, Hkv, ps, D, BF, bits=bits, bounds=True)
    s = dict(kp=kp, vp=vp, bounds=bounds, ps=ps, fr=T.rotary_freqs([D // 2], device="cuda"))
    s["table"] = torch.randperm(60, generator=gen, device="cuda").int().view(B, 20)
    w = dict(page_table=s["table"], kv_lens=i32([old] * B))
    k, v = (rows(gen, B, Hkv, old, D, BF) for _ in range(2))
    T.cache_append(k, v, kp, vp, freqs=s["fr"], bounds=bounds, **w)
    for n, h in (("q", Hq), ("k", Hkv), ("v", Hkv)):
        s[n] = rows(gen, B, h, S, D, BF)
    s["lens"] = i32([old + S, old // 2 + S, S])
    return s


@pytest.mark.parametrize("bits", [16, 4])
def test_on_another_stream_and_on_two(T, bits):
    states = [step_state(T, bits, seed=n) for n in (1, 2)]
    want = [step(T, s) for s in states]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = [None, None]
    for _ in range(5):
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                got[i] = step(T, states[i])
    torch.cuda.synchronize()
    for a, b in zip(want, got):
        assert all(torch.equal(x, y) for x, y in zip(a, b))


@pytest.mark.parametrize("bits,S", [(16, 1), (4, 1), (4, 5), (16, 90)])
def test_graph_capture(T, bits, S):
    """A step captured twice and replayed with other tokens and lengths, eager
    work between; every replay against the eager step on a copy of the cache."""
    s = step_state(T, bits, S)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(T, s)
    torch.cuda.current_stream().wait_stream(side)
    graphs, outs = [], []
    for _ in range(2):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            outs.append(step(T, s))
    for n in range(4):
        other = step_state(T, bits, S, seed=20 + n)
        for name in ("q", "k", "v"):
            s[name].copy_(other[name])
        s["lens"] += i32([1, 30, 3])
        copy = dict(s, **{x: s[x].clone() for x in ("kp", "vp", "bounds")})
        want = [x.clone() for x in step(T, copy)]
        torch.cuda.synchronize()
        for g, out in zip(graphs, outs):
            g.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(x, y) for x, y in zip(want, out))
            assert all(torch.equal(copy[x].view(torch.uint8), s[x].view(torch.uint8)) for x in ("kp", "vp", "bounds"))


def test_results_are_reproducible(T):
    for bits in (16, 4):
        for kv, S in (([5000, 3000], 1), ([3000, 900], 70)):
            cache, q, o = attn_case(dict(kv=kv, S=S, Hq=8, D=128), bits, BF)
            a, b = (T.cache_attention(q, cache["k"], cache["v"], return_lse=True, **where(cache)) for _ in range(2))
            assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def test_pages_with_nan_are_selected(T):
    """A key that is NaN makes its page's bounds NaN on one side, and the page
    comes first."""
    s = step_state(T, 16, old=640)
    k = rows(gen_of(9), 1, 2, 640, 128, BF)
    k[0, :, 5 * 64 + 9, 7] = math.nan
    k[0, :, 2 * 64 + 1, 100] = -math.inf
    w = dict(page_table=s["table"][:1].contiguous(), kv_lens=i32([640]))
    T.cache_append(k, k, s["kp"], s["vp"], bounds=s["bounds"], **w)
    sel = T.cache_select(s["q"][:1], s["bounds"], page_size=64, count=3, **w)
    assert (sel == i32([2, 5, 9])).all()


def test_nothing_to_do(T):
    """Empty batches, no rows, no pages, a table of no width."""
    kp, vp, bounds = T.cache_pages(4, 2, 32, 64, BF, bounds=True)
    fr = T.rotary_freqs([32], device="cuda")
    for B, S, width in ((0, 3, 2), (2, 0, 2), (2, 3, 0)):
        k = torch.zeros(B, 2, S, 64, dtype=BF, device="cuda")
        w = dict(page_table=torch.zeros(B, width, dtype=torch.int32, device="cuda"),
                 kv_lens=torch.full((B,), 3, dtype=torch.int32, device="cuda"))
        pos = torch.zeros(1, B, S, dtype=torch.int32, device="cuda")
        assert T.cache_append(k, k, kp, vp, q=k, freqs=fr, bounds=bounds, **w).shape == k.shape
        assert T.cache_append(k, k, kp, vp, q=k, freqs=fr, positions=pos, **w).shape == k.shape
        assert T.cache_append(k, k, kp, vp, **w) is None
        sel = T.cache_select(k, bounds, page_size=32, count=2, **w)
        assert sel.shape == (B, 2, S, 2) and (width or (sel == -1).all())
        for s in (None, sel):
            out, lse = T.cache_attention(k, kp, vp, selected=s, return_lse=True, **w)
            assert out.shape == k.shape and (width or ((out == 0).all() and (lse == -math.inf).all()))
        x, y = T.cache_read(kp, vp, seqlen=S, dtype=BF, **w)
        assert x.shape == (B, 2, S, 64) and (x == 0).all()
    torch.cuda.synchronize()
    assert (kp == 0).all() and (bounds == 0).all()


def test_lengths_out_of_range_are_taken_into_it(T):
    """Lengths below 0, past the pages and past the rows."""
    for bits in (16, 4):
        cache, q, o = attn_case(dict(kv=[128, 128, 128], S=4, Hq=4), bits, BF)
        for kv, new in (([-5, 1 << 30, 2147483647], [4, 4, 4]), ([128, 100, 3], [-7, 9, 2147483647])):
            lens, fresh = i32(kv), i32(new)
            out, lse = T.cache_attention(q, cache["k"], cache["v"], page_table=cache["table"], kv_lens=lens,
                                         new_lens=fresh, return_lse=True)
            c = dict(cache, kv=[max(0, min(128, n)) for n in kv], new=[max(0, min(4, n)) for n in new])
            want, wlse, off, lse_off = O.attend(q, c)
            within("out", out, want, off)
            within("lse", lse, wlse, lse_off)
            k = rows(gen_of(1), 3, 2, 4, 64, BF)
            T.cache_append(k, k, cache["k"], cache["v"], page_table=cache["table"], kv_lens=lens, new_lens=fresh)
            b = torch.zeros(cache["k"].shape[0], 2, 2, 64, dtype=BF, device="cuda")
            sel = T.cache_select(q, b, page_table=cache["table"], kv_lens=lens, new_lens=fresh, page_size=64, count=2)
            assert torch.equal(sel, O.select(q, b, c, 2))
            T.cache_read(cache["k"], cache["v"], page_table=cache["table"], kv_lens=lens, seqlen=200, dtype=BF)
    torch.cuda.synchronize()


def test_library_checks(T):
    """Schemas and fake implementations agree with what the operators do."""
    checks = ("test_schema", "test_faketensor")
    ops = torch.ops.shaobo_fa3
    for bits in (16, 4):
        s = step_state(T, bits, 2)
        w = (s["table"], s["lens"])
        for op, args in (
                ("cache_append", (s["k"], s["v"], s["kp"], s["vp"], *w, None, s["q"], None, s["fr"], False, s["bounds"])),
                ("cache_append", (s["k"], s["v"], s["kp"], s["vp"], *w)),
                ("cache_attn", (s["q"], s["kp"], s["vp"], *w)),
                ("cache_select", (s["q"], s["bounds"], *w, 64, 3)),
                ("cache_read", (s["kp"], s["vp"], *w, 100, BF))):
            torch.library.opcheck(getattr(ops, op).default, args, test_utils=checks)


def test_refusals(T):
    s = step_state(T, 16, 2)
    ops = torch.ops.shaobo_fa3
    q, k, v, kp, vp, t, n = (s[x] for x in ("q", "k", "v", "kp", "vp", "table", "lens"))
    four = T.cache_pages(60, 2, 64, 128, BF, bits=4)[0]
    a = ops.cache_attn
    refused("must be \\[batch", lambda: a(q[0], kp, vp, t, n))
    refused("fp16 or bf16", lambda: a(q.float(), kp, vp, t, n))
    refused("type", lambda: a(q.half(), kp, vp, t, n))
    refused("alike", lambda: a(q, kp, vp[:, :, :32], t, n))
    refused("alike", lambda: a(q, kp, four, t, n))
    refused("same GPU", lambda: a(q, kp, vp.cpu(), t, n))
    refused("head_dim 128, rows of 64", lambda: a(q[..., :64], kp, vp, t, n))
    refused("page_size", lambda: a(q, kp[:, :, :16], vp[:, :, :16], t, n))
    refused("page_size", lambda: a(q, kp[:, :, :48], vp[:, :, :48], t, n))
    refused("int32 \\[batch, width\\]", lambda: a(q, kp, vp, t.long(), n))
    refused("int32 \\[batch, width\\]", lambda: a(q, kp, vp, t.cpu(), n))
    refused("rows must be contiguous", lambda: a(q, kp, vp, t.t().contiguous().t(), n))
    refused("batch", lambda: a(q, kp, vp, t[:2], n[:2]))
    refused("kv_lens", lambda: a(q, kp, vp, t, n.long()))
    refused("kv_lens", lambda: a(q, kp, vp, t, n[:2]))
    refused("new_lens", lambda: a(q, kp, vp, t, n, n[:1]))
    refused("heads", lambda: a(q[:, :3], kp, vp, t, n))
    refused("16 bytes", lambda: a(q, torch.zeros(60, 2, 64, 132, dtype=BF, device="cuda")[..., :128], vp, t, n))
    refused("two axes", lambda: a(q, torch.zeros(60, 2, 64, 80, dtype=torch.uint8, device="cuda")[..., :68], four, t, n))
    refused("64 or 128", lambda: a(q[..., :96], *(torch.zeros(60, 2, 64, 52, dtype=torch.uint8, device="cuda"),) * 2, t, n))
    refused("needs causal", lambda: a(q, kp, vp, t, n, None, False, None, 0.0, None, n))
    refused("softcap", lambda: a(q, kp, vp, t, n, None, True, None, -1.0))
    refused("finite", lambda: a(q, kp, vp, t, n, None, True, math.nan))
    refused("slopes", lambda: a(q, kp, vp, t, n, None, True, None, 0.0, torch.ones(3, device="cuda")))
    sel = torch.zeros(3, 2, 2, 4, dtype=torch.int32, device="cuda")
    refused("selected", lambda: a(q, kp, vp, t, n, None, True, None, 0.0, None, None, sel.long()))
    refused("selected", lambda: a(q, kp, vp, t, n, None, True, None, 0.0, None, None, sel[:, :1].contiguous()))
    refused("selected", lambda: a(q, kp, vp, t, n, None, True, None, 0.0, None, None, sel[..., :2]))
    refused("selected", lambda: a(q, kp, vp, t, n, None, True, None, 0.0, None, None, sel[..., :0]))
    p = ops.cache_append
    refused("heads", lambda: p(k[:, :1], v[:, :1], kp, vp, t, n))
    refused("other rows", lambda: p(k, v[:, :, :1], kp, vp, t, n))
    refused("other rows", lambda: p(k, v, kp, vp, t, n, None, q[:, :, :1]))
    refused("several axes", lambda: p(k, v, kp, vp, t, n, None, q, None, T.rotary_freqs([32, 32], device="cuda")))
    refused("need freqs", lambda: p(k, v, kp, vp, t, n, None, q, torch.zeros(1, 3, 2, device="cuda")))
    refused("positions", lambda: p(k, v, kp, vp, t, n, None, q, torch.zeros(1, 3, 1, device="cuda"), s["fr"]))
    refused("positions", lambda: p(k, v, kp, vp, t, n, None, q, torch.zeros(1, 3, 2, device="cuda").short(), s["fr"]))
    refused("pairs", lambda: p(k, v, kp, vp, t, n, None, q, None, s["fr"][:, :12].contiguous()))
    refused("bounds", lambda: p(k, v, kp, vp, t, n, bounds=s["bounds"][:-1]))
    refused("bounds", lambda: p(k, v, kp, vp, t, n, bounds=s["bounds"].half()))
    c = ops.cache_select
    refused("count", lambda: c(q, s["bounds"], t, n, 64, 0))
    refused("page_size", lambda: c(q, s["bounds"], t, n, 100, 3))
    refused("bounds", lambda: c(q, s["bounds"].float(), t, n, 64, 3))
    refused("heads", lambda: c(q[:, :3], s["bounds"], t, n, 64, 3))
    r = ops.cache_read
    refused("fp16 or bf16", lambda: r(kp, vp, t, n, 10, torch.float32))
    refused("type", lambda: r(kp, vp, t, n, 10, HF))
    refused("seqlen", lambda: r(kp, vp, t, n, -1, BF))
    refused("seqlen", lambda: r(kp, vp, t, n, 1 << 25, BF))
    # (under grad mode: no gradient)
    refused("no gradient", lambda: T.cache_attention(q.clone().requires_grad_(), kp, vp, page_table=t, kv_lens=n))
    refused("no gradient", lambda: T.cache_append(k.clone().requires_grad_(), v, kp, vp, page_table=t, kv_lens=n))
    with torch.no_grad():
        T.cache_attention(q.clone().requires_grad_(), kp, vp, page_table=t, kv_lens=n)
    torch.cuda.synchronize()


def test_no_gradient_is_dropped(T):
    """Whichever tensor requires a gradient or has a tangent, functions and operators
    refuse the call; under no_grad, and for tensors without, they run."""
    import torch.autograd.forward_ad as fw
    s = step_state(T, 16, 2)
    x = dict(s, slopes=torch.rand(8, device="cuda"), pos=torch.zeros(1, 3, 2, device="cuda"))
    ops, w = torch.ops.shaobo_fa3, (s["table"], s["lens"])
    names = dict(page_table=s["table"], kv_lens=s["lens"])
    calls = [
        ("k v kp vp q pos fr bounds", lambda y: ops.cache_append(y["k"], y["v"], y["kp"], y["vp"], *w, None, y["q"], y["pos"],
                                                                 y["fr"], False, y["bounds"])),
        ("k v kp vp q pos fr bounds", lambda y: T.cache_append(y["k"], y["v"], y["kp"], y["vp"], q=y["q"], positions=y["pos"],
                                                               freqs=y["fr"], bounds=y["bounds"], **names)),
        ("q kp vp slopes", lambda y: ops.cache_attn(y["q"], y["kp"], y["vp"], *w, None, True, None, 0.0, y["slopes"])),
        ("q kp vp slopes", lambda y: T.cache_attention(y["q"], y["kp"], y["vp"], slopes=y["slopes"], **names)),
        ("q bounds", lambda y: ops.cache_select(y["q"], y["bounds"], *w, 64, 3)),
        ("q bounds", lambda y: T.cache_select(y["q"], y["bounds"], page_size=64, count=3, **names)),
        ("kp vp", lambda y: ops.cache_read(y["kp"], y["vp"], *w, 10, BF)),
        ("kp vp", lambda y: T.cache_read(y["kp"], y["vp"], seqlen=10, **names)),
    ]
    for takes, call in calls:
        call(x)
        for name in takes.split():
            y = dict(x)
            y[name] = x[name].clone().requires_grad_()
            refused("no gradient", lambda: call(y))
            with torch.no_grad():
                call(y)
            with fw.dual_level():
                y[name] = fw.make_dual(x[name].clone(), torch.ones_like(x[name]))
                refused("no gradient", lambda: call(y))
    torch.cuda.synchronize()


def test_appends_count_as_writes(T):
    """Autograd's version counters of what an append writes: a value that a backward
    has yet to read is missed.  Tensors without counters are written too."""
    s = step_state(T, 16, 2)
    w = dict(page_table=s["table"], kv_lens=s["lens"])
    x = torch.ones((), device="cuda", requires_grad=True)
    y = (s["kp"].float().sum() + (s["vp"] * x).float().sum())  # (x's gradient needs the values)
    before = [s[n]._version for n in ("kp", "vp", "bounds")]
    T.cache_append(s["k"], s["v"], s["kp"], s["vp"], bounds=s["bounds"], **w)
    assert all(s[n]._version > v for n, v in zip(("kp", "vp", "bounds"), before))
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()
    with torch.inference_mode():
        kp, vp, bounds = T.cache_pages(60, 2, 64, 128, BF, bounds=True)
        T.cache_append(s["k"], s["v"], kp, vp, bounds=bounds, **w)
        assert kp.abs().sum() > 0 and bounds.abs().sum() > 0
    torch.cuda.synchronize()


@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("S,direct", [(1, False), (5, False), (3, True)])
def test_a_step_is_traced(T, bits, S, direct):
    """A step as one traced and functionalized graph: outputs and cache as the eager
    step's, call after call; with and without queries and bounds."""
    ops = torch.ops.shaobo_fa3

    def run(k, v, kp, vp, q, fr, bounds, table, lens):
        w = dict(page_table=table, kv_lens=lens)
        if direct:
            qt, = ops.cache_append(k, v, kp, vp, table, lens, None, q, None, fr, False, bounds)
            assert ops.cache_append(k, v, kp, vp, table, lens, None, None, None, fr) == []
        else:
            qt = T.cache_append(k, v, kp, vp, q=q, freqs=fr, bounds=bounds, **w)
            assert T.cache_append(k, v, kp, vp, freqs=fr, **w) is None
        sel = T.cache_select(qt, bounds, page_size=64, count=4, **w)
        return (qt, sel, *T.cache_attention(qt, kp, vp, return_lse=True, **w),
                T.cache_attention(qt, kp, vp, selected=sel, **w))

    names = ("k", "v", "kp", "vp", "q", "fr", "bounds", "table", "lens")
    torch._dynamo.reset()
    traced = torch.compile(run, backend="aot_eager", fullgraph=True)
    s = step_state(T, bits, S)
    with torch.no_grad():
        for n in range(3):
            other = step_state(T, bits, S, seed=30 + n)
            for name in ("q", "k", "v"):
                s[name].copy_(other[name])
            s["lens"] += S
            copy = dict(s, **{x: s[x].clone() for x in ("kp", "vp", "bounds")})
            want = run(*(copy[x] for x in names))
            got = traced(*(s[x] for x in names))
            torch.cuda.synchronize()
            assert all(torch.equal(x, y) for x, y in zip(want, got))
            assert all(torch.equal(copy[x].view(torch.uint8), s[x].view(torch.uint8)) for x in ("kp", "vp", "bounds"))


def test_an_append_into_a_tensor(T):
    """cache_append_into: a tensor beside q, q itself, no q; what does not fit."""
    s = step_state(T, 16, 5)
    op, w = torch.ops.shaobo_fa3.cache_append_into, (s["table"], s["lens"], None)
    kp, vp, bounds = (s[n].clone() for n in ("kp", "vp", "bounds"))
    want = T.cache_append(s["k"], s["v"], kp, vp, q=s["q"], freqs=s["fr"], bounds=bounds, page_table=s["table"],
                          kv_lens=s["lens"])
    room = torch.full((3, 5, 8, 144), 7.0, dtype=BF, device="cuda")
    for out in (room[..., 8:136].transpose(1, 2), torch.zeros_like(s["q"])):
        assert op(s["k"], s["v"], s["kp"], s["vp"], *w, s["q"], None, s["fr"], False, s["bounds"], out) is None
        assert torch.equal(out, want) and torch.equal(kp, s["kp"]) and torch.equal(vp, s["vp"])
        assert torch.equal(bounds, s["bounds"])
    assert (room[..., :8] == 7.0).all() and (room[..., 136:] == 7.0).all()
    q = s["q"].clone()
    op(s["k"], s["v"], s["kp"], s["vp"], *w, q, None, s["fr"], False, None, q)
    assert torch.equal(q, want)
    op(s["k"], s["v"], s["kp"], s["vp"], *w, None, None, s["fr"])
    assert torch.equal(kp, s["kp"])
    for q_out in (None, want[:, :4], want[:, :, :4], want.half(), want.cpu(), want[:2]):
        refused("q_out", lambda: op(s["k"], s["v"], s["kp"], s["vp"], *w, s["q"], None, s["fr"], False, None, q_out))
    refused("q_out", lambda: op(s["k"], s["v"], s["kp"], s["vp"], *w, None, None, s["fr"], False, None, want))
    refused("no gradient", lambda: op(s["k"], s["v"], s["kp"], s["vp"], *w, s["q"], None, s["fr"], False, None,
                                      want.clone().requires_grad_()))
    args = (s["k"], s["v"], s["kp"], s["vp"], *w, s["q"], None, s["fr"], False, s["bounds"], torch.empty_like(s["q"]))
    torch.library.opcheck(op.default, args, test_utils=("test_schema", "test_faketensor"))
    torch.cuda.synchronize()


@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("S,new", [(1, None), (4, None), (40, None), (9, [5, 0, 9, 2, 7, 1])])
def test_tokens_past_the_table_are_not_written(T, bits, S, new):
    """Lengths past the table's places: nothing held is written over, tokens that are
    in the table go to their places, keys and queries turn by theirs -- as under a
    wider table whose further pages are none."""
    ps, width, B, D = 32, 2, 6, 64
    gen = gen_of(6)
    k, v, q = (rows(gen, B, h, S, D, BF) for h in (2, 2, 4))
    fr = T.rotary_freqs([D // 2], device="cuda")
    lens = i32([64, 65, 66, 64 + S, 64 + S // 2, 1 << 20])
    table = torch.randperm(B * width, generator=gen, device="cuda").int().view(B, width)
    results = []
    for t in (table, torch.cat((table, torch.full((B, 1 << 15), -1, device="cuda").int()), 1)):
        kp, vp, bounds = T.cache_pages(B * width, 2, ps, D, BF, bits=bits, bounds=True)
        old = rows(gen_of(7), B, 2, 64, D, BF)
        T.cache_append(old, old, kp, vp, page_table=table, kv_lens=i32([64] * B), bounds=bounds)
        qt = T.cache_append(k, v, kp, vp, q=q, freqs=fr, bounds=bounds, page_table=t, kv_lens=lens,
                            new_lens=None if new is None else i32(new))
        results.append((kp.view(torch.uint8), vp.view(torch.uint8), bounds, qt))
    for a, b in zip(*results):
        assert torch.equal(a, b)
    # lengths that no table has
    kp, vp, bounds = (x.clone() for x in (kp, vp, bounds))
    T.cache_append(k, v, kp, vp, q=q, freqs=fr, bounds=bounds, page_table=table, kv_lens=i32([2147483647] * B))
    torch.cuda.synchronize()
    assert torch.equal(kp.view(torch.uint8), results[0][0]) and torch.equal(vp.view(torch.uint8), results[0][1])
    assert torch.equal(bounds, results[0][2])


def test_written_tensors_that_overlap_are_refused(T):
    """Pages that are one memory, by a stride of zero or k's and v's the same, are
    read but not written; likewise q's output."""
    for bits in (16, 4):
        s = step_state(T, bits, 2)
        w = dict(page_table=s["table"], kv_lens=s["lens"])
        kp, vp = s["kp"], s["vp"]
        for k_pages, v_pages in ((kp[:1].expand(60, -1, -1, -1), vp), (kp, vp[:, :1].expand(-1, 2, -1, -1)), (kp, kp)):
            refused("overlap", lambda: T.cache_append(s["k"], s["v"], k_pages, v_pages, **w))
            if k_pages.shape == v_pages.shape:
                T.cache_attention(s["q"], k_pages, v_pages, **w)
                T.cache_read(k_pages, v_pages, seqlen=10, dtype=BF, **w)
        op, a = torch.ops.shaobo_fa3.cache_append_into, (s["k"], s["v"], kp, vp, s["table"], s["lens"], None)
        room = torch.zeros(5, 8, 2, 128, dtype=BF, device="cuda")
        room[1:4] = s["q"]
        for q, q_out in ((s["q"], s["q"][:1].expand(3, -1, -1, -1)), (room[1:4], room[:3]), (room[1:4], room[2:])):
            refused("overlap|apart", lambda: op(*a, q, None, s["fr"], False, None, q_out))
        op(*a, room[1:4], None, s["fr"], False, None, room[1:4])
        # one pool, k's and v's pages in turn, beside pages of their own
        pool = torch.zeros(61, *kp.shape[1:], dtype=kp.dtype, device="cuda")
        even = dict(page_table=(2 * torch.randperm(30, generator=gen_of(1), device="cuda")).int().view(3, 10),
                    kv_lens=i32([300, 64, 2]))
        apart = [torch.zeros_like(kp), torch.zeros_like(vp)]
        T.cache_append(s["k"], s["v"], *apart, **even)
        T.cache_append(s["k"], s["v"], pool[:-1], pool[1:], **even)
        assert torch.equal(pool[:-1][::2], apart[0][::2]) and torch.equal(pool[1:][::2], apart[1][::2])
    torch.cuda.synchronize()


def test_a_token_whose_own_page_is_none(T):
    """Its own page is left out of the list as any absent page is; the others stay."""
    s = step_state(T, 16)
    table = s["table"].clone()
    s["lens"] = i32([901, 451, 1])
    table[0, 14], table[0, 2], table[1, 7], table[2, 0] = -1, 60, -5, 1 << 30
    w = dict(page_table=table, kv_lens=s["lens"])
    sel = T.cache_select(s["q"], s["bounds"], page_size=64, count=20, **w)
    want = [[n for n in range(14) if n != 2], list(range(7)), []]
    for b, pages in enumerate(want):
        assert (sel[b, :, 0] == i32(pages + [-1] * (20 - len(pages)))).all()
    few = T.cache_select(s["q"], s["bounds"], page_size=64, count=3, **w)
    cache = dict(table=table, kv=[901, 451, 1], new=[1] * 3, page_size=64)
    assert torch.equal(few, O.select(s["q"], s["bounds"], cache, 3)) and (few[0] >= 0).all()


@pytest.mark.parametrize("bits,dtype", [(16, BF), (4, BF), (4, HF)])
@pytest.mark.parametrize("S", [1, 3, 100])
def test_large_values(T, S, bits, dtype):
    """V up to the size that the header promises: |v| times 2^8 times the keys below 2^127
    (in fp16 the type's own largest)."""
    kv = 500  # < 2^9
    cache, q, o = attn_case(dict(kv=[kv, 70], S=S, Hq=8, D=128), bits, dtype)
    top = 2.0 ** 110 if dtype == BF else 65504.0
    x = O.rows_of(cache["v"], bits)
    factor = top / float(x.abs().max())
    if bits == 16:
        cache["v"] = (cache["v"].double() * factor).to(dtype)
    else:
        code, scale = O.parts(cache["v"])
        cache["v"] = O.pack(code, (scale.double() * factor).float())
    assert float(O.rows_of(cache["v"], bits).abs().max()) > 0.99 * top
    out, _ = check_attn(T, cache, q, o)
    assert torch.isfinite(out).all()


@pytest.mark.parametrize("bits", [16, 4])
def test_an_append_takes_lengths_into_their_range(T, bits):
    """Lengths below 0, more new tokens than rows or than the sequence has, fewer
    than none: the same rows written as with lengths in range."""
    gen = gen_of(2)
    k, v, q = (rows(gen, 6, h, 9, 64, BF) for h in (2, 2, 4))
    fr = T.rotary_freqs([32], device="cuda")
    table = torch.randperm(24, generator=gen, device="cuda").int().view(6, 4)
    got = []
    for kv, new in (([-5, 100, 100, 3, 3, -2147483648], [4, 2147483647, -7, 2147483647, 5, -2147483648]),
                    ([0, 100, 100, 3, 3, 0], [4, 9, 0, 9, 5, 0])):
        kp, vp, bounds = T.cache_pages(24, 2, 32, 64, BF, bits=bits, bounds=True)
        qt = T.cache_append(k, v, kp, vp, q=q, freqs=fr, bounds=bounds, page_table=table, kv_lens=i32(kv), new_lens=i32(new))
        got.append((kp, vp, bounds, qt))
    torch.cuda.synchronize()
    for a, b in zip(*got):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))
    want = torch.zeros(24, 32, dtype=torch.bool, device="cuda")  # the rows that hold tokens
    for b, places in ((1, range(91, 100)), (3, range(3)), (4, range(3))):
        for p in places:
            want[table[b, p // 32], p % 32] = True
    written = kp != 0 if bits == 16 else O.parts(kp)[1][..., None] != 0
    assert torch.equal(written.any(-1).any(1), want)
