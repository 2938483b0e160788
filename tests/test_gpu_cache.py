"""The paged cache's kernels against their definitions (cache_oracle.py):
appended rows, codes, bounds and selected pages exactly, attention element by
element within counted roundings -- lengths around the edges of pages, blocks
and tiles, padding, pages that are none, every option, both widths."""
import math

import pytest

import attn_oracle as A
import cache_oracle as O
import shaobo_fa3 as F
from test_gpu_attn import i32, within

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


def make_cache(gen, kv, new, Hkv=2, D=64, ps=64, bits=16, dtype=BF, width=None, spare=3, std=1.0):
    """A cache of random rows, pages in random order, -1 behind each sequence."""
    kv, new = list(kv), list(new)
    used = [-(-max(0, n) // ps) for n in kv]
    width = max(used + [1]) if width is None else width
    used = [min(u, width) for u in used]
    pages = sum(used) + spare
    order = torch.randperm(pages, generator=gen, device="cuda")
    table = torch.full((len(kv), width), -1, dtype=torch.int32, device="cuda")
    at = 0
    for b, n in enumerate(used):
        table[b, :n] = order[at:at + n].int()
        at += n
    c = dict(bits=bits, table=table, kv=kv, new=new, page_size=ps, D=D, dtype=dtype)
    for n in ("k", "v"):
        x = (torch.randn(pages, Hkv, ps, D, generator=gen, device="cuda") * std).to(dtype)
        c[n] = O.pack(*O.codes_of(x)) if bits == 4 else x
    return c


def rows(gen, B, H, S, D, dtype, bshd=False, std=1.0):
    shape = (B, S, H, D) if bshd else (B, H, S, D)
    x = (torch.randn(shape, generator=gen, device="cuda") * std).to(dtype)
    return x.transpose(1, 2) if bshd else x


def where(c):
    """The operators' arguments for a cache's sequences."""
    return dict(page_table=c["table"], kv_lens=i32(c["kv"]), new_lens=i32(c["new"]))


def gen_of(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


# ---------------------------------------------------------------------------
ATTN = [
    # one token: caches around the edges of blocks, tiles and pages
    dict(kv=[1], D=128), dict(kv=[31, 32, 33]), dict(kv=[63, 64, 65], D=128), dict(kv=[127, 128, 129], ps=32),
    dict(kv=[300, 5], D=128, Hq=8), dict(kv=[1000, 257, 512], ps=128, Hq=4), dict(kv=[2049], ps=1024, D=128),
    dict(kv=[700, 64], Hq=32, Hkv=2, D=128), dict(kv=[333], Hq=7, Hkv=1, bshd=True),
    dict(kv=[400, 90], Hq=40, Hkv=2, D=128), dict(kv=[150, 41], Hq=64, Hkv=1),
    # key axes long enough to be cut
    dict(kv=[5000], D=128, Hq=8, Hkv=2), dict(kv=[9000, 100], ps=32, Hq=4), dict(kv=[20000], ps=256, Hq=2, Hkv=1, D=128),
    # a few tokens, and parts of prompts
    dict(kv=[77, 140], S=3, D=128, Hq=8), dict(kv=[260, 33], S=9, Hq=12, Hkv=4), dict(kv=[5], S=5),
    dict(kv=[64, 130], S=64, D=128), dict(kv=[500, 257], S=100, Hq=4, ps=32), dict(kv=[300], S=300, D=128, bshd=True),
    dict(kv=[1500, 700], S=129, Hq=8, D=128, ps=128), dict(kv=[4000], S=70, Hq=8, Hkv=2, ps=32, D=128),
    dict(kv=[900, 1100, 64, 70], S=64, Hq=16, Hkv=8, D=128), dict(kv=[640], S=513, Hq=2, Hkv=1, ps=32),
    # padding, no tokens, fewer places than rows
    dict(kv=[40, 90, 70], new=[1, 0, 7], S=7, Hq=4), dict(kv=[300, 200], new=[130, 0], S=130, D=128),
    dict(kv=[10, 0], S=40, Hq=4), dict(kv=[0, 3], S=1), dict(kv=[20], new=[20], S=33, D=128),
    dict(kv=[100, 30], S=140, ps=32, D=128), dict(kv=[2000, 1700], new=[33, 64], S=64, D=128, Hq=8),
    # options
    dict(kv=[500, 90], S=3, causal=False, Hq=4, D=128), dict(kv=[200, 300], S=150, causal=False),
    dict(kv=[400], softcap=5.0, std=4.0, Hq=4, D=128), dict(kv=[300, 200], S=100, softcap=150.0, std=20.0),
    dict(kv=[400, 90], slopes=1, Hq=8), dict(kv=[400, 900], S=130, slopes=2, D=128, Hq=4),
    dict(kv=[333], S=5, slopes=1, softcap=20.0, Hq=4, D=128), dict(kv=[333, 290], S=140, slopes=1, softcap=9.0, ps=32),
    dict(kv=[300, 250], S=100, prefix=[220, 1000], Hq=4), dict(kv=[200, 70], S=40, prefix=[170, -3], D=128),
    dict(kv=[400], scale=-0.3, D=128), dict(kv=[400, 50], S=130, scale=0.0), dict(kv=[64], S=9, scale=-0.2, softcap=3.0),
    # pages that are none, anywhere
    dict(kv=[400, 130], holes=[0, 3], Hq=4, D=128), dict(kv=[500], S=150, holes=[0, 1, 4, 7], ps=32),
    dict(kv=[640, 70], S=70, holes=[2, 5, 9], ps=32, D=128, Hq=4), dict(kv=[100, 100], S=3, holes=[0, 1]),
    dict(kv=[3000], S=9, holes=[3, 4, 5, 6, 20], Hq=8, D=128), dict(kv=[700], S=200, holes=[0, 2, 10], D=128, prefix=[600]),
]


def attn_case(case, bits, dtype, seed=3):
    c = dict(Hq=2, Hkv=2, D=64, S=1, ps=64, causal=True, std=1.0, bshd=False)
    c.update(case)
    gen = gen_of(seed)
    cache = make_cache(gen, c["kv"], c.get("new", [c["S"]] * len(c["kv"])), c["Hkv"], c["D"], c["ps"],
                       bits, dtype)
    for n, h in enumerate(c.get("holes", ())):
        if h < cache["table"].shape[1]:
            cache["table"][:, h] = (-1, cache["k"].shape[0], -2 ** 31, 2 ** 31 - 1)[n % 4]
    Hq = max(c["Hq"], c["Hkv"])
    q = rows(gen, len(c["kv"]), Hq, c["S"], c["D"], dtype, c["bshd"], c["std"])
    o = dict(causal=c["causal"], softcap=c.get("softcap", 0.0), scale=c.get("scale"))
    if c.get("slopes") == 1:
        o["slopes"] = torch.exp2(-torch.arange(1, Hq + 1, device="cuda").float())
    elif c.get("slopes") == 2:
        o["slopes"] = torch.rand(len(c["kv"]), Hq, generator=gen, device="cuda")
    if "prefix" in c:
        o["prefix"] = c["prefix"]
    return cache, q, o


def check_attn(T, cache, q, o, selected=None):
    kw = dict(causal=o["causal"], softmax_scale=o["scale"], softcap=o["softcap"],
              slopes=o.get("slopes"), selected=selected, return_lse=True)
    if "prefix" in o:
        kw["prefix_lens"] = i32(o["prefix"])
    out, lse = T.cache_attention(q, cache["k"], cache["v"], **where(cache), **kw)
    torch.cuda.synchronize()
    assert out.shape == q.shape and out.dtype == q.dtype and lse.dtype == torch.float32
    want, wlse, off, lse_off = O.attend(q, cache, selected=selected, **o)
    within("lse", lse, wlse, lse_off)
    within("out", out, want, off)
    return out, lse


def ids(c):
    return "-".join(f"{k}{v}" for k, v in c.items()).replace(" ", "")


@pytest.mark.parametrize("bits,dtype", [(16, BF), (4, BF), (16, HF), (4, HF)])
@pytest.mark.parametrize("case", ATTN, ids=ids)
def test_attention_against_fp64(T, case, bits, dtype):
    check_attn(T, *attn_case(case, bits, dtype))


@pytest.mark.parametrize("case", [
    dict(kv=[100], D=8), dict(kv=[500], D=40, S=3), dict(kv=[200, 90], D=96, S=100), dict(kv=[90], D=120, S=9),
    dict(kv=[3000], D=72, Hq=4),
], ids=ids)
def test_head_dims_that_are_no_whole_tile(T, case):
    check_attn(T, *attn_case(case, 16, BF))


SPARSE = [
    dict(kv=[300], D=128, Hq=8, count=3), dict(kv=[1000, 64, 10], Hq=4, count=4, ps=32),
    dict(kv=[5000, 2000], Hq=8, Hkv=2, D=128, count=33), dict(kv=[700], S=5, Hq=6, Hkv=2, count=2, ps=128),
    dict(kv=[260, 90], new=[3, 0], S=4, Hq=4, count=3, D=128), dict(kv=[3], S=5, count=2),
    dict(kv=[900], Hq=40, Hkv=1, count=5, D=128), dict(kv=[900], Hq=40, Hkv=1, S=3, count=5), dict(kv=[40], count=9),
    dict(kv=[800], softcap=4.0, std=3.0, count=6), dict(kv=[800, 300], slopes=1, count=6, Hq=4, D=128),
    dict(kv=[640], S=70, count=4, Hq=4, ps=32), dict(kv=[9000], count=100, Hq=8, ps=64, D=128),
    dict(kv=[500], causal=False, S=2, count=3),
]


@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("case", SPARSE, ids=ids)
def test_selected_pages(T, case, bits, dtype):
    """Random lists: any order, numbers that are no page, -1 among them."""
    cache, q, o = attn_case(case, bits, dtype, 5)
    gen, N = gen_of(6), cache["table"].shape[1]
    B, Hkv, S, count = q.shape[0], cache["k"].shape[1], q.shape[2], case["count"]
    sel = torch.stack([torch.randperm(max(N, count), generator=gen, device="cuda")[:count]
                       for _ in range(B * Hkv * S)]).view(B, Hkv, S, count).int()
    sel = torch.where(torch.rand(sel.shape, generator=gen, device="cuda") < 0.1, -1, sel)
    check_attn(T, cache, q, o, sel.contiguous())


@pytest.mark.parametrize("bits", [16, 4])
def test_a_page_listed_twice_counts_twice(T, bits):
    cache, q, o = attn_case(dict(kv=[300], Hq=4, D=128), bits, BF)
    check_attn(T, cache, q, o, i32([[[[1, 1, 4]], [[0, 2, 0]]]]))


@pytest.mark.parametrize("bits", [16, 4])
def test_no_page_listed(T, bits):
    cache, q, o = attn_case(dict(kv=[300, 200], Hq=4, S=2), bits, BF)
    sel = i32([[[[-1, 7], [0, -1]], [[99, -5], [-1, -1]]]] * 2)
    out, lse = check_attn(T, cache, q, o, sel)
    assert (out[:, 2:] == 0).all() and torch.isinf(lse[:, 2:]).all()


# ---------------------------------------------------------------------------
APPEND = [
    dict(kv=[1]), dict(kv=[65, 33], D=128, Hq=4), dict(kv=[100, 64, 31], S=5, Hq=4, ps=32),
    dict(kv=[40], S=40, D=128, Hq=2, bshd=True), dict(kv=[300, 200], S=130, D=128, Hq=8, Hkv=8),
    dict(kv=[500], S=211, Hkv=5, Hq=15, ps=128, bshd=True), dict(kv=[90, 0, 70], new=[5, 0, 17], S=17, Hq=4),
    dict(kv=[20, 10], S=33, Hq=2), dict(kv=[200], S=64, D=128, pairs=32, Hq=4), dict(kv=[200], S=20, pairs=0, Hq=4),
    dict(kv=[77, 80], S=19, D=128, inter=True, Hq=4), dict(kv=[90], S=33, pairs=8, inter=True, D=128),
    dict(kv=[129], S=100, axes=2, D=128, Hq=4), dict(kv=[70, 60], S=9, axes=3, inter=True, Hq=2),
    dict(kv=[1030], S=1000, ps=1024, D=128), dict(kv=[70, 95], S=50, holes=[1], ps=32, Hq=2),
    dict(kv=[10000], S=3, place="far", axes=1, D=128, Hq=2), dict(kv=[50], S=17, q=False, D=128),
    dict(kv=[33, 65, 97, 1, 2, 3, 4, 5], Hq=8, Hkv=4, D=128),
]


def append_case(case, bits, dtype, seed=9):
    c = dict(Hkv=2, D=64, S=1, ps=64, bshd=False, axes=0, inter=False, q=True)
    c.update(case)
    c.setdefault("Hq", c["Hkv"])
    gen, B = gen_of(seed), len(c["kv"])
    cache = make_cache(gen, c["kv"], c.get("new", [c["S"]] * B), c["Hkv"], c["D"], c["ps"], bits, dtype)
    for n, h in enumerate(c.get("holes", ())):
        cache["table"][:, h] = (-1, cache["k"].shape[0])[n % 2]
    k, v = (rows(gen, B, c["Hkv"], c["S"], c["D"], dtype, c["bshd"]) for _ in range(2))
    q = rows(gen, B, c["Hq"], c["S"], c["D"], dtype, c["bshd"]) if c["q"] else None
    P = c.get("pairs", c["D"] // 2)
    o = dict(freqs=None, positions=None, interleaved=c["inter"])
    if P:
        o["freqs"] = (10000.0 ** (-torch.arange(P, device="cuda").double() / P)).float()[None]
    if c["axes"]:
        owner = torch.arange(P, device="cuda") * c["axes"] // P
        o["freqs"] = torch.where(owner == torch.arange(c["axes"], device="cuda")[:, None], o["freqs"], 0.0)
        top = 2 ** 21 if c.get("place") == "far" else 500
        o["positions"] = torch.randint(0, top, (c["axes"], B, c["S"]), generator=gen, device="cuda")
    return cache, k, v, q, o


def check_append(T, cache, k, v, q, o, bounds=None):
    """One append against the definition; the cache's tensors are written."""
    before = {n: cache[n].clone() for n in ("k", "v")}
    old = None if bounds is None else bounds.clone()
    got = T.cache_append(k, v, cache["k"], cache["v"], q=q, bounds=bounds, **where(cache), **o)
    torch.cuda.synchronize()
    fresh = dict(cache, **before)
    if q is not None:
        want, off = O.turned(q, cache, o["freqs"], o["positions"], o["interleaved"])
        within("q", got, want, off)
    else:
        assert got is None
    kt, off = O.turned(k, cache, o["freqs"], o["positions"], o["interleaved"])
    # the keys in 16 bits, which codes and bounds go by: off the formula's by one rounding
    k16 = k
    if o["freqs"] is not None:
        k16 = T.cache_append(k, v, *T.cache_pages(0, k.shape[1], cache["page_size"], k.shape[3], k.dtype)[:2],
                             q=k, **where(cache), **o)
        within("k", k16, kt, off)
    want = {n: fresh[n].clone() for n in ("k", "v")}
    ps, seen = cache["page_size"], {}
    for b in range(k.shape[0]):
        kv, new = O.clipped(cache, b)
        for i in range(new):
            place = kv - new + i
            page = int(cache["table"][b, place // ps]) if place >= 0 else -1
            if not 0 <= page < cache["k"].shape[0]:
                continue
            for n, x in (("k", k16), ("v", v)):
                seen.setdefault((n, page), []).append((place % ps, x[b, :, i]))
    for (n, page), items in seen.items():
        at = torch.tensor([r for r, _ in items], device="cuda")
        x = torch.stack([y for _, y in items], 1)  # [H, rows, D]
        if cache["bits"] == 16:
            want[n][page, :, at] = x
        else:
            code, scale = O.parts(want[n][page:page + 1])
            c, s = O.codes_of(x)
            code[0, :, at], scale[0, :, at] = c.int(), s
            want[n][page] = O.pack(code, scale)[0]
        if n == "k" and bounds is not None:
            low, high = x.float().amin(1), x.float().amax(1)
            if int(at.min()) > 0:
                low, high = torch.minimum(low, old[page, :, 0].float()), \
                    torch.maximum(high, old[page, :, 1].float())
            old[page, :, 0], old[page, :, 1] = low.to(k.dtype), high.to(k.dtype)
    for n in ("k", "v"):  # bit by bit: rows that are not written stay as they were
        assert torch.equal(cache[n].view(torch.uint8), want[n].view(torch.uint8)), n
    if bounds is not None:
        assert torch.equal(bounds, old)


@pytest.mark.parametrize("bits,dtype", [(16, BF), (4, BF), (16, HF), (4, HF)])
@pytest.mark.parametrize("with_bounds", [False, True])
@pytest.mark.parametrize("case", APPEND, ids=ids)
def test_append(T, case, with_bounds, bits, dtype):
    cache, k, v, q, o = append_case(case, bits, dtype)
    bounds = None
    if with_bounds:
        n = cache["k"].shape[0]
        b = torch.randn(n, k.shape[1], 2, k.shape[3], generator=gen_of(1), device="cuda").to(dtype)
        bounds = b.sort(2)[0].contiguous()
    check_append(T, cache, k, v, q, o, bounds)


@pytest.mark.parametrize("D", [8, 24, 72, 96, 120])
def test_append_other_head_dims(T, D):
    gen = gen_of(2)
    cache = make_cache(gen, [70, 40], [33, 9], 3, D, 32)
    k, v, q = (rows(gen, 2, h, 33, D, BF) for h in (3, 3, 6))
    P = D // 16 * 8
    f = None if P == 0 else torch.rand(1, P, generator=gen, device="cuda")
    bounds = torch.zeros(cache["k"].shape[0], 3, 2, D, dtype=BF, device="cuda")
    check_append(T, cache, k, v, q, dict(freqs=f, positions=None, interleaved=False), bounds)


@pytest.mark.parametrize("bits,dtype", [(16, BF), (4, HF)])
@pytest.mark.parametrize("kind", [torch.int32, torch.int64, torch.float32])
@pytest.mark.parametrize("case", [
    dict(kv=[33, 65], D=128, Hq=4, axes=1), dict(kv=[129], S=100, axes=2, D=128, Hq=4), dict(kv=[70, 60], S=9, axes=3, inter=True, Hq=2),
    dict(kv=[10000], S=3, place="far", axes=1, D=128, Hq=2), dict(kv=[40, 90], new=[3, 5], S=7, axes=2),
], ids=ids)
def test_append_takes_positions_of_any_type(T, case, kind, bits, dtype):
    """int32, int64 and fp32 (with quarters), below 0 too; as they lie, or a row of
    positions that the batch shares and reads with strides."""
    cache, k, v, q, o = append_case(case, bits, dtype)
    x = (o["positions"] - 250).to(kind)
    if kind == torch.float32:
        x = x + 0.25 * torch.randint(0, 4, x.shape, generator=gen_of(3), device="cuda")
    check_append(T, cache, k, v, q, dict(o, positions=x))
    shared = x[:, :1].transpose(0, 2).contiguous().transpose(0, 2).expand_as(x)
    bounds = torch.zeros(cache["k"].shape[0], k.shape[1], 2, k.shape[3], dtype=dtype, device="cuda")
    check_append(T, cache, k, v, q, dict(o, positions=shared), bounds)


def special_rows(dtype):
    """Rows at the levels' borders and of odd sizes: [n, 64]."""
    x = torch.zeros(16, 64)
    for r, top in enumerate((6.0, 12.0, 3.0, 96.0, 7.0, 1.0)):
        mids = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0]) * top / 6
        x[r, :7], x[r, 7:14], x[r, 14] = mids, -mids, top
        x[r, 15:22] = mids * 1.01
        x[r, 22:29] = mids * 0.99
    x[7] = torch.randn(64, generator=torch.Generator().manual_seed(0)) * torch.finfo(dtype).max / 8
    x[8, 3] = torch.finfo(dtype).max
    x[9, 5] = torch.finfo(dtype).smallest_normal
    x[10, 9] = -torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps  # the smallest at all
    x[11] = -0.0
    x[12] = torch.linspace(-1, 1, 64)
    x[13, 0], x[13, 1] = math.inf, 1.0
    x[14, 2] = math.nan
    return x.to(dtype)


@pytest.mark.parametrize("dtype", [BF, HF])
def test_codes_at_the_levels_borders(T, dtype):
    x = special_rows(dtype).cuda()[None, None]
    k, v, _ = T.cache_pages(1, 1, 32, 64, dtype, bits=4)
    T.cache_append(x, x.flip(3).contiguous(), k, v, page_table=i32([[0]]), kv_lens=i32([16]))
    for pages, y in ((k, x), (v, x.flip(3))):
        code, scale = O.parts(pages)
        c, s = O.codes_of(y)
        assert torch.equal(code[0, 0, :16], c[0, 0].int())
        assert torch.equal(scale[0, 0, :16].nan_to_num(nan=-1.0), s[0, 0].nan_to_num(nan=-1.0))
        assert (scale[0, 0, 16:] == 0).all() and torch.isnan(scale[0, 0, 13:15]).all()
    a, b = T.cache_read(k, v, page_table=i32([[0]]), kv_lens=i32([16]), seqlen=16, dtype=dtype)
    # (the widest gap between levels is 2 of 6, a value off by half of it: a sixth of the largest)
    top = x.double().abs().amax(-1, keepdim=True)
    fine = torch.isfinite(top[..., 0])
    assert ((a.double() - x.double()).abs()[fine] <= (top / 6 * 1.001 + 2.0 ** -24)[fine]).all()
    assert torch.isnan(a[0, 0, 13:15]).all() and torch.isnan(b[0, 0, 13:15]).all()


@pytest.mark.parametrize("bits,dtype", [(16, BF), (4, BF), (16, HF), (4, HF)])
@pytest.mark.parametrize("kv,seqlen,ps,D", [([70, 0, 33], 70, 32, 64), ([129, 64], 200, 64, 128), ([5], 3, 128, 64)])
def test_read(T, kv, seqlen, ps, D, bits, dtype):
    cache = make_cache(gen_of(4), kv, [0] * len(kv), 3, D, ps, bits, dtype)
    if cache["table"].shape[1] > 1:
        cache["table"][0, 1] = cache["k"].shape[0] + 5
    got = T.cache_read(cache["k"], cache["v"], page_table=cache["table"], kv_lens=i32(kv), seqlen=seqlen,
                       dtype=dtype)
    for b in range(len(kv)):
        for x, y in zip(got, O.sequence(cache, b)[:2]):
            n = min(seqlen, y.shape[1])
            # (level times scale is exact in fp64 and rounded to fp32, then to the type)
            assert torch.equal(x[b, :, :n], y[:, :n].float().to(dtype))
            assert (x[b, :, n:] == 0).all()


# ---------------------------------------------------------------------------
SELECT = [
    dict(kv=[1], count=1), dict(kv=[300, 65], count=3, Hq=8, D=128), dict(kv=[2000], count=7, ps=32, Hq=5, Hkv=1),
    dict(kv=[5000, 129, 64], count=20, Hq=8, Hkv=2, D=128, ps=32), dict(kv=[700, 70], S=6, count=4, Hq=6, Hkv=2),
    dict(kv=[90, 50], new=[2, 0], S=4, count=3), dict(kv=[3], S=5, count=2), dict(kv=[600], count=64),
    dict(kv=[640, 300], count=4, holes=[0, 3, 9], Hq=4), dict(kv=[40000], count=100, ps=32, Hq=2, Hkv=1),
    dict(kv=[150000], count=64, ps=32, Hq=4, Hkv=1), dict(kv=[9000], count=1, ps=64), dict(kv=[9000], count=2, D=40),
    dict(kv=[4000], S=2, count=30, Hq=36, Hkv=2, D=128),
]


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("kind", ["random", "equal", "coarse", "wild"])
@pytest.mark.parametrize("case", SELECT, ids=ids)
def test_select(T, case, kind, dtype):
    """Equal scores (bounds of few different values, or one), infinities and NaN in bounds."""
    c = dict(Hq=2, Hkv=2, D=64, S=1, ps=64)
    c.update(case)
    gen, B = gen_of(8), len(c["kv"])
    new = c.get("new", [c["S"]] * B)
    used = [-(-n // c["ps"]) for n in c["kv"]]
    pages = sum(used) + 2
    order = torch.randperm(pages, generator=gen, device="cuda").int()
    table = torch.full((B, max(used)), -1, dtype=torch.int32, device="cuda")
    at = 0
    for b, n in enumerate(used):
        table[b, :n] = order[at:at + n]
        at += n
    for n, h in enumerate(c.get("holes", ())):
        table[:, min(h, table.shape[1] - 1)] = (-1, pages)[n % 2]
    x = torch.randn(pages, c["Hkv"], 2, c["D"], generator=gen, device="cuda")
    if kind == "equal":
        x = x[:1].expand_as(x)
    elif kind == "coarse":
        x = x[torch.randint(0, min(pages, 5), (pages,), generator=gen, device="cuda")]
    x = x.sort(2)[0].to(dtype).contiguous()
    if kind == "wild":
        x[::3, :, 1, 5] = math.inf
        x[1::5, :, :, 0] = math.nan
        x[2::7, :, 0, 3] = -math.inf
    q = rows(gen, B, c["Hq"], c["S"], c["D"], dtype)
    cache = dict(table=table, kv=c["kv"], new=new, page_size=c["ps"])
    got = T.cache_select(q, x, page_table=table, kv_lens=i32(c["kv"]), new_lens=i32(new), page_size=c["ps"],
                         count=c["count"])
    torch.cuda.synchronize()
    assert torch.equal(got, O.select(q, x, cache, c["count"]))


@pytest.mark.parametrize("kind", ["random", "equal", "coarse", "wild"])
@pytest.mark.parametrize("count", [1, 64, 600])
@pytest.mark.parametrize("width", [511, 512, 513, 1023, 1024, 1025, 2048, 2049, 4096, 4097])
def test_select_at_the_pick_kernels_widths(T, width, count, kind):
    """Tables as wide as a thread of the pick kernels has pages for, in registers or
    not, and one more or less: all of it used, and half."""
    gen, ps, D = gen_of(width), 32, 64
    pages = width + 2
    x = torch.randn(pages, 1, 2, D, generator=gen, device="cuda")
    if kind == "equal":
        x = x[:1].expand_as(x)
    elif kind == "coarse":
        x = x[torch.randint(0, 5, (pages,), generator=gen, device="cuda")]
    x = x.sort(2)[0].to(BF).contiguous()
    if kind == "wild":
        x[::3, :, 1, 5], x[1::5, :, :, 0], x[2::7, :, 0, 3] = math.inf, math.nan, -math.inf
    q = rows(gen, 1, 2, 1, D, BF)
    table = torch.randperm(pages, generator=gen, device="cuda")[None, :width].int().contiguous()
    for kv in (ps * width, ps * (width // 2) + 5):
        got = T.cache_select(q, x, page_table=table, kv_lens=i32([kv]), page_size=ps, count=count)
        torch.cuda.synchronize()
        assert torch.equal(got, O.select(q, x, dict(table=table, kv=[kv], new=[1], page_size=ps), count))
