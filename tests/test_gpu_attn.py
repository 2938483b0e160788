"""The attention layer's kernels against fp64 (attn_oracle.py), element by
element within bounds that count the roundings: lengths around the tiles'
edges, head counts, head dims, types, layouts, every mask and option, key
axes long enough to be split, and what masked places may hold."""
import ctypes
import math

import pytest

import attn_oracle as A
import shaobo_fa3 as F

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


def randn(gen, B, H, S, D, dtype, bshd=False, std=1.0):
    if bshd:
        return (torch.randn(B, S, H, D, generator=gen, device="cuda") * std).to(dtype).transpose(1, 2)
    return (torch.randn(B, H, S, D, generator=gen, device="cuda") * std).to(dtype)


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def within(name, got, want, off):
    """got equals want within off, element by element; infinities where want's are."""
    got = got.double()
    fin = torch.isfinite(want)
    assert torch.equal(torch.isfinite(got), fin), name + ": not finite in other places"
    assert torch.equal(got[~fin], want[~fin]), name
    d = (got - want)[fin].abs() - off[fin]
    worst = float(d.max()) if d.numel() else -1.0
    assert worst <= 0.0, f"{name}: {worst:.3e} over its bound"


def make(case, seed=3):
    """Inputs of a case: (q, k, v, dout, options)."""
    c = dict(B=2, Hq=2, Hkv=2, Sq=64, Sk=None, D=64, dtype=BF, bshd=False, std=1.0, causal=True)
    c.update(case)
    Sk = c["Sq"] if c["Sk"] is None else c["Sk"]
    gen = torch.Generator(device="cuda").manual_seed(seed)
    q = randn(gen, c["B"], c["Hq"], c["Sq"], c["D"], c["dtype"], c["bshd"], c["std"])
    k, v = (randn(gen, c["B"], c["Hkv"], Sk, c["D"], c["dtype"], c["bshd"]) for _ in range(2))
    do = randn(gen, c["B"], c["Hq"], c["Sq"], c["D"], c["dtype"], c["bshd"])
    o = dict(causal=c["causal"])
    for n in ("softcap", "softmax_scale"):
        if n in c:
            o[n] = c[n]
    if c.get("slopes"):
        h = torch.arange(1, c["Hq"] + 1, device="cuda", dtype=torch.float32)
        o["slopes"] = torch.exp2(-h) if c["slopes"] == 1 else \
            torch.rand(c["B"], c["Hq"], generator=gen, device="cuda")
    if "docs" in c:  # document lengths around c["docs"], -1 for some of the rest
        def ids(n):
            steps = torch.rand(c["B"], n, generator=gen, device="cuda") < 1.0 / c["docs"]
            x = steps.int().cumsum(1).int() * 3
            x[:, n - n // 9:] = -1
            return x.contiguous()
        o["documents"] = ids(c["Sq"])
        if Sk != c["Sq"]:
            o["documents_k"] = ids(Sk)
    if "prefix" in c:
        o["prefix_lens"] = i32(c["prefix"])
    if "kv" in c:
        o["kv_lens"] = i32(c["kv"])
    return q, k, v, do, o


def op_args(o):
    return (o["causal"], o.get("softmax_scale"), o.get("softcap", 0.0), o.get("slopes"),
            o.get("documents"), o.get("documents_k"), o.get("prefix_lens"), o.get("kv_lens"))


def oracle_options(o):
    o = dict(o)
    if "softmax_scale" in o:
        o["scale"] = o.pop("softmax_scale")
    return o


def run_both(q, k, v, do, o):
    """Forward and backward on the GPU, both checked."""
    ops = torch.ops.shaobo_fa3
    out, lse = ops.attn_forward(q, k, v, *op_args(o))
    torch.cuda.synchronize()
    assert out.dtype == q.dtype and out.shape == q.shape and lse.dtype == torch.float32
    want, wlse, off, lse_off = A.forward(q, k, v, **oracle_options(o))
    within("lse", lse, wlse, lse_off)
    within("out", out, want, off)
    grads = dict(zip(("dq", "dk", "dv", "delta"),
                     ops.attn_backward(do, q, k, v, out, lse, *op_args(o))))
    torch.cuda.synchronize()
    for n, (g, b) in A.backward(do, q, k, v, out, lse, **oracle_options(o)).items():
        within(n, grads[n], g, b)
    return out, lse, grads


CASES = [
    # lengths around the 16-row, 32-row, 64-key and 128-row edges
    dict(Sq=1), dict(Sq=2, D=128), dict(Sq=15, dtype=HF), dict(Sq=17, D=128, causal=False),
    dict(Sq=31), dict(Sq=33, D=128, dtype=HF), dict(Sq=63), dict(Sq=65, causal=False),
    dict(Sq=127, D=128), dict(Sq=128, D=128, dtype=HF), dict(Sq=129, D=128),
    dict(Sq=191, causal=False, dtype=HF), dict(Sq=257, D=128, bshd=True), dict(Sq=300, B=1),
    # fewer and more keys than queries (rows that see none, a cache)
    dict(Sq=100, Sk=40), dict(Sq=70, Sk=3, D=128), dict(Sq=40, Sk=333, D=128),
    dict(Sq=40, Sk=333, causal=False, dtype=HF), dict(Sq=1, Sk=200, D=128), dict(Sq=5, Sk=129),
    # grouped and shared heads
    dict(Sq=130, Hq=8, Hkv=2, D=128), dict(Sq=77, Hq=6, Hkv=2, bshd=True), dict(Sq=50, Hq=7, Hkv=1),
    dict(Sq=140, Hq=16, Hkv=16, B=1, D=128), dict(Sq=3, Hq=12, Hkv=4, Sk=90, D=128),
    dict(Sq=90, Hq=8, Hkv=8, B=4, causal=False),
    # head dims that are no whole tile
    dict(Sq=70, D=8), dict(Sq=70, D=24, dtype=HF, bshd=True), dict(Sq=70, D=56), dict(Sq=130, D=72),
    dict(Sq=130, D=96, bshd=True), dict(Sq=130, D=120, causal=False, dtype=HF),
    # capped scores, small and large caps and scores
    dict(Sq=150, softcap=5.0, std=3.0), dict(Sq=150, softcap=30.0, std=8.0, D=128),
    dict(Sq=150, softcap=101.0, std=3.0, D=128), dict(Sq=150, softcap=1000.0, std=20.0, dtype=HF),
    dict(Sq=66, softcap=0.5, std=10.0, causal=False, dtype=HF),
    # distance bias
    dict(Sq=150, slopes=1), dict(Sq=150, slopes=2, D=128, causal=False), dict(Sq=9, Sk=300, slopes=2),
    dict(Sq=130, slopes=1, softcap=20.0, D=128, dtype=HF), dict(Sq=100, Sk=50, slopes=1, causal=False),
    # caps and scales at the ends of their range
    dict(Sq=70, softcap=1e-38, D=128), dict(Sq=70, softcap=1e30), dict(Sq=70, softcap=1e-30, softmax_scale=1e8),
    dict(Sq=70, softmax_scale=1e-35), dict(Sq=70, softmax_scale=1e-35, slopes=1), dict(Sq=70, softcap=100.0, std=30.0),
    # prefixes: none, inside a tile, past the keys
    dict(Sq=150, prefix=[0, 70]), dict(Sq=150, prefix=[149, 1000], D=128),
    dict(Sq=200, prefix=[65, -5], softcap=10.0, Hq=4), dict(Sq=40, Sk=100, prefix=[90, 10], slopes=1),
    # documents: long, short, of one token, with padding
    dict(Sq=300, docs=100.0), dict(Sq=300, docs=10.0, D=128), dict(Sq=300, docs=1.0, causal=False),
    dict(Sq=513, docs=200.0, causal=False, D=128, Hq=4), dict(Sq=64, docs=1e9),
    dict(Sq=100, Sk=260, docs=40.0, causal=False), dict(Sq=300, docs=60.0, prefix=[100, 200]),
    dict(Sq=300, docs=60.0, softcap=10.0, slopes=1, dtype=HF),
    # keys in use: none, one, some, all, out of range (taken into it)
    dict(Sq=70, kv=[0, 1]), dict(Sq=70, kv=[69, 70], D=128), dict(Sq=70, kv=[-4, 1000]),
    dict(Sq=5, Sk=200, kv=[5, 131], D=128), dict(Sq=5, Sk=200, kv=[3, 64], causal=False),
    dict(Sq=33, Sk=160, kv=[100, 20], docs=30.0, causal=False), dict(Sq=33, Sk=160, kv=[100, 20], slopes=1),
    # scales: given, negative, zero
    dict(Sq=80, softmax_scale=0.3), dict(Sq=80, softmax_scale=-0.2, D=128),
    dict(Sq=80, softmax_scale=0.0), dict(Sq=80, softmax_scale=-0.2, softcap=3.0),
    dict(Sq=80, softmax_scale=0.0, slopes=1), dict(Sq=80, softmax_scale=-0.2, docs=20.0),
]


@pytest.mark.parametrize("case", CASES, ids=lambda c: "-".join(
    f"{k}{str(v).replace('torch.', '')}" for k, v in c.items()))
def test_against_fp64(T, case):
    print("[case]", case, flush=True)
    run_both(*make(case))


# Key axes long enough to be split between workgroups: parts that end inside a
# tile, that a row sees nothing of, and that no row sees anything of.
SPLIT = [
    dict(B=1, Hq=8, Hkv=8, Sq=1, Sk=2049), dict(B=2, Hq=8, Hkv=2, Sq=1, Sk=5000, D=128, kv=[5000, 70]),
    dict(B=3, Hq=4, Hkv=1, Sq=1, Sk=1500, D=128, kv=[0, 1, 1500]),
    dict(B=1, Hq=4, Hkv=4, Sq=1024, causal=True, D=128), dict(B=1, Hq=2, Hkv=1, Sq=900, prefix=[700]),
    dict(B=1, Hq=2, Hkv=2, Sq=1111, docs=150.0, softcap=20.0, D=128, dtype=HF),
    dict(B=1, Hq=2, Hkv=2, Sq=3, Sk=4097, slopes=1, D=128), dict(B=1, Hq=2, Hkv=2, Sq=700, Sk=1300, D=80),
    dict(B=1, Hq=16, Hkv=2, Sq=2, Sk=2500, softcap=30.0, std=5.0, bshd=True),
    dict(B=2, Hq=24, Hkv=8, Sq=7, Sk=1999, dtype=HF, kv=[1999, 8]),
    dict(B=1, Hq=4, Hkv=4, Sq=1, Sk=1500, docs=1e9, causal=False), dict(B=1, Hq=5, Hkv=5, Sq=1, Sk=900, D=40),
]


@pytest.mark.parametrize("case", SPLIT, ids=lambda c: "-".join(
    f"{k}{str(v).replace('torch.', '')}" for k, v in c.items()))
def test_long_key_axis(T, case):
    print("[case]", case, flush=True)
    run_both(*make(case))


@pytest.mark.parametrize("causal,D,cap", [(True, 64, 0.0), (False, 128, 0.0), (False, 64, 8.0)])
def test_steep_and_rising_bias(T, causal, D, cap):
    """Slopes from one that hides all but the next keys to ones below zero
    (far keys weigh most): every row's scores, sums and their gradients."""
    print("[case] slopes", causal, D, cap, flush=True)
    q, k, v, do, o = make(dict(Sq=700, B=1, Hq=8, Hkv=4, D=D, causal=causal))
    o["slopes"] = torch.tensor([300.0, 20.0, 3.0, 1.0, 0.7, 0.05, -0.02, -0.5], device="cuda")
    if cap:
        o["softcap"] = cap
    run_both(q, k, v, do, o)


def test_bias_at_far_places(T):
    """Places past 2^24, where fp32 no longer tells neighbours apart: distances
    are differences of whole numbers."""
    print("[case] far places", flush=True)
    Sk, D = (1 << 24) + 300, 8
    gen = torch.Generator(device="cuda").manual_seed(5)
    k, v = (torch.randn(1, 1, Sk, D, generator=gen, device="cuda").to(HF) for _ in range(2))
    q = torch.randn(1, 1, 5, D, generator=gen, device="cuda").to(HF)
    slopes = torch.full((1,), 0.9, device="cuda")
    out, lse = torch.ops.shaobo_fa3.attn_forward(q, k, v, True, None, 0.0, slopes)
    # keys further than 2000 back weigh less than e^-1700
    want, wlse, off, lse_off = A.forward(q, k[:, :, -2000:], v[:, :, -2000:], True, slopes=slopes)
    within("lse", lse, wlse, lse_off)
    within("out", out, want, off)
    g = torch.ops.shaobo_fa3.attn_backward(torch.ones_like(q), q, k, v, out, lse, True, None, 0.0, slopes)
    w = A.backward(torch.ones_like(q), q, k[:, :, -2000:], v[:, :, -2000:], out, lse, True, slopes=slopes)
    within("dq", g[0], *w["dq"])
    within("dk", g[1][:, :, -2000:], *w["dk"])
    within("dv", g[2][:, :, -2000:], *w["dv"])


# Backwards cut in every way: whole and halved jobs, parts over the heads and
# over the query tiles, the parts' masks and last tiles.
CUTS = [
    dict(B=1, Hq=8, Hkv=1, Sq=700, D=128), dict(B=1, Hq=6, Hkv=1, Sq=333, D=64, docs=70.0, dtype=HF),
    dict(B=1, Hq=3, Hkv=1, Sq=500, D=128, softcap=20.0, prefix=[100]), dict(B=1, Hq=1, Hkv=1, Sq=1500, D=64),
    dict(B=1, Hq=5, Hkv=5, Sq=800, D=128, causal=False, slopes=1), dict(B=8, Hq=8, Hkv=8, Sq=290, D=128),
    dict(B=8, Hq=16, Hkv=8, Sq=200, D=64, dtype=HF, softcap=200.0), dict(B=8, Hq=32, Hkv=8, Sq=130, D=128, bshd=True),
    dict(B=2, Hq=16, Hkv=2, Sq=100, Sk=900, D=96), dict(B=2, Hq=4, Hkv=2, Sq=900, Sk=70, D=128, causal=False),
    dict(B=1, Hq=12, Hkv=2, Sq=260, D=128, kv=[100]), dict(B=12, Hq=24, Hkv=12, Sq=140, D=128, docs=50.0, slopes=2),
]


@pytest.mark.parametrize("case", CUTS, ids=lambda c: "-".join(
    f"{k}{str(v).replace('torch.', '')}" for k, v in c.items()))
def test_backward_cuts(T, case):
    print("[case]", case, flush=True)
    run_both(*make(case))


@pytest.mark.parametrize("Sq,Sk,causal", [(0, 5, True), (5, 0, True), (0, 0, False), (7, 0, False)])
def test_no_queries_or_no_keys(T, Sq, Sk, causal):
    print("[case] empty", Sq, Sk, flush=True)
    q, k, v, do, o = make(dict(Sq=Sq, Sk=Sk, causal=causal))
    for docs in (False, True):
        if docs:
            o["documents"] = torch.zeros(2, Sq, dtype=torch.int32, device="cuda")
            o["documents_k"] = torch.zeros(2, Sk, dtype=torch.int32, device="cuda")
        out, lse = torch.ops.shaobo_fa3.attn_forward(q, k, v, *op_args(o))
        g = torch.ops.shaobo_fa3.attn_backward(do, q, k, v, out, lse, *op_args(o))
        torch.cuda.synchronize()
        assert out.shape == q.shape and (out == 0).all() and (lse == -math.inf).all()
        assert [x.shape for x in g] == [q.shape, k.shape, v.shape, lse.shape]
        assert all((x == 0).all() for x in g)


def test_empty_batch(T):
    q, k, v, do, o = make(dict(B=0))
    out, lse = torch.ops.shaobo_fa3.attn_forward(q, k, v, True)
    g = torch.ops.shaobo_fa3.attn_backward(do, q, k, v, out, lse, True)
    assert out.shape == q.shape and [x.shape for x in g] == [q.shape, k.shape, v.shape, lse.shape]


JUNK = (math.nan, math.inf, -math.inf)


@pytest.mark.parametrize("D,dtype", [(64, HF), (128, BF)])
@pytest.mark.parametrize("extra", [{}, dict(softcap=10.0), dict(slopes=1)])
def test_masked_places_may_hold_anything(T, D, dtype, extra):
    """Keys behind kv_lens, padding keys and rows, and rows that see nothing
    hold NaN and infinities: same outputs as with zeros there."""
    print("[case] junk", D, dtype, extra, flush=True)
    q, k, v, do, o = make(dict(Sq=150, Sk=200, kv=[130, 200], D=D, dtype=dtype, Hq=4, docs=40.0,
                               causal=False, **extra))
    o["documents"][0, 3:9] = -7
    o["documents"][1, 60:70] = 99999  # (a document without keys)
    o["documents_k"][0, 20:30] = -2147483648
    clean = run_both(q, k, v, do, o)
    gen = torch.Generator(device="cuda").manual_seed(8)

    def spoil(x, rows):  # rows: [B, S] truth values
        junk = torch.tensor(JUNK, device="cuda", dtype=x.dtype)[
            torch.randint(0, 3, x.shape, generator=gen, device="cuda")]
        return torch.where(rows[:, None, :, None], junk, x)

    seen = torch.stack([A.visible(b, 150, 200, False, o["documents"], o["documents_k"], None,
                                  o["kv_lens"], "cuda")[0] for b in range(2)])
    rows = ~seen.any(2)
    assert rows.any() and not rows.all()
    in_use = torch.arange(200, device="cuda")[None] < o["kv_lens"][:, None]
    keys = ~in_use | (o["documents_k"] < 0)
    got_out, got_lse = torch.ops.shaobo_fa3.attn_forward(
        spoil(q, rows), spoil(k, keys), spoil(v, keys), *op_args(o))
    torch.cuda.synchronize()
    assert torch.equal(got_out, clean[0]) and torch.equal(got_lse, clean[1])
    got = torch.ops.shaobo_fa3.attn_backward(
        spoil(do, rows), spoil(q, rows), spoil(k, keys), spoil(v, keys), got_out, got_lse,
        *op_args(o))
    torch.cuda.synchronize()
    for x, n in zip(got, ("dq", "dk", "dv", "delta")):
        assert torch.equal(x, clean[2][n]), n


def test_causal_rows_without_keys_may_hold_anything(T):
    """More queries than keys: the first rows see nothing."""
    q, k, v, do, o = make(dict(Sq=100, Sk=30, D=128))
    out, lse, grads = run_both(q, k, v, do, o)
    assert (lse[:, :, :70] == -math.inf).all() and (out[:, :, :70] == 0).all()
    q2, do2 = q.clone(), do.clone()
    q2[:, :, :70], do2[:, :, :70] = math.nan, math.inf
    out2, lse2 = torch.ops.shaobo_fa3.attn_forward(q2, k, v, *op_args(o))
    got = torch.ops.shaobo_fa3.attn_backward(do2, q2, k, v, out2, lse2, *op_args(o))
    torch.cuda.synchronize()
    assert torch.equal(out2, out) and torch.equal(lse2, lse)
    for x, n in zip(got, ("dq", "dk", "dv", "delta")):
        assert torch.equal(x, grads[n]), n


@pytest.mark.parametrize("extra", [{}, dict(softcap=10.0), dict(slopes=1), dict(causal=False),
                                   dict(docs=40.0)], ids=lambda e: "-".join(e) or "causal")
@pytest.mark.parametrize("Sq,Sk", [(1, 1), (1, 70), (1, 3000), (150, 150), (40, 3000), (600, 600)])
def test_visible_nan_shows(T, Sq, Sk, extra):
    """A row whose Q is NaN, or that sees a key that is, has NaN for output and
    log-sum-exp, never the zeros of a row that sees nothing; rows that see
    nothing stay zeros."""
    print("[case] visible NaN", Sq, Sk, extra, flush=True)
    q, k, v, do, o = make(dict(Sq=Sq, Sk=Sk, D=128, Hq=4, **extra))
    docs = o.get("documents")
    if docs is not None and Sq > 2:
        docs[0, Sq - 2] = 99999  # (a document without keys)
    see = A.visible(0, Sq, Sk, o["causal"], docs, o.get("documents_k"), None, None, "cuda")[0]
    q2 = q.clone()
    q2[0, 1] = math.nan
    out, lse = torch.ops.shaobo_fa3.attn_forward(q2, k, v, *op_args(o))
    rows = see.any(1)
    assert torch.isnan(out[0, 1][rows]).all() and torch.isnan(lse[0, 1][rows]).all()
    assert (out[0, 1][~rows] == 0).all() and (lse[0, 1][~rows] == -math.inf).all()
    assert torch.isfinite(out[1]).all() and torch.isfinite(out[0, 2:]).all()
    for j in {0, Sk // 2, Sk - 1}:
        k2 = k.clone()
        k2[0, 1, j, 5] = math.nan  # (KV head 1: query heads 2 and 3)
        out, lse = torch.ops.shaobo_fa3.attn_forward(q, k2, v, *op_args(o))
        assert torch.isnan(out[0, 2:][:, see[:, j]]).all(), j
        assert torch.isnan(lse[0, 2:][:, see[:, j]]).all(), j
        assert (out[0, 2:][:, ~rows] == 0).all() and (lse[0, 2:][:, ~rows] == -math.inf).all()
        assert torch.isfinite(out[1]).all() and torch.isfinite(out[0, :2]).all()


def test_strides(T):
    """Heads of one packed tensor, expanded keys, and rows far apart."""
    print("[case] strides", flush=True)
    gen = torch.Generator(device="cuda").manual_seed(2)
    qkv = torch.randn(2, 90, 4 + 2 + 2, 64, generator=gen, device="cuda").to(BF)
    q, k, v = (t.transpose(1, 2) for t in qkv.split([4, 2, 2], 2))
    do = torch.randn(2, 4, 90, 64, generator=gen, device="cuda").to(BF)
    run_both(q, k, v, do, dict(causal=True))
    one = torch.randn(1, 1, 90, 64, generator=gen, device="cuda").to(BF)
    run_both(q, one.expand(2, 2, 90, 64), one.expand(2, 2, 90, 64), do, dict(causal=True))
    wide = torch.randn(2, 4, 90, 3, 64, generator=gen, device="cuda").to(BF)
    run_both(wide[:, :, :, 1], k, wide[:, :2, :, 2], do.transpose(2, 3).contiguous().transpose(2, 3)
             .contiguous(), dict(causal=False))
    # documents and slopes of every batch entry alike, without copies
    docs = (torch.arange(90, device="cuda") // 30).int()[None].expand(2, 90)
    run_both(q, k, v, do, dict(causal=True, documents=docs,
                               slopes=torch.rand(1, 4, device="cuda").expand(2, 4)))


def test_offsets_past_32_bits(T):
    """A cache whose rows lie 2^20 elements apart: its last keys are 4.4e9
    elements (8.8e9 bytes) from its first."""
    print("[case] far rows", flush=True)
    S, D = 4200, 128
    far = torch.empty(S << 20, dtype=BF, device="cuda").view(1, 1, S, 1 << 20)
    k, v = far[..., :D], far[..., D:2 * D]
    gen = torch.Generator(device="cuda").manual_seed(4)
    k.copy_(torch.randn(1, 1, S, D, generator=gen, device="cuda"))
    v.copy_(torch.randn(1, 1, S, D, generator=gen, device="cuda"))
    q = torch.randn(1, 2, 3, D, generator=gen, device="cuda").to(BF)
    for o in (dict(causal=True), dict(causal=False, documents=torch.ones(1, 3, dtype=torch.int32, device="cuda"),
                                      documents_k=(torch.arange(S, device="cuda")[None] % 2).int().contiguous())):
        run_both(q, k, v, torch.randn(1, 2, 3, D, generator=gen, device="cuda").to(BF), o)
    # and queries
    run_both(far[:, :, 4100:, :D], k[:, :, :70], v[:, :, :70],
             torch.randn(1, 1, 100, D, generator=gen, device="cuda").to(BF), dict(causal=False))
    del far, k, v
    torch.cuda.empty_cache()


def test_outputs_stay_inside_their_views(T):
    """The C entries write nothing between or behind the rows they are given."""
    print("[case] guards", flush=True)
    lib = F.load()
    B, Hq, Hkv, S, D = 2, 4, 2, 77, 72
    gen = torch.Generator(device="cuda").manual_seed(7)
    ins = {n: torch.randn(B, S, h, D, generator=gen, device="cuda").to(BF)
           for n, h in (("q", Hq), ("k", Hkv), ("v", Hkv), ("dout", Hq))}
    want, lse = torch.ops.shaobo_fa3.attn_forward(*(ins[n].transpose(1, 2) for n in "qkv"), True)
    grads = torch.ops.shaobo_fa3.attn_backward(ins["dout"].transpose(1, 2),
                                               *(ins[n].transpose(1, 2) for n in "qkv"), want, lse,
                                               True)
    p = F.AttnParams()
    lib.shaobo_fa3_attn_params_init(ctypes.byref(p))
    p.batch, p.seqlen_q, p.seqlen_k, p.num_heads_q, p.num_heads_kv, p.head_dim = B, S, S, Hq, Hkv, D
    p.dtype, p.causal = F.DTYPE_BF16, 1
    bufs = {}

    def put(name, t, h):
        x = getattr(p, name)
        x.data = t.data_ptr()
        x.batch_stride, x.head_stride, x.row_stride = t.stride(0), t.stride(2), t.stride(1)

    for n, h in (("q", Hq), ("k", Hkv), ("v", Hkv), ("dout", Hq)):
        put(n, ins[n], h)
    for n, h in (("out", Hq), ("dq", Hq), ("dk", Hkv), ("dv", Hkv)):
        bufs[n] = torch.full((B, S + 2, h + 1, D + 8), -7.0, dtype=BF, device="cuda")
        put(n, bufs[n][:, 1:S + 1, :h, :D], h)
    rows = torch.full((B * Hq * S + 8,), -7.0, device="cuda")
    d = torch.full((B * Hq * S + 8,), -7.0, device="cuda")
    p.softmax_lse, p.softmax_d = rows.data_ptr(), d.data_ptr()
    n = max(lib.shaobo_fa3_attn_fwd_workspace_bytes(ctypes.byref(p)),
            lib.shaobo_fa3_attn_bwd_workspace_bytes(ctypes.byref(p)))
    ws = torch.full((n + 512,), 0x5A, dtype=torch.uint8, device="cuda")
    p.workspace, p.workspace_bytes = ws.data_ptr(), n
    stream = ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)
    assert lib.shaobo_fa3_attn_fwd(ctypes.byref(p), stream) == F.SUCCESS
    assert lib.shaobo_fa3_attn_bwd(ctypes.byref(p), stream) == F.SUCCESS
    torch.cuda.synchronize()
    for name, h, x in (("out", Hq, want), ("dq", Hq, grads[0]), ("dk", Hkv, grads[1]),
                       ("dv", Hkv, grads[2])):
        got = bufs[name]
        assert torch.equal(got[:, 1:S + 1, :h, :D], x.transpose(1, 2)), name
        got[:, 1:S + 1, :h, :D] = -7.0
        assert (got == -7.0).all(), name
    assert torch.equal(rows[:-8], lse.flatten()) and (rows[-8:] == -7.0).all()
    assert torch.equal(d[:-8], grads[3].flatten()) and (d[-8:] == -7.0).all()
    assert (ws[n:] == 0x5A).all()
    # without softmax_d, on the null stream (out is read: it was wiped above)
    bufs["out"][:, 1:S + 1, :Hq, :D] = want.transpose(1, 2)
    p.softmax_d = None
    assert lib.shaobo_fa3_attn_bwd(ctypes.byref(p), None) == F.SUCCESS
    torch.cuda.synchronize()
    assert torch.equal(bufs["dk"][:, 1:S + 1, :Hkv, :D], grads[1].transpose(1, 2))


def test_results_are_reproducible(T):
    for case in (dict(Sq=700, Hq=8, Hkv=2, D=128, docs=150.0, B=1), dict(Sq=1, Sk=3000, Hq=8, Hkv=2, softcap=9.0)):
        q, k, v, do, o = make(case)
        a = torch.ops.shaobo_fa3.attn_forward(q, k, v, *op_args(o))
        b = torch.ops.shaobo_fa3.attn_forward(q, k, v, *op_args(o))
        g = torch.ops.shaobo_fa3.attn_backward(do, q, k, v, *a, *op_args(o))
        h = torch.ops.shaobo_fa3.attn_backward(do, q, k, v, *a, *op_args(o))
        assert all(torch.equal(x, y) for x, y in zip(a + g, b + h))


def test_gradients_against_differences(T):
    """The kernels' gradients along random directions against central
    differences of the fp64 forward, within the summed bounds of their
    elements (and 1e-6 for the differences' third order)."""
    q, k, v, do, o = make(dict(Sq=60, Hq=4, D=64, dtype=HF, softcap=3.0, slopes=1, prefix=[20, 0],
                               docs=25.0, std=2.0))
    out, lse = torch.ops.shaobo_fa3.attn_forward(q, k, v, *op_args(o))
    grads = torch.ops.shaobo_fa3.attn_backward(do, q, k, v, out, lse, *op_args(o))
    exact, exact_lse, out_off, _ = A.forward(q, k, v, **oracle_options(o))
    bounds = A.backward(do, q, k, v, out, lse, **oracle_options(o))
    # delta comes from the rounded out: off by sum |dO| out_off
    ddelta = (do.double().abs() * out_off).sum(-1)
    gen = torch.Generator(device="cuda").manual_seed(9)
    for i, (n, g) in enumerate(zip(("dq", "dk", "dv"), grads)):
        d = torch.randn(g.shape, generator=gen, device="cuda").double()
        ends = []
        for step in (1e-4, -1e-4):
            x = [q.double(), k.double(), v.double()]
            x[i] = x[i] + step * d
            ends.append(float((A.forward(*x, **oracle_options(o))[0] * do.double()).sum()))
        off = float((bounds[n][1] * d.abs()).sum())
        # sum_j p_ij = 1: a delta off by x moves ds_ij by p_ij x
        far = {"dq": k, "dk": q}.get(n)
        if far is not None:
            off += float(ddelta.sum() * far.double().abs().amax() * d.abs().amax() * 64 ** 0.5)
        assert abs((ends[0] - ends[1]) / 2e-4 - float((g.double() * d).sum())) <= off + 1e-3, n


# ---------------------------------------------------------------------------
ROTARY = [
    dict(S=1), dict(S=7, axes=3, dtype=HF), dict(S=33, D=64, P=16, axes=2, interleaved=True),
    dict(S=100, D=72, P=32, dtype=torch.float32), dict(S=100, D=80, P=40, interleaved=True, dtype=torch.float32),
    dict(S=64, H=(3, 1), B=3, bshd=True, axes=4), dict(S=19, D=512, P=256), dict(S=5, D=16, P=8),
    dict(S=50, positions=torch.int64, start=3_000_000_000), dict(S=50, positions=torch.float32, axes=2),
    dict(S=50, H=(5,), interleaved=True), dict(S=1100, B=1, bshd=True), dict(S=4100, B=2, H=(2, 1), D=64, P=32),
    dict(S=4100, B=2, H=(2, 1), D=64, P=24, bshd=True, axes=3), dict(S=50, start=-40), dict(S=0),
]


def rotary_inputs(c):
    c = dict(dict(B=2, H=(4, 2), D=128, P=64, axes=1, dtype=BF, bshd=False, interleaved=False,
                  positions=torch.int32, start=0), **c)
    gen = torch.Generator(device="cuda").manual_seed(11)
    xs = [randn(gen, c["B"], h, c["S"], c["D"], c["dtype"], c["bshd"]) for h in c["H"]]
    pos = torch.randint(0, 5000, (c["axes"], c["B"], c["S"]), generator=gen, device="cuda") + c["start"]
    pos = pos.float() + 0.25 if c["positions"] == torch.float32 else pos.to(c["positions"])
    freqs = 10000.0 ** (-torch.rand(c["axes"], c["P"], generator=gen, device="cuda"))
    return xs, pos, freqs, c["interleaved"]


@pytest.mark.parametrize("case", ROTARY, ids=str)
def test_rotary_against_fp64(T, case):
    print("[case] rotary", case, flush=True)
    xs, pos, freqs, inter = rotary_inputs(case)
    for inverse in (False, True):
        ys = torch.ops.shaobo_fa3.rotary(xs, pos, freqs, inter, inverse)
        torch.cuda.synchronize()
        assert len(ys) == len(xs)
        for x, y in zip(xs, ys):
            assert y.dtype == x.dtype and y.shape == x.shape
            within("rotary", y, *A.rotary(x, pos, freqs, inter, inverse))


def test_rotary_strides_and_in_place(T):
    gen = torch.Generator(device="cuda").manual_seed(12)
    qkv = torch.randn(2, 40, 6, 64, generator=gen, device="cuda").to(BF)
    q, k = qkv[:, :, :4].transpose(1, 2), qkv[:, :, 4:5].transpose(1, 2)
    pos = torch.arange(40, device="cuda").expand(3, 2, 40)  # (strides 0, 0, 1)
    freqs = T.rotary_freqs([8, 12, 12], device="cuda")
    ys = torch.ops.shaobo_fa3.rotary([q, k], pos, freqs)
    torch.cuda.synchronize()
    for x, y in zip((q, k), ys):
        within("rotary", y, *A.rotary(x, pos, freqs, False))
    # three axes that agree turn as one does
    one = torch.ops.shaobo_fa3.rotary([q], pos[:1], T.rotary_freqs([32], device="cuda"))[0]
    assert torch.equal(one, ys[0])
    # the C entry on its own input
    lib, p = F.load(), F.RotaryParams()
    lib.shaobo_fa3_rotary_params_init(ctypes.byref(p))
    p.batch, p.seqlen, p.head_dim, p.pairs, p.axes, p.tensors = 2, 40, 64, 32, 3, 1
    p.dtype, p.position_type = F.DTYPE_BF16, F.POSITIONS_INT64
    p.positions, p.freqs = pos.data_ptr(), freqs.data_ptr()
    p.position_axis_stride, p.position_batch_stride, p.position_row_stride = pos.stride()
    p.heads[0] = 4
    rest = qkv[:, :, 4:].clone()
    for t in (p.in_[0], p.out[0]):
        t.data, t.batch_stride, t.head_stride, t.row_stride = (q.data_ptr(), *q.stride()[:3])
    assert lib.shaobo_fa3_rotary(ctypes.byref(p), torch.cuda.current_stream().cuda_stream) == F.SUCCESS
    torch.cuda.synchronize()
    assert torch.equal(q, ys[0]) and torch.equal(qkv[:, :, 4:], rest)


# ---------------------------------------------------------------------------
def layer(T, q, k, v, pos, freqs, **options):
    q, k = T.rotary(q, k, positions=pos, freqs=freqs)
    return T.score_attention(q, k, v, **options)


def layer_inputs(S=200, seed=21, dtype=HF):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    q = torch.randn(2, S, 4, 64, generator=gen, device="cuda").to(dtype).transpose(1, 2)
    k, v = (torch.randn(2, S, 2, 64, generator=gen, device="cuda").to(dtype).transpose(1, 2)
            for _ in range(2))
    i = torch.arange(S, device="cuda", dtype=torch.int32)
    pos = torch.stack((i // 16, i // 4 % 4, i % 4))[:, None].expand(3, 2, S)
    docs = (i // 70)[None].expand(2, S).contiguous()
    docs[1, 150:] = -1
    return q, k, v, pos, T_freqs(), docs


def T_freqs():
    import shaobo_fa3_torch
    return shaobo_fa3_torch.rotary_freqs([8, 12, 12], device="cuda")


def test_attention_layer_and_its_gradient(T):
    """Rotary positions, attention, loss and back: against the same layer in
    fp64, the gradients within 8 u of each tensor's norm.  (Seven roundings lie
    between q and dq: the rotated q and k, P, out, dS, dq, the rotation back;
    each is off by u / sqrt(3) of a norm on average, 8 u covers their sum in
    the worst direction of all.)"""
    q, k, v, pos, freqs, docs = layer_inputs()
    leaves = [t.detach().clone(memory_format=torch.preserve_format).requires_grad_() for t in (q, k, v)]
    opts = dict(causal=True, softcap=8.0, documents=docs)
    out = layer(T, *leaves, pos, freqs, **opts)
    w = torch.randn(out.shape, device="cuda", generator=torch.Generator(device="cuda").manual_seed(1))
    grads = torch.autograd.grad((out.float() * w).sum(), leaves)
    ref = [t.detach().double().requires_grad_() for t in leaves]

    def turn(x):
        a = (pos.double()[..., None] * freqs.double()[:, None, None]).sum(0)[:, None]
        lo, hi = x[..., :32], x[..., 32:]
        return torch.cat((lo * a.cos() - hi * a.sin(), hi * a.cos() + lo * a.sin()), -1)

    qr, kr = turn(ref[0]), turn(ref[1]).repeat_interleave(2, 1)
    s = 8.0 * torch.tanh((qr @ kr.transpose(2, 3).contiguous()) / 8.0 / 8.0)
    seen = torch.stack([A.visible(b, 200, 200, True, docs, None, None, None, "cuda")[0]
                        for b in range(2)])[:, None]
    p = torch.exp(s) * seen
    z = p.sum(-1, keepdim=True)
    want = (p / torch.where(z == 0, torch.ones_like(z), z)) @ ref[2].repeat_interleave(2, 1)
    wgrads = torch.autograd.grad((want * w.double()).sum(), ref)
    u = torch.finfo(HF).eps / 2
    for n, x, y in (("out", out.detach(), want.detach()), *zip(("dq", "dk", "dv"), grads, wgrads)):
        assert x.dtype == HF and x.shape == y.shape
        assert float((x.double() - y).norm()) <= 8 * u * float(y.norm()), n


def test_gradients_of_expanded_and_odd_layouts(T):
    """Inputs expanded over heads, a gradient that arrives expanded, outputs
    used in part, tensors that need no gradient."""
    q, k, v, pos, freqs, docs = layer_inputs(dtype=BF)
    one = k[:, :1].detach().clone().requires_grad_()
    qq = q.detach().clone().requires_grad_()
    out, lse = T.score_attention(qq, one.expand(2, 2, 200, 64), v, return_lse=True)
    assert not lse.requires_grad
    out.sum().backward()  # (dout: one number, expanded)
    full = k[:, :1].expand(2, 2, 200, 64).contiguous().detach().requires_grad_()
    q2 = q.detach().clone().requires_grad_()
    T.score_attention(q2, full, v).backward(torch.ones_like(out))
    assert torch.equal(qq.grad, q2.grad)
    assert torch.equal(one.grad, full.grad.sum(1, keepdim=True))
    x = T.rotary(qq, positions=pos, freqs=freqs)
    (g,) = torch.autograd.grad(x[..., 0].sum(), qq)
    assert g.shape == qq.shape and torch.isfinite(g.float()).all()
    with torch.no_grad():
        assert not T.score_attention(qq, one.expand(2, 2, 200, 64), v).requires_grad


def test_serving_equals_the_prompt(T):
    """Token by token over a cache with free rows behind the last one: the
    outputs of the whole prompt's rows, within both bounds; the cache's free
    rows hold NaN and stay as they are."""
    S, D, B = 70, 128, 3
    gen = torch.Generator(device="cuda").manual_seed(31)
    q = randn(gen, B, 8, S, D, BF)
    k, v = randn(gen, B, 2, S, D, BF), randn(gen, B, 2, S, D, BF)
    slopes = torch.rand(8, generator=gen, device="cuda")
    whole, lse, off, lse_off = A.forward(q, k, v, True, softcap=20.0, slopes=slopes)
    kc, vc = (torch.full((B, 2, 256, D), math.nan, dtype=BF, device="cuda") for _ in range(2))
    for t in (0, 1, 31, 63, 64, 69):
        n = t + 1
        kc[:, :, :n], vc[:, :, :n] = k[:, :, :n], v[:, :, :n]
        o, l = T.score_attention(q[:, :, t:n], kc, vc, softcap=20.0, slopes=slopes,
                                 kv_lens=i32([n] * B), return_lse=True)
        within("out", o, whole[:, :, t:n], off[:, :, t:n])
        within("lse", l, lse[:, :, t:n], lse_off[:, :, t:n])
        assert torch.isnan(kc[:, :, n:]).all()


def test_other_stream(T):
    """Inputs made and used on a stream of their own."""
    want = run_both(*make(dict(Sq=300, Hq=8, Hkv=2, D=128, docs=60.0)))
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        q, k, v, do, o = make(dict(Sq=300, Hq=8, Hkv=2, D=128, docs=60.0))
        out, lse = torch.ops.shaobo_fa3.attn_forward(q, k, v, *op_args(o))
        g = torch.ops.shaobo_fa3.attn_backward(do, q, k, v, out, lse, *op_args(o))
    s.synchronize()
    assert torch.equal(out, want[0]) and all(torch.equal(x, want[2][n]) for x, n in zip(g, ("dq", "dk", "dv", "delta")))


def test_two_streams_at_once(T):
    cases = [make(dict(Sq=500, Hq=8, Hkv=2, D=128, docs=90.0), seed) for seed in (1, 2)]
    want = [torch.ops.shaobo_fa3.attn_forward(q, k, v, *op_args(o)) for q, k, v, _, o in cases]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = [None, None]
    for _ in range(5):
        for i, (q, k, v, _, o) in enumerate(cases):
            with torch.cuda.stream(streams[i]):
                got[i] = torch.ops.shaobo_fa3.attn_forward(q, k, v, *op_args(o))
    torch.cuda.synchronize()
    for a, b in zip(want, got):
        assert all(torch.equal(x, y) for x, y in zip(a, b))


@pytest.mark.parametrize("case", [
    dict(B=1, Hq=8, Hkv=2, Sq=1, Sk=3000, D=128, softcap=20.0, kv=[2000]),
    dict(Sq=260, Hq=4, Hkv=2, D=128, docs=60.0), dict(Sq=130, slopes=1)],
    ids=["split", "documents", "bias"])
def test_graph_capture(T, case):
    """Captured once, replayed with other inputs, with eager work between."""
    print("[case] graph", case, flush=True)
    q, k, v, do, o = make(case)
    D = q.shape[3]
    pos = torch.arange(q.shape[2], device="cuda", dtype=torch.int32).expand(1, q.shape[0], -1).contiguous()
    freqs = T.rotary_freqs([D // 2], device="cuda")

    def step():
        (qr,) = torch.ops.shaobo_fa3.rotary([q], pos, freqs)
        out, lse = torch.ops.shaobo_fa3.attn_forward(qr, k, v, *op_args(o))
        return (qr, out, lse, *torch.ops.shaobo_fa3.attn_backward(do, qr, k, v, out, lse, *op_args(o)))

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step()
    torch.cuda.current_stream().wait_stream(s)
    graph, second = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    with torch.cuda.graph(second):
        other = step()
    for seed in (4, 5, 6, 7):
        q2, k2, v2, do2, o2 = make(case, seed)
        for a, b in ((q, q2), (k, k2), (v, v2), (do, do2)):
            a.copy_(b)
        for n in ("documents", "kv_lens"):
            if n in o:
                o[n].copy_(o2[n] if n == "documents" else o[n] - 111)
        pos += 1000
        want = [x.clone() for x in step()]
        torch.cuda.synchronize()
        graph.replay()
        second.replay()
        torch.cuda.synchronize()
        for x, y, z in zip(want, got, other):
            assert torch.equal(x, y) and torch.equal(x, z)


def test_training_step_captured(T):
    """Rotary, attention and their gradient through autograd in one graph,
    replayed between eager steps."""
    q, k, v, do, o = make(dict(Sq=130, Hq=4, Hkv=2, D=128, docs=60.0, softcap=20.0))
    q, k, v = (x.detach().requires_grad_() for x in (q, k, v))
    pos = torch.arange(130, device="cuda").expand(1, 2, 130)
    freqs = T.rotary_freqs([64], device="cuda")

    def step():
        qr, kr = T.rotary(q, k, positions=pos, freqs=freqs)
        out = T.score_attention(qr, kr, v, causal=True, softcap=20.0, documents=o["documents"])
        return torch.autograd.grad(out, (q, k, v), do)

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        for _ in range(2):
            step()
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for seed in (4, 5, 6):
        with torch.no_grad():
            for a, b in zip((q, k, v, do), make(dict(Sq=130, Hq=4, Hkv=2, D=128), seed)):
                a.copy_(b)
        want = [x.clone() for x in step()]
        graph.replay()
        torch.cuda.synchronize()
        for x, y in zip(want, got):
            assert torch.equal(x, y)


def test_operators_under_torch_library_checks(T):
    """Schemas and fake implementations agree with what the operators do."""
    q, k, v, do, o = make(dict(Sq=70, Hq=4, Hkv=2, docs=30.0, bshd=True))
    out, lse = torch.ops.shaobo_fa3.attn_forward(q, k, v, *op_args(o))
    pos = torch.arange(70, device="cuda").expand(1, 2, 70)
    freqs = T.rotary_freqs([32], device="cuda")
    checks = ("test_schema", "test_faketensor")
    for op, args in (("attn_forward", (q, k, v, *op_args(o))),
                     ("attn_backward", (do, q, k, v, out, lse, *op_args(o))),
                     ("rotary", ([q, k], pos, freqs))):
        torch.library.opcheck(getattr(torch.ops.shaobo_fa3, op).default, args, test_utils=checks)


# ---------------------------------------------------------------------------
def refused(match, fn, error=ValueError):
    with pytest.raises(error, match=match):
        fn()


def test_attention_refusals(T):
    q, k, v, do, o = make(dict(Sq=32))
    f = torch.ops.shaobo_fa3.attn_forward
    refused("must be \\[batch", lambda: f(q[0], k, v, True))
    refused("does not match", lambda: f(q, k[:, :, :5], v, True))
    refused("does not match", lambda: f(q, k[:1], v[:1], True))
    refused("does not match", lambda: f(q[:, :1], k, v, True))
    refused("one type", lambda: f(q, k.half(), v, True))
    refused("one type", lambda: f(q.float(), k.float(), v.float(), True))
    refused("same GPU", lambda: f(q, k.cpu(), v, True))
    refused("multiple of 8", lambda: f(q[..., :20], k[..., :20], v[..., :20], True))
    refused("contiguous", lambda: f(q.transpose(2, 3).contiguous().transpose(2, 3), k, v, True))
    odd = torch.zeros(2, 2, 32, 68, dtype=BF, device="cuda")
    refused("16 bytes", lambda: f(odd[..., :64], k, v, True))
    refused("aligned", lambda: f(q, torch.zeros(2 * 2 * 32 * 64 + 4, dtype=BF, device="cuda")[4:].view(2, 2, 32, 64), v, True))
    refused("finite", lambda: f(q, k, v, True, math.nan))
    refused("softcap", lambda: f(q, k, v, True, None, -1.0))
    refused("softcap", lambda: f(q, k, v, True, None, math.inf))
    refused("softcap", lambda: f(q, k, v, True, None, 1e-50))
    refused("slopes", lambda: f(q, k, v, True, None, 0.0, torch.ones(3, device="cuda")))
    refused("slopes", lambda: f(q, k, v, True, None, 0.0, torch.ones(2, device="cuda").half()))
    refused("slopes", lambda: f(q, k, v, True, None, 0.0, torch.ones(2)))
    ids = torch.zeros(2, 32, dtype=torch.int32, device="cuda")
    refused("int32", lambda: f(q, k, v, True, documents=ids.long()))
    refused("documents", lambda: f(q, k, v, True, documents=ids[:, :31]))
    refused("needs documents", lambda: f(q, k, v, True, documents_k=ids))
    refused("documents_k must be given", lambda: f(q, k[:, :, :20], v[:, :, :20], True, documents=ids))
    refused("along the sequence", lambda: f(q, k, v, True, documents=ids.t().contiguous().t()))
    refused("needs causal", lambda: f(q, k, v, False, prefix_lens=i32([1, 2])))
    refused("prefix_lens", lambda: f(q, k, v, True, prefix_lens=i32([1])))
    refused("kv_lens", lambda: f(q, k, v, True, kv_lens=i32([1, 2]).cpu()))
    out, lse = f(q, k, v, True)
    g = torch.ops.shaobo_fa3.attn_backward
    refused("like q", lambda: g(do[:, :1], q, k, v, out, lse, True))
    refused("like q", lambda: g(do, q, k, v, out.half(), lse, True))
    refused("softmax_lse", lambda: g(do, q, k, v, out, lse.double(), True))
    refused("softmax_lse", lambda: g(do, q, k, v, out, lse[:, :, :31], True))
    refused("contiguous", lambda: g(do[..., :1].expand(2, 2, 32, 64), q, k, v, out, lse, True))


def test_rotary_refusals(T):
    x = torch.zeros(2, 3, 8, 64, dtype=BF, device="cuda")
    pos = torch.zeros(1, 2, 8, dtype=torch.int32, device="cuda")
    fr = torch.zeros(1, 32, device="cuda")
    f = torch.ops.shaobo_fa3.rotary
    refused("one or two", lambda: f([x, x, x], pos, fr))
    refused("\\[batch", lambda: f([x[0]], pos, fr))
    refused("heads only", lambda: f([x, x[:, :, :4]], pos, fr))
    refused("heads only", lambda: f([x, x.half()], pos, fr))
    refused("fp16, bf16 or fp32", lambda: f([x.double()], pos, fr))
    refused("positions", lambda: f([x], pos[:, :, :7], fr))
    refused("positions", lambda: f([x], pos.short(), fr))
    refused("positions", lambda: f([x], pos.cpu(), fr))
    refused("freqs", lambda: f([x], pos, fr.double()))
    refused("pairs", lambda: f([x], pos, fr[:, :12].contiguous()))
    refused("pairs", lambda: f([x], pos, torch.zeros(1, 40, device="cuda")))
    refused("axes", lambda: f([x], pos.expand(5, 2, 8), fr.expand(5, 32).contiguous()))
    refused("head_dim", lambda: f([torch.zeros(2, 3, 8, 60, dtype=BF, device="cuda")], pos, fr))
    refused("16 bytes", lambda: f([torch.zeros(2, 3, 8, 68, dtype=BF, device="cuda")[..., :64]], pos, fr))
