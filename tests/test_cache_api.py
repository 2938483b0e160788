"""The paged cache without a GPU: parameter checks and workspace sizes of the C
entries, refusals that return before any HIP call, the operators' fake
implementations, the kernels' resources, and the oracle of the GPU tests."""
import ctypes
import math
import os

import pytest

import attn_oracle as A
import cache_oracle as O
import resource_gate as gate
import shaobo_fa3 as F

torch = pytest.importorskip("torch")

PTR = 1 << 20  # a non-null address; nothing here reads it
PARAMS = {"append": F.CacheAppendParams, "attn": F.CacheAttnParams, "select": F.CacheSelectParams,
          "read": F.CacheReadParams}


@pytest.fixture(scope="module")
def lib():
    return F.load()


def make(lib, what, **kw):
    """Plausible parameters, every pointer set (to memory nothing may touch)."""
    p = PARAMS[what]()
    getattr(lib, f"shaobo_fa3_cache_{what}_params_init")(ctypes.byref(p))
    c = p.cache
    c.batch, c.num_heads_kv, c.head_dim, c.pages, c.page_size, c.width = 2, 4, 128, 40, 64, 16
    for t in (c.k, c.v):
        t.data, t.page_stride, t.head_stride, t.row_stride = PTR, 4 * 64 * 128, 64 * 128, 128
    c.page_table, c.page_table_stride, c.kv_lens = PTR, 16, PTR
    p.seqlen = 3
    for n in ("q", "k", "v", "out", "q_out"):
        if hasattr(p, n):
            t = getattr(p, n)
            t.data, t.batch_stride, t.head_stride, t.row_stride = PTR, 4096, 512, 128
    if hasattr(p, "num_heads_q"):
        p.num_heads_q = 8
    if what == "select":
        p.count, p.selected, c.bounds = 4, PTR, PTR
    if what == "attn":
        p.softmax_lse = PTR
    if hasattr(p, "workspace"):
        p.workspace, p.workspace_bytes = PTR, 1 << 40
    for n, x in kw.items():
        obj = p
        *path, last = n.split("__")
        for part in path:
            obj = getattr(obj, part)
        setattr(obj, last, x)
    return p


def call(lib, what, p):
    return getattr(lib, f"shaobo_fa3_cache_{what}")(ctypes.byref(p), None)


def test_struct_sizes(lib):
    for what, cls in PARAMS.items():
        p = cls()
        ctypes.memset(ctypes.byref(p), 0x5A, ctypes.sizeof(p))
        init = getattr(lib, f"shaobo_fa3_cache_{what}_params_init")
        init(ctypes.byref(p))
        assert p.struct_size == ctypes.sizeof(cls)
        assert p.seqlen == 0 and p.cache.bits == 16 and p.cache.page_size == 64 and p.cache.k.data is None
        init(None)  # tolerated
        assert getattr(lib, f"shaobo_fa3_cache_{what}")(None, None) == F.INVALID_VALUE


CACHE = [
    ({"struct_size": 8}, F.INVALID_VALUE), ({"cache__batch": -1}, F.INVALID_VALUE), ({"seqlen": -1}, F.INVALID_VALUE),
    ({"cache__num_heads_kv": 0}, F.INVALID_VALUE), ({"cache__head_dim": 0}, F.INVALID_VALUE),
    ({"cache__pages": -1}, F.INVALID_VALUE), ({"cache__width": -1}, F.INVALID_VALUE),
    ({"cache__bits": 8}, F.INVALID_VALUE), ({"cache__page_size": 0}, F.INVALID_VALUE),
    ({"cache__dtype": F.DTYPE_FP8}, F.UNSUPPORTED), ({"cache__dtype": F.DTYPE_FP32}, F.UNSUPPORTED),
    ({"cache__head_dim": 136}, F.UNSUPPORTED), ({"cache__head_dim": 100}, F.UNSUPPORTED),
    ({"cache__bits": 4, "cache__head_dim": 96}, F.UNSUPPORTED),
    ({"cache__page_size": 16}, F.UNSUPPORTED), ({"cache__page_size": 48}, F.UNSUPPORTED),
    ({"cache__page_size": 2048}, F.UNSUPPORTED), ({"cache__width": 1 << 25}, F.UNSUPPORTED),
    ({"cache__batch": 1 << 23, "seqlen": 2}, F.UNSUPPORTED), ({"seqlen": 1 << 24}, F.UNSUPPORTED),
]
STRIDES = [
    ({"cache__k__page_stride": 4}, F.UNSUPPORTED), ({"cache__v__head_stride": 12}, F.UNSUPPORTED),
    ({"cache__k__row_stride": 130}, F.UNSUPPORTED),
    ({"cache__bits": 4, "cache__v__page_stride": 24}, F.UNSUPPORTED),
]
POINTERS = [{"cache__page_table": None}, {"cache__kv_lens": None}]
PAGES = [{"cache__k__data": None}, {"cache__v__data": PTR + 8}]


@pytest.mark.parametrize("what", list(PARAMS))
def test_the_cache_is_checked(lib, what):
    for change, status in CACHE + (STRIDES if what != "select" else []):
        assert call(lib, what, make(lib, what, **change)) == status, change
    for change in POINTERS + (PAGES if what != "select" else [{"cache__bounds": None}, {"cache__bounds": PTR + 8}]):
        assert call(lib, what, make(lib, what, **change)) == F.INVALID_VALUE, change


@pytest.mark.parametrize("what", list(PARAMS))
def test_empty_calls_need_no_memory(lib, what):
    for change in ({"cache__batch": 0}, {"seqlen": 0}):
        p = make(lib, what, **change)
        p.cache.k.data = p.cache.v.data = p.cache.page_table = p.cache.kv_lens = None
        assert call(lib, what, p) == F.SUCCESS


@pytest.mark.parametrize("what,change,status", [
    ("attn", {"num_heads_q": 0}, F.INVALID_VALUE), ("attn", {"num_heads_q": 6}, F.INVALID_VALUE),
    ("attn", {"num_heads_q": 1 << 17}, F.UNSUPPORTED), ("attn", {"causal": 2}, F.INVALID_VALUE),
    ("attn", {"softmax_scale_is_set": 1, "softmax_scale": math.nan}, F.INVALID_VALUE),
    ("attn", {"softmax_scale_is_set": 3}, F.INVALID_VALUE), ("attn", {"softcap": -1.0}, F.INVALID_VALUE),
    ("attn", {"softcap": math.inf}, F.INVALID_VALUE), ("attn", {"prefix_lens": PTR}, F.INVALID_VALUE),
    ("attn", {"count": -1}, F.INVALID_VALUE), ("attn", {"selected": PTR}, F.INVALID_VALUE),
    ("attn", {"selected": PTR, "count": 1 << 21}, F.UNSUPPORTED), ("attn", {"q__row_stride": 12}, F.UNSUPPORTED),
    ("attn", {"out__head_stride": 4}, F.UNSUPPORTED), ("attn", {"q__data": None}, F.INVALID_VALUE),
    ("attn", {"out__data": PTR + 2}, F.INVALID_VALUE), ("attn", {"softmax_lse": None}, F.INVALID_VALUE),
    ("attn", {"workspace": None}, F.INVALID_VALUE), ("attn", {"workspace_bytes": 16}, F.INVALID_VALUE),
    ("attn", {"workspace": PTR + 64}, F.INVALID_VALUE),
    ("select", {"num_heads_q": 6}, F.INVALID_VALUE), ("select", {"count": 0}, F.INVALID_VALUE),
    ("select", {"count": 1 << 21}, F.UNSUPPORTED), ("select", {"q__head_stride": 4}, F.UNSUPPORTED),
    ("select", {"q__data": PTR + 8}, F.INVALID_VALUE), ("select", {"selected": None}, F.INVALID_VALUE),
    ("select", {"workspace": None}, F.INVALID_VALUE), ("select", {"workspace_bytes": 8}, F.INVALID_VALUE),
    ("append", {"num_heads_q": -1}, F.INVALID_VALUE), ("append", {"num_heads_q": 1 << 17}, F.UNSUPPORTED),
    ("append", {"positions": PTR}, F.INVALID_VALUE), ("append", {"freqs": PTR, "pairs": 12}, F.UNSUPPORTED),
    ("append", {"freqs": PTR, "pairs": 72}, F.UNSUPPORTED), ("append", {"freqs": PTR, "pairs": 64, "axes": 0}, F.INVALID_VALUE),
    ("append", {"freqs": PTR, "pairs": 64, "axes": 2}, F.INVALID_VALUE),
    ("append", {"freqs": PTR, "pairs": 64, "axes": 5, "positions": PTR}, F.UNSUPPORTED),
    ("append", {"freqs": PTR, "pairs": 64, "interleaved": 2}, F.INVALID_VALUE),
    ("append", {"freqs": PTR, "pairs": 64, "positions": PTR, "position_type": 7}, F.INVALID_VALUE),
    ("append", {"k__row_stride": 4}, F.UNSUPPORTED), ("append", {"q_out__head_stride": 4}, F.UNSUPPORTED),
    ("append", {"v__data": None}, F.INVALID_VALUE), ("append", {"q__data": None}, F.INVALID_VALUE),
    ("append", {"q_out__data": PTR + 4}, F.INVALID_VALUE), ("append", {"cache__bounds": PTR + 8}, F.INVALID_VALUE),
    ("read", {"k__row_stride": 4}, F.UNSUPPORTED), ("read", {"v__data": None}, F.INVALID_VALUE),
])
def test_calls_are_checked_before_any_launch(lib, what, change, status):
    p = make(lib, what, **change)
    assert call(lib, what, p) == status
    pointers = status == F.INVALID_VALUE and any(n in str(change) for n in ("data", "workspace", "lse", "'selected': None"))
    if what in ("attn", "select") and not pointers:
        assert getattr(lib, f"shaobo_fa3_cache_{what}_validate")(ctypes.byref(p)) == status
        assert getattr(lib, f"shaobo_fa3_cache_{what}_workspace_bytes")(ctypes.byref(p)) == 0


def test_workspaces(lib):
    def need(what, **kw):
        p = make(lib, what, **kw)
        assert getattr(lib, f"shaobo_fa3_cache_{what}_validate")(ctypes.byref(p)) == F.SUCCESS
        return getattr(lib, f"shaobo_fa3_cache_{what}_workspace_bytes")(ctypes.byref(p))

    # a key a page of every token and KV head
    assert need("select") == 2 * 4 * 3 * 16 * 8
    # few rows over long sequences: parts of fp32 outputs and log-sum-exps
    n = need("attn", seqlen=1, cache__width=512)
    assert n % 256 == 0 and n >= 2 * 2 * 8 * (128 + 1) * 4
    # many sequences fill the chip by themselves
    assert need("attn", cache__batch=512, seqlen=1) == 0
    # fewer listed pages, fewer parts
    assert need("attn", seqlen=1, cache__width=512, selected=PTR, count=8) < n


@pytest.mark.parametrize("heads,seqlen,status", [
    (8, 1 << 20, F.UNSUPPORTED), (1, (1 << 23) + 1, F.UNSUPPORTED), (8, (1 << 20) - 1, F.SUCCESS),
    (1, (1 << 23) - 1, F.SUCCESS), (1 << 16, 128, F.UNSUPPORTED), (1 << 16, 127, F.SUCCESS),
])
@pytest.mark.parametrize("width", [0, 1, 64])
def test_selection_of_more_rows_than_a_launch_takes(lib, heads, seqlen, status, width):
    """Picking has a workgroup of 512 threads for every token and KV head, and a launch
    fewer than 2^32 threads: refused at 2^23 rows, before anything is launched."""
    p = make(lib, "select", cache__batch=1, cache__num_heads_kv=heads, num_heads_q=heads, seqlen=seqlen,
             cache__width=width)
    assert lib.shaobo_fa3_cache_select_validate(ctypes.byref(p)) == status
    n = lib.shaobo_fa3_cache_select_workspace_bytes(ctypes.byref(p))
    assert n == (-(-heads * seqlen * width * 8 // 256) * 256 if status == F.SUCCESS else 0)
    if status != F.SUCCESS:
        assert call(lib, "select", p) == status


# ---------------------------------------------------------------------------
@pytest.fixture(scope="module")
def T():
    import shaobo_fa3_torch
    assert shaobo_fa3_torch._ATTN, "lib/_fa3_torch_attn.so is not built"
    return shaobo_fa3_torch


def test_fake_implementations(T):
    from torch._subclasses.fake_tensor import FakeTensorMode
    ops = torch.ops.shaobo_fa3
    with FakeTensorMode():
        q = torch.empty(2, 33, 8, 64, dtype=torch.bfloat16, device="cuda").transpose(1, 2)
        k = torch.empty(2, 4, 33, 64, dtype=torch.bfloat16, device="cuda")
        t = torch.empty(2, 9, dtype=torch.int32, device="cuda")
        for bits, row in ((16, 64), (4, 36)):
            kp, vp, b = T.cache_pages(7, 4, 32, 64, torch.bfloat16, bits=bits, bounds=True)
            assert kp.shape == (7, 4, 32, row) and b.shape == (7, 4, 2, 64)
            assert ops.cache_append(k, k, kp, vp, t, t[:, 0]) == []
            y, = ops.cache_append(k, k, kp, vp, t, t[:, 0], None, q)
            assert y.shape == q.shape and y.stride() == q.stride()
            out, lse = ops.cache_attn(q, kp, vp, t, t[:, 0])
            assert out.shape == q.shape and lse.shape == (2, 8, 33) and lse.dtype == torch.float32
            x, y = ops.cache_read(kp, vp, t, t[:, 0], 50, torch.bfloat16)
            assert x.shape == y.shape == (2, 4, 50, 64)
        sel = ops.cache_select(q, b, t, t[:, 0], 32, 5)
        assert sel.shape == (2, 4, 33, 5) and sel.dtype == torch.int32


def test_appends_are_functionalized(T):
    """A program that appends, with and without queries and bounds, becomes one graph
    that returns what it wrote."""
    from torch._functorch.aot_autograd import aot_export_module
    from torch._subclasses.fake_tensor import FakeTensorMode

    class Step(torch.nn.Module):
        def __init__(self, f):
            super().__init__()
            self.f = f

        def forward(self, *tensors):
            return self.f(*tensors)

    def functions(k, v, kp, vp, t, n, q, b):
        qt = T.cache_append(k, v, kp, vp, page_table=t, kv_lens=n, q=q, bounds=b)
        assert T.cache_append(k, v, kp, vp, page_table=t, kv_lens=n) is None
        return qt, T.cache_attention(qt, kp, vp, page_table=t, kv_lens=n)

    def operators(k, v, kp, vp, t, n, q, b):
        qt, = torch.ops.shaobo_fa3.cache_append(k, v, kp, vp, t, n, None, q, bounds=b)
        assert torch.ops.shaobo_fa3.cache_append(k, v, kp, vp, t, n) == []
        return qt, *torch.ops.shaobo_fa3.cache_attn(qt, kp, vp, t, n)

    for f, outs in ((functions, 2), (operators, 3)):
        with FakeTensorMode(), torch.no_grad():
            k = torch.empty(2, 4, 33, 64, dtype=torch.bfloat16, device="cuda")
            q = torch.empty(2, 33, 8, 64, dtype=torch.bfloat16, device="cuda").transpose(1, 2)
            t = torch.empty(2, 9, dtype=torch.int32, device="cuda")
            kp, vp, b = T.cache_pages(7, 4, 32, 64, torch.bfloat16, bounds=True)
            graph, signature = aot_export_module(Step(f), (k, k, kp, vp, t, t[:, 0], q, b), trace_joint=False)
        assert sorted(signature.user_inputs_to_mutate.values()) == sorted(signature.user_inputs[n] for n in (2, 3, 7))
        assert len(signature.user_outputs) == outs
        assert str(graph.graph).count("cache_append_into") == 2


def test_refusals_without_a_gpu(T):
    q = torch.zeros(1, 1, 4, 64, dtype=torch.bfloat16)
    t = torch.zeros(1, 1, dtype=torch.int32)
    with pytest.raises(NotImplementedError):
        torch.ops.shaobo_fa3.cache_attn(q, q, q, t, t[0])
    with pytest.raises(ValueError, match="no gradient"):
        T.cache_attention(q.requires_grad_(), q, q, page_table=t, kv_lens=t[0])
    with pytest.raises(ValueError, match="no gradient"):
        T.cache_append(q, q, q, q, page_table=t, kv_lens=t[0])
    with pytest.raises(ValueError, match="16 bits or in 4"):
        T.cache_pages(1, 1, 32, 64, bits=8, device="cpu")


def test_no_tensor_of_a_call_loses_its_gradient(T):
    """Whichever tensor requires one, the call is refused (under no_grad it goes on, to
    an operator that has no CPU kernel)."""
    def tensors():
        x = {n: torch.zeros(1, 1, 32, 64, dtype=torch.bfloat16) for n in ("q", "k", "v", "k_pages", "v_pages")}
        x["bounds"] = torch.zeros(1, 1, 2, 64, dtype=torch.bfloat16)
        x["slopes"], x["freqs"], x["positions"] = torch.zeros(1), torch.zeros(1, 8), torch.zeros(1, 1, 32)
        return x

    t = torch.zeros(1, 1, dtype=torch.int32)
    w = dict(page_table=t, kv_lens=t[0])
    calls = {
        T.cache_append: lambda x: T.cache_append(x["k"], x["v"], x["k_pages"], x["v_pages"], q=x["q"], freqs=x["freqs"],
                                                 positions=x["positions"], bounds=x["bounds"], **w),
        T.cache_attention: lambda x: T.cache_attention(x["q"], x["k_pages"], x["v_pages"], slopes=x["slopes"], **w),
        T.cache_select: lambda x: T.cache_select(x["q"], x["bounds"], page_size=32, count=1, **w),
        T.cache_read: lambda x: T.cache_read(x["k_pages"], x["v_pages"], seqlen=1, **w),
    }
    takes = {T.cache_append: "k v k_pages v_pages q freqs positions bounds", T.cache_attention: "q k_pages v_pages slopes",
             T.cache_select: "q bounds", T.cache_read: "k_pages v_pages"}
    for f, call_ in calls.items():
        for name in takes[f].split():
            x = tensors()
            x[name].requires_grad_()
            with pytest.raises(ValueError, match="no gradient"):
                call_(x)
            with torch.no_grad(), pytest.raises(NotImplementedError):
                call_(x)


def test_a_missing_library_is_said(T, monkeypatch):
    monkeypatch.setattr(T, "_ATTN", False)
    q = torch.zeros(1, 1, 4, 64, dtype=torch.bfloat16)
    for f in (lambda: T.cache_attention(q, q, q, page_table=q, kv_lens=q),
              lambda: T.cache_append(q, q, q, q, page_table=q, kv_lens=q),
              lambda: T.cache_select(q, q, page_table=q, kv_lens=q, page_size=32, count=1),
              lambda: T.cache_read(q, q, page_table=q, kv_lens=q, seqlen=1)):
        with pytest.raises(RuntimeError, match="make -C flash-attention3_amd torch"):
            f()


def test_kernels_share_a_cu():
    """As many workgroups of the kernels fit a CU as the plans count on."""
    kernels, bad = gate.check(gate.LIB_PATH)
    assert bad == []
    few = [k for k in kernels if "cache_few_kernel" in k[".name"]]
    tile = [k for k in kernels if "cache_tile_kernel" in k[".name"]]
    assert len(few) == 128 and len(tile) == 64 and os.path.exists(gate.LIB_PATH)
    for k in few:
        # template arguments: D, type, cap, bias, four, 16-row blocks, dealt
        args = k[".name"].split("cache_few_kernelI")[1].split("EEE")[0]
        d, four, blocks = 64 if "Li64E" in args else 128, args.split("E")[4] == "Lb1", int(args.split("E")[5][2:])
        n = (5 if d == 64 else 4 if four else 3) - blocks
        assert k[".vgpr_count"] <= 512 // n // 8 * 8, k[".name"]
        assert n * k[".group_segment_fixed_size"] <= gate.LDS_BYTES, k[".name"]
    for k in tile:
        n = 3 if "ILi64E" in k[".name"] else 2
        assert k[".vgpr_count"] + k[".agpr_count"] <= 512 // n // 8 * 8, k[".name"]
        assert n * k[".group_segment_fixed_size"] <= gate.LDS_BYTES, k[".name"]
    for what in ("cache_append_kernel", "cache_read_kernel", "cache_score_kernel", "cache_pick_kernel"):
        assert any(what in k[".name"] for k in kernels), what


# ---------------------------------------------------------------------------
def test_oracle_codes():
    """The nearest level, ties to the even code; what codes and scales stand
    for is off by half a level's gap at most."""
    x = torch.tensor([[0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0, -0.25, -5.0, 0.26, -4.99, 0.0, -0.0, 0.74, 3.49]])
    code, scale = O.codes_of(x)
    assert float(scale) == 1.0
    assert code.tolist() == [[0, 2, 2, 4, 4, 6, 6, 7, 8, 14, 1, 14, 0, 0, 1, 5]]
    x = torch.randn(2, 3, 32, 64, generator=torch.Generator().manual_seed(1)).bfloat16()
    back = O.rows_of(O.pack(*O.codes_of(x)), 4)
    top = x.double().abs().amax(-1, keepdim=True) / 6
    t = x.double().abs() / top
    gap = torch.where(t < 2, 0.25, torch.where(t < 4, 0.5, 1.0))
    assert ((back - x.double()).abs() <= gap * top * (1 + 1e-6)).all()
    wild = x.clone()
    wild[0, 0, 0, 0], wild[1, 2, 5, 9] = math.inf, math.nan
    assert torch.isnan(O.rows_of(O.pack(*O.codes_of(wild)), 4)).any(-1).sum() == 2


@pytest.mark.parametrize("bits", [16, 4])
def test_oracle_attends_as_over_a_dense_cache(bits):
    """A cache in any page order against attn_oracle over the rows it stands for."""
    gen = torch.Generator().manual_seed(2)
    ps, D, H, B = 32, 64, 2, 2
    kv, S = [70, 45], 3
    pages = torch.randn(2, 9, H, ps, D, generator=gen).bfloat16()
    table = torch.randperm(9, generator=gen)[:6].int().view(2, 3)
    k, v = (O.pack(*O.codes_of(p)) if bits == 4 else p for p in pages)
    cache = dict(k=k, v=v, bits=bits, table=table, kv=kv, new=[S, S], page_size=ps, D=D, dtype=torch.bfloat16)
    q = torch.randn(B, 4, S, D, generator=gen).bfloat16()
    got = O.attend(q, cache, softcap=3.0)
    for b in range(B):
        kd, vd, ok = O.sequence(cache, b)
        assert ok.all() and kd.shape == (H, kv[b], D)
        want = A.forward(q[b:b + 1], kd[None], vd[None], True, softcap=3.0)
        assert torch.allclose(got[0][b:b + 1], want[0]) and torch.allclose(got[1][b:b + 1], want[1])
    # a page that is none hides its keys; listed pages hide the others
    table[0, 1] = 9
    hidden = O.attend(q, cache)
    kd, vd, ok = O.sequence(cache, 0)
    assert ok.sum() == 70 - 32
    some = torch.tensor([[[[0, 2]] * S] * H] * B)
    listed = O.attend(q, dict(cache, table=table.clone()), selected=some)
    assert torch.allclose(listed[0][0], hidden[0][0])
    twice = O.attend(q, cache, selected=torch.tensor([[[[0, 2, 0, 2]] * S] * H] * B))
    assert torch.allclose(twice[0], listed[0]) and torch.allclose(twice[1], listed[1] + math.log(2))


def test_oracle_selects():
    """Own page first, the largest scores, ties to the lower page; what is not
    finite before all numbers."""
    D, ps = 8, 32
    q = torch.ones(1, 2, 1, D).bfloat16()
    q[0, 1] = -1
    b = torch.zeros(6, 1, 2, D).bfloat16()
    b[1, 0, 1, 0], b[3, 0, 0, 0], b[4, 0, 1, 2] = 2.0, -3.0, 1.0  # scores: 0 2 0 3 1 (0)
    cache = dict(table=torch.arange(6).int()[None], kv=[6 * ps - 1], new=[1], page_size=ps)
    for count, want in ((1, [5]), (2, [3, 5]), (3, [1, 3, 5]), (4, [1, 3, 4, 5]), (5, [0, 1, 3, 4, 5]),
                        (7, [0, 1, 2, 3, 4, 5, -1])):
        assert O.select(q, b, cache, count).flatten().tolist() == want
    b[2, 0, 0, 7] = math.nan
    assert O.select(q, b, cache, 2).flatten().tolist() == [2, 5]
