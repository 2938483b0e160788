"""The attention layer without a GPU: parameter checks and workspace sizes of
the C entries, refusals that return before any HIP call, the operators' fake
implementations, and the oracle of the GPU tests against autograd and against
differences."""
import ctypes
import math

import pytest

import attn_oracle as A
import shaobo_fa3 as F

torch = pytest.importorskip("torch")


@pytest.fixture(scope="module")
def lib():
    return F.load()


def params(lib, **kw):
    p = F.AttnParams()
    lib.shaobo_fa3_attn_params_init(ctypes.byref(p))
    p.batch, p.seqlen_q, p.seqlen_k = 2, 100, 300
    p.num_heads_q, p.num_heads_kv, p.head_dim = 4, 2, 128
    for n in ("q", "k", "v", "out", "dout", "dq", "dk", "dv"):
        t = getattr(p, n)
        t.batch_stride, t.head_stride, t.row_stride = 128 * 4 * 300, 128 * 300, 128
    for n, x in kw.items():
        obj = p
        *path, last = n.split("__")
        for part in path:
            obj = getattr(obj, part)
        setattr(obj, last, x)
    return p


def test_struct_sizes(lib):
    for cls, init in ((F.AttnParams, lib.shaobo_fa3_attn_params_init),
                      (F.RotaryParams, lib.shaobo_fa3_rotary_params_init)):
        p = cls()
        ctypes.memset(ctypes.byref(p), 0x5A, ctypes.sizeof(p))
        init(ctypes.byref(p))
        assert p.struct_size == ctypes.sizeof(cls)
        assert p.batch == 0 and p.dtype == F.DTYPE_FP16
        init(None)  # tolerated


PTR = 1 << 20  # a non-null address; nothing here reads it


@pytest.mark.parametrize("change,status", [
    ({}, F.SUCCESS),
    ({"struct_size": 8}, F.INVALID_VALUE),
    ({"batch": -1}, F.INVALID_VALUE),
    ({"seqlen_q": -1}, F.INVALID_VALUE),
    ({"num_heads_kv": 0}, F.INVALID_VALUE),
    ({"num_heads_kv": 3}, F.INVALID_VALUE),
    ({"head_dim": 0}, F.INVALID_VALUE),
    ({"causal": 2}, F.INVALID_VALUE),
    ({"softmax_scale_is_set": 2}, F.INVALID_VALUE),
    ({"softmax_scale_is_set": 1, "softmax_scale": math.nan}, F.INVALID_VALUE),
    ({"softmax_scale_is_set": 1, "softmax_scale": math.inf}, F.INVALID_VALUE),
    ({"softmax_scale_is_set": 1, "softmax_scale": -0.5}, F.SUCCESS),
    ({"softmax_scale_is_set": 1, "softmax_scale": 1e31}, F.INVALID_VALUE),
    ({"softcap": 1e31}, F.INVALID_VALUE),
    ({"softcap": 1e30}, F.SUCCESS),
    ({"softcap": -1.0}, F.INVALID_VALUE),
    ({"softcap": math.inf}, F.INVALID_VALUE),
    ({"softcap": math.nan}, F.INVALID_VALUE),
    ({"documents_q": PTR}, F.INVALID_VALUE),
    ({"documents_k": PTR}, F.INVALID_VALUE),
    ({"documents_q": PTR, "documents_k": PTR}, F.SUCCESS),
    ({"prefix_lens": PTR}, F.INVALID_VALUE),  # not causal
    ({"prefix_lens": PTR, "causal": 1}, F.SUCCESS),
    ({"dtype": F.DTYPE_FP8}, F.UNSUPPORTED),
    ({"dtype": F.DTYPE_FP32}, F.UNSUPPORTED),
    ({"head_dim": 136}, F.UNSUPPORTED),
    ({"head_dim": 100}, F.UNSUPPORTED),
    ({"head_dim": 40}, F.SUCCESS),
    ({"k__row_stride": 132}, F.UNSUPPORTED),
    ({"out__head_stride": 4}, F.UNSUPPORTED),
    ({"k__row_stride": 0, "k__batch_stride": -128}, F.SUCCESS),
    ({"seqlen_k": (1 << 30) + 1}, F.UNSUPPORTED),
    ({"batch": 1 << 29}, F.UNSUPPORTED),
    ({"seqlen_q": 1 << 30, "num_heads_q": 8}, F.UNSUPPORTED),
    ({"batch": 1 << 20, "num_heads_q": 32, "num_heads_kv": 32}, F.UNSUPPORTED),  # (2^24 jobs and more)
    ({"seqlen_q": 0}, F.SUCCESS),
    ({"seqlen_k": 0}, F.SUCCESS),
])
def test_validation(lib, change, status):
    p = params(lib, **change)
    assert lib.shaobo_fa3_attn_fwd_validate(ctypes.byref(p)) == status
    assert lib.shaobo_fa3_attn_bwd_validate(ctypes.byref(p)) == status
    if status != F.SUCCESS:
        assert lib.shaobo_fa3_attn_fwd_workspace_bytes(ctypes.byref(p)) == 0
        assert lib.shaobo_fa3_attn_bwd_workspace_bytes(ctypes.byref(p)) == 0
        assert lib.shaobo_fa3_attn_fwd(ctypes.byref(p), None) == status
        assert lib.shaobo_fa3_attn_bwd(ctypes.byref(p), None) == status


def test_backward_checks_its_own_tensors(lib):
    p = params(lib, dk__row_stride=12)
    assert lib.shaobo_fa3_attn_fwd_validate(ctypes.byref(p)) == F.SUCCESS
    assert lib.shaobo_fa3_attn_bwd_validate(ctypes.byref(p)) == F.UNSUPPORTED


def test_null(lib):
    for f in (lib.shaobo_fa3_attn_fwd_validate, lib.shaobo_fa3_attn_bwd_validate):
        assert f(None) == F.INVALID_VALUE
    for f in (lib.shaobo_fa3_attn_fwd, lib.shaobo_fa3_attn_bwd, lib.shaobo_fa3_rotary):
        assert f(None, None) == F.INVALID_VALUE


def full(lib, **kw):
    """Parameters whose pointers are all set (to memory nothing may touch)."""
    p = params(lib)
    for n in ("q", "k", "v", "out", "dout", "dq", "dk", "dv"):
        getattr(p, n).data = PTR
    p.softmax_lse = p.softmax_d = PTR
    p.documents_q = p.documents_k = PTR
    p.workspace, p.workspace_bytes = PTR, 1 << 40
    for n, x in kw.items():
        obj = p
        *path, last = n.split("__")
        for part in path:
            obj = getattr(obj, part)
        setattr(obj, last, x)
    return p


@pytest.mark.parametrize("change,both", [
    ({"q__data": None}, True), ({"k__data": None}, True), ({"v__data": None}, True),
    ({"out__data": None}, True), ({"softmax_lse": None}, True), ({"workspace": None}, True),
    ({"workspace_bytes": 16}, True), ({"workspace": PTR + 16}, True), ({"q__data": PTR + 8}, True),
    ({"dout__data": None}, False), ({"dq__data": None}, False), ({"dk__data": None}, False),
    ({"dv__data": PTR + 2}, False),
])
def test_pointers_are_checked_before_any_launch(lib, change, both):
    p = full(lib, **change)
    if both:
        assert lib.shaobo_fa3_attn_fwd(ctypes.byref(p), None) == F.INVALID_VALUE
    assert lib.shaobo_fa3_attn_bwd(ctypes.byref(p), None) == F.INVALID_VALUE


def test_empty_calls_need_no_memory(lib):
    for change in ({"batch": 0}, {"seqlen_q": 0}):
        p = params(lib, **change)
        assert lib.shaobo_fa3_attn_fwd(ctypes.byref(p), None) == F.SUCCESS
    p = params(lib, batch=0)
    assert lib.shaobo_fa3_attn_bwd(ctypes.byref(p), None) == F.SUCCESS


def test_workspace_grows_with_what_it_holds(lib):
    def need(backward=False, **kw):
        p = params(lib, **kw)
        f = lib.shaobo_fa3_attn_bwd_workspace_bytes if backward else \
            lib.shaobo_fa3_attn_fwd_workspace_bytes
        return f(ctypes.byref(p))

    # a long key axis and few rows: parts of fp32 outputs and log-sum-exps
    one = need(batch=1, seqlen_q=1, seqlen_k=8192)
    assert one % 256 == 0 and one >= 2 * 4 * (128 + 1) * 4
    # many rows, no documents: nothing
    assert need(batch=64, seqlen_q=4096, seqlen_k=4096) == 0
    docs = need(batch=64, seqlen_q=4096, seqlen_k=4096, documents_q=PTR, documents_k=PTR)
    assert docs == 64 * 64 * 8
    # backward: two fp32 rows and a flag per 64 of them
    rows = 2 * 4 * 128
    assert need(True) >= rows * 8 + rows // 64 * 4


def test_backward_cuts_few_heads_into_parts(lib):
    """One KV head for many query heads: dK and dV are summed from parts, two
    fp32 tensors each; many KV heads: they are not."""
    def need(**kw):
        p = params(lib, **kw)
        return lib.shaobo_fa3_attn_bwd_workspace_bytes(ctypes.byref(p))

    few = need(batch=1, seqlen_q=4096, seqlen_k=4096, num_heads_q=8, num_heads_kv=1)
    assert few >= 2 * 2 * 4096 * 128 * 4
    many = need(batch=4, seqlen_q=4096, seqlen_k=4096, num_heads_q=32, num_heads_kv=32)
    assert many < 4 * 32 * 4096 * 8 + 4 * 32 * 64 * 4 + 3 * 256 + 1


def rotary_params(lib, **kw):
    p = F.RotaryParams()
    lib.shaobo_fa3_rotary_params_init(ctypes.byref(p))
    p.batch, p.seqlen, p.head_dim, p.pairs, p.axes = 2, 10, 128, 64, 3
    p.heads[0] = p.heads[1] = 4
    p.positions = p.freqs = PTR
    for k in range(2):
        for t in (p.in_[k], p.out[k]):
            t.data, t.batch_stride, t.head_stride, t.row_stride = PTR, 5120, 1280, 128
    for n, x in kw.items():
        setattr(p, n, x)
    return p


@pytest.mark.parametrize("change,status", [
    ({"struct_size": 4}, F.INVALID_VALUE), ({"batch": -1}, F.INVALID_VALUE),
    ({"tensors": 3}, F.INVALID_VALUE), ({"tensors": 0}, F.INVALID_VALUE),
    ({"axes": 0}, F.INVALID_VALUE), ({"axes": 5}, F.UNSUPPORTED),
    ({"position_type": 3}, F.INVALID_VALUE), ({"interleaved": 2}, F.INVALID_VALUE),
    ({"inverse": -1}, F.INVALID_VALUE), ({"dtype": F.DTYPE_FP8}, F.UNSUPPORTED),
    ({"pairs": 65}, F.UNSUPPORTED), ({"pairs": 72}, F.UNSUPPORTED), ({"pairs": 0}, F.UNSUPPORTED),
    ({"head_dim": 132}, F.UNSUPPORTED), ({"head_dim": 520}, F.UNSUPPORTED),
    ({"positions": None}, F.INVALID_VALUE), ({"freqs": None}, F.INVALID_VALUE),
    ({"seqlen": 1 << 30}, F.UNSUPPORTED), ({"seqlen": 1 << 23}, F.UNSUPPORTED), ({"batch": 0}, F.SUCCESS), ({"seqlen": 0}, F.SUCCESS),
])
def test_rotary_validation(lib, change, status):
    assert lib.shaobo_fa3_rotary(ctypes.byref(rotary_params(lib, **change)), None) == status


def test_rotary_checks_every_tensor(lib):
    for k in range(2):
        p = rotary_params(lib, tensors=2)
        p.heads[k] = 0
        assert lib.shaobo_fa3_rotary(ctypes.byref(p), None) == F.INVALID_VALUE
        for side in ("in_", "out"):
            p = rotary_params(lib, tensors=2)
            getattr(p, side)[k].row_stride = 130
            assert lib.shaobo_fa3_rotary(ctypes.byref(p), None) == F.UNSUPPORTED
            p = rotary_params(lib, tensors=2)
            getattr(p, side)[k].data = PTR + 4
            assert lib.shaobo_fa3_rotary(ctypes.byref(p), None) == F.INVALID_VALUE


# ---------------------------------------------------------------------------
@pytest.fixture(scope="module")
def T():
    import shaobo_fa3_torch
    assert shaobo_fa3_torch._ATTN, "lib/_fa3_torch_attn.so is not built"
    return shaobo_fa3_torch


def test_fake_implementations(T):
    from torch._subclasses.fake_tensor import FakeTensorMode
    with FakeTensorMode():
        q = torch.empty(2, 8, 33, 64, dtype=torch.bfloat16, device="cuda")
        k = torch.empty(2, 50, 4, 64, dtype=torch.bfloat16, device="cuda").transpose(1, 2)
        out, lse = torch.ops.shaobo_fa3.attn_forward(q, k, k, True)
        assert out.shape == q.shape and out.dtype == q.dtype
        assert lse.shape == (2, 8, 33) and lse.dtype == torch.float32
        dq, dk, dv, d = torch.ops.shaobo_fa3.attn_backward(out, q, k, k, out, lse, True)
        assert dq.shape == q.shape and dk.shape == dv.shape == k.shape and d.shape == lse.shape
        assert dk.stride() == k.stride()
        ys = torch.ops.shaobo_fa3.rotary([q, k], q, q, False, False)
        assert [y.shape for y in ys] == [q.shape, k.shape]


def test_cpu_tensors_are_refused(T):
    q = torch.zeros(1, 1, 4, 64, dtype=torch.bfloat16)
    with pytest.raises(NotImplementedError):
        torch.ops.shaobo_fa3.attn_forward(q, q, q, True)


def test_gradients_of_parameters_without_one_are_refused(T):
    q = torch.zeros(1, 2, 4, 64, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="slopes"):
        T.score_attention(q, q, q, slopes=torch.ones(2, requires_grad=True))
    with pytest.raises(ValueError, match="freqs"):
        T.rotary(q, positions=torch.zeros(1, 1, 4), freqs=torch.ones(1, 8, requires_grad=True))


def test_rotary_freqs(T):
    f = T.rotary_freqs([2, 3, 3], theta=100.0)
    one = T.rotary_freqs([8], theta=100.0)
    assert f.shape == (3, 8) and torch.equal(f.sum(0), one[0])
    assert (f != 0).sum(1).tolist() == [2, 3, 3]
    assert abs(float(one[0, 4]) - 0.1) < 1e-8


def test_a_missing_library_is_said(T, monkeypatch):
    monkeypatch.setattr(T, "_ATTN", False)
    q = torch.zeros(1, 1, 4, 64, dtype=torch.bfloat16)
    with pytest.raises(RuntimeError, match="make -C flash-attention3_amd torch"):
        T.score_attention(q, q, q)
    with pytest.raises(RuntimeError, match="make -C flash-attention3_amd torch"):
        T.rotary(q, positions=q, freqs=q)


# The oracle: its gradients are autograd's and the differences' of its forward.
ORACLE = [
    dict(causal=True),
    dict(causal=False, softcap=1.5),
    dict(causal=True, softcap=0.7, slopes=True, prefix_lens=[4, 0]),
    dict(causal=False, slopes=True, documents=True),
    dict(causal=True, kv_lens=[3, 9], documents=None),
]


def oracle_inputs(case, Sq=7, Sk=9):
    gen = torch.Generator().manual_seed(5)
    B, Hq, Hkv, D = 2, 4, 2, 8
    q, do = (torch.randn(B, Hq, Sq, D, generator=gen).double() for _ in range(2))
    k, v = (torch.randn(B, Hkv, Sk, D, generator=gen).double() for _ in range(2))
    case = dict(case)
    if case.get("slopes"):
        case["slopes"] = torch.tensor([0.5, 0.25, 0.125, 0.0625])
    if case.get("documents"):
        case["documents"] = torch.randint(-1, 3, (B, Sq), generator=gen, dtype=torch.int32)
        case["documents_k"] = torch.randint(-1, 3, (B, Sk), generator=gen, dtype=torch.int32)
    return q, k, v, do, case


def plain(q, k, v, case):
    """The forward in differentiable fp64 operations, written apart."""
    B, Hq, Sq, D = q.shape
    G, Sk = Hq // k.shape[1], k.shape[2]
    rows = []
    for b in range(B):
        seen, dist, _ = A.visible(b, Sq, Sk, case["causal"], case.get("documents"),
                                  case.get("documents_k"), case.get("prefix_lens"),
                                  case.get("kv_lens"))
        for h in range(Hq):
            s = q[b, h] @ k[b, h // G].t() / math.sqrt(D)
            if case.get("softcap"):
                s = case["softcap"] * torch.tanh(s / case["softcap"])
            if case.get("slopes") is not None:
                s = s - float(case["slopes"][h]) * dist.abs()
            w = torch.exp(s) * seen
            z = w.sum(1, keepdim=True)
            rows.append((w / torch.where(z == 0, torch.ones_like(z), z)) @ v[b, h // G])
    return torch.stack(rows).view(B, Hq, Sq, D)


@pytest.mark.parametrize("case", ORACLE)
def test_oracle_gradients(case):
    q, k, v, do, case = oracle_inputs(case)
    out, lse, _, _ = A.forward(q, k, v, **case)
    leaves = [t.clone().requires_grad_() for t in (q, k, v)]
    want = plain(*leaves, case)
    assert torch.allclose(out, want.detach(), atol=1e-12)
    grads = torch.autograd.grad((want * do).sum(), leaves)
    got = A.backward(do, q, k, v, out, lse, **case)
    for n, g in zip(("dq", "dk", "dv"), grads):
        assert torch.allclose(got[n][0], g, atol=1e-11), n
    # central differences along one direction: third-order terms at 1e-5 are ~1e-10
    gen = torch.Generator().manual_seed(6)
    for n, i in (("dq", 0), ("dk", 1), ("dv", 2)):
        d = torch.randn((q, k, v)[i].shape, generator=gen).double()
        d /= d.norm()
        ends = []
        for step in (1e-5, -1e-5):
            x = [q, k, v]
            x[i] = x[i] + step * d
            ends.append(float((A.forward(*x, **case)[0] * do).sum()))
        assert abs((ends[0] - ends[1]) / 2e-5 - float((got[n][0] * d).sum())) < 1e-7, n


def test_oracle_rotary_is_a_rotation():
    gen = torch.Generator().manual_seed(1)
    x = torch.randn(2, 3, 5, 48, generator=gen)
    pos = torch.randint(0, 1000000, (2, 2, 5), generator=gen)
    freqs = torch.rand(2, 16, generator=gen)
    for inter in (False, True):
        y, off = A.rotary(x, pos, freqs, inter)
        assert torch.equal(y[..., 32:], x[..., 32:].double()) and (off[..., 32:] == 0).all()
        back, _ = A.rotary(y, pos, freqs, inter, True)
        assert torch.allclose(back, x.double(), atol=1e-9)
        assert torch.allclose(y.norm(dim=-1), x.double().norm(dim=-1))
