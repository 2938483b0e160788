"""The attention layer where autograd, other rows' values and padding meet it
in ways that the plain cases do not."""
import functools
import math
from concurrent.futures import ThreadPoolExecutor
from fractions import Fraction

import pytest

import attn_differences as X
import attn_oracle as A
import shaobo_fa3 as F
from test_gpu_attn import BF, HF, make, op_args, oracle_options, randn, within

torch = pytest.importorskip("torch")
import torch.utils.checkpoint  # noqa: E402

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def T():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    F.load()
    import shaobo_fa3_torch
    assert shaobo_fa3_torch._ATTN, "lib/_fa3_torch_attn.so is not built"
    return shaobo_fa3_torch


@pytest.mark.parametrize("dtype,offset", [(HF, 3), (BF, 1), (BF, 8)])
def test_gradients_that_start_anywhere(T, dtype, offset):
    """An output joined with others in one vector: its gradient is a view into
    that vector's, contiguous from whatever element on."""
    print("[case] gradient at element", offset, dtype, flush=True)
    gen = torch.Generator(device="cuda").manual_seed(41)
    q, k, v = (randn(gen, 2, h, 128, 64, dtype) for h in (4, 2, 2))
    pos = torch.arange(128, device="cuda").expand(1, 2, 128)
    freqs = T.rotary_freqs([32], device="cuda")
    w = torch.randn(offset + q.numel(), generator=gen, device="cuda").to(dtype)

    def grads(f, xs, joined):
        xs = [x.detach().clone().requires_grad_() for x in xs]
        y = f(*xs)
        if joined:
            torch.cat([torch.zeros(offset, dtype=dtype, device="cuda"), y.flatten()]).backward(w)
        else:
            y.backward(w[offset:].clone().view(y.shape))
        return [x.grad for x in xs]

    for f, xs in ((lambda *x: T.score_attention(*x), (q, k, v)),
                  (lambda x: T.rotary(x, positions=pos, freqs=freqs), (q,)),
                  (lambda *x: T.attention(*x), (q, k, v))):
        for a, b in zip(grads(f, xs, True), grads(f, xs, False)):
            assert torch.equal(a, b)


@pytest.mark.parametrize("where", ["q", "k", "v", "dout"])
@pytest.mark.parametrize("case", [
    dict(Sq=150, D=128, Hq=4, docs=40.0), dict(Sq=150, D=64, dtype=HF, Hq=4, docs=40.0),
    dict(Sq=150, D=128, Hq=4, docs=40.0, causal=False, softcap=10.0), dict(Sq=100, Sk=60, D=128, slopes=1),
    dict(Sq=100, Sk=60, D=72, dtype=HF, softcap=200.0), dict(Sq=70, D=64, kv=[9, 70]),
    # (jobs of whole 128 rows)
    dict(B=12, Hq=24, Hkv=12, Sq=600, D=128, docs=40.0)], ids=str)
def test_gradients_of_rows_without_keys(T, case, where):
    """A NaN in what some rows see (or in their own Q or dO): the rows of its
    tiles that see nothing have a gradient of zero all the same, and other
    batch entries stay as they are."""
    print("[case] keyless rows", case, where, flush=True)
    q, k, v, do, o = make(case)
    B, _, Sq, _ = q.shape
    Sk = k.shape[2]
    if "docs" in case:
        o["documents_k"] = o["documents"].clone()
        o["documents"][0, 60:70] = 99999  # (a document without keys)
    seen = A.visible(0, Sq, Sk, o["causal"], o.get("documents"), o.get("documents_k"), None,
                     o.get("kv_lens"), "cuda")[0]
    rows, keys = seen.any(1), seen.any(0)
    assert rows.any() and not rows.all()
    for bad in (math.nan, math.inf):
        x = dict(q=q, k=k, v=v, dout=do)
        x[where] = x[where].clone()
        hit = rows if where in ("q", "dout") else keys
        x[where][0, 0, hit.nonzero()[0, 0], 5] = bad
        out, lse = torch.ops.shaobo_fa3.attn_forward(x["q"], x["k"], x["v"], *op_args(o))
        dq, dk, dv, delta = torch.ops.shaobo_fa3.attn_backward(
            x["dout"], x["q"], x["k"], x["v"], out, lse, *op_args(o))
        torch.cuda.synchronize()
        assert (lse[0, :, ~rows] == -math.inf).all()
        for t in (out[0], dq[0]):
            assert (t[:, ~rows] == 0).all()
        assert (delta[0, :, ~rows] == 0).all()
        for t in (out, dq, dk, dv, delta):
            assert torch.isfinite(t[1:]).all()


@pytest.mark.parametrize("Sq,causal", [(150, True), (150, False), (1111, True)])
@pytest.mark.parametrize("pad", [-1, -2, -3, -4, -2147483648])
def test_every_negative_document_is_padding(T, pad, Sq, causal):
    """Padding on both sides under any negative document, a NaN in a key that
    the other rows see, junk in the padding: its rows stay zeros, and take no
    part in the backward."""
    print("[case] padding", pad, Sq, causal, flush=True)
    q, k, v, do, o = make(dict(Sq=Sq, D=128, Hq=4, causal=causal))
    ids = torch.zeros(2, Sq, dtype=torch.int32, device="cuda")
    ids[0, 100:110] = pad
    ids[1, 7] = pad
    o["documents"] = ids
    here = ids < 0
    k[:, 0, 60, 3] = math.nan
    q, do = (torch.where(here[:, None, :, None], math.nan, t).to(BF) for t in (q, do))
    out, lse = torch.ops.shaobo_fa3.attn_forward(q, k, v, *op_args(o))
    dq, dk, dv, delta = torch.ops.shaobo_fa3.attn_backward(do, q, k, v, out, lse, *op_args(o))
    torch.cuda.synchronize()
    for b in range(2):
        assert (lse[b, :, here[b]] == -math.inf).all()
        assert all((t[b, :, here[b]] == 0).all() for t in (out, dq, delta))
        # (KV head 1 holds no NaN that counts)
        assert all(torch.isfinite(t[b, 2:]).all() for t in (out, dq, delta))
        assert all(torch.isfinite(t[b, 1]).all() for t in (dk, dv))


def test_launches_that_do_not_fit_are_value_errors(T):
    """More rows or positions than a launch takes: refused as every other
    argument is, before any memory is taken for outputs."""
    ops = torch.ops.shaobo_fa3
    row = torch.zeros(1, 1, 1, 8, dtype=BF, device="cuda")
    for B, H, S in ((1 << 19, 32, 1), (1, 16, 1 << 23), (1 << 12, 1 << 12, 1)):
        q = row.expand(B, H, S, 8)
        torch.cuda.synchronize()
        torch.cuda.reset_peak_memory_stats()
        before = torch.cuda.max_memory_allocated()
        with pytest.raises(ValueError, match="shaobo_fa3_attn_fwd"):
            ops.attn_forward(q, q, q, True)
        assert torch.cuda.max_memory_allocated() == before
    # (a backward whose lse is there is asked for its own launch)
    q = row.expand(1, 16, 1 << 22, 8)
    lse = torch.zeros(1, 16, 1 << 22, device="cuda")
    with pytest.raises(ValueError, match="shaobo_fa3_attn_bwd"):
        ops.attn_backward(q, q, q, q, q, lse, True)


@pytest.mark.parametrize("case", [
    dict(Sq=60, Hq=4, D=64, dtype=HF, softcap=3.0, slopes=1, prefix=[20, 0], docs=25.0, std=2.0),
    dict(Sq=60, Hq=4, D=128, softcap=3.0, slopes=1, prefix=[20, 0], docs=25.0, std=2.0),
    dict(Sq=140, Hq=4, D=64, dtype=HF), dict(Sq=90, Sk=150, D=72, causal=False, slopes=2, kv=[150, 101]),
    dict(Sq=70, Hq=6, Hkv=1, D=128, dtype=HF, softcap=150.0, std=20.0, softmax_scale=-0.1)], ids=str)
def test_gradients_of_every_head_against_differences(T, case):
    """dq, dk and dv of each (batch entry, head) along themselves against
    central differences of the fp64 forward; every tolerance, made from the
    counted roundings, is a tenth of its derivative at most."""
    print("[case] differences", case, flush=True)
    q, k, v, do, o = make(case)
    out, lse = torch.ops.shaobo_fa3.attn_forward(q, k, v, *op_args(o))
    grads = dict(zip(("dq", "dk", "dv"),
                     torch.ops.shaobo_fa3.attn_backward(do, q, k, v, out, lse, *op_args(o))))

    def fail(n, b, h, off, tol, slope):
        raise AssertionError(f"{n}[{b}, {h}]: {off:.3e} off a derivative of {slope:.3e}, "
                             f"{tol:.3e} allowed")

    assert X.blocks(q, k, v, do, out, lse, grads, oracle_options(o), fail) >= X.LEAST


@pytest.mark.parametrize("case", [
    dict(B=1, Hq=8, Hkv=1, Sq=700, D=128),                     # dK and dV from parts
    dict(B=2, Hq=8, Hkv=2, Sq=500, D=128, docs=90.0, softcap=20.0),
    dict(B=1, Hq=8, Hkv=2, Sq=3, Sk=5000, D=128, slopes=1)], ids=str)
def test_backwards_on_two_streams_at_once(T, case):
    """Each call has scratch of its own: row statistics, flags, document
    ranges and parts pass between up to three kernels of each."""
    print("[case] two streams", case, flush=True)
    inputs = [make(case, seed) for seed in (1, 2)]
    ops = torch.ops.shaobo_fa3

    def step(q, k, v, do, o):
        out, lse = ops.attn_forward(q, k, v, *op_args(o))
        return (out, lse, *ops.attn_backward(do, q, k, v, out, lse, *op_args(o)))

    want = [step(*x) for x in inputs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = [[], []]
    for _ in range(6):
        for i, x in enumerate(inputs):
            with torch.cuda.stream(streams[i]):
                got[i].append(step(*x))
    torch.cuda.synchronize()
    for a, runs in zip(want, got):
        for b in runs:
            assert all(torch.equal(x, y) for x, y in zip(a, b))


def test_training_steps_in_two_threads(T):
    """Two host threads, a stream each: their steps are those of one."""
    print("[case] two threads", flush=True)
    inputs = [make(dict(B=2, Hq=6, Hkv=2, Sq=300, D=64, docs=70.0), seed) for seed in (1, 2)]

    def step(q, k, v, do, o):
        xs = [t.detach().clone().requires_grad_() for t in (q, k, v)]
        out = T.score_attention(*xs, causal=True, documents=o["documents"])
        out.backward(do)
        return [out.detach()] + [t.grad for t in xs]

    want = [step(*x) for x in inputs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]

    def work(i):
        with torch.cuda.stream(streams[i]):
            runs = [step(*inputs[i]) for _ in range(6)]
            streams[i].synchronize()
        return runs

    with ThreadPoolExecutor(2) as pool:
        for a, runs in zip(want, pool.map(work, range(2))):
            for b in runs:
                assert all(torch.equal(x, y) for x, y in zip(a, b))


TURN = Fraction(62831853071795864769252867665590057683943387987502116419498891846, 10 ** 64)  # 2 pi


@pytest.mark.parametrize("inverse", [False, True])
@pytest.mark.parametrize("bits,axes,kind", [
    (20, 1, torch.int32), (31, 3, torch.int32), (32, 1, torch.int64), (40, 2, torch.int64),
    (53, 1, torch.int64), (53, 4, torch.int64), (24, 2, torch.float32), (50, 1, torch.float32)],
    ids=str)
def test_rotary_at_far_positions(T, bits, axes, kind, inverse):
    """Positions up to 2^53 against angles reduced as exact fractions.  The
    angle's fp32 remainder and the sine are off by 2^-22 together (as at near
    positions), the products and their sum by 2^-23 each."""
    print("[case] far positions", bits, axes, kind, flush=True)
    gen = torch.Generator(device="cuda").manual_seed(bits)
    P, S = 32, 24
    pos = torch.randint(2 ** (bits - 1), 2 ** bits, (axes, 1, S), generator=gen, device="cuda")
    pos[:, :, ::2] *= -1
    pos = pos.to(kind)
    freqs = torch.rand(axes, P, generator=gen, device="cuda")
    freqs[:, 0] = 1.0
    x = torch.randn(1, 2, S, 2 * P, generator=gen, device="cuda")
    (y,) = torch.ops.shaobo_fa3.rotary([x], pos, freqs, False, inverse)
    torch.cuda.synchronize()
    at = [[Fraction(n) for n in row] for row in pos[:, 0].tolist()]
    per = [[Fraction(f) for f in row] for row in freqs.tolist()]
    angle = torch.empty(S, P, dtype=torch.float64)
    for s in range(S):
        for p in range(P):
            turns = sum(at[a][s] * per[a][p] for a in range(axes)) / TURN
            angle[s, p] = float((turns - round(turns)) * TURN)
    if inverse:
        angle = -angle
    a, b = x.double().cpu().split(P, 3)
    got = y.double().cpu().split(P, 3)
    for g, want in zip(got, (a * angle.cos() - b * angle.sin(), b * angle.cos() + a * angle.sin())):
        off = (a.abs() + b.abs()) * 2.0 ** -21 + 2.0 ** -24 * want.abs()
        assert ((g - want).abs() <= off).all(), float(((g - want).abs() - off).max())


@pytest.mark.parametrize("B,Hq,Hkv,S,D,causal,dtype", [
    (1, 4, 4, 384, 128, True, HF), (2, 8, 2, 256, 64, True, BF), (1, 4, 1, 512, 128, False, BF),
    (2, 3, 3, 128, 64, False, HF)])
def test_the_forward_feeds_either_backward(T, monkeypatch, B, Hq, Hkv, S, D, causal, dtype):
    """Without options both backwards are the gradient of attn_forward, within
    the oracle's bound.  The other one's operands may carry the scale: a score
    is off by half a step of each of its products then, and an operand of the
    last products by half a step more, as much as dS (so twice that bound)."""
    print("[case] either backward", B, Hq, Hkv, S, D, causal, dtype, flush=True)
    q, k, v, do, o = make(dict(B=B, Hq=Hq, Hkv=Hkv, Sq=S, D=D, causal=causal, dtype=dtype))
    out, lse = torch.ops.shaobo_fa3.attn_forward(q, k, v, causal)
    both = (torch.ops.shaobo_fa3.attn_backward(do, q, k, v, out, lse, causal),
            torch.ops.shaobo_fa3.flash_attn_backward(do, q, k, v, out, lse, causal))
    torch.cuda.synchronize()
    init, u = A.Head.__init__, torch.finfo(dtype).eps / 2

    def scaled(self, q, k, scale, *rest):
        init(self, q, k, scale, *rest)
        self.dx = self.dx + u * scale * (self.q.abs() @ self.k.abs().t().contiguous()) * self.seen

    want = [A.backward(do, q, k, v, out, lse, causal)]
    monkeypatch.setattr(A.Head, "__init__", scaled)
    want.append(A.backward(do, q, k, v, out, lse, causal))
    for times, grads, w in zip((1, 2), both, want):
        for n, g in zip(("dq", "dk", "dv", "delta"), grads):
            within(n, g, w[n][0], times * w[n][1])


@pytest.mark.parametrize("causal", [True, False])
def test_documents_are_any_numbers(T, causal):
    """Only the numbers' order and sign count, up to the type's last ones."""
    print("[case] document numbers", causal, flush=True)
    q, k, v, do, o = make(dict(Sq=400, Hq=4, D=64, causal=causal))
    small = torch.tensor([0, 1, 2, 3, -1], dtype=torch.int32, device="cuda")
    large = torch.tensor([0, 70000, 2147483646, 2147483647, -2147483648], dtype=torch.int32, device="cuda")
    for pick in (torch.arange(400, device="cuda") // 90, torch.arange(400, device="cuda") * 7 % 5,
                 torch.full((400,), 3, device="cuda")):
        got = []
        for names in (small, large):
            o["documents"] = names[pick][None].expand(2, 400).contiguous()
            out, lse = torch.ops.shaobo_fa3.attn_forward(q, k, v, *op_args(o))
            got.append((out, lse, *torch.ops.shaobo_fa3.attn_backward(do, q, k, v, out, lse, *op_args(o))))
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(*got))


def test_layers_under_tracing_and_recomputation(T):
    """The layer traced through the operators' fake implementations, and
    recomputed in its backward: the eager step's outputs and gradients."""
    print("[case] tracing", flush=True)
    q, k, v, do, o = make(dict(Sq=100, Hq=4, D=64, docs=30.0, bshd=True))
    pos = torch.arange(100, device="cuda").expand(1, 2, 100)
    freqs = T.rotary_freqs([32], device="cuda")

    def layer(q, k, v):
        q, k = T.rotary(q, k, positions=pos, freqs=freqs)
        return T.score_attention(q, k, v, softcap=10.0, documents=o["documents"])

    def step(f):
        xs = [t.detach().clone(memory_format=torch.preserve_format).requires_grad_() for t in (q, k, v)]
        out = f(*xs)
        out.backward(do)
        return [out.detach()] + [x.grad for x in xs]

    want = step(layer)
    traced = torch.compile(layer, backend="aot_eager")
    again = functools.partial(torch.utils.checkpoint.checkpoint, layer, use_reentrant=False)
    for f in (traced, again):
        assert all(torch.equal(x, y) for x, y in zip(want, step(f)))
