"""The attention layer where autograd, other rows' values and padding meet it
in ways that the plain cases do not."""
import math

import pytest

import attn_oracle as A
import shaobo_fa3 as F
from test_gpu_attn import BF, HF, i32, make, op_args, randn, run_both

torch = pytest.importorskip("torch")
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
