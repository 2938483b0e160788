"""The check of gradients against differences (attn_differences.py) tells right
gradients from wrong ones: the oracle's, rounded as a kernel rounds, pass, and
the same with a mistake in them do not."""
import pytest

import attn_differences as X
import attn_oracle as A

torch = pytest.importorskip("torch")


def inputs(dtype, D):
    gen = torch.Generator().manual_seed(3)

    def rn(H, std=1.0):
        return (torch.randn(2, H, 60, D, generator=gen) * std).to(dtype)

    q, k, v, do = rn(4, 2.0), rn(2), rn(2), rn(4)
    docs = (torch.arange(60) // 25).int()[None].expand(2, 60).contiguous()
    docs[:, 54:] = -1
    return q, k, v, do, dict(causal=True, softcap=3.0, slopes=torch.exp2(-torch.arange(1, 5).float()),
                             documents=docs, prefix_lens=[20, 0])


def count(q, k, v, do, o, change=lambda n, t: t, backward=A.backward):
    out, lse, _, _ = A.forward(q, k, v, **o)
    out, lse = out.to(q.dtype), lse.float()
    grads = {n: change(n, x[0].to(q.dtype)) for n, x in backward(do, q, k, v, out, lse, **o).items()}
    bad = []
    ratio = X.blocks(q, k, v, do, out, lse, grads, o, lambda *a: bad.append(a))
    return len(bad), ratio


@pytest.mark.parametrize("dtype,D", [(torch.float16, 64), (torch.bfloat16, 128)])
def test_right_gradients_pass(dtype, D):
    bad, ratio = count(*inputs(dtype, D))
    assert bad == 0 and ratio >= X.LEAST


MISTAKES = {
    "zeros": lambda n, t: t * 0, "negated": lambda n, t: -t, "5 % more": lambda n, t: t * 1.05,
    "other head": lambda n, t: t.flip(1), "other entry": lambda n, t: t.flip(0),
    "a row on": lambda n, t: t.roll(1, 2), "not scaled": lambda n, t: t * 8,
}


@pytest.mark.parametrize("what", MISTAKES)
def test_wrong_gradients_do_not(what):
    bad, _ = count(*inputs(torch.float16, 64), MISTAKES[what])
    assert bad == 2 * (4 + 2 + 2)  # (every block of dq, dk and dv)


@pytest.mark.parametrize("what", ["tanh's slope", "delta", "a head of the group"])
def test_wrong_formulas_do_not(what, monkeypatch):
    """Mistakes in the oracle's own backward."""
    def backward(do, q, k, v, out, lse, **o):
        with monkeypatch.context() as m:
            if what == "tanh's slope":
                init = A.Head.__init__

                def flat(self, *a):
                    init(self, *a)
                    self.slope = torch.ones_like(self.s)
                m.setattr(A.Head, "__init__", flat)
            elif what == "delta":
                out = out * 0
            else:
                do = do.clone()
                do[:, 1::2] = 0
            return A.backward(do, q, k, v, out, lse, **o)

    bad, _ = count(*inputs(torch.float16, 64), backward=backward)
    # dq and dk of every head (a head left out: dq of two heads, dk and dv of all)
    assert bad == {"tanh's slope": 12, "delta": 12, "a head of the group": 12}[what]
