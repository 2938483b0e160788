"""What autograd may hand the attention layer's functions as a gradient, and
what they pass on to the operators: rows of whole 16-byte chunks that start at
a 16-byte boundary."""
import pytest

torch = pytest.importorskip("torch")


@pytest.fixture(scope="module")
def T():
    import shaobo_fa3_torch
    return shaobo_fa3_torch


def gradient_of_cat(shape, dtype, offset):
    """The gradient of a tensor that was joined behind `offset` others in one
    vector: contiguous, and a view into that vector's gradient."""
    x = torch.zeros(shape, dtype=dtype, requires_grad=True)
    caught = []
    x.register_hook(caught.append)
    y = torch.cat([torch.zeros(offset, dtype=dtype), x.flatten()])
    y.backward(torch.arange(y.numel(), dtype=torch.float32).to(dtype))
    return caught[0]


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("offset", [0, 1, 3, 4, 8])
def test_rows_start_at_16_bytes(T, dtype, offset):
    g = gradient_of_cat((2, 3, 5, 16), dtype, offset)
    assert g.is_contiguous() and g.storage_offset() == offset
    t = T._in_rows(g)
    assert torch.equal(t, g)
    assert t.storage_offset() * t.element_size() % 16 == 0 and t.is_contiguous()
    if offset * g.element_size() % 16 == 0:
        assert t is g  # (nothing to copy)


def test_rows_of_any_layout(T):
    x = torch.arange(2 * 3 * 8 * 16, dtype=torch.float32).to(torch.bfloat16).view(2, 3, 8, 16)
    for t in (x.transpose(1, 2), x[..., :8], x[:, 1:], x.transpose(2, 3), x[..., 1:9],
              x[..., :1].expand(2, 3, 8, 16), x[:, :1].expand(2, 3, 8, 16)):
        y = T._in_rows(t)
        assert torch.equal(y, t) and y.stride(-1) == 1
        assert y.storage_offset() % 8 == 0 and all(s % 8 == 0 for s in y.stride()[:-1])
