"""Sizes at the ends of their types: refused on the host, before any HIP call."""
import ctypes

import pytest

import shaobo_fa3 as F

PTR = 1 << 20  # a non-null address; nothing here reads it
MOST = (1 << 31) - 1


@pytest.fixture(scope="module")
def lib():
    return F.load()


@pytest.mark.parametrize("pairs", [1 << 30, (1 << 30) + 8, MOST - 7, 72])
@pytest.mark.parametrize("interleaved", [0, 1])
def test_rotary_pairs_whose_double_leaves_its_type(lib, pairs, interleaved):
    p = F.RotaryParams()
    lib.shaobo_fa3_rotary_params_init(ctypes.byref(p))
    p.batch, p.seqlen, p.head_dim, p.pairs, p.heads[0] = 1, 4, 128, pairs, 1
    p.interleaved = interleaved
    p.positions = p.freqs = PTR
    for t in (p.in_[0], p.out[0]):
        t.data, t.batch_stride, t.head_stride, t.row_stride = PTR, 512, 512, 128
    assert lib.shaobo_fa3_rotary(ctypes.byref(p), None) == F.UNSUPPORTED
