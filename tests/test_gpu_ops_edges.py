"""The layer operators (``ops``) at the ends of their stated ranges: the largest windows and sums, biases of minus infinity and of the
type's lowest value, values that are not finite, the smallest numbers; against 64-bit forms."""
import math

import numpy as np
import pytest

from conftest import pkg

torch = pytest.importorskip("torch")

from test_gpu_ops import BF16, F32, HEADS, L, attend, attention_64, check_attention, normal, offsets, ops

pytestmark = pytest.mark.gpu


# ---- windows --------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype,nh,nkv,hd", HEADS)
@pytest.mark.parametrize("ql,kl", [([5], [2]), ([40], [3]), ([300, 2, 7], [90, 4, 0]), ([300, 200], [3000, 5])])
@pytest.mark.parametrize("window", [2**31 - 1, 2**31 - 5, 2**20])
def test_the_largest_windows_see_every_key(dtype, nh, nkv, hd, ql, kl, window):
    """More queries than keys put the first queries at negative places: a window that reaches every key is no window, to the bit."""
    q, k, v = normal(1, sum(ql), nh, hd, scale=2.0, dtype=dtype), normal(2, sum(kl), nkv, hd, dtype=dtype), normal(3, sum(kl), nkv, hd, dtype=dtype)
    opt = dict(scale=hd ** -0.5, softcap=30.0)
    got = attend(q, k, v, ql, kl, window=window, **opt)
    check_attention(q, k, v, ql, kl, got, window=window, **opt)
    want = attend(q, k, v, ql, kl, **opt)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
