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


# ---- capped scores ------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype,nh,nkv,hd", HEADS)
@pytest.mark.parametrize("ql,kl", [([390], [390]), ([3], [390]), ([60], [4000])])
@pytest.mark.parametrize("softcap", [1.0, 5.0, 30.0])
@pytest.mark.parametrize("hidden", [50.0, math.inf, math.nan])
def test_a_capped_score_does_not_depend_on_its_neighbours(dtype, nh, nkv, hd, ql, kl, softcap, hidden):
    """Scores below and past half the cap are computed differently; which way goes by the score alone, not by hidden keys nor by
    other rows' scores."""
    q, k, v = normal(51, sum(ql), nh, hd, scale=0.5, dtype=dtype), normal(52, sum(kl), nkv, hd, dtype=dtype), normal(53, sum(kl), nkv, hd, dtype=dtype)
    k_doc = (torch.arange(sum(kl)) % 7 == 3).to(torch.int32).cuda()
    q_doc = torch.zeros(sum(ql), dtype=torch.int32, device="cuda")
    opt = dict(scale=hd ** -0.5, softcap=softcap, q_doc=q_doc, k_doc=k_doc)
    want = attend(q, k, v, ql, kl, **opt)
    check_attention(q, k, v, ql, kl, want, **opt)
    other = k.clone()
    other[k_doc == 1] *= hidden
    got = attend(q, other, v, ql, kl, **opt)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    louder = q.clone()
    louder[::2] *= 20.0
    got = attend(louder, k, v, ql, kl, **opt)
    check_attention(louder, k, v, ql, kl, got, **opt)
    assert torch.equal(got[0][1::2], want[0][1::2]) and torch.equal(got[1][1::2], want[1][1::2])


@pytest.mark.parametrize("dtype,nh,nkv,hd", HEADS)
@pytest.mark.parametrize("nq", [3, 200])
@pytest.mark.parametrize("scale,softcap", [(0.0625, 1000.0), (0.0625, 6.0), (-0.125, 20.0), (3.0, 2.0)])
def test_capped_scores_near_and_far_from_the_cap(dtype, nh, nkv, hd, nq, scale, softcap):
    ql, kl = [nq], [333]
    q, k, v = normal(54, nq, nh, hd, dtype=dtype), normal(55, 333, nkv, hd, dtype=dtype), normal(56, 333, nkv, hd, dtype=dtype)
    opt = dict(scale=scale, softcap=softcap)
    check_attention(q, k, v, ql, kl, attend(q, k, v, ql, kl, **opt), **opt)
