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


# ---- values that are not finite ---------------------------------------------------------------------------
def places(ql, kl):
    """Place of each query row among its sequence's keys, and its sequence."""
    at = [(nk - nq + t, b) for b, (nq, nk) in enumerate(zip(ql, kl)) for t in range(nq)]
    return torch.tensor([a for a, _ in at]).cuda(), torch.tensor([b for _, b in at]).cuda()


BF16_HEADS = [(BF16, 4, 2, 64), (BF16, 2, 1, 128), (BF16, 4, 2, 256), (BF16, 4, 1, 512), (BF16, 3, 1, 128), (BF16, 3, 3, 80)]


@pytest.mark.parametrize("dtype,nh,nkv,hd", HEADS)
@pytest.mark.parametrize("ql,kl", [([390], [390]), ([5, 3], [200, 700]), ([60], [4000]), ([40, 300], [900, 300])])
def test_any_number_of_hidden_values_may_not_be_finite(dtype, nh, nkv, hd, ql, kl):
    """Dozens of NaN and infinite rows of V in a hidden document, and past a causal bound: the other rows keep their bits."""
    q, k, v = normal(31, sum(ql), nh, hd, scale=2.0, dtype=dtype), normal(32, sum(kl), nkv, hd, dtype=dtype), normal(33, sum(kl), nkv, hd, dtype=dtype)
    n = sum(kl)
    j = torch.arange(n)
    k_doc = ((j % 9 == 4) | ((j > n // 2) & (j < n // 2 + 40))).to(torch.int32).cuda()
    q_doc = torch.zeros(sum(ql), dtype=torch.int32, device="cuda")
    opt = dict(scale=hd ** -0.5, softcap=30.0, q_doc=q_doc, k_doc=k_doc)
    clean = attend(q, k, v, ql, kl, **opt)
    check_attention(q, k, v, ql, kl, clean, **opt)
    bad = v.clone()
    bad[k_doc == 1] = math.nan
    bad[(k_doc == 1) & (j.cuda() % 2 == 0)] = math.inf
    got = attend(q, k, bad, ql, kl, **opt)
    assert torch.equal(got[0], clean[0]) and torch.equal(got[1], clean[1])
    # the last 70 keys of every sequence, seen by its last queries alone
    opt = dict(scale=hd ** -0.5, causal=True)
    clean = attend(q, k, v, ql, kl, **opt)
    bad, place, seq = v.clone(), *places(ql, kl)
    sees = torch.zeros(sum(ql), dtype=torch.bool, device="cuda")
    for b, end in enumerate(np.cumsum(kl)):
        bad[int(end) - 70 : int(end)] = math.nan
        sees |= (seq == b) & (place >= kl[b] - 70)
    out, lse = attend(q, k, bad, ql, kl, **opt)
    assert torch.equal(out[~sees], clean[0][~sees]) and torch.equal(lse, clean[1])
    assert not bool(torch.isfinite(out[sees]).any())


@pytest.mark.parametrize("dtype,nh,nkv,hd", HEADS)
@pytest.mark.parametrize("ql,kl", [([390], [390]), ([3], [700]), ([2], [5003]), ([60], [4000]), ([17, 200], [1500, 200])])
@pytest.mark.parametrize("window", [-1, 60])
def test_visible_infinities_keep_their_sign_and_channel(dtype, nh, nkv, hd, ql, kl, window):
    """A channel that meets one kind of infinity becomes it, one that meets both or a NaN becomes NaN, for the rows that see
    the key; all else keeps its bits."""
    q, k, v = normal(41, sum(ql), nh, hd, scale=2.0, dtype=dtype), normal(42, sum(kl), nkv, hd, dtype=dtype), normal(43, sum(kl), nkv, hd, dtype=dtype)
    opt = dict(scale=hd ** -0.5, causal=True, window=window)
    clean = attend(q, k, v, ql, kl, **opt)
    bad, place, seq = v.clone(), *places(ql, kl)
    want = clean[0].double()
    G = nh // nkv
    for b, (end, n) in enumerate(zip(np.cumsum(kl), kl)):
        for back, ch, e in ((1, 0, math.inf), (2, 0, math.inf), (2, 1, -math.inf), (3, 2, math.nan), (40, 3, math.inf), (50, 3, -math.inf),
                            (30, hd - 1, -math.inf), (130, hd // 2, math.inf)):
            key = n - back
            bad[int(end) - back, 0, ch] = e
            rows = (seq == b) & (place >= key)
            if window >= 0:
                rows &= place - key <= window
            want[rows, :G, ch] += e  # the first K/V head's query heads
    out, lse = attend(q, k, bad, ql, kl, **opt)
    kept = torch.isfinite(want)
    assert torch.equal(out[kept], clean[0][kept]) and torch.equal(lse, clean[1])
    assert torch.equal(torch.isnan(out), torch.isnan(want))
    assert torch.equal(out[torch.isinf(want)].double(), want[torch.isinf(want)])
    assert L.load().eg2_device_status() == 0


@pytest.mark.parametrize("dtype,nh,nkv,hd,nq", [h + (64,) for h in BF16_HEADS] + [(BF16, 1, 1, 64, 20_000), (BF16, 1, 1, 128, 20_000)])
def test_a_value_that_is_not_finite_in_a_long_sequence(dtype, nh, nkv, hd, nq):
    """200,000 keys, one of them infinite, one NaN in one channel, one NaN and hidden from all but the last query; with the key axis
    split and whole: no wait runs out."""
    n = 200_000
    q, k, v = normal(44, nq, nh, hd, scale=2.0, dtype=dtype), normal(45, n, nkv, hd, dtype=dtype), normal(46, n, nkv, hd, dtype=dtype)
    opt = dict(scale=hd ** -0.5, causal=True)
    clean = attend(q, k, v, [nq], [n], **opt)
    v[777] = math.inf * v[777].sign()
    v[n - 30, :, 5] = math.nan
    v[n - 1] = math.nan
    out, lse = attend(q, k, v, [nq], [n], **opt)
    torch.cuda.synchronize()
    assert L.load().eg2_device_status() == 0
    assert torch.equal(lse, clean[1])
    assert bool(torch.isnan(out[-1]).all()) and bool(torch.isnan(out[nq - 30 :, :, 5]).all())
    sign = v[777].repeat_interleave(nh // nkv, 0)
    assert torch.equal(out[: nq - 30], sign.expand(nq - 30, nh, hd))


# ---- biases of minus infinity ---------------------------------------------------------------------------
@pytest.mark.parametrize("dtype,nh,nkv,hd", HEADS)
@pytest.mark.parametrize("ql,kl", [([150], [150]), ([3], [150]), ([70, 330], [70, 330]), ([2], [5003]), ([100], [4000])])
@pytest.mark.parametrize("heads", ["all", "first"])
def test_biases_of_minus_infinity_hide_keys(dtype, nh, nkv, hd, ql, kl, heads):
    """A bias of -infinity is a mask: what keys hold under it (NaN, infinities, in K or in V) reaches no row, to the bit."""
    R = 9
    table = normal(11, nh, 2 * R + 1, scale=2.0)
    hide = slice(0, nh if heads == "all" else 1)
    table[hide, 2 * R] = -math.inf     # keys R and more ahead
    table[hide, : R - 4] = -math.inf   # keys 5 and more behind
    table[hide, R + 2] = -math.inf     # and one in between
    q, k, v = normal(12, sum(ql), nh, hd, scale=2.0, dtype=dtype), normal(13, sum(kl), nkv, hd, dtype=dtype), normal(14, sum(kl), nkv, hd, dtype=dtype)
    opt = dict(scale=hd ** -0.5, softcap=20.0, table=table)
    clean = attend(q, k, v, ql, kl, **opt)
    check_attention(q, k, v, ql, kl, clean, **opt)
    place, seq = places(ql, kl)
    start = torch.tensor(np.cumsum([0] + kl)[:-1]).cuda()
    for what, bad in (("v", math.nan), ("v", -math.inf), ("k", math.nan), ("k", math.inf)):
        kk, vv = k.clone(), v.clone()
        sees = torch.zeros(sum(ql), nh, dtype=torch.bool, device="cuda")
        for b, n in enumerate(kl):
            for key in {0, n // 2, n - 1}:
                (vv if what == "v" else kk)[int(start[b]) + key] = bad
                bias = table.T[(key - place).clamp(-R, R) + R]  # [rows, nh]
                sees |= (seq == b)[:, None] & (bias != -math.inf)
        out, lse = attend(q, kk, vv, ql, kl, **opt)
        assert torch.equal(out[~sees], clean[0][~sees]) and torch.equal(lse[~sees], clean[1][~sees])
        if what == "v":
            assert not bool(torch.isfinite(out[sees]).any())
    assert L.load().eg2_device_status() == 0


@pytest.mark.parametrize("dtype,nh,nkv,hd", HEADS)
@pytest.mark.parametrize("ql,kl", [([150], [150]), ([3], [150]), ([2], [5003]), ([100], [4000])])
def test_rows_that_a_bias_hides_whole_are_empty(dtype, nh, nkv, hd, ql, kl):
    table = torch.zeros(nh, 5, device="cuda")
    table[-1] = -math.inf
    q, k, v = normal(15, sum(ql), nh, hd, dtype=dtype), normal(16, sum(kl), nkv, hd, dtype=dtype), normal(17, sum(kl), nkv, hd, dtype=dtype)
    k[:, -1, ::3], v[:, -1, ::2] = math.nan, math.inf
    out, lse = attend(q, k, v, ql, kl, scale=hd ** -0.5, table=table)
    assert bool((out[:, -1] == 0).all()) and bool((lse[:, -1] == -math.inf).all())


# ---- the parts of a split key axis under large biases -----------------------------------------------------
@pytest.mark.parametrize("dtype,nh,nkv,hd", HEADS)
@pytest.mark.parametrize("nq", [1, 3, 100, 330])
@pytest.mark.parametrize("bias", [torch.finfo(F32).min, -1e30, -1e6, -1e5, 3e4])
@pytest.mark.parametrize("docs", [False, True])
def test_parts_are_weighted_by_their_sums_under_any_bias(dtype, nh, nkv, hd, nq, bias, docs):
    """All scores equal: every visible key weighs the same, however few of them a part of the key axis holds and however large
    the bias is that all scores carry. Values rise along the keys, so that a part's wrong share shows."""
    ql, kl = [nq], [5003]
    q = torch.zeros(nq, nh, hd, dtype=dtype, device="cuda")
    k = normal(21, 5003, nkv, hd, dtype=dtype)
    v = (normal(22, 5003, nkv, hd) + torch.linspace(-2.0, 4.0, 5003).cuda()[:, None, None]).to(dtype)
    q_doc = k_doc = None
    if docs:  # visible: the first 40 keys, every 7th up to 3,000, all past 4,900
        j = torch.arange(5003)
        k_doc = ((j < 40) | ((j < 3000) & (j % 7 == 0)) | (j > 4900)).to(torch.int32).cuda()
        q_doc = torch.ones(nq, dtype=torch.int32, device="cuda")
    got = attend(q, k, v, ql, kl, table=torch.full((nh, 3), bias).cuda(), q_doc=q_doc, k_doc=k_doc)
    # The weights do not depend on the common bias (in 64 bits, too, the log-sum beside -1e30 would lose the sum).
    want, wlse, mag, _ = attention_64(q, k, v, ql, kl, q_doc=q_doc, k_doc=k_doc)
    out, lse = got
    rel = 2.0**-8 if dtype == BF16 else 2.0**-14  # bf16: the result's rounding; f32: a running sum of 5,003 terms
    assert bool(((out.double() - want).abs() <= rel * (mag + want.abs())).all())
    # bias and sum in units of log 2 and back: four roundings of 2^-24
    bias = max(bias, -1e30)
    assert bool(((lse.double() - (wlse + bias)).abs() <= 2.0**-22 * abs(bias) + 2.0**-18 * wlse.abs()).all())


@pytest.mark.parametrize("dtype,nh,nkv,hd", HEADS)
@pytest.mark.parametrize("ql,kl", [([390], [390]), ([3], [390]), ([3], [5003]), ([60], [4000]), ([200], [3000])])
def test_a_nan_counts_however_small_its_weight(dtype, nh, nkv, hd, ql, kl):
    """Scores so far apart that nearly all weights are zero in 32 bits: a row that sees a NaN in V is still NaN, in a masked tile, a part
    of the key axis or a warp whose weight has vanished as in any other."""
    q, k, v = normal(47, sum(ql), nh, hd, scale=2.0, dtype=dtype), normal(48, sum(kl), nkv, hd, dtype=dtype), normal(49, sum(kl), nkv, hd, dtype=dtype)
    n = kl[0]
    k_doc = (torch.arange(n) % 5 == 1).to(torch.int32).cuda()
    q_doc = torch.zeros(sum(ql), dtype=torch.int32, device="cuda")
    opt = dict(scale=100.0, causal=True, q_doc=q_doc, k_doc=k_doc)
    clean = attend(q, k, v, ql, kl, **opt)
    assert bool(torch.isfinite(clean[0]).all())
    place, _ = places(ql, kl)
    for key in (3, n // 2 // 5 * 5, (n - 2) // 5 * 5, 6):  # the last one is hidden
        bad = v.clone()
        bad[key] = math.nan
        out, lse = attend(q, k, bad, ql, kl, **opt)
        sees = place >= key if key != 6 else torch.zeros_like(place, dtype=torch.bool)
        assert torch.equal(lse, clean[1])
        assert bool(torch.isnan(out[sees]).all()) and torch.equal(out[~sees], clean[0][~sees])


# ---- 8-bit integers -------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("k", [1, 7, 64, 200, 777, 1000, 3000, 8192, 20_000])
@pytest.mark.parametrize("top", [1e-30, 3.8e-37, 3.7e-37, 1e-37, 1.2e-38, 1e-38, 1e-39, 2e-40])
def test_quantize_rows_of_the_smallest_numbers(dtype, k, top):
    """127 / top does not fit 32 bits below 3.73e-37. The numbers are the definition's all the same: zeros stay zero, the largest is
    127, and q * scale is within half a step of x and the rounding of the scale, half of 2^-149 where it is subnormal, 127 times."""
    x = normal(61, 5, k).clamp(-3, 3) * (top / 4)
    x[:, 0] = top
    x[1] *= -1.0
    x[2, 1:] = 0.0
    x[3, ::2] = 0.0
    x[4] = 0.0
    x = x.to(dtype)
    q, scale = ops.quantize_rows(x)
    y = x.double()
    most = y.abs().amax(1)
    np.testing.assert_array_equal(scale.cpu().numpy(), most.float().cpu().numpy() / np.float32(127.0))
    exact = y * (127.0 / most.clamp(min=1e-300))[:, None]
    # two roundings of 2^-24 each of a number of at most 127: nothing but a tie within 127 * 2^-22 may go the other way
    assert bool(((q.double() - exact).abs() <= 0.5 + 127 * 2.0**-22).all())
    assert bool((q[x == 0] == 0).all()) and bool((q.long().abs().amax(1)[most > 0] == 127).all())
    back = q.double() * scale.double()[:, None]
    assert bool(((back - y).abs() <= scale.double()[:, None] * (0.5 + 127 * 2.0**-22) + 127 * 2.0**-150 + most[:, None] * 2.0**-24).all())


def test_quantize_rows_of_a_row_of_the_most_columns():
    k = 2**31 - 1
    x = torch.zeros(1, k, dtype=BF16, device="cuda")
    x[0, 0], x[0, -1], x[0, -400], x[0, k // 2] = 2.0, -4.0, 1.0, 3.0
    q, scale = ops.quantize_rows(x)
    assert float(scale[0]) == float(np.float32(4.0) / np.float32(127.0))
    assert [int(q[0, c]) for c in (0, k - 1, k - 400, k // 2)] == [64, -127, 32, 95]  # 63.5 to even, 31.75, 95.25
    assert int((q != 0).sum()) == 4


@pytest.mark.parametrize("m,n", [(3, 2), (200, 70), (1800, 1600)])
@pytest.mark.parametrize("k", [ops.I8_MAX_K, ops.I8_MAX_K - 16])
def test_gemm_i8_sums_of_the_lowest_values(m, n, k):
    """-128 on both sides over the most columns allowed: 2^31 itself; and the other corners of the range."""
    a = torch.full((m, k), -128, dtype=torch.int8, device="cuda")
    w = torch.full((n, k), -128, dtype=torch.int8, device="cuda")
    a[1::3], a[2::3, -1] = 127, 0
    w[1::2] = 127
    one = torch.ones(max(m, n), device="cuda")
    got = ops.gemm_i8(a, one[:m], w, one[:n], out_dtype=F32)
    rows = [(-128, k), (127, k), (-128, k - 1)]  # value and count of a row's factors
    want = torch.tensor([[np.float32(va * c * vw) for vw in (-128, 127)] for va, c in rows]).cuda()
    assert torch.equal(got, want[torch.arange(m) % 3][:, torch.arange(n) % 2])


# ---- numbers that do not fit the C call ----------------------------------------------------------------------
@pytest.mark.parametrize("change", [dict(window=2**31), dict(window=-(2**40)), dict(scale=1e39), dict(softcap=1e300), dict(softcap=math.nan),
                                    dict(max_q=2**31), dict(max_k=2**40), dict(max_q=-1)])
def test_attention_refuses_numbers_that_do_not_fit(change):
    q = normal(71, 4, 2, 64, dtype=BF16)
    a = dict(max_q=4, max_k=4)
    a.update(change)
    with pytest.raises(L.Eg2Error):
        ops.attention_masked(q, q, q, offsets([4]), offsets([4]), a.pop("max_q"), a.pop("max_k"), **a)


# ---- graphs ------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("nq", [700, 2])
def test_the_calls_can_be_captured_in_a_graph(nq):
    """All of them in one graph, the attention's workspace among them (few queries split the key axis); replayed on other
    inputs it gives what the calls give."""
    nh, nkv, hd, nk = 4, 2, 128, 3000
    x = normal(81, nk, 512, dtype=BF16)
    w, ws = ops.quantize_rows(normal(82, (nh + 2 * nkv) * hd, 512, scale=512**-0.5))
    steps = torch.from_numpy(ops.rotary_steps(hd)[0].view(np.int64)).cuda()
    pos = torch.arange(nk, dtype=torch.int32).cuda()
    q_off, k_off = offsets([nq]), offsets([nk])

    def layer():
        qkv = ops.gemm_i8(*ops.quantize_rows(x), w, ws)
        q, k, v = (t.unflatten(1, (-1, hd)) for t in qkv.split([nh * hd, nkv * hd, nkv * hd], 1))
        q, k = ops.rotary(q, k, pos, steps)
        return ops.attention_masked(q[nk - nq :], k, v, q_off, k_off, nq, nk, scale=hd**-0.5, softcap=30.0, causal=True, return_lse=True)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        layer()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = layer()
    for seed in (83, 84):
        x.copy_(normal(seed, nk, 512, dtype=BF16))
        graph.replay()
        torch.cuda.synchronize()
        want = layer()
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    assert L.load().eg2_device_status() == 0


# ---- scales and caps at the ends of 32 bits -------------------------------------------------------------------------
@pytest.mark.parametrize("dtype,nh,nkv,hd", HEADS)
@pytest.mark.parametrize("nq", [3, 200])
def test_caps_and_scales_at_the_ends_of_the_type(dtype, nh, nkv, hd, nq):
    """A cap near the type's largest value caps nothing; one near its smallest leaves all scores equal; a score of zero is zero
    under any scale."""
    ql, kl = [nq], [333]
    q, k, v = normal(91, nq, nh, hd, dtype=dtype), normal(92, 333, nkv, hd, dtype=dtype), normal(93, 333, nkv, hd, dtype=dtype)
    scale = hd ** -0.5
    for softcap in (1e30, 2.3e38, torch.finfo(F32).max):
        check_attention(q, k, v, ql, kl, attend(q, k, v, ql, kl, scale=scale, softcap=softcap), scale=scale)
    zero = q.clone()
    zero[:, :, :] = 0.0
    for opt in (dict(scale=torch.finfo(F32).max), dict(scale=-3e38), dict(scale=3e38, softcap=2.0), dict(scale=1.0, softcap=1e-40)):
        check_attention(zero, k, v, ql, kl, attend(zero, k, v, ql, kl, **opt), scale=1.0)
    # every score is within 1e-38 of zero, whatever its sign
    got = attend(q, k, v, ql, kl, scale=scale, softcap=1e-40)
    check_attention(zero, k, v, ql, kl, got, scale=1.0)


def test_gemm_i8_of_one_row_from_a_buffer_of_any_stride():
    buf = torch.randint(-127, 128, (8, 1000), dtype=torch.int8, generator=torch.Generator().manual_seed(94)).cuda()
    w, ws = ops.quantize_rows(normal(95, 40, 777))
    one = torch.ones(1, device="cuda")
    for row in (0, 2, 4):  # 16-byte aligned
        a = buf[row : row + 1, :777]
        got = ops.gemm_i8(a, one, w, ws, out_dtype=F32)
        want = (a.double() @ w.double().T) * ws.double()
        assert bool(((got.double() - want).abs() <= 2.0**-22 * want.abs()).all())
        assert torch.equal(ops.gemm_i8(w, ws, a, one, out_dtype=F32).T, got)
