"""The layer operators (``ops``) against plain forms in 64 bits: rotary positions, masked attention and the
matrix product in 8-bit integers, at the sizes, strides and masks where they can go wrong."""
import math

import numpy as np
import pytest

from conftest import pkg

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu

L = pkg("lib")
ops = pkg("ops")
BF16, F32 = torch.bfloat16, torch.float32


def normal(seed, *shape, scale=1.0, dtype=F32):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=g) * scale).to(dtype).cuda()


# ---- rotary -------------------------------------------------------------------------------------------
def rotary_64(x, pos, steps, layout, rot, m, inverse):
    """From whole numbers: the phase modulo 2^64 exactly, then double precision."""
    phase = np.array([[(int(p) * int(s)) % 2**64 for s in steps] for p in pos], dtype=np.float64).reshape(len(pos), -1)
    t = torch.from_numpy(phase * 2.0**-64 * 2 * math.pi).cuda()
    c, s = (m * torch.cos(t))[:, None], (m * torch.sin(t))[:, None] * (-1 if inverse else 1)
    y = x.double().clone()
    a, b = (y[..., : rot // 2], y[..., rot // 2 : rot]) if layout == "half" else (y[..., 0:rot:2], y[..., 1:rot:2])
    u, v = a * c - b * s, b * c + a * s
    if layout == "half":
        y[..., : rot // 2], y[..., rot // 2 : rot] = u, v
    else:
        y[..., 0:rot:2], y[..., 1:rot:2] = u, v
    return y


def rotary_tolerance(x, want, m):
    """The angle is good to 2^-23 of itself (its f32 form, at most pi) plus the cosine's 2^-22, the products and
    their sum to 2^-23 of m (|a| + |b|): 16 * 2^-23 m max|x| covers all; then one rounding of the result."""
    unit = 2.0**-8 if x.dtype == BF16 else 2.0**-24  # half a unit in the last of 8 or 24 bits
    return 16 * 2.0**-23 * m * float(x.double().abs().max()) + unit * want.abs()


def steps_for(rot, scaling="none", factor=4.0):
    steps, m = ops.rotary_steps(rot, 10000.0, scaling, factor, 4096)
    return steps, torch.from_numpy(steps.view(np.int64)).cuda(), m


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("hd,rot", [(64, 64), (256, 256), (512, 512), (80, 80), (96, 48), (64, 2), (64, 34), (50, 30), (7, 4)])
@pytest.mark.parametrize("rows,nh,nkv", [(1, 4, 2), (37, 3, 1), (37, 5, 0)])
def test_rotary(dtype, layout, hd, rot, rows, nh, nkv):
    q = normal(1, rows, nh, hd, dtype=dtype)
    k = normal(2, rows, nkv, hd, dtype=dtype) if nkv else None
    # Positions from the first to the ends of the type, negative ones among them.
    pos = np.array([0, 1, 2**31 - 1, -(2**31), -1, 131071, 999_999, 5], np.int64)
    pos = np.resize(pos, rows)
    steps, dev, m = steps_for(rot, "yarn")
    p = torch.from_numpy(pos.astype(np.int32)).cuda()
    for inverse in (False, True):
        got = ops.rotary(q, k, p, dev, layout=layout, rot_dim=rot, magnitude=m, inverse=inverse)
        for x, y in zip((q, k), got):
            if x is None:
                assert y is None
                continue
            want = rotary_64(x, pos, steps, layout, rot, m, inverse)
            assert y.dtype == dtype and y.shape == x.shape
            assert bool(((y.double() - want).abs() <= rotary_tolerance(x, want, m)).all())
            assert torch.equal(y[..., rot:], x[..., rot:])


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("shift", [0, 1])
def test_rotary_strided_and_in_place(dtype, layout, shift):
    """q and k inside rows of a fused projection, at an even or odd element of the buffer, rotated in place: the
    same bits as from copies, and nothing else touched."""
    rows, nh, nkv, hd = 33, 4, 2, 128
    width = (nh + 2 * nkv) * hd + 2 * shift
    flat = normal(3, rows * width + 16, dtype=dtype)
    fused = flat[shift : shift + rows * width].view(rows, width)
    before = flat.clone()
    q, k = fused[:, : nh * hd].unflatten(1, (nh, hd)), fused[:, nh * hd : (nh + nkv) * hd].unflatten(1, (nkv, hd))
    steps, dev, m = steps_for(hd)
    pos = torch.arange(rows, dtype=torch.int32).cuda() * 1000
    want_q, want_k = ops.rotary(q.contiguous(), k.contiguous(), pos, dev, layout=layout)
    got_q, got_k = ops.rotary(q, k, pos, dev, layout=layout)
    assert torch.equal(got_q, want_q) and torch.equal(got_k, want_k)
    assert torch.equal(flat, before)
    ops.rotary(q, k, pos, dev, layout=layout, out=(q, k))
    assert torch.equal(q, want_q) and torch.equal(k, want_k)
    rest = torch.ones(rows, width, dtype=torch.bool)
    rest[:, : (nh + nkv) * hd] = False
    old = before[shift : shift + rows * width].view(rows, width)
    assert torch.equal(fused[rest.cuda()], old[rest.cuda()])


@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_rotary_inverse_is_the_gradient(layout):
    """The rotation is linear, so <R x, y> = <x, R^T y>, and (R(x + h e) - R(x)) / h is R's column whatever h."""
    rows, nh, hd, rot = 9, 2, 96, 64
    x, y = normal(4, rows, nh, hd), normal(5, rows, nh, hd)
    pos = torch.arange(rows, dtype=torch.int32).cuda() * 777
    _, dev, m = steps_for(rot, "yarn")
    call = lambda t, inv=False: ops.rotary(t, None, pos, dev, layout=layout, rot_dim=rot, magnitude=m, inverse=inv)[0].double()
    left, right = (call(x) * y.double()).sum(), (x.double() * call(y, True)).sum()
    # 2 n terms of size about 1, each off by at most 16 * 2^-23 m: the sum of absolute errors bounds the difference.
    assert abs(float(left - right)) <= 32 * 2.0**-23 * m * float((x.abs() * 4 * y.abs().amax()).sum())
    grad = call(y, True)
    for r, h, c in [(0, 0, 0), (3, 1, 5), (8, 0, 63), (8, 1, 64), (4, 1, 95)]:
        e = torch.zeros_like(x)
        e[r, h, c] = 1.0  # differences of a linear map with step 1: no truncation error
        diff = float(((call(x + e) - call(x)) * y.double()).sum())
        # each of the two touched outputs is off by at most 2 * 16 * 2^-23 m max|x + e|, times |y|
        tol = 64 * 2.0**-23 * m * float((x.abs().max() + 1) * y.abs().max()) * 2
        assert abs(diff - float(grad[r, h, c])) <= tol


def test_rotary_wide_buffers():
    """Rows 600 MB apart: offsets beyond 32 bits."""
    hd, rows = 64, 9
    ld = 300_000_000
    flat = torch.zeros((rows - 1) * ld + 2 * hd, dtype=BF16, device="cuda")
    q = flat.as_strided((rows, 2, hd), (ld, hd, 1))
    q.copy_(normal(6, rows, 2, hd, dtype=BF16))
    steps, dev, m = steps_for(hd)
    pos = torch.arange(rows, dtype=torch.int32).cuda()
    got, _ = ops.rotary(q, None, pos, dev)
    want = rotary_64(q, range(rows), steps, "half", hd, m, False)
    assert bool(((got.double() - want).abs() <= rotary_tolerance(q, want, m)).all())


# ---- attention -----------------------------------------------------------------------------------------
def attention_64(q, k, v, ql, kl, *, scale=1.0, softcap=0.0, window=-1, causal=False, prefix=None, q_doc=None, k_doc=None,
                 slopes=None, table=None):
    """(out, lse, sum_j p_j |v_j|, the largest scale * sum_d |q_d k_d|) in double precision."""
    nh, hd, nkv = q.shape[1], q.shape[2], k.shape[1]
    out = torch.zeros(q.shape, dtype=torch.float64, device="cuda")
    mag = torch.zeros_like(out)
    lse = torch.full(q.shape[:2], -math.inf, dtype=torch.float64, device="cuda")
    big, q0, k0 = 0.0, 0, 0
    for b, (nq, nk) in enumerate(zip(ql, kl)):
        i = torch.arange(nk - nq, nk, device="cuda")[:, None]
        j = torch.arange(nk, device="cuda")[None]
        seen = torch.ones(nq, nk, dtype=torch.bool, device="cuda")
        if window >= 0:
            seen &= (i - j).abs() <= window
        if causal:
            seen &= (j <= i) | (j < (prefix[b] if prefix is not None else 0))
        if q_doc is not None:
            seen &= q_doc[q0 : q0 + nq][:, None] == k_doc[k0 : k0 + nk][None]
        for h in range(nh):
            if nq == 0 or nk == 0:
                continue
            g = h // (nh // nkv)
            qq, kk, vv = q[q0 : q0 + nq, h].double(), k[k0 : k0 + nk, g].double(), v[k0 : k0 + nk, g].double()
            used = seen.any(0)
            kk, vv = torch.where(used[:, None], kk, 0.0), torch.where(used[:, None], vv, 0.0)
            big = max(big, float((qq.abs() @ kk.abs().T).max()) * abs(scale))
            x = qq @ kk.T * scale
            if softcap:
                x = softcap * torch.tanh(x / softcap)
            if slopes is not None:
                x = x - float(slopes[h]) * (j - i).abs()
            if table is not None:
                R = table.shape[1] // 2
                x = x + table[h].double()[(j - i).clamp(-R, R) + R]
            x = torch.where(seen, x, -math.inf)
            z = torch.logsumexp(x, 1)
            p = torch.where(seen, torch.exp(x - z[:, None]), 0.0)
            lse[q0 : q0 + nq, h] = z
            out[q0 : q0 + nq, h] = p @ vv
            mag[q0 : q0 + nq, h] = p @ vv.abs()
        q0, k0 = q0 + nq, k0 + nk
    return out, lse, mag, big


def offsets(lens):
    return torch.tensor(np.cumsum([0] + list(lens)), dtype=torch.int32).cuda()


def check_attention(q, k, v, ql, kl, got, **opt):
    """|out - want| against the errors the operator's arithmetic allows.

    A score is off by at most d = (hd + 16) 2^-24 (sum_d |q_d k_d| scale) from the f32 sum and, with a bias, the
    rounding of scores of up to a few hundred (2^-24 * 512); a capped bf16 score by a further 2^-13 (its tanh, in
    units of the cap). Weights are then off by 2 d relatively, bf16 ones by another 2^-8 for their rounding before
    the product with v; the result by the rounding of its type. The log-sum is off by d and 2^-20."""
    out, lse = got
    want, wlse, mag, big = attention_64(q, k, v, ql, kl, **opt)
    bf = q.dtype == BF16
    d = (q.shape[2] + 16) * 2.0**-24 * big
    if opt.get("slopes") is not None or opt.get("table") is not None:
        d += 2.0**-15
    if bf and opt.get("softcap"):
        d += 2.0**-13
    rel = 2 * d + (2.0**-8 if bf else 2.0**-18)
    n = sum(ql)
    assert out.dtype == q.dtype and not bool(torch.isnan(out[:n]).any())
    err = (out[:n].double() - want[:n]).abs()
    tol = rel * mag[:n] + (2.0**-8 if bf else 2.0**-23) * want[:n].abs() + 1e-30
    assert bool((err <= tol).all()), float((err / tol).max())
    live = torch.isfinite(wlse[:n])
    assert torch.equal(lse[:n] == -math.inf, ~live)
    assert bool(((lse[:n].double() - wlse[:n]).abs()[live] <= d + 2.0**-18 * wlse[:n].abs()[live] + 2.0**-18).all())


def attend(q, k, v, ql, kl, *, prefix=None, table=None, **opt):
    return ops.attention_masked(q, k, v, offsets(ql), offsets(kl), max(ql), max(kl), return_lse=True,
                                prefix_len=None if prefix is None else torch.tensor(prefix, dtype=torch.int32).cuda(),
                                dist_bias=table, **opt)


def run_case(dtype, nh, nkv, hd, ql, kl, seed=7, **opt):
    q, k, v = normal(seed, sum(ql), nh, hd, scale=2.0, dtype=dtype), normal(seed + 1, sum(kl), nkv, hd, dtype=dtype), \
        normal(seed + 2, sum(kl), nkv, hd, dtype=dtype)
    opt.setdefault("scale", hd ** -0.5)
    check_attention(q, k, v, ql, kl, attend(q, k, v, ql, kl, **opt), **opt)


HEADS = [(BF16, 4, 2, 64), (BF16, 2, 1, 128), (BF16, 4, 2, 256), (BF16, 4, 1, 512), (BF16, 3, 1, 128), (BF16, 2, 2, 64),
         (BF16, 3, 3, 80), (BF16, 6, 2, 50), (F32, 4, 2, 64), (F32, 3, 1, 80), (F32, 4, 1, 256), (F32, 2, 1, 512), (F32, 2, 2, 7)]


@pytest.mark.parametrize("dtype,nh,nkv,hd", HEADS)
@pytest.mark.parametrize("softcap", [0.0, 5.0, 30.0])
def test_attention_lengths(dtype, nh, nkv, hd, softcap):
    """Lengths around the tiles' edges, one and none among them."""
    run_case(dtype, nh, nkv, hd, [1, 2, 0, 63, 64, 65, 127, 128, 129, 300], [1, 2, 0, 63, 64, 65, 127, 128, 129, 300],
             softcap=softcap)


@pytest.mark.parametrize("dtype,nh,nkv,hd", HEADS)
@pytest.mark.parametrize("window,causal,prefix", [(0, False, False), (7, False, False), (200, False, False), (-1, True, False),
                                                  (-1, True, True), (50, True, True), (2**31 - 1, False, False)])
def test_attention_windows_and_prefixes(dtype, nh, nkv, hd, window, causal, prefix):
    lens = [1, 70, 257, 390]
    run_case(dtype, nh, nkv, hd, lens, lens, window=window, causal=causal, prefix=[0, 70, 100, 500] if prefix else None)


@pytest.mark.parametrize("dtype,nh,nkv,hd", HEADS)
@pytest.mark.parametrize("ordered", [True, False])
def test_attention_documents(dtype, nh, nkv, hd, ordered):
    """Documents in order and scattered; a query whose document has no key, keys that no query wants."""
    lens = [5, 200, 410]
    rng = np.random.default_rng(3)
    doc = np.concatenate([np.sort(rng.integers(-3, 9, n)) if ordered else rng.integers(-3, 4, n) for n in lens])
    k_doc = torch.tensor(doc, dtype=torch.int32).cuda()
    q_doc = k_doc.clone()
    q_doc[[2, 100, 300]] = 77
    q_doc[205:340] = 78 if not ordered else q_doc[205:340]
    run_case(dtype, nh, nkv, hd, lens, lens, q_doc=q_doc, k_doc=k_doc, window=150)


@pytest.mark.parametrize("dtype,nh,nkv,hd", HEADS)
@pytest.mark.parametrize("softcap", [0.0, 20.0])
@pytest.mark.parametrize("bias", ["slopes", "table 0", "table 9", "table 200", "table 1024", "both"])
def test_attention_biases(dtype, nh, nkv, hd, softcap, bias):
    lens = [3, 130, 420]
    slopes = table = None
    if bias in ("slopes", "both"):
        slopes = torch.tensor([0.5 ** (h + 1) for h in range(nh)]).cuda()
    if bias != "slopes":
        R = 9 if bias == "both" else int(bias.split()[1])
        table = normal(11, nh, 2 * R + 1, scale=2.0)
    run_case(dtype, nh, nkv, hd, lens, lens, softcap=softcap, slopes=slopes, table=table, causal=bias == "both")


@pytest.mark.parametrize("dtype,nh,nkv,hd", HEADS)
@pytest.mark.parametrize("nq", [1, 3, 17])
@pytest.mark.parametrize("causal", [False, True])
def test_attention_few_queries_over_many_keys(dtype, nh, nkv, hd, nq, causal):
    """The form for single tokens: the key axis may be split; more queries than keys in one sequence."""
    slopes = torch.tensor([2.0 ** -(h + 3) for h in range(nh)]).cuda()
    run_case(dtype, nh, nkv, hd, [nq, nq, 0, nq], [3000, 2, 5, 1111], causal=causal, softcap=15.0, slopes=slopes)
    run_case(dtype, nh, nkv, hd, [nq], [5003], causal=causal, window=700)


@pytest.mark.parametrize("dtype,nh,nkv,hd", HEADS)
@pytest.mark.parametrize("nq", [100, 330])
@pytest.mark.parametrize("docs", [False, True])
def test_attention_split_over_many_rows(dtype, nh, nkv, hd, nq, docs):
    """Hundreds of queries over a split key axis: parts without a key of a row's, rows without any key."""
    ql, kl, q_doc, k_doc = [nq, 0, 5], [4000, 3, 40], None, None
    if docs:
        k_doc = (torch.arange(sum(kl), dtype=torch.int32) // 600).cuda()
        q_doc = (torch.arange(sum(ql), dtype=torch.int32) % 9).cuda()
    run_case(dtype, nh, nkv, hd, ql, kl, softcap=20.0, q_doc=q_doc, k_doc=k_doc)
    run_case(dtype, nh, nkv, hd, ql, kl, causal=True, window=900, q_doc=q_doc, k_doc=k_doc)


@pytest.mark.parametrize("dtype,nh,nkv,hd", HEADS)
@pytest.mark.parametrize("few", [False, True])
def test_hidden_keys_may_hold_anything(dtype, nh, nkv, hd, few):
    """NaN and infinities in keys and values that the masks hide -- rows between sequences, other documents, keys
    outside the window, ahead of a causal query -- reach nothing; a row that sees one is not finite."""
    kl = [150, 333]
    ql = [2, 3] if few else kl
    q = normal(21, sum(ql), nh, hd, scale=2.0, dtype=dtype)
    k, v = normal(22, sum(kl) + 90, nkv, hd, dtype=dtype), normal(23, sum(kl) + 90, nkv, hd, dtype=dtype)
    for t in (k, v):  # 90 rows of no sequence after the two
        t[sum(kl) :] = math.nan
    gap = 40  # the second sequence's first keys belong to a document that no query asks for
    k_doc = torch.zeros(sum(kl) + 90, dtype=torch.int32).cuda()
    k_doc[150 : 150 + gap] = 5
    q_doc = torch.zeros(sum(ql), dtype=torch.int32).cuda()
    k[150 : 150 + gap : 2] = math.inf
    v[150 : 150 + gap : 3] = -math.inf
    v[151 : 150 + gap : 3] = math.nan
    opt = dict(scale=hd ** -0.5, q_doc=q_doc, k_doc=k_doc[: sum(kl)])
    got = ops.attention_masked(q, k, v, offsets(ql), offsets(kl), max(ql), max(kl), return_lse=True, scale=opt["scale"],
                               q_doc=q_doc, k_doc=k_doc)
    check_attention(q, k[: sum(kl)], v[: sum(kl)], ql, kl, got, **opt)
    # Causal: the last key's value is NaN. Only the last query of the sequence sees it.
    v2 = normal(24, sum(kl), nkv, hd, dtype=dtype)
    clean = attend(q, k[: sum(kl)], v2, ql, kl, causal=True, **opt)
    v2[149] = math.nan
    out, lse = attend(q, k[: sum(kl)], v2, ql, kl, causal=True, **opt)
    last = ql[0] - 1
    rest = torch.arange(sum(ql), device="cuda") != last
    assert not bool(torch.isfinite(out[last]).any())
    assert torch.equal(out[rest], clean[0][rest]) and torch.equal(lse[rest], clean[1][rest])


@pytest.mark.parametrize("dtype,nh,nkv,hd", [(BF16, 4, 2, 128), (BF16, 4, 1, 512), (F32, 4, 2, 64)])
def test_scores_at_the_ends_of_the_range(dtype, nh, nkv, hd):
    """Very large scores and biases: one weight is all, nothing overflows; a bias of the type's lowest value."""
    lens = [140]
    q, k, v = (normal(s, 140, n, hd, dtype=dtype) for s, n in ((31, nh), (32, nkv), (33, nkv)))
    for scale in (1e4, -1e4):
        out, lse = attend(q, k, v, lens, lens, scale=scale)
        assert bool(torch.isfinite(out).all()) and bool(torch.isfinite(lse).all())
    out, lse = attend(q, k, v, lens, lens, scale=1e4, softcap=50.0)
    want, wlse, _, _ = attention_64(q, k, v, lens, lens, scale=1e4, softcap=50.0)
    # scores of +-50 up to 2^-13 of tanh units: weights off by 2^-12 and bf16's 2^-8, in f32 by 50 * 2^-21
    tol = 2.0**-7 if dtype == BF16 else 2.0**-12
    assert bool(((out.double() - want).abs() <= tol * (1 + want.abs())).all())
    table = torch.full((nh, 3), torch.finfo(F32).min).cuda()
    table[:, 1] = 0.0
    out, _ = attend(q, k, v, lens, lens, table=table)
    own = v.repeat_interleave(nh // nkv, 1)
    assert torch.equal(out, own)  # each row is left with itself


def test_attention_strides_slices_and_streams():
    """q, k, v inside fused rows, a strided out, rows of no sequence untouched, on a stream of its own; unaligned
    buffers give the same within the operator's errors."""
    nh, nkv, hd = 4, 2, 128
    ql = [33, 0, 200]
    rows = sum(ql) + 7
    for shift in (0, 1):
        width = (nh + 2 * nkv) * hd
        flat = normal(41, rows * width + 8, dtype=BF16)
        fused = flat[shift : shift + rows * width].view(rows, width)
        q, k, v = (fused[:, a * hd : b * hd].unflatten(1, (b - a, hd)) for a, b in ((0, nh), (nh, nh + nkv), (nh + nkv, nh + 2 * nkv)))
        out = torch.full((rows, 2 * nh * hd), 3.0, dtype=BF16, device="cuda")
        view = out[:, nh * hd :].unflatten(1, (nh, hd))
        off = offsets(ql)
        st = torch.cuda.Stream()
        st.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(st):
            got, lse = ops.attention_masked(q, k, v, off, off, 200, 200, scale=hd ** -0.5, out=view, return_lse=True)
        torch.cuda.current_stream().wait_stream(st)
        n = sum(ql)
        check_attention(q[:n], k[:n], v[:n], ql, ql, (got[:n], lse[:n]), scale=hd ** -0.5)
        assert bool((out[:, : nh * hd] == 3.0).all()) and bool((out[n:] == 3.0).all())


def test_attention_twice_gives_the_same_bits():
    for nq in (1, 300):
        ql, kl = [nq, nq], [4000, 300]
        q, k, v = normal(51, 2 * nq, 4, 128, dtype=BF16), normal(52, 4300, 2, 128, dtype=BF16), normal(53, 4300, 2, 128, dtype=BF16)
        a, b = (attend(q, k, v, ql, kl, softcap=30.0, causal=True) for _ in range(2))
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    assert L.load().eg2_device_status() == 0


def test_attention_offsets_beyond_the_buffers_stay_inside():
    """Offsets are device data the host cannot check: lengths are cut to the buffers and to max_q / max_k."""
    q, k, v = (normal(s, 50, 2, 64, dtype=BF16) for s in (61, 62, 63))
    off = torch.tensor([0, 1000], dtype=torch.int32).cuda()
    a = ops.attention_masked(q, k, v, off, off, 50, 50)
    b = ops.attention_masked(q, k, v, offsets([50]), offsets([50]), 50, 50)
    assert torch.equal(a, b)
    ops.attention_masked(q, k, v, -off, off.flip(0).contiguous(), 50, 50)
    torch.cuda.synchronize()


# ---- 8-bit integers ---------------------------------------------------------------------------------------
def quantize_plain(x):
    """The definition in f32, operation for operation (each is one IEEE rounding)."""
    x = x.float().cpu().numpy()
    top = np.abs(x).max(1).astype(np.float32)
    with np.errstate(divide="ignore"):
        inv = np.where(top > 0, np.float32(127.0) / top, np.float32(0.0)).astype(np.float32)
    return np.rint(x * inv[:, None]).astype(np.int8), (top / np.float32(127.0)).astype(np.float32)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("rows,k", [(1, 1), (3, 7), (17, 512), (5, 777), (2, 8192), (33, 96), (1, 100_000), (300, 4)])
def test_quantize_rows(dtype, rows, k):
    x = normal(71, rows, k, dtype=dtype)
    x[0, 0] = 0.0
    if rows > 2:
        x[1] = 0.0
        x[2] *= 1e30
    q, scale = ops.quantize_rows(x)
    want_q, want_s = quantize_plain(x)
    np.testing.assert_array_equal(q.cpu().numpy(), want_q)
    np.testing.assert_array_equal(scale.cpu().numpy(), want_s)
    assert q.stride(0) % 16 == 0 and q.data_ptr() % 16 == 0


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_quantize_rows_strides_and_values_without_a_scale(dtype):
    flat = normal(72, 9 * 131 + 1, dtype=dtype)
    x = flat[1:].view(9, 131)[:, :130]
    q, scale = ops.quantize_rows(x)
    want_q, want_s = quantize_plain(x)
    np.testing.assert_array_equal(q.cpu().numpy(), want_q)
    np.testing.assert_array_equal(scale.cpu().numpy(), want_s)
    y = normal(73, 4, 64, dtype=dtype)
    y[1, 3], y[2, 5], y[3, 6] = math.nan, math.inf, -math.inf
    q, scale = ops.quantize_rows(y)
    assert bool(torch.isnan(scale[1:]).all()) and bool((q[1:] == 0).all()) and bool(torch.isfinite(scale[0]))
    w, ws = ops.quantize_rows(normal(74, 5, 64))
    out = ops.gemm_i8(q, scale, w, ws)
    assert bool(torch.isnan(out[1:]).all()) and bool(torch.isfinite(out[0]).all())


def ints(seed, *shape):
    g = torch.Generator().manual_seed(seed)
    rows, k = shape
    buf = torch.full((rows, (k + 15) // 16 * 16 + 16), 99, dtype=torch.int8)
    buf[:, :k] = torch.randint(-128, 128, shape, generator=g, dtype=torch.int8)
    return buf.cuda()[:, :k]  # what lies past column k must not matter


def check_gemm(a, w, bias, out_dtype, got, a_scale, w_scale):
    s = a.double() @ w.double().T  # exact: below 2^53
    want = s * a_scale.double()[:, None] * w_scale.double()
    mag = want.abs()
    if bias is not None:
        want = want + bias.double()
        mag = mag + bias.double().abs()
    # the sum's rounding to f32, two products and the bias: 4 roundings of 2^-24; then the result's own
    tol = 4 * 2.0**-24 * mag + (2.0**-8 * want.abs() if out_dtype == BF16 else 0.0) + 1e-38
    assert got.dtype == out_dtype
    assert bool(((got.double() - want).abs() <= tol).all())


@pytest.mark.parametrize("m", [1, 2, 7, 8, 9, 17, 64, 65, 129, 300])
@pytest.mark.parametrize("n,k", [(1, 1), (5, 16), (64, 33), (100, 512), (257, 777), (513, 128), (1000, 2100)])
@pytest.mark.parametrize("out_dtype", [BF16, F32])
def test_gemm_i8(m, n, k, out_dtype):
    a, w = ints(81, m, k), ints(82, n, k)
    sa, sw = normal(83, m).abs() + 0.1, normal(84, n).abs() + 0.1
    for bias in (None, normal(85, n)):
        check_gemm(a, w, bias, out_dtype, ops.gemm_i8(a, sa, w, sw, bias=bias, out_dtype=out_dtype), sa, sw)


@pytest.mark.parametrize("m,n,k", [(1000, 768, 512), (777, 2048, 1111), (4500, 300, 64), (600, 5000, 256)])
def test_gemm_i8_large(m, n, k):
    a, w = ints(86, m, k), ints(87, n, k)
    sa, sw, bias = normal(88, m).abs() + 0.1, normal(89, n).abs() + 0.1, normal(90, n)
    for dt in (BF16, F32):
        check_gemm(a, w, bias, dt, ops.gemm_i8(a, sa, w, sw, bias=bias, out_dtype=dt), sa, sw)


@pytest.mark.parametrize("m", [3, 200])
def test_gemm_i8_sums_at_their_largest(m):
    """All factors -128 or 127 over the most columns allowed: the sums come within 2 % of 2^31, and stay exact."""
    k = ops.I8_MAX_K
    a = torch.full((m, k), 127, dtype=torch.int8, device="cuda")
    w = torch.full((2, k), 127, dtype=torch.int8, device="cuda")
    w[1] = -127
    one = torch.ones(max(m, 2), device="cuda")
    got = ops.gemm_i8(a, one[:m], w, one[:2], out_dtype=F32)
    total = 127 * 127 * k
    want = torch.tensor([np.float32(total), -np.float32(total)]).cuda().expand(m, 2)
    assert torch.equal(got, want)


@pytest.mark.parametrize("m", [5, 150])
def test_gemm_i8_into_a_slice(m):
    n, k = 70, 48
    a, w = ints(91, m, k), ints(92, n, k)
    sa, sw = normal(93, m).abs(), normal(94, n).abs()
    for dt in (BF16, F32):
        whole = torch.full((m + 2, n + 9), 5.0, dtype=dt, device="cuda")
        view = whole[1 : m + 1, 3 : 3 + n]
        got = ops.gemm_i8(a, sa, w, sw, out=view)
        assert got.data_ptr() == view.data_ptr()
        check_gemm(a, w, None, dt, got, sa, sw)
        rest = torch.ones_like(whole, dtype=torch.bool)
        rest[1 : m + 1, 3 : 3 + n] = False
        assert bool((whole[rest] == 5.0).all())


def test_int8_linear_is_near_the_real_product():
    """Quantised rows times quantised weights: within the sum of half steps of the exact product."""
    x, w = normal(95, 40, 512, dtype=BF16), normal(96, 96, 512)
    q, s = ops.quantize_rows(x)
    wq, ws = ops.quantize_rows(w)
    got = ops.gemm_i8(q, s, wq, ws, out_dtype=F32).double()
    want = x.double() @ w.double().T
    # |x w - x' w'| <= |x - x'| |w| + |x'| |w - w'|, each off by at most half a step (and 2^-20 of it)
    half = 0.5 * (1 + 2.0**-20)
    tol = half * s.double()[:, None] * w.double().abs().sum(1) + half * ws.double() * (q.double() * s.double()[:, None]).abs().sum(1)[:, None]
    assert bool(((got - want).abs() <= tol + 1e-4).all())


def test_empty_inputs():
    assert ops.quantize_rows(torch.zeros(0, 8, device="cuda"))[0].shape == (0, 8)
    w, ws = ops.quantize_rows(normal(97, 5, 16))
    assert ops.gemm_i8(torch.zeros(0, 16, dtype=torch.int8, device="cuda"), torch.zeros(0, device="cuda"), w, ws).shape == (0, 5)
    off = torch.zeros(1, dtype=torch.int32, device="cuda")
    q = torch.zeros(0, 2, 64, dtype=BF16, device="cuda")
    assert ops.attention_masked(q, q, q, off, off, 0, 0).shape == (0, 2, 64)
    # keys only; queries without keys
    off2, off0 = torch.tensor([0, 3], dtype=torch.int32).cuda(), torch.tensor([0, 0], dtype=torch.int32).cuda()
    k = normal(98, 3, 2, 64, dtype=BF16)
    out, lse = ops.attention_masked(k, q, q, off2, off0, 3, 0, return_lse=True)
    assert bool((out == 0).all()) and bool((lse == -math.inf).all())
    assert ops.rotary(q, None, torch.zeros(0, dtype=torch.int32, device="cuda"), torch.zeros(32, dtype=torch.int64, device="cuda"))[0].shape == q.shape


# ---- together ------------------------------------------------------------------------------------------------
def test_example_layer_is_near_its_32_bit_form():
    """The example's encoder layer (all operators in one pass) against its plain 32-bit form: 8-bit weights and
    activations are off by up to half a step in 127 of each row's largest value, about 1 % of the typical one (rows of
    512 normal values: the largest is near 3.5, half a step 0.014), so a product is off by about sqrt(2) * 0.8 % of its
    norm; four products in a row and bf16 activations stay within 5 %."""
    import importlib.util
    from pathlib import Path

    spec = importlib.util.spec_from_file_location("encoder_layer_int8", Path(__file__).parents[1] / "examples" / "encoder_layer_int8.py")
    ex = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(ex)
    for scaling, factor in (("none", 1.0), ("yarn", 4.0)):
        layer = ex.EncoderLayer8(seed=3, window=100, scaling=scaling, factor=factor, original_len=256)
        x = normal(99, 700, 512, dtype=BF16)
        pos, doc, off = ex.packed(700, 300)
        got, want = layer(x, pos, doc, off, 700).float(), layer.in_32_bits(x, pos, doc)
        assert float((got - want).norm() / want.norm()) < 0.05
        cos = torch.nn.functional.cosine_similarity(got, want, 1)
        assert float(cos.min()) > 0.995
