"""The layer operators' host side, without a GPU: rotary frequencies against their definition, and every
refusal that is decided before a launch (no pointer below is ever read)."""
import ctypes as C
import math

import numpy as np
import pytest

from conftest import pkg

L = pkg("lib")
torch = pytest.importorskip("torch")
ops = pkg("ops")


def definition(rot, theta, scaling, factor, original):
    if scaling == "ntk":
        theta = theta * factor ** (rot / max(1, rot - 2))
    f = np.array([theta ** (-2.0 * i / rot) for i in range(rot // 2)])
    m = 1.0
    if scaling == "linear":
        f = f / factor
    if scaling == "yarn":
        pair = lambda turns: rot * math.log(original / (turns * 2 * math.pi)) / (2 * math.log(theta))
        lo, hi = max(0, math.floor(pair(32))), min(rot - 1, math.ceil(pair(1)))
        r = np.clip((np.arange(rot // 2) - lo) / max(hi - lo, 0.001), 0, 1)
        f = f * (1 - r) + f / factor * r
        m = 0.1 * math.log(factor) + 1
    return f, m


@pytest.mark.parametrize("scaling", ["none", "linear", "ntk", "yarn"])
@pytest.mark.parametrize("rot", [2, 6, 64, 80, 512])
@pytest.mark.parametrize("theta,factor", [(10000.0, 1.0), (10000.0, 8.0), (1e6, 32.0)])
def test_rotary_steps_follow_the_definition(scaling, rot, theta, factor):
    steps, m = ops.rotary_steps(rot, theta, scaling, factor, 4096)
    f, want_m = definition(rot, theta, scaling, factor, 4096.0)
    # pow differs by a few units of 2^-53; the fixed-point grid is 2^-64 of a turn.
    got = steps.astype(np.float64) * 2.0**-64 * 2 * math.pi
    assert np.all(np.abs(got - f) <= 1e-14 * f + 2.0**-62)
    assert abs(m - want_m) <= 2.0**-23 * want_m


def test_rotary_steps_refusals():
    for args in [(0,), (3,), (-2,), (64, 1.0), (64, math.nan), (64, math.inf), (64, 1e4, "linear", 0.5),
                 (64, 1e4, "ntk", math.nan), (64, 1e4, "yarn", 4.0, 0.0), (64, 1e4, "stretch")]:
        with pytest.raises(L.Eg2Error):
            ops.rotary_steps(*args)


FAKE = 4096  # never read: each call below is refused before a launch


def rotary_rc(**change):
    a = dict(kind=L.EG2_BF16, layout=0, inverse=0, q=FAKE, ldq=512, nh=2, k=FAKE, ldk=256, nkv=1, qo=FAKE, ldqo=512, ko=FAKE,
             ldko=256, pos=FAKE, rows=4, hd=256, rot=256, steps=FAKE, m=1.0)
    a.update(change)
    return L.load().eg2_rotary(*a.values(), None)


@pytest.mark.parametrize("change", [dict(kind=1), dict(kind=9), dict(layout=2), dict(layout=-1), dict(rows=-1), dict(nh=-1),
                                    dict(nh=0, nkv=0), dict(hd=0), dict(rot=0), dict(rot=3), dict(rot=258), dict(ldq=511),
                                    dict(ldk=255), dict(ldqo=511), dict(ldko=255), dict(q=0), dict(qo=0), dict(k=0),
                                    dict(ko=0), dict(pos=0), dict(steps=0), dict(rows=1 << 50)])
def test_rotary_refuses(change):
    assert rotary_rc(**change) == -1


def masked(**change):
    a = dict(kind=L.EG2_BF16, q=FAKE, k=FAKE, v=FAKE, out=FAKE, lse=0, ldq=512, ldk=256, ldv=256, ldo=512, q_off=FAKE, k_off=FAKE,
             q_rows=8, k_rows=8, n_seq=1, max_q=8, max_k=8, nh=4, nkv=2, hd=128, scale=1.0, softcap=0.0, window=-1, causal=0,
             prefix_len=0, q_doc=0, k_doc=0, slopes=0, dist_bias=0, dist_radius=0)
    a.update(change)
    return L.MaskedAttention(*a.values())


@pytest.mark.parametrize("change", [dict(kind=1), dict(n_seq=-1), dict(max_q=-1), dict(max_k=(1 << 20) + 1), dict(q_rows=-1),
                                    dict(nh=0), dict(nkv=0), dict(nkv=3), dict(hd=0), dict(hd=513), dict(ldq=511),
                                    dict(ldk=255), dict(ldv=255), dict(ldo=511), dict(scale=math.nan), dict(softcap=-1.0),
                                    dict(softcap=math.inf), dict(q_doc=FAKE), dict(k_doc=FAKE), dict(prefix_len=FAKE),
                                    dict(dist_bias=FAKE, dist_radius=-1), dict(dist_bias=FAKE, dist_radius=1025)])
def test_attention_masked_refuses(change):
    a = masked(**change)
    assert L.load().eg2_attention_masked_workspace(C.byref(a)) == -1
    assert L.load().eg2_attention_masked(C.byref(a), None, 0, None) == -1


@pytest.mark.parametrize("change", [dict(q=0), dict(k=0), dict(v=0), dict(out=0), dict(q_off=0), dict(k_off=0)])
def test_attention_masked_refuses_missing_buffers(change):
    a = masked(**change)
    assert L.load().eg2_attention_masked(C.byref(a), None, 0, None) == -1


def test_empty_calls_do_nothing():
    for change in (dict(q_rows=0), dict(n_seq=0), dict(max_q=0)):
        a = masked(**change)
        assert L.load().eg2_attention_masked(C.byref(a), None, 0, None) == 0
    assert rotary_rc(rows=0) == 0
    assert L.load().eg2_quantize_rows(L.EG2_BF16, None, 8, None, 16, None, 0, 8, None) == 0
    assert L.load().eg2_gemm_i8(None, 16, None, None, 16, None, None, None, 8, 0, 8, 16, 0, None) == 0


@pytest.mark.parametrize("i,bad", [(0, 1), (2, 7), (4, 7), (6, -1), (7, 0), (1, 0), (3, 0), (5, 0)])
def test_quantize_rows_refuses(i, bad):
    a = [L.EG2_F32, FAKE, 8, FAKE, 16, FAKE, 4, 8]
    a[i] = bad
    assert L.load().eg2_quantize_rows(*a, None) == -1


@pytest.mark.parametrize("i,bad", [(0, 0), (0, FAKE + 8), (1, 24), (1, 0), (2, 0), (3, 0), (3, FAKE + 1), (4, 17), (5, 0),
                                   (7, 0), (8, 7), (9, -1), (10, 0), (11, 0), (11, 131073)])
def test_gemm_i8_refuses(i, bad):
    a = [FAKE, 32, FAKE, FAKE, 32, FAKE, None, FAKE, 8, 4, 8, 32, 0]
    a[i] = bad
    assert L.load().eg2_gemm_i8(*a, None) == -1


def test_python_layer_refuses_host_tensors_and_wrong_types():
    q, k = torch.zeros(3, 4, 8), torch.zeros(3, 2, 8)
    pos, steps = torch.zeros(3, dtype=torch.int32), torch.zeros(4, dtype=torch.int64)
    off = torch.tensor([0, 3], dtype=torch.int32)
    calls = [
        lambda: ops.rotary(q, k, pos, steps),                                  # not on a GPU
        lambda: ops.rotary(q, k, pos.long(), steps),
        lambda: ops.rotary(q, k.double(), pos, steps),
        lambda: ops.rotary(q, k, pos, steps, rot_dim=5),
        lambda: ops.rotary(q, k, pos, steps, rot_dim=10),
        lambda: ops.rotary(q, k, pos, steps[:3]),
        lambda: ops.rotary(q, k, pos, steps, layout="both"),
        lambda: ops.rotary(q.transpose(0, 1), None, pos, steps),
        lambda: ops.attention_masked(q, k, k, off, off, 3, 3),                 # not on a GPU
        lambda: ops.attention_masked(q, k, k[:, :1], off, off, 3, 3),
        lambda: ops.attention_masked(q[:, :3], k, k, off, off, 3, 3),
        lambda: ops.attention_masked(q, k, k, off.long(), off, 3, 3),
        lambda: ops.attention_masked(q, k, k, off, off, 3, 3, prefix_len=off[:1]),
        lambda: ops.attention_masked(q, k, k, off, off, 3, 3, q_doc=pos),
        lambda: ops.attention_masked(q, k, k, off, off, 3, 3, slopes=torch.zeros(3)),
        lambda: ops.attention_masked(q, k, k, off, off, 3, 3, dist_bias=torch.zeros(4, 4)),
        lambda: ops.quantize_rows(q),
        lambda: ops.quantize_rows(q[0]),                                       # not on a GPU
        lambda: ops.quantize_rows(q[0].half()),
        lambda: ops.quantize_rows(torch.zeros(4, 0)),
        lambda: ops.gemm_i8(torch.zeros(2, 8, dtype=torch.int8), torch.zeros(2), torch.zeros(2, 8, dtype=torch.int8), torch.zeros(2)),
        lambda: ops.gemm_i8(torch.zeros(2, 16, dtype=torch.int8), torch.zeros(2), torch.zeros(2, 16, dtype=torch.int8), torch.zeros(3)),
        lambda: ops.gemm_i8(torch.zeros(2, 16, dtype=torch.int8), torch.zeros(2), torch.zeros(2, 16), torch.zeros(2)),
    ]
    for call in calls:
        with pytest.raises(L.Eg2Error):
            call()
