"""Refusals of the layer operators at the ends of the C types, without a GPU (no pointer below is ever read)."""
import pytest

from conftest import pkg

L = pkg("lib")

FAKE = 4096


@pytest.mark.parametrize("m,n", [(4, 2**31 - 1), (4, 2**30 + 1), (2**30 + 1, 4), (2**62, 4)])
def test_gemm_i8_refuses_what_its_tile_numbers_cannot_hold(m, n):
    a = [FAKE, 32, FAKE, FAKE, 32, FAKE, None, FAKE, 2**31, m, n, 32, 0]
    assert L.load().eg2_gemm_i8(*a, None) == -1


@pytest.mark.parametrize("hd", [2**31 - 2, 2**30 + 2])
def test_rotary_refuses_heads_whose_channels_it_cannot_number(hd):
    a = [L.EG2_BF16, 0, 0, FAKE, hd, 1, None, 0, 0, FAKE, hd, None, 0, FAKE, 4, hd, 2, FAKE, 1.0, None]
    assert L.load().eg2_rotary(*a) == -1


def test_python_layer_refuses_sizes_that_do_not_fit_the_c_call():
    """C ints would keep the low 32 bits of these sizes and compute a part of the result. No memory behind the tensors."""
    torch = pytest.importorskip("torch")
    ops = pkg("ops")
    empty = lambda *s, dtype=torch.bfloat16: torch.empty(*s, dtype=dtype, device="meta")
    i8, f32 = torch.int8, torch.float32
    big = 2**32 + 16
    calls = [
        ("2\\^31", lambda: ops.rotary_steps(2**32 + 64)),
        ("2\\^31", lambda: ops.quantize_rows(empty(1, big))),
        ("2\\^31", lambda: ops.gemm_i8(empty(1, 16, dtype=i8), empty(1, dtype=f32), empty(big, 16, dtype=i8), empty(big, dtype=f32))),
        ("2\\^31", lambda: ops.rotary(empty(1, big, 2), None, empty(1, dtype=torch.int32), empty(1, dtype=torch.int64))),
        ("2\\^31", lambda: ops.attention_masked(empty(1, big, 8), empty(1, 1, 8), empty(1, 1, 8), empty(2, dtype=torch.int32),
                                                empty(2, dtype=torch.int32), 1, 1)),
    ]
    for match, call in calls:
        with pytest.raises(L.Eg2Error, match=match):
            call()
