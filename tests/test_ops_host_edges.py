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
