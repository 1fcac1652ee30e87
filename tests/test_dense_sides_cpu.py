"""The backward's entry: which of its outputs may be left out."""
import ctypes

import pytest

from sparseattention_b200 import _lib

P = ctypes.c_void_p(0x1000)
V, NULL = _lib.HsaView(0x1000, 0, 0), _lib.HsaView(None, 0, 0)


def bwd(dq, dk, dv):
    return _lib.load().hsa_dense_attn_bwd(V, V, V, V, None, P, V, dq, dk, dv, None, None, 0, 0, 0, None, 0, 1, 4, 4, 2, 2, 64, 0.125, 1, 0, None)


@pytest.mark.parametrize("sides", [(V, V, V), (NULL, V, V), (V, NULL, NULL)])
def test_a_side_may_be_left_out(sides):
    assert bwd(*sides) == -4                                 # the next check: no workspace


@pytest.mark.parametrize("sides", [(NULL, NULL, NULL), (V, V, NULL), (V, NULL, V), (NULL, V, NULL)])
def test_but_not_both_and_not_half_of_one(sides):
    assert bwd(*sides) == -1
