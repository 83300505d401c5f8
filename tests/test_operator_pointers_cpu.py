"""Pointers that the operators' C entry points refuse on the host, where a kernel would otherwise access misaligned memory.  No GPU:
nothing is launched, the addresses are never dereferenced."""
import ctypes

import pytest

from sru_b200 import _lib


def last_error():
    return _lib.lib().sru_b200_last_error().decode()


@pytest.mark.parametrize("dtype,size", [(_lib.SRU_F32, 4), (_lib.SRU_F16, 2), (_lib.SRU_BF16, 2)])
def test_linear_recurrence_pairs_of_the_gradient(dtype, size):
    """grad_u is written a pair (x, g) at a time, so it has to be aligned to a pair and not only to an element."""
    L = _lib.lib()
    at = ctypes.c_void_p
    args = (at(256), None, at(256), None, None, None, 4, 2, 8, 32, 16, 16, 8, 0, dtype, None, 0, None)
    assert L.sru_b200_linear_recurrence_backward(at(256 + size), None, None, *args) == -1
    assert "pairs of grad_u" in last_error()


def test_linear_recurrence_scratch():
    L = _lib.lib()
    at = ctypes.c_void_p
    g = L.sru_b200_linear_recurrence_backward
    sizes = (4, 2, 8, 32, 16, 16, 8, 0, _lib.SRU_BF16)
    assert g(at(256), None, None, at(256), None, at(258), None, None, None, *sizes, None, 0, None) == -1
    assert "states" in last_error()
    assert g(at(256), at(256), None, at(256), None, at(256), None, None, None, *sizes, at(258), 1 << 20, None) == -3
    assert "aligned" in last_error()
    f = L.sru_b200_linear_recurrence_forward
    assert f(at(256), None, at(257), at(256), None, None, None, 4, 2, 8, 32, 16, 0, _lib.SRU_BF16, None) == -1
    assert "states" in last_error()
