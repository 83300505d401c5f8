"""Refusals of the operators around the recurrent layers, without a GPU: bad arguments end as errors on the host."""
import ctypes

import pytest
import torch

from sru_b200 import _lib


def last_error():
    return _lib.lib().sru_b200_last_error().decode()


def test_linear_recurrence_refuses_cpu_tensors():
    from sru_b200 import gated_linear_recurrence
    with pytest.raises(_lib.SruB200Error, match="no CPU path"):
        gated_linear_recurrence(torch.zeros(2, 1, 8))


def test_linear_recurrence_c_arguments():
    L = _lib.lib()
    one = ctypes.c_void_p(16)      # never dereferenced: every call below is refused on the host
    f = L.sru_b200_linear_recurrence_forward
    assert f(None, None, None, None, None, None, None, 4, 2, 8, 32, 16, 0, _lib.SRU_F32, None) == -1
    assert "must not be null" in last_error()
    assert f(one, None, None, one, None, None, None, -1, 2, 8, 32, 16, 0, _lib.SRU_F32, None) == -1
    assert f(one, None, None, one, None, None, None, 4, 2, 0, 32, 16, 0, _lib.SRU_F32, None) == -1
    assert f(one, None, None, one, None, None, None, 4, 2, 8, 32, 16, 0, _lib.SRU_F64, None) == -2
    assert f(one, None, None, one, None, None, None, 4, 2, 8, 31, 16, 0, _lib.SRU_F32, None) == -1
    assert "aligned" in last_error()
    assert f(one, None, None, ctypes.c_void_p(18), None, None, None, 4, 2, 8, 32, 16, 0, _lib.SRU_BF16, None) == -1
    assert f(one, None, None, one, None, None, None, 0, 2, 8, 32, 16, 0, _lib.SRU_F32, None) == 0      # nothing to do
    g = L.sru_b200_linear_recurrence_backward
    assert g(one, None, None, one, None, None, None, None, None, 4, 2, 8, 32, 16, 16, 8, 0, 0, None, 0, None) == -1
    assert g(one, one, None, one, one, one, None, None, None, 4, 2, 8, 32, 16, 16, 8, 0, 0, None, 0, None) == -3
    assert L.sru_b200_linear_recurrence_states_bytes(17, 3, 5) == 3 * 3 * 5 * 4
    assert L.sru_b200_linear_recurrence_states_bytes(0, 3, 5) == 0


def test_embedding_refuses_cpu_tensors():
    from sru_b200 import embedding_lookup
    with pytest.raises(_lib.SruB200Error, match="no CPU path"):
        embedding_lookup(torch.zeros(3, dtype=torch.long), torch.zeros(5, 8))


def test_embedding_c_arguments():
    L = _lib.lib()
    one = ctypes.c_void_p(16)      # never dereferenced: every call below is refused on the host
    f, g = L.sru_b200_embedding_forward, L.sru_b200_embedding_backward
    assert f(None, one, one, 3, 5, 8, 8, 1.0, 8, 0, 0, None) == -1
    assert f(one, one, one, 3, 0, 8, 8, 1.0, 8, 0, 0, None) == -1
    assert f(one, one, one, 3, 5, 8, 7, 1.0, 8, 0, 0, None) == -1
    assert f(one, one, one, 3, 5, 8, 8, 1.0, 2, 0, 0, None) == -1
    assert f(one, one, one, 1 << 31, 5, 8, 8, 1.0, 8, 0, 0, None) == -1
    assert f(one, one, one, 3, 1 << 31, 8, 8, 1.0, 8, 0, 0, None) == -1
    assert f(one, one, one, 3, 5, 8, 8, 1.0, 8, _lib.SRU_BF16, _lib.SRU_F32, None) == -2
    assert f(one, one, one, 3, 5, 8, 8, 1.0, 8, _lib.SRU_F64, _lib.SRU_F64, None) == -2
    assert f(None, None, None, 0, 5, 8, 8, 1.0, 8, 0, 0, None) == 0
    assert g(None, one, one, 3, 5, 8, -1, 1.0, 8, 0, 0, None, 0, None) == -1
    assert g(one, one, one, 3, 5, 8, -1, 1.0, 8, 0, 0, None, 0, None) == -3
    assert g(one, one, one, 3, 5, 8, -1, 1.0, 8, 0, 0, ctypes.c_void_p(8), 1 << 20, None) == -3
    assert "aligned" in last_error()


def test_orthogonalize_refuses_cpu_tensors():
    from sru_b200 import orthogonalize
    with pytest.raises(_lib.SruB200Error, match="no CPU path"):
        orthogonalize(torch.zeros(3, 4))


def test_orthogonalize_c_arguments():
    L = _lib.lib()
    one = ctypes.c_void_p(256)     # never dereferenced: every call below is refused on the host
    f = L.sru_b200_orthogonalize
    tail = (3.4, -4.7, 2.0, 1e-7)
    big = 1 << 30
    assert f(one, one, -1, 4, 5, 20, 5, 1, 5, *tail, 0, 2, one, big, None) == -1
    assert f(one, one, 1, 1 << 21, 5, 20, 5, 1, 5, *tail, 0, 2, one, big, None) == -1
    assert f(one, one, 1, 4, 5, 20, 5, 1, -1, *tail, 0, 2, one, big, None) == -1
    assert f(one, one, 1, 4, 5, 20, 5, 1, 5, 3.4, -4.7, 2.0, -1.0, 0, 2, one, big, None) == -1
    assert f(one, one, 1, 4, 5, 20, 5, 1, 5, 3.4, -4.7, 2.0, float("nan"), 0, 2, one, big, None) == -1
    assert f(one, one, 1, 4, 5, 20, 5, 1, 5, *tail, _lib.SRU_F64, 2, one, big, None) == -2
    assert f(one, one, 1, 4, 5, 20, 5, 1, 5, *tail, 0, _lib.SRU_F32, one, big, None) == -2
    assert f(None, one, 1, 4, 5, 20, 5, 1, 5, *tail, 0, 2, one, big, None) == -1
    assert f(one, one, 1, 4, 5, 20, 10, 2, 5, *tail, 0, 2, one, big, None) == -1
    assert f(one, one, 1, 4, 5, 20, 5, 1, 5, *tail, 0, 2, None, 0, None) == -3
    assert f(one, one, 1, 4, 5, 20, 5, 1, 5, *tail, 0, 2, ctypes.c_void_p(16), big, None) == -3
    assert f(one, one, 0, 4, 5, 20, 5, 1, 5, *tail, 0, 2, None, 0, None) == 0


@pytest.mark.parametrize("timed", [False, True])
def test_refusals_come_as_the_packages_error(timed, monkeypatch):
    """Through the native operator and through the Python form that a timer sees alike."""
    from sru_b200 import embedding_lookup, gated_linear_recurrence, orthogonalize
    monkeypatch.setattr(_lib, "timer", object() if timed else None)
    with pytest.raises(_lib.SruB200Error, match="no CPU path"):
        gated_linear_recurrence(torch.zeros(2, 1, 8))
    with pytest.raises(_lib.SruB200Error, match="no CPU path"):
        embedding_lookup(torch.zeros(3, dtype=torch.long), torch.zeros(5, 8))
    with pytest.raises(_lib.SruB200Error, match="no CPU path"):
        orthogonalize(torch.zeros(3, 4))
    assert isinstance(_lib.refused(RuntimeError("x")), _lib.SruB200Error)
    oom = torch.OutOfMemoryError("x")
    assert _lib.refused(oom) is oom
