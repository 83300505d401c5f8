"""A timer and NVTX ranges look at the operators around the layers as they run otherwise: the same native nodes, one span per
forward and per backward pass, on whatever graph they hang."""
import pytest
import torch

from sru_b200 import _lib, embedding_lookup, gated_linear_recurrence, orthogonalize

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def step(seed=0):
    g = torch.Generator().manual_seed(seed)
    table = torch.randn(30, 32, generator=g).to(DEV).requires_grad_()
    bias = torch.rand(16, generator=g).to(DEV).requires_grad_()
    tokens = torch.randint(0, 30, (50, 3), generator=g).to(DEV)
    x = embedding_lookup(tokens, table, scale=2.0)
    h, c = gated_linear_recurrence(x * 1.5, None, bias)
    h1, c1 = gated_linear_recurrence(x[3], c, bias)
    nodes = {t.grad_fn.name() for t in (h, c1)}
    grads = torch.autograd.grad(h.square().sum() + c1.sum(), (table, bias))
    return nodes, [h.detach(), c1.detach(), *grads, orthogonalize(grads[0])]


def test_the_timed_step_is_the_same_step(monkeypatch):
    nodes, want = step()
    launches = _lib.launch_count
    step()
    launches = _lib.launch_count - launches
    monkeypatch.setattr(_lib, "timer", _lib.KernelTimer())
    before = _lib.launch_count
    timed_nodes, got = step()
    assert _lib.launch_count - before == launches
    assert timed_nodes == nodes                     # the same kind of node in the graph
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    spans = _lib.timer.summary()
    assert {k: v[0] for k, v in spans.items()} == {"embedding_fwd": 1, "embedding_bwd": 1, "linear_recurrence_fwd": 2,
                                                   "linear_recurrence_bwd": 2, "orthogonalize": 1}
    assert all(v[1] > 0 for v in spans.values())


def test_spans_only_where_a_backward_pass_runs(monkeypatch):
    monkeypatch.setattr(_lib, "timer", _lib.KernelTimer())
    u = torch.randn(20, 2, 16, device=DEV, requires_grad=True)
    with torch.no_grad():
        gated_linear_recurrence(u)
    h, _ = gated_linear_recurrence(u)
    assert set(_lib.timer.summary()) == {"linear_recurrence_fwd"}
    h.sum().backward(retain_graph=True)
    h.sum().backward()
    assert _lib.timer.summary()["linear_recurrence_bwd"][0] == 2
    with pytest.raises(_lib.SruB200Error):
        gated_linear_recurrence(u.double())
    h, _ = gated_linear_recurrence(u)
    monkeypatch.setattr(_lib, "timer", None)        # taken off before the backward pass
    h.sum().backward()


def test_nvtx_ranges():
    want = step(1)
    _lib.set_nvtx_ranges(True)
    try:
        got = step(1)
    finally:
        _lib.set_nvtx_ranges(False)
    assert got[0] == want[0] and all(torch.equal(a, b) for a, b in zip(got[1], want[1]))
