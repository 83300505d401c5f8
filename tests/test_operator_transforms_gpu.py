"""Derivatives and transforms that the operators do not have end as errors, not as wrong numbers."""
import pytest
import torch
from torch.autograd import forward_ad

from sru_b200 import _lib, embedding_lookup, gated_linear_recurrence, orthogonalize

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.mark.parametrize("which", ["u", "c0", "bias"])
@pytest.mark.parametrize("learns", [False, True])
def test_recurrence_refuses_tangents(which, learns):
    args = {"u": torch.randn(9, 2, 8, device=DEV), "c0": torch.randn(2, 4, device=DEV), "bias": torch.randn(4, device=DEV)}
    if learns:
        args = {k: t.requires_grad_() for k, t in args.items()}
    with forward_ad.dual_level():
        dual = dict(args)
        dual[which] = forward_ad.make_dual(args[which], torch.ones_like(args[which]))
        with pytest.raises(_lib.SruB200Error, match="forward-mode derivative, and %s" % which):
            gated_linear_recurrence(**dual)
        with torch.no_grad(), pytest.raises(_lib.SruB200Error, match="forward-mode"):
            gated_linear_recurrence(**dual)
        dual[which] = forward_ad.unpack_dual(dual[which]).primal
        h, c = gated_linear_recurrence(**dual)              # without its tangent it is welcome
    assert torch.equal(h, gated_linear_recurrence(**args)[0])


def test_lookup_refuses_tangents():
    w, t = torch.randn(5, 8, device=DEV), torch.tensor([1, 4], device=DEV)
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(w, torch.ones_like(w))
        for table in (dual, dual.t().contiguous().t()):
            with pytest.raises(_lib.SruB200Error, match="forward-mode"):
                embedding_lookup(t, table)
        assert forward_ad.unpack_dual(orthogonalize(dual)).tangent is None      # documented: a constant
    assert torch.equal(embedding_lookup(t, w), w[t])


def test_functional_derivatives():
    """The functional derivatives stop before a kernel runs."""
    u, w, t = torch.randn(2, 9, 2, 8, device=DEV), torch.randn(5, 8, device=DEV), torch.tensor([1, 4], device=DEV)
    calls = [lambda: torch.func.grad(lambda x: gated_linear_recurrence(x)[0].sum())(u[0]),
             lambda: torch.func.grad(lambda x: embedding_lookup(t, x).sum())(w),
             lambda: torch.func.grad(lambda x: orthogonalize(x).float().sum())(w),
             lambda: torch.func.jvp(lambda x: gated_linear_recurrence(x)[0], (u[0],), (u[1],)),
             lambda: torch.func.jvp(lambda x: embedding_lookup(t, x), (w,), (w,))]
    before = _lib.launch_count
    for call in calls:
        with pytest.raises(_lib.SruB200Error):
            call()
    assert _lib.launch_count == before
    _lib.check_device_error()


def test_vmap():
    """vmap takes the calls one by one; gradients flow through it."""
    u, w, t = torch.randn(3, 9, 2, 8, device=DEV), torch.randn(5, 8, device=DEV), torch.tensor([[1, 4], [0, 1], [1, 1]], device=DEV)
    a, b = u.clone().requires_grad_(), u.clone().requires_grad_()
    h = torch.func.vmap(lambda x: gated_linear_recurrence(x)[0])(a)
    want = torch.stack([gated_linear_recurrence(x)[0] for x in b])
    h.square().sum().backward()
    want.square().sum().backward()
    assert torch.equal(h, want) and torch.equal(a.grad, b.grad)
    assert torch.equal(torch.func.vmap(lambda x: embedding_lookup(x, w))(t), w[t])
    assert torch.equal(torch.func.vmap(orthogonalize)(u[0]), orthogonalize(u[0]))
