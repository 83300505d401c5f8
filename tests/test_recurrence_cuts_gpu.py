"""Gated linear recurrence: what must not depend on how a column's time is cut into slices.

An infinite state is multiplied by gates that are closed but not 0 (f = sigmoid(-30) = 9e-14; the smallest gate the
kernels know is 2^-126), so it stays infinite for ever, whatever the product of the gates underflows to.  The definition in 64
bits says where infinities and NaN stand; finite values are right to the bound of the small tests (half a step of the type
and 1e-5 of the largest finite value).
"""
import pytest
import torch

from sru_b200 import _lib, gated_linear_recurrence

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
INF = float("inf")


def plain(u, c, gh, dc, reverse):
    """h, last state, and the gradients of u and of the first state by the chain rule, step by step in 64 bits."""
    times = range(u.size(0) - 1, -1, -1) if reverse else range(u.size(0))
    h, gu, before = torch.empty_like(gh), torch.empty_like(u), torch.empty_like(gh)
    for t in times:
        f = torch.sigmoid(u[t, :, 1::2])
        before[t] = c
        h[t] = c = f * c + (1 - f) * u[t, :, 0::2]
    for t in reversed(times):
        f = torch.sigmoid(u[t, :, 1::2])
        total = dc + gh[t]
        gu[t, :, 0::2] = (1 - f) * total
        gu[t, :, 1::2] = total * (before[t] - u[t, :, 0::2]) * f * (1 - f)
        dc = f * total
    return h, c, gu, dc


def same(got, want, half):
    got = got.detach().double().cpu()
    assert torch.equal(got.isnan(), want.isnan())
    assert torch.equal(got.isinf(), want.isinf()) and torch.equal(got[got.isinf()], want[want.isinf()])
    fine = want.isfinite()
    if fine.any():
        bound = half * want[fine].abs() + 1e-5 * float(want[fine].abs().max())
        assert bool(((got[fine] - want[fine]).abs() <= bound).all())


@pytest.mark.parametrize("slices", [None, 1, 2, 3, 8, 9, 24, 64])
@pytest.mark.parametrize("L,B,d", [(600, 2, 68), (530, 1, 33)])
@pytest.mark.parametrize("reverse", [False, True])
def test_infinities_stay_behind_closed_gates(slices, L, B, d, reverse):
    g = torch.Generator().manual_seed(L + d)
    for dtype in (F32, BF16):
        u = torch.randn(L, B, 2 * d, generator=g)
        u[..., 1::2] -= 30.0
        u[..., 0::2] = (u[..., 0::2].abs() + 0.1) * (1 - 2 * (torch.arange(L) % 2)).view(L, 1, 1)    # no two neighbours alike
        c0, gl = torch.randn(B, d, generator=g), torch.randn(B, d, generator=g)
        gh = torch.randn(L, B, d, generator=g).to(dtype)
        c0[0, 1], c0[B - 1, d - 2] = INF, -INF             # an infinite state handed in
        u[L // 3, 0, 2 * 5], u[L // 2, B - 1, 2 * 7] = INF, -INF        # one that an input makes
        gl[0, 3] = INF                                     # and infinite gradients
        gh[L // 2, 0, 9] = -INF
        u = u.to(dtype)
        want = plain(u.double(), c0.double(), gh.double(), gl.double(), reverse)
        dev = [u.to(DEV).requires_grad_(), c0.to(DEV).requires_grad_()]
        with _lib.options(linrec_slices=slices):
            h, c = gated_linear_recurrence(*dev, reverse=reverse)
            torch.autograd.backward([h, c], [gh.to(DEV), gl.to(DEV)])
        half = torch.finfo(dtype).eps / 2
        for got, ref, bound in zip((h, c, dev[0].grad, dev[1].grad), want, (half, 0.0, half, 0.0)):
            same(got, ref, bound)
    _lib.check_device_error()
