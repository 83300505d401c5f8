"""Gated linear recurrence (sru_b200_linear_recurrence_forward / _backward) against the definition in 64 bits.

Tolerances, per element: half a step of the output's type relative to the value (finfo.eps / 2), plus REL of the tensor's
largest value for the float32 arithmetic.  A step adds at most 8 roundings of 2^-24 (three of them in the gate's exponential
and reciprocal, relative to f c + (1 - f) x), and with the logits used here (N(0, 1) + bias in [0, 2]) the geometric mean of
f is below 0.86, so an error is remembered for about 7 steps, 16 allowed: 16 * 8 * 2^-24 = 7.6e-6, rounded up to 1e-5.
grad_bias sums L * B values that are each right to that bound.
"""
import pytest
import torch

from sru_b200 import _lib
from sru_b200.linear_recurrence import gated_linear_recurrence

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
REL = 1e-5
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


def plain(u, c0, bias, mask, reverse):
    """float64, step by step, on the CPU; differentiable."""
    L, B, w = u.shape
    x, g = u[..., 0::2], u[..., 1::2]
    c = torch.zeros(B, w // 2, dtype=u.dtype) if c0 is None else c0
    h = [None] * L
    for t in (range(L - 1, -1, -1) if reverse else range(L)):
        f = torch.sigmoid(g[t] if bias is None else g[t] + bias)
        n = f * c + (1 - f) * x[t]
        if mask is not None:
            live = (mask[t] == 0).unsqueeze(1)
            c = torch.where(live, n, c)
            h[t] = torch.where(live, n, torch.zeros_like(n))
        else:
            c = n
            h[t] = n
    return (torch.stack(h) if L else x), c


def make(L, B, d, dtype, seed, init=True, bias=True, mask=True):
    g = torch.Generator().manual_seed(seed)
    u = torch.randn(L, B, 2 * d, generator=g).to(dtype)
    c0 = torch.randn(B, d, generator=g) if init else None
    b = torch.rand(d, generator=g) * 2 if bias else None
    m = None
    if mask:
        m = torch.rand(L, B, generator=g) < 0.25
        m[:, B // 2] = True                         # one sequence is all padding
    gh = torch.randn(L, B, d, generator=g).to(dtype)
    gl = torch.randn(B, d, generator=g)
    return u, c0, b, m, gh, gl


def near(new, ref, what):
    new, ref = new.detach().double().cpu(), ref.detach().double()
    assert new.shape == ref.shape, what
    if ref.numel() == 0:
        return
    half = 0.0 if what in ("c_last", "grad_c0", "grad_bias") else torch.finfo(what[1]).eps / 2
    top = float(ref.abs().max())
    bad = (new - ref).abs() - (half * ref.abs() + REL * top)
    assert float(bad.max()) <= 0, (what, float((new - ref).abs().max()), top)


def check(L, B, d, dtype, reverse=False, seed=0, **kw):
    u, c0, b, m, gh, gl = make(L, B, d, dtype, seed, **kw)
    leaves = [None if t is None else t.double().requires_grad_() for t in (u, c0, b)]
    h_ref, c_ref = plain(*leaves, m, reverse)
    torch.autograd.backward([h_ref, c_ref], [gh.double(), gl.double()])
    dev = [None if t is None else t.to(DEV).requires_grad_() for t in (u, c0, b)]
    h, c = gated_linear_recurrence(*dev, None if m is None else m.to(DEV), reverse=reverse)
    assert h.dtype == dtype and c.dtype == F32
    torch.autograd.backward([h, c], [gh.to(DEV), gl.to(DEV)])
    near(h, h_ref, ("h", dtype))
    near(c, c_ref, "c_last")
    near(dev[0].grad, leaves[0].grad, ("grad_u", dtype))
    if c0 is not None:
        near(dev[1].grad, leaves[1].grad, "grad_c0")
    if b is not None:
        dg = float(leaves[0].grad[..., 1::2].abs().max()) if u.numel() else 0.0
        want = torch.zeros(d, dtype=torch.float64) if leaves[2].grad is None else leaves[2].grad
        err = (dev[2].grad.double().cpu() - want).abs().max()
        assert float(err) <= REL * L * B * max(dg, 1e-30), float(err)
    with torch.no_grad():
        h2, c2 = gated_linear_recurrence(*dev, None if m is None else m.to(DEV), reverse=reverse)
    assert torch.equal(h, h2) and torch.equal(c, c2)
    _lib.check_device_error()


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("L,B,d", [(1, 1, 1), (1, 3, 33), (2, 2, 31), (15, 1, 32), (16, 3, 64), (17, 2, 65), (33, 5, 7),
                                   (129, 2, 200), (300, 4, 96), (257, 1, 513)])
def test_lengths_and_widths(L, B, d, dtype):
    check(L, B, d, dtype, seed=L * 31 + d)
    check(L, B, d, dtype, seed=L * 37 + d, reverse=True)


@pytest.mark.parametrize("init", [False, True])
@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("mask", [False, True])
@pytest.mark.parametrize("reverse", [False, True])
def test_options(init, bias, mask, reverse):
    for dtype in (F32, BF16):
        check(70, 3, 40, dtype, seed=5, init=init, bias=bias, mask=mask, reverse=reverse)


@pytest.mark.parametrize("L,B,d", [(2100, 1, 40), (1500, 2, 130), (4097, 1, 32), (700, 8, 1024), (130, 40, 520)])
def test_few_and_many_columns(L, B, d):
    """Sizes on both sides of every rule that spreads the work."""
    check(L, B, d, BF16, seed=L, mask=False)
    check(L, B, d, F32, seed=L + 1, reverse=True)


@pytest.mark.parametrize("slices", [1, 2, 3, 7, 8, 9, 16, 24, 33, 64])
def test_every_cut_of_time(slices):
    """The number of slices a column's time is cut into (option linrec_slices) changes only the order of roundings."""
    with _lib.options(linrec_slices=slices):
        check(700, 3, 70, BF16, seed=slices)
        check(1025, 2, 33, F32, seed=slices, reverse=True)
        check(8 * slices + 1, 2, 64, F16, seed=slices, mask=False)


def test_empty():
    for L, B in ((0, 3), (4, 0), (0, 0)):
        check(L, B, 8, F32, mask=False)


def test_gradient_against_differences():
    """<gradient, v> against central differences of the definition in 64 bits along random directions v (step 1e-4:
    truncation about 1e-8 of the third derivative); the gradient's own error is REL of its norm at most."""
    L, B, d = 60, 3, 24
    u, c0, b, m, gh, gl = make(L, B, d, F32, 11)
    dev = [t.to(DEV).requires_grad_() for t in (u, c0, b)]
    h, c = gated_linear_recurrence(*dev, m.to(DEV))
    torch.autograd.backward([h, c], [gh.to(DEV), gl.to(DEV)])

    def loss(*leaves):
        hh, cc = plain(*leaves, m, False)
        return float((hh * gh.double()).sum() + (cc * gl.double()).sum())
    for seed in range(3):
        g = torch.Generator().manual_seed(100 + seed)
        base = [t.double() for t in (u, c0, b)]
        v = [torch.randn(t.shape, generator=g, dtype=torch.float64) for t in base]
        eps = 1e-4
        diff = (loss(*[t + eps * w for t, w in zip(base, v)]) - loss(*[t - eps * w for t, w in zip(base, v)])) / (2 * eps)
        own = sum(float((t.grad.double().cpu() * w).sum()) for t, w in zip(dev, v))
        size = sum(float((t.grad.double().cpu() * w).abs().sum()) for t, w in zip(dev, v))
        assert abs(own - diff) <= 1e-5 * size, (own, diff, size)


def test_what_padding_holds_is_not_looked_at():
    """NaN, infinities and the type's lowest value at padded positions of u and of grad_h change nothing."""
    for dtype in (F32, F16, BF16):
        u, c0, b, m, gh, gl = make(90, 4, 48, dtype, 3)
        outs = []
        for fill in (0.0, float("nan"), float("inf"), -float("inf"), torch.finfo(dtype).min):
            uu, gg = u.clone(), gh.clone()
            uu[m] = fill
            gg[m] = fill
            dev = [t.to(DEV).requires_grad_() for t in (uu, c0, b)]
            h, c = gated_linear_recurrence(*dev, m.to(DEV))
            torch.autograd.backward([h, c], [gg.to(DEV), gl.to(DEV)])
            outs.append([h, c] + [t.grad for t in dev])
            assert not h[m.to(DEV)].any() and not dev[0].grad[m.to(DEV)].any()
        for other in outs[1:]:
            assert all(torch.equal(a, o) for a, o in zip(outs[0], other))
        # the sequence that is all padding hands its state and its gradient through unchanged
        assert torch.equal(outs[0][1][2].cpu(), c0[2]) and torch.equal(outs[0][3][2].cpu(), gl[2])


def test_saturated_gates():
    """Logits of +-inf and of the type's extremes: f is exactly 0 or 1 (to 2^-120), nothing overflows; NaN stays NaN."""
    for dtype in (F32, F16, BF16):
        top = torch.finfo(dtype).max
        g = torch.tensor([float("inf"), -float("inf"), top, -top, 100.0, -100.0, float("nan"), 0.0], dtype=dtype)
        u = torch.stack([torch.full_like(g, 3.0), g], dim=-1).view(1, 1, -1).repeat(20, 2, 1).to(DEV).requires_grad_()
        h, c = gated_linear_recurrence(u, torch.full((2, 8), 2.0, device=DEV))
        want = torch.tensor([2.0, 3.0, 2.0, 3.0, 2.0, 3.0, float("nan"), 3.0])
        torch.testing.assert_close(h[-1, 0].float().cpu(), want, equal_nan=True, atol=1e-3, rtol=0)
        h.nan_to_num().sum().backward()
        grad = u.grad[..., [0, 1, 2, 3, 4, 5, 6, 7, 8, 9, 10, 11, 14, 15]]
        assert torch.isfinite(grad).all()


def test_strides_and_unused_gradients():
    """Batch-first views, slices and broadcast gradients, h or c_last alone in the loss."""
    u, c0, b, m, gh, gl = make(50, 4, 24, BF16, 9)
    want = gated_linear_recurrence(u.to(DEV), c0.to(DEV), b.to(DEV), m.to(DEV))
    batch_first = u.transpose(0, 1).contiguous().to(DEV).transpose(0, 1)
    wide = torch.randn(53, 5, 60, device=DEV).to(BF16)
    wide[2:52, 1:, 4:52] = u.to(DEV)
    odd = torch.zeros(50 * 4 * 48 + 1, device=DEV, dtype=BF16)[1:].view(50, 4, 48).copy_(u)
    apart = torch.zeros(50, 4, 96, device=DEV, dtype=BF16)[..., ::2].copy_(u)
    for v in (batch_first, wide[2:52, 1:, 4:52], odd, apart):
        got = gated_linear_recurrence(v, c0.to(DEV), b.to(DEV), m.t().contiguous().t().to(DEV))
        assert all(torch.equal(x, y) for x, y in zip(got, want))
        v = v.detach().requires_grad_()
        h, c = gated_linear_recurrence(v, c0.to(DEV), b.to(DEV), m.to(DEV))
        h.sum().backward()
        w = u.to(DEV).requires_grad_()
        h, c = gated_linear_recurrence(w, c0.to(DEV), b.to(DEV), m.to(DEV))
        h.backward(torch.ones_like(h))
        assert torch.equal(v.grad, w.grad)
    w = u.to(DEV).requires_grad_()
    b2 = b.to(DEV).requires_grad_()
    gated_linear_recurrence(w, None, b2, m.to(DEV))[1].sum().backward()
    leaves = [u.double().requires_grad_(), b.double().requires_grad_()]
    plain(leaves[0], None, leaves[1], m, False)[1].sum().backward()
    near(w.grad, leaves[0].grad, ("grad_u", BF16))
    assert float((b2.grad.double().cpu() - leaves[1].grad).abs().max()) <= REL * 200 * float(leaves[0].grad.abs().max())


def test_single_steps_equal_the_sequence():
    """Token by token, the state handed on: the same arithmetic as one pass in a single walk over time."""
    u, c0, b, m, *_ = (None if t is None else t.to(DEV) for t in make(12, 5, 80, BF16, 2))
    with torch.no_grad(), _lib.options(linrec_slices=1):
        h, c = gated_linear_recurrence(u, c0, b, m)
        state = c0
        for t in range(12):
            ht, state = gated_linear_recurrence(u[t], state, b, m[t])
            assert ht.shape == (5, 80)
            assert torch.equal(ht, h[t])
        assert torch.equal(state, c)


def test_same_bits_again_and_on_another_stream():
    u, c0, b, m, gh, gl = (t.to(DEV) for t in make(1000, 3, 200, BF16, 4))

    def once():
        dev = [t.clone().requires_grad_() for t in (u, c0, b)]
        h, c = gated_linear_recurrence(*dev, m)
        torch.autograd.backward([h, c], [gh, gl])
        return [h.detach(), c.detach()] + [t.grad for t in dev]
    first = once()
    assert all(torch.equal(x, y) for x, y in zip(first, once()))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = once()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    assert all(torch.equal(x, y) for x, y in zip(first, other))


def test_captured_step_replays():
    """Forward and backward in one graph; replays on new values give the eager results."""
    u, c0, b, m, gh, gl = (t.to(DEV) for t in make(400, 2, 96, BF16, 8))
    dev = [t.clone().requires_grad_() for t in (u, c0, b)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            h, c = gated_linear_recurrence(*dev, m)
            torch.autograd.grad([h, c], dev, [gh, gl])
            del h, c
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        h, c = gated_linear_recurrence(*dev, m)
        grads = torch.autograd.grad([h, c], dev, [gh, gl])
    for seed in (21, 22):
        new = make(400, 2, 96, BF16, seed)
        with torch.no_grad():
            for t, v in zip(dev, new):
                t.copy_(v)
        graph.replay()
        torch.cuda.synchronize()
        eager = [t.detach().clone().requires_grad_() for t in dev]
        he, ce = gated_linear_recurrence(*eager, m)
        want = torch.autograd.grad([he, ce], eager, [gh, gl])
        assert torch.equal(h, he) and torch.equal(c, ce) and all(torch.equal(x, y) for x, y in zip(grads, want))


def test_no_write_outside_the_outputs():
    """Every output lies between bands of a bit pattern that have to survive, in each type, ragged everywhere."""
    L_ = _lib.lib()
    for dtype in (F32, BF16):
        for L, B, d in ((37, 3, 41), (530, 1, 70), (16, 2, 32)):
            u, c0, b, m, gh, gl = (t.to(DEV) for t in make(L, B, d, dtype, 1))
            es = u.element_size()
            sizes = {"h": L * B * d * es, "last": B * d * 4, "states": int(L_.sru_b200_linear_recurrence_states_bytes(L, B, d)),
                     "gu": L * B * 2 * d * es, "gb": d * 4, "gi": B * d * 4,
                     "ws": int(L_.sru_b200_linear_recurrence_backward_workspace_bytes(L, B, d, _lib.DTYPE_CODE[dtype]))}
            bufs = {k: torch.full((n + 512,), 0xA5, dtype=torch.uint8, device=DEV) for k, n in sizes.items()}
            at = {k: t.data_ptr() + 256 for k, t in bufs.items()}
            st = torch.cuda.current_stream().cuda_stream
            code = _lib.DTYPE_CODE[dtype]
            mask = m.contiguous()
            _lib.check(L_.sru_b200_linear_recurrence_forward(
                at["h"], at["last"], at["states"], u.data_ptr(), b.data_ptr(), c0.data_ptr(), mask.data_ptr(), L, B, d,
                B * 2 * d, 2 * d, 0, code, st))
            _lib.check(L_.sru_b200_linear_recurrence_backward(
                at["gu"], at["gb"], at["gi"], u.data_ptr(), b.data_ptr(), at["states"], mask.data_ptr(), gh.data_ptr(),
                gl.data_ptr(), L, B, d, B * 2 * d, 2 * d, B * d, d, 0, code, at["ws"], sizes["ws"], st))
            torch.cuda.synchronize()
            for k, t in bufs.items():
                assert (t[:256] == 0xA5).all() and (t[256 + sizes[k]:] == 0xA5).all(), (k, dtype, L, B, d)
            h, _ = gated_linear_recurrence(u, c0, b, mask)
            assert torch.equal(bufs["h"][256:256 + sizes["h"]].view(dtype).view(L, B, d), h)
