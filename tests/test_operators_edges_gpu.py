"""Recurrence, embedding and orthogonalised update where indexes are large, strides are zero and single values are not finite.

Large tensors are compared on windows.  With logits in [-2, 2] the gate is below 0.881, so that a window that starts 256 steps
early from another state has forgotten it to 0.881^256 < 1e-14 of its size; in the windows the tolerances are those of the
small tests: half a step of the type relative to the value and 1e-5 of the largest value for float32 arithmetic.  What
only spreads the same sums differently has the same bits.
"""
import pytest
import torch

from sru_b200 import _lib, embedding_lookup, gated_linear_recurrence, orthogonalize

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
REL = 1e-5


def plain(u, c, bias):
    h = []
    for t in range(u.size(0)):
        f = torch.sigmoid(u[t, :, 1::2] + bias)
        c = f * c + (1 - f) * u[t, :, 0::2]
        h.append(c)
    return torch.stack(h), c


def near(new, ref, half):
    new, ref = new.detach().double().cpu(), ref.detach()
    assert new.shape == ref.shape
    bad = (new - ref).abs() - (half * ref.abs() + REL * float(ref.abs().max()))
    assert float(bad.max()) <= 0, float((new - ref).abs().max())


@pytest.mark.parametrize("L,B,d", [(70000, 2, 8192), (70000, 2, 8191), (600, 512, 4096), (600, 512, 4095)])
def test_recurrence_offsets_past_32_bits(L, B, d):
    """u has more than 2^31 elements: in slices and in one walk, with and without the copy engine's alignment."""
    torch.manual_seed(L + d)
    u = torch.empty(L, B, 2 * d, device=DEV, dtype=F16).normal_().clamp_(-2, 2)
    assert u.numel() > 2 ** 31
    u.requires_grad_()
    c0 = torch.randn(B, d, device=DEV, requires_grad=True)
    bias = torch.zeros(d, device=DEV)
    gh = torch.empty(L, B, d, device=DEV, dtype=F16).normal_()
    gl = torch.randn(B, d, device=DEV)
    h, c = gated_linear_recurrence(u, c0, bias)
    torch.autograd.backward([h, c], [gh, gl])
    _lib.check_device_error()
    half, W, K = torch.finfo(F16).eps / 2, min(L, 456), 200
    for b in (0, B - 1):
        for j in (0, d - 6):
            cols, pairs = slice(j, j + 6), slice(2 * j, 2 * j + 12)
            for first in (True, False):
                t = slice(0, W) if first else slice(L - W, L)
                uw = u.detach()[t, b:b + 1, pairs].double().cpu().requires_grad_()
                start = c0.detach()[b:b + 1, cols].double().cpu() if first else torch.zeros(1, 6, dtype=torch.float64)
                start.requires_grad_()
                hw, cw = plain(uw, start, 0.0)
                end = gl[b:b + 1, cols].double().cpu() if not first else torch.zeros_like(cw)
                torch.autograd.backward([hw, cw], [gh[t, b:b + 1, cols].double().cpu(), end])
                k = slice(0, K) if first else slice(W - K, W)
                at = slice(0, K) if first else slice(L - K, L)
                near(h[at, b:b + 1, cols], hw[k], half)
                near(u.grad[at, b:b + 1, pairs], uw.grad[k], half)
                if first:
                    near(c0.grad[b:b + 1, cols], start.grad, 0.0)
                else:
                    near(c[b:b + 1, cols], cw, 0.0)


@pytest.mark.parametrize("L,B,d,dtype", [(300, 4, 512, BF16), (64, 256, 1024, F16), (40, 3, 33, F32), (300, 4, 512, F32)])
def test_recurrence_repeated_rows(L, B, d, dtype):
    """Gradients and inputs that repeat one row over time, over the batch, or over both (stride 0): the same bits as copies."""
    g = torch.Generator().manual_seed(d)
    u = torch.randn(L, B, 2 * d, generator=g).to(dtype).to(DEV)
    bias = torch.rand(d, generator=g).to(DEV)
    rows = torch.randn(L, B, d, generator=g).to(dtype).to(DEV)

    def step(u, gh, reverse):
        u = u.detach().requires_grad_()
        b = bias.detach().requires_grad_()
        h, c = gated_linear_recurrence(u, None, b, reverse=reverse)
        h.backward(gh)
        return h.detach(), c.detach(), u.grad, b.grad

    for reverse in (False, True):
        for gh in (rows[:1].expand(L, B, d), rows[:, :1].expand(L, B, d), rows[:1, :1].expand(L, B, d), rows[:1, :1, :1].expand(L, B, d)):
            got, want = step(u, gh, reverse), step(u, gh.contiguous(), reverse)
            assert all(torch.equal(x, y) for x, y in zip(got, want))
        for v in (u[:1].expand(L, B, 2 * d), u[:, :1].expand(L, B, 2 * d), u[:1, :1].expand(L, B, 2 * d)):
            with torch.no_grad():
                got, want = gated_linear_recurrence(v, None, bias, reverse=reverse), gated_linear_recurrence(v.contiguous(), None, bias, reverse=reverse)
            assert all(torch.equal(x, y) for x, y in zip(got, want))
    _lib.check_device_error()


@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
@pytest.mark.parametrize("L,B,d", [(300, 3, 128), (64, 256, 1024), (50, 3, 33)])
def test_recurrence_keeps_what_is_not_finite_to_its_column(L, B, d, bad):
    """One such input reaches its column from its step on, one such gradient its column up to its step; nothing else."""
    g = torch.Generator().manual_seed(d)
    clean = torch.randn(L, B, 2 * d, generator=g).to(DEV)
    gh0 = torch.randn(L, B, d, generator=g).to(DEV)
    t, b, j = L // 2 + 3, B - 1, d // 2

    def step(u, gh):
        u = u.detach().requires_grad_()
        bias = torch.zeros(d, device=DEV, requires_grad=True)
        c0 = torch.zeros(B, d, device=DEV, requires_grad=True)
        h, c = gated_linear_recurrence(u, c0, bias)
        h.backward(gh)
        return h.detach(), c.detach(), u.grad, c0.grad, bias.grad

    base = step(clean, gh0)
    u = clean.clone()
    u[t, b, 2 * j] = bad
    h, c, gu, gc, gb = step(u, gh0)
    touched = torch.zeros(L, B, d, dtype=torch.bool, device=DEV)
    touched[t:, b, j] = True
    assert torch.equal(h[~touched], base[0][~touched]) and not h[touched].isfinite().any()
    assert torch.equal(c.isfinite(), ~touched[-1]) and torch.equal(c[~touched[-1]], base[1][~touched[-1]])
    # dx does not look at the states; dg does, where x or the state in front of it is not finite
    assert torch.equal(gu[..., 0::2], base[2][..., 0::2]) and torch.equal(gc, base[3])
    assert torch.equal(gu[..., 1::2][~touched], base[2][..., 1::2][~touched])
    other = torch.arange(d, device=DEV) != j
    assert torch.equal(gb[other], base[4][other]) and not gb[j].isfinite()
    gh = gh0.clone()
    gh[t, b, j] = bad
    h, c, gu, gc, gb = step(clean, gh)
    touched = torch.zeros(L, B, d, dtype=torch.bool, device=DEV)
    touched[:t + 1, b, j] = True
    assert torch.equal(h, base[0]) and torch.equal(c, base[1])
    both = touched.repeat_interleave(2, dim=2)
    assert torch.equal(gu[~both], base[2][~both]) and not gu[t, b, 2 * j].isfinite()
    assert torch.equal(gc[~touched[0]], base[3][~touched[0]])
    assert torch.equal(gb[other], base[4][other])


def test_recurrence_input_changed_before_backward():
    """The saved input is the caller's own memory where its layout fits: a change in place is noticed."""
    u = torch.randn(40, 2, 64, device=DEV)
    w = u.clone().requires_grad_()
    v = w * 1.0
    h, _ = gated_linear_recurrence(v)
    v.mul_(2.0)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        h.sum().backward()
    tokens = torch.tensor([1, 2], device=DEV)
    table = torch.randn(4, 8, device=DEV, requires_grad=True)
    y = embedding_lookup(tokens, table)
    tokens.zero_()
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()


def test_embedding_offsets_past_32_bits():
    """More than 2^31 elements of y and its gradient, and of the table and its gradient."""
    torch.manual_seed(0)
    n, v, d = 600_000, 1000, 4096
    tokens = torch.randint(0, v, (n,), device=DEV)
    tokens[-1] = 7
    table = torch.randn(v, d, device=DEV).half().requires_grad_()
    y = embedding_lookup(tokens, table, scale=1.5)
    assert y.numel() > 2 ** 31
    scaled = (table.detach().float() * 1.5).half()
    for i in range(0, n, 50_000):
        assert torch.equal(y.detach()[i:i + 50_000], scaled[tokens[i:i + 50_000]])
    dy = torch.empty_like(y).normal_()
    y.backward(dy)
    for k in (0, 7, int(tokens[0]), v - 1):
        rows = dy[tokens == k].double() * 1.5
        want, size, m = rows.sum(0), rows.abs().sum(0), rows.size(0)
        err = (table.grad[k].double() - want).abs()
        assert bool((err <= 1.01 * (m + 2) * 2.0 ** -24 * size + 1.01 * torch.finfo(F16).eps / 2 * want.abs() + 2.0 ** -24).all())
    del y, dy, table, scaled
    n, v = 5000, 600_000
    tokens = torch.randint(0, v, (n,), device=DEV)
    tokens[:3] = v - 1
    table = torch.empty(v, d, device=DEV, dtype=F16).normal_().requires_grad_()
    y = embedding_lookup(tokens, table)
    assert torch.equal(y, table.detach()[tokens])
    y.backward(torch.ones_like(y))
    count = torch.bincount(tokens, minlength=v)
    for i in range(0, v, 100_000):
        assert torch.equal(table.grad[i:i + 100_000], count[i:i + 100_000].half().unsqueeze(1).expand(-1, d))
    _lib.check_device_error()


def test_orthogonalize_offsets_past_32_bits():
    """A batch of more than 2^31 elements, its first and its last matrix.  In the Frobenius norm: 1.5 times what rounding the
    iterates and products to fp16 does to float64 steps, half a step of bf16, and 1e-4."""
    torch.manual_seed(1)
    batch, rows, cols = 300, 130, 60_000
    g = torch.empty(batch, rows, cols, device=DEV, dtype=BF16).normal_()
    assert g.numel() > 2 ** 31
    got = orthogonalize(g)
    eye = torch.eye(rows, dtype=torch.float64, device=DEV)

    def steps64(x, r):
        x = r(x.double() / (x.double().norm() + 1e-7))
        for _ in range(5):
            a = r(x @ x.T)
            x = r(r(3.4445 * eye - 4.7750 * a + 2.0315 * (a @ a)) @ x)
        return x

    for z in (0, batch - 1):
        want, model = steps64(g[z], lambda t: t), steps64(g[z], lambda t: t.half().double())
        assert float((got[z].double() - want).norm()) <= 1.5 * float((model - want).norm()) + (2.0 ** -8 + 1e-4) * float(want.norm())
    _lib.check_device_error()


@pytest.mark.parametrize("rows,cols", [(48, 80), (300, 200)])
def test_orthogonalize_one_bad_matrix_of_a_batch(rows, cols):
    g = torch.randn(5, rows, cols, generator=torch.Generator().manual_seed(3)).to(DEV)
    want = orthogonalize(g)
    for bad in (float("nan"), float("inf")):
        h = g.clone()
        h[2, 5, 7] = bad
        got = orthogonalize(h)
        assert got[2].isnan().all()
        assert torch.equal(got[[0, 1, 3, 4]], want[[0, 1, 3, 4]])
    _lib.check_device_error()


def test_orthogonalize_repeated_rows():
    g = torch.randn(4, 60, 90, device=DEV)
    for v in (g[:1].expand(4, 60, 90), g[:, :1].expand(4, 60, 90), g[..., :1].expand(4, 60, 90), torch.randn(300, 1, device=DEV).expand(300, 200)):
        assert torch.equal(orthogonalize(v), orthogonalize(v.contiguous()))


def test_orthogonalize_on_two_streams():
    """Matrices in one SM, in clusters, split between clusters' pairs and with a launch per product, on two streams at once
    and in one captured graph: the bits of calls of their own."""
    g = torch.Generator().manual_seed(4)
    sizes = [(1, 100, 300), (3, 200, 300), (1, 64, 4200), (2, 700, 900), (1, 500, 2000)]
    mats = [torch.randn(*s, generator=g).to(DEV) for s in sizes]
    want = [orthogonalize(m) for m in mats]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(3):
        got = []
        for k, st in enumerate(streams):
            with torch.cuda.stream(st):
                got += [orthogonalize(m) for m in (mats if k else mats[::-1])]
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want[::-1] + want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = [orthogonalize(m) for m in mats]
    for _ in range(2):
        graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(out, want))
    _lib.check_device_error()
