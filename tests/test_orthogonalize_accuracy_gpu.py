"""How far the orthogonalised update is off exact steps: the figures that its documentation gives, as they stand there.

bfloat16 results: 1.3 to 1.5 times what rounding X to eleven bits and A and M to fp16 does to 64-bit steps (1.5e-3; 4.0e-3; 2.1e-2; 4.3e-2
at the most over these sizes), and on top what rounding the exact result to bfloat16 alone does (1.7e-3).  What storing the gradient
as bfloat16 costs is computed from the exact steps of the rounded gradient.  float16 results: their own rounding (2.07e-4 for
values spread evenly between fp16's steps) and half as much again; for the four directions 485 times what float32 sums of 2304 terms
are off, a few 2^-24, comes to twice the rounding."""
import pytest
import torch

from sru_b200 import orthogonalize

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def exact(g):
    x = g.double()
    x = x.mT if x.size(0) > x.size(1) else x
    x = x / (x.norm() + 1e-7)
    eye = torch.eye(x.size(0), dtype=torch.float64)
    for _ in range(5):
        a = x @ x.mT
        x = (3.4445 * eye - 4.7750 * a + 2.0315 * (a @ a)) @ x
    return x.mT if g.size(0) > g.size(1) else x


def with_values(m, n, values, g):
    left = torch.linalg.qr(torch.randn(m, m, generator=g, dtype=torch.float64))[0]
    right = torch.linalg.qr(torch.randn(n, m, generator=g, dtype=torch.float64))[0]
    return (left * values) @ right.T


def gradient(kind, m, n):
    g = torch.Generator().manual_seed(m + n)
    i = torch.arange(1, m + 1, dtype=torch.float64)
    noise = torch.randn(m, n, generator=g, dtype=torch.float64)
    if kind == "noise":
        return noise.float()
    if kind == "sixteen":
        strong = torch.randn(m, 16, generator=g, dtype=torch.float64) @ torch.randn(16, n, generator=g, dtype=torch.float64)
        return ((0.25 * strong + noise) * 1e-3).float()
    if kind == "four":
        strong = torch.randn(m, 4, generator=g, dtype=torch.float64) @ torch.randn(4, n, generator=g, dtype=torch.float64)
        return (strong + 0.01 * noise).float()
    return with_values(m, n, 1 / i if kind == "1/i" else 1 / i ** 2, g).float()


SIZES = [(128, 384), (256, 1024), (512, 2048), (768, 2304)]
KINDS = [("noise", 2e-3, 3e-4), ("sixteen", 2e-3, 3e-4), ("1/i", 6e-3, 3e-4), ("1/i^2", 3e-2, 3e-4), ("four", 6e-2, 7e-4)]


@pytest.mark.parametrize("m,n", SIZES)
@pytest.mark.parametrize("kind,bfloat16,float16", KINDS)
def test_documented_accuracy(m, n, kind, bfloat16, float16):
    g = gradient(kind, m, n)
    want = exact(g)
    norm = float(want.norm())
    rounding = float((want.bfloat16().double() - want).norm()) / norm
    assert rounding <= 1.8e-3
    for grad, ref in ((g, want), (g.mT, want.mT)):
        got = orthogonalize(grad.to(DEV)).cpu()
        assert got.dtype == torch.bfloat16
        err = float((got.double() - ref).norm()) / norm
        assert err <= bfloat16 + rounding, err
        fine = orthogonalize(grad.to(DEV), out_dtype=torch.float16).cpu().double()
        assert float((fine - ref).norm()) <= float16 * norm
    if kind in ("1/i", "1/i^2", "four"):
        stored = float((exact(g.bfloat16()) - want).norm()) / norm
        assert err <= stored / 4 + rounding, (err, stored)


@pytest.mark.parametrize("rows,cols", [(100, 120), (120, 100), (128, 768), (16, 700), (200, 300), (300, 200), (200, 304), (700, 900), (900, 704),
                                       (704, 900), (64, 4200), (4200, 64), (1100, 1030), (1100, 1032), (20, 500)])
@pytest.mark.parametrize("out", [torch.bfloat16, torch.float16])
def test_no_row_is_scaled(rows, cols, out):
    """X <- 3.1416 X once: M = 3.1416 I, which fp16 holds as 3.1406, 3.1e-4 less.  The result as a multiple of the exact one: the
    elements' roundings (1.7e-3 in the mean to bfloat16, 2.1e-4 to eleven bits) average out over at least 10000 of them to 1.7e-5;
    allowed is 1.2e-4."""
    g = torch.randn(rows, cols, generator=torch.Generator().manual_seed(rows + cols))
    want = 3.1416 * g.double() / (g.double().norm() + 1e-7)
    got = orthogonalize(g.to(DEV), steps=1, coefficients=(3.1416, 0.0, 0.0), out_dtype=out).cpu().double()
    ratio = float((got * want).sum() / want.square().sum())
    assert abs(ratio - 1.0) <= 1.2e-4, ratio
