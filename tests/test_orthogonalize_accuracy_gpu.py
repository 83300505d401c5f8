"""How far the orthogonalised update is off exact steps: the figures that its documentation gives, as they stand there.

They are 1.4 to 1.7 times what rounding X to eleven bits and A and M to fp16 does to 64-bit steps (1.5e-3; 4.0e-3; 2.1e-2; 4.3e-2 at
the most over these sizes), and the result's own rounding to fp16 (at most 2^-11 = 4.9e-4) is allowed on top.  What storing the gradient
as bfloat16 costs is computed from the exact steps of the rounded gradient."""
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


@pytest.mark.parametrize("m,n", [(128, 384), (256, 1024), (512, 2048), (768, 2304)])
@pytest.mark.parametrize("kind,documented", [("noise", 2.5e-3), ("sixteen", 2.5e-3), ("1/i", 6e-3), ("1/i^2", 3e-2), ("four", 6e-2)])
def test_documented_accuracy(m, n, kind, documented):
    g = gradient(kind, m, n)
    want = exact(g)
    norm = float(want.norm())
    for grad, ref in ((g, want), (g.mT, want.mT)):
        got = orthogonalize(grad.to(DEV), out_dtype=torch.float16).cpu().double()
        err = float((got - ref).norm()) / norm
        assert err <= documented + 2.0 ** -11, err
    if kind in ("1/i", "1/i^2", "four"):
        stored = float((exact(g.bfloat16()) - want).norm()) / norm
        assert err <= stored / 4 + 2.0 ** -11, (err, stored)
