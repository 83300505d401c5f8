"""The orthogonalised update at the ends of its inputs' and its iterates' range."""
import pytest
import torch

from sru_b200 import _lib, orthogonalize

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
SHAPES = [(50, 70), (70, 50), (200, 300), (300, 200), (700, 900), (1, 700), (64, 4200), (4200, 64)]     # every way an update is carried out


@pytest.mark.parametrize("rows,cols", SHAPES)
@pytest.mark.parametrize("dtype,scales", [(F32, (-149, -140, -126, -70, 0, 100, 121)), (BF16, (-133, -100, 121)), (F16, (-24, 9))])
def test_powers_of_two_do_not_change_the_result(rows, cols, dtype, scales):
    """Whole numbers below 128 times 2^s are held exactly, down to the subnormal end of each type; norm, first iterate and all
    that follows scale exactly, so the result has the same bits, also where 1 / norm leaves float32."""
    g = torch.Generator().manual_seed(rows)
    whole = torch.randint(-127, 128, (rows, cols), generator=g).double()
    whole[0, 0] = 1.0
    want = orthogonalize(whole.to(dtype).to(DEV), eps=0.0, out_dtype=BF16)
    assert want.isfinite().all() and want.any()
    for s in scales:
        scaled = (whole * 2.0 ** s).to(dtype)
        assert torch.equal(scaled.double(), whole * 2.0 ** s)
        assert torch.equal(orthogonalize(scaled.to(DEV), eps=0.0, out_dtype=BF16), want), s
    _lib.check_device_error()


@pytest.mark.parametrize("rows,cols", SHAPES)
def test_zeros(rows, cols):
    """0 / eps is 0 for every eps that is not 0, and 0 / 0 is not a number."""
    for dtype in (F32, BF16):
        zeros = torch.zeros(rows, cols, device=DEV, dtype=dtype)
        for eps in (1e-7, 1e-30, 1e-60, 5e-324, 1e300):
            assert not orthogonalize(zeros, eps=eps).any(), eps
        assert orthogonalize(zeros, eps=0.0).isnan().all()
        assert not orthogonalize(torch.ones_like(zeros), eps=1e300).any()


def steps64(g, rounded, abc=(3.4445, -4.7750, 2.0315), steps=5):
    """The steps in 64 bits; rounded: with A and M rounded to fp16 and X to fp16's eleven bits, not to its range."""
    half = (lambda t: t.half().double()) if rounded else (lambda t: t)
    held = (lambda t: (t * 4096).half().double() / 4096) if rounded else (lambda t: t)
    x = g.double()
    x = x.mT if x.size(0) > x.size(1) else x
    x = held(x / (x.norm() + 1e-7))
    eye = torch.eye(x.size(0), dtype=torch.float64)
    for _ in range(steps):
        a = half(x @ x.mT)
        x = held(half(abc[0] * eye + abc[1] * a + abc[2] * (a @ a)) @ x)
    return x.mT if g.size(0) > g.size(1) else x


@pytest.mark.parametrize("rows,cols", [(128, 384), (384, 128), (256, 1024), (500, 500), (900, 700), (64, 4200), (1024, 1536)])
@pytest.mark.parametrize("large", [1e4, 1e5])
def test_one_row_far_above_the_others(rows, cols, large):
    """The elements of the other rows lie where fp16 is subnormal and has a few bits left; 2^12 X keeps all eleven.  bfloat16 result:
    1.5 times what the roundings do to 64-bit steps without a range (0.8e-3 to 2.2e-3 of the norm), and what rounding the exact
    result does.  float16 result: half as much again as rounding the exact result."""
    g = torch.randn(rows, cols, generator=torch.Generator().manual_seed(rows + cols))
    g[3] *= large
    want, model = steps64(g, False), steps64(g, True)
    assert float((model - want).norm()) <= 2.3e-3 * float(want.norm())
    got = orthogonalize(g.to(DEV)).cpu().double()
    assert float((got - want).norm()) <= 1.5 * float((model - want).norm()) + float((want.bfloat16().double() - want).norm())
    got = orthogonalize(g.to(DEV), out_dtype=F16).cpu().double()
    assert float((got - want).norm()) <= 1.5 * float((want.half().double() - want).norm())


@pytest.mark.parametrize("rows,cols", SHAPES)
@pytest.mark.parametrize("a", [3.0, -2.0, 8.0, 12.0])
def test_coefficients_that_let_the_iterates_grow(rows, cols, a):
    """X <- a X three times: |a|^3 X_0 whatever power of two is held (9, 11, 5 and 3 of the usual 12).  X_0, each of
    three steps and the result round to eleven bits (relative 2^-11; where fp16 is subnormal, half of its smallest step, which
    later steps multiply; a bfloat16 result by 2^-8 at the end), and nothing overflows (A = X X^T is at most 12^4).  The bound holds
    for a float16 result, whose iterates have more bits, too."""
    g = torch.randn(rows, cols, generator=torch.Generator().manual_seed(rows))
    want = a ** 3 * g.double() / (g.double().norm() + 1e-7)
    tiny = 2.0 ** -25 * (abs(a) ** 3 + a ** 2 + abs(a) + 2)
    for out, rounding in ((F16, 0.0), (BF16, 2.0 ** -8)):
        got = orthogonalize(g.to(DEV), steps=3, coefficients=(a, 0.0, 0.0), out_dtype=out).cpu().double()
        assert got.isfinite().all()
        assert bool(((got - want).abs() <= (5.05 * 2.0 ** -11 + rounding * 1.01) * want.abs() + tiny).all())
    _lib.check_device_error()


@pytest.mark.parametrize("rows,cols", SHAPES)
def test_no_steps(rows, cols):
    """G / |G| alone, rounded to eleven bits and to the result's type."""
    g = torch.randn(rows, cols, generator=torch.Generator().manual_seed(rows))
    want = g.double() / (g.double().norm() + 1e-7)
    for out in (F16, BF16):
        got = orthogonalize(g.to(DEV), steps=0, out_dtype=out).cpu().double()
        bound = (2.0 ** -11 + torch.finfo(out).eps / 2) * 1.01 * want.abs() + (2.0 ** -25 if out == F16 else 2.0 ** -37)
        assert bool(((got - want).abs() <= bound).all())
