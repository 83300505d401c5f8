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
