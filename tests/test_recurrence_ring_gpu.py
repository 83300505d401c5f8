"""Gated linear recurrence in one walk over time with the copy engine's ring, where nothing is whole: lengths that are no multiple
of a chunk, columns that are no multiple of a warp's 64 or a CTA's 128, padded chunks, CTAs with a single scanning warp.

The same definition in 64 bits and the same tolerances as the tests of the other forms; slices are held at 1 by the option, or come
out as 1 by themselves where there are many columns."""
import pytest
import torch

from sru_b200 import _lib, gated_linear_recurrence
from test_linear_recurrence_gpu import check, make

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("L,B,d", [(37, 3, 68), (129, 2, 200), (70, 3, 40), (16, 2, 4), (300, 4, 192), (17, 1, 128), (23, 2, 132),
                                   (31, 1, 64), (100, 2, 260)])
def test_ragged_sizes(L, B, d, dtype):
    with _lib.options(linrec_slices=1):
        for mask in (False, True):
            for reverse in (False, True):
                check(L, B, d, dtype, reverse=reverse, seed=L + d + 2 * mask + reverse, mask=mask, init=mask != reverse)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_many_columns(dtype):
    """One walk by the library's own rule."""
    check(70, 64, 900, dtype, seed=1)
    check(41, 64, 900, dtype, seed=2, reverse=True)


@pytest.mark.parametrize("slices", [1, None])
def test_what_padding_holds_is_not_looked_at(slices):
    for L, B, d in ((91, 4, 132), (45, 3, 68)):
        for dtype in (F32, BF16):
            u, c0, b, m, gh, gl = make(L, B, d, dtype, 3)
            m[20:50, 0] = True                              # whole chunks of padding, and partly padded ones at either end
            outs = []
            for fill in (0.0, float("nan"), float("inf"), torch.finfo(dtype).min):
                uu, gg = u.clone(), gh.clone()
                uu[m], gg[m] = fill, fill
                dev = [t.to(DEV).requires_grad_() for t in (uu, c0, b)]
                with _lib.options(linrec_slices=slices):
                    h, c = gated_linear_recurrence(*dev, m.to(DEV))
                    torch.autograd.backward([h, c], [gg.to(DEV), gl.to(DEV)])
                outs.append([h, c] + [t.grad for t in dev])
            for other in outs[1:]:
                assert all(torch.equal(a, o) for a, o in zip(outs[0], other))


@pytest.mark.parametrize("slices", [1, 2, 9, None])
@pytest.mark.parametrize("L,B,d", [(37, 3, 68), (1003, 1, 36), (129, 2, 200), (300, 4, 192), (23, 2, 132), (70, 64, 900)])
def test_no_write_outside_the_outputs(L, B, d, slices):
    """Every output lies between bands of a bit pattern that have to survive."""
    L_ = _lib.lib()
    st = torch.cuda.current_stream().cuda_stream
    for dtype in (F32, BF16):
        for reverse in (0, 1):
            u, c0, b, m, gh, gl = (t.to(DEV) for t in make(L, B, d, dtype, 1))
            es, code = u.element_size(), _lib.DTYPE_CODE[dtype]
            with _lib.options(linrec_slices=slices):
                sizes = {"h": L * B * d * es, "last": B * d * 4, "states": int(L_.sru_b200_linear_recurrence_states_bytes(L, B, d)),
                         "gu": L * B * 2 * d * es, "gb": d * 4, "gi": B * d * 4,
                         "ws": int(L_.sru_b200_linear_recurrence_backward_workspace_bytes(L, B, d, code))}
                bufs = {k: torch.full((n + 512,), 0xA5, dtype=torch.uint8, device=DEV) for k, n in sizes.items()}
                at = {k: t.data_ptr() + 256 for k, t in bufs.items()}
                _lib.check(L_.sru_b200_linear_recurrence_forward(
                    at["h"], at["last"], at["states"], u.data_ptr(), b.data_ptr(), c0.data_ptr(), m.data_ptr(), L, B, d,
                    B * 2 * d, 2 * d, reverse, code, st))
                _lib.check(L_.sru_b200_linear_recurrence_backward(
                    at["gu"], at["gb"], at["gi"], u.data_ptr(), b.data_ptr(), at["states"], m.data_ptr(), gh.data_ptr(),
                    gl.data_ptr(), L, B, d, B * 2 * d, 2 * d, B * d, d, reverse, code, at["ws"], sizes["ws"], st))
                h, _ = gated_linear_recurrence(u, c0, b, m, reverse=bool(reverse))
            torch.cuda.synchronize()
            for k, t in bufs.items():
                assert (t[:256] == 0xA5).all() and (t[256 + sizes[k]:] == 0xA5).all(), (k, dtype, reverse)
            assert torch.equal(bufs["h"][256:256 + sizes["h"]].view(dtype).view(L, B, d), h)
