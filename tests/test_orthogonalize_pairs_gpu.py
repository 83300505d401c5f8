"""The orthogonalised update into float16: iterates of 22 bits, so that the result is the exact steps rounded once.

Tolerance: half as much again as rounding the exact result to fp16 alone does, in the Frobenius norm.  The pairs' own rounding is
2^-22 and the float32 sums' a few 2^-24 relative, fifteen times, multiplied by at most some tens along the singular directions that a
gradient of this kind has (a^5 = 485 only where they are 0): 1e-5 to 5e-5 against 2.07e-4.  Elements, at most: half a step of fp16 (2^-11
relative, 2^-25 where it is subnormal) and 2^-11 of the norm's root mean square, by the same count."""
import pytest
import torch

from sru_b200 import _lib, orthogonalize

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


def exact(g, steps=5, abc=(3.4445, -4.7750, 2.0315)):
    x = g.double()
    x = x.mT if x.size(-2) > x.size(-1) else x
    x = x / (torch.linalg.matrix_norm(x, keepdim=True) + 1e-7)
    eye = torch.eye(x.size(-2), dtype=torch.float64)
    for _ in range(steps):
        a = x @ x.mT
        x = (abc[0] * eye + abc[1] * a + abc[2] * (a @ a)) @ x
    return x.mT if g.size(-2) > g.size(-1) else x


def gradient(batch, rows, cols, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    strong = torch.randn(batch, rows, 4, generator=g) @ torch.randn(batch, 4, cols, generator=g)
    return ((strong + torch.randn(batch, rows, cols, generator=g)) * 1e-3).to(dtype)


def check(g, **kw):
    got = orthogonalize(g.to(DEV), out_dtype=F16, **kw)
    _lib.check_device_error()
    assert got.dtype == F16 and got.shape == g.shape and got.is_contiguous()
    got, want = got.cpu().double(), exact(g, **kw)
    for z in range(g.size(0)) if g.dim() == 3 else [...]:
        err, w = got[z] - want[z], want[z]
        assert float(err.norm()) <= 1.5 * float((w.half().double() - w).norm()) + 1e-6, (tuple(g.shape), z)
        rms = float(w.norm()) / w.numel() ** 0.5
        assert bool((err.abs() <= 2.0 ** -11 * (w.abs() + rms) + 2.0 ** -25).all())
    return got


@pytest.mark.parametrize("rows,cols", [(1, 1), (1, 7), (9, 1), (2, 3), (8, 8), (31, 33), (64, 64), (100, 257), (127, 128), (128, 129),
                                       (129, 128), (255, 256), (256, 300), (257, 257), (384, 385), (130, 1000), (1000, 130), (513, 640),
                                       (700, 520), (64, 4100), (4200, 65), (1100, 1030), (1, 2000), (2000, 3)])
def test_sizes(rows, cols):
    """One tile and several, whole and ragged, wide and tall, split reductions and not, aligned results and not."""
    check(gradient(1, rows, cols, F32, rows * 7 + cols)[0])
    check(gradient(2, rows, cols, F16, rows * 5 + cols))


@pytest.mark.parametrize("batch,rows,cols", [(3, 72, 200), (40, 24, 40), (7, 33, 4160), (2, 500, 1700), (15, 100, 2000), (33, 128, 300),
                                             (6, 1024, 530), (300, 9, 14)])
def test_batches_and_types(batch, rows, cols):
    for dtype in (F32, F16, BF16):
        check(gradient(batch, rows, cols, dtype, rows + cols))


@pytest.mark.parametrize("steps", [0, 1, 2, 3])
def test_steps(steps):
    check(gradient(1, 90, 152, F32, 6)[0], steps=steps)
    check(gradient(1, 151, 90, F32, 6)[0], steps=steps)


def test_other_coefficients():
    g = gradient(1, 60, 80, F32, 8)[0]
    got = orthogonalize(g.to(DEV), steps=6, coefficients=(1.5, -0.5, 0.0), out_dtype=F16).cpu().double()
    want = exact(g, 6, (1.5, -0.5, 0.0))
    assert float((got - want).norm()) <= 1.5 * float((want.half().double() - want).norm())


def test_layouts():
    g = gradient(3, 65, 140, F32, 2)
    dev = g.to(DEV)
    want = orthogonalize(dev, out_dtype=F16)
    wide = torch.zeros(3, 70, 200, device=DEV)
    wide[:, 2:67, 9:149] = dev
    apart = torch.zeros(3, 65, 280, device=DEV)[:, :, ::2].copy_(dev)
    for v in (dev.mT.contiguous().mT, wide[:, 2:67, 9:149], apart, dev.transpose(0, 1).contiguous().transpose(0, 1)):
        assert torch.equal(orthogonalize(v, out_dtype=F16), want)
    for z in range(3):
        assert torch.equal(orthogonalize(dev[z], out_dtype=F16), want[z])
    assert torch.equal(orthogonalize(dev.mT, out_dtype=F16), want.mT)


def test_one_bad_matrix_of_a_batch():
    for rows, cols in ((48, 80), (300, 200)):
        g = torch.randn(5, rows, cols, generator=torch.Generator().manual_seed(3)).to(DEV)
        want = orthogonalize(g, out_dtype=F16)
        for bad in (float("nan"), float("inf")):
            h = g.clone()
            h[2, 5, 7] = bad
            got = orthogonalize(h, out_dtype=F16)
            assert got[2].isnan().all() and torch.equal(got[[0, 1, 3, 4]], want[[0, 1, 3, 4]])
    assert not orthogonalize(torch.zeros(40, 60, device=DEV), out_dtype=F16).any()
    _lib.check_device_error()


def test_same_bits_again_other_streams_and_captured():
    mats = [gradient(b, r, c, F32, r).to(DEV) for b, r, c in ((1, 100, 300), (3, 200, 300), (1, 64, 4200), (2, 700, 900))]

    def both():
        return [orthogonalize(m, out_dtype=o) for m in mats for o in (F16, BF16)]
    want = both()
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream(), torch.cuda.Stream()], []
    for st in streams:
        with torch.cuda.stream(st):
            got.append(both())
    torch.cuda.synchronize()
    for g in got:
        assert all(torch.equal(a, b) for a, b in zip(g, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = both()
    for _ in range(2):
        graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(out, want))
    _lib.check_device_error()


@pytest.mark.parametrize("out", [F16, BF16])
@pytest.mark.parametrize("batch,rows,cols", [(1, 130, 67), (3, 65, 300), (2, 257, 301), (2, 333, 140), (1, 500, 2011), (2, 900, 30), (20, 140, 150),
                                             (1, 1100, 1030), (1, 100, 300)])
def test_no_write_outside_the_outputs(batch, rows, cols, out):
    """With the workspace of exactly the size that this type of result asks for; the other entry gives the larger of both."""
    L_ = _lib.lib()
    st = torch.cuda.current_stream().cuda_stream
    code = _lib.DTYPE_CODE[out]
    g = gradient(batch, rows, cols, F32, rows).to(DEV)
    need = int(L_.sru_b200_orthogonalize_workspace_bytes_for(batch, rows, cols, code))
    assert need <= int(L_.sru_b200_orthogonalize_workspace_bytes(batch, rows, cols))
    sizes = {"out": batch * rows * cols * 2, "ws": need}
    bufs = {k: torch.full((n + 512,), 0xA5, dtype=torch.uint8, device=DEV) for k, n in sizes.items()}
    at = {k: t.data_ptr() + 256 for k, t in bufs.items()}
    args = (at["out"], g.data_ptr(), batch, rows, cols, rows * cols, cols, 1, 5, 3.4445, -4.7750, 2.0315, 1e-7, _lib.SRU_F32, code, at["ws"])
    assert L_.sru_b200_orthogonalize(*args, need - 1, st) == -3
    _lib.check(L_.sru_b200_orthogonalize(*args, need, st))
    torch.cuda.synchronize()
    for k, t in bufs.items():
        assert (t[:256] == 0xA5).all() and (t[256 + sizes[k]:] == 0xA5).all(), k
    assert torch.equal(bufs["out"][256:256 + sizes["out"]].view(out).view(batch, rows, cols), orthogonalize(g, out_dtype=out))


def test_offsets_past_32_bits():
    """A batch whose pairs have more than 2^32 elements, its first and its last matrix; wide, and tall.

    On top of the rounding, float32 sums over n = 60000: the tensor cores add 16 columns at a time and cut the sum off, by 2^-23 of
    it at most, so that A is off by at most e = n / 16 * 2^-23.  A step takes that to sigma |b sigma^2 + 2 c sigma^4| e, at most 1.2 e for
    sigma up to 1.2, and later steps, whose slope is about 0.7 around 1, to a third of that again and again: 2.5 e."""
    torch.manual_seed(1)
    batch, rows, cols = 300, 130, 60_000
    g = torch.empty(batch, rows, cols, device=DEV, dtype=BF16).normal_()
    assert g.numel() > 2 ** 31
    eye = torch.eye(rows, dtype=torch.float64, device=DEV)
    for grad in (g, g.view(batch, cols, rows)):
        got = orthogonalize(grad, out_dtype=F16)
        for z in (0, batch - 1):
            x = grad[z].double()
            x = x.mT if x.size(0) > x.size(1) else x
            x = x / (x.norm() + 1e-7)
            for _ in range(5):
                a = x @ x.T
                x = (3.4445 * eye - 4.7750 * a + 2.0315 * (a @ a)) @ x
            own = got[z].double()
            own = own.mT if own.size(0) > own.size(1) else own
            # elements near 1 / sqrt(60000): fp16 has its eleven bits there
            assert float((own - x).norm()) <= 1.5 * float((x.half().double() - x).norm()) + 2.5 * cols / 16 * 2.0 ** -23 * float(x.norm())
        del got
    _lib.check_device_error()
