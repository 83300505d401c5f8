"""Newton-Schulz orthogonalisation (sru_b200_orthogonalize) against the steps in 64 bits.

Tolerance.  The kernels round X, A = X X^T and M = a I + b A + c A A to fp16 in every step and accumulate in float32.  The
same steps in float64 with those roundings (``model``) give the size of their effect without running a kernel; the
kernels' float32 sums (2^-24 a term, thousands of terms, against fp16's 2^-11) only move some of the roundings to the other
neighbour.  Allowed: 1.5 times the model's error in the Frobenius norm and 3 times its largest entry, plus half a step of
the output's type.  1e-4 of the norm is granted where the model's own error is next to nothing (rank-one matrices).
"""
import pytest
import torch

from sru_b200 import _lib, orthogonalize

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
ABC = (3.4445, -4.7750, 2.0315)


def steps64(g, steps, rounded, abc=ABC, eps=1e-7):
    r = (lambda t: t.half().double()) if rounded else (lambda t: t)
    x = g.double()
    tall = x.size(-2) > x.size(-1)
    x = x.mT if tall else x
    x = r(x / (torch.linalg.matrix_norm(x, keepdim=True) + eps))
    eye = torch.eye(x.size(-2), dtype=torch.float64)
    for _ in range(steps):
        a = r(x @ x.mT)
        x = r(r(abc[0] * eye + abc[1] * a + abc[2] * (a @ a)) @ x)
    return x.mT if tall else x


def gradient(batch, rows, cols, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    strong = torch.randn(batch, rows, 4, generator=g) @ torch.randn(batch, 4, cols, generator=g)
    return ((strong + torch.randn(batch, rows, cols, generator=g)) * 1e-3).to(dtype)


def check(g, out_dtype=None, steps=5, dev=None, **kw):
    got = orthogonalize(g.to(DEV) if dev is None else dev, steps=steps, out_dtype=out_dtype, **kw)
    _lib.check_device_error()
    out_dtype = out_dtype or (BF16 if g.dtype == F32 else g.dtype)
    assert got.dtype == out_dtype and got.shape == g.shape and got.is_contiguous()
    got = got.cpu().double()
    half = torch.finfo(out_dtype).eps / 2
    for z in range(g.size(0)) if g.dim() == 3 else [None]:
        one, out = (g, got) if z is None else (g[z], got[z])
        want, model = steps64(one, steps, False), steps64(one, steps, True)
        norm, top = float(want.norm()), float(want.abs().max())
        err, most = float((out - want).norm()), float((out - want).abs().max())
        assert err <= 1.5 * float((model - want).norm()) + (half + 1e-4) * norm, (one.shape, err / norm)
        assert most <= 3 * float((model - want).abs().max()) + (half + 1e-3) * top, (one.shape, most, top)
    return got


@pytest.mark.parametrize("rows,cols", [(1, 1), (1, 7), (9, 1), (2, 3), (8, 8), (31, 33), (64, 64), (100, 257), (127, 128),
                                       (128, 129), (129, 128), (255, 256), (256, 300), (257, 257), (384, 385), (130, 1000),
                                       (1000, 130), (513, 640), (700, 520)])
def test_sizes(rows, cols):
    check(gradient(1, rows, cols, F32, rows * 7 + cols)[0])
    check(gradient(2, rows, cols, BF16, rows * 5 + cols))


@pytest.mark.parametrize("dtype,out", [(F32, F16), (F32, BF16), (F16, F16), (F16, BF16), (BF16, F16), (BF16, None)])
def test_types_and_batches(dtype, out):
    check(gradient(3, 72, 200, dtype, 3), out)
    check(gradient(5, 200, 72, dtype, 4), out)
    check(gradient(40, 24, 40, dtype, 5), out)


@pytest.mark.parametrize("rows,cols", [(1024, 1100), (1280, 640), (900, 2304)])
def test_larger(rows, cols):
    got = check(gradient(1, rows, cols, BF16, 1)[0])
    values = torch.linalg.svdvals(got)
    assert float(values[0]) < 1.3


@pytest.mark.parametrize("rows,cols", [(128, 768), (768, 128), (128, 769), (770, 127), (128, 255), (120, 511), (65, 512),
                                       (64, 513), (16, 700), (3, 768), (129, 768), (129, 640)])
def test_where_one_cta_takes_the_matrix(rows, cols):
    """Both sides of the sizes at which a matrix stays in one SM's shared memory, and of its column groups."""
    check(gradient(1, rows, cols, F32, rows + cols)[0], F16)
    check(gradient(4, rows, cols, F16, rows + cols), BF16)


@pytest.mark.parametrize("batch,rows,cols", [(6, 1024, 1030), (3, 1500, 1100), (7, 1040, 1024)])
def test_both_tile_widths(batch, rows, cols):
    """More tiles than pairs of SMs: the symmetric products run on 256-column tiles."""
    g = gradient(batch, rows, cols, BF16, 2).to(DEV)
    many, few = orthogonalize(g), orthogonalize(g[:1])
    # one matrix alone takes the narrow tiles: the same sums in the same order
    assert float((many[:1].float() - few.float()).norm()) <= 2.0 ** -9 * float(few.float().norm())
    one = g[batch - 1].cpu()
    err, want = many[batch - 1].cpu().double(), steps64(one, 5, False)
    model = steps64(one, 5, True)
    assert float((err - want).norm()) <= 1.5 * float((model - want).norm()) + (2.0 ** -8 + 1e-4) * float(want.norm())


@pytest.mark.parametrize("batch,rows,cols", [(1, 130, 200), (7, 201, 333), (8, 140, 260), (15, 200, 136), (16, 130, 200),
                                             (1, 130, 1700), (1, 1700, 129), (2, 60, 1000), (9, 1000, 100), (1, 385, 390),
                                             (3, 500, 505), (1, 384, 1024), (1, 384, 1100), (7, 400, 1300), (6, 1101, 450)])
def test_where_one_cluster_takes_the_matrix(batch, rows, cols):
    """Both sides of the sizes and batches at which a cluster takes a matrix through all steps; with and without several
    pairs to a tile, wide and tall, rows of the result aligned and not."""
    check(gradient(batch, rows, cols, F32, rows + cols), BF16)
    for steps in (1, 2):
        check(gradient(batch, rows, cols, F16, rows + cols), F16, steps=steps)


@pytest.mark.parametrize("batch,rows,cols", [(1, 64, 4100), (7, 33, 4160), (1, 500, 4133), (2, 500, 1700), (15, 100, 4000),
                                             (1, 900, 1200), (16, 129, 2000), (33, 128, 900), (1, 4200, 257)])
def test_reductions_split_between_pairs(batch, rows, cols):
    """X X^T of few tiles over a long reduction: two, four and eight pairs of SMs to a tile."""
    g = gradient(batch, rows, cols, BF16, rows + cols)
    got = orthogonalize(g.to(DEV))
    for z in (0, batch - 1):
        want, model = steps64(g[z], 5, False), steps64(g[z], 5, True)
        err = float((got[z].cpu().double() - want).norm())
        assert err <= 1.5 * float((model - want).norm()) + (2.0 ** -8 / 2 + 1e-4) * float(want.norm()), (z, err)
    _lib.check_device_error()


def test_singular_values_gather_around_one():
    g = torch.Generator().manual_seed(9)
    got = orthogonalize(torch.randn(300, 900, generator=g).to(DEV)).double().cpu()
    values = torch.linalg.svdvals(got)
    assert 0.6 < float(values[-1]) and float(values[0]) < 1.3       # the coefficients' own range is 0.68 to 1.13


@pytest.mark.parametrize("steps", [0, 1, 2, 3, 8])
def test_steps(steps):
    check(gradient(1, 90, 150, F32, 6)[0], steps=steps)
    check(gradient(1, 150, 90, F32, 6)[0], F16, steps=steps)


def test_coefficients():
    """The classical cubic step (1.5, -0.5, 0)."""
    g = gradient(1, 60, 80, F32, 8)[0]
    got = orthogonalize(g.to(DEV), steps=12, coefficients=(1.5, -0.5, 0.0), out_dtype=F16).cpu().double()
    want = steps64(g, 12, False, (1.5, -0.5, 0.0))
    model = steps64(g, 12, True, (1.5, -0.5, 0.0))
    assert float((got - want).norm()) <= 1.5 * float((model - want).norm()) + 2.0 ** -10 * float(want.norm())


@pytest.mark.parametrize("rows,cols", [(1, 2000), (2000, 1), (3, 900), (900, 5), (7, 4099), (1100, 16)])
def test_long_and_thin(rows, cols):
    check(gradient(1, rows, cols, F32, rows + 3 * cols)[0])
    check(gradient(2, rows, cols, F16, rows + 5 * cols))


def test_many_small_matrices():
    """More matrices than SMs, in one SM's shared memory and beyond."""
    g = gradient(400, 20, 28, BF16, 7)
    got = check(g)
    dev = g.to(DEV)
    assert torch.equal(orthogonalize(dev[399]).cpu().double(), got[399])
    g = gradient(150, 140, 20, F32, 8)
    got = orthogonalize(g.to(DEV))
    assert torch.equal(orthogonalize(g[149].to(DEV)), got[149])


def test_layouts():
    """Transposed views, slices, batches apart, and strides that have to be copied."""
    g = gradient(3, 65, 140, F32, 2)
    dev = g.to(DEV)
    want = orthogonalize(dev)
    wide = torch.zeros(3, 70, 200, device=DEV)
    wide[:, 2:67, 9:149] = dev
    apart = torch.zeros(3, 65, 280, device=DEV)[:, :, ::2].copy_(dev)
    for v in (dev.mT.contiguous().mT, wide[:, 2:67, 9:149], apart, dev.transpose(0, 1).contiguous().transpose(0, 1)):
        assert torch.equal(orthogonalize(v), want)
    for z in range(3):
        assert torch.equal(orthogonalize(dev[z]), want[z])
    # the steps commute with the transpose: the same iterates
    assert torch.equal(orthogonalize(dev.mT), want.mT)


def test_extreme_values():
    """Zeros, tiny and huge entries (their squares leave float32), one infinity, one NaN, eps."""
    assert not orthogonalize(torch.zeros(40, 60, device=DEV)).any()
    g = gradient(1, 50, 70, F32, 12)[0]
    base = orthogonalize(g.to(DEV), eps=0.0)
    for scale in (2.0 ** -100, 2.0 ** 100):
        assert torch.equal(orthogonalize((g * scale).to(DEV), eps=0.0), base)
    check(g * 1e-7)                                   # eps is of the norm's size
    for bad in (float("inf"), float("nan")):
        h = g.clone()
        h[3, 4] = bad
        assert orthogonalize(h.to(DEV)).isnan().all()
    assert orthogonalize(torch.zeros(0, 5, device=DEV)).shape == (0, 5)
    assert orthogonalize(torch.zeros(0, 4, 5, device=DEV, dtype=F16)).shape == (0, 4, 5)


def test_same_bits_again_other_stream_and_captured():
    g = gradient(2, 300, 420, BF16, 14).to(DEV)
    first = orthogonalize(g)
    assert torch.equal(first, orthogonalize(g))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = orthogonalize(g)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    assert torch.equal(first, other)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = orthogonalize(g)
    g.copy_(gradient(2, 300, 420, BF16, 15))
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, orthogonalize(g))


def test_no_write_outside_the_outputs():
    L_ = _lib.lib()
    st = torch.cuda.current_stream().cuda_stream
    for batch, rows, cols in ((1, 130, 67), (3, 65, 300), (2, 257, 301), (2, 333, 140), (1, 500, 2011), (2, 900, 30), (20, 140, 150)):
        g = gradient(batch, rows, cols, F32, rows).to(DEV)
        sizes = {"out": batch * rows * cols * 2, "ws": int(L_.sru_b200_orthogonalize_workspace_bytes(batch, rows, cols))}
        bufs = {k: torch.full((n + 512,), 0xA5, dtype=torch.uint8, device=DEV) for k, n in sizes.items()}
        at = {k: t.data_ptr() + 256 for k, t in bufs.items()}
        _lib.check(L_.sru_b200_orthogonalize(at["out"], g.data_ptr(), batch, rows, cols, rows * cols, cols, 1, 5, *ABC, 1e-7,
                                             _lib.SRU_F32, _lib.SRU_BF16, at["ws"], sizes["ws"], st))
        torch.cuda.synchronize()
        for k, t in bufs.items():
            assert (t[:256] == 0xA5).all() and (t[256 + sizes[k]:] == 0xA5).all(), (k, rows, cols)
        assert torch.equal(bufs["out"][256:256 + sizes["out"]].view(BF16).view(batch, rows, cols), orthogonalize(g))
