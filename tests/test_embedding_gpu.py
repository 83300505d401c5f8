"""Scaled embedding lookup and its gradient (sru_b200_embedding_forward / _backward) against 64 bits.

Tolerances, per element.  y: the product of two float32 values (the scale itself rounded once), 2^-23 relative, plus half a
step of y's type.  Gradient: a float32 sum of m terms in any order is off by at most (m - 1) 2^-24 sum|terms| to first
order; with the scale's and the product's rounding (m + 2) 2^-24, taken 1.01 times, plus half a step of the table's type.
"""
import pytest
import torch

from sru_b200 import _lib, embedding_lookup

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
PAIRS = [(F32, F32), (F32, F16), (F32, BF16), (F16, F16), (BF16, BF16)]


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def check(tokens, vocabulary, hidden, table_dtype, out_dtype, scale=1.7, padding=None, seed=0):
    g = torch.Generator().manual_seed(seed)
    w = torch.randn(vocabulary, hidden, generator=g).to(table_dtype)
    n = tokens.numel()
    dy = torch.randn(n, hidden, generator=g).to(out_dtype)
    dev = w.to(DEV).requires_grad_()
    y = embedding_lookup(tokens.to(DEV), dev, scale=scale, padding_idx=padding, out_dtype=out_dtype)
    assert y.dtype == out_dtype and y.shape == (*tokens.shape, hidden)
    y.backward(dy.to(DEV).view_as(y))
    flat = tokens.reshape(-1).long()
    ref = w.double()[flat] * scale
    err = (y.detach().cpu().double().view(n, hidden) - ref).abs()
    tiny = torch.finfo(out_dtype).smallest_normal * half_step(out_dtype) * 2      # subnormal results: half their fixed step
    assert bool((err <= (2.0 ** -23 + half_step(out_dtype)) * ref.abs() + tiny).all())
    terms = dy.double() * scale
    if padding is not None:
        terms[flat == padding % vocabulary] = 0
    want = torch.zeros(vocabulary, hidden, dtype=torch.float64).index_add_(0, flat, terms)
    size = torch.zeros(vocabulary, hidden, dtype=torch.float64).index_add_(0, flat, terms.abs())
    count = torch.bincount(flat, minlength=vocabulary).double().unsqueeze(1)
    assert dev.grad.dtype == table_dtype
    err = (dev.grad.cpu().double() - want).abs()
    assert bool((err <= 1.01 * (count + 2) * 2.0 ** -24 * size + half_step(table_dtype) * want.abs() * 1.01 + tiny).all()), float(err.max())
    assert not dev.grad[(count[:, 0] == 0).to(DEV)].any()
    _lib.check_device_error()
    return y, dev.grad


@pytest.mark.parametrize("table_dtype,out_dtype", PAIRS)
@pytest.mark.parametrize("n,vocabulary,hidden", [(1, 1, 1), (1, 300, 8), (31, 5, 33), (32, 7, 64), (33, 1000, 7), (64, 3, 256),
                                                 (500, 70000, 40), (1000, 255, 130), (1000, 256, 512), (257, 257, 1000)])
def test_sizes_and_types(n, vocabulary, hidden, table_dtype, out_dtype):
    g = torch.Generator().manual_seed(n + vocabulary)
    tokens = torch.randint(0, vocabulary, (n,), generator=g)
    check(tokens, vocabulary, hidden, table_dtype, out_dtype)
    check(tokens.to(torch.int32), vocabulary, hidden, table_dtype, out_dtype, padding=int(tokens[0]))


@pytest.mark.parametrize("n", [1, 31, 32, 33, 63, 64, 65, 96, 1024, 1025, 2500, 8192, 9000])
def test_one_token_everywhere(n):
    """One run over all tiles; and the same with one other token at either end and in the middle."""
    for hidden in (8, 33, 300):
        tokens = torch.full((n,), 4)
        check(tokens, 6, hidden, F32, F32)
        for at in (0, n // 2, n - 1):
            tokens = torch.full((n,), 4)
            tokens[at] = 2
            check(tokens, 6, hidden, BF16, BF16)


@pytest.mark.parametrize("n", [1, 31, 32, 33, 63, 64, 65, 96, 1025])
def test_one_token_in_a_large_table(n):
    """The same runs where the gradient takes three launches instead of one."""
    for hidden in (64, 65):
        tokens = torch.full((n,), 5000)
        check(tokens, 6000, hidden, F32, F32)
        tokens[n // 2] = 2
        check(tokens, 6000, hidden, BF16, BF16, padding=5999)
        check(tokens, 6000, hidden, F32, F16, padding=2)


def test_uneven_frequencies():
    """Runs of every length at every offset against the tiles: token k occurs k times, shuffled."""
    tokens = torch.repeat_interleave(torch.arange(120), torch.arange(120))
    tokens = tokens[torch.randperm(tokens.numel(), generator=torch.Generator().manual_seed(1))]
    check(tokens, 120, 72, F32, BF16, padding=119)
    check(tokens.sort().values, 66000, 72, F32, F32)
    check(tokens.flip(0).view(2, 1190, 3), 120, 16, F16, F16, padding=-3)


def test_many_tokens():
    g = torch.Generator().manual_seed(0)
    tokens = (torch.rand(70000, generator=g) ** 4 * 20000).long()
    check(tokens, 20000, 24, F32, F32)


def test_large_vocabulary_and_long_runs():
    """Keys of three radix digits, rows far apart; 200000 positions, half of them one token (thousands of tiles in a run)."""
    g = torch.Generator().manual_seed(6)
    check(torch.randint(0, 17_000_000, (500,), generator=g), 17_000_000, 2, F16, F16)
    tokens = torch.randint(0, 3000, (200_000,), generator=g)
    tokens[torch.rand(200_000, generator=g) < 0.5] = 1234
    check(tokens, 3000, 12, F32, F32)


def test_all_padding_and_empty():
    check(torch.full((40,), 3), 9, 16, F32, F32, padding=3)
    check(torch.zeros(0, dtype=torch.long), 9, 16, F32, F32)
    check(torch.zeros(3, 0, dtype=torch.long), 9, 16, BF16, BF16)


def test_layouts():
    """Rows of a wider table, misaligned bases, strided tokens and broadcast gradients."""
    g = torch.Generator().manual_seed(2)
    tokens = torch.randint(0, 50, (6, 8), generator=g).to(DEV)
    w = torch.randn(50, 64, generator=g).to(DEV)
    want = embedding_lookup(tokens, w, scale=3.0)
    wide = torch.zeros(50, 100, device=DEV)
    wide[:, 5:69] = w
    odd = torch.zeros(50 * 64 + 1, device=DEV)[1:].view(50, 64).copy_(w)
    for table in (wide[:, 5:69], odd, w.t().contiguous().t()):
        assert torch.equal(embedding_lookup(tokens, table, scale=3.0), want)
    assert torch.equal(embedding_lookup(tokens.t().contiguous().t(), w, scale=3.0), want)
    a, b = w.clone().requires_grad_(), wide.clone().requires_grad_()
    embedding_lookup(tokens, a, scale=3.0).sum().backward()
    embedding_lookup(tokens, b[:, 5:69], scale=3.0).sum().backward()
    assert torch.equal(a.grad, b.grad[:, 5:69])


def test_gradient_against_differences():
    """The lookup is linear in the table: the difference along any direction v equals <gradient, v>."""
    g = torch.Generator().manual_seed(3)
    tokens = torch.randint(0, 40, (300,), generator=g)
    w, v = torch.randn(40, 24, generator=g, dtype=torch.float64), torch.randn(40, 24, generator=g, dtype=torch.float64)
    dy = torch.randn(300, 24, generator=g)
    dev = w.float().to(DEV).requires_grad_()
    embedding_lookup(tokens.to(DEV), dev, scale=2.0).backward(dy.to(DEV))
    diff = float((((w + 0.5 * v)[tokens] - (w - 0.5 * v)[tokens]) * 2.0 * dy.double()).sum())
    own = (dev.grad.double().cpu() * v)
    assert abs(float(own.sum()) - diff) <= 64 * 2.0 ** -24 * float(own.abs().sum()) + 1e-9


def test_a_token_outside_the_table():
    """Reads nothing: zeros, no gradient, and an error that the host can ask for."""
    w = torch.randn(10, 16, device=DEV, requires_grad=True)
    for bad in (10, -1, 2 ** 31 - 1, 2 ** 40, -2 ** 40):
        tokens = torch.tensor([1, bad, 3, 1], device=DEV)
        y = embedding_lookup(tokens, w)
        with pytest.raises(_lib.SruB200Error, match="outside its embedding table"):
            _lib.check_device_error()
        assert not y[1].any() and torch.equal(y[0], w[1])
        (grad,) = torch.autograd.grad(y, w, torch.ones_like(y))
        with pytest.raises(_lib.SruB200Error, match="outside its embedding table"):
            _lib.check_device_error()
        want = torch.zeros(10, 16, device=DEV)
        want[1], want[3] = 2.0, 1.0
        assert torch.equal(grad, want)
    _lib.check_device_error()


def test_same_bits_again_other_stream_and_captured():
    g = torch.Generator().manual_seed(5)
    tokens = torch.randint(0, 300, (5000,), generator=g).to(DEV)
    w = torch.randn(300, 96, generator=g).to(DEV).requires_grad_()
    dy = torch.randn(5000, 96, generator=g).to(DEV).to(BF16)

    def once():
        y = embedding_lookup(tokens, w, scale=1.3, padding_idx=7, out_dtype=BF16)
        return y.detach(), torch.autograd.grad(y, w, dy)[0]
    first = once()
    assert all(torch.equal(x, y) for x, y in zip(first, once()))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = once()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    assert all(torch.equal(x, y) for x, y in zip(first, other))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = once()
    tokens.copy_(torch.randint(0, 300, (5000,), generator=g))
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(x, y) for x, y in zip(out, once()))


def test_no_write_outside_the_outputs():
    L_ = _lib.lib()
    st = torch.cuda.current_stream().cuda_stream
    for dtype, n, v, d in ((F32, 70, 37, 41), (BF16, 333, 5, 72), (F32, 64, 300, 4)):
        g = torch.Generator().manual_seed(n)
        tokens = torch.randint(0, v, (n,), generator=g).to(DEV)
        w, dy = torch.randn(v, d, generator=g).to(dtype).to(DEV), torch.randn(n, d, generator=g).to(dtype).to(DEV)
        es, code = w.element_size(), _lib.DTYPE_CODE[dtype]
        sizes = {"y": n * d * es, "gw": v * d * es, "ws": int(L_.sru_b200_embedding_backward_workspace_bytes(n, v, d))}
        bufs = {k: torch.full((m + 512,), 0xA5, dtype=torch.uint8, device=DEV) for k, m in sizes.items()}
        at = {k: t.data_ptr() + 256 for k, t in bufs.items()}
        _lib.check(L_.sru_b200_embedding_forward(at["y"], tokens.data_ptr(), w.data_ptr(), n, v, d, d, 2.0, 8, code, code, st))
        _lib.check(L_.sru_b200_embedding_backward(at["gw"], tokens.data_ptr(), dy.data_ptr(), n, v, d, -1, 2.0, 8, code, code,
                                                  at["ws"], sizes["ws"], st))
        torch.cuda.synchronize()
        for k, t in bufs.items():
            assert (t[:256] == 0xA5).all() and (t[256 + sizes[k]:] == 0xA5).all(), (k, dtype)
