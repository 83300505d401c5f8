"""The embedding gradient's separate kernels (sort, sums and fill, join) between bands of a bit pattern that have to survive: sizes
on the far side of the rule that takes small gradients in one launch, with long runs, ragged rows and every token absent but one."""
import pytest
import torch

from sru_b200 import _lib

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


@pytest.mark.parametrize("n,v,d", [(3000, 37, 41), (333, 6000, 72), (2500, 5, 72), (2049, 1, 8), (5000, 70001, 33), (40, 9000, 65)])
@pytest.mark.parametrize("table,out,token", [(F32, F32, torch.int64), (F32, BF16, torch.int32), (BF16, BF16, torch.int64), (F16, F16, torch.int32)])
def test_no_write_outside_the_outputs(n, v, d, table, out, token):
    L_ = _lib.lib()
    st = torch.cuda.current_stream().cuda_stream
    g = torch.Generator().manual_seed(n)
    tokens = torch.randint(0, v, (n,), generator=g)
    tokens[n // 3:n // 2] = v - 1                           # a run over several tiles, up to the table's last row
    dy = torch.randn(n, d, generator=g).to(out)
    tk, dev = tokens.to(token).to(DEV), dy.to(DEV)
    sizes = {"gw": v * d * table.itemsize, "ws": int(L_.sru_b200_embedding_backward_workspace_bytes(n, v, d))}
    bufs = {k: torch.full((m + 512,), 0xA5, dtype=torch.uint8, device=DEV) for k, m in sizes.items()}
    before = _lib.launch_count
    _lib.check(L_.sru_b200_embedding_backward(bufs["gw"].data_ptr() + 256, tk.data_ptr(), dev.data_ptr(), n, v, d, -1, 2.0,
                                              tk.element_size(), _lib.DTYPE_CODE[table], _lib.DTYPE_CODE[out],
                                              bufs["ws"].data_ptr() + 256, sizes["ws"], st))
    torch.cuda.synchronize()
    assert _lib.launch_count - before == (1 if n <= 2048 and (n * out.itemsize + v * table.itemsize) * d <= 1 << 20 else 3)
    for k, t in bufs.items():
        assert (t[:256] == 0xA5).all() and (t[256 + sizes[k]:] == 0xA5).all(), k
    got = bufs["gw"][256:256 + sizes["gw"]].view(table).view(v, d).cpu().double()
    terms = dy.double() * 2.0
    want = torch.zeros(v, d, dtype=torch.float64).index_add_(0, tokens, terms)
    size = torch.zeros(v, d, dtype=torch.float64).index_add_(0, tokens, terms.abs())
    count = torch.bincount(tokens, minlength=v).double().unsqueeze(1)
    # float32 sums of `count` terms in any order, and half a step of the table's type (its smallest one where that is larger)
    bound = 1.01 * ((count + 2) * 2.0 ** -24 * size + torch.finfo(table).eps / 2 * want.abs()) + torch.finfo(table).smallest_normal * torch.finfo(table).eps
    assert bool(((got - want).abs() <= bound).all())
