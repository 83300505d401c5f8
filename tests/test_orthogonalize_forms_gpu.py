"""Which form an update of some hundreds of rows takes, by its launches: one cluster for all steps (norm, first iterate, cluster, and a
copy of the result where its rows are not aligned), or a launch per product; and that both are right at the sizes where the rule
changes from one to the other."""
import pytest
import torch

from sru_b200 import _lib, orthogonalize

pytestmark = pytest.mark.gpu
DEV = "cuda:0"

CLUSTER = [(1, 130, 200), (1, 500, 504), (1, 200, 768), (1, 256, 1024), (7, 256, 512), (7, 300, 1504), (6, 512, 2048), (15, 384, 384)]
LAUNCHES = [(1, 200, 2048), (1, 384, 1024), (1, 512, 1024), (5, 512, 2048), (10, 512, 512), (3, 300, 1504), (6, 600, 600), (16, 200, 300)]


@pytest.mark.parametrize("batch,rows,cols,cluster", [(*s, True) for s in CLUSTER] + [(*s, False) for s in LAUNCHES])
def test_form(batch, rows, cols, cluster):
    g = torch.randn(batch, rows, cols, generator=torch.Generator().manual_seed(rows + cols))
    dev = g.to(DEV)
    before = _lib.launch_count
    got = orthogonalize(dev)
    n = _lib.launch_count - before
    assert n <= 4 if cluster else n >= 17
    before = _lib.launch_count
    turned = orthogonalize(dev.mT.contiguous())
    assert (_lib.launch_count - before <= 4) == cluster         # the rule looks at the smaller and the larger side
    _lib.check_device_error()
    x = g[batch - 1].double()
    x = x / (x.norm() + 1e-7)
    eye = torch.eye(rows, dtype=torch.float64)
    for _ in range(5):
        a = x @ x.mT
        x = (3.4445 * eye - 4.7750 * a + 2.0315 * (a @ a)) @ x
    rounding = float((x.bfloat16().double() - x).norm())
    for out in (got[batch - 1].cpu().double(), turned[batch - 1].cpu().double().mT):
        # the documented 2e-3 for gradients that are mostly noise, and what rounding the exact result does
        assert float((out - x).norm()) <= 2e-3 * float(x.norm()) + rounding
