"""``_lib.launch_count`` against the kernel nodes of a captured graph: what the library says it launched is what a stream saw.

The captured calls run no kernels but the library's (contiguous inputs of the types that the kernels take), so every kernel node
of the graph is one of its launches."""
import pytest
import torch
from cuda.bindings import runtime

from sru_b200 import _lib, embedding_lookup, gated_linear_recurrence, orthogonalize
from sru_b200.modules import SRU
from sru_b200.projection import gemm

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
F32, BF16 = torch.float32, torch.bfloat16


def kernel_nodes(graph):
    raw = runtime.cudaGraph_t(graph.raw_cuda_graph())
    rc, _, count = runtime.cudaGraphGetNodes(raw)
    assert rc == runtime.cudaError_t.cudaSuccess
    rc, nodes, count = runtime.cudaGraphGetNodes(raw, count)
    assert rc == runtime.cudaError_t.cudaSuccess
    kinds = [runtime.cudaGraphNodeGetType(n)[1] for n in nodes[:count]]
    return sum(k == runtime.cudaGraphNodeType.cudaGraphNodeTypeKernel for k in kinds)


def counted(call):
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph(keep_graph=True)
    before = _lib.launch_count
    with torch.cuda.graph(graph):
        out = call()
    n = _lib.launch_count - before
    assert n == kernel_nodes(graph)
    graph.replay()
    torch.cuda.synchronize()
    assert _lib.launch_count - before == n          # replays are not counted
    del out
    return n


def test_recurrence():
    u = torch.randn(700, 2, 64, device=DEV).to(BF16).requires_grad_()
    b = torch.rand(32, device=DEV, requires_grad=True)
    gh = torch.randn(700, 2, 32, device=DEV).to(BF16)
    with torch.no_grad():
        assert counted(lambda: gated_linear_recurrence(u, None, b)) == 1
        assert counted(lambda: gated_linear_recurrence(u[0], None, b)) == 1
    assert counted(lambda: torch.autograd.grad(gated_linear_recurrence(u, None, b)[0], (u, b), gh)) == 3
    assert counted(lambda: torch.autograd.grad(gated_linear_recurrence(u)[0], u, gh)) == 2


@pytest.mark.parametrize("n,vocabulary,launches", [(60, 100, 2), (5000, 6000, 4)])
def test_embedding(n, vocabulary, launches):
    t = torch.randint(0, vocabulary, (n,), device=DEV)
    w = torch.randn(vocabulary, 64, device=DEV, requires_grad=True)
    dy = torch.randn(n, 64, device=DEV)
    assert counted(lambda: torch.autograd.grad(embedding_lookup(t, w), w, dy)) == launches


@pytest.mark.parametrize("shape,launches", [((100, 300), 1), ((256, 1024), 3), ((256, 1025), 18), ((2048, 2048), 17), ((700, 900), None),
                                            ((64, 4200), None)])
def test_orthogonalize(shape, launches):
    g = torch.randn(shape, device=DEV)
    n = counted(lambda: orthogonalize(g))
    assert launches is None or n == launches


def test_products_and_layers():
    a, b = torch.randn(256, 512, device=DEV).to(BF16), torch.randn(512, 384, device=DEV).to(BF16)
    assert counted(lambda: gemm(a, b)) == 1
    long_a, long_b = torch.randn(65536, 128, device=DEV).to(BF16), torch.randn(65536, 128, device=DEV).to(BF16)
    assert counted(lambda: gemm(long_a, long_b, trans_a=True)) == 2          # slabs of the reduction, then their sum
    model = SRU(64, 64, num_layers=2).to(DEV).to(BF16).eval()
    x = torch.randn(40, 3, 64, device=DEV).to(BF16)

    def forward():
        with torch.no_grad():
            return model(x)
    before = _lib.launch_count
    forward()
    forward()
    assert _lib.launch_count - before >= 8          # per layer and call a product and a scan at least, from the native loop


def test_refused_calls_and_timed_calls(monkeypatch):
    u = torch.randn(9, 2, 8, device=DEV)
    before = _lib.launch_count
    for bad in (lambda: gated_linear_recurrence(u.double()), lambda: orthogonalize(u[0, 0]),
                lambda: embedding_lookup(torch.zeros(2, device=DEV), u[0])):
        with pytest.raises(_lib.SruB200Error):
            bad()
    assert _lib.launch_count == before
    monkeypatch.setattr(_lib, "timer", _lib.KernelTimer())
    gated_linear_recurrence(u)
    orthogonalize(u[:, 0])
    assert _lib.launch_count == before + 2
