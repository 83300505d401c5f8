"""The operators around the recurrent layers together: a training step through all of them against 64 bits, their native
and their Python form, refusals of what the documentation does not allow, two calls at once."""
import subprocess
import sys

import pytest
import torch

from conftest import ROOT
from sru_b200 import _lib, embedding_lookup, gated_linear_recurrence, orthogonalize
from sru_b200.projection import project

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


@pytest.fixture
def timed(monkeypatch):
    """The Python form of the operators, which is the one that a KernelTimer sees."""
    def install():
        monkeypatch.setattr(_lib, "timer", _lib.KernelTimer())
    return install


def test_native_and_python_forms_give_the_same_bits(timed):
    g = torch.Generator().manual_seed(0)
    u = torch.randn(60, 3, 80, generator=g).to(BF16).to(DEV)
    c0, bias = torch.randn(3, 40, generator=g).to(DEV), torch.rand(40, generator=g).to(DEV).to(F16)
    mask = (torch.rand(60, 3, generator=g) < 0.3).to(DEV)
    table, tokens = torch.randn(30, 24, generator=g).to(DEV), torch.randint(0, 30, (4, 25), generator=g).to(DEV)
    weight = torch.randn(50, 70, generator=g).to(DEV)

    def everything():
        leaves = [t.clone().requires_grad_() for t in (u, c0, bias, table)]
        h, c = gated_linear_recurrence(leaves[0], leaves[1], leaves[2], mask, reverse=True)
        h1, c1 = gated_linear_recurrence(leaves[0][5], leaves[1], leaves[2], mask[5])
        y = embedding_lookup(tokens, leaves[3], scale=0.5, padding_idx=-2, out_dtype=F16)
        (h.float().square().sum() + c.sum() + h1.float().sum() + 2 * c1.sum() + y.float().square().sum()).backward()
        with torch.no_grad():
            quiet = [*gated_linear_recurrence(u, None, bias), embedding_lookup(tokens.int(), table)]
        return [h, c, h1, c1, y] + [t.grad for t in leaves] + quiet + [orthogonalize(weight)]
    native = everything()
    timed()
    python = everything()
    names = _lib.timer.summary()
    assert {"linear_recurrence_fwd", "linear_recurrence_bwd", "embedding_fwd", "embedding_bwd", "orthogonalize"} <= set(names)
    assert all(a.dtype == b.dtype and torch.equal(a, b) for a, b in zip(native, python))


def test_from_a_scripted_program():
    """TorchScript programs and C++ hosts find the operators by name."""
    _lib.load_torch_ops()

    @torch.jit.script
    def program(tokens: torch.Tensor, table: torch.Tensor, u: torch.Tensor):
        y = torch.ops.sru_b200.embedding_lookup(tokens, table, 2.0)
        h, c = torch.ops.sru_b200.gated_linear_recurrence(u)
        return y, h, c, torch.ops.sru_b200.orthogonalize(table)
    g = torch.Generator().manual_seed(1)
    tokens, table = torch.randint(0, 30, (5, 7), generator=g).to(DEV), torch.randn(30, 24, generator=g).to(DEV)
    u = torch.randn(20, 3, 16, generator=g).to(DEV)
    want = [embedding_lookup(tokens, table, scale=2.0), *gated_linear_recurrence(u), orthogonalize(table)]
    assert all(torch.equal(a, b) for a, b in zip(program(tokens, table, u), want))


@pytest.mark.parametrize("python", [False, True])
def test_differentiable_once(python, timed):
    """A second derivative is an error, not a wrong number; the orthogonalised update has no derivative at all."""
    if python:
        timed()
    u = torch.randn(9, 2, 8, device=DEV, requires_grad=True)
    h, _ = gated_linear_recurrence(u)
    (grad,) = torch.autograd.grad(h.square().sum(), u, create_graph=True)
    with pytest.raises(RuntimeError, match="differentiable once|once_differentiable"):
        grad.sum().backward()
    w = torch.randn(9, 8, device=DEV, requires_grad=True)
    y = embedding_lookup(torch.tensor([1, 2], device=DEV), w)
    (grad,) = torch.autograd.grad(y.square().sum(), w, create_graph=True)
    with pytest.raises(RuntimeError, match="differentiable once|once_differentiable"):
        grad.sum().backward()
    assert not orthogonalize(w).requires_grad and not orthogonalize(w.square()).requires_grad


@pytest.mark.parametrize("python", [False, True])
def test_refusals(python, timed):
    if python:
        timed()
    u = torch.zeros(4, 2, 8, device=DEV)
    for args in ((u.double(),), (u[0, 0],), (torch.zeros(4, 2, 7, device=DEV),), (u, torch.zeros(2, 5, device=DEV)),
                 (u, torch.zeros(2, 4)), (u, None, torch.zeros(5, device=DEV)), (u, None, None, torch.zeros(2, 4, device=DEV)),
                 (u, torch.zeros(2, 4, device=DEV, dtype=torch.long)), (u[0], None, None, torch.zeros(4, 2, device=DEV))):
        with pytest.raises(_lib.SruB200Error):
            gated_linear_recurrence(*args)
    w, t = torch.zeros(5, 8, device=DEV), torch.zeros(3, dtype=torch.long, device=DEV)
    for args in ((t.float(), w), (t.short(), w), (t.cpu(), w), (t, w[0]), (t, w.double()), (t, torch.zeros(0, 8, device=DEV)),
                 (t, w, 1.0, 5), (t, w, 1.0, -6), (t, w.half(), 1.0, None, F32), (t, w, 1.0, None, torch.float64)):
        with pytest.raises(_lib.SruB200Error):
            embedding_lookup(*args)
    for args in ((w[0],), (w.double(),), (w.long(),), (w, -1), (w, 5, (1.0, 2.0)), (w, 5, (1.0, 2.0, 3.0), -1.0),
                 (w, 5, (1.0, 2.0, 3.0), 1e-7, F32)):
        with pytest.raises(_lib.SruB200Error):
            orthogonalize(*args)


def test_a_training_step():
    """tokens -> table -> projection -> recurrence -> loss -> gradients -> orthogonalised update, in bf16 with float32
    masters, against the same step in 64 bits.

    Roundings to bf16 (half a step, 2^-9 of a binade's top, at most 2^-8 of a value): table rows, weight, u, h, and in the
    backward pass grad_h, grad_u, grad_y.  Each enters a sum of hundreds of terms with random signs, so a gradient's relative
    error in the Frobenius norm is at most about sqrt(7) 2^-8 / sqrt(3) = 6e-3 if they are independent and the sums keep
    relative errors; doubled for the recurrence's memory: 1.2e-2."""
    g = torch.Generator().manual_seed(7)
    L, B, V, n, d = 48, 8, 90, 64, 96
    tokens = torch.randint(0, V, (L, B), generator=g)
    mask = torch.arange(L).view(L, 1) >= torch.randint(20, L + 1, (B,), generator=g).view(1, B)
    table = torch.randn(V, n, generator=g) * n ** -0.5
    weight = torch.randn(n, 2 * d, generator=g) * n ** -0.5
    bias = torch.rand(d, generator=g) * 2
    c0 = torch.randn(B, d, generator=g) * 0.3
    target = torch.randn(L, B, d, generator=g)

    leaves = [t.clone().to(DEV).requires_grad_() for t in (table, weight, bias, c0)]
    with torch.autocast("cuda", dtype=BF16):
        y = embedding_lookup(tokens.to(DEV), leaves[0], scale=n ** 0.5, padding_idx=0, out_dtype=BF16)
        u = project(y.view(L * B, n), leaves[1]).view(L, B, 2 * d)
        h, c = gated_linear_recurrence(u, leaves[3], leaves[2], mask.to(DEV))
    assert y.dtype == BF16 and u.dtype == BF16 and h.dtype == BF16
    loss = (h.float() * target.to(DEV)).sum() + c.square().sum()
    loss.backward()
    update = orthogonalize(leaves[1].grad)

    ref = [t.double().requires_grad_() for t in (table, weight, bias, c0)]
    yr = ref[0][tokens] * n ** 0.5
    ur = yr @ ref[1]
    state, out = ref[3], []
    for t in range(L):
        f = torch.sigmoid(ur[t, :, 1::2] + ref[2])
        new = f * state + (1 - f) * ur[t, :, 0::2]
        live = ~mask[t].unsqueeze(1)
        state = torch.where(live, new, state)
        out.append(torch.where(live, new, torch.zeros_like(new)))
    ((torch.stack(out) * target.double()).sum() + state.square().sum()).backward()
    ref[0].grad[0] = 0                                    # padding_idx
    for got, want in zip(leaves, ref):
        err = float((got.grad.double().cpu() - want.grad).norm() / want.grad.norm())
        assert err <= 1.2e-2, err
    # the update of the gradient that the kernels found: its singular vectors, all singular values near 1
    uu, _, vv = torch.linalg.svd(leaves[1].grad.double().cpu(), full_matrices=False)
    values = torch.linalg.svdvals(update.double().cpu())
    assert float(values[0]) < 1.3 and float((update.double().cpu() * (uu @ vv)).sum()) > 0.5 * values.numel()
    _lib.check_device_error()


def test_two_streams_at_once():
    """Calls whose kernels may overlap on the GPU share nothing: results as alone."""
    g = torch.Generator().manual_seed(3)
    sets = []
    for k in range(2):
        sets.append((torch.randn(900, 2, 128, generator=g).to(BF16).to(DEV), torch.rand(64, generator=g).to(DEV),
                     torch.randint(0, 500, (3000,), generator=g).to(DEV), torch.randn(500, 64, generator=g).to(DEV),
                     torch.randn(300, 400, generator=g).to(DEV)))

    def work(s):
        u, b, t, w, m = s
        u, b, w = (x.clone().requires_grad_() for x in (u, b, w))
        h, c = gated_linear_recurrence(u, None, b)
        y = embedding_lookup(t, w)
        grads = torch.autograd.grad(h.float().sum() + c.sum() + y.square().sum(), (u, b, w))
        return [h, c, y, orthogonalize(m), *grads]
    alone = [[x.detach().clone() for x in work(s)] for s in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    together = [None, None]
    for _ in range(5):
        for k, st in enumerate(streams):
            with torch.cuda.stream(st):
                together[k] = work(sets[k])
    torch.cuda.synchronize()
    for a, b in zip(alone, together):
        assert all(torch.equal(x, y) for x, y in zip(a, b))


FIRST_CALL_CAPTURED = """
import torch
from sru_b200 import _lib, embedding_lookup, gated_linear_recurrence, orthogonalize
_lib.load_torch_ops()
u = torch.randn(300, 2, 64, device="cuda").bfloat16()
w, t, m = torch.randn(50, 32, device="cuda"), torch.randint(0, 50, (200,), device="cuda"), torch.randn(200, 300, device="cuda")
small = torch.randn(20, 30, device="cuda")
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    out = [*gated_linear_recurrence(u), embedding_lookup(t, w), orthogonalize(m), orthogonalize(small)]
graph.replay()
torch.cuda.synchronize()
want = [*gated_linear_recurrence(u), embedding_lookup(t, w), orthogonalize(m), orthogonalize(small)]
assert all(torch.equal(a, b) for a, b in zip(out, want))
_lib.check_device_error()
print("same")
"""


def test_the_first_call_of_a_process_may_be_a_captured_one():
    run = subprocess.run([sys.executable, "-c", FIRST_CALL_CAPTURED], cwd=ROOT, capture_output=True, text=True, timeout=300)
    assert run.returncode == 0 and "same" in run.stdout, run.stderr[-2000:]


def test_capture_while_an_eager_graph_lives():
    """The framework ties a leaf's gradient node to the stream it was first used on for as long as a graph holds it, so a
    backward pass is captured on leaves of its own (sharing the storage) when an eager graph of the originals is alive."""
    g = torch.Generator().manual_seed(4)
    u = torch.randn(40, 2, 64, generator=g).to(BF16).to(DEV).requires_grad_()
    w = torch.randn(50, 32, generator=g).to(DEV).requires_grad_()
    t = torch.randint(0, 50, (200,), generator=g).to(DEV)

    def forward(u, w):
        return gated_linear_recurrence(u)[0].float().square().sum() + embedding_lookup(t, w).square().sum()
    eager = forward(u, w)
    own = [x.detach().requires_grad_() for x in (u, w)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        torch.autograd.grad(forward(*own), own)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = torch.autograd.grad(forward(*own), own)
    graph.replay()
    want = torch.autograd.grad(eager, (u, w))
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(captured, want))
