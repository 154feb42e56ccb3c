"""torch.library.opcheck and torch.compile of the token operators; captured training steps."""
import pytest
import torch

import torch_point_ops_b200 as tpo

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _tokens(*shape, grad=False):
    return torch.randn(*shape, device=DEV, requires_grad=grad)


def test_opcheck_layer_norm():
    N = torch.ops.torch_point_ops_b200_norm
    x, w, b = _tokens(6, 32, grad=True), _tokens(32, grad=True), _tokens(32, grad=True)
    torch.library.opcheck(N.layer_norm.default, (x, w, b, 1e-5))
    torch.library.opcheck(N.layer_norm.default, (x, None, None, 1e-5))
    x, w, b = x.detach(), w.detach(), b.detach()
    torch.library.opcheck(N.layer_norm_forward.default, (x, w, b, 1e-5))
    y, mean, rstd = N.layer_norm_forward(x, w, b, 1e-5)
    for need in ((True, True, True), (True, False, True), (False, True, False)):
        torch.library.opcheck(N.layer_norm_backward.default, (torch.randn_like(y), x, w, b, mean, rstd, *need))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_opcheck_attention(dtype):
    A = torch.ops.torch_point_ops_b200_attention
    q, k, v = (_tokens(50, h, 16).to(dtype).requires_grad_() for h in (4, 2, 2))
    off = torch.tensor([0, 20, 50], device=DEV)
    torch.library.opcheck(A.packed_attention.default, (q, k, v, off, None, True, 0.25))
    q, k, v = q.detach(), k.detach(), v.detach()
    torch.library.opcheck(A.packed_attention_forward.default, (q, k, v, off, off, True, 0.25))
    o, lse = A.packed_attention_forward(q, k, v, off, off, True, 0.25)
    for need in ((True, True), (True, False), (False, True)):
        torch.library.opcheck(A.packed_attention_backward.default,
                              (torch.randn_like(o), q, k, v, o, lse, off, off, True, 0.25, *need))
    cache = _tokens(2, 30, 2, 16).to(dtype)
    torch.library.opcheck(A.cached_attention.default, (q[:2], cache, cache, torch.tensor([3, 30], device=DEV), 0.25))


def test_compile():
    norm = tpo.LayerNorm(64).to(DEV)
    off = torch.tensor([0, 20, 50], device=DEV)

    def f(x):
        y = norm(x).view(50, 4, 16)
        return tpo.packed_attention(y, y, y, off, causal=True)

    x = _tokens(50, 64, grad=True)
    do = _tokens(50, 4, 16)
    eager, compiled = f(x), torch.compile(f, fullgraph=True)(x)
    assert torch.equal(eager, compiled)
    assert torch.equal(*(torch.autograd.grad(t, x, do)[0] for t in (eager, compiled)))
    q, cache, lengths = _tokens(2, 4, 16), _tokens(2, 30, 2, 16), torch.tensor([3, 30], device=DEV)
    with torch.no_grad():
        assert torch.equal(torch.compile(tpo.cached_attention, fullgraph=True)(q, cache, cache, lengths),
                           tpo.cached_attention(q, cache, cache, lengths))


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
def test_captured_training_step(dtype):
    # forward and backward in one graph, replayed with other values and other lengths
    g = torch.Generator().manual_seed(0)
    x = torch.randn(300, 4, 64, generator=g).to(DEV, dtype).requires_grad_()
    do = torch.randn(300, 4, 64, generator=g).to(DEV, dtype)
    off = torch.tensor([0, 100, 100, 300], device=DEV)

    def step():
        o = tpo.packed_attention(y := tpo.layer_norm(x), y, y, off, causal=True)
        return o.detach(), torch.autograd.grad(o, x, do)[0]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    for new in ([0, 250, 251, 280], [0, 0, 300, 300]):
        off.copy_(torch.tensor(new))
        with torch.no_grad():
            x.mul_(-1.5)
        graph.replay()
        for a, b in zip(captured, step()):
            assert torch.equal(a, b)
