"""Layer norm against a plain 64-bit implementation with element-wise bounds (token_reference.py)."""
import pytest
import torch

import token_reference as R
import torch_point_ops_b200 as tpo

pytestmark = pytest.mark.gpu
DEV = "cuda"
TYPES = [(torch.float32, torch.float32), (torch.float16, torch.float16), (torch.float16, torch.float32),
         (torch.bfloat16, torch.bfloat16), (torch.bfloat16, torch.float32), (torch.float64, torch.float64)]


def _inputs(rows, width, dtype, wdtype, seed=0, shift=1.0):
    g = torch.Generator().manual_seed(seed + rows * 131 + width)
    x = torch.randn(rows, width, generator=g) * 1.5 + shift * torch.randn(rows, 1, generator=g)
    w = 1 + 0.3 * torch.randn(width, generator=g)
    b = 0.3 * torch.randn(width, generator=g)
    dy = torch.randn(rows, width, generator=g)
    return x.to(DEV, dtype), w.to(DEV, wdtype), b.to(DEV, wdtype), dy.to(DEV, dtype)


def _run(x, w, b, dy, eps=1e-5):
    leaves = [t.detach().requires_grad_() for t in (x, w, b) if t is not None]
    it = iter(leaves)
    args = [next(it) if t is not None else None for t in (x, w, b)]
    y = tpo.layer_norm(*args, eps)
    grads = torch.autograd.grad(y, leaves, dy)
    it = iter(grads)
    return y.detach(), [next(it) if t is not None else None for t in (x, w, b)]


# widths at and around every switch of kernel (256, 512, 1024, 2048, 4096, 8192), with and
# without whole 16-byte vectors; row counts below, at and beyond the resident blocks
SHAPES = [(1, 1), (1, 2), (3, 7), (5, 8), (2, 31), (64, 33), (17, 255), (9, 256), (9, 257), (700, 384), (13, 512),
          (13, 520), (5, 771), (6, 1024), (6, 1032), (4, 2048), (3, 2049), (3, 2056), (2, 4096), (2, 4104), (2, 8191),
          (2, 8192), (2, 8193), (3, 10000), (40, 9000), (2371, 64), (5000, 40), (1200, 1100)]


@pytest.mark.parametrize("dtype,wdtype", TYPES)
@pytest.mark.parametrize("rows,width", SHAPES)
def test_forward_backward(rows, width, dtype, wdtype):
    x, w, b, dy = _inputs(rows, width, dtype, wdtype)
    y, (dx, dw, db) = _run(x, w, b, dy)
    ref = R.layer_norm(x, w, b, 1e-5, dy)
    assert y.dtype == dtype and dx.dtype == dtype and dw.dtype == wdtype and db.dtype == wdtype
    for name, t in (("y", y), ("dx", dx), ("dw", dw), ("db", db)):
        R.check(t, ref[name], name)


@pytest.mark.parametrize("width", [40, 129, 1000, 9001])
@pytest.mark.parametrize("has_w,has_b", [(False, False), (True, False), (False, True)])
def test_without_parameters(width, has_w, has_b):
    x, w, b, dy = _inputs(50, width, torch.float32, torch.float32)
    w, b = w if has_w else None, b if has_b else None
    y, (dx, dw, db) = _run(x, w, b, dy)
    ref = R.layer_norm(x, w, b, 1e-5, dy)
    R.check(y, ref["y"])
    R.check(dx, ref["dx"])
    if has_w:
        R.check(dw, ref["dw"])
    if has_b:
        R.check(db, ref["db"])
    with torch.no_grad():
        assert torch.equal(tpo.layer_norm(x, w, b), y)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_large_mean_small_spread(dtype):
    # one-pass moments in fp32 would cancel: the mean is 1000 times the spread
    g = torch.Generator().manual_seed(3)
    x = (1000 + torch.randn(64, 700, generator=g)).to(DEV, dtype)
    R.check(tpo.layer_norm(x), R.layer_norm(x, None, None, 1e-5)["y"])


def test_constant_rows_and_zero_eps():
    x = torch.full((4, 100), 3.0, device=DEV)
    assert torch.equal(tpo.layer_norm(x), torch.zeros_like(x))
    assert torch.isnan(tpo.layer_norm(x, eps=0.0)).all()  # 0 * inf, as the formula says


@pytest.mark.parametrize("width", [64, 300, 5000, 9000])
def test_nonfinite_rows_stay_in_their_row(width):
    x, w, b, dy = _inputs(20, width, torch.float32, torch.float32)
    clean, _ = _run(x, w, b, dy)
    bad = x.clone()
    bad[3, 5], bad[7, 0] = float("nan"), float("inf")
    y, (dx, _, _) = _run(bad, w, b, dy)
    keep = [i for i in range(20) if i not in (3, 7)]
    assert torch.isnan(y[[3, 7]]).all() and torch.equal(y[keep], clean[keep]) and torch.isfinite(dx[keep]).all()


def test_shapes_strides_and_offsets():
    base = torch.randn(6, 50, 3, 160, device=DEV)
    w, b = torch.randn(160, device=DEV), torch.randn(160, device=DEV)
    for x in (base, base[:, ::2, 1], base[2, :, 0], base.transpose(0, 1), base[..., 0, :].reshape(300, 160)[1::3]):
        want = R.layer_norm(x.reshape(-1, 160), w, b, 1e-5)["y"]
        got = tpo.layer_norm(x, w, b)
        assert got.shape == x.shape and got.is_contiguous()
        R.check(got.reshape(-1, 160), want)
    # rows that do not start on 16 bytes, and a transposed matrix
    x = torch.randn(40, 129, device=DEV)[:, 1:]
    R.check(tpo.layer_norm(x), R.layer_norm(x, None, None, 1e-5)["y"])
    x = torch.randn(128, 40, device=DEV).t()
    R.check(tpo.layer_norm(x), R.layer_norm(x, None, None, 1e-5)["y"])
    x = torch.randn(64, device=DEV)
    R.check(tpo.layer_norm(x)[None], R.layer_norm(x[None], None, None, 1e-5)["y"])
    # one row seen many times
    x = torch.randn(1, 64, device=DEV).expand(30, 64).requires_grad_()
    (dx,) = torch.autograd.grad(tpo.layer_norm(x), x, torch.ones(30, 64, device=DEV))
    assert dx.shape == (30, 64)


def test_expanded_and_strided_gradient():
    x, w, b, _ = _inputs(30, 96, torch.float32, torch.float32)
    x.requires_grad_(), w.requires_grad_(), b.requires_grad_()
    gx, gw, gb = torch.autograd.grad(tpo.layer_norm(x, w, b).sum(), (x, w, b))  # grad: one value expanded
    ref = R.layer_norm(x.detach(), w.detach(), b.detach(), 1e-5, torch.ones_like(x))
    R.check(gx, ref["dx"]), R.check(gw, ref["dw"]), R.check(gb, ref["db"])
    dy = torch.randn(30, 192, device=DEV)[:, ::2]
    gx, gw, gb = torch.autograd.grad(tpo.layer_norm(x, w, b), (x, w, b), dy)
    ref = R.layer_norm(x.detach(), w.detach(), b.detach(), 1e-5, dy)
    R.check(gx, ref["dx"]), R.check(gw, ref["dw"]), R.check(gb, ref["db"])


@pytest.mark.parametrize("shape", [(0, 64), (4, 0), (0, 0), (2, 0, 64)])
def test_empty(shape):
    x = torch.randn(shape, device=DEV, requires_grad=True)
    w = torch.randn(shape[-1], device=DEV, requires_grad=True)
    b = torch.randn(shape[-1], device=DEV, requires_grad=True)
    y = tpo.layer_norm(x, w, b)
    dx, dw, db = torch.autograd.grad(y, (x, w, b), torch.ones_like(y))
    assert y.shape == x.shape and dx.shape == x.shape
    assert torch.equal(dw, torch.zeros_like(w)) and torch.equal(db, torch.zeros_like(b))


def test_differences():
    # 64-bit rows against central differences of the operator itself
    g = torch.Generator().manual_seed(1)
    x, w, b = (torch.randn(s, generator=g, dtype=torch.float64).to(DEV).requires_grad_() for s in ((5, 37), (37,), (37,)))
    assert torch.autograd.gradcheck(lambda *a: tpo.layer_norm(*a), (x, w, b), eps=1e-6, atol=1e-7, rtol=1e-6)


def test_same_bits_every_run_and_on_another_stream():
    x, w, b, dy = _inputs(3000, 640, torch.bfloat16, torch.float32)
    y, g = _run(x, w, b, dy)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        y2, g2 = _run(x, w, b, dy)
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(y, y2) and all(torch.equal(p, q) for p, q in zip(g, g2))


def test_graph_capture():
    x, w, b, _ = _inputs(500, 320, torch.float32, torch.float32)
    tpo.layer_norm(x, w, b)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = tpo.layer_norm(x, w, b)
    x.copy_(torch.randn_like(x))
    graph.replay()
    R.check(y, R.layer_norm(x, w, b, 1e-5)["y"])


def test_module():
    m = tpo.LayerNorm(48).to(DEV)
    x = torch.randn(7, 48, device=DEV)
    R.check(m(x), R.layer_norm(x, m.weight.detach(), m.bias.detach(), m.eps)["y"])
    assert len(list(m.parameters())) == 2 and not list(tpo.LayerNorm(48, affine=False).parameters())
    with pytest.raises(ValueError):
        m(torch.randn(7, 47, device=DEV))


def test_refusals():
    x = torch.randn(4, 8, device=DEV)
    w = torch.randn(8, device=DEV)
    for args in ((x, torch.randn(7, device=DEV)), (x, w, torch.randn(8, 1, device=DEV)), (x, w.half()), (x.double(), w),
                 (x, w, w.double()), (x.int(), None), (x, w.cpu()), (torch.tensor(1.0, device=DEV),)):
        with pytest.raises((RuntimeError, IndexError)):
            tpo.layer_norm(*args)
    with pytest.raises((RuntimeError, NotImplementedError)):
        tpo.layer_norm(x.cpu())
    with pytest.raises(RuntimeError):
        tpo.layer_norm(x, eps=-1.0)
    with pytest.raises(RuntimeError):
        tpo.layer_norm(x, eps=float("nan"))


def test_second_differentiation_raises():
    x = torch.randn(4, 8, device=DEV, requires_grad=True)
    (g,) = torch.autograd.grad(tpo.layer_norm(x).square().sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="second differentiation"):
        torch.autograd.grad(g.sum(), x)
