"""Layer norm at the ends of the number range: rows whose mean is large beside their spread."""
import pytest
import torch

import token_reference as R
import torch_point_ops_b200 as tpo

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("dtype,wdtype", [(torch.float32, torch.float32), (torch.bfloat16, torch.float32),
                                          (torch.bfloat16, torch.bfloat16), (torch.float64, torch.float64)])
@pytest.mark.parametrize("width", [40, 42, 48, 200, 9001])
def test_gradient_of_constant_rows_of_large_values(width, dtype, wdtype):
    # mean * rstd is beyond the type's range, mean and (x - mean) * rstd are not
    g = torch.Generator().manual_seed(width)
    value = 2.0 ** (1016 if dtype == torch.float64 else 120)
    value *= 1.0 if width < 1000 else 2.0 ** -6  # the row's sum stays finite
    x = torch.full((6, width), value, device=DEV, dtype=dtype)
    # a power of two times whole numbers sums exactly; the reciprocal of the width must give the mean back
    size = torch.tensor(float(width), dtype=torch.promote_types(dtype, torch.float32))
    assert float(size * (1 / size)) == 1.0
    w, b = ((1 + torch.randn(width, generator=g) / 4).to(DEV, wdtype) for _ in range(2))
    dy = torch.randn(6, width, generator=g).to(DEV, dtype)
    leaves = [t.detach().requires_grad_() for t in (x, w, b)]
    got = dict(zip(("dx", "dw", "db"), torch.autograd.grad(tpo.layer_norm(*leaves), leaves, dy)))
    ref = R.layer_norm(torch.zeros_like(x), w, b, 1e-5, dy)  # centred, such rows are zeros
    for name, t in got.items():
        R.check(t, ref[name], name)


# one, several and many rows per block, registers and loops, whole vectors and single elements
WIDTHS = [100, 1000, 1001, 2000, 5000, 8192, 9001]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16, torch.float64])
@pytest.mark.parametrize("width", WIDTHS)
def test_constant_rows(width, dtype):
    # the exact result is 0: a mean off by one step of the type would be magnified by 1 / sqrt(eps)
    f = R.U[torch.float64 if dtype == torch.float64 else torch.float32]
    for value in (1000.0, 50000.0, 0.1, 4097.0):
        x = torch.full((9, width), value, device=DEV, dtype=dtype)
        value = float(x[0, 0])
        y = tpo.layer_norm(x).double()
        # the mean is off by ACC + 2 roundings of itself, what is left of that by as many of what it is
        assert (y.abs() <= ((R.ACC + 2) * f) ** 2 * value / 1e-5 ** 0.5).all(), float(y.abs().max())


@pytest.mark.parametrize("width", WIDTHS)
def test_rows_far_from_zero(width):
    # a spread of a hundredth around 1000; 64 bits of the same inputs
    g = torch.Generator().manual_seed(width)
    x = (1000 + 0.01 * torch.randn(50, width, generator=g)).to(DEV)
    d = x.double()
    mean = d.mean(1, keepdim=True)
    var = (d - mean).square().mean(1, keepdim=True)
    rstd = (var + 1e-5).rsqrt()
    want = (d - mean) * rstd
    # centring is exact here (both within a factor of two); the mean's two-step error as above; the variance's
    # sum, its root and the products are relative to the result
    bound = R.SLACK * (((R.ACC + 2) * R.F) ** 2 * 1000 * rstd + (R.ACC + 16) * R.F * (want.abs() + 1))
    assert ((tpo.layer_norm(x).double() - want).abs() <= bound).all()
    # and the backward's mean is rounded once, not ACC times
    _, m, _ = torch.ops.torch_point_ops_b200_norm.layer_norm_forward(x, None, None, 1e-5)
    assert ((m.double()[:, None] - mean).abs() <= 1.01 * R.F * mean).all()


def test_variance_beyond_the_range():
    # the squares overflow: an infinite variance, not a NaN
    for width in (64, 1000, 9001):
        x = (1e30 * (1 + torch.rand(4, width, generator=torch.Generator().manual_seed(1)))).to(DEV)
        assert torch.equal(tpo.layer_norm(x), torch.zeros_like(x))
