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
