"""How near 16-bit packed attention comes to 64 bits, against what rounding the exact results to the
type costs by itself.

A sum over terms that were each rounded once is off by about as much as its own rounding (both are
relative, and random terms add up like the sum does): together sqrt(2).  That is what P costs o and
dv, and dS costs dk.  dq's dS has a second 16-bit value, so its own rounding is nearly all of it; one
value, or a delta from the rounded o alone in dk, would show (1.4 and more; 1.5 to 1.6)."""
import math

import pytest
import torch

import token_reference as R
import torch_point_ops_b200 as tpo

pytestmark = pytest.mark.gpu
DEV = "cuda"
MOST = {"o": 1.5, "dq": 1.25, "dk": 1.5, "dv": 1.5}


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("causal", [False, True])
def test_root_mean_square_error(causal, D, dtype):
    g = torch.Generator().manual_seed(D)
    off = [0, 500, 1500]
    q, k, v, do = (torch.randn(off[-1], h, D, generator=g).to(DEV, dtype) for h in (4, 2, 2, 4))
    leaves = [t.detach().requires_grad_() for t in (q, k, v)]
    o = tpo.packed_attention(*leaves, torch.tensor(off, device=DEV), causal=causal)
    got = dict(zip(MOST, [o.detach(), *torch.autograd.grad(o, leaves, do)]))
    ref = R.packed(q, k, v, off, off, causal, 1 / math.sqrt(D), do)
    ratio = {}
    for name, t in got.items():
        exact = ref[name][0]
        own = (exact.to(dtype).double() - exact).square().mean().sqrt()
        ratio[name] = float((t.double() - exact).square().mean().sqrt() / own)
    assert all(ratio[n] <= MOST[n] for n in MOST), ratio
    print(ratio)
