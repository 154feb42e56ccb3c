"""Packed attention where offsets, counts and shapes grow: element offsets beyond 32 bits, more
clouds than a warp holds, long clouds beside many empty ones."""
import math

import pytest
import torch

import token_reference as R
import torch_point_ops_b200 as tpo

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _run(q, k, v, do, off, off_k, causal):
    leaves = [t.detach().requires_grad_() for t in (q, k, v)]
    o = tpo.packed_attention(*leaves, off, off_k, causal)
    return dict(zip(("o", "dq", "dk", "dv"), [o.detach()] + list(torch.autograd.grad(o, leaves, do))))


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
def test_element_offsets_beyond_32_bits(dtype):
    # 300 tokens 8 million elements apart: the last ones lie 2.4e9 elements into the buffer
    T, hop = 300, 8_000_000
    buffer = torch.empty(hop * (T - 1) + 4 * 128, dtype=dtype, device=DEV)
    views = [buffer.as_strided((T, 2, 64), (hop, 64, 1), 128 * i) for i in range(4)]
    g = torch.Generator().manual_seed(0)
    small = [torch.randn(T, 2, 64, generator=g).to(DEV, dtype) for _ in range(4)]
    for view, t in zip(views, small):
        view.copy_(t)
    off = torch.tensor([0, 170, T], device=DEV)
    far, near = _run(*views, off, None, True), _run(*small, off, None, True)
    for name in near:
        assert torch.equal(far[name], near[name]), name
    ref = R.packed(*small[:3], [0, 170, T], [0, 170, T], True, 0.125, small[3])
    for name, t in near.items():
        R.check(t, ref[name], name)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("clouds", [28, 29, 30, 31, 32, 33, 1100])
def test_many_clouds(clouds, causal, dtype):
    g = torch.Generator().manual_seed(clouds)
    lengths = torch.randint(0, 9, (clouds,), generator=g)
    lengths[clouds // 2], lengths[-1] = 300, 140
    more = lengths + torch.randint(-2, 3, (clouds,), generator=g)
    off, off_k = tpo.packed_offsets(lengths), tpo.packed_offsets(more.clamp(min=0))
    q, do = (torch.randn(int(off[-1]), 2, 64, generator=g).to(DEV, dtype) for _ in range(2))
    k, v = (torch.randn(int(off_k[-1]), 1, 64, generator=g).to(DEV, dtype) for _ in range(2))
    got = _run(q, k, v, do, off.to(DEV), off_k.to(DEV), causal)
    ref = R.packed(q, k, v, off, off_k, causal, 0.125, do)
    for name, t in got.items():
        R.check(t, ref[name], name)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_no_clouds_and_no_tokens(dtype):
    q = torch.randn(70, 2, 64, device=DEV).to(dtype)
    none = _run(q, q, q, q, torch.tensor([0], device=DEV), None, True)  # tokens, but no cloud
    assert all(torch.equal(t, torch.zeros_like(t)) for t in none.values())
    empty = q[:0]
    assert all(t.shape == (0, 2, 64) for t in _run(empty, empty, empty, empty, torch.tensor([0, 0], device=DEV), None, True).values())
    # queries without keys, keys without queries
    got = _run(q, empty, empty, q, torch.tensor([0, 70], device=DEV), torch.tensor([0, 0], device=DEV), False)
    assert not got["o"].any() and not got["dq"].any()
    got = _run(empty, q, q, empty, torch.tensor([0, 0], device=DEV), torch.tensor([0, 70], device=DEV), False)
    assert not got["dk"].any() and not got["dv"].any() and got["dk"].shape == q.shape


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
def test_one_long_cloud(dtype):
    # 20000 tokens: hundreds of steps of the running maximum and sum; rows checked on a sample
    T = 20000
    g = torch.Generator().manual_seed(3)
    q, k, v = (torch.randn(T, 1, 64, generator=g).to(DEV, dtype) for _ in range(3))
    off = torch.tensor([0, T], device=DEV)
    with torch.no_grad():
        o = tpo.packed_attention(q, k, v, off, causal=True)
    for row in (0, 1, 63, 127, 128, 255, 256, 5000, 12345, T - 1):
        seen = torch.ones(1, row + 1, dtype=torch.bool, device=DEV)
        ref = R.attend(q[row:row + 1, 0], k[:row + 1, 0], v[:row + 1, 0], seen, 1 / math.sqrt(64))["o"]
        R.check(o[row:row + 1, 0], ref, f"row {row}")
