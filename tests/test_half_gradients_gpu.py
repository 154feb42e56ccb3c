"""float16 gradients of packed attention over the type's range: large and small values, long clouds.

The kernels hold P and dS in 16 bits beside a power of two, so multiplying v or the gradient by a
power of two must multiply the results by it, bit for bit where they stay normal numbers."""
import math

import pytest
import torch

import token_reference as R
import torch_point_ops_b200 as tpo

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _gradients(q, k, v, do, offsets, offsets_k=None, causal=False):
    leaves = [t.detach().requires_grad_() for t in (q, k, v)]
    o = tpo.packed_attention(*leaves, torch.tensor(offsets, device=DEV),
                             None if offsets_k is None else torch.tensor(offsets_k, device=DEV), causal)
    return dict(zip(("dq", "dk", "dv"), torch.autograd.grad(o, leaves, do)))


def _inputs(T, H, Hk, D, seed=0):
    g = torch.Generator().manual_seed(seed + T + D)
    return [torch.randn(T, h, D, generator=g).to(DEV, torch.float16) for h in (H, Hk, Hk, H)]


@pytest.mark.parametrize("D", [40, 64, 128])
@pytest.mark.parametrize("size", [100.0, 1200.0, 3000.0, 10000.0])
def test_aligned_rows_of_large_values(size, D):
    # rows of v with one sign each and a constant gradient: the largest dS that these sizes can give
    T = 150
    q, k, v, do = _inputs(T, 2, 1, D)
    sign = torch.where(torch.arange(T, device=DEV) % 3 == 0, -1.0, 1.0)
    v = (size * sign)[:, None, None].expand(T, 1, D).half().contiguous()
    do = torch.full_like(do, 2.0 ** -10)
    off = [0, 2, T]  # a cloud of two keys too
    for causal in (False, True):
        ref = R.packed(q, k, v, off, off, causal, 1 / math.sqrt(D), do)
        for name, t in _gradients(q, k, v, do, off, causal=causal).items():
            assert torch.isfinite(t).all(), name
            R.check(t, ref[name], name)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("by_v,by_do", [(2.0 ** -10, 1.0), (2.0 ** 8, 2.0 ** -6), (1.0, 2.0 ** -8), (2.0 ** 11, 2.0 ** -12),
                                        (2.0 ** -6, 2.0 ** 6), (2.0 ** 4, 2.0 ** 4)])
def test_powers_of_two_pass_through(by_v, by_do, causal, D):
    q, k, v, do = _inputs(700, 4, 2, D)
    # few bits, so that no factor rounds an input; v of one sign, so that no output is subnormal
    v, do = 1 + (v.abs() * 64).round() / 64, (do * 64).round() / 64
    off = [0, 300, 333, 700]
    base = _gradients(q, k, v, do, off, causal=causal)
    got = _gradients(q, k, v * by_v, do * by_do, off, causal=causal)
    for name, f in (("dq", by_v * by_do), ("dk", by_v * by_do), ("dv", by_do)):
        # subnormal results are rounded to half a step there and to half a step here; others not at all
        assert ((got[name].double() - base[name].double() * f).abs() <= 2.0 ** -24 * max(f, 1.0)).all(), name


def test_one_large_row_among_small_ones():
    # a cloud's scale is its own: its neighbour holds values 2^14 times as large
    q, k, v, do = _inputs(400, 2, 2, 64)
    alone = _gradients(q[:200], k[:200], v[:200], do[:200], [0, 200])
    v[200:] *= 2.0 ** 14
    both = _gradients(q, k, v, do, [0, 200, 400])
    for name, t in alone.items():
        assert torch.equal(both[name][:200], t), name
    # an unseen token of no cloud likewise
    v[200:] = float("inf")
    some = _gradients(q, k, v, do, [0, 200])
    for name, t in alone.items():
        assert torch.equal(some[name][:200], t), name


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("keys", [300, 50000, 99000])
def test_gradient_of_values_of_long_clouds(keys, D):
    # flat rows: every probability is 1 / keys, far below the smallest normal number for many keys
    rows, each = 2048, 16.0
    q = torch.zeros(rows, 1, D, device=DEV, dtype=torch.float16)
    _, k, v, _ = _inputs(keys, 1, 1, D)
    do = torch.full_like(q, each)
    dv = _gradients(q, k, v, do, [0, rows], [0, keys])["dv"].double()
    want = rows * each / keys
    # one rounding of P, one of the result, each 2^-11 at most; fp32: the log-sum-exp's three roundings
    # and the sum over the rows (a chain of rows / 8 and a tree)
    off = 2 * 2.0 ** -11 + (3 * math.log2(keys) + rows / 8 + 64) * R.F
    assert ((dv - want).abs() <= off * want).all(), float((dv / want - 1).abs().max())


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("before", [0, 300])
def test_keys_that_are_not_seen_leave_the_scale_alone(before, D):
    # later keys of a causal cloud hold values 2^12 times as large: tiles of queries that see none of them
    q, k, v, do = _inputs(700, 2, 1, D)
    rows = 700 - before  # so many queries, the last ones
    off, off_k = [0, rows], [0, 700]
    args = lambda v: (q[:rows], k, v, do[:rows], off, off_k, True)
    base = _gradients(*args(v))["dq"]
    last = 512 - before  # queries below see keys below 512 only, and start tiles of their own
    v = v.clone()
    v[512:] *= 2.0 ** 12
    seen = last // 128 * 128
    got = _gradients(*args(v))["dq"]
    assert seen > 0 and torch.equal(got[:seen], base[:seen])
    assert torch.isfinite(got).all()


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("rows,keys", [(1, 3000), (3, 1000), (5, 130), (200, 5000)])
def test_few_rows_over_many_tiles_of_large_values(rows, keys, D):
    # the largest value of the last tile counts, however few queries there are
    q, k, v, do = _inputs(keys, 2, 1, D)
    v[-1] = 4000.0
    v[-2] = -4000.0
    k[-2:] = 3 * q[0, 0]  # and it is attended to
    do = torch.full_like(do, 2.0 ** -9)
    ref = R.packed(q[:rows], k, v, [0, rows], [0, keys], True, 1 / math.sqrt(D), do[:rows])
    for name, t in _gradients(q[:rows], k, v, do[:rows], [0, rows], [0, keys], True).items():
        assert torch.isfinite(t).all(), name
        R.check(t, ref[name], name)
