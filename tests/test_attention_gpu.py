"""Attention over packed clouds and over a cache against a plain 64-bit implementation
with element-wise bounds (token_reference.py)."""
import math

import pytest
import torch

import capi_util as C
import token_reference as R
import torch_point_ops_b200 as tpo

pytestmark = pytest.mark.gpu
DEV = "cuda"
TYPES = [torch.float32, torch.float16, torch.bfloat16]


def _offsets(lengths):
    return torch.tensor([0] + list(lengths)).cumsum(0)


def _packed_inputs(lq, lk, H, Hk, D, dtype, seed=0, grow=1.0):
    g = torch.Generator().manual_seed(seed + 7 * sum(lq) + D)
    q = torch.randn(sum(lq), H, D, generator=g) * grow
    k, v = (torch.randn(sum(lk), Hk, D, generator=g) * s for s in (grow, 1.0))
    do = torch.randn(sum(lq), H, D, generator=g)
    return [t.to(DEV, dtype) for t in (q, k, v, do)]


def _check_packed(q, k, v, do, offsets, offsets_k, causal, scale=None):
    leaves = [t.detach().requires_grad_() for t in (q, k, v)]
    o = tpo.packed_attention(*leaves, offsets.to(DEV), None if offsets_k is None else offsets_k.to(DEV), causal, scale)
    dq, dk, dv = torch.autograd.grad(o, leaves, do)
    ref = R.packed(q, k, v, offsets, offsets if offsets_k is None else offsets_k, causal,
                   scale or 1 / math.sqrt(q.shape[-1]), do)
    got = {"o": o.detach(), "dq": dq, "dk": dk, "dv": dv}
    for name, t in got.items():
        assert t.dtype == q.dtype
        R.check(t, ref[name], name)
    with torch.no_grad():
        alone = tpo.packed_attention(q, k, v, offsets.to(DEV), None if offsets_k is None else offsets_k.to(DEV), causal, scale)
    assert torch.equal(alone, o)
    return got


# lengths at and around the kernels' tiles of 64, 128 and 256 rows, empty clouds first, last and between
LENGTHS = [[1], [2, 1, 3], [63, 64, 65], [127, 1, 128, 129], [0, 5, 0, 0, 200, 0], [255, 257, 31], [513], [40] * 37]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("lengths", LENGTHS, ids=str)
def test_lengths(lengths, causal, dtype):
    args = _packed_inputs(lengths, lengths, 4, 2, 64, dtype)
    _check_packed(*args, _offsets(lengths), None, causal)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("D", [1, 3, 8, 24, 33, 40, 64, 72, 80, 96, 104, 128, 130, 136, 200, 256])
def test_widths(D, dtype):
    lengths = [70, 0, 190, 3]
    args = _packed_inputs(lengths, lengths, 2, 1, D, dtype)
    for causal in (False, True):
        _check_packed(*args, _offsets(lengths), None, causal)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("H,Hk", [(1, 1), (3, 3), (6, 2), (8, 1), (12, 4)])
def test_heads(H, Hk, dtype):
    lengths = [150, 20]
    args = _packed_inputs(lengths, lengths, H, Hk, 128, dtype)
    _check_packed(*args, _offsets(lengths), None, True)


# keys before the queries, fewer keys than queries (causal: the first rows see nothing), none at all
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("lq,lk", [([5, 1, 130], [70, 300, 131]), ([200, 64, 10], [3, 0, 9]), ([0, 300], [40, 140]),
                                   ([1, 1, 1], [1, 500, 0]), ([0], [9]), ([400], [129])], ids=str)
def test_lengths_of_keys(lq, lk, causal, dtype):
    args = _packed_inputs(lq, lk, 4, 2, 64, dtype)
    _check_packed(*args, _offsets(lq), _offsets(lk), causal)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("D", [64, 128])
def test_long(D, dtype):
    lengths = [1500, 700]
    args = _packed_inputs(lengths, lengths, 2, 1, D, dtype)
    for causal in (False, True):
        _check_packed(*args, _offsets(lengths), None, causal)


@pytest.mark.parametrize("dtype", TYPES)
def test_peaked_and_flat_scores(dtype):
    lengths = [300, 77]
    for grow in (4.0, 0.01):  # scores of +-100 after the scale, and all alike
        args = _packed_inputs(lengths, lengths, 2, 2, 64, dtype, grow=grow)
        _check_packed(*args, _offsets(lengths), None, True)
    args = _packed_inputs(lengths, lengths, 2, 2, 64, dtype)
    _check_packed(*args, _offsets(lengths), None, False, scale=0.5)
    # every row's maximum grows with the key: the running maximum moves in each tile
    q, k, v, do = _packed_inputs([600], [600], 1, 1, 64, dtype)
    q.fill_(1.0), k.copy_((torch.arange(600, device=DEV) / 64)[:, None, None].expand_as(k))
    _check_packed(q, k, v, do, _offsets([600]), None, True)


@pytest.mark.parametrize("scale", [2.0 ** -14, 2.0 ** 6])
def test_small_and_large_gradients_in_half(scale):
    # dS of fp16 must not drown in the type's smallest step, nor overflow
    q, k, v, do = _packed_inputs([700], [700], 2, 1, 64, torch.float16)
    leaves = [t.detach().requires_grad_() for t in (q, k, v)]
    off = _offsets([700])
    grads = torch.autograd.grad(tpo.packed_attention(*leaves, off.to(DEV)), leaves, (do * scale).half())
    ref = R.packed(q, k, v, off, off, False, 0.125, (do * scale).half())
    for name, t in zip(("dq", "dk", "dv"), grads):
        R.check(t, ref[name], name)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("D", [64, 128, 40])
def test_neighbours_hold_anything(D, dtype):
    # a cloud between two that are full of NaN and infinities
    lengths = [50, 90, 200]
    q, k, v, do = _packed_inputs(lengths, lengths, 2, 1, D, dtype)
    off = _offsets(lengths)
    bad = [t.clone() for t in (q, k, v, do)]
    for t in bad:
        t[:50], t[140:] = float("nan"), float("inf")
    for causal in (False, True):
        def run(a):
            leaves = [t.detach().requires_grad_() for t in a[:3]]
            o = tpo.packed_attention(*leaves, off.to(DEV), causal=causal)
            return [o.detach()] + list(torch.autograd.grad(o, leaves, a[3]))
        for a, b in zip(run([q, k, v, do]), run(bad)):
            assert torch.equal(a[50:140], b[50:140])


@pytest.mark.parametrize("dtype", TYPES)
def test_tokens_of_no_cloud(dtype):
    # a buffer with room before the first and after the last cloud, full of NaN there
    q, k, v, do = _packed_inputs([700], [700], 2, 2, 64, dtype)
    off = torch.tensor([100, 130, 400])
    for t in (q, k, v, do):
        t[:100], t[400:] = float("nan"), float("nan")
    got = _check_packed(q, k, v, do, off, None, True)
    for t in got.values():
        assert torch.equal(t[:100], torch.zeros_like(t[:100])) and torch.equal(t[400:], torch.zeros_like(t[400:]))
    flags = C.ctypes.c_uint(0)
    assert C.lib().tpo_device_error_flags(C.ctypes.byref(flags), 1) == 0 and flags.value == 0


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("D", [64, 96, 33])
def test_strides(D, dtype):
    # slices of one projection, heads before tokens, a broadcast key head, a strided width
    lengths = [90, 35, 128]
    T, off = sum(lengths), _offsets(lengths)
    g = torch.Generator().manual_seed(D)
    qkv = torch.randn(T, 3, 4, D, generator=g).to(DEV, dtype)
    do = torch.randn(4, T, D, generator=g).to(DEV, dtype).transpose(0, 1)
    _check_packed(qkv[:, 0], qkv[:, 1], qkv[:, 2], do, off, None, True)
    ht = torch.randn(3, 4, T, D, generator=g).to(DEV, dtype)
    _check_packed(ht[0].transpose(0, 1), ht[1].transpose(0, 1), ht[2].transpose(0, 1), do, off, None, False)
    one = torch.randn(T, 1, D, generator=g).to(DEV, dtype)
    _check_packed(qkv[:, 0], one.expand(T, 4, D), one.expand(T, 4, D), do, off, None, True)
    wide = torch.randn(T, 4, 2 * D, generator=g).to(DEV, dtype)
    _check_packed(wide[..., ::2], qkv[:, 1], wide[..., 1::2], wide[..., :D], off, None, False)
    odd = torch.randn(T * 4 * D + 1, generator=g).to(DEV, dtype)[1:].view(T, 4, D)  # rows off the 16-byte grid
    _check_packed(odd, qkv[:, 1], odd, do, off, None, True)


def test_gradient_of_a_broadcast_input():
    off = _offsets([60, 40])
    q, k, v, do = _packed_inputs([60, 40], [60, 40], 4, 1, 32, torch.float32)
    shared = k.detach().requires_grad_()
    many = tpo.packed_attention(q, shared.expand(100, 4, 32), v.expand(100, 4, 32), off.to(DEV))
    (a,) = torch.autograd.grad(many, shared, do)
    (b,) = torch.autograd.grad(tpo.packed_attention(q, shared, v, off.to(DEV)), shared, do)
    ref = R.packed(q, k, v, off, off, False, 1 / math.sqrt(32), do)["dk"]
    R.check(b, ref)
    R.check(a, (ref[0], 4 * ref[1]))  # four gradients rounded and then summed


def test_gradients_that_are_not_wanted():
    off = _offsets([80]).to(DEV)
    q, k, v, do = _packed_inputs([80], [80], 2, 2, 64, torch.bfloat16)
    full = [t.detach().requires_grad_() for t in (q, k, v)]
    want = torch.autograd.grad(tpo.packed_attention(*full, off), full, do)
    for i in range(3):
        leaves = [t.detach().requires_grad_(j == i) for j, t in enumerate((q, k, v))]
        (g,) = torch.autograd.grad(tpo.packed_attention(*leaves, off), leaves[i], do)
        assert torch.equal(g, want[i])


def test_differences():
    """Directional central differences of the operator: D(h) is off the derivative by about
    |D(2h) - D(h)| / 3 (the next term falls by 4 per halving; doubled below) and by the outputs' own error over h."""
    lengths = [20, 45]
    off = _offsets(lengths)
    q, k, v, do = _packed_inputs(lengths, lengths, 4, 2, 24, torch.float32)
    grads = torch.autograd.grad(tpo.packed_attention(*(leaves := [t.detach().requires_grad_() for t in (q, k, v)]),
                                                     off.to(DEV), causal=True), leaves, do)
    noise = float((R.packed(q, k, v, off, off, True, 1 / math.sqrt(24))["o"][1] * do.double().abs()).sum())
    g = torch.Generator().manual_seed(5)
    for i in range(3):
        way = torch.randn((q, k, v)[i].shape, generator=g).to(DEV)
        way = way / way.norm()

        def loss(h):
            args = [q, k, v]
            args[i] = args[i] + h * way
            # the step that was really taken
            return float((tpo.packed_attention(*args, off.to(DEV), causal=True).double() * do.double()).sum())

        h = 2.0 ** -4
        d1, d2 = ((loss(s) - loss(-s)) / (2 * s) for s in (h, 2 * h))
        exact = float((grads[i].double() * way.double()).sum())
        # inputs after the step are rounded to fp32 too: F * |x| per element, through the gradient
        rounding = R.F * float((grads[i].double().abs() * ((q, k, v)[i].double().abs() + 1)).sum()) / h
        assert abs(d1 - exact) <= 2 * abs(d2 - d1) / 3 + noise / h + rounding


@pytest.mark.parametrize("dtype", TYPES)
def test_same_bits_every_run_and_on_another_stream(dtype):
    lengths = [400, 33, 250]
    off = _offsets(lengths).to(DEV)
    q, k, v, do = _packed_inputs(lengths, lengths, 4, 2, 64, dtype)

    def run():
        leaves = [t.detach().requires_grad_() for t in (q, k, v)]
        o = tpo.packed_attention(*leaves, off, causal=True)
        return [o.detach()] + list(torch.autograd.grad(o, leaves, do))

    first = run()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        second = run()
    torch.cuda.current_stream().wait_stream(s)
    assert all(torch.equal(a, b) for a, b in zip(first, second))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_graph_capture_with_new_lengths(dtype):
    # the captured launch must not depend on the lengths: they change between replays
    q, k, v, _ = _packed_inputs([500], [500], 2, 1, 64, dtype)
    off = torch.tensor([0, 100, 100, 500], device=DEV)
    tpo.packed_attention(q, k, v, off, causal=True)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        o = tpo.packed_attention(q, k, v, off, causal=True)
    for new in ([0, 250, 251, 480], [0, 0, 500, 500]):
        off.copy_(torch.tensor(new))
        graph.replay()
        R.check(o, R.packed(q, k, v, new, new, True, 0.125)["o"])


def test_int32_and_host_offsets():
    q, k, v, _ = _packed_inputs([60, 40], [60, 40], 2, 2, 64, torch.float32)
    off = _offsets([60, 40])
    want = tpo.packed_attention(q, k, v, off.to(DEV))
    assert torch.equal(tpo.packed_attention(q, k, v, off.int().to(DEV)), want)
    assert torch.equal(tpo.packed_attention(q, k, v, off), want)
    assert torch.equal(tpo.packed_offsets(torch.tensor([60, 40])), off)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("bad", [[0, 90, 40, 100], [0, 50, 1000], [-7, 50, 100], [0, 2 ** 40, 100]], ids=str)
def test_bad_offsets_are_flagged(bad, dtype):
    q, k, v, do = _packed_inputs([100], [100], 2, 2, 64, dtype)
    leaves = [t.detach().requires_grad_() for t in (q, k, v)]
    o = tpo.packed_attention(*leaves, torch.tensor(bad, device=DEV), causal=True)
    torch.autograd.grad(o, leaves, do)
    flags = C.ctypes.c_uint(0)
    assert C.lib().tpo_device_error_flags(C.ctypes.byref(flags), 1) == 0 and flags.value == 4
    assert C.lib().tpo_device_error_flags(C.ctypes.byref(flags), 0) == 0 and flags.value == 0


def test_packed_refusals():
    q = torch.randn(10, 4, 16, device=DEV)
    k = torch.randn(10, 2, 16, device=DEV)
    off = torch.tensor([0, 10], device=DEV)
    bad = [(q, k, k[:9], off), (q, k, k.half(), off), (q, k[..., :8], k[..., :8], off), (q[0], k, k, off),
           (q[:, :3], k, k, off), (q, k[:, :0], k[:, :0], off), (q.double(), k.double(), k.double(), off),
           (q.int(), k.int(), k.int(), off), (q, k, k, off.float()), (q, k, k, off[None]), (q, k, k, off[:0]),
           (q, k[:9], k[:9], off), (q, k, k, off, torch.tensor([0, 5, 10], device=DEV)), (q, k.cpu(), k, off),
           (torch.randn(10, 4, 257, device=DEV),) * 3 + (off,)]
    for args in bad:
        with pytest.raises(RuntimeError):
            tpo.packed_attention(*args)
    with pytest.raises((RuntimeError, NotImplementedError)):
        tpo.packed_attention(q.cpu(), k.cpu(), k.cpu(), off.cpu())
    for scale in (0.0, -1.0, float("inf"), float("nan")):
        with pytest.raises(ValueError):
            tpo.packed_attention(q, k, k, off, scale=scale)


def test_second_differentiation_raises():
    q = torch.randn(10, 2, 16, device=DEV, requires_grad=True)
    off = torch.tensor([0, 10], device=DEV)
    (g,) = torch.autograd.grad(tpo.packed_attention(q, q, q, off).square().sum(), q, create_graph=True)
    with pytest.raises(RuntimeError, match="second differentiation"):
        torch.autograd.grad(g.sum(), q)


def test_module():
    q, k, v, _ = _packed_inputs([30], [30], 2, 1, 32, torch.float32)
    off = _offsets([30]).to(DEV)
    assert torch.equal(tpo.PackedAttention(causal=True, scale=0.3)(q, k, v, off),
                       tpo.packed_attention(q, k, v, off, causal=True, scale=0.3))
    with pytest.raises(ValueError):
        tpo.PackedAttention(scale=-1.0)


# ------------------------------------------------------------------ cache
def _cached_inputs(N, P, H, Hk, D, dtype, seed=0):
    g = torch.Generator().manual_seed(seed + P * 3 + D)
    return [torch.randn(s, generator=g).to(DEV, dtype) for s in ((N, H, D), (N, P, Hk, D), (N, P, Hk, D))]


def _check_cached(q, k, v, lengths, scale=None):
    o = tpo.cached_attention(q, k, v, torch.tensor(lengths, device=DEV), scale)
    assert o.dtype == q.dtype
    R.check(o, R.cached(q, k, v, lengths, scale or 1 / math.sqrt(q.shape[-1]))["o"])
    return o


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("P,lengths", [(1, [1, 0]), (16, [16, 15, 1, 0]), (17, [17, 8]), (130, [130, 128, 129, 127]),
                                       (1000, [1000, 3, 0, 513]), (5000, [5000, 4097])], ids=str)
def test_cached_lengths(P, lengths, dtype):
    _check_cached(*_cached_inputs(len(lengths), P, 4, 2, 64, dtype), lengths)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("D", [1, 7, 8, 24, 32, 40, 64, 80, 96, 120, 128, 136, 200, 255, 256])
def test_cached_widths(D, dtype):
    _check_cached(*_cached_inputs(2, 300, 4, 2, D, dtype), [300, 41])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("H,Hk", [(1, 1), (2, 1), (3, 1), (4, 4), (5, 1), (8, 1), (9, 3), (16, 1), (24, 1), (40, 2)])
def test_cached_heads(H, Hk, dtype):
    _check_cached(*_cached_inputs(2, 200, H, Hk, 128, dtype), [200, 77])


@pytest.mark.parametrize("dtype", TYPES)
def test_cached_split_axis(dtype):
    _check_cached(*_cached_inputs(1, 40000, 4, 1, 64, dtype), [39001])
    _check_cached(*_cached_inputs(3, 9000, 2, 2, 128, dtype), [9000, 0, 1])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("D", [64, 128, 33])
def test_cached_unwritten_slots_hold_anything(D, dtype):
    q, k, v = _cached_inputs(3, 700, 4, 2, D, dtype)
    lengths = [500, 0, 33]
    want = _check_cached(q, k, v, lengths)
    for n, length in enumerate(lengths):
        k[n, length:], v[n, length:] = float("nan"), float("inf")
    assert torch.equal(_check_cached(q, k, v, lengths), want)
    assert torch.equal(want[1], torch.zeros_like(want[1]))


@pytest.mark.parametrize("dtype", TYPES)
def test_cached_strides_and_lengths_out_of_range(dtype):
    q, k, v = _cached_inputs(2, 90, 4, 4, 64, dtype)
    want = _check_cached(q, k, v, [90, 17])
    heads_first = [t.transpose(1, 2).contiguous().transpose(1, 2) for t in (k, v)]
    assert torch.equal(tpo.cached_attention(q, *heads_first, torch.tensor([90, 17], device=DEV)), want)
    both = torch.stack([k, v], 2)
    assert torch.equal(tpo.cached_attention(q, both[:, :, 0], both[:, :, 1], torch.tensor([90, 17], device=DEV)), want)
    assert torch.equal(tpo.cached_attention(q, k, v, torch.tensor([1000, 17], device=DEV, dtype=torch.int32)), want)
    assert not tpo.cached_attention(q, k, v, torch.tensor([-5, 17], device=DEV))[0].any()
    odd = torch.randn(2 * 90 * 4 * 64 + 1, device=DEV).to(dtype)[1:].view(2, 90, 4, 64)
    _check_cached(q, odd, odd, [90, 17])
    wide = torch.randn(2, 90, 4, 128, device=DEV).to(dtype)
    _check_cached(q, wide[..., ::2], wide[..., 1::2], [90, 17])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("H,Hk,D", [(4, 2, 64), (20, 1, 128), (6, 2, 200), (3, 3, 33)])
@pytest.mark.parametrize("P", [32, 65, 127, 129, 255, 257, 513, 1024, 1025])
def test_cached_short_axes(P, H, Hk, D, dtype):
    # lengths that end in each part of the axis, leave parts empty, or all of it
    lengths = [P, 1, 0, P // 2 + 1, P - 1, P // 8]
    q, k, v = _cached_inputs(len(lengths), P, H, Hk, D, dtype)
    for n, length in enumerate(lengths):
        k[n, length:], v[n, length:] = math.nan, math.inf
    want = _check_cached(q, k, v, lengths)
    for _ in range(20):  # and the same bits each time
        assert torch.equal(tpo.cached_attention(q, k, v, torch.tensor(lengths, device=DEV)), want)


def test_cached_offsets_beyond_32_bits():
    # the last cloud's cache starts 2.2e9 elements into the tensor
    P, N = 70000, 250
    k = torch.zeros(N, P, 1, 128, dtype=torch.bfloat16, device=DEV)
    tail = torch.randn(2, 300, 128, device=DEV).to(torch.bfloat16)
    k[N - 1, P - 300:, 0], k[0, :300, 0] = tail[0], tail[1]
    q = torch.randn(N, 2, 128, device=DEV).to(torch.bfloat16)
    o = tpo.cached_attention(q, k, k, torch.full((N,), P, device=DEV))
    for n in (0, N - 1):
        R.check(o[n:n + 1], R.cached(q[n:n + 1], k[n:n + 1], k[n:n + 1], [P], 1 / math.sqrt(128))["o"])


def test_cached_matches_packed():
    # one token over a cache is the last row of causal attention
    q, k, v = _cached_inputs(1, 333, 8, 2, 64, torch.float32)
    o = tpo.cached_attention(q, k, v, torch.tensor([333], device=DEV))
    packed = tpo.packed_attention(q, k[0], v[0], torch.tensor([0, 1], device=DEV), torch.tensor([0, 333], device=DEV), causal=True)
    ref = R.cached(q, k, v, [333], 0.125)["o"]
    R.check(o, ref), R.check(packed, ref)


def test_cached_graph_capture_with_new_lengths():
    q, k, v = _cached_inputs(2, 3000, 4, 2, 64, torch.bfloat16)
    lengths = torch.tensor([5, 3000], device=DEV)
    tpo.cached_attention(q, k, v, lengths)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        o = tpo.cached_attention(q, k, v, lengths)
    for new in ([2000, 6], [0, 1]):
        lengths.copy_(torch.tensor(new))
        graph.replay()
        R.check(o, R.cached(q, k, v, new, 0.125)["o"])


def test_cached_refusals():
    q, k, v = _cached_inputs(2, 10, 4, 2, 16, torch.float32)
    n = torch.tensor([3, 4], device=DEV)
    for args in ((q, k, v[:, :9], n), (q, k.half(), v, n), (q[:1], k, v, n), (q[:, :3], k, v, n), (q, k, v, n[:1]),
                 (q, k, v, n.float()), (q[0], k, v, n), (q.double(), k.double(), v.double(), n),
                 (torch.randn(2, 4, 300, device=DEV), torch.randn(2, 5, 4, 300, device=DEV), torch.randn(2, 5, 4, 300, device=DEV), n)):
        with pytest.raises(RuntimeError):
            tpo.cached_attention(*args)
    with pytest.raises(RuntimeError, match="no backward"):
        tpo.cached_attention(q.requires_grad_(), k, v, n)
    with pytest.raises(ValueError):
        tpo.cached_attention(q.detach(), k, v, n, scale=0.0)
    assert tpo.cached_attention(q[:0].detach(), k[:0], v[:0], n[:0]).shape == (0, 4, 16)
    assert not tpo.cached_attention(q.detach(), k[:, :0], v[:, :0], n).any()
