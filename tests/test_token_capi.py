"""C ABI of the token operators: argument checks (no kernel is launched, CPU only), and the
entry points driven without torch's binding (GPU)."""
import ctypes
import math

import pytest
import torch

import token_reference as R
from capi_util import I64, VP, lib, p, stream

F = ctypes.c_float
DT = {torch.float32: 0, torch.float16: 1, torch.float64: 2, torch.bfloat16: 3}


class Packed(ctypes.Structure):
    _fields_ = [("dtype", ctypes.c_int), ("causal", ctypes.c_int)] + [
        (n, I64) for n in ("clouds", "heads", "kv_heads", "width", "tokens_q", "tokens_k")] + [
        ("offsets_q", VP), ("offsets_k", VP), ("scale", F), ("q", VP), ("k", VP), ("v", VP)] + [
        (n, I64) for n in ("q_token_stride", "q_head_stride", "k_token_stride", "k_head_stride", "v_token_stride",
                           "v_head_stride")]


def _size(name, *args):
    f = getattr(lib(), name)
    f.restype = ctypes.c_size_t
    return f(*args)


def _good():
    return dict(dtype=0, causal=1, clouds=1, heads=4, kv_heads=2, width=16, tokens_q=8, tokens_k=8, offsets_q=16,
                offsets_k=16, scale=0.25, q=16, k=16, v=16, q_token_stride=64, q_head_stride=16, k_token_stride=32,
                k_head_stride=16, v_token_stride=32, v_head_stride=16)


@pytest.mark.parametrize("change,status", [
    (dict(dtype=2), 1), (dict(dtype=7), 1), (dict(clouds=-1), 1), (dict(tokens_q=-1), 1), (dict(tokens_k=2 ** 31), 1),
    (dict(heads=3), 1), (dict(heads=0), 1), (dict(kv_heads=0), 1), (dict(width=0), 1), (dict(width=257), 2),
    (dict(scale=0.0), 1), (dict(scale=-1.0), 1), (dict(scale=math.inf), 1), (dict(scale=math.nan), 1),
    (dict(q_token_stride=-1), 1), (dict(v_head_stride=-1), 1), (dict(offsets_q=None), 1), (dict(offsets_k=None), 1),
    (dict(q=None), 1), (dict(v=None), 1)], ids=str)
def test_packed_arguments(change, status):
    prob = Packed(**{**_good(), **change})
    assert lib().tpo_packed_attention_fwd(ctypes.byref(prob), VP(16), VP(0), VP(0)) == status
    assert len(lib().tpo_status_string(status)) > 10
    ws = ctypes.c_size_t(1 << 20)
    assert lib().tpo_packed_attention_bwd(ctypes.byref(prob), VP(16), VP(16), VP(16), I64(64), I64(16), VP(16), VP(16),
                                          VP(16), VP(256), ws, VP(0)) == status


def test_packed_outputs_and_workspace():
    good = Packed(**_good())
    L = lib()
    need = _size("tpo_packed_attention_bwd_workspace_size", I64(8), I64(4))
    assert need >= 2 * 8 * 4 * 4 and _size("tpo_packed_attention_bwd_workspace_size", I64(-1), I64(4)) == 0
    assert L.tpo_packed_attention_fwd(None, VP(16), VP(0), VP(0)) == 1
    assert L.tpo_packed_attention_fwd(ctypes.byref(good), VP(0), VP(0), VP(0)) == 1
    assert L.tpo_packed_attention_fwd(ctypes.byref(Packed(**{**_good(), "tokens_q": 0, "q": None})), VP(0), VP(0), VP(0)) == 0
    bwd = lambda dk, dv, ws, n: L.tpo_packed_attention_bwd(ctypes.byref(good), VP(16), VP(16), VP(16), I64(64), I64(16),
                                                           VP(16), VP(dk), VP(dv), VP(ws), ctypes.c_size_t(n), VP(0))
    assert bwd(16, 0, 256, need) == 1 and bwd(16, 16, 0, need) == 3 and bwd(16, 16, 256, need - 1) == 3
    assert bwd(16, 16, 264, need) == 3


def test_layer_norm_arguments():
    L = lib()
    fwd = lambda dt, wd, rows, width, eps=1e-5, x=16, y=16, xs=8, mean=16, rstd=16: L.tpo_layer_norm_fwd(
        dt, wd, VP(x), I64(xs), VP(16), VP(16), I64(rows), I64(width), ctypes.c_double(eps), VP(y), VP(mean), VP(rstd), VP(0))
    assert fwd(7, 0, 2, 8) == 1 and fwd(0, 1, 2, 8) == 1 and fwd(0, 2, 2, 8) == 1 and fwd(2, 0, 2, 8) == 1
    assert fwd(0, 0, -1, 8) == 1 and fwd(0, 0, 2, -8) == 1 and fwd(0, 0, 2, 2 ** 31) == 1 and fwd(0, 0, 2, 8, xs=-1) == 1
    assert fwd(0, 0, 2, 8, eps=-1.0) == 1 and fwd(0, 0, 2, 8, eps=math.nan) == 1
    assert fwd(0, 0, 2, 8, x=0) == 1 and fwd(0, 0, 2, 8, y=0) == 1 and fwd(0, 0, 2, 8, mean=0) == 1
    assert fwd(0, 0, 0, 8) == 0 and fwd(1, 0, 2, 0) == 0
    need = _size("tpo_layer_norm_bwd_workspace_size", 0, I64(50), I64(64))
    assert need > 0 and _size("tpo_layer_norm_bwd_workspace_size", 0, I64(0), I64(64)) == 0
    bwd = lambda ws, n, dy=16: L.tpo_layer_norm_bwd(0, 0, VP(16), I64(64), VP(dy), I64(64), VP(16), VP(16), VP(16), I64(50),
                                                    I64(64), VP(16), VP(16), VP(16), VP(ws), ctypes.c_size_t(n), VP(0))
    assert bwd(0, need) == 3 and bwd(16, need - 1) == 3 and bwd(24, need) == 3 and bwd(16, need, dy=0) == 1


def test_cached_arguments():
    L = lib()
    two, three = (I64 * 2)(64, 16), (I64 * 3)(512, 32, 16)
    bad = (I64 * 3)(512, -32, 16)

    def call(dtype=0, N=2, P=16, H=4, Hk=2, D=16, scale=0.25, q=16, k=16, lengths=16, o=16, ks=three, ws=16, n=1 << 24):
        return L.tpo_cached_attention(dtype, VP(q), two, VP(k), ks, VP(16), three, VP(lengths), I64(N), I64(P), I64(H),
                                      I64(Hk), I64(D), F(scale), VP(o), VP(ws), ctypes.c_size_t(n), VP(0))

    for change in (dict(dtype=2), dict(dtype=9), dict(N=-1), dict(N=70000), dict(P=-1), dict(H=3), dict(Hk=0), dict(D=0),
                   dict(scale=0.0), dict(scale=math.nan), dict(q=0), dict(k=0), dict(lengths=0), dict(o=0), dict(ks=bad)):
        assert call(**change) == 1, change
    assert call(D=300) == 2
    need = _size("tpo_cached_attention_workspace_size", I64(1), I64(4), I64(2), I64(100000), I64(16))
    assert need > 0 and call(N=1, P=100000, ws=0) == 3 and call(N=1, P=100000, n=need - 1) == 3
    assert call(N=0) == 0


def test_shapes_under_fake_tensors():
    from torch._subclasses.fake_tensor import FakeTensorMode

    import torch_point_ops_b200 as tpo

    with FakeTensorMode(allow_non_fake_inputs=True):
        x = torch.empty(5, 7, 32, device="cuda", dtype=torch.bfloat16)
        assert torch.ops.torch_point_ops_b200_norm.layer_norm(x, None, None, 1e-5).shape == (5, 7, 32)
        y, mean, rstd = torch.ops.torch_point_ops_b200_norm.layer_norm_forward(x, None, None, 1e-5)
        assert y.dtype == torch.bfloat16 and mean.shape == rstd.shape == (35,) and mean.dtype == torch.float32
        q, k = torch.empty(10, 4, 16, device="cuda"), torch.empty(12, 2, 16, device="cuda")
        off = torch.empty(3, device="cuda", dtype=torch.int64)
        o, lse = torch.ops.torch_point_ops_b200_attention.packed_attention_forward(q, k, k, off, off, True, 0.25)
        assert o.shape == q.shape and lse.shape == (4, 10)
        assert tpo.cached_attention(q, torch.empty(10, 20, 2, 16, device="cuda"), torch.empty(10, 20, 2, 16, device="cuda"),
                                    torch.empty(10, device="cuda", dtype=torch.int64)).shape == q.shape


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
def test_entry_points_without_the_binding(dtype):
    L, dev = lib(), "cuda"
    g = torch.Generator().manual_seed(0)
    q, go = (torch.randn(150, 4, 64, generator=g).to(dev, dtype) for _ in range(2))
    k, v = (torch.randn(150, 2, 64, generator=g).to(dev, dtype) for _ in range(2))
    off = torch.tensor([0, 100, 150], device=dev)
    prob = Packed(dtype=DT[dtype], causal=1, clouds=2, heads=4, kv_heads=2, width=64, tokens_q=150, tokens_k=150,
                  offsets_q=off.data_ptr(), offsets_k=off.data_ptr(), scale=0.125, q=q.data_ptr(), k=k.data_ptr(),
                  v=v.data_ptr(), q_token_stride=256, q_head_stride=64, k_token_stride=128, k_head_stride=64,
                  v_token_stride=128, v_head_stride=64)
    o, dq, dk, dv = (torch.full_like(t, float("nan")) for t in (q, q, k, v))
    lse = torch.full((4, 150), float("nan"), device=dev)
    assert L.tpo_packed_attention_fwd(ctypes.byref(prob), p(o), p(lse), stream()) == 0
    n = _size("tpo_packed_attention_bwd_workspace_size", I64(150), I64(4))
    ws = torch.full((n,), 255, dtype=torch.uint8, device=dev)  # its contents on entry do not matter
    assert L.tpo_packed_attention_bwd(ctypes.byref(prob), p(o), p(lse), p(go), I64(256), I64(64), p(dq), p(dk), p(dv),
                                      p(ws), ctypes.c_size_t(n), stream()) == 0
    ref = R.packed(q, k, v, [0, 100, 150], [0, 100, 150], True, 0.125, go)
    for name, t in (("o", o), ("dq", dq), ("dk", dk), ("dv", dv)):
        R.check(t, ref[name], name)
    scores = 0.125 * q[:100, 0].double() @ k[:100, 0].double().T
    want = scores.masked_fill(~torch.ones(100, 100, dtype=torch.bool, device=dev).tril(), -math.inf).logsumexp(1)
    # fp32 sums of 64 products and 100 exponentials
    assert (lse[0, :100].double() - want).abs().max() < 200 * 2.0 ** -24 * (1 + scores.abs().max())

    x, w, b = (torch.randn(s, generator=g).to(dev, dtype) for s in ((90, 72), (72,), (72,)))
    y, dx, dw, db = (torch.full_like(t, float("nan")) for t in (x, x, w, b))
    mean, rstd = (torch.empty(90, device=dev) for _ in range(2))
    assert L.tpo_layer_norm_fwd(DT[dtype], DT[dtype], p(x), I64(72), p(w), p(b), I64(90), I64(72), ctypes.c_double(1e-5),
                                p(y), p(mean), p(rstd), stream()) == 0
    dy = torch.randn(90, 72, generator=g).to(dev, dtype)
    n = _size("tpo_layer_norm_bwd_workspace_size", DT[dtype], I64(90), I64(72))
    ws = torch.full((n,), 255, dtype=torch.uint8, device=dev)
    assert L.tpo_layer_norm_bwd(DT[dtype], DT[dtype], p(x), I64(72), p(dy), I64(72), p(w), p(mean), p(rstd), I64(90),
                                I64(72), p(dx), p(dw), p(db), p(ws), ctypes.c_size_t(n), stream()) == 0
    ref = R.layer_norm(x, w, b, 1e-5, dy)
    for name, t in (("y", y), ("dx", dx), ("dw", dw), ("db", db)):
        R.check(t, ref[name], name)

    cache = torch.randn(2, 2, 5000, 2, 64, generator=g).to(dev, dtype)
    lengths = torch.tensor([5000, 77], device=dev)
    q2 = q[:2].contiguous()
    out = torch.full_like(q2, float("nan"))
    n = _size("tpo_cached_attention_workspace_size", I64(2), I64(4), I64(2), I64(5000), I64(64))
    ws = torch.full((max(n, 1),), 255, dtype=torch.uint8, device=dev)
    s3 = (I64 * 3)(5000 * 128, 128, 64)
    assert L.tpo_cached_attention(DT[dtype], p(q2), (I64 * 2)(256, 64), p(cache[0]), s3, p(cache[1]), s3, p(lengths),
                                  I64(2), I64(5000), I64(4), I64(2), I64(64), F(0.125), p(out), p(ws),
                                  ctypes.c_size_t(n), stream()) == 0
    R.check(out, R.cached(q2, cache[0], cache[1], [5000, 77], 0.125)["o"])
