"""The token operators' C entry points: outputs at any address of their type."""
import ctypes

import pytest
import torch

import token_reference as R
from capi_util import I64, lib, p, stream
from test_token_capi import DT, F, Packed, _size

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _off(shape, dtype, by):
    """A tensor whose first element lies `by` elements behind a 16-byte boundary, and its guards."""
    n = 1
    for d in shape:
        n *= d
    buffer = torch.full((n + 16,), 7.0, dtype=dtype, device=DEV)
    return buffer[by:by + n].view(shape), (buffer[:by], buffer[by + n:])


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("which", ["o", "dq", "dk", "dv", "all"])
def test_attention_outputs_off_the_16_byte_grid(which, D, dtype):
    T, H, Hk, scale = 150, 4, 2, 0.125
    g = torch.Generator().manual_seed(D)
    q, go = (torch.randn(T, H, D, generator=g).to(DEV, dtype) for _ in range(2))
    k, v = (torch.randn(T, Hk, D, generator=g).to(DEV, dtype) for _ in range(2))
    off = torch.tensor([0, 100, T], device=DEV)
    prob = Packed(dtype=DT[dtype], causal=1, clouds=2, heads=H, kv_heads=Hk, width=D, tokens_q=T, tokens_k=T,
                  offsets_q=off.data_ptr(), offsets_k=off.data_ptr(), scale=scale, q=q.data_ptr(), k=k.data_ptr(),
                  v=v.data_ptr(), q_token_stride=H * D, q_head_stride=D, k_token_stride=Hk * D, k_head_stride=D,
                  v_token_stride=Hk * D, v_head_stride=D)
    lse = torch.empty(H, T, device=DEV)
    n = _size("tpo_packed_attention_bwd_workspace_size", I64(T), I64(H))
    ws = torch.empty(n, dtype=torch.uint8, device=DEV)
    ref = R.packed(q, k, v, [0, 100, T], [0, 100, T], True, scale, go)
    for by in (1, 3, 4):
        out = {name: _off(t.shape, dtype, by if which in (name, "all") else 0)
               for name, t in (("o", q), ("dq", q), ("dk", k), ("dv", k))}
        assert lib().tpo_packed_attention_fwd(ctypes.byref(prob), p(out["o"][0]), p(lse), stream()) == 0
        assert lib().tpo_packed_attention_bwd(ctypes.byref(prob), p(out["o"][0]), p(lse), p(go), I64(H * D), I64(D),
                                              p(out["dq"][0]), p(out["dk"][0]), p(out["dv"][0]), p(ws),
                                              ctypes.c_size_t(n), stream()) == 0
        for name, (t, guards) in out.items():
            R.check(t, ref[name], name)
            assert all((x == 7).all() for x in guards)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("P", [200, 5000])
def test_cached_output_off_the_16_byte_grid(P, dtype):
    g = torch.Generator().manual_seed(P)
    q = torch.randn(2, 4, 64, generator=g).to(DEV, dtype)
    k, v = (torch.randn(2, P, 2, 64, generator=g).to(DEV, dtype) for _ in range(2))
    lengths = torch.tensor([P, 77], device=DEV)
    n = _size("tpo_cached_attention_workspace_size", I64(2), I64(4), I64(2), I64(P), I64(64))
    ws = torch.empty(max(n, 1), dtype=torch.uint8, device=DEV)
    s3 = (I64 * 3)(P * 128, 128, 64)
    out, guards = _off(q.shape, dtype, 1)
    assert lib().tpo_cached_attention(DT[dtype], p(q), (I64 * 2)(256, 64), p(k), s3, p(v), s3, p(lengths), I64(2), I64(P),
                                      I64(4), I64(2), I64(64), F(0.125), p(out), p(ws), ctypes.c_size_t(n), stream()) == 0
    R.check(out, R.cached(q, k, v, [P, 77], 0.125)["o"])
    assert all((x == 7).all() for x in guards)


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
def test_layer_norm_outputs_off_the_16_byte_grid(dtype):
    rows, width = 40, 256
    g = torch.Generator().manual_seed(0)
    x, dy = (torch.randn(rows, width, generator=g).to(DEV, dtype) for _ in range(2))
    w, b = (torch.randn(width, generator=g).to(DEV, dtype) for _ in range(2))
    outs = [_off(s, dtype, 1) for s in ((rows, width), (rows, width), (width,), (width,))]
    (y, dx, dw, db), guards = [o[0] for o in outs], [x for o in outs for x in o[1]]
    mean, rstd = (torch.empty(rows, device=DEV) for _ in range(2))
    n = _size("tpo_layer_norm_bwd_workspace_size", DT[dtype], I64(rows), I64(width))
    ws = torch.empty(n, dtype=torch.uint8, device=DEV)
    assert lib().tpo_layer_norm_fwd(DT[dtype], DT[dtype], p(x), I64(width), p(w), p(b), I64(rows), I64(width),
                                    ctypes.c_double(1e-5), p(y), p(mean), p(rstd), stream()) == 0
    assert lib().tpo_layer_norm_bwd(DT[dtype], DT[dtype], p(x), I64(width), p(dy), I64(width), p(w), p(mean), p(rstd),
                                    I64(rows), I64(width), p(dx), p(dw), p(db), p(ws), ctypes.c_size_t(n), stream()) == 0
    ref = R.layer_norm(x, w, b, 1e-5, dy)
    for name, t in (("y", y), ("dx", dx), ("dw", dw), ("db", db)):
        R.check(t, ref[name], name)
    assert all((x == 7).all() for x in guards)
