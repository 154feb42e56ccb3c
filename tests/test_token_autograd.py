"""Forward-mode derivatives of the token operators: refused, never silently zero."""
import pytest
import torch
import torch.autograd.forward_ad as fw
from torch._subclasses.fake_tensor import FakeTensorMode

import torch_point_ops_b200 as tpo


def _calls(rand, ints):
    """(operator's call on its differentiable inputs, those inputs)."""
    q, kv, cache = rand(10, 4, 16), rand(10, 2, 16), rand(2, 5, 2, 16)
    off, lengths = ints(2), ints(2)
    return {
        "layer_norm": (lambda x, w, b: tpo.layer_norm(x, w, b), [rand(3, 8), rand(8), rand(8)]),
        "packed_attention": (lambda q, k, v: tpo.packed_attention(q, k, v, off), [q, kv, rand(10, 2, 16)]),
        "cached_attention": (lambda q, k, v: tpo.cached_attention(q, k, v, lengths), [rand(2, 4, 16), cache, rand(2, 5, 2, 16)]),
    }


@pytest.mark.parametrize("which", [0, 1, 2])
@pytest.mark.parametrize("name", ["layer_norm", "packed_attention", "cached_attention"])
def test_tangents_are_refused(name, which):
    with FakeTensorMode():
        call, args = _calls(lambda *s: torch.empty(s, device="cuda"), lambda n: torch.empty(n, device="cuda", dtype=torch.int64))[name]
        with fw.dual_level():
            args[which] = fw.make_dual(args[which], torch.empty_like(args[which]))
            with pytest.raises(RuntimeError, match="forward-mode"):
                call(*args)
            with torch.no_grad(), pytest.raises(RuntimeError, match="forward-mode"):
                call(*args)
        # and without a tangent as ever
        with fw.dual_level():
            assert call(*[fw.unpack_dual(t).primal for t in args]).shape == args[0].shape


@pytest.mark.gpu
@pytest.mark.parametrize("name", ["layer_norm", "packed_attention", "cached_attention"])
def test_jvp_and_jacfwd_are_refused(name):
    call, args = _calls(lambda *s: torch.randn(s, device="cuda"),
                        lambda n: torch.tensor([0, 10][:n] if name == "packed_attention" else [3, 5][:n], device="cuda"))[name]
    with pytest.raises(RuntimeError, match="forward-mode"):
        torch.func.jvp(lambda x: call(x, *args[1:]), (args[0],), (torch.ones_like(args[0]),))
    with pytest.raises(RuntimeError):
        torch.func.jacfwd(lambda x: call(x, *args[1:]))(args[0])
