"""Layer norm over the last dimension, forward and backward, in one kernel each
(plus the reduction of the parameter gradients)."""
import torch

from .. import _lib

_ops = _lib.norm_ops


def _stat_dtype(x):
    return torch.float64 if x.dtype == torch.float64 else torch.float32


def _rows(x):
    return x.numel() // x.shape[-1] if x.shape[-1] else 0


@torch.library.register_fake("torch_point_ops_b200_norm::layer_norm")
def _(x, weight, bias, eps):
    return x.new_empty(x.shape)


@torch.library.register_fake("torch_point_ops_b200_norm::layer_norm_forward")
def _(x, weight, bias, eps):
    stat = x.new_empty(_rows(x), dtype=_stat_dtype(x))
    return x.new_empty(x.shape), stat, torch.empty_like(stat)


@torch.library.register_fake("torch_point_ops_b200_norm::layer_norm_backward")
def _(grad, x, weight, bias, mean, rstd, need_x, need_weight, need_bias):
    width = x.shape[-1]
    return (x.new_empty(x.shape if need_x else 0),
            (x if weight is None else weight).new_empty(width if need_weight else 0),
            (x if bias is None else bias).new_empty(width if need_bias else 0))


def layer_norm(x: torch.Tensor, weight: torch.Tensor = None, bias: torch.Tensor = None,
               eps: float = 1e-5) -> torch.Tensor:
    """y = (x - mean) / sqrt(var + eps) * weight + bias over the last dimension.

    Args:
        x: (..., C) CUDA tensor; float32, float16, bfloat16 or float64
        weight, bias: (C,) or None; x's dtype, or float32 where x has 16 bits
        eps: added to the (biased) variance
    Returns:
        (..., C), x's dtype.  Moments and sums are held in float32 (float64 for
        float64); differentiable once in x, weight and bias (reverse mode), with
        the same bits in every run.
    """
    return _ops.layer_norm(x, weight, bias, eps)


from .norm import LayerNorm  # noqa: E402

__all__ = ["layer_norm", "LayerNorm"]
