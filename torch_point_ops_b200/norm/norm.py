"""LayerNorm module."""
import torch

from . import layer_norm


class LayerNorm(torch.nn.Module):
    """Layer norm over the last dimension, with weight and bias unless affine=False."""

    def __init__(self, width, eps=1e-5, affine=True, device=None, dtype=None):
        super().__init__()
        if width < 1:
            raise ValueError(f"width must be >= 1, but got {width}")
        if eps < 0:
            raise ValueError(f"eps must not be negative, but got {eps}")
        self.width = width
        self.eps = eps
        if affine:
            self.weight = torch.nn.Parameter(torch.ones(width, device=device, dtype=dtype))
            self.bias = torch.nn.Parameter(torch.zeros(width, device=device, dtype=dtype))
        else:
            self.register_parameter("weight", None)
            self.register_parameter("bias", None)

    def forward(self, x):
        if x.shape[-1] != self.width:
            raise ValueError(f"expected a last dimension of {self.width}, but got {x.shape[-1]}")
        return layer_norm(x, self.weight, self.bias, self.eps)

    def extra_repr(self):
        return f"{self.width}, eps={self.eps}, affine={self.weight is not None}"
