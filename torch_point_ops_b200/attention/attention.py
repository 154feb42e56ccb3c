"""PackedAttention module."""
import torch

from . import packed_attention


class PackedAttention(torch.nn.Module):
    """packed_attention with its options held by a module."""

    def __init__(self, causal=False, scale=None):
        super().__init__()
        if scale is not None and not scale > 0:
            raise ValueError(f"scale must be positive, but got {scale}")
        self.causal = causal
        self.scale = scale

    def forward(self, q, k, v, offsets, offsets_k=None):
        return packed_attention(q, k, v, offsets, offsets_k, causal=self.causal, scale=self.scale)

    def extra_repr(self):
        return f"causal={self.causal}, scale={self.scale}"
