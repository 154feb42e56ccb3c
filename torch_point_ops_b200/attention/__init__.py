"""Attention over the tokens of point clouds: packed clouds of different sizes
(training, whole prompts) and one token per cloud over a cache (generation)."""
import math

import torch

from .. import _lib

_ops = _lib.attention_ops


@torch.library.register_fake("torch_point_ops_b200_attention::packed_attention")
def _(q, k, v, offsets, offsets_k, causal, scale):
    return q.new_empty(q.shape)


@torch.library.register_fake("torch_point_ops_b200_attention::packed_attention_forward")
def _(q, k, v, offsets, offsets_k, causal, scale):
    return q.new_empty(q.shape), q.new_empty((q.shape[1], q.shape[0]), dtype=torch.float32)


@torch.library.register_fake("torch_point_ops_b200_attention::packed_attention_backward")
def _(grad, q, k, v, o, lse, offsets, offsets_k, causal, scale, need_q, need_kv):
    return (q.new_empty(q.shape if need_q else 0), k.new_empty(k.shape if need_kv else 0),
            v.new_empty(v.shape if need_kv else 0))


@torch.library.register_fake("torch_point_ops_b200_attention::cached_attention")
def _(q, k, v, lengths, scale):
    return q.new_empty(q.shape)


def packed_offsets(lengths: torch.Tensor) -> torch.Tensor:
    """Offsets (N + 1,) int64 of clouds with `lengths` (N,) packed one after another."""
    return torch.nn.functional.pad(lengths.to(torch.int64).cumsum(0), (1, 0))


def _scale(scale, width):
    if scale is None:
        return 1.0 / math.sqrt(width) if width else 1.0
    if not 0 < scale < math.inf:
        raise ValueError(f"scale must be positive and finite, but got {scale}")
    return float(scale)


def packed_attention(
    q: torch.Tensor,
    k: torch.Tensor,
    v: torch.Tensor,
    offsets: torch.Tensor,
    offsets_k: torch.Tensor = None,
    causal: bool = False,
    scale: float = None,
) -> torch.Tensor:
    """softmax(scale * q k^T) v within each cloud of a packed batch.

    Args:
        q: (T, H, D) queries of all clouds one after another (CUDA; float32,
            float16 or bfloat16; D <= 256); any strides, copied only where the
            last dimension is not contiguous
        k, v: (Tk, Hk, D), H a multiple of Hk: query head h reads h // (H // Hk)
        offsets: (N + 1,) int64 (int32 is converted): cloud i has the queries
            [offsets[i], offsets[i + 1])
        offsets_k: the same for the keys; None: the same tokens as the queries
        causal: query i of a cloud with nq queries and nk keys sees the keys
            j <= i + nk - nq, so the last query sees all of them
        scale: positive; None: 1 / sqrt(D)
    Returns:
        (T, H, D).  A query that sees no key, and a token outside of every
        cloud, gives zeros and has zero gradients.  Differentiable once in q, k,
        v (reverse mode), with the same bits in every run.  Nothing from another cloud enters a
        result; within a causal cloud a value that is not finite may
        reach earlier queries of its own tile of 128 keys.
    """
    return _ops.packed_attention(q, k, v, offsets, offsets_k, causal, _scale(scale, q.shape[-1]))


def cached_attention(
    q: torch.Tensor,
    k_cache: torch.Tensor,
    v_cache: torch.Tensor,
    lengths: torch.Tensor,
    scale: float = None,
) -> torch.Tensor:
    """One query token per cloud against the first lengths[n] tokens of its cache.

    Args:
        q: (N, H, D) (CUDA; float32, float16 or bfloat16; D <= 256)
        k_cache, v_cache: (N, P, Hk, D), H a multiple of Hk; any strides with a
            contiguous last dimension
        lengths: (N,) int64 (int32 is converted), clamped to [0, P]
        scale: positive; None: 1 / sqrt(D)
    Returns:
        (N, H, D); zeros where lengths[n] is 0.  Slots at or beyond lengths[n]
        are not read.  No backward pass.
    """
    return _ops.cached_attention(q, k_cache, v_cache, lengths, _scale(scale, q.shape[-1]))


from .attention import PackedAttention  # noqa: E402

__all__ = ["packed_attention", "cached_attention", "packed_offsets", "PackedAttention"]
