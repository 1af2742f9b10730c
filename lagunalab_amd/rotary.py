"""Rotary embeddings as the paged cache's append takes them: frequencies on the device, the factor on rotated
dims, and which dims make a pair."""
from __future__ import annotations

import math

import torch

from .attention import rope_frequencies


class Rotary:
    """A rotary embedding of the first ``2 len(inv_freq)`` dims of a head: pair ``i`` turns by ``position *
    inv_freq[i]`` radians (fp32, on the device) and is scaled by ``mscale``. Pairs are dims ``i`` and ``i +
    len(inv_freq)``, or with ``interleaved`` dims ``2 i`` and ``2 i + 1``; the other dims stay."""

    __slots__ = ("inv_freq", "dims", "mscale", "interleaved")

    def __init__(self, inv_freq: torch.Tensor, mscale: float = 1.0, interleaved: bool = False):
        if inv_freq.dtype != torch.float32 or inv_freq.dim() != 1:
            raise ValueError(f"frequencies must be float32 [pairs], got {tuple(inv_freq.shape)} {inv_freq.dtype}")
        if not math.isfinite(mscale):
            raise ValueError(f"a factor of {mscale}")
        self.inv_freq, self.mscale, self.interleaved = inv_freq.contiguous(), float(mscale), bool(interleaved)
        self.dims = 2 * inv_freq.shape[0]  # rotated dims of a head

    @classmethod
    def of(cls, params: dict, device="cuda", interleaved: bool = False, head_dim: int = 128) -> "Rotary":
        """Of a rope config, as :func:`lagunalab_amd.attention.rope_frequencies` reads it."""
        inv_freq, dims, mscale = rope_frequencies(head_dim, params)
        if dims != 2 * len(inv_freq):
            raise ValueError(f"{dims} rotated dims are not pairs")
        return cls(inv_freq.to(device), mscale, interleaved)
