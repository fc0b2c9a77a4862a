"""Norms before and after the blocks of a transformer, joined with the residual stream around them.

One launch forward and two backward (three where the column sums have a kernel of their own) for what the encoder layers with layer norms do between two blocks
(reference: models/indexed_latticeformer_encoder.py:848-877, ``torch.nn.LayerNorm`` and additions): the block's output is
normed itself if asked for, gated, scaled and added to the scaled residual stream, and the sum is normed for what follows.
Also reachable as ``cuda_funcs.residual_norm``.  The checks, the library's calls and the autograd function are native
(csrc/host_module.cpp).
"""
from __future__ import annotations

from typing import Optional

import torch

from . import _lib

MAX_DIM = 16384        # channels (the native checks hold the same number)
_native = None


def residual_norm(x: torch.Tensor, block: Optional[torch.Tensor] = None, weight: Optional[torch.Tensor] = None,
                  bias: Optional[torch.Tensor] = None, *, norm: Optional[str] = "layer", eps: float = 1e-5,
                  gate: Optional[torch.Tensor] = None, residual_scale: float = 1.0, block_scale: float = 1.0,
                  block_norm: Optional[str] = None, block_weight: Optional[torch.Tensor] = None,
                  block_bias: Optional[torch.Tensor] = None, block_eps: float = 1e-5, keep_residual: bool = True,
                  twice_differentiable: bool = False):
    """h = residual_scale x + block_scale gate N_b(block),  y = N(h): the residual stream after a block and its norm for the next.

    ``norm``, ``block_norm``: "layer" ((h - mean) / sqrt(var + eps) weight + bias), "rms" (h / sqrt(mean h^2 + eps) weight + bias)
    or None.  Weights and biases may be left out (1 and 0).  ``block`` may be left out (h = residual_scale x), and with it ``gate``
    and ``block_norm``.  ``gate``: a factor per channel (D), per element (the shape of x), or per leading index ((B, 1, D) for x of
    (B, T, D)).  Returns (h, y); y alone with ``keep_residual`` False; h alone with ``norm`` None.

    x, block and gate have one type, float32, bfloat16 or float16, which is that of the results; weights and biases have it too,
    or float32.  Everything between is in float32, and rounded once.  Up to 16384 channels.  All gradients are there, with
    sums over rows in a fixed order; a gradient of a gradient raises, but with ``twice_differentiable`` (a layer norm of x or of x + block):
    a backward pass that is itself recorded then goes through the framework's operations."""
    global _native
    if _native is None:
        _native = _lib.load_host().residual_norm
    if torch.autograd.forward_ad._current_level >= 0:
        raise RuntimeError("a residual norm has no forward-mode derivative")
    kinds = _lib.NORM_KINDS
    if norm not in kinds or block_norm not in kinds:
        raise ValueError(f"norm {norm!r}, block_norm {block_norm!r}: \"layer\", \"rms\" or None")
    return _native(x, block, gate, weight, bias, block_weight, block_bias, kinds[norm], eps, kinds[block_norm], block_eps, residual_scale,
                   block_scale, keep_residual, twice_differentiable)
