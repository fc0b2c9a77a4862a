"""Norms before and after the blocks of a transformer, joined with the residual stream around them.

One launch forward (and two backward) for what the encoder layers with layer norms do between two blocks
(reference: models/indexed_latticeformer_encoder.py:848-877, ``torch.nn.LayerNorm`` and additions): the block's output is
normed itself if asked for, gated, scaled and added to the scaled residual stream, and the sum is normed for what follows.
Also reachable as ``cuda_funcs.residual_norm``.
"""
from __future__ import annotations

import ctypes
from typing import Optional

import torch
from torch.autograd.function import once_differentiable

from . import _lib

MAX_DIM = 16384


def _rows(t: torch.Tensor):
    """``t`` as rows of its last dimension and the distance between them in elements: in place if the rows lie evenly and
    their elements next to each other, else copied."""
    D = t.shape[-1]
    if t.is_contiguous():
        return t, D
    if t.dim() == 2 and t.stride(1) == 1 and t.stride(0) >= D:
        return t, t.stride(0)
    return t.contiguous(), D


def _gate_rows(gate: torch.Tensor, x: torch.Tensor) -> int:
    """How many rows the gate has: 1 (a scale per channel), one for as many rows of ``x`` after one another, or one for each."""
    D = x.shape[-1]
    if gate.dim() == 1 and gate.shape[0] == D:
        return 1
    if gate.dim() == x.dim() and gate.shape[-1] == D:
        lead = gate.shape[:-1]
        k = 0
        while k < len(lead) and lead[k] == x.shape[k]:
            k += 1
        if all(n == 1 for n in lead[k:]):
            rows = 1
            for n in lead[:k]:
                rows *= n
            return rows
    raise ValueError(f"gate of shape {tuple(gate.shape)} for x of shape {tuple(x.shape)}: its last dimension must be that of x, and "
                     "its leading dimensions none, or those of x up to some dimension and 1 from there on")


class ResidualNormHIP(torch.autograd.Function):
    """(h, y) or y or h; see ``residual_norm``.  ``spec``: (norm, eps, block_norm, block_eps, residual_scale, block_scale, keep)."""

    @staticmethod
    def forward(ctx, x, block, gate, weight, bias, block_weight, block_bias, spec):
        out, stats, h = _forward(x, block, gate, weight, bias, block_weight, block_bias, spec, True)
        # In float32 h is what the norm saw: where it is there anyway, and nothing else needs the block's output, it is kept
        # instead of x and block.  16 bits hold it rounded: the backward pass puts it together again.
        ctx.joined = h is not None and x.dtype == torch.float32 and gate is None and spec[2] is None
        ctx.has_block = block is not None
        ctx.spec, ctx.shape = spec, x.shape
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(h if ctx.joined else x, None if ctx.joined else block, gate, weight, bias, block_weight, block_bias, stats)
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, *grads):
        x, block, gate, weight, bias, block_weight, block_bias, stats = ctx.saved_tensors
        norm, _, block_norm, _, residual_scale, block_scale, keep = ctx.spec
        gh = grads[0] if keep else None
        gy = grads[-1] if norm is not None else None
        need = ctx.needs_input_grad
        if gh is None and gy is None:
            return (None,) * 8
        like = lambda t, yes: torch.empty(t.shape, dtype=t.dtype, device=t.device) if yes and t is not None else None  # noqa: E731
        args, held = _args(x, block, gate, weight, bias, block_weight, block_bias, ctx.spec)
        gh, gy = (None if g is None else g.contiguous() for g in (gh, gy))
        dgate, dw, db, dwf, dbf = (like(t, n) for t, n in zip((gate, weight, bias, block_weight, block_bias), need[2:]))
        if args.rows == 0:
            zero = lambda t: None if t is None else t.zero_()  # noqa: E731
            empty = torch.empty(ctx.shape, dtype=x.dtype, device=x.device)
            return (empty if need[0] else None, empty.clone() if need[1] else None, zero(dgate), zero(dw), zero(db), zero(dwf),
                    zero(dbf), None)
        dx = torch.empty(ctx.shape, dtype=x.dtype, device=x.device) if need[0] else None
        same = gate is None and block_norm is None and residual_scale == block_scale
        dblock = (dx if same and dx is not None else torch.empty(ctx.shape, dtype=x.dtype, device=x.device)) if need[1] else None
        if ctx.joined:
            args.joined = 1
        lib, dev = _lib.load(), x.device
        ref = ctypes.byref(args)
        # (scratch of its own for every call: two captured passes never share it)
        scratch = torch.empty(lib.cfh_residual_norm_backward_workspace_bytes(ref), dtype=torch.uint8, device=dev)
        address = lambda t: None if t is None else t.data_ptr()  # noqa: E731
        with torch.cuda.device(dev), _timed("residual_norm_backward", dev):
            rc = lib.cfh_residual_norm_backward(
                ref, stats.data_ptr(), address(gh), address(gy), address(dx), address(dblock), address(dgate), address(dw),
                address(db), address(dwf), address(dbf), scratch.data_ptr(), scratch.numel(), _lib.raw_stream(dev))
        _lib.check(rc, "cfh_residual_norm_backward")
        del held
        return dx, dblock, dgate, dw, db, dwf, dbf, None


def _timed(name, dev):
    from .cuda_funcs import _timed as timed
    return timed(name, dev)


def _args(x, block, gate, weight, bias, block_weight, block_bias, spec):
    """The library's argument structure and the tensors that it points to."""
    norm, eps, block_norm, block_eps, residual_scale, block_scale, _ = spec
    x, xs = _rows(x)
    D = x.shape[-1]
    a = _lib.CfhResidualNorm()
    a.struct_size = ctypes.sizeof(_lib.CfhResidualNorm)
    a.dtype = a.weight_dtype = _lib.ELEMENT_TYPES[x.dtype]
    a.norm, a.block_norm = _lib.NORM_KINDS[norm], _lib.NORM_KINDS[block_norm]
    a.eps, a.block_eps, a.residual_scale, a.block_scale = eps, block_eps, residual_scale, block_scale
    a.rows, a.dim, a.x_stride = x.numel() // D, D, xs
    held = [x]
    a.x = x.data_ptr()
    if block is not None:
        block, a.block_stride = _rows(block)
        a.block = block.data_ptr()
        held.append(block)
    if gate is not None:
        a.gate_rows = _gate_rows(gate, x)
        gate = gate.contiguous()
        a.gate = gate.data_ptr()
        held.append(gate)
    for name, t in (("weight", weight), ("bias", bias), ("block_weight", block_weight), ("block_bias", block_bias)):
        if t is not None:
            t = t.contiguous()
            a.weight_dtype = _lib.ELEMENT_TYPES[t.dtype]
            setattr(a, name, t.data_ptr())
            held.append(t)
    return a, held


def _forward(x, block, gate, weight, bias, block_weight, block_bias, spec, train):
    """(what the caller gets, the row statistics or None, h or None)."""
    norm, keep = spec[0], spec[6]
    args, held = _args(x, block, gate, weight, bias, block_weight, block_bias, spec)
    new = lambda: torch.empty(x.shape, dtype=x.dtype, device=x.device)  # noqa: E731
    h = new() if keep else None
    y = new() if norm is not None else None
    stats = torch.empty((args.rows, 4), dtype=torch.float32, device=x.device) if train else None
    lib, dev = _lib.load(), x.device
    with torch.cuda.device(dev), _timed("residual_norm_forward", dev):
        rc = lib.cfh_residual_norm_forward(ctypes.byref(args), None if h is None else h.data_ptr(), None if y is None else y.data_ptr(),
                                           None if stats is None else stats.data_ptr(), _lib.raw_stream(dev))
    _lib.check(rc, "cfh_residual_norm_forward")
    del held
    return ((h, y) if keep and y is not None else h if y is None else y), stats, h


def residual_norm(x: torch.Tensor, block: Optional[torch.Tensor] = None, weight: Optional[torch.Tensor] = None,
                  bias: Optional[torch.Tensor] = None, *, norm: Optional[str] = "layer", eps: float = 1e-5,
                  gate: Optional[torch.Tensor] = None, residual_scale: float = 1.0, block_scale: float = 1.0,
                  block_norm: Optional[str] = None, block_weight: Optional[torch.Tensor] = None,
                  block_bias: Optional[torch.Tensor] = None, block_eps: float = 1e-5, keep_residual: bool = True):
    """h = residual_scale x + block_scale gate N_b(block),  y = N(h): the residual stream after a block and its norm for the next.

    ``norm``, ``block_norm``: "layer" ((h - mean) / sqrt(var + eps) weight + bias), "rms" (h / sqrt(mean h^2 + eps) weight + bias)
    or None.  Weights and biases may be left out (1 and 0).  ``block`` may be left out (h = residual_scale x), and with it ``gate``
    and ``block_norm``.  ``gate``: a factor per channel (D), per element (the shape of x), or per leading index ((B, 1, D) for x of
    (B, T, D)).  Returns (h, y); y alone with ``keep_residual`` False; h alone with ``norm`` None.

    x, block and gate have one type, float32, bfloat16 or float16, which is that of the results; weights and biases have it too,
    or float32.  Everything between is in float32, and rounded once.  Up to 16384 channels.  All gradients are there (once: a
    gradient of a gradient raises), with sums over rows in a fixed order."""
    _lib.require_gpu(x, block, gate, weight, bias, block_weight, block_bias)
    if norm not in _lib.NORM_KINDS or block_norm not in _lib.NORM_KINDS:
        raise ValueError(f"norm {norm!r}, block_norm {block_norm!r}: \"layer\", \"rms\" or None")
    if x.dtype not in _lib.ELEMENT_TYPES:
        raise TypeError(f"x of {x.dtype}: float32, bfloat16 or float16")
    if x.dim() < 1 or not 1 <= x.shape[-1] <= MAX_DIM:
        raise ValueError(f"x of shape {tuple(x.shape)}: 1 to {MAX_DIM} channels")
    if eps < 0.0 or block_eps < 0.0:
        raise ValueError("eps and block_eps must not be negative")
    if norm is None and not keep_residual:
        raise ValueError("norm None with keep_residual False: nothing is left to return")
    if norm is None and (weight is not None or bias is not None):
        raise ValueError("weight and bias belong to a norm")
    if block_norm is None and (block_weight is not None or block_bias is not None):
        raise ValueError("block_weight and block_bias belong to a block_norm")
    if block is None and (gate is not None or block_norm is not None):
        raise ValueError("gate and block_norm belong to a block")
    for name, t in (("block", block), ("gate", gate)):
        if t is not None and t.dtype != x.dtype:
            raise TypeError(f"{name} of {t.dtype}, x of {x.dtype}: they must have one type")
    if block is not None and block.shape != x.shape:
        raise ValueError(f"block of shape {tuple(block.shape)}, x of shape {tuple(x.shape)}")
    D, kind = x.shape[-1], None
    for name, t in (("weight", weight), ("bias", bias), ("block_weight", block_weight), ("block_bias", block_bias)):
        if t is None:
            continue
        if t.shape != (D,):
            raise ValueError(f"{name} of shape {tuple(t.shape)} for {D} channels")
        if t.dtype not in (x.dtype, torch.float32) or (kind or t.dtype) != t.dtype:
            raise TypeError(f"{name} of {t.dtype}: weights and biases have one type, that of x or float32")
        kind = t.dtype
    tensors = (x, block, gate, weight, bias, block_weight, block_bias)
    if any(t is not None and t.device != x.device for t in tensors):
        raise RuntimeError("the tensors are on different devices")
    if gate is not None:
        _gate_rows(gate, x)
    spec = (norm, float(eps), block_norm, float(block_eps), float(residual_scale), float(block_scale), bool(keep_residual))
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors):
        return ResidualNormHIP.apply(*tensors, spec)
    return _forward(*tensors, spec, False)[0]
