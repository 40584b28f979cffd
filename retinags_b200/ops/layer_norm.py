"""Layer norm over the channels of rendered features, with its backward pass.

Blended features are weighted sums over the splats of a pixel, so their size follows the pixel's coverage; the norm
takes that out ahead of a classifier (``ops.label_loss``).  The input may be rows (..., C) or, as the renderer writes an
image, channel planes (``image.permute(1, 2, 0)`` of a (C,H,W) image), both read where they lie (planes of more than 512
channels, and any other layout, are copied into rows); the output is dense rows in ``out_dtype``.  Sums are held in 32 bits
whatever the types.
"""
from __future__ import annotations

import torch

from . import native
from .pack8 import BLOCK, DTYPES, alloc_codes, as_rows, dense, dtype_code, empty_like_layout, restored

MAX_PLANES = 512  # channels up to which planes are read and written where they lie; more are copied into rows and back


def _scratch(device: torch.device, n: int, c: int) -> torch.Tensor:
    return torch.empty(native.size_of("norm_scratch_bytes", device, n, c), dtype=torch.uint8, device=device)


class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps, out_dtype, keep):
        flat, ld, planes = as_rows(x, "layer_norm")
        n, c = flat.shape
        out_planes = planes
        if planes and c > MAX_PLANES:
            flat, ld, planes = flat.contiguous(), c, 0
        dev = x.device
        y = torch.empty(x.shape, dtype=out_dtype, device=dev)
        p_code = DTYPES[weight.dtype if weight is not None else bias.dtype if bias is not None else torch.float32]
        codes = exponents = None
        # bias alone needs no input in the backward pass
        if keep == "int8" and (ctx.needs_input_grad[0] or ctx.needs_input_grad[1]):
            codes, exponents = alloc_codes(x.shape, planes, dev)
        if n:
            native.call("norm_fwd", dev, flat, DTYPES[x.dtype], ld, planes, weight, bias, p_code, n, c, eps, y, DTYPES[out_dtype],
                        codes, exponents)
        ctx.save_for_backward(flat if codes is None else None, codes, exponents, weight)
        ctx.layout = (codes is not None, x.shape, x.dtype, planes, out_planes, n, c, p_code, eps, weight.dtype if weight is not None else None,
                      bias.dtype if bias is not None else None)
        return y

    @staticmethod
    def backward(ctx, dy):
        # (the wrapper that refuses a second derivative costs as much as a launch: only where one is being recorded)
        return _norm_backward_once(ctx, dy) if torch.is_grad_enabled() else _norm_backward(ctx, dy)


def _norm_backward(ctx, dy):
    coded, shape, x_dtype, planes, out_planes, n, c, p_code, eps, w_dtype, b_dtype = ctx.layout
    flat, codes, exponents, weight = ctx.saved_tensors
    dev, ld = dy.device, c
    if coded:
        codes = dense(restored(codes, shape, torch.int8, dev, "layer_norm"), planes)
        exponents = dense(restored(exponents, (*shape[:-1], (c + BLOCK - 1) // BLOCK), torch.uint8, dev, "layer_norm"), planes)
    elif restored(flat, (n, c), x_dtype, dev, "layer_norm").is_contiguous():
        planes = 0
    else:
        flat, ld, planes = as_rows(flat, "layer_norm")
        if planes and c > MAX_PLANES:
            flat, ld, planes = flat.contiguous(), c, 0
    if w_dtype is not None:
        weight = restored(weight, (c,), w_dtype, dev, "layer_norm").contiguous()
    need_x, need_w, need_b = ctx.needs_input_grad[:3]
    dyf, ldy, _ = as_rows(dy, "layer_norm", planes_ok=False)
    dx = empty_like_layout(shape, planes, x_dtype, dev) if need_x else None
    new = torch.empty if n else torch.zeros
    dw = new(c, dtype=w_dtype, device=dev) if need_w else None
    db = new(c, dtype=b_dtype, device=dev) if need_b else None
    if n:
        native.call("norm_bwd", dev, flat, DTYPES[x_dtype], ld, planes, codes, exponents, dyf, DTYPES[dyf.dtype], ldy, weight, p_code,
                    n, c, eps, _scratch(dev, n, c), dx, dw, db)
    if dx is not None and out_planes != planes:
        dx = empty_like_layout(shape, out_planes, x_dtype, dev).copy_(dx)
    return dx, dw, db, None, None, None


_norm_backward_once = torch.autograd.function.once_differentiable(_norm_backward)


def layer_norm(x: torch.Tensor, weight: torch.Tensor | None = None, bias: torch.Tensor | None = None, eps: float = 1e-5,
               out_dtype: torch.dtype | None = None, keep: str = "input") -> torch.Tensor:
    """``(x - mean) / sqrt(var + eps) * weight + bias`` over the last dimension of ``x`` (..., C), as dense rows.

    ``x`` and ``out_dtype`` (default: that of ``x``) are float32 or bfloat16; ``weight`` and ``bias`` (C) are of one of
    these types, both of the same.  ``keep`` says what waits for the backward pass: ``"input"`` the tensor itself,
    ``"int8"`` its 8-bit form (``ops.pack8``); the gradients are then those of the norm at the restored values, and the
    input's memory is free as soon as nothing else holds it.  A step of the codes is 1/254 to 1/127 of the largest magnitude
    among 32 channels, so the gradients suffer where channels differ little beside their size: with 64 channels of spread 0.1
    the gradient of ``x`` is off by 0.2 % (in norm) around 0, by 1 % around 1, 4 % around 5 and 18 % around 20, that of
    ``weight`` by about four times as much.
    """
    dtype_code(x, "layer_norm")
    out_dtype = x.dtype if out_dtype is None else out_dtype
    if out_dtype not in DTYPES:
        raise TypeError(f"layer_norm: out_dtype float32 or bfloat16 expected, got {out_dtype}")
    if keep != "input" and keep != "int8":
        raise ValueError(f"layer_norm: keep is 'input' or 'int8', got {keep!r}")
    if not eps >= 0.0:
        raise ValueError(f"layer_norm: eps >= 0 expected, got {eps}")
    shape = x.shape
    if len(shape) < 1 or shape[-1] < 1:
        raise ValueError(f"layer_norm: shape (..., C) with at least one channel expected, got {tuple(shape)}")
    if weight is not None:
        weight = _param(x, weight, shape[-1], "weight")
    if bias is not None:
        bias = _param(x, bias, shape[-1], "bias")
        if weight is not None and weight.dtype != bias.dtype:
            raise TypeError(f"layer_norm: weight and bias of one type expected, got {weight.dtype} and {bias.dtype}")
    if not torch.is_grad_enabled():
        keep = "input"  # no backward pass will read codes
    return _LayerNorm.apply(x, weight, bias, float(eps), out_dtype, keep)


def _param(x: torch.Tensor, p: torch.Tensor, c: int, name: str) -> torch.Tensor:
    if p.dtype not in DTYPES:
        raise TypeError(f"layer_norm {name}: float32 or bfloat16 expected, got {p.dtype}")
    if p.dim() != 1 or p.shape[0] != c:
        raise ValueError(f"layer_norm: {name} of shape ({c},) expected, got {tuple(p.shape)}")
    if p.device != x.device:
        raise ValueError(f"layer_norm: {name} on {x.device} expected, got {p.device}")
    return p if p.is_contiguous() else p.contiguous()
