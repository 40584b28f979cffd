"""Softmax cross entropy of linear scores against a vocabulary of labels, without the scores in memory.

The loss of a label field: rendered features (..., C) are scored against V labels (classes, instances, entries of a
codebook) by ``features @ weight.T + bias``.  At 1600 x 1036 pixels the scores of 1024 labels are 6.8 GB in 32 bits;
the kernels (``csrc/rgs_label.cu``) walk the vocabulary in pieces, keep two numbers per pixel for the backward pass
(the largest score and the logarithm of the sum of exponentials below it) and compute the scores anew there.  Stands beside the photometric loss of
``ops.loss``; the readable definition is ``utils.loss.label_loss``.
"""
from __future__ import annotations

import torch

from . import native
from .pack8 import DTYPES, as_rows, dtype_code, restored

MAX_CHANNELS = 1024
_REDUCTIONS = ("mean", "sum", "none")
_LIMIT = 2 ** 31 - 1


def _scratch(x: torch.Tensor, ldx: int, w: torch.Tensor, ldw: int, backward: int) -> torch.Tensor:
    """Workspace of one pass; it depends on whether the kernels can read the rows as they lie (16-byte boundaries) and on the
    gradients that a backward pass is to give (1, and 2 for features, 4 for weight, 8 for bias)."""
    device = x.device
    direct = (ldx % 8 == 0 and x.data_ptr() % 16 == 0) + 2 * (ldw % 8 == 0 and w.data_ptr() % 16 == 0)
    size = native.size_of("label_scratch_bytes", device, x.shape[0], x.shape[1], w.shape[0], DTYPES[x.dtype], direct, backward)
    return torch.empty(size, dtype=torch.uint8, device=device)


class _LabelLoss(torch.autograd.Function):
    @staticmethod
    def forward(ctx, features, weight, bias, labels, reduction):
        dev = features.device
        x, ldx, _ = as_rows(features, "label_loss", planes_ok=False)
        w, ldw, _ = as_rows(weight, "label_loss", planes_ok=False)
        y = labels if labels.dim() == 1 and labels.is_contiguous() else labels.reshape(-1).contiguous()
        n, c = x.shape
        v = w.shape[0]
        per_row = reduction == "none"
        new = torch.empty if n else torch.zeros
        # kept for the backward pass: m and log z of every pixel, number of pixels that count, flags
        state = torch.empty(2 * n + 2, dtype=torch.float32, device=dev)
        lse = state.data_ptr()
        losses = torch.empty(n, dtype=torch.float32, device=dev) if per_row else None
        result = None if per_row else new((), dtype=torch.float32, device=dev)
        b_code = DTYPES[bias.dtype] if bias is not None else 0
        if n:
            scratch = _scratch(x, ldx, w, ldw, 0)
            native.call("label_fwd", dev, x, ldx, w, ldw, bias, y, y.element_size(), n, c, v, DTYPES[x.dtype], b_code,
                        int(reduction == "mean"), scratch, scratch.numel(), lse, losses, result, lse + 8 * n)
        ctx.save_for_backward(x, w, bias, y, state)
        ctx.args = (features.shape, n, c, v, features.dtype, bias.dtype if bias is not None else None, y.dtype, dev, b_code, reduction)
        return losses.view(features.shape[:-1]) if per_row else result

    @staticmethod
    def backward(ctx, gout):
        # (the wrapper that refuses a second derivative costs as much as a launch: only where one is being recorded)
        return _label_backward_once(ctx, gout) if torch.is_grad_enabled() else _label_backward(ctx, gout)


def _saved_rows(t: torch.Tensor, shape, dtype: torch.dtype, device: torch.device):
    restored(t, shape, dtype, device, "label_loss")
    return (t, shape[1]) if t.is_contiguous() else as_rows(t, "label_loss", planes_ok=False)[:2]


def _label_backward(ctx, gout):
    x_shape, n, c, v, dtype, b_dtype, y_dtype, dev, b_code, reduction = ctx.args
    x, w, bias, y, state = ctx.saved_tensors
    x, ldx = _saved_rows(x, (n, c), dtype, dev)
    w, ldw = _saved_rows(w, (v, c), dtype, dev)
    y = restored(y, (n,), y_dtype, dev, "label_loss").contiguous()
    state = restored(state, (2 * n + 2,), torch.float32, dev, "label_loss").contiguous()
    if b_dtype is not None:
        bias = restored(bias, (v,), b_dtype, dev, "label_loss").contiguous()
    g = gout if gout.dim() < 2 and gout.is_contiguous() else gout.reshape(-1).contiguous()
    new = torch.empty if n else torch.zeros
    dx = torch.empty(x_shape, dtype=x.dtype, device=dev) if ctx.needs_input_grad[0] else None
    dw = new((v, c), dtype=w.dtype, device=dev) if ctx.needs_input_grad[1] else None
    db = new(v, dtype=bias.dtype, device=dev) if ctx.needs_input_grad[2] else None
    if n and (dx is not None or dw is not None or db is not None):
        scratch = _scratch(x, ldx, w, ldw, 1 + 2 * (dx is not None) + 4 * (dw is not None) + 8 * (db is not None))
        native.call("label_bwd", dev, x, ldx, w, ldw, bias, y, y.element_size(), n, c, v, DTYPES[x.dtype], b_code, state, g,
                    int(reduction == "none"), int(reduction == "mean"), state.data_ptr() + 8 * n,
                    scratch, scratch.numel(), dx, dw, db)
    return dx, dw, db, None, None


_label_backward_once = torch.autograd.function.once_differentiable(_label_backward)


def label_loss(features: torch.Tensor, weight: torch.Tensor, labels: torch.Tensor, bias: torch.Tensor | None = None,
               reduction: str = "mean") -> torch.Tensor:
    """Cross entropy (float32) of ``features @ weight.T + bias`` against ``labels``.

    ``features`` (..., C) and ``weight`` (V, C) are float32 or bfloat16, both of one type, with C up to 1024;
    ``labels`` (...) int64 or int32; ``bias`` (V) of the features' type or float32 (``-inf`` takes a label out).  A label
    outside [0, V) marks a pixel without one: its loss and gradient are zero, whatever its features hold, and it does not
    count in the mean.  ``reduction``: ``"mean"`` over the pixels that count (0 if none does), ``"sum"``, ``"none"``
    (one loss per pixel).  Differentiable (once) in features, weight and bias.

    Products of bfloat16 inputs are exact and summed in 32 bits; ``exp(score - lse) - [label]`` is rounded to bfloat16
    for the products with features and weight.  float32 inputs go through the same tensor-core products in three
    bfloat16 pieces each; their gradients are off by 1 to 3 millionths of their size (elementary 32-bit operations: half to
    one and a half).  Where a wait inside the kernels runs out the numbers that hang on it are NaN.

    Features are read as rows; planes (``image.permute(1, 2, 0)``) are copied into rows first.  Gradients form the scores anew
    for every 256 channels in bfloat16 and every 64 in float32, so wide features cost more than their width: 66560 pixels x
    4096 labels take 0.38, 0.69, 2.1 and 9.3 ms a step at 64, 256, 512 and 1024 bfloat16 channels, and 0.9, 7.4, 26 and 108 ms in
    float32 (where the scores fit, two products with them in memory are faster above 256 channels: 18 and 31 ms).
    Workspace beside the results: a copy of features or weight that do not start on 16 bytes (float32: 6 bytes a channel of
    each), some 50 bytes a pixel and a label, and for gradients partial sums in 32 bits, up to 2 GiB and one result each for features
    and weight.
    """
    code = dtype_code(features, "label_loss features")
    if weight.dtype != features.dtype:
        raise TypeError(f"label_loss: weight of type {features.dtype} expected, got {weight.dtype}")
    if reduction not in _REDUCTIONS:
        raise ValueError(f"label_loss: reduction is one of {_REDUCTIONS}, got {reduction!r}")
    if features.dim() < 1 or weight.dim() != 2 or features.shape[-1] != weight.shape[1]:
        raise ValueError(f"label_loss: features (..., C) and weight (V, C) expected, got {tuple(features.shape)} and {tuple(weight.shape)}")
    c, v = features.shape[-1], weight.shape[0]
    if not 1 <= c <= MAX_CHANNELS:
        raise ValueError(f"label_loss: 1 to {MAX_CHANNELS} channels expected, got {c}")
    if v < 1:
        raise ValueError("label_loss: the vocabulary is empty")
    if labels.dtype not in (torch.int64, torch.int32):
        raise TypeError(f"label_loss: int64 or int32 labels expected, got {labels.dtype}")
    if labels.shape != features.shape[:-1]:
        raise ValueError(f"label_loss: labels of shape {tuple(features.shape[:-1])} expected, got {tuple(labels.shape)}")
    if labels.numel() > _LIMIT or v > _LIMIT:
        raise ValueError("label_loss: at most 2^31 - 1 pixels and labels")
    if bias is not None:
        if bias.shape != (v,):
            raise ValueError(f"label_loss: bias of shape ({v},) expected, got {tuple(bias.shape)}")
        if DTYPES.get(bias.dtype, -1) not in (0, code):
            raise TypeError(f"label_loss: bias of type {features.dtype} or float32 expected, got {bias.dtype}")
    device = features.device
    for name, t in (("weight", weight), ("labels", labels), ("bias", bias)):
        if t is not None and t.device != device:
            raise ValueError(f"label_loss: {name} on {features.device} expected, got {t.device}")
    return _LabelLoss.apply(features, weight, bias.contiguous() if bias is not None else None, labels, reduction)
