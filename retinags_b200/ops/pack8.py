"""Feature rows in 8 bits: blocks of 32 channels that share a power of two.

``pack8(x)`` keeps a float tensor (..., C) as one signed byte per element and one exponent byte per 32 channels of a row
(the last block of a row may be shorter); ``Packed8.unpack`` gives the values back.  With e the smallest integer for
which ``127 * 2**e >= max|x|`` over a block (at least -126) an element becomes ``round(x / 2**e)``, halves to even: the
error is at most ``2**(e-1)``, between 1/254 and 1/127 of the block's largest magnitude, and because every step is exact
the codes are the same on every device (magnitudes above ``63 * 2**122`` count as that, so that values stay finite).  A block that holds an infinity or a NaN stands for NaN throughout.

Made for what waits between the passes of a training step (``layer_norm(keep="int8")`` keeps its input this way and
its backward pass reads the codes): 1.03 bytes an element in place of 4.
"""
from __future__ import annotations

from dataclasses import dataclass

import torch

from . import native

BLOCK = 32
DTYPES = {torch.float32: 0, torch.bfloat16: 1}


def dtype_code(t: torch.Tensor, what: str) -> int:
    code = DTYPES.get(t.dtype)
    if code is None:
        raise TypeError(f"{what}: float32 or bfloat16 expected, got {t.dtype}")
    check_device(t, what)
    return code


def check_device(t: torch.Tensor, what: str) -> None:
    if not (t.is_cuda or t.is_cpu):
        raise ValueError(f"{what}: a tensor on the CPU or a CUDA device expected, got {t.device}")


def as_rows(x: torch.Tensor, what: str, planes_ok: bool = True):
    """(tensor (N,C), leading stride, planes) of a tensor (..., C): rows with unit channel stride, or channel planes with unit row
    stride (``image.permute(1, 2, 0)`` of a (C,H,W) image), without a copy; any other layout is copied into rows."""
    if x.dim() < 1 or x.shape[-1] < 1:
        raise ValueError(f"{what}: shape (..., C) with at least one channel expected, got {tuple(x.shape)}")
    c = x.shape[-1]
    n = x.numel() // c
    if n > 2 ** 31 - 1:
        raise ValueError(f"{what}: at most 2^31 - 1 rows, got {n}")
    if n == 0:
        return x.reshape(0, c), c, 0
    if x.is_contiguous():
        return x if x.dim() == 2 else x.view(n, c), c, 0
    try:
        flat = x.view(n, c)
    except RuntimeError:
        return x.contiguous().view(n, c), c, 0
    s0, s1 = flat.stride()
    if (s1 == 1 or c == 1) and (n == 1 or s0 >= c):
        return flat, max(s0, c), 0
    if planes_ok and (s0 == 1 or n == 1) and s1 >= n:
        return flat, s1, 1
    return flat.contiguous(), c, 0


def restored(t, shape, dtype: torch.dtype, device: torch.device, what: str) -> torch.Tensor:
    """A saved tensor as autograd gives it back.  Saved-tensor hooks (offloading, compression) may restore it with other strides, so
    nothing about its layout is kept across the passes; another shape, type or device is refused."""
    if t is None or t.shape != shape or t.dtype is not dtype or t.device != device:
        got = "nothing" if t is None else f"{t.dtype} of shape {tuple(t.shape)} on {t.device}"
        raise RuntimeError(f"{what}: a saved tensor came back as {got}, {dtype} of shape {tuple(shape)} on {device} expected")
    return t


def empty_like_layout(shape, planes: int, dtype, device) -> torch.Tensor:
    """Tensor (..., C) stored as dense rows, or as dense channel planes."""
    if planes:
        return torch.empty((shape[-1], *shape[:-1]), dtype=dtype, device=device).movedim(0, -1)
    return torch.empty(tuple(shape), dtype=dtype, device=device)


def dense(t: torch.Tensor, planes: int) -> torch.Tensor:
    """``t`` in the order in which it is read: dense rows, or dense planes as (C, ...); a copy only if it is a slice or a view."""
    return (t.movedim(-1, 0) if planes else t).contiguous()


@dataclass
class Packed8:
    """Codes (..., C) int8 and exponent bytes (..., ceil(C/32)) uint8, both stored in the layout of the packed tensor."""

    codes: torch.Tensor
    exponents: torch.Tensor
    planes: int
    dtype: torch.dtype  # of the packed tensor

    @property
    def shape(self) -> torch.Size:
        return self.codes.shape

    @property
    def nbytes(self) -> int:
        return self.codes.numel() + self.exponents.numel()

    def unpack(self, dtype: torch.dtype | None = None) -> torch.Tensor:
        """The values that the codes stand for, as ``dtype`` (default: the type that was packed), in the same layout."""
        dtype = self.dtype if dtype is None else dtype
        if dtype not in DTYPES:
            raise TypeError(f"unpack: float32 or bfloat16 expected, got {dtype}")
        codes, exponents = self.codes, self.exponents
        check_device(codes, "unpack")
        if codes.dtype != torch.int8 or exponents.dtype != torch.uint8:
            raise TypeError(f"unpack: int8 codes and uint8 exponents expected, got {codes.dtype} and {exponents.dtype}")
        if codes.dim() < 1 or codes.shape[-1] < 1:
            raise ValueError(f"unpack: codes (..., C) with at least one channel expected, got {tuple(codes.shape)}")
        c = codes.shape[-1]
        if exponents.shape != (*codes.shape[:-1], (c + BLOCK - 1) // BLOCK):
            raise ValueError(f"unpack: one exponent to {BLOCK} channels expected, got {tuple(exponents.shape)} for {tuple(codes.shape)}")
        if exponents.device != codes.device:
            raise ValueError(f"unpack: exponents on {codes.device} expected, got {exponents.device}")
        n = codes.numel() // c
        if n > 2 ** 31 - 1:
            raise ValueError(f"unpack: at most 2^31 - 1 rows, got {n}")
        out = empty_like_layout(codes.shape, self.planes, dtype, codes.device)
        if n:
            native.call("unpack8", codes.device, dense(codes, self.planes), dense(exponents, self.planes), int(bool(self.planes)), n, c,
                        out, DTYPES[dtype])
        return out


def alloc_codes(shape, planes: int, device):
    """Uninitialised codes and exponents for a tensor (..., C)."""
    blocks = (shape[-1] + BLOCK - 1) // BLOCK
    return (empty_like_layout(shape, planes, torch.int8, device),
            empty_like_layout((*shape[:-1], blocks), planes, torch.uint8, device))


def pack8(x: torch.Tensor) -> Packed8:
    """Pack a float32 or bfloat16 tensor (..., C); rows or channel planes are read where they lie.

    A form to keep values in: no gradient passes through it (``pack8(x).unpack()`` is detached from ``x``)."""
    code = dtype_code(x, "pack8")
    flat, ld, planes = as_rows(x.detach(), "pack8")
    codes, exponents = alloc_codes(x.shape, planes, x.device)
    if flat.shape[0]:
        native.call("pack8", x.device, flat, code, ld, planes, flat.shape[0], flat.shape[1], codes, exponents)
    return Packed8(codes, exponents, planes, x.dtype)
