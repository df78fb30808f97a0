"""Root-mean-square norm of rows with the residual's addition, an output in 8 bits and the gradient, on the
HIP kernels of csrc/spr_rms_norm.hip.

    s = x + residual (rounded once, to the residual's type);  y = s / sqrt(mean(s^2) + epsilon) * weight

over the last dim of x [..., C], C up to 16384, sums in fp32: a row whose sum of squares leaves its range gives
what fp32 gives (zeros above 1.8e19, and with epsilon 0 infinities below 1e-23).  The norm reads s as it is stored.  x and the
residual are bf16, fp16 or fp32, the residual of x's type or fp32; the weight is [C] of x's type or fp32,
or None.  Rows may have any strides as long as they are packed and their dims merge into two (a Q or K
slice of a projection, seen by heads); others are copied.  None of the functions is recorded by autograd:
inputs that require a gradient are refused while it records, and those with a tangent; `rms_norm_backward` is the
gradient."""

from __future__ import annotations

import torch

from .. import _lib
from .fp8 import BLOCK, CODES, no_gradient

MAX_WIDTH = 16384


def _by_rows(x: torch.Tensor) -> tuple[torch.Tensor, int, int, int, int]:
    """x [..., C] as [n0, n1, C]: (x or a copy, n0, n1, stride of n0, stride of n1)."""
    rows = x.numel() // x.shape[-1]
    if x.is_contiguous():
        return x, rows, 1, x.shape[-1], 0
    dims = []  # the leading dims, merged where the outer one continues the inner one
    for n, s in zip(x.shape[:-1], x.stride()[:-1]):
        if n == 1:
            continue
        if dims and dims[-1][1] == n * s:
            dims[-1] = (dims[-1][0] * n, s)
        else:
            dims.append((n, s))
    if len(dims) > 2 or (x.shape[-1] > 1 and x.stride(-1) != 1):
        return x.contiguous(), rows, 1, x.shape[-1], 0
    dims = [(1, 0)] * (2 - len(dims)) + dims
    (n0, s0), (n1, s1) = dims
    return x, n0, n1, s0, s1


def _split(x: torch.Tensor, n0: int, n1: int) -> tuple[torch.Tensor, int, int]:
    """x's strides over rows counted as n0 x n1 (a copy where they are not that regular)."""
    x, m0, m1, s0, s1 = _by_rows(x)
    if (m0, m1) == (n0, n1):
        return x, s0, s1
    if m1 == 1 or m0 == 1:  # one stride for all rows
        step = s0 if m1 == 1 else s1
        return x, step * n1, step
    x = x.contiguous()
    return x, x.shape[-1] * n1, x.shape[-1]


def _check(x: torch.Tensor, weight: torch.Tensor | None, epsilon: float, what: str) -> tuple[torch.Size, int, int, int]:
    """(x's shape, its last dim, codes of x's and of the weight's type)."""
    shape, code = x.shape, _lib.DTYPE_CODE.get(x.dtype)
    if len(shape) < 1 or code is None:
        raise RuntimeError(f"{what}: x must be [..., C] in bfloat16, float16 or float32, got {x.dtype} {tuple(x.shape)}")
    width, weight_code = shape[-1], 0
    if not 1 <= width <= MAX_WIDTH:
        raise RuntimeError(f"{what}: width {width} not in 1 .. {MAX_WIDTH}")
    if x.numel() // width >= 1 << 31:  # the entry points count rows in 32 bits
        raise RuntimeError(f"{what}: too many rows in {tuple(x.shape)}")
    if weight is not None:
        weight_code = _lib.DTYPE_CODE.get(weight.dtype)
        if weight.shape != (width,) or weight_code not in (code, 2):
            raise RuntimeError(f"{what}: weight must be [{width}] in {x.dtype} or float32, got {weight.dtype} "
                               f"{tuple(weight.shape)}")
    if not 0.0 <= epsilon < float("inf"):
        raise RuntimeError(f"{what}: epsilon must be finite and not negative, got {epsilon}")
    return shape, width, code, weight_code


def _norm(x, weight, residual, epsilon, fp8: bool, what: str):
    dev = _lib.require_gpu(x, weight, residual, what=what)
    no_gradient(what, x, weight, residual)
    shape, width, code, weight_code = _check(x, weight, epsilon, what)
    total, r_code = None, 0
    if residual is not None:
        r_code = _lib.DTYPE_CODE.get(residual.dtype)
        if residual.shape != shape or r_code not in (code, 2):
            raise RuntimeError(f"{what}: residual must be {tuple(x.shape)} in {x.dtype} or float32, got {residual.dtype} "
                               f"{tuple(residual.shape)}")
        total = residual.new_empty(shape)
    scales = None
    if fp8:
        rows = shape[:-1]
        out = x.new_empty((*rows, -(-width // 16) * 16), dtype=CODES)
        scales = x.new_empty((*rows, -(-width // BLOCK)), dtype=torch.uint8)
    else:
        out = x.new_empty(shape)
    if x.numel() > 0:
        x, n0, n1, s0, s1 = _by_rows(x)
        r_at = r0 = r1 = 0
        if residual is not None:
            residual, r0, r1 = _split(residual, n0, n1)
            r_at = residual.data_ptr()
        weight = None if weight is None else weight.contiguous()
        _lib.launch("spr_rms_norm", dev, x.data_ptr(), s0, s1, r_at, r0, r1, n0, n1, width, code, r_code,
                    _lib.ptr(weight), weight_code, float(epsilon), out.data_ptr(), _lib.ptr(scales), _lib.ptr(total))
    return out, scales, total


def rms_norm(x: torch.Tensor, weight: torch.Tensor | None = None, *, residual: torch.Tensor | None = None,
             epsilon: float = 1e-6):
    """y in x's type; with a residual (y, s)."""
    out, _, total = _norm(x, weight, residual, epsilon, False, "RMS norm")
    return out if residual is None else (out, total)


def rms_norm_fp8(x: torch.Tensor, weight: torch.Tensor | None = None, *, residual: torch.Tensor | None = None,
                 epsilon: float = 1e-6):
    """y in 8 bits, as fp8_quantize(y) of an unrounded y gives it: codes [..., C rounded up to 16] and scales
    [..., C / 128 rounded up], what fp8_matmul takes (as [rows, width]); with a residual (codes, scales, s)."""
    codes, scales, total = _norm(x, weight, residual, epsilon, True, "RMS norm to 8 bits")
    return (codes, scales) if residual is None else (codes, scales, total)


def rms_norm_backward(dy: torch.Tensor, s: torch.Tensor, weight: torch.Tensor | None = None, *,
                      dsum: torch.Tensor | None = None, epsilon: float = 1e-6):
    """The gradient of rms_norm: (dx, dweight) from dy, the s that the norm read (x without a residual) and
    `dsum`, the gradient that reaches s on its other way (the residual's).  dx, in s's type, is the gradient of
    x and of the residual; dweight is fp32 [C], None without a weight.  dy is of x's type, s and dsum of that
    or fp32.  The weight's gradient is added up in an order that the sizes alone decide."""
    what = "RMS norm's gradient"
    dev = _lib.require_gpu(dy, s, weight, dsum, what=what)
    no_gradient(what, dy, s, weight, dsum)
    _, width, code, weight_code = _check(dy, weight, epsilon, what)
    for t, name in ((s, "s"), (dsum, "dsum")):
        if t is not None and (t.shape != dy.shape or t.dtype not in (dy.dtype, torch.float32) or t.dtype != s.dtype):
            raise RuntimeError(f"{what}: {name} must be {tuple(dy.shape)} in {dy.dtype} or float32 (one type for both), "
                               f"got {t.dtype} {tuple(t.shape)}")
    dx = s.new_empty(s.shape)
    dweight = None if weight is None else dy.new_empty(width, dtype=torch.float32)
    if dy.numel() == 0:
        return dx, dweight if dweight is None else dweight.zero_()
    dy, n0, n1, y0, y1 = _by_rows(dy)
    s, s0, s1 = _split(s, n0, n1)
    d0 = d1 = 0
    if dsum is not None:
        dsum, d0, d1 = _split(dsum, n0, n1)
    weight = None if weight is None else weight.contiguous()
    need = 0 if dweight is None else _lib.query("spr_rms_norm_backward_workspace", n0 * n1, width)
    ws = _lib.workspace(need, dev) if need > 0 else None
    _lib.launch("spr_rms_norm_backward", dev, dy.data_ptr(), y0, y1, s.data_ptr(), s0, s1, _lib.ptr(dsum), d0, d1, n0, n1,
                width, code, _lib.DTYPE_CODE[s.dtype], _lib.ptr(weight), weight_code, float(epsilon), dx.data_ptr(),
                _lib.ptr(dweight), _lib.ptr(ws), need)
    return dx, dweight
