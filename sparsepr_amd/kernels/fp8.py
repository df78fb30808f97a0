"""8-bit matrices and their product on the HIP kernels of csrc/spr_fp8.hip and csrc/spr_fp8_matmul.hip.

A matrix in 8 bits is two tensors:
  codes   float8_e4m3fn [rows, wide], wide = the row's width rounded up to 16, zeros behind the width
  scales  uint8 [rows, blocks], blocks = the width / 128 rounded up: the byte b of 128 values of a row
          stands for 2^(b - 127); or [rows / 128 rounded up, blocks] for 128 x 128 values ("square")
The exponent is the smallest one with which the group's largest magnitude is at most 448, so scaling
is exact and a value is off by half a step of its code alone.  A group with an infinity or a NaN has the
byte 255 and is NaN.

The products of a linear layer y = x W^T are all `fp8_matmul`, which sums along the rows of both sides:
  y   fp8_matmul(*fp8_quantize(x), *fp8_quantize(w, square=True))
  dx  fp8_matmul(*fp8_quantize(dy), *fp8_quantize(w, square=True, transpose=True))
  dw  fp8_matmul(*fp8_quantize(dy, transpose=True), *fp8_quantize(x, transpose=True))
Square blocks hold the same values either way round, so y and dx see one weight.  None of the functions
is recorded by autograd: inputs that require a gradient are refused while it records, and those with a tangent."""

from __future__ import annotations

import torch
from torch.autograd import forward_ad

from .. import _lib

BLOCK = 128
MAX_SIZE = 1 << 30  # of a dim: the entry points count columns in 32 bits
MAX_SUM = 1 << 22  # terms of a product, and bytes from row to row
ROWS = (1 << 24) - 1  # that one launch quantises, with scales of their own
GROUPS = (1 << 28) - 65  # of 128 values, the same
CODES = torch.float8_e4m3fn


def no_gradient(what: str, *tensors: torch.Tensor | None) -> None:
    """Refuse what autograd would lose without a word: gradients that it records, and tangents (forward mode; no_grad
    does not stop those, so they are looked for wherever a level is open)."""
    for t in tensors:
        if t is None:
            continue
        if t.requires_grad and torch.is_grad_enabled():
            raise RuntimeError(f"{what}: autograd does not record this call; call it under torch.no_grad() and use the "
                               "gradient functions beside it")
        if forward_ad._current_level >= 0 and forward_ad.unpack_dual(t).tangent is not None:
            raise RuntimeError(f"{what}: autograd's forward mode would lose a tangent in this call; give it the primal")


def _packed_rows(x: torch.Tensor, rows: int, width: int) -> tuple[torch.Tensor, int]:
    """x [R, C] and its row stride: itself where rows are packed, else a copy."""
    step, packed = x.stride()
    if packed == 1 or width == 1:
        return x, step if rows > 1 else width
    return x.contiguous(), width


def _check_matrix(codes: torch.Tensor, scales: torch.Tensor, what: str, name: str) -> tuple[int, int, int]:
    """(rows, width, whether a scale is of 128 rows) of an 8-bit matrix."""
    shape = codes.shape
    if codes.dtype is not CODES or len(shape) != 2:
        raise RuntimeError(f"{what}: {name} must be float8_e4m3fn [rows, width], got {codes.dtype} {tuple(codes.shape)}")
    rows, width = shape
    blocks = -(-width // BLOCK)
    if rows > MAX_SIZE or width > MAX_SIZE:
        raise RuntimeError(f"{what}: {name} is {tuple(codes.shape)}, {MAX_SIZE} rows or columns at most")
    if width % 16 != 0:
        raise RuntimeError(f"{what}: the width of {name} ({width}) must be a multiple of 16 (zeros behind the row)")
    shape = scales.shape
    if scales.dtype is not torch.uint8 or len(shape) != 2 or shape[1] != blocks \
            or (shape[0] != rows and shape[0] != -(-rows // BLOCK)):
        raise RuntimeError(f"{what}: the scales of {name} must be uint8 [{rows} or {-(-rows // BLOCK)}, {blocks}], got "
                           f"{scales.dtype} {tuple(scales.shape)}")
    return rows, width, int(shape[0] != rows)


def _as_read(codes: torch.Tensor, scales: torch.Tensor, rows: int, width: int,
             most: int = 1 << 62) -> tuple[torch.Tensor, int, torch.Tensor, int]:
    """Codes with packed rows that start on 16 bytes, at most `most` bytes apart, and scales with packed rows, and their
    row strides."""
    ld, packed = codes.stride()
    if rows == 1:
        ld = width
    if packed != 1 or ld % 16 != 0 or not width <= ld <= most or codes.data_ptr() % 16 != 0:  # (the width is 16 or more)
        codes, ld = codes.clone(memory_format=torch.contiguous_format), width
    scales_ld, packed = scales.stride()
    if packed != 1 and width > BLOCK:
        scales = scales.contiguous()
        scales_ld = scales.stride(0)
    return codes, ld, scales, scales_ld


def fp8_quantize(x: torch.Tensor, *, square: bool = False, transpose: bool = False):
    """x [R, C] in bf16, fp16 or fp32 -> (codes, scales), see the module's text.

    `square`: one scale for 128 x 128 values, else for 128 values of a row.  `transpose`: the 8-bit matrix
    of x^T, codes [C, R rounded up to 16], its groups along x's columns.  R and C are at most 2^30, with either R
    at most 65535 * 128 and R C / 128 below 2^28.  Without them more than 2^24 rows take several launches."""
    what = "8-bit quantisation"
    dev = _lib.require_gpu(x, what=what)
    no_gradient(what, x)
    shape, code = x.shape, _lib.DTYPE_CODE.get(x.dtype)
    if len(shape) != 2 or code is None:
        raise RuntimeError(f"{what}: x must be [rows, width] in bfloat16, float16 or float32, got {x.dtype} "
                           f"{tuple(x.shape)}")
    height, across = shape
    if height > MAX_SIZE or across > MAX_SIZE:
        raise RuntimeError(f"{what}: x is {tuple(x.shape)}, {MAX_SIZE} rows or columns at most")
    rows, width = (across, height) if transpose else (height, across)
    codes = x.new_empty((rows, -(-width // 16) * 16), dtype=CODES)
    scales = x.new_empty((-(-rows // BLOCK) if square else rows, -(-width // BLOCK)), dtype=torch.uint8)
    if height > 0 and across > 0:
        x, ld = _packed_rows(x, height, across)
        groups = -(-across // BLOCK)
        step = height
        if not square and not transpose and (height > ROWS or height * groups > GROUPS):
            step = min(ROWS, GROUPS // groups)
        for r in range(0, height, step):
            _lib.launch("spr_fp8_quantize", dev, x.data_ptr() + r * ld * x.element_size(), ld, min(step, height - r), across,
                        code, int(square), int(transpose), codes.data_ptr() + r * codes.shape[1],
                        scales.data_ptr() + r * groups)
    return codes, scales


def fp8_dequantize(codes: torch.Tensor, scales: torch.Tensor, *, dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """The values of an 8-bit matrix, [rows, wide] in `dtype`: exact in fp32, and in bf16 but at the ends of its
    range (fp16 rounds and overflows)."""
    what = "8-bit values"
    dev = _lib.require_gpu(codes, scales, what=what)
    no_gradient(what, codes)
    rows, width, square = _check_matrix(codes, scales, what, "codes")
    code = _lib.DTYPE_CODE.get(dtype)
    if code is None:
        raise RuntimeError(f"{what}: dtype must be bfloat16, float16 or float32, got {dtype}")
    out = codes.new_empty((rows, width), dtype=dtype)
    if rows > 0 and width > 0:
        codes, ld, scales, scales_ld = _as_read(codes, scales, rows, width)
        _lib.launch("spr_fp8_dequantize", dev, codes.data_ptr(), ld, scales.data_ptr(), scales_ld, square, rows, width,
                    code, out.data_ptr())
    return out


def fp8_matmul(a: torch.Tensor, a_scales: torch.Tensor, b: torch.Tensor, b_scales: torch.Tensor, *,
               bias: torch.Tensor | None = None, out_dtype: torch.dtype = torch.bfloat16,
               fast_sums: bool = False) -> torch.Tensor:
    """a b^T + bias for 8-bit matrices a [M, K] and b [N, K]: out [M, N] in `out_dtype` (bf16, fp16 or fp32),
    summed in fp32 and rounded once.  bias [N] in any of the three types.  The values are multiplied as
    fp8_dequantize gives them in bf16, exact for scale bytes 3 to 246.

    `fast_sums`, for outputs in 16 bits: up to twice the rate, on the 8-bit matrix instruction.  It adds eight
    neighbouring products at a time and keeps digits down to 2^-13 of the largest of them (the sums of the eights
    are fp32).  What it cuts is 5e-5 of the norm on normal rows, a thirtieth of bf16's own rounding and a quarter
    of fp16's; where large products cancel it may be all of an output.

    Codes whose rows are not packed, do not start on 16 bytes or are more than 2^22 bytes apart are copied first."""
    what = "8-bit product"
    dev = _lib.require_gpu(a, a_scales, b, b_scales, bias, what=what)
    no_gradient(what, a, b, bias)
    m, k, a_square = _check_matrix(a, a_scales, what, "a")
    n, kb, b_square = _check_matrix(b, b_scales, what, "b")
    if k != kb:
        raise RuntimeError(f"{what}: a is [{m}, {k}], b [{n}, {kb}]")
    if k > MAX_SUM:
        raise RuntimeError(f"{what}: sums of {k} terms, {MAX_SUM} are taken")
    code, bias_at, bias_code = _lib.DTYPE_CODE.get(out_dtype), 0, 0
    if code is None:
        raise RuntimeError(f"{what}: out_dtype must be bfloat16, float16 or float32, got {out_dtype}")
    if fast_sums and code == 2:
        raise RuntimeError(f"{what}: fast sums are for outputs in 16 bits, got {out_dtype}")
    if bias is not None:
        bias_code = _lib.DTYPE_CODE.get(bias.dtype)
        if bias.shape != (n,) or bias_code is None:
            raise RuntimeError(f"{what}: bias must be [{n}] in bfloat16, float16 or float32, got {bias.dtype} "
                               f"{tuple(bias.shape)}")
        bias = bias.contiguous()
        bias_at = bias.data_ptr()
    out = a.new_empty((m, n), dtype=out_dtype)
    if k == 0:  # (no rows that a weight's gradient would be summed over)
        return out.zero_() if bias is None else out.copy_(bias)
    if m > 0 and n > 0:
        a, a_ld, a_scales, a_scales_ld = _as_read(a, a_scales, m, k, MAX_SUM)
        b, b_ld, b_scales, b_scales_ld = _as_read(b, b_scales, n, k, MAX_SUM)
        _lib.launch("spr_fp8_matmul_ex", dev, a.data_ptr(), a_ld, a_scales.data_ptr(), a_scales_ld, a_square, b.data_ptr(),
                    b_ld, b_scales.data_ptr(), b_scales_ld, b_square, m, n, k, bias_at, bias_code, code, int(fast_sums),
                    out.data_ptr())
    return out
