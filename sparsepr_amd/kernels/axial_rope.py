"""Rotary positions with several axes (time, height, width for a video; height, width for an image; one for
text) on the HIP kernel of csrc/spr_axial_rope.hip.

Pair i of a head's rotated dims turns by positions[..., axis[i]] * freqs[i] radians:
    (a, b) -> (a cos - b sin, b cos + a sin)
`pairs` says which dims a pair is: "interleaved" (2i, 2i + 1), or "halves" (i, i + R / 2) of R rotated dims.
Dims from R on are copied.  The angle is kept in 64 bits until whole turns are off it."""

from __future__ import annotations

import torch

from .. import _lib
from .fp8 import no_gradient

POSITION_CODE = {torch.int32: 0, torch.int64: 1, torch.float32: 2, torch.float64: 3}


def axial_frequencies(axis_dims, *, theta: float = 10000.0, device: torch.device | str | None = None):
    """(freqs float64 [R / 2], axis int32 [R / 2]) for axes of axis_dims[a] dims each, one behind the other (Wan:
    44, 42, 42 of 128): pair j of an axis of n dims has theta^(-2 j / n) radians a step."""
    for n in axis_dims:
        if n < 0 or n % 2 != 0:
            raise RuntimeError(f"axial RoPE: dims of an axis must be even, got {tuple(axis_dims)}")
    if not 0.0 < theta < float("inf"):
        raise RuntimeError(f"axial RoPE: theta must be positive and finite, got {theta}")
    freqs = [theta ** (-j / n) for n in axis_dims for j in range(0, n, 2)]
    axis = [a for a, n in enumerate(axis_dims) for _ in range(0, n, 2)]
    dev = torch.device("cuda" if device is None else device)
    return torch.tensor(freqs, dtype=torch.float64, device=dev), torch.tensor(axis, dtype=torch.int32, device=dev)


def grid_positions(frames: int, height: int, width: int, *, first=(0, 0, 0), device: torch.device | str | None = None):
    """int32 [frames * height * width, 3]: the (time, height, width) of a video's tokens, frame by frame and line
    by line, from `first` on."""
    dev = torch.device("cuda" if device is None else device)
    axes = [torch.arange(n, dtype=torch.int32, device=dev) + f for n, f in zip((frames, height, width), first)]
    return torch.stack(torch.meshgrid(*axes, indexing="ij"), -1).reshape(-1, 3)


def _strided(x: torch.Tensor) -> tuple[torch.Tensor, int, int, int]:
    """x [B, H, T, D] and its strides over the first three dims; a copy where rows are not packed."""
    b, h, t, d = x.stride()
    if d != 1 and x.shape[3] > 1:
        x = x.contiguous()
        b, h, t, d = x.stride()
    return x, b, h, t


def axial_rope(q: torch.Tensor, k: torch.Tensor | None, positions: torch.Tensor, freqs: torch.Tensor,
               axis: torch.Tensor, *, pairs: str = "interleaved", inverse: bool = False):
    """Q [B, Hq, T, D] and K [B, Hkv, T, D] (or None) turned: new contiguous tensors (q', k'), what the attention
    takes.  bf16, fp16 or fp32, any strides with packed rows (a projection's [B, T, H, D], transposed), D a
    multiple of 8 up to 1024.  positions [T, A] or [B, T, A], int32, int64, float32 or float64; freqs float64 and
    axis int32 [R / 2] (axial_frequencies), R a multiple of 8.  An axis that the positions do not have gives NaN.

    `inverse` turns back: with the gradients of q' and k' it gives those of q and k.  Autograd does not record the
    call: inputs that require a gradient are refused while it records, and those with a tangent."""
    what = "axial RoPE"
    dev = _lib.require_gpu(q, k, positions, freqs, axis, what=what)
    no_gradient(what, q, k, positions, freqs)
    shape, dtype = q.shape, _lib.DTYPE_CODE.get(q.dtype)
    if len(shape) != 4 or dtype is None:
        raise RuntimeError(f"{what}: q must be [B, H, T, D] in bfloat16, float16 or float32, got {q.dtype} "
                           f"{tuple(q.shape)}")
    b, h, t, d = shape
    hk = 0
    if k is not None:
        shape = k.shape
        hk = shape[1] if len(shape) == 4 else -1
        if shape != (b, hk, t, d) or k.dtype is not q.dtype:
            raise RuntimeError(f"{what}: k must be [{b}, heads, {t}, {d}] in {q.dtype}, got {k.dtype} {tuple(shape)}")
    if pairs != "interleaved" and pairs != "halves":
        raise RuntimeError(f"{what}: pairs must be 'interleaved' or 'halves', got {pairs!r}")
    place = positions.shape
    axes = place[-1] if len(place) > 1 else 0
    code = POSITION_CODE.get(positions.dtype)
    if code is None or (place != (t, axes) and place != (b, t, axes)):
        raise RuntimeError(f"{what}: positions must be [{t}, axes] or [{b}, {t}, axes] in int32, int64, float32 or "
                           f"float64, got {positions.dtype} {tuple(positions.shape)}")
    turns = freqs.shape
    if freqs.dtype is not torch.float64 or axis.dtype is not torch.int32 or len(turns) != 1 \
            or axis.shape != turns or not freqs.is_contiguous() or not axis.is_contiguous():
        raise RuntimeError(f"{what}: freqs must be contiguous float64 and axis contiguous int32 of one length, got "
                           f"{freqs.dtype} {tuple(freqs.shape)} / {axis.dtype} {tuple(axis.shape)}")
    rotated = 2 * turns[0]
    if d % 8 != 0 or not 8 <= d <= 1024 or rotated % 8 != 0 or rotated > d:
        raise RuntimeError(f"{what}: {rotated} rotated dims of {d} (both multiples of 8, D at most 1024)")
    if h >= 1 << 20 or hk >= 1 << 20:
        raise RuntimeError(f"{what}: {h} and {hk} heads")
    if not 1 <= axes <= 16:
        raise RuntimeError(f"{what}: {axes} axes, 1 to 16 are taken")
    q_out = q.new_empty((b, h, t, d))
    k_out = None if k is None else q.new_empty((b, hk, t, d))
    if b * t * (h + hk) > 0:
        positions = positions.contiguous()
        kb = kh = kt = k_at = k_to = 0
        q, qb, qh, qt = _strided(q)
        if k is not None:
            k, kb, kh, kt = _strided(k)
            k_at, k_to = k.data_ptr(), k_out.data_ptr()
        _lib.launch("spr_axial_rope", dev, q.data_ptr(), qb, qh, qt, h, k_at, kb, kh, kt, hk, dtype, b, t, d, rotated,
                    positions.data_ptr(), code, t * axes if len(place) == 3 else 0, axes, freqs.data_ptr(),
                    axis.data_ptr(), int(pairs == "halves"), int(inverse), q_out.data_ptr(), k_to)
    return q_out, k_out
