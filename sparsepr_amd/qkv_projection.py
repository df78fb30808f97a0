"""QKVProjection: what a model's block does in front of the attention, with the weights in 8 bits.

    front = QKVProjection(weight, heads=40, norm_weight=g, axis_dims=(44, 42, 42))   # once: weight [3 * 40 * 128, C]
    positions = grid_positions(21, 30, 52)                                           # or any [T, 3] / [B, T, 3]
    q, k, v, x = front(y, positions, residual=x)       # x + y normed to 8 bits, projected, Q and K turned by place
    out = SparsePRAttention(config)(q, k, v)

The norm of the hidden rows is the root-mean-square one.  With another norm in front (a layer norm with a scale and a
shift by time step, as Wan's blocks have it), `norm=False` takes rows as the caller has normed them.

The hidden rows are read once between the residual's addition and the 8-bit product; nothing is rounded to 16
bits in between.  The product's outputs are rounded to x's type, Q and K again where they are normed and where they
are turned.  All calls are kernels/rms_norm.py's, kernels/fp8.py's and kernels/axial_rope.py's, on torch's
current stream; none waits for the GPU, and a captured graph replays what an eager call does."""

from __future__ import annotations

import torch

from .kernels.axial_rope import axial_frequencies, axial_rope
from .kernels.fp8 import fp8_matmul, fp8_quantize
from .kernels.rms_norm import rms_norm, rms_norm_fp8


class QKVProjection:
    def __init__(self, weight: torch.Tensor, *, heads: int, kv_heads: int | None = None, axis_dims, theta: float = 10000.0,
                 pairs: str = "interleaved", norm_weight: torch.Tensor | None = None, bias: torch.Tensor | None = None,
                 q_norm: torch.Tensor | None = None, k_norm: torch.Tensor | None = None, epsilon: float = 1e-6,
                 fast_sums: bool = False,
                 norm: bool = True):
        """weight [(heads + 2 kv_heads) D, C]: the rows of Q, then K, then V, quantised here once (128 x 128 blocks).
        norm_weight [C] and bias as in rms_norm and fp8_matmul.  q_norm and k_norm norm Q and K before they are
        turned: [D] every head by itself, [heads * D] all channels together.  axis_dims: the rotated dims of each
        axis of the positions (axial_frequencies).  fast_sums: the product's (fp8_matmul).  norm False:
        x has been normed, and is quantised as it is."""
        kv_heads = heads if kv_heads is None else kv_heads
        what = "QKV projection"
        if heads < 1 or kv_heads < 1 or heads % kv_heads != 0:
            raise RuntimeError(f"{what}: {heads} query heads on {kv_heads} kv heads")
        if weight.dim() != 2 or weight.shape[0] % (heads + 2 * kv_heads) != 0 or weight.numel() == 0:
            raise RuntimeError(f"{what}: weight {tuple(weight.shape)} is not [({heads} + 2 * {kv_heads}) D, C]")
        if norm_weight is not None and not norm:
            raise RuntimeError(f"{what}: norm_weight is for a norm of x, which norm=False leaves to the caller")
        self.heads, self.kv_heads, self.norm = heads, kv_heads, norm
        self.head_dim = weight.shape[0] // (heads + 2 * kv_heads)
        for t, h, name in ((q_norm, heads, "q_norm"), (k_norm, kv_heads, "k_norm")):
            if t is not None and t.shape not in ((self.head_dim,), (h * self.head_dim,)):
                raise RuntimeError(f"{what}: {name} must be [{self.head_dim}] or [{h * self.head_dim}], got {tuple(t.shape)}")
        self.width = weight.shape[1]
        self.weight = fp8_quantize(weight, square=True)
        self.norm_weight, self.bias, self.q_norm, self.k_norm = norm_weight, bias, q_norm, k_norm
        self.freqs, self.axis = axial_frequencies(axis_dims, theta=theta, device=weight.device)
        self.pairs, self.epsilon, self.fast_sums = pairs, epsilon, fast_sums

    def _heads(self, x: torch.Tensor, heads: int, weight: torch.Tensor | None) -> torch.Tensor:
        """x [B, T, heads * D] -> [B, heads, T, D], normed where there is a weight."""
        if weight is not None and weight.shape[0] != self.head_dim:
            x = rms_norm(x, weight, epsilon=self.epsilon)
        x = x.unflatten(-1, (heads, self.head_dim))
        if weight is not None and weight.shape[0] == self.head_dim:
            x = rms_norm(x, weight, epsilon=self.epsilon)
        return x.transpose(1, 2)

    def __call__(self, x: torch.Tensor, positions: torch.Tensor, *, residual: torch.Tensor | None = None):
        """x [B, T, C] -> Q [B, heads, T, D], K and V [B, kv_heads, T, D] in x's type (V a view of the projection),
        and with a residual the sum x + residual as well."""
        if x.dim() != 3 or x.shape[2] != self.width:
            raise RuntimeError(f"QKV projection: x must be [B, T, {self.width}], got {tuple(x.shape)}")
        if not self.norm and residual is not None:
            raise RuntimeError("QKV projection: a residual is added in front of the norm, which norm=False leaves to the caller")
        total = []
        if self.norm:
            codes, scales, *total = rms_norm_fp8(x, self.norm_weight, residual=residual, epsilon=self.epsilon)
            codes, scales = codes.flatten(0, 1), scales.flatten(0, 1)
        else:
            codes, scales = fp8_quantize(x.flatten(0, 1))
        y = fp8_matmul(codes, scales, *self.weight, bias=self.bias, out_dtype=x.dtype,
                       fast_sums=self.fast_sums)
        q_dims, kv_dims = self.heads * self.head_dim, self.kv_heads * self.head_dim
        q, k, v = y.view(*x.shape[:2], q_dims + 2 * kv_dims).split((q_dims, kv_dims, kv_dims), -1)
        q, k = axial_rope(self._heads(q, self.heads, self.q_norm), self._heads(k, self.kv_heads, self.k_norm), positions,
                          self.freqs, self.axis, pairs=self.pairs)
        return q, k, self._heads(v, self.kv_heads, None), *total
