"""The hidden rows to Q, K, V and through the attention layer, and back through the gradients: the operators
together, as a block uses them."""

import numpy as np
import pytest
import torch

from tests import _fp8_model as model

pytestmark = pytest.mark.gpu


def _f64(t):
    return t.double().cpu().numpy()


def _front(dev, seed, heads, kv_heads, d, width, dtype, **kw):
    from sparsepr_amd.qkv_projection import QKVProjection

    g = torch.Generator(device=dev).manual_seed(seed)
    w = torch.randn((heads + 2 * kv_heads) * d, width, generator=g, device=dev) / width**0.5
    norm = 1 + 0.2 * torch.randn(width, generator=g, device=dev)
    x, res = (torch.randn(2, 150, width, generator=g, device=dev).to(dtype) for _ in range(2))
    return QKVProjection(w.to(dtype), heads=heads, kv_heads=kv_heads, norm_weight=norm, **kw), w.to(dtype), norm, x, res


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("heads,kv_heads,d,width,dims,pairs", [(6, 6, 64, 500, (16, 24, 24), "interleaved"),
                                                              (8, 2, 128, 640, (44, 42, 42), "halves")])
def test_projection_against_the_formula_in_64_bits(dev, dtype, heads, kv_heads, d, width, dims, pairs):
    """Rows and weights are off by half a step of their codes, 2^-4 of a value (2^-10 of its group's scale below the
    smallest normal code, 2^-9 / 224 of the group's largest): together 2^-3 + 2^-8 of the products' magnitudes, and
    half a step of the output's type twice (after the product and after the turn)."""
    from sparsepr_amd.kernels.axial_rope import grid_positions

    front, w, norm, x, res = _front(dev, d, heads, kv_heads, d, width, dtype, axis_dims=dims, pairs=pairs,
                                    bias=torch.linspace(-1, 1, (heads + 2 * kv_heads) * d, device=dev))
    positions = grid_positions(3, 5, 10, first=(40, 0, 0), device=dev)
    q, k, v, s = front(x, positions, residual=res)
    assert s.dtype == dtype and q.dtype == dtype and v.shape == (2, kv_heads, 150, d)
    y = model.norm(_f64(s).reshape(300, width), _f64(norm), 1e-6)
    want, size = y @ _f64(w).T + _f64(front.bias), np.abs(y) @ np.abs(_f64(w)).T
    top_y, top_w = np.abs(y).max(1, keepdims=True), np.abs(_f64(w)).max()
    low = 2.0**-9 / 224 * (top_y * np.abs(_f64(w)).sum(1) + top_w * np.abs(y).sum(1, keepdims=True))
    step = torch.finfo(dtype).eps
    bound = (2.0**-3 + 2.0**-8) * size + 1.1 * low + step * (np.abs(want) + size) + 1e-6 * size
    parts = np.split(np.stack([want, bound]).reshape(2, 2, 150, -1, d), [heads, heads + kv_heads], axis=3)
    p = np.broadcast_to(_f64(positions), (2, 150, 3))
    for got, (value, off), turned in ((q, parts[0], True), (k, parts[1], True), (v, parts[2], False)):
        value, off = value.transpose(0, 2, 1, 3), off.transpose(0, 2, 1, 3)
        if turned:
            value, _ = model.rotate(value, p, _f64(front.freqs), front.axis.cpu().numpy(), pairs)
            _, off = model.rotate(off, p, _f64(front.freqs), front.axis.cpu().numpy(), pairs)  # an error's length at both dims
        assert (np.abs(_f64(got) - value) <= off).all()


def test_projection_is_its_operators_one_by_one_and_replays(dev):
    from sparsepr_amd.kernels.axial_rope import axial_rope
    from sparsepr_amd.kernels.fp8 import fp8_matmul
    from sparsepr_amd.kernels.rms_norm import rms_norm, rms_norm_fp8

    for whole in (False, True):
        h, hk, d = 4, 2, 64
        qn = 1 + 0.1 * torch.arange(h * d if whole else d, device=dev) / 64
        kn = 1 - 0.1 * torch.arange(hk * d if whole else d, device=dev) / 256
        front, _, norm, x, res = _front(dev, 5, h, hk, d, 384, torch.bfloat16, axis_dims=(24, 20, 20), q_norm=qn, k_norm=kn)
        positions = torch.randint(0, 500, (2, 150, 3), generator=torch.Generator(device=dev).manual_seed(1), device=dev)
        inputs = [(x, res, positions), (res, x, positions + 3), (x * 2, x, positions * 2)]
        eager = [front(a, p, residual=b) for a, b, p in inputs]
        codes, scales, s = rms_norm_fp8(x, norm, residual=res)
        y = fp8_matmul(codes.view(300, -1), scales.view(300, -1), *front.weight).view(2, 150, -1)
        q, k, v = (t.contiguous() for t in y.split((h * d, hk * d, hk * d), -1))
        if whole:
            q, k = rms_norm(q, qn), rms_norm(k, kn)
        q, k, v = (t.view(2, 150, -1, d) for t in (q, k, v))
        if not whole:
            q, k = rms_norm(q, qn), rms_norm(k, kn)
        q, k = axial_rope(q.transpose(1, 2), k.transpose(1, 2), positions, front.freqs, front.axis)
        for got, want in zip(eager[0], (q, k, v.transpose(1, 2), s)):
            assert torch.equal(got, want)
        a, b, p = (t.clone() for t in inputs[0])
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = front(a, p, residual=b)
        for (u, w, z), want in zip(inputs, eager):
            a.copy_(u), b.copy_(w), p.copy_(z)
            graph.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(o, e) for o, e in zip(out, want))


def test_projection_feeds_the_attention_layer_and_the_cache(dev):
    from sparsepr_amd.kernels.axial_rope import grid_positions
    from sparsepr_amd.kv4_cache import KV4Cache
    from sparsepr_amd.layer import SparsePRAttention, SparsePRConfig
    from sparsepr_amd.qkv_projection import QKVProjection

    g = torch.Generator(device=dev).manual_seed(3)
    h, d, width, n = 2, 128, 256, 2 * 32 * 32
    w = (torch.randn(3 * h * d, width, generator=g, device=dev) / 16).to(torch.bfloat16)
    front = QKVProjection(w, heads=h, axis_dims=(44, 42, 42))
    x = torch.randn(1, n, width, generator=g, device=dev).to(torch.bfloat16)
    q, k, v = front(x, grid_positions(2, 32, 32, device=dev))
    cfg = SparsePRConfig(num_q_centroids=16, num_k_centroids=32, kmeans_iters=3, top_p=0.9, probe_rows=16)
    out = SparsePRAttention(cfg)(q, k, v)
    assert out.shape == (1, h, n, d) and bool(torch.isfinite(out.float()).all())
    assert torch.equal(out, SparsePRAttention(cfg)(q.contiguous(), k.contiguous(), v.contiguous()))
    cache = KV4Cache(num_pages=40, num_kv_heads=h, head_dim=d, max_sequences=1, device=dev)
    cache.append(k, v)
    token, key, value = front(x[:, -1:], torch.tensor([[2, 0, 0]], device=dev))  # the next frame's first token
    cache.append(key, value)
    assert torch.isfinite(cache.attend(token, causal=True).float()).all()
    cache.check()


def test_gradients_through_the_chain(dev):
    """d/dx of sum(q gq + k gk + v gv) through the turn, the 8-bit product and the norm.  The product's gradient is
    off by at most (2^-3 + 2^-8) |dy| |W| and what small codes lose, as above; the turn and the norm's gradient are
    linear in it, and add 1e-5 of the magnitudes that they add up."""
    from sparsepr_amd.kernels.axial_rope import axial_rope, grid_positions
    from sparsepr_amd.kernels.fp8 import fp8_matmul, fp8_quantize
    from sparsepr_amd.kernels.rms_norm import rms_norm_backward

    h, hk, d, width = 4, 2, 64, 320
    front, w, norm, x, _ = _front(dev, 8, h, hk, d, width, torch.float32, axis_dims=(24, 20, 20))
    positions = grid_positions(3, 5, 10, device=dev)
    g = torch.Generator(device=dev).manual_seed(9)
    gq, gk, gv = (torch.randn(2, n, 150, d, generator=g, device=dev) for n in (h, hk, hk))
    # the library's way back
    bq, bk = axial_rope(gq, gk, positions, front.freqs, front.axis, inverse=True)
    dy = torch.cat([t.transpose(1, 2).flatten(2) for t in (bq, bk, gv)], -1).view(300, -1)
    dn = fp8_matmul(*fp8_quantize(dy), *fp8_quantize(w, square=True, transpose=True), out_dtype=torch.float32)
    dx, dg = rms_norm_backward(dn.view(2, 150, width), x, norm)
    # torch's, in 64 bits and without the 8-bit rounding
    x64, n64, w64 = x.double().requires_grad_(), norm.double().requires_grad_(), w.double()
    y = (x64 * torch.rsqrt((x64 * x64).mean(-1, keepdim=True) + 1e-6) * n64) @ w64.t()
    q, k, v = (t.unflatten(-1, (-1, d)).transpose(1, 2) for t in y.split((h * d, hk * d, hk * d), -1))
    angle = positions.double()[:, front.axis.long()] * front.freqs
    turn = lambda t: torch.view_as_real(torch.view_as_complex(t.contiguous().unflatten(-1, (-1, 2)))  # noqa: E731
                                        * torch.polar(torch.ones_like(angle), angle)).flatten(-2)
    ((turn(q) * gq).sum() + (turn(k) * gk).sum() + (v * gv).sum()).backward()
    dy64, w64 = _f64(dy), _f64(w)
    low = 2.0**-9 / 224 * (np.abs(dy64).max(1, keepdims=True) * np.abs(w64).sum(0)
                           + np.abs(w64).max() * np.abs(dy64).sum(1, keepdims=True))
    off = (2.0**-3 + 2.0**-8 + 1e-5) * (np.abs(dy64) @ np.abs(w64)) + 1.1 * low
    s, n = np.abs(_f64(x).reshape(300, width)), np.abs(_f64(norm))
    r = 1 / np.sqrt((s * s).mean(-1, keepdims=True) + 1e-6)
    bound = r * (off * n + s * r * r * (off * n * s).mean(-1, keepdims=True)) * 1.01
    assert (np.abs(_f64(dx).reshape(300, width) - _f64(x64.grad).reshape(300, width)) <= bound).all()
    assert (np.abs(_f64(dg) - _f64(n64.grad)) <= (off * s * r).sum(0) * 1.01).all()


def test_refusals(dev):
    from sparsepr_amd.qkv_projection import QKVProjection

    w = torch.zeros(192, 64, device=dev)
    for kw, text in [(dict(heads=0), "0 query heads"), (dict(heads=3, kv_heads=2), "3 query heads on 2"), (dict(heads=5), "weight"),
                     (dict(heads=1, q_norm=w[0, :7]), "q_norm must be"), (dict(heads=1, axis_dims=(63,)), "must be even")]:
        with pytest.raises(RuntimeError, match=text):
            QKVProjection(w, **{"axis_dims": (64,), **kw})
    front = QKVProjection(w, heads=1, axis_dims=(64,))
    with pytest.raises(RuntimeError, match=r"x must be \[B, T, 64\]"):
        front(w[None, :, :32], torch.zeros(192, 1, device=dev))
    with pytest.raises(RuntimeError, match="positions must be"):
        front(w[None], torch.zeros(191, 1, device=dev))


def test_inputs_whose_gradient_or_tangent_would_be_lost_are_refused(dev):
    """Every tensor input of every function in front of the attention."""
    from torch.autograd import forward_ad

    from sparsepr_amd.kernels.axial_rope import axial_frequencies, axial_rope
    from sparsepr_amd.kernels.fp8 import fp8_dequantize, fp8_matmul, fp8_quantize
    from sparsepr_amd.kernels.rms_norm import rms_norm, rms_norm_backward, rms_norm_fp8
    from sparsepr_amd.qkv_projection import QKVProjection

    x, w, place = torch.randn(4, 64, device=dev), torch.ones(64, device=dev), torch.ones(4, 1, device=dev)
    codes, scales = fp8_quantize(x)
    freqs, axis = axial_frequencies((64,))
    front = QKVProjection(torch.randn(192, 64, device=dev), heads=1, axis_dims=(64,))
    calls = [(rms_norm, x, w), (lambda a, b, c: rms_norm(a, b, residual=c), x, w, x), (rms_norm_fp8, x, w),
             (lambda a, b, c: rms_norm_fp8(a, b, residual=c), x, w, x),
             (lambda a, b, c, d: rms_norm_backward(a, b, c, dsum=d), x, x, w, x), (fp8_quantize, x),
             (lambda a: fp8_dequantize(a, scales), codes),
             (lambda a, b, c: fp8_matmul(a, scales, b, scales, bias=c), codes, codes, w[:4]),
             (lambda a, b, c, d: axial_rope(a, b, c, d, axis), x[None, None], x[None, None], place, freqs),
             (lambda a, b: front(a, place, residual=b), x[None], x[None])]
    for call, *given in calls:
        call(*given)
        for i, t in enumerate(given):
            leaf = t.float().clone().requires_grad_()
            with pytest.raises(RuntimeError, match="autograd does not record"):
                call(*given[:i], leaf.to(t.dtype), *given[i + 1:])
            with forward_ad.dual_level():
                call(*given)
                dual = forward_ad.make_dual(t.float(), torch.ones_like(t, dtype=torch.float32)).to(t.dtype)
                with torch.no_grad(), pytest.raises(RuntimeError, match="forward mode"):
                    call(*given[:i], dual, *given[i + 1:])


@pytest.mark.parametrize("norms", [None, "head", "all"])
@pytest.mark.parametrize("b,t", [(0, 150), (2, 0), (0, 0)])
def test_no_batch_and_no_tokens(dev, b, t, norms):
    h, hk, d = 4, 2, 64
    qn, kn = (None if norms is None else torch.ones(d if norms == "head" else n * d, device=dev) for n in (h, hk))
    front, *_ = _front(dev, 2, h, hk, d, 384, torch.bfloat16, axis_dims=(24, 20, 20), q_norm=qn, k_norm=kn)
    x = torch.zeros(b, t, 384, device=dev, dtype=torch.bfloat16)
    for places in (torch.zeros(t, 3, device=dev), torch.zeros(b, t, 3, device=dev)):
        for residual in (None, x, x.float()):
            q, k, v, *total = front(x, places, residual=residual)
            assert q.shape == (b, h, t, d) and k.shape == v.shape == (b, hk, t, d) and v.dtype == x.dtype
            assert [s.shape for s in total] == ([] if residual is None else [(b, t, 384)])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_rows_that_the_caller_has_normed(dev, dtype):
    """A layer norm with a scale and a shift per batch in front, as the operators one by one give it, and replayed."""
    from sparsepr_amd.kernels.axial_rope import axial_rope
    from sparsepr_amd.kernels.fp8 import fp8_matmul, fp8_quantize
    from sparsepr_amd.qkv_projection import QKVProjection

    h, hk, d, width = 4, 2, 64, 500
    g = torch.Generator(device=dev).manual_seed(6)
    w = (torch.randn((h + 2 * hk) * d, width, generator=g, device=dev) / width**0.5).to(dtype)
    x, scale, shift = (torch.randn(2, n, width, generator=g, device=dev).to(dtype) for n in (150, 1, 1))
    x = torch.nn.functional.layer_norm(x, (width,)) * (1 + scale) + shift
    front = QKVProjection(w, heads=h, kv_heads=hk, axis_dims=(24, 20, 20), norm=False)
    places = torch.randint(0, 500, (150, 3), generator=g, device=dev)
    q, k, v = front(x, places)
    codes, scales = fp8_quantize(x.view(300, width))
    y = fp8_matmul(codes, scales, *fp8_quantize(w, square=True), out_dtype=dtype).view(2, 150, -1)
    want_q, want_k, want_v = (t.unflatten(-1, (-1, d)).transpose(1, 2) for t in y.split((h * d, hk * d, hk * d), -1))
    want_q, want_k = axial_rope(want_q, want_k, places, front.freqs, front.axis)
    assert torch.equal(q, want_q) and torch.equal(k, want_k) and torch.equal(v, want_v)
    assert all(torch.equal(a, b) for a, b in zip(front(x.transpose(0, 1).contiguous().transpose(0, 1), places), (q, k, v)))
    assert front(x[:0], places)[2].shape == (0, hk, 150, d) and front(x[:, :0], places[:0])[0].shape == (2, h, 0, d)
    buffer, graph = x.clone(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = front(buffer, places)
    for t in (x, 2 * x, x.flip(1)):
        eager = front(t, places)
        buffer.copy_(t)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, eager))
    with pytest.raises(RuntimeError, match="a residual is added in front of the norm"):
        front(x, places, residual=x)
    with pytest.raises(RuntimeError, match="norm_weight is for a norm of x"):
        QKVProjection(w, heads=h, kv_heads=hk, axis_dims=(64,), norm=False, norm_weight=w[0])
