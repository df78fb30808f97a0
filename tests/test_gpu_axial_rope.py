"""Rotary positions with several axes on the GPU against the formula in 64 bits.

A turn below one half, rounded to fp32, is off by 2^-26, its angle by 2 pi of that, 9.4e-8; sine and cosine are off by
at most 2^-23 (two steps below one), the two products and their sum by 2^-23 of the pair's length: 3.4e-7 of it
together, and half a step of the output's type."""

import numpy as np
import pytest
import torch

from tests import _fp8_model as model

pytestmark = pytest.mark.gpu

DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
HALF = {t: torch.finfo(t).eps / 2 for t in DT.values()}
TINY = {torch.bfloat16: 2.0**-134, torch.float16: 2.0**-25, torch.float32: 2.0**-126}


def _f64(t):
    return t.double().cpu().numpy()


def _check(x, got, positions, freqs, axis, pairs, inverse):
    assert got.shape == x.shape and got.dtype == x.dtype and got.is_contiguous()
    p = _f64(positions)
    p = np.broadcast_to(p if p.ndim == 3 else p[None], (x.shape[0], *p.shape[-2:]))
    want, size = model.rotate(_f64(x), p, _f64(freqs), axis.cpu().numpy(), pairs, inverse)
    assert (np.abs(_f64(got) - want) <= HALF[x.dtype] * np.abs(want) + 3.5e-7 * size + TINY[x.dtype]).all()
    r = 2 * len(freqs)
    assert torch.equal(got[..., r:], x[..., r:])


CASES = [(1, 1, 1, 1, 64, (64,)), (1, 1, 40, 8, 128, (44, 42, 42)), (2, 37, 3, 3, 128, (32, 48, 48)), (3, 50, 16, 4, 80, (32, 32)),
         (1, 300, 5, 0, 96, (24, 24)), (2, 11, 4, 2, 256, (64, 64, 64)), (1, 4099, 24, 24, 64, (16, 24, 24)), (1, 3, 2, 1, 8, (8,)),
         (1, 9, 2, 2, 1024, (512, 256, 256)), (2, 5, 3, 1, 72, (40, 16))]


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("pairs", ["interleaved", "halves"])
@pytest.mark.parametrize("b,t,h,hk,d,dims", CASES)
def test_rotation_and_its_inverse(dev, dtype, pairs, b, t, h, hk, d, dims):
    from sparsepr_amd.kernels.axial_rope import axial_frequencies, axial_rope

    g = torch.Generator().manual_seed(t + d)
    # as a projection leaves them, [B, T, H, D], seen by heads
    q, k = (torch.randn(b, t, n, d, generator=g).to(DT[dtype]).to(dev).transpose(1, 2) for n in (h, hk))
    freqs, axis = axial_frequencies(dims)
    kind = [torch.int32, torch.int64, torch.float32, torch.float64][(t + d + len(dims)) % 4]
    positions = (torch.rand(b, t, len(dims), generator=g, dtype=torch.float64) * 119000).to(kind).to(dev)
    for inverse in (False, True):
        got = axial_rope(q, k if hk else None, positions, freqs, axis, pairs=pairs, inverse=inverse)
        _check(q, got[0], positions, freqs, axis, pairs, inverse)
        if hk:
            _check(k, got[1], positions, freqs, axis, pairs, inverse)
        else:
            assert got[1] is None
    one = axial_rope(q, None, positions[0], freqs, axis, pairs=pairs)[0]  # one set of places for the whole batch
    _check(q, one, positions[0], freqs, axis, pairs, False)


def test_far_places(dev):
    """A hundred million steps on, where an angle in fp32 has no digit left."""
    from sparsepr_amd.kernels.axial_rope import axial_frequencies, axial_rope

    freqs, axis = axial_frequencies((32, 32))
    q = torch.randn(1, 2, 64, 64, generator=torch.Generator().manual_seed(1)).to(dev)
    positions = (torch.arange(64, device=dev)[:, None] * torch.tensor([1562501, -937501], device=dev)).contiguous()
    _check(q, axial_rope(q, None, positions, freqs, axis)[0], positions, freqs, axis, "interleaved", False)


def test_many_tokens_and_many_heads(dev):
    """More rows than a launch that gives every head its own lanes would take at once, checked at some tokens."""
    from sparsepr_amd.kernels.axial_rope import axial_frequencies, axial_rope, grid_positions

    freqs, axis = axial_frequencies((44, 42, 42))
    positions = grid_positions(21, 30, 52, first=(7, 0, 0))
    q = torch.randn(1, 32760, 40, 128, generator=torch.Generator(device=dev).manual_seed(1), device=dev).to(torch.bfloat16)
    q = q.transpose(1, 2)
    got, _ = axial_rope(q, None, positions, freqs, axis)
    at = torch.tensor([0, 1, 51, 52, 1559, 1560, 16379, 32758, 32759], device=dev)
    _check(q[:, :, at], got[:, :, at].contiguous(), positions[at], freqs, axis, "interleaved", False)


def test_inverse_undoes_and_keeps_lengths_and_products(dev):
    """Rotations of Q and K at places p and p + n: their products go by n alone (fp32: 2^-20 of the lengths)."""
    from sparsepr_amd.kernels.axial_rope import axial_frequencies, axial_rope

    freqs, axis = axial_frequencies((32, 48, 48))
    g = torch.Generator(device=dev).manual_seed(2)
    q, k = (torch.randn(1, 4, 1, 128, generator=g, device=dev).expand(1, 4, 20, 128) for _ in range(2))
    p = torch.randint(0, 1000, (20, 3), generator=g, device=dev)
    a, _ = axial_rope(q, None, p, freqs, axis)
    b, _ = axial_rope(k, None, p + torch.tensor([3, -2, 9], device=dev), freqs, axis)
    dots = (a.double() * b.double()).sum(-1)
    size = a.double().norm(dim=-1) * b.double().norm(dim=-1)
    assert ((dots - dots[..., :1]).abs() <= 2.0**-20 * size).all()
    back, _ = axial_rope(a, None, p, freqs, axis, inverse=True)
    assert ((back - q).abs() <= 2.0**-20 * q.norm(dim=-1, keepdim=True)).all()


def test_strides_offsets_and_own_frequencies(dev):
    from sparsepr_amd.kernels.axial_rope import axial_rope

    g = torch.Generator(device=dev).manual_seed(3)
    base = torch.randn(2, 9, 3, 6, 72, generator=g, device=dev).to(torch.bfloat16)
    freqs = torch.rand(20, generator=g, device=dev, dtype=torch.float64)
    axis = torch.tensor([2, 0, 1, 1] * 5, dtype=torch.int32, device=dev)
    p = torch.randint(-50, 50, (2, 9, 3), generator=g, device=dev, dtype=torch.int32)
    q = base[:, :, 1].transpose(1, 2)
    for x, y in ((q[..., 8:], q[..., :-8]), (q[..., 1:65], q[..., 3:67]), (q[:, ::2, :, :64], q[:, 1::2, :, :64]),
                 (q[:, :1, :, :64].expand(2, 5, 9, 64), q[..., :64]), (q[..., :64].contiguous(), q[..., 7:71].contiguous()),
                 (base[..., 2, :, :].permute(0, 2, 1, 3)[..., :64], q[:, :, :, 8:])):
        for got, z in zip(axial_rope(x, y, p, freqs, axis, pairs="halves"), (x, y)):
            _check(z, got, p, freqs, axis, "halves", False)
    odd = base.permute(0, 3, 4, 1, 2)[:, :, :64, :, 0].transpose(2, 3)
    flipped = base[:, :, 0].permute(0, 2, 3, 1).contiguous()[:, :, :64].transpose(2, 3)  # rows not packed: copied
    for x in (odd, flipped):
        _check(x, axial_rope(x, None, p, freqs, axis)[0], p, freqs, axis, "interleaved", False)


def test_nan_places_missing_axes_and_no_rotation(dev):
    from sparsepr_amd.kernels.axial_rope import axial_rope

    q = torch.randn(1, 2, 4, 64, generator=torch.Generator().manual_seed(4)).to(dev)
    freqs = torch.ones(16, dtype=torch.float64, device=dev)
    axis = torch.tensor([0] * 8 + [1] * 8, dtype=torch.int32, device=dev)
    p = torch.zeros(4, 2, device=dev)
    p[1, 0], p[2, 1] = float("nan"), float("inf")
    y = axial_rope(q, None, p, freqs, axis)[0]
    nan = torch.isnan(y)
    assert nan[:, :, 1, :16].all() and not nan[:, :, 1, 16:].any() and nan[:, :, 2, 16:32].all() and not nan[:, :, 2, 32:].any()
    assert torch.equal(y[:, :, [0, 3]], q[:, :, [0, 3]])
    axis[9], axis[10] = 2, -1  # axes that the positions do not have
    y = axial_rope(q, None, p[:1].expand(4, 2), freqs, axis)[0]
    nan = torch.isnan(y)
    assert nan[..., 18:22].all() and not nan[..., :18].any() and not nan[..., 22:].any()
    assert torch.equal(axial_rope(q, None, p, freqs[:0], axis[:0])[0], q)


def test_empty_and_refused(dev):
    from sparsepr_amd.kernels.axial_rope import axial_rope

    q = torch.zeros(2, 3, 5, 64, device=dev)
    f, a = torch.ones(32, dtype=torch.float64, device=dev), torch.zeros(32, dtype=torch.int32, device=dev)
    p = torch.zeros(5, 1, device=dev)
    assert axial_rope(q[:, :, :0], q[:, :1, :0], p[:0], f, a)[1].shape == (2, 1, 0, 64)
    assert axial_rope(q[:, :0], q, p, f, a)[0].shape == (2, 0, 5, 64)
    for bad, text in [(lambda: axial_rope(q[0], None, p, f, a), "q must be"), (lambda: axial_rope(q.double(), None, p, f, a), "q must be"),
                      (lambda: axial_rope(q, q.half(), p, f, a), "k must be"), (lambda: axial_rope(q, q[:, :, :4], p, f, a), "k must be"),
                      (lambda: axial_rope(q, q, p[:4], f, a), "positions must be"), (lambda: axial_rope(q, q, p.half(), f, a), "positions must be"),
                      (lambda: axial_rope(q, q, p[None], f, a), "positions must be"), (lambda: axial_rope(q, q, p, f.float(), a), "freqs must be"),
                      (lambda: axial_rope(q, q, p, f, a.long()), "freqs must be"), (lambda: axial_rope(q, q, p, f[:30], a[:30]), "60 rotated"),
                      (lambda: axial_rope(q[..., :60], None, p, f[:28], a[:28]), "56 rotated dims of 60"),
                      (lambda: axial_rope(q, q, p[:, :0], f, a), "0 axes"), (lambda: axial_rope(q, q, p, f, a, pairs="both"), "pairs must be"),
                      (lambda: axial_rope(q.clone().requires_grad_(), None, p, f, a), "autograd"),
                      (lambda: axial_rope(q, q, p.cpu(), f, a), "require GPU tensors")]:
        with pytest.raises(RuntimeError, match=text):
            bad()


def test_replays_and_another_stream(dev):
    from sparsepr_amd.kernels.axial_rope import axial_frequencies, axial_rope

    freqs, axis = axial_frequencies((16, 24, 24))
    g = torch.Generator(device=dev).manual_seed(5)
    q, p = torch.zeros(1, 4, 1, 64, device=dev), torch.zeros(1, 3, dtype=torch.int32, device=dev)
    inputs = [(torch.randn(1, 4, 1, 64, generator=g, device=dev), torch.randint(0, 99, (1, 3), generator=g, device=dev).int())
              for _ in range(4)]
    eager = [axial_rope(x, x, y, freqs, axis) for x, y in inputs]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        beside = axial_rope(inputs[0][0], None, inputs[0][1], freqs, axis)[0]
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(beside, eager[0][0])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = axial_rope(q, q, p, freqs, axis)
    for (x, y), want in zip(inputs, eager):
        q.copy_(x), p.copy_(y)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out[0], want[0]) and torch.equal(out[1], want[1])


def test_more_heads_than_an_entry_point_counts(dev):
    from sparsepr_amd.kernels.axial_rope import axial_frequencies, axial_rope

    freqs, axis = axial_frequencies((8,))
    one, place = torch.zeros(1, 1, 1, 8, device=dev), torch.zeros(1, 1, device=dev)
    many = one.expand(1, 2**32 + 1, 1, 8)
    for q, k in ((many, None), (one, many)):
        with pytest.raises(RuntimeError, match="heads"):
            axial_rope(q, k, place, freqs, axis)


def test_the_digits_of_a_turn_below_fp32_count(dev):
    """Pairs (1, 0) come back as cosine and sine.  Were the turn cut to fp32, their errors would be the dropped part times
    the derivative: 1 by regression on that.  With it they are the roundings of sine and cosine, at most 2^-22 each and
    unrelated to the dropped part (5e-8 on average): 400,000 of them bring the regression to 0 within
    2^-22 / 5e-8 / 632 = 0.008 as a standard deviation, and six of those are allowed."""
    from sparsepr_amd.kernels.axial_rope import axial_rope

    g = torch.Generator(device=dev).manual_seed(8)
    q = torch.zeros(1, 1, 50000, 8, device=dev)
    q[..., 0::2] = 1
    p = torch.rand(50000, 1, generator=g, device=dev, dtype=torch.float64) * 1000
    freqs = torch.rand(4, generator=g, device=dev, dtype=torch.float64) + 0.1
    y = _f64(axial_rope(q, None, p, freqs, torch.zeros(4, dtype=torch.int32, device=dev))[0])[0, 0]
    turn = _f64(p) * (_f64(freqs) / (2 * np.pi))
    part = turn - np.rint(turn)
    dropped = (part - part.astype(np.float32)) * 2 * np.pi
    c, s = np.cos(2 * np.pi * part), np.sin(2 * np.pi * part)
    error = np.concatenate([y[:, 0::2] - c, y[:, 1::2] - s])
    along = np.concatenate([s * dropped, -c * dropped])
    assert np.abs(error).max() <= 2.0**-22
    assert abs((error * along).sum() / (along * along).sum()) <= 0.05
