"""The 4-bit K/V cache without a GPU: the encoder's definition, and the refusals that the host gives."""

import numpy as np
import pytest
import torch

from tests import _kv4_model as model


def test_encoder_picks_the_nearest_value_of_the_best_scale():
    rng = np.random.default_rng(1)
    x = rng.standard_normal((200, 64)) * np.exp(4 * rng.standard_normal((200, 1)))
    codes, scales = model.encode(x)
    y = model.decode(codes, scales)
    s = np.ldexp(1.0, scales.astype(int) - 127).repeat(32, -1).reshape(x.shape)
    top = np.abs(x).reshape(200, 2, 32).max(-1).repeat(32, -1).reshape(x.shape)
    assert (top < 7 * s).all() and (top >= 3.5 * s).all()
    # half a step of the grid: 0.25 below 2, 0.5 below 4, 1 above, in units of the scale
    a = np.abs(x) / s
    assert (np.abs(x - y) <= s * np.where(a < 2, 0.25, np.where(a < 4, 0.5, 1.0))).all()
    # what is stored is stored again as it is, in bf16 too
    assert np.array_equal(model.decode(*model.encode(y)), y)
    assert np.array_equal(torch.from_numpy(y).to(torch.bfloat16).double().numpy(), y)


def test_the_page_lists_agree_with_themselves():
    m = model.Pages(8, 4, 4, 32)
    assert m.reserve([0, 1], [70, 32]) == (0, [0, 0])
    assert m.table[0, :3].tolist() == [0, 1, 2] and m.table[1, 0] == 3
    assert m.fork([0], [2], True) == (0, [(2, 4)])
    assert m.refs.tolist() == [2, 2, 1, 1, 1, 0, 0, 0]
    assert m.free([0]) == 0 and m.lengths[0] == 0 and m.refs.tolist() == [1, 1, 0, 1, 1, 0, 0, 0]
    assert m.free([2], [0], [1]) == 0 and m.lengths[2] == 38 and m.table[2].tolist() == [1, 4, -1, -1]
    assert m.compact() == (3, [(3, 0), (4, 2)]) and m.table[2, :2].tolist() == [1, 2] and m.table[1, 0] == 0


def _lib():
    from sparsepr_amd import _lib

    return _lib.load()


def test_entry_points_refuse_bad_arguments_before_any_launch():
    lib = _lib()

    def attention(**kw):
        a = dict(dtype=0, batch=1, heads=4, kv_heads=2, rows=1, d=128, num_pages=4, page_size=64, sequences=1, wide=4,
                 scale=0.1, q=16, q_t=128, ws=None, longest=256)
        a.update(kw)
        st = lib.spr_kv4_attention(a["q"], 512, 128, a["q_t"], a["dtype"], a["batch"], a["heads"], a["kv_heads"],
                                   a["rows"], a["d"], 16, a["num_pages"], a["page_size"], 16, a["sequences"], a["wide"],
                                   16, None, None, 0, a["scale"], a["longest"], 16, None, a["ws"], 0, None)
        return st, lib.spr_last_error().decode()

    for kw, text in [
        (dict(dtype=2), "dtype code 2"), (dict(d=96), "head dim 96"), (dict(page_size=48), "page size 48"),
        (dict(page_size=512), "page size 512"), (dict(num_pages=0), "0 pages"), (dict(wide=2**24 + 1), "block table"),
        (dict(heads=3), "3 query heads on 2"), (dict(scale=0.0), "scale must be positive"),
        (dict(scale=float("inf")), "scale must be positive"), (dict(scale=float("nan")), "scale must be positive"), (dict(scale=2e38), "at most 1e38"), (dict(heads=70000, kv_heads=70000), "on 70000 kv heads"),
        (dict(q=8), "16-byte aligned"), (dict(q_t=100), "multiples of 8"), (dict(batch=70000), "batch 70000"),
        (dict(rows=2**20), "too many"), (dict(longest=-1), "max_length -1"),
    ]:
        st, said = attention(**kw)
        assert st == 1 and text in said, (kw, st, said)
    st, said = attention(wide=4096, longest=4096 * 64)  # keys in shares, and no workspace for them
    assert st == 3 and "workspace" in said
    assert attention(rows=0)[0] == 0 and attention(batch=0)[0] == 0

    rows = [16, 4, 2, 64, 128, 16, 1, 4, None, 16, None, 16, 16, 0, 1, 1, 256, 128, 128, 256, 128, 128, None]
    for at, bad, text in [(3, 16, "page size 16"), (4, 32, "head dim 32"), (13, 5, "dtype code 5"), (11, 24, "aligned"),
                          (18, 4, "multiples of 16 bytes"), (2, 0, "kv heads 0"), (14, -1, "batch -1")]:
        args = list(rows)
        args[at] = bad
        assert lib.spr_kv4_store(*args) == 1 and text in lib.spr_last_error().decode(), (at, bad)
    load = [16, 4, 2, 64, 128, 16, 1, 4, None, 16, 16, 16, 16, 0, 1, 1, None]
    for at, bad, text in [(3, 33, "page size 33"), (4, 256, "head dim 256"), (13, -1, "dtype code -1"), (11, 4, "aligned")]:
        args = list(load)
        args[at] = bad
        assert lib.spr_kv4_load(*args) == 1 and text in lib.spr_last_error().decode(), (at, bad)
    assert lib.spr_kv4_reserve(16, 16, 16, 16, None, 3, 2, 4, 64, 8, 16, None, 16, 1 << 20, None) == 1
    assert "3 counts for 2 sequences" in lib.spr_last_error().decode()
    assert lib.spr_kv4_reserve(16, 16, 16, 16, 16, 1, 2, 4, 64, 8, 16, None, None, 0, None) == 3
    assert lib.spr_kv4_free(16, 16, 16, 16, None, None, 5000, 2, 4, 64, 8, None, 16, 1 << 20, None) == 1
    assert "5000 sequences in one call" in lib.spr_last_error().decode()
    assert lib.spr_kv4_free(16, 16, 16, 16, None, None, 65, 2, 4, 64, 8, None, 16, 16, None) == 3
    assert lib.spr_kv4_fork(16, 24, 0, 1, 16, 16, 16, 16, 16, 1, 2, 4, 64, 8, 1, None, 16, 1 << 20, None) == 1
    assert lib.spr_kv4_fork(16, 32, 64, 2, 16, 16, 16, 16, 16, 1, 2, 4, 64, 8, 1, None, 16, 1 << 20, None) == 1
    assert lib.spr_kv4_compact(16, 32, 0, 1, 16, 16, 2, 4, 0, 16, 16, 1 << 20, None) == 1
    assert lib.spr_kv4_compact(16, 32, 0, 1, 16, 16, 2, 4, 8, 16, None, 0, None) == 3
    # nothing to do
    assert lib.spr_kv4_free(None, None, None, None, None, None, 0, 2, 4, 64, 8, None, None, 0, None) == 0


def test_python_refuses_cpu_tensors_and_bad_geometry():
    from sparsepr_amd.kernels import kv4
    from sparsepr_amd.kv4_cache import KV4Cache

    pages = torch.zeros((2, 1, kv4.kv4_page_bytes(32, 64)), dtype=torch.uint8)
    table, ints = torch.zeros((1, 2), dtype=torch.int32), torch.zeros(1, dtype=torch.int32)
    x = torch.zeros((1, 1, 1, 64), dtype=torch.bfloat16)
    for call in (
        lambda: kv4.kv4_store(pages, table, x, x, ints),
        lambda: kv4.kv4_load(pages, table, ints, ints, 1, 64),
        lambda: kv4.kv4_attention(x, pages, table, ints),
        lambda: kv4.kv4_reserve(table, ints, ints, 32, ints),
        lambda: kv4.kv4_free(table, ints, ints, 32, ints),
        lambda: kv4.kv4_fork(pages, table, ints, ints, 32, ints, ints),
        lambda: kv4.kv4_compact(pages, table, ints),
    ):
        with pytest.raises(RuntimeError, match="require GPU tensors"):
            call()
    assert kv4.kv4_page_bytes(64, 128) == 64 * 136 == _lib().spr_kv4_page_bytes(1, 64, 128)
    for args, text in [((64, 96), "head dim 96"), ((48, 64), "page size 48")]:
        with pytest.raises(RuntimeError, match=text):
            kv4.kv4_page_bytes(*args)
    for kw, text in [(dict(num_pages=0), "num_pages"), (dict(layers=0), "layers"), (dict(page_size=100), "page size"),
                     (dict(max_pages=2**26), "2\\^30 tokens")]:
        args = dict(num_pages=4, num_kv_heads=1, head_dim=64, max_sequences=1, device="cpu") | kw
        with pytest.raises(RuntimeError, match=text):
            KV4Cache(**args)


def test_calls_of_more_rows_than_a_launch_has_threads_are_refused():
    lib = _lib()
    for d, rows in ((128, 2**28), (64, 2**29)):
        assert lib.spr_kv4_store(16, 4, 1, 64, d, 16, 1, 4, None, 16, None, 16, 16, 0, 1, rows, 0, 0, 0, 0, 0, 0, None) == 1
        assert f"{rows} rows of 1 heads are too many" in lib.spr_last_error().decode()
        assert lib.spr_kv4_load(16, 4, 1, 64, d, 16, 1, 4, None, 16, 16, 16, 16, 0, 1, rows, None) == 1
        assert f"{rows} rows of 1 heads are too many" in lib.spr_last_error().decode()
    assert lib.spr_kv4_attention(16, 0, 0, 0, 0, 65535, 129, 129, 33, 64, 16, 4, 64, 16, 1, 4, 16, None, 16, 0, 0.1, 256,
                                 16, None, None, 0, None) == 1
    assert "33 rows of 129 heads in 65535 sequences are too many" in lib.spr_last_error().decode()


def test_more_pages_of_all_layers_than_an_index_counts_are_refused():
    lib = _lib()
    pages, layers = 2**28, 8
    space = lib.spr_kv4_pages_workspace(pages)
    assert lib.spr_kv4_fork(16, 16, 16 * pages, layers, 16, 16, 16, 16, 16, 1, 2, 4, 64, pages, 1, None, 16, space, None) == 1
    assert "8 layers" in lib.spr_last_error().decode()
    assert lib.spr_kv4_compact(16, 16, 16 * pages, layers, 16, 16, 2, 4, pages, 16, 16, space, None) == 1
    assert "8 layers" in lib.spr_last_error().decode()
