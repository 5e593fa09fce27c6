"""The lists by which a step's tokens are dealt out to their adapters, and what the C entry points of the 8-bit rows, their product and the
adapters refuse: no device is needed for either."""
import ctypes

import numpy as np
import pytest

from roost_b200.kernels import build, library


@pytest.mark.parametrize("seed", range(20))
def test_every_token_with_an_adapter_stands_in_one_tile(seed):
    rng = np.random.default_rng(seed)
    n = int(rng.integers(1, 50))
    counts = rng.integers(0, 200 if seed % 2 else 2, n).tolist()
    slots = rng.integers(-1, 6, n).tolist()
    of = np.repeat(slots, counts)
    rows, tiles, tile_rows = library.adapter_lists(counts, slots)
    assert rows.dtype == np.int32 and tiles.dtype == np.int32 and tiles.shape[1:] == (3,)
    seen = []
    for slot, first, end in tiles:
        assert 0 <= first < end <= rows.size and end - first <= tile_rows <= library.ADAPTER_TILE_ROWS
        assert (of[rows[first:end]] == slot).all()
        seen += rows[first:end].tolist()
    assert sorted(seen) == np.flatnonzero(of >= 0).tolist()


def test_no_tokens_no_tiles():
    for counts, slots in (([], []), ([0, 0], [1, 2]), ([3, 2], [-1, -1])):
        rows, tiles, _ = library.adapter_lists(counts, slots)
        assert rows.size == 0 and tiles.shape == (0, 3)


def test_lists_refuse():
    for counts, slots in (([1], [0, 1]), ([-1], [0])):
        with pytest.raises(library.KernelError):
            library.adapter_lists(counts, slots)


@pytest.fixture(scope="module")
def lib():
    try:
        path = build.library_path()
    except build.BuildError as e:
        pytest.skip(str(e))
    so = ctypes.CDLL(str(path))
    for name in ("roost_quantise_e4m3", "roost_silu_mul_e4m3", "roost_rms_norm_e4m3", "roost_gemm_e4m3", "roost_adapters_add"):
        getattr(so, name).argtypes = library._SIGNATURES[name]
    return so


FAKE = 1 << 20     # an address that no refused call reads


def test_entry_points_refuse_before_they_launch(lib):
    P = FAKE
    widths = (ctypes.c_int * 9)(*[8] * 9)
    quantise = dict(x=P, ldx=64, q=P, scale=P, rows=2, cols=64, dtype=1, stream=None)
    silu = dict(x=P, q=P, scale=P, tokens=2, inter=64, block=0, dtype=1, stream=None)
    norm = dict(x=P, residual=P, w=P, q=P, scale=P, kept=None, rows=None, n_out=2, hidden=64, eps=1e-6, dtype=1, residual_dtype=1, wdtype=0, stream=None)
    gemm = dict(q=P, qs=P, w=P, ws=P, out=P, m=2, n=64, k=64, ldq=64, ldw=64, ldo=64, out_dtype=1, stream=None)
    add = dict(y=P, ldy=64, x=P, ldx=64, a=P, b=P, h=P, scales=P, ranks=None, rows=P, tiles=P, n_tiles=1, tile_rows=64, listed=2, tokens=2, slots=1, n_parts=1, widths=widths, rank=8,
               inputs=64, dtype=1, y_dtype=1, stream=None)
    cases = [("roost_quantise_e4m3", quantise, [dict(rows=-1), dict(cols=0), dict(ldx=63), dict(cols=60000, ldx=60000), dict(x=None), dict(q=None), dict(dtype=2)]),
             ("roost_silu_mul_e4m3", silu, [dict(tokens=-1), dict(inter=0), dict(block=12), dict(block=128), dict(block=-8), dict(inter=60000), dict(scale=None), dict(dtype=7)]),
             ("roost_rms_norm_e4m3", norm, [dict(n_out=-1), dict(hidden=0), dict(eps=0.0), dict(wdtype=2), dict(dtype=0), dict(dtype=2), dict(hidden=60000), dict(w=None)]),
             ("roost_gemm_e4m3", gemm, [dict(m=-1), dict(n=0), dict(k=0), dict(ldq=63), dict(ldw=63), dict(ldo=63), dict(q=None), dict(ws=None), dict(out_dtype=2)]),
             ("roost_adapters_add", add, [dict(n_tiles=-1), dict(slots=0), dict(rank=0), dict(inputs=0), dict(n_parts=0), dict(n_parts=9), dict(rank=513), dict(n_parts=8, rank=65),
                                          dict(widths=None), dict(ldy=7), dict(ldx=63), dict(dtype=0), dict(dtype=3), dict(y_dtype=4), dict(y=None), dict(tiles=None), dict(h=None), dict(tile_rows=0), dict(tile_rows=65),
                                          dict(widths=(ctypes.c_int * 1)(0))])]
    for name, good, bad in cases:
        for change in bad:
            assert getattr(lib, name)(*{**good, **change}.values()) != 0, (name, change)
    # nothing to do: no launch, no error
    for name, good, empty in (("roost_quantise_e4m3", quantise, dict(rows=0, x=None)), ("roost_silu_mul_e4m3", silu, dict(tokens=0)), ("roost_rms_norm_e4m3", norm, dict(n_out=0)),
                              ("roost_gemm_e4m3", gemm, dict(m=0)), ("roost_adapters_add", add, dict(n_tiles=0)), ("roost_adapters_add", add, dict(listed=0))):
        assert getattr(lib, name)(*{**good, **empty}.values()) == 0, (name, empty)
