"""CPU: the float64 restatement of the 8-bit cache against torch's own conversions, and the refusals of the C entries and of the wrappers."""
import ctypes

import numpy as np
import pytest
import torch

from oracle import kv8_ref as R
from pegainfer_amd import ffi, ops_blocks as B


def test_e4m3_numbers_and_codes_are_torchs():
    every = torch.arange(256, dtype=torch.uint8)
    want = every.view(torch.float8_e4m3fn).float().numpy()
    got = R.number(every.numpy(), "e4m3")
    assert np.array_equal(np.isnan(got), np.isnan(want)) and np.array_equal(np.nan_to_num(got), np.nan_to_num(want))
    x = torch.cat([torch.linspace(-448, 448, 20001), torch.randn(20000) * 2.0 ** -7, torch.tensor([0.0, -0.0, 464.0 - 16])])
    assert np.array_equal(R.code(x.numpy(), "e4m3"), x.to(torch.float8_e4m3fn).view(torch.uint8).numpy())


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
def test_the_exponent_is_the_least_that_reaches(fmt):
    top = R.TOP[fmt]
    for a in [0.0, 1e-40, 1.0, top, np.nextafter(top, 1e9), top / 2, top * 2.0 ** 100, 3.3e38, 1e-3]:
        e = R.exponent(a, fmt)
        assert top * 2.0 ** e >= a and (e == R.LEAST or top * 2.0 ** (e - 1) < a)


def test_repeated_rescaling_of_int8_stays_within_one_step():
    """half a step at every doubling of the scale: 1/2 + 1/4 + ... of the last step"""
    x = np.random.RandomState(0).randn(4000) * 40
    y, scale = R.number(R.code(x, "int8"), "int8"), 1.0
    for _ in range(5):
        y, scale = R.number(R.code(y / 2, "int8"), "int8"), scale * 2
    assert np.abs(y * scale - x).max() < scale


@pytest.mark.parametrize("dim", [64, 128, 256])
def test_a_blocks_layout_is_a_permutation(dim):
    for side in (0, 1):
        at = np.concatenate([R.offsets(dim, side, t) for t in range(16)])
        assert np.array_equal(np.sort(at), np.arange(16 * dim))


def _cache(**kw):
    at = 1 << 20      # never followed: every call below is refused before a launch
    c = dict(codes=at, scales=at, code_page_stride=2 * 2 * 16 * 64, scale_page_stride=4, format=0, n_pages=3, kv_heads=2, dim=64, page_indptr=at, page_ids=at,
             n_page_ids=3, n_entries=1)
    return B.Kv8Cache(**{**c, **kw})


def test_c_entries_refuse(built_libs):
    L, at, bad = ffi.lib(), 1 << 20, 1
    ref = ctypes.addressof
    wrong = [dict(codes=None), dict(codes=at + 8), dict(scales=None), dict(code_page_stride=2 * 2 * 16 * 64 - 16), dict(code_page_stride=2 * 2 * 16 * 64 + 8),
             dict(scale_page_stride=3), dict(format=2), dict(dim=96), dict(kv_heads=0), dict(n_pages=0), dict(n_entries=65536), dict(n_entries=-1), dict(page_indptr=None), dict(page_ids=None)]
    for w in wrong:
        c = _cache(**w)
        assert L.pegainfer_kv8_append(ref(c), at, at, 128, 128, at, at, 4, 4, 0, None) == bad, w
        assert L.pegainfer_kv8_read(ref(c), at, at, at, at, 4, 4, 0, None) == bad, w
        assert L.pegainfer_kv8_evict(ref(c), at, 32, at, at, at, 3, 8, 0, 0, 100, at, None) == bad, w
    c = _cache()
    for k, v, ks, vs, n, m, dt in [(None, at, 128, 128, 4, 4, 0), (at, at + 2, 128, 128, 4, 4, 0), (at, at, 120, 128, 4, 4, 0), (at, at, 128, 132, 4, 4, 0), (at, at, 128, 128, -1, 4, 0),
                                   (at, at, 128, 128, 4, -1, 0), (at, at, 128, 128, 4, 4, 2), (at, at, 128, 130, 4, 4, 1)]:
        assert L.pegainfer_kv8_append(ref(c), k, v, ks, vs, at, at, n, m, dt, None) == bad
    for budget, first, last in [(0, 0, 0), (8, -1, 0), (8, 0, -1), (8, 5, 4), (8, 2 ** 31 - 1, 1)]:
        assert L.pegainfer_kv8_evict(ref(c), at, 32, at, at, at, 3, budget, first, last, 100, at, None) == bad
    assert L.pegainfer_kv8_evict(ref(c), at, 31, at, at, at, 3, 8, 0, 0, 100, at, None) == bad
    good = dict(q=at, q_row_stride=256, out=at, out_row_stride=256, row0=at, starts=at, n_rows=4, max_rows=4, max_len=9, heads=4, scale=1.0, dtype=0)
    for w in [dict(q=None), dict(q=at + 4), dict(q_row_stride=255), dict(out_row_stride=260), dict(heads=3), dict(heads=0), dict(scale=-1.0), dict(scale=float('nan')), dict(n_rows=-1), dict(max_len=-1), dict(dtype=3), dict(row0=None),
              dict(mass_out=at, mass_out_page_stride=31, workspace=at), dict(mass_out=at, mass_out_page_stride=32, mass_keep=1.0, workspace=at),
              dict(mass_out=at, mass_out_page_stride=32), dict(n_rows=2 ** 31 - 1, max_rows=1)]:
        d = B.Kv8AttnDesc(**{**good, **w})
        assert L.pegainfer_kv8_attention(ref(c), ref(d), None) == bad, w
    assert L.pegainfer_kv8_attention(None, ref(B.Kv8AttnDesc(**good)), None) == bad and L.pegainfer_kv8_attention(ref(c), None, None) == bad
    # nothing to do: no launch, no pointer looked at
    assert L.pegainfer_kv8_append(ref(c), None, None, 0, 0, None, None, 0, 0, 0, None) == 0
    assert L.pegainfer_kv8_attention(ref(c), ref(B.Kv8AttnDesc(dtype=1, heads=4)), None) == 0


def test_wrappers_refuse_what_is_not_on_the_device():
    i = torch.zeros(2, dtype=torch.int32)
    for dt in (torch.uint8, torch.int8):
        with pytest.raises(ValueError, match="kv8"):
            B.kv8_append(torch.zeros(1, 2, 64), torch.zeros(1, 2, 64), torch.zeros(3, 2, 2, 1024, dtype=dt), torch.zeros(3, 2, 2), i, i[:1], i, i)


def test_what_is_not_cut_needs_no_workspace(built_libs):
    """the wrapper asks for the size of a workspace only beyond KV8_WHOLE tokens"""
    L, ref = ffi.lib(), ctypes.addressof
    text = open(ffi.INCLUDE + "/pegainfer_kernels_blocks.h").read()
    assert "PEGAINFER_KV8_WHOLE = %d " % B.KV8_WHOLE in text
    for kv, dim in [(1, 64), (8, 128), (2, 256)]:
        for entries in (1, 3, 400):
            c = _cache(kv_heads=kv, dim=dim, code_page_stride=2 * kv * 16 * dim, scale_page_stride=2 * kv, n_entries=entries, n_page_ids=5)
            for rows in (1, 5, 40, 1000, 100000):
                for dtype in (0, 1):
                    assert L.pegainfer_kv8_attention_workspace(ref(c), rows, rows, B.KV8_WHOLE, 4 * kv, dtype, 0) == 0
                    assert L.pegainfer_kv8_attention_workspace(ref(c), rows, rows, B.KV8_WHOLE, 4 * kv, dtype, 1) >= rows * 4 * kv
    # a long cache is cut where that fills the chip: one entry's is, that of 400 entries of 2 heads is not
    assert L.pegainfer_kv8_attention_workspace(ref(c), 1, 1, 10 ** 6, 2, 0, 0) == 0
    assert L.pegainfer_kv8_attention_workspace(ref(_cache()), 1, 1, 10 ** 6, 2, 0, 0) > 0
