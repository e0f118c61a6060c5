"""CPU: the ends of the 8-bit cache's ranges in the float64 restatement, and the refusals at them."""
import ctypes
import os
import subprocess
import sys

import numpy as np
import pytest

from oracle import kv8_ref as R
from pegainfer_amd import ffi, ops_blocks as B

LARGEST = {"e4m3": 240 * 2.0 ** 120, "int8": 127 * 2.0 ** 121}      # code * 2^e: the next one up is 2^128


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
@pytest.mark.parametrize("x", [3.4028234e38, 3.3895314e38, 3.3e38, 3.2e38, 3.1e38, 2.9e38, np.inf])
def test_what_is_kept_of_a_finite_value_is_finite(fmt, x):
    """a value next to fp32's largest is not rounded to 2^128: e4m3 within its half step (2^-4 of the value), int8 within a 127th of the block's largest, as elsewhere"""
    k = np.full((3, 1, 64), x, np.float32)
    k[1], k[2] = -k[1], 2.9e38
    codes, scales = np.zeros((1, 2, 1, 1024), np.uint8), np.zeros((1, 2, 1), np.float32)
    R.append(k, k, codes, scales, fmt, [0, 3], [0], ([0, 1], [0]))
    for got in R.read(codes, scales, fmt, 64, [0, 3], [0], ([0, 1], [0])):
        assert np.isfinite(got.astype(np.float32)).all() and np.abs(got).max() <= LARGEST[fmt]
        if np.isfinite(x):
            assert (np.abs(got - k) <= (2.0 ** -4 * np.abs(k) if fmt == "e4m3" else np.abs(k).max() / 127)).all()


def test_rows_into_a_weighed_cache_need_its_weights(built_libs):
    L, at = ffi.lib(), 1 << 20      # never followed: every call is refused before a launch
    c = B.Kv8Cache(codes=at, scales=at, code_page_stride=2 * 2 * 16 * 64, scale_page_stride=4, format=0, n_pages=3, kv_heads=2, dim=64, page_indptr=at, page_ids=at,
                   n_page_ids=3, n_entries=1)
    for mass, apart, k in [(None, 32, at), (at, 31, at), (at, 32, None), (at, 32, at + 8)]:
        assert L.pegainfer_kv8_append_weighed(ctypes.addressof(c), mass, apart, k, at, 128, 128, at, at, 4, 4, 0, None) == 1
    assert L.pegainfer_kv8_append_weighed(None, at, 32, at, at, 128, 128, at, at, 4, 4, 0, None) == 1
    assert L.pegainfer_kv8_append_weighed(ctypes.addressof(c), at, 32, None, None, 0, 0, None, None, 0, 4, 0, None) == 0


def test_a_hint_of_no_rows_is_no_call_without_rows(built_libs):
    """max_rows is about the most rows of an entry: whatever it says, the call's rows are looked at, and refused where they are wrong"""
    L, at, ref = ffi.lib(), 1 << 20, ctypes.addressof
    c = B.Kv8Cache(codes=at, scales=at, code_page_stride=2 * 2 * 16 * 64, scale_page_stride=4, format=0, n_pages=3, kv_heads=2, dim=64, page_indptr=at, page_ids=at,
                   n_page_ids=3, n_entries=1)
    assert L.pegainfer_kv8_append(ref(c), None, at, 128, 128, at, at, 4, 0, 0, None) == 1
    assert L.pegainfer_kv8_read(ref(c), at, at, None, at, 4, 0, 0, None) == 1
    d = B.Kv8AttnDesc(q=None, q_row_stride=256, out=at, out_row_stride=256, row0=at, starts=at, n_rows=4, max_rows=0, max_len=9, heads=4, scale=1.0, dtype=0)
    assert L.pegainfer_kv8_attention(ref(c), ref(d), None) == 1
    for max_len in (9, 5000):
        for mass in (0, 1):
            assert L.pegainfer_kv8_attention_workspace(ref(c), 4, 0, max_len, 4, 0, mass) == L.pegainfer_kv8_attention_workspace(ref(c), 4, 1, max_len, 4, 0, mass)


def test_the_wrappers_import_beside_a_torch_without_a_gpu_build():
    """what such a torch lacks is looked up by the calls alone, which refuse first"""
    code = ("import torch\n"
            "for name in ('_cuda_getDevice', '_cuda_getCurrentRawStream'):\n"
            "    if hasattr(torch._C, name): delattr(torch._C, name)\n"
            "from pegainfer_amd import ops, ops_blocks as B\n"
            "i = torch.zeros(2, dtype=torch.int32)\n"
            "try: B.kv8_read(torch.zeros(3, 2, 2, 1024, dtype=torch.int8), torch.zeros(3, 2, 2), i, i[:1], i, i, 1)\n"
            "except ValueError as e: print('refused', e)\n")
    p = subprocess.run([sys.executable, "-c", code], cwd=os.path.dirname(os.path.dirname(os.path.abspath(__file__))), capture_output=True, text=True, timeout=120)
    assert p.returncode == 0 and "refused kv8" in p.stdout, p.stderr
