"""The 8-bit paged cache on the device at the ends of its ranges, and with what a pool of pages held before."""
import numpy as np
import pytest
import torch

from oracle import kv8_ref as R
from pegainfer_amd import ops_blocks as B
from kv8_common import Cache, TORCH, codes_of

pytestmark = pytest.mark.gpu
TYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}


def i32(*x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
def test_values_next_to_the_largest_stay_finite(fmt, dtype):
    """e4m3: within half a step, 2^-4 of the value (2^-10 of the scale's step at the least); int8: within a 127th of the block's largest"""
    top = torch.finfo(TYPES[dtype]).max
    c = Cache([0, 3], [16, 5], 1, 64, fmt, seed=3)
    d = c.device()
    x = torch.zeros(21, 1, 64)
    for i, v in enumerate([top, -top, 3.3e38, 3.2e38, 3.1e38, 2.9e38, 1.5e38, 1.0, 0.0]):
        x[:, 0, i] = v
    x[17:, 0, 10], x[2, 0, 11] = torch.inf, -torch.inf
    x = x.to(TYPES[dtype])
    codes, scales = c.codes.copy(), c.scales.copy()
    rows = x.float().numpy()
    R.append(rows, rows, codes, scales, fmt, c.row0, c.starts, c.tables)
    B.kv8_append(x.cuda(), x.cuda(), d.codes, d.scales, d.row0, d.starts, d.indptr, d.ids)
    assert np.array_equal(codes_of(d), codes) and np.array_equal(d.scales.cpu().numpy(), scales)
    for t in TYPES.values():
        for got in B.kv8_read(d.codes, d.scales, d.row0, d.starts, d.indptr, d.ids, 21, dtype=t):
            assert torch.isfinite(got).all()
            there = np.isfinite(rows)
            off = np.abs(got.double().cpu().numpy() - rows.astype(np.float64))[there]
            most = 2.0 ** -4 * np.abs(rows.astype(np.float64)) + 2.0 ** (120 - 10) if fmt == "e4m3" else np.full(rows.shape, float(top) / 127)
            assert (off <= most[there]).all()
    # a row that sees its own token alone gives its values
    for t in TYPES.values():
        out = B.kv8_attention(torch.zeros(1, 2, 64, dtype=t, device="cuda"), d.codes, d.scales, i32(0, 1, 1), d.starts * 0, d.indptr, d.ids, 1.0)
        want = B.kv8_read(d.codes, d.scales, i32(0, 1, 1), d.starts * 0, d.indptr, d.ids, 1, dtype=t)[1]
        assert torch.equal(out, want.expand(1, 2, 64))
