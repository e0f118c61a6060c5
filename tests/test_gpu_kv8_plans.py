"""The 8-bit cache's attention in every way that a call is cut: orders of the work, splits and joins, heads of 256 values."""
import numpy as np
import pytest
import torch

from oracle import kv8_ref as R
from pegainfer_amd import ops_blocks as B
from kv8_common import Cache, attention_bound, mass_bound
from test_gpu_kv8_ops import attend, rows_of

pytestmark = pytest.mark.gpu
TYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}


def values(c, e, side):
    """an entry's keys or values [slots, kv_heads, dim]"""
    n = c.starts[e] + c.rows[e]
    pages = np.array(c.ids[c.indptr[e]:c.indptr[e] + (n + 15) // 16], int)
    at = np.stack([R.offsets(c.dim, side, t) for t in range(16)])                       # [16, dim]
    x = R.number(c.codes[pages, side][:, :, at], c.fmt) * c.scales[pages, side][:, :, None, None].astype(np.float64)
    return x.transpose(0, 2, 1, 3).reshape(-1, c.kv, c.dim)[:n]


def reference(q, c, scale):
    """R.attention entry by entry and head by head, for caches whose pages are all there"""
    H = q.shape[1]
    group = H // c.kv
    out, spread, reach, mass = np.zeros(q.shape), np.zeros(q.shape), np.zeros(q.shape[:2]), []
    for e in range(c.B):
        a, n, length = c.row0[e], c.rows[e], c.starts[e] + c.rows[e]
        weight = np.zeros((c.kv, length if n else 0))
        for g in range(c.kv if n else 0):
            k, v = (values(c, e, side)[:, g] for side in (0, 1))               # no NaN: the caches here are not `dirty`
            seen = np.arange(length) <= c.starts[e] + np.arange(n)[:, None]
            for h in range(g * group, (g + 1) * group):
                x = q[a:a + n, h].astype(np.float64)
                z = np.where(seen, x @ k.T * scale, -np.inf)
                p = np.exp(z - z.max(-1, keepdims=True))
                p /= p.sum(-1, keepdims=True)
                out[a:a + n, h], spread[a:a + n, h] = p @ v, p @ np.abs(v)
                reach[a:a + n, h] = np.where(seen, np.abs(x) @ np.abs(k).T, 0).max(-1) * scale
                weight[g] += p.sum(0)
        mass.append(weight)
    return out, mass, spread, reach


def check(c, heads, dtype, hints, weigh):
    """outputs and weights against the reference, every row behind and every slot without a token as it was"""
    d, n, scale = c.device(), c.row0[-1], c.dim ** -0.5
    q, qd = rows_of(np.random.RandomState(1), n + 2, heads, c.dim, dtype)
    out = torch.full((n + 2, heads, c.dim), 7.0, dtype=dtype, device="cuda")
    B.kv8_attention(qd, d.codes, d.scales, d.row0, d.starts, d.indptr, d.ids, scale, max_rows=hints[0], max_len=hints[1], out=out,
                    **(dict(mass=d.mass, mass_keep=0.5) if weigh else {}))
    assert (out[n:] == 7).all()
    want, mass, spread, reach = reference(q[:n], c, scale)
    length = max(s + r for s, r in zip(c.starts, c.rows))
    err = np.abs(out[:n].double().cpu().numpy() - want)
    bound = attention_bound(spread, reach, want, c.dim, length, dtype)
    assert np.isfinite(err).all() and (err <= bound).all(), ((err / bound).max(), np.argwhere(err > bound)[:5])
    end, full, most = d.mass.cpu().numpy().astype(np.float64), c.mass.astype(np.float64), np.zeros(c.mass.shape)
    for e in range(c.B if weigh else 0):
        for s in range(mass[e].shape[1]):
            p = c.ids[c.indptr[e] + s // 16]
            full[p, :, s % 16] = 0.5 * full[p, :, s % 16] + mass[e][:, s]
            most[p, :, s % 16] = mass_bound(mass[e][:, s], reach.max(), c.dim, length, c.rows[e] * heads // c.kv) + 2.0 ** -23 * np.abs(full[p, :, s % 16])
    off = np.abs(end - full)
    assert np.isfinite(off).all() and (off <= most).all(), np.argwhere(off > most)[:5]


# More tiles of rows than a round holds (256 compute units / (kv heads * entries)): entries change places from round to round, and where two rounds are all the second
# begins with the shortest.  Entries of fewer tiles than the hint's, hints under and over the rows there are.
@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
@pytest.mark.parametrize("dtype,entries,kv,group,dim,most,hints", [
    ("bf16", 16, 8, 2, 64, 150, (150, 130)),       # prompts, 3 tiles of 2 a round: two rounds
    ("bf16", 16, 4, 4, 128, 150, None),            # 5 tiles of 4
    ("bf16", 16, 8, 1, 256, 290, (290, 140)),      # 3 of 2
    ("bf16", 24, 8, 2, 64, 170, (170, 70, 300)),   # 3 of 1: more than two rounds
    ("bf16", 40, 8, 1, 64, 100, (100, 40)),        # two row tiles, 4 of 1 (2 of 1: two rounds)
    ("bf16", 16, 8, 1, 256, 100, (100, 70)),       # 4 and 3 of 2
    ("fp32", 16, 8, 1, 64, 120, (120, 70, 17)),    # 4, 3 and 1 of 2
    ("fp32", 16, 4, 1, 256, 110, (110, 80)),       # one row tile, 7 and 5 of 4
])
def test_work_in_every_order(fmt, dtype, entries, kv, group, dim, most, hints):
    rng = np.random.RandomState(entries + dim)
    rows = [most] + [int(x) for x in rng.randint(17, most, entries - 2)] + [0]
    c = Cache([int(x) for x in rng.randint(0, 60, entries)], rows, kv, dim, fmt, seed=dim, dirty=False)
    for hint in hints or (most,):
        check(c, kv * group, TYPES[dtype], (hint, most + 60), True)


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
def test_split_keys_and_entries_that_change_places(dtype):
    """3 tiles of rows, 2 a round, the keys of each in two splits"""
    rng = np.random.RandomState(5)
    rows = [90] + [int(x) for x in rng.randint(17, 90, 15)]
    c = Cache([1010] + [int(x) for x in rng.randint(0, 400, 15)], rows, 8, 64, "int8", seed=6, dirty=False)
    for weigh in (False, True):
        check(c, 8, TYPES[dtype], (90, 1100), weigh)


# ---- heads of 256 values ----
@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
@pytest.mark.parametrize("weigh", [False, True])
def test_two_row_tiles_of_256_values(fmt, weigh):
    """20 to 100 rows a kv head, over few tokens, over more than a run of 64 blocks, split"""
    for c in (Cache([0, 33, 10], [20, 25, 9], 2, 256, fmt, seed=1, dirty=True), Cache([2300], [8], 1, 256, fmt, seed=2), Cache([1300, 5], [23, 6], 1, 256, fmt, seed=3, layers=2)):
        attend(c, 4 * c.kv, torch.bfloat16, weigh=weigh)


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("weigh", [False, True])
def test_steps_of_256_values_over_long_caches(fmt, dtype, weigh):
    """ten and more splits of few rows, seven of 16 entries, runs of more than 64 blocks with nothing cut"""
    c = Cache([3000, 17, 1499], [1, 1, 2], 1, 256, fmt, seed=4)
    attend(c, 4, TYPES[dtype], weigh=weigh)
    attend(c, 4, TYPES[dtype], weigh=weigh, hints=(2, 1024))
    attend(Cache([1700] + [100] * 15, [1] * 16, 2, 256, fmt, seed=5), 4, TYPES[dtype], weigh=weigh, hints=(1, 1800))


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
@pytest.mark.parametrize("weigh", [False, True])
def test_prompts_of_256_values_over_long_caches(fmt, weigh):
    """both sets of codes across runs of 64 blocks and splits, whole (one split of 70 blocks) and cut in four"""
    attend(Cache([2300], [40], 1, 256, fmt, seed=6), 4, torch.bfloat16, weigh=weigh)
    attend(Cache([1100, 0], [35, 33], 1, 256, fmt, seed=7), 4, torch.bfloat16, weigh=weigh, hints=(35, 1000))


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
@pytest.mark.parametrize("dim", [128, 256])
def test_fp32_prompts_whose_weights_are_cut_in_slices(fmt, dim):
    attend(Cache([100, 7], [60, 45], 1, dim, fmt, seed=8), 4, torch.float32, weigh=True, keep=0.5)
    attend(Cache([1200], [70], 1, dim, fmt, seed=9), 4, torch.float32, weigh=True)


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
def test_a_workgroup_a_row_joins_many_splits(dtype):
    """of 256 values; the join looks at sixteen splits at a time, two to eight waves apart"""
    for kv, rows in ((16, 1), (2, 3)):
        c = Cache([2600 + 10 * kv], [rows], kv, 256, "int8", seed=kv, dirty=False)
        attend(c, 4 * kv, TYPES[dtype], weigh=False)


@pytest.mark.parametrize("weigh", [False, True])
def test_a_wave_a_row_joins_more_than_eight_splits(weigh):
    check(Cache([4700], [32], 1, 256, "e4m3", seed=10, dirty=False), 64, torch.bfloat16, (32, 4740), weigh)
