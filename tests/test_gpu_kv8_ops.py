"""The 8-bit paged cache on the device against its float64 restatement: movers bit for bit, attention and weights within derived bounds."""
import numpy as np
import pytest
import torch

from oracle import kv8_ref as R
from pegainfer_amd import ops_blocks as B
from kv8_common import Cache, TORCH, attention_bound, codes_of, mass_bound

pytestmark = pytest.mark.gpu
TYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}


def rows_of(rng, n, heads, dim, dtype, size=1.0):
    """values that dtype holds, as numpy float32 and on the device, inside a wider row (a view of a projection)"""
    x = torch.from_numpy((rng.randn(n, heads, dim) * size).astype(np.float32)).to(dtype)
    wide = torch.zeros(n, heads * dim + 32, dtype=dtype, device="cuda")
    view = wide[:, 16:16 + heads * dim].unflatten(1, (heads, dim))
    view.copy_(x)
    return x.float().numpy(), view


def same(d, c, codes, scales):
    got = codes_of(d)
    bad = np.argwhere(got != codes)
    assert len(bad) == 0, (len(bad), bad[:4], got[tuple(bad[0])], codes[tuple(bad[0])])
    assert np.array_equal(d.scales.cpu().numpy(), scales)


# ---- rows in and out ----
@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("kv,dim", [(1, 64), (3, 128), (2, 256)])
def test_append_and_read(fmt, dtype, kv, dim):
    c = Cache([0, 5, 16, 31, 40, 7, 0], [1, 1, 33, 1, 0, 9, 17], kv, dim, fmt, seed=dim + kv, layers=2)
    d = c.device()
    k, kd = rows_of(c.rng, c.row0[-1] + 2, kv, dim, TYPES[dtype], 3.0)
    v, vd = rows_of(c.rng, c.row0[-1] + 2, kv, dim, TYPES[dtype], 0.01)
    codes, scales = c.codes.copy(), c.scales.copy()
    R.append(k, v, codes, scales, fmt, c.row0, c.starts, c.tables)
    B.kv8_append(kd, vd, d.codes, d.scales, d.row0, d.starts, d.indptr, d.ids)
    same(d, c, codes, scales)
    assert (d.pool[:, 0] == 0).all()                                    # the other layer's part
    for hint in (None, 1, 33):
        out = tuple(torch.full((c.row0[-1] + 2, kv, dim), 7.0, dtype=TYPES[dtype], device="cuda") for _ in range(2))
        got = B.kv8_read(d.codes, d.scales, d.row0, d.starts, d.indptr, d.ids, c.row0[-1] + 2, dtype=TYPES[dtype], max_rows=hint, out=out)
        for x, y in zip(got, R.read(codes, scales, fmt, dim, c.row0, c.starts, c.tables)):
            assert np.array_equal(x[:-2].double().cpu().numpy(), y) and (x[-2:] == 7).all()


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
def test_append_values_at_the_ends_of_their_range(fmt):
    c = Cache([0, 3], [16, 5], 2, 64, fmt, seed=3)
    d = c.device()
    k = np.zeros((21, 2, 64), np.float32)
    k[0, 0, :6] = [np.inf, -np.inf, np.nan, 448, -448.5, 1e-3]
    k[1, 1, :3] = [np.nan, np.inf, 0.0]                                   # no finite value but 0
    k[16, 0, :4] = [3.3e38, -3.3e38, 1e38, 1e-38]
    k[17, 1, :4] = [1e-40, -1e-40, 2.0 ** -126, 0.0]
    v = -k[::-1].copy()
    codes, scales = c.codes.copy(), c.scales.copy()
    R.append(k, v, codes, scales, fmt, c.row0, c.starts, c.tables)
    B.kv8_append(torch.from_numpy(k).cuda(), torch.from_numpy(v).cuda(), d.codes, d.scales, d.row0, d.starts, d.indptr, d.ids)
    same(d, c, codes, scales)


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
def test_append_token_by_token(fmt):
    """a block whose scale grows with every token, then shrinks in the next block"""
    c = Cache([0], [40], 2, 128, fmt, seed=5)
    d = c.device()
    codes, scales = c.codes.copy(), c.scales.copy()
    for t in range(40):
        k, kd = rows_of(c.rng, 1, 2, 128, torch.bfloat16, 1.7 ** (t if t < 16 else -t))
        v, vd = rows_of(c.rng, 1, 2, 128, torch.bfloat16, 1.3 ** t)
        R.append(k, v, codes, scales, fmt, [0, 1], [t], c.tables)
        B.kv8_append(kd, vd, d.codes, d.scales, torch.tensor([0, 1], dtype=torch.int32, device="cuda"), torch.tensor([t], dtype=torch.int32, device="cuda"), d.indptr, d.ids)
        same(d, c, codes, scales)


# ---- attention ----
def attend(c, heads, dtype, weigh=False, keep=1.0, separate=False, hints=(None, None), q_size=1.0, seed=0, d=None):
    d = d or c.device()
    n = c.row0[-1]
    q, qd = rows_of(np.random.RandomState(seed), n + 2, heads, c.dim, dtype, q_size)
    out = torch.full((n + 2, heads, c.dim), 7.0, dtype=dtype, device="cuda")
    scale = c.dim ** -0.5
    kw = {}
    if weigh:
        kw = dict(mass=d.mass, mass_keep=keep)
        if separate:
            kw["mass_out"] = torch.full_like(d.mass, 5.0)
    got = B.kv8_attention(qd, d.codes, d.scales, d.row0, d.starts, d.indptr, d.ids, scale, max_rows=hints[0], max_len=hints[1], out=out, **kw)
    assert (got[n:] == 7).all()
    want, mass, spread, reach = R.attention(q[:n], c.codes, c.scales, c.fmt, c.row0, c.starts, c.tables, scale)
    length = max([s + r for s, r in zip(c.starts, c.rows)] + [1])
    err = np.abs(got[:n].double().cpu().numpy() - want)
    bound = attention_bound(spread, reach, want, c.dim, length, dtype)
    assert np.isfinite(err).all() and (err <= bound).all(), (err.max(), (err / bound).max(), np.argwhere(err > bound)[:5])
    if weigh:
        end = kw.get("mass_out", d.mass).cpu().numpy().astype(np.float64)
        full = np.full_like(c.mass, 5.0, dtype=np.float64) if separate else c.mass.astype(np.float64)
        most, rest = np.zeros_like(full), np.ones(full.shape, bool)
        for e in range(c.B):
            for s in range(mass[e].shape[1]):
                p = R.page_of(c.tables, e, s // 16, c.pages)
                if p < 0:
                    continue
                rest[p, :, s % 16] = False
                full[p, :, s % 16] = (0 if keep == 0 else keep * c.mass[p, :, s % 16].astype(np.float64)) + mass[e][:, s]
                most[p, :, s % 16] = mass_bound(mass[e][:, s], reach.max(), c.dim, length, c.rows[e] * heads // c.kv) + 2.0 ** -23 * np.abs(full[p, :, s % 16])
        assert np.array_equal(end[rest], full[rest], equal_nan=True)     # slots without a token stay as they were
        off = np.where(rest, 0.0, np.abs(end - full))
        assert np.isfinite(off).all() and (off <= most).all(), ((off / np.maximum(most, 1e-300)).max(), np.argwhere(off > most)[:5])
    return d, got


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("kv,group,dim", [(1, 1, 64), (2, 3, 64), (2, 4, 128), (1, 17, 128), (2, 4, 256)])
def test_attention_of_ragged_batches(fmt, dtype, kv, group, dim):
    c = Cache([0, 0, 15, 16, 17, 100, 333, 0, 64], [1, 2, 1, 1, 1, 1, 1, 0, 5], kv, dim, fmt, seed=group)
    attend(c, kv * group, TYPES[dtype])
    c = Cache([0, 33, 0, 250], [70, 18, 16, 21], kv, dim, fmt, seed=group + 1, layers=2)
    for hints in [(None, None), (1, 1), (70, 280)]:
        attend(c, kv * group, TYPES[dtype], hints=hints)


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
def test_attention_over_a_long_cache_and_of_many_rows(fmt, dtype):
    attend(Cache([3000, 17, 1499], [1, 1, 2], 1, 128, fmt, seed=1), 4, TYPES[dtype])
    attend(Cache([100, 700], [150, 40], 1, 64, fmt, seed=2), 2, TYPES[dtype])


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
def test_attention_with_sharp_and_flat_scores(dtype):
    for size in (0.0, 30.0):
        attend(Cache([200, 5], [3, 1], 2, 128, "int8", seed=4), 4, TYPES[dtype], q_size=size)


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("kv,group,dim", [(1, 1, 64), (2, 3, 128), (2, 4, 256), (1, 17, 64)])
def test_weights_of_cached_tokens(fmt, dtype, kv, group, dim):
    steps = Cache([0, 15, 16, 100, 333, 0], [1, 1, 1, 1, 1, 0], kv, dim, fmt, seed=group)
    prompts = Cache([0, 33, 0, 250], [70, 18, 16, 21], kv, dim, fmt, seed=group + 1, layers=2)
    for c in (steps, prompts):
        attend(c, kv * group, TYPES[dtype], weigh=True)
        attend(c, kv * group, TYPES[dtype], weigh=True, keep=0.5, separate=True, hints=(1, 1))
    c.mass[:] = np.nan
    attend(c, kv * group, TYPES[dtype], weigh=True, keep=0.0)


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("most", [1, 512, 513, 1024, 1025, 5000])
def test_weights_whatever_the_hints(dtype, most):
    """a step's weights by the attention itself, by a launch of its own, and beside the join of split keys; entries of more rows and tokens than was said"""
    steps = Cache([511, 512, 20, 1300, 0], [1, 1, 1, 1, 1], 2, 64, "e4m3", seed=most)
    mixed = Cache([600, 3, 0, 40], [1, 20, 0, 2], 1, 128, "int8", seed=most)
    for c, group in ((steps, 4), (mixed, 3)):
        attend(c, c.kv * group, TYPES[dtype], weigh=True, keep=0.5, hints=(1, most))


def test_weights_of_many_rows():
    attend(Cache([0, 300], [200, 90], 1, 64, "e4m3", seed=9), 4, torch.bfloat16, weigh=True)


def test_runs_repeat_bit_for_bit():
    c = Cache([900, 40, 0], [1, 33, 100], 2, 128, "e4m3", seed=6)
    d, a = attend(c, 8, torch.bfloat16, weigh=True, keep=0.0)
    first = d.mass.clone()
    for _ in range(3):
        _, b = attend(c, 8, torch.bfloat16, weigh=True, keep=0.0, d=d)
        assert torch.equal(a, b) and torch.equal(d.mass, first)


@pytest.mark.parametrize("rows", [1, 20, 80])
def test_a_row_that_is_not_a_number_spoils_itself_alone(rows):
    c = Cache([50], [rows], 1, 128, "e4m3", seed=30)
    d = c.device()
    q = torch.randn(rows, 4, 128, device="cuda").bfloat16()
    want = B.kv8_attention(q, d.codes, d.scales, d.row0, d.starts, d.indptr, d.ids, 0.1)
    q[0, 1, 5], q[rows - 1, 2, 7] = float("nan"), float("inf")
    got = B.kv8_attention(q, d.codes, d.scales, d.row0, d.starts, d.indptr, d.ids, 0.1)
    spoiled = torch.zeros(rows, 4, dtype=torch.bool)
    spoiled[0, 1] = spoiled[rows - 1, 2] = True
    assert torch.equal(got[~spoiled], want[~spoiled]) and torch.isnan(got[0, 1]).all()


# A key that comes late and takes nearly all of a row gives its values: its own weight may not be rounded, so that what is left is the output's rounding, 2^-8 of it,
# the others' weights, 2^-8 each of their small share, and the fp32 terms: scores below 48 off by (dim + 4) 2^-24 each and sums over 1024 tokens.
@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
@pytest.mark.parametrize("rows", [1, 16, 96])
def test_a_late_key_with_nearly_all_of_a_row(fmt, rows):
    n, dim, heads = 1024, 64, 4
    rng = np.random.RandomState(31)
    k, v = torch.zeros(n, 1, dim), torch.from_numpy(rng.randn(n, 1, dim).astype(np.float32))
    k[:, 0, 1] = -1.0                                                    # far below, but for one token in 32 of the first 256, at zero, ...
    k[0:256:32, 0, 1] = 0.0
    late = 600                                                           # ... and one above them, behind every wave's first tokens
    k[late, 0, 0], k[late, 0, 1] = 1.0, 0.0
    c = Cache([0], [n], 1, dim, fmt, seed=31)
    d = c.device()
    codes, scales = c.codes.copy(), c.scales.copy()
    R.append(k.numpy(), v.numpy(), codes, scales, fmt, c.row0, c.starts, c.tables)
    B.kv8_append(k.cuda(), v.cuda(), d.codes, d.scales, d.row0, d.starts, d.indptr, d.ids)
    same(d, c, codes, scales)
    kk, vv = (x[:, 0] for x in R.read(codes, scales, fmt, dim, c.row0, c.starts, c.tables))
    q = torch.from_numpy(rng.randn(rows, heads, dim).astype(np.float32))
    q[..., 0] = torch.linspace(3.6, 5.4, rows * heads).view(rows, heads)    # factors of e^3.6 to e^5.4: 36 to 222 times the others at zero
    q[..., 1] = 40.0
    q = q.bfloat16()
    at = lambda *x: torch.tensor(x, dtype=torch.int32, device="cuda")    # noqa: E731
    got = B.kv8_attention(q.cuda(), d.codes, d.scales, at(0, rows), at(n - rows), d.indptr, d.ids, 1.0).double().cpu().numpy()
    z = q.double().numpy() @ kk.T
    for i in range(rows):
        z[i, :, n - rows + i + 1:] = -np.inf
    p = np.exp(z - z.max(-1, keepdims=True))
    p /= p.sum(-1, keepdims=True)
    want, most = p @ vv, p[..., late, None] * np.abs(vv[late])
    small = 2 * (2 * (dim + 4) * 48 + n + 16) * 2.0 ** -24
    bound = 2.0 ** -8 * np.abs(want) + (1 + 2.0 ** -8) * (2.0 ** -8 * (p @ np.abs(vv) - most) * 2 + small * (p @ np.abs(vv)))
    off = np.abs(got - want)
    assert (off <= bound).all(), ((off / bound).max(), np.argwhere(off > bound)[:5])


@pytest.mark.parametrize("entries,kv,group", [(300, 1, 1), (3, 9, 1), (2, 1, 64), (1, 40, 2)])
def test_attention_of_many_entries_and_heads(entries, kv, group):
    rng = np.random.RandomState(entries)
    c = Cache([int(x) for x in rng.randint(0, 90, entries)], [1] * entries, kv, 64, "int8", seed=5)
    attend(c, kv * group, torch.bfloat16, weigh=True)


def test_no_rows_and_no_pages():
    c = Cache([20, 3], [0, 0], 2, 64, "e4m3")
    d = c.device()
    out = torch.full((3, 4, 64), 7.0, device="cuda")
    mass = d.mass.clone()
    B.kv8_attention(torch.zeros_like(out), d.codes, d.scales, d.row0, d.starts, d.indptr, d.ids, 1.0, out=out, mass=d.mass)
    pool = d.pool.clone()
    B.kv8_append(torch.zeros(3, 2, 64, device="cuda"), torch.zeros(3, 2, 64, device="cuda"), d.codes, d.scales, d.row0, d.starts, d.indptr, d.ids)
    assert (out == 7).all() and torch.equal(d.mass, mass) and torch.equal(d.pool, pool)
    # rows of entries that own no pages at all: zeros, nothing written, nothing kept
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    row0, starts, none = i32([0, 1, 3]), i32([0, 40]), i32([])
    B.kv8_append(torch.ones(3, 2, 64, device="cuda"), torch.ones(3, 2, 64, device="cuda"), d.codes, d.scales, row0, starts, i32([0, 0, 0]), none)
    B.kv8_attention(torch.ones_like(out), d.codes, d.scales, row0, starts, i32([0, 0, 0]), none, 1.0, out=out, mass=d.mass)
    k, v = B.kv8_read(d.codes, d.scales, row0, starts, i32([0, 0, 0]), none, 3)
    kept = B.kv8_evict(d.codes, d.scales, d.mass, i32([5, 40]), i32([0, 0, 0]), none, i32([0, 0, 0]), none, 16, 2, 2)
    assert (out == 0).all() and (k == 0).all() and (v == 0).all() and torch.equal(d.mass, mass) and torch.equal(d.pool, pool)
    assert (kept == -1).all()


def test_lengths_and_starts_of_any_size_end():
    """what a table says of a length goes no further than the entry's pages: these calls end at once, and give what the pages hold"""
    c = Cache([31, 15], [1, 1], 2, 64, "int8", seed=33)
    d = c.device()
    q = torch.randn(2, 4, 64, device="cuda").bfloat16()
    want = B.kv8_attention(q, d.codes, d.scales, d.row0, d.starts, d.indptr, d.ids, 0.1)
    weights = torch.zeros_like(d.mass)
    B.kv8_attention(q, d.codes, d.scales, d.row0, d.starts, d.indptr, d.ids, 0.1, mass_out=weights, mass_keep=0.0)
    far = torch.tensor([2 ** 31 - 5000, 2 ** 30], dtype=torch.int32, device="cuda")           # every slot of the pages lies before them
    for row0, rows in ((d.row0, q), (torch.tensor([0, 100, 200], dtype=torch.int32, device="cuda"), torch.randn(200, 4, 64, device="cuda").bfloat16())):
        again = torch.zeros_like(d.mass)
        got = B.kv8_attention(rows, d.codes, d.scales, row0, far, d.indptr, d.ids, 0.1, mass_out=again, mass_keep=0.0)
        assert torch.isfinite(got).all()
        if rows is q:
            assert torch.equal(got, want) and torch.equal(again, weights)
    free = [p for p in range(c.pages) if p not in c.ids]
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    for lens in ([2 ** 31 - 1, -5], [2 ** 30, 2 ** 31 - 1]):
        kept = B.kv8_evict(d.codes, d.scales, d.mass, i32(lens), d.indptr, d.ids, i32([0, 1, 2]), i32(free[:2]), 10, 2, 3)
        assert kept[0, :, :2].tolist() == [[0, 1]] * 2 and kept[0, :, -3:].tolist() == [[29, 30, 31]] * 2
        assert (kept[1] == -1).all() if lens[1] < 0 else kept[1, :, -3:].tolist() == [[13, 14, 15]] * 2


def test_rows_in_and_out_at_the_last_slots_of_32_bits():
    """starts that have no page, and a grid that reaches past 2^31 behind them: the walks end, nothing is written, what is read is 0"""
    c = Cache([0, 0], [16, 7984], 1, 64, "int8", seed=34)
    d = c.device()
    rows = torch.randn(8000, 1, 64, device="cuda").bfloat16()
    pool, scales = d.pool.clone(), d.scales.clone()
    for start in (2 ** 31 - 1 - 32 - 7984, 2 ** 31 - 40000, 2 ** 30):
        at = torch.tensor([start, start], dtype=torch.int32, device="cuda")
        for most in (None, 1, 8000, 2 ** 40):
            B.kv8_append(rows, rows, d.codes, d.scales, d.row0, at, d.indptr, d.ids, max_rows=most)
            k, v = B.kv8_read(d.codes, d.scales, d.row0, at, d.indptr, d.ids, 8000, max_rows=most)
            assert (k == 0).all() and (v == 0).all()
    assert torch.equal(d.pool, pool) and torch.equal(d.scales.nan_to_num(7), scales.nan_to_num(7))
    many = torch.empty(2 ** 26 + 1, dtype=torch.int32, device="cuda")
    with pytest.raises(RuntimeError):
        B.kv8_append(rows, rows, d.codes, d.scales, d.row0, d.starts, d.indptr, many)


def test_tables_that_lead_nowhere():
    """pages out of range, tables that end early, rows out of range, entries that start nowhere: not there, and nothing else is touched"""
    c = Cache([20, 40, 5, 33, 70], [4, 1, 1, 2, 1], 2, 64, "int8", seed=8)
    c.ids[c.indptr[0]] = -3
    c.ids[c.indptr[1] + 1] = c.pages
    c.ids[c.indptr[2]] = 2 ** 31 - 1                   # all its tokens: zeros
    c.indptr[5] -= 1                                   # the last entry's last page: its newest token
    d, out = attend(c, 4, torch.bfloat16, weigh=True)
    assert (out[5] == 0).all()
    codes, scales = c.codes.copy(), c.scales.copy()
    k, kd = rows_of(c.rng, c.row0[-1], 2, 64, torch.float32)
    R.append(k, k, codes, scales, "int8", c.row0, c.starts, c.tables)
    B.kv8_append(kd, kd, d.codes, d.scales, d.row0, d.starts, d.indptr, d.ids)
    same(d, c, codes, scales)
    for x, y in zip(B.kv8_read(d.codes, d.scales, d.row0, d.starts, d.indptr, d.ids, c.row0[-1]), R.read(codes, scales, "int8", 64, c.row0, c.starts, c.tables)):
        assert np.array_equal(x.double().cpu().numpy(), y)
    # an entry that starts before 0, one whose rows lie behind the rows there are
    d.starts[0] = -1
    d.row0[5] = 100
    out = torch.full((9, 4, 64), 7.0, dtype=torch.bfloat16, device="cuda")
    B.kv8_attention(torch.zeros_like(out), d.codes, d.scales, d.row0, d.starts, d.indptr, d.ids, 1.0, out=out)
    assert (out[:4] == 7).all() and (out[4:] != 7).all()


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_prompts_over_pages_that_are_not_there(fmt, dim):
    """many rows: whole blocks missing, at the ends and in the middle; scales that nothing but 0 is left of beside the scores'"""
    c = Cache([40, 0], [150, 90], 2, dim, fmt, seed=21, layers=2)
    c.ids[c.indptr[0]], c.ids[c.indptr[0] + 5], c.ids[c.indptr[1] + 2] = -1, c.pages, 2 ** 31 - 1
    c.indptr[2] -= 1
    attend(c, 4, torch.bfloat16, weigh=True)
    c.scales[:] = 2.0 ** -100
    attend(c, 4, torch.bfloat16, weigh=True)


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
def test_prompts_split_over_a_long_cache(fmt):
    """a portion of a prompt over more than a run of 64 blocks, few enough rows that the keys are split"""
    attend(Cache([2300], [40], 1, 128, fmt, seed=22), 4, torch.bfloat16, weigh=True)
    attend(Cache([1500, 30], [33, 129], 1, 64, fmt, seed=23), 4, torch.bfloat16)


# ---- eviction ----
def run_evict(c, lens, budget, first, last, dst_extra=0):
    """entries of `lens` tokens over c's pages; fresh pages behind c's own"""
    n = [(min(x, budget) + 15) // 16 + dst_extra for x in lens]
    free = [p for p in range(c.pages) if p not in c.ids]
    assert len(free) >= sum(n)
    dst = [int(x) for x in np.concatenate([[0], np.cumsum(n)])], free[:sum(n)]
    d = c.device()
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    codes, scales, mass = c.codes.copy(), c.scales.copy(), c.mass.copy()
    want = R.evict(codes, scales, c.fmt, c.dim, mass, lens, c.tables, dst, budget, first, last)
    for hint in (None, 1):
        kept = B.kv8_evict(d.codes, d.scales, d.mass, i32(lens), d.indptr, d.ids, i32(dst[0]), i32(dst[1]), budget, first, last, max_len=hint)
        assert np.array_equal(kept.cpu().numpy(), want)
        same(d, c, codes, scales)
        assert np.array_equal(d.mass.cpu().numpy(), mass, equal_nan=True)
    return d, kept, dst


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
@pytest.mark.parametrize("kv,dim", [(1, 64), (3, 128), (2, 256)])
@pytest.mark.parametrize("budget,first,last", [(1, 0, 0), (16, 4, 4), (37, 0, 20), (64, 64, 0), (50, 1, 49), (200, 3, 5)])
def test_evict(fmt, kv, dim, budget, first, last):
    lens = [0, 1, 16, 37, 150, 200, 201, 64]
    c = Cache(lens, [0] * 8, kv, dim, fmt, seed=budget, pages=150, dirty=False, layers=2)
    run_evict(c, lens, budget, first, last)


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
def test_evict_equal_and_odd_weights(fmt):
    lens = [120, 120, 120]
    c = Cache(lens, [0] * 3, 2, 64, fmt, seed=1, pages=60, dirty=False)
    c.mass[:, 0] = np.random.RandomState(0).choice(np.array([0.0, -0.0, 1.0, -1.0], np.float32), c.mass[:, 0].shape)
    c.mass[:, 1] = np.random.RandomState(1).choice(np.array([np.nan, np.inf, -np.inf, 1e-40, 0.0], np.float32), c.mass[:, 1].shape)
    run_evict(c, lens, 50, 2, 10)
    run_evict(c, lens, 100, 0, 0)


def test_weights_at_any_four_bytes():
    """weights and scales whose pages lie an odd number of values apart, from an odd place: what aligned ones give, and nothing between them is touched"""
    lens = [300, 41]
    c = Cache([x - 1 for x in lens], [1, 1], 3, 64, "e4m3", seed=12, dirty=False, pages=60)
    a, b = c.device(), c.device()
    apart = 3 * 16 + 3
    room = torch.full((c.pages * apart + 5,), 9.0, device="cuda")
    b.mass = room[5:].as_strided((c.pages, 3, 16), (apart, 16, 1))
    b.mass.copy_(a.mass)
    scales = torch.zeros(c.pages * 7 + 1, device="cuda")[1:].as_strided((c.pages, 2, 3), (7, 3, 1))
    scales.copy_(b.scales)
    b.scales = scales
    q = torch.randn(2, 6, 64, device="cuda").bfloat16()
    free = torch.tensor([p for p in range(c.pages) if p not in c.ids], dtype=torch.int32, device="cuda")
    dst = torch.tensor([0, 7, 10], dtype=torch.int32, device="cuda")
    got = []
    for d in (a, b):
        out = B.kv8_attention(q, d.codes, d.scales, d.row0, d.starts, d.indptr, d.ids, 0.125, mass=d.mass, mass_keep=0.5)
        kept = B.kv8_evict(d.codes, d.scales, d.mass, d.lens, d.indptr, d.ids, dst, free, 100, 5, 9)
        got.append((out, kept, d.mass.contiguous(), d.scales.contiguous(), d.codes.contiguous().view(torch.uint8)))
    for x, y in zip(*got):
        assert torch.equal(x, y)
    rest = torch.ones_like(room, dtype=torch.bool)
    rest[5:].as_strided((c.pages, 3, 16), (apart, 16, 1)).fill_(False)
    assert (room[rest] == 9).all()


def test_evict_of_many_tokens_and_of_shared_pages():
    lens = [2500, 1030, 2500]
    c = Cache(lens, [0] * 3, 2, 64, "int8", seed=2, pages=700, dirty=False)
    a, b = c.indptr[0], c.indptr[2]
    c.ids[b:b + 100] = c.ids[a:a + 100]                # the third entry's first 1600 tokens are the first one's
    run_evict(c, lens, 1029, 4, 100, dst_extra=1)


@pytest.mark.parametrize("first,last", [(0, 0), (4, 100), (700, 329)])
def test_evict_whatever_the_hint(first, last):
    """the weights of the first max_len tokens are kept at hand, the others' looked up again: ends of that part inside and at the ends of every wave's run"""
    lens = [2500, 1030, 40000]
    c = Cache(lens, [0] * 3, 1, 64, "int8", seed=3, dirty=False)
    d, got = c.device(), []
    dst = torch.zeros(4, dtype=torch.int32, device="cuda")               # no pages to move to: the slots that stay are what is looked at
    order = [c.mass[[c.ids[i] for i in range(c.indptr[e], c.indptr[e + 1])], 0].reshape(-1)[:n] for e, n in enumerate(lens)]
    for most in (None, 0, 1, 63, 64, 256, 1000, 1024, 2047, 2304, 2499, 2500, 20000, 36865, 10 ** 6):
        kept = B.kv8_evict(d.codes, d.scales, d.mass, d.lens, d.indptr, d.ids, dst, dst[:0], 1029, first, last, max_len=most)
        got.append(kept.cpu().numpy()[:, 0])
    for e, n in enumerate(lens):
        between = np.argsort(-order[e][first:n - last], kind="stable")[:1029 - first - last] + first
        want = np.sort(np.concatenate([np.arange(first), between, np.arange(n - last, n)]))
        for g in got:
            assert np.array_equal(g[e], want), (e, np.argwhere(g[e] != want)[:4])


def test_evict_with_pages_that_are_not_there():
    lens = [100, 90]
    c = Cache(lens, [0] * 2, 2, 64, "e4m3", seed=2, pages=60, dirty=False)
    c.ids[2], c.ids[c.indptr[1] + 1] = -1, 10 ** 6
    run_evict(c, lens, 40, 20, 5)
    run_evict(c, lens, 90, 0, 0)


# ---- together, as a server uses them ----
@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
def test_prompt_steps_eviction_steps(fmt):
    """prompts in, their weights, steps, a cut to a budget, steps behind it: against the restatement all the way"""
    kv, H, dim, budget, heads_of = 2, 6, 64, 48, 3
    c = Cache([0, 0], [90, 37], kv, dim, fmt, seed=11, pages=40, dirty=False, extra=1)
    d = c.device()
    free = [p for p in range(c.pages) if p not in c.ids]
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    codes, scales, mass = c.codes.copy(), c.scales.copy(), c.mass.copy()
    tables, starts, rows = c.tables, [0, 0], [90, 37]

    def step(keep):
        row0 = [0, rows[0], rows[0] + rows[1]]
        (k, kd), (v, vd), (q, qd) = (rows_of(c.rng, row0[-1], h, dim, torch.bfloat16) for h in (kv, kv, H))
        t = i32(row0), i32(starts), i32(tables[0]), i32(tables[1])
        B.kv8_append(kd, vd, d.codes, d.scales, *t)
        R.append(k, v, codes, scales, fmt, row0, starts, tables)
        same(d, c, codes, scales)
        out = B.kv8_attention(qd, d.codes, d.scales, *t, 0.125, mass=d.mass, mass_keep=keep)
        want, new, spread, reach = R.attention(q, codes, scales, fmt, row0, starts, tables, 0.125)
        err = np.abs(out.double().cpu().numpy() - want)
        assert (err <= attention_bound(spread, reach, want, dim, 128, torch.bfloat16)).all()
        for e in range(2):
            for s in range(new[e].shape[1]):
                p = R.page_of(tables, e, s // 16, c.pages)
                mass[p, :, s % 16] = (keep * mass[p, :, s % 16] if keep else 0) + new[e][:, s]
                off = np.abs(d.mass[p, :, s % 16].cpu().numpy() - mass[p, :, s % 16])
                assert (off <= mass_bound(new[e][:, s], reach.max(), dim, 128, rows[e] * heads_of) + 1e-5 * mass[p, :, s % 16]).all()
        mass[:] = d.mass.cpu().numpy()                   # from here on the device's own sums
        starts[:] = [s + r for s, r in zip(starts, rows)]

    step(0.0)
    rows = [1, 1]
    for _ in range(3):
        step(1.0)
    n = [(min(x, budget) + 15) // 16 + 1 for x in starts]
    dst = [0, n[0], n[0] + n[1]], free[:sum(n)]
    kept = B.kv8_evict(d.codes, d.scales, d.mass, i32(starts), i32(tables[0]), i32(tables[1]), i32(dst[0]), i32(dst[1]), budget, 4, 16)
    assert np.array_equal(kept.cpu().numpy(), R.evict(codes, scales, fmt, dim, mass, list(starts), tables, dst, budget, 4, 16))
    same(d, c, codes, scales)
    assert np.array_equal(d.mass.cpu().numpy(), mass)
    tables, starts[:] = dst, [min(x, budget) for x in starts]
    for _ in range(4):
        step(0.9)


def test_a_captured_step_replays_with_other_tables():
    """append, attention with weights: captured once, replayed as the sequences grow, against the same calls outside the graph"""
    kv, H, dim = 2, 8, 128
    c = Cache([30, 200, 0], [1, 1, 1], kv, dim, "e4m3", seed=12, pages=60, dirty=False, extra=2)
    a, b = c.device(), c.device()
    k, q = torch.randn(3, kv, dim, device="cuda").bfloat16(), torch.randn(3, H, dim, device="cuda").bfloat16()
    out = torch.zeros_like(q)

    def step(d, out):
        B.kv8_append(k, k, d.codes, d.scales, d.row0, d.starts, d.indptr, d.ids, max_rows=1)
        B.kv8_attention(q, d.codes, d.scales, d.row0, d.starts, d.indptr, d.ids, 0.1, max_rows=1, max_len=256, out=out, mass=d.mass)

    warm = c.device()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(warm, out)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(a, out)
    for i in range(4):
        k.copy_(torch.randn(3, kv, dim, device="cuda") * (i + 1))
        q.copy_(torch.randn(3, H, dim, device="cuda"))
        graph.replay()
        eager = torch.zeros_like(q)
        step(b, eager)
        torch.cuda.synchronize()
        assert torch.equal(out, eager) and torch.equal(a.pool, b.pool) and torch.equal(a.scales, b.scales) and torch.equal(a.mass, b.mass), i
        for d in (a, b):
            d.starts += 1


def test_a_captured_prompt_and_eviction_replay():
    """a portion of a prompt with weights, the cut and what is read back, captured once and replayed over other values, with eager work in between"""
    kv, H, dim, budget = 2, 8, 64, 100
    c = Cache([40, 0], [150, 60], kv, dim, "int8", seed=31, pages=80, dirty=False)
    free = [p for p in range(c.pages) if p not in c.ids]
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    dst, ids = i32([0, 7, 14]), i32(free[:14])
    zeros = i32([0, 0])
    back0 = i32([0, 100, 160])
    a, b = c.device(), c.device()
    k, q = torch.randn(210, kv, dim, device="cuda"), torch.randn(210, H, dim, device="cuda")

    def step(d):
        t = d.row0, d.starts, d.indptr, d.ids
        B.kv8_append(k, k, d.codes, d.scales, *t)
        out = B.kv8_attention(q, d.codes, d.scales, *t, 0.2, mass=d.mass, mass_keep=0.5)
        kept = B.kv8_evict(d.codes, d.scales, d.mass, d.lens, d.indptr, d.ids, dst, ids, budget, 4, 10)
        return (out, kept) + B.kv8_read(d.codes, d.scales, back0, zeros, dst, ids, 160)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(c.device())
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step(a)
    for i in range(4):
        k.copy_(torch.randn_like(k) * (i + 1))
        q.copy_(torch.randn_like(q))
        graph.replay()
        want = step(b)
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(got, want)) and torch.equal(a.mass, b.mass) and torch.equal(a.pool, b.pool) and torch.equal(a.scales, b.scales), i


def test_two_streams_at_once():
    """the same operators on two streams, each with its cache: workspaces are not shared"""
    c = [Cache([700, 30], [1, 20], 2, 128, f, seed=s) for s, f in enumerate(TORCH)]
    d = [x.device() for x in c]
    q = torch.randn(21, 8, 128, device="cuda").bfloat16()
    run = lambda x: B.kv8_attention(q, x.codes, x.scales, x.row0, x.starts, x.indptr, x.ids, 0.1, mass=x.mass, mass_keep=0.0)  # noqa: E731
    want = [(run(x).clone(), x.mass.clone()) for x in d]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in d]
    for _ in range(5):
        got = []
        for x, s in zip(d, streams):
            with torch.cuda.stream(s):
                got.append(run(x))
        torch.cuda.synchronize()
        for x, g, w in zip(d, got, want):
            assert torch.equal(g, w[0]) and torch.equal(x.mass, w[1])


def test_a_cache_that_passes_32_bits():
    """pages 96 MiB apart: the last ones lie 4.5 GiB behind the first"""
    kv, dim, pages, apart = 2, 128, 48, 96 << 20
    c = Cache([200, 100], [1, 3], kv, dim, "int8", seed=13, pages=pages, dirty=False)
    d = c.device()
    pool = torch.empty(pages * apart, dtype=torch.int8, device="cuda")
    codes = pool.as_strided((pages, 2, kv, 16 * dim), (apart, kv * 16 * dim, 16 * dim, 1))
    codes.copy_(d.codes)
    d.codes = codes
    k, kd = rows_of(c.rng, 4, kv, dim, torch.bfloat16)
    R.append(k, k, c.codes, c.scales, "int8", c.row0, c.starts, c.tables)
    B.kv8_append(kd, kd, d.codes, d.scales, d.row0, d.starts, d.indptr, d.ids)
    assert np.array_equal(codes.cpu().numpy().view(np.uint8), c.codes) and np.array_equal(d.scales.cpu().numpy(), c.scales)
    attend(c, 4, torch.bfloat16, weigh=True, d=d)


def test_wrappers_refuse():
    c = Cache([20], [4], 2, 64, "e4m3")
    d = c.device()
    q = torch.zeros(4, 4, 64, dtype=torch.bfloat16, device="cuda")
    k = torch.zeros(4, 2, 64, dtype=torch.bfloat16, device="cuda")
    t = (d.row0, d.starts, d.indptr, d.ids)
    go = lambda **kw: B.kv8_attention(**{**dict(q=q, codes=d.codes, scales=d.scales, row0=d.row0, starts=d.starts, page_indptr=d.indptr, page_ids=d.ids, scale=1.0), **kw})  # noqa: E731
    assert go().shape == q.shape
    for kw in [dict(q=q.half()), dict(q=q.float()[..., ::2]), dict(q=q[:, :3]), dict(q=q[..., :32]), dict(q=q.cpu()), dict(q=q.transpose(0, 1)), dict(codes=d.pool[:, -1]),
               dict(codes=d.codes[..., :1000]), dict(codes=d.codes.cpu()), dict(scales=d.scales[:-1]), dict(scales=d.scales.double()), dict(row0=d.row0.long()), dict(row0=d.row0.cpu()),
               dict(starts=d.indptr), dict(page_indptr=d.starts), dict(out=q.float()), dict(out=q[:2]), dict(out=q), dict(scale=-1.0), dict(scale=float("nan")), dict(mass=d.mass[..., :8]), dict(mass=d.mass.double()),
               dict(mass_out=d.mass), dict(page_ids=d.ids[None]), dict(max_rows=-1), dict(max_len=-1)]:
        with pytest.raises((ValueError, RuntimeError)):
            go(**kw)
    with pytest.raises(ValueError):
        B.kv8_append(k, k.float(), d.codes, d.scales, *t)
    with pytest.raises(ValueError):
        B.kv8_append(k[:, :1], k[:, :1], d.codes, d.scales, *t)
    with pytest.raises(ValueError):
        B.kv8_read(d.codes, d.scales, *t, 4, dtype=torch.float16)
    for budget, first, last in [(0, 0, 0), (8, 5, 4), (8, -1, 0)]:
        with pytest.raises(ValueError):
            B.kv8_evict(d.codes, d.scales, d.mass, d.lens, d.indptr, d.ids, d.indptr, d.ids, budget, first, last)
    none = torch.zeros(0, 4, 64, dtype=torch.bfloat16, device="cuda")
    zero = torch.zeros(1, dtype=torch.int32, device="cuda")
    assert B.kv8_attention(none, d.codes, d.scales, zero, zero[:0], zero, d.ids, 1.0).shape == (0, 4, 64)      # no entries
