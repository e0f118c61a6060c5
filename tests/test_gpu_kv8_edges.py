"""The 8-bit paged cache on the device at the ends of its ranges, and with what a pool of pages held before."""
import numpy as np
import pytest
import torch

from oracle import kv8_ref as R
from pegainfer_amd import ops_blocks as B
from kv8_common import Cache, attention_bound, codes_of, mass_bound
from test_gpu_kv8_ops import attend

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


# ---- weights of pages that another entry gave back ----
@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("kv,dim", [(1, 64), (3, 128), (2, 256)])
def test_appended_tokens_weigh_nothing(fmt, dtype, kv, dim):
    c = Cache([0, 5, 16, 31, 40, 7, 0], [1, 1, 33, 1, 0, 9, 17], kv, dim, fmt, seed=kv, layers=2)
    c.ids[c.indptr[2]], c.ids[c.indptr[6]] = -1, c.pages                 # pages that are not there
    k = torch.randn(c.row0[-1], kv, dim, device="cuda").to(TYPES[dtype])
    want = c.mass.copy()
    for e in range(c.B):
        for s in range(c.starts[e], (c.starts[e] + c.rows[e] + 15) // 16 * 16 if c.rows[e] else 0):
            p = R.page_of(c.tables, e, s // 16, c.pages)
            if p >= 0:
                want[p, :, s % 16] = 0
    for most in (None, 1, 33):
        a, b = c.device(), c.device()
        for d, kw in ((a, {}), (b, dict(mass=b.mass))):
            B.kv8_append(k, k, d.codes, d.scales, d.row0, d.starts, d.indptr, d.ids, max_rows=most, **kw)
        assert np.array_equal(b.mass.cpu().numpy(), want) and np.array_equal(a.mass.cpu().numpy(), c.mass)
        assert torch.equal(a.pool, b.pool) and torch.equal(a.scales, b.scales)
    with pytest.raises(ValueError):
        B.kv8_append(k, k, b.codes, b.scales, b.row0, b.starts, b.indptr, b.ids, mass=b.mass[..., :8])


def test_a_pool_that_pages_come_back_to():
    """a session over pages that another one left: its weights, what it evicts and what it answers are those over a fresh pool"""
    kv, H, dim, pages, budget = 2, 4, 64, 12, 40
    order = i32(*range(1, pages))
    rows = torch.randn(70, kv, dim, device="cuda").bfloat16()
    q = torch.randn(70, H, dim, device="cuda").bfloat16()

    def session(codes, scales, mass, n):
        """a prompt, steps, a cut, a step behind it"""
        got = []
        for start, m in [(0, n)] + [(n + i, 1) for i in range(5)]:
            t = i32(0, m), i32(start), i32(0, 7), order
            B.kv8_append(rows[start:start + m], rows[start:start + m], codes, scales, *t, mass=mass)
            got.append(B.kv8_attention(q[:m], codes, scales, *t, 0.125, mass=mass))
        got.append(B.kv8_evict(codes, scales, mass, i32(n + 5), i32(0, 7), order, i32(0, 4), order[7:], budget, 2, 8))
        t = i32(0, 1), i32(min(budget, n + 5)), i32(0, 4), order[7:]
        B.kv8_append(rows[:1], rows[:1], codes, scales, *t, mass=mass)
        return got + [B.kv8_attention(q[:1], codes, scales, *t, 0.125, mass=mass)]

    def pool():
        return torch.zeros(pages, 2, kv, 16 * dim, dtype=torch.int8, device="cuda"), torch.ones(pages, 2, kv, device="cuda"), torch.zeros(pages, kv, 16, device="cuda")

    used, fresh = pool(), pool()
    session(*used, 61)
    for a, b in zip(session(*used, 50), session(*fresh, 50)):
        assert torch.equal(a, b)
    assert torch.equal(used[2][order[7:10].long()], fresh[2][order[7:10].long()])


def test_a_hint_of_no_rows_gives_what_any_gives():
    c = Cache([20, 0, 600], [4, 20, 1], 2, 64, "e4m3", seed=41, dirty=False)
    a, b = c.device(), c.device()
    k, q = torch.randn(25, 2, 64, device="cuda").bfloat16(), torch.randn(25, 4, 64, device="cuda").bfloat16()
    got = []
    for d, most in ((a, 0), (b, 1)):
        t = d.row0, d.starts, d.indptr, d.ids
        B.kv8_append(k, k, d.codes, d.scales, *t, max_rows=most)
        for length in (700, 3000):
            got.append((B.kv8_attention(q, d.codes, d.scales, *t, 0.1, max_rows=most, max_len=length, mass=d.mass, out=torch.full_like(q, 7.0)),
                        *B.kv8_read(d.codes, d.scales, *t, 25, max_rows=most, out=(torch.full_like(k, 7.0), torch.full_like(k, 7.0)))))
    for x, y in zip(got[:2], got[2:]):
        assert all(torch.equal(i, j) for i, j in zip(x, y))
    assert torch.equal(a.pool, b.pool) and torch.equal(a.scales, b.scales) and torch.equal(a.mass, b.mass)


# ---- entries of more rows than the call said ----
@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("kv,group,dim", [(2, 1, 64), (1, 3, 128), (1, 2, 256)])
def test_weights_of_more_rows_than_were_said(fmt, dtype, kv, group, dim):
    """the weights of a step's call where an entry brings a portion: over few tokens, over a run of keys, over split ones; pages that are not there"""
    c = Cache([40, 9, 0], [70, 1, 33], kv, dim, fmt, seed=dim, layers=2)
    c.ids[c.indptr[0] + 1] = -1
    for length in (300, 1000, 9000):
        attend(c, kv * group, TYPES[dtype], weigh=True, keep=0.5, hints=(1, length))
    attend(Cache([1100, 3], [20, 1], kv, dim, fmt, seed=dim + 1), kv * group, TYPES[dtype], weigh=True, hints=(1, 1200), keep=0.0)


def test_a_portion_among_single_tokens_is_not_a_cliff():
    """the default hint is the average of the rows: with weights, a portion that it does not fit takes a few times what it takes with a hint of its own, not 66 times"""
    n, kv, dim, ctx = 256, 8, 128, 300
    c = Cache([ctx] * 32, [n] + [1] * 31, kv, dim, "int8", seed=50, dirty=False)
    d = c.device()
    q = torch.randn(c.row0[-1], kv, dim, device="cuda").bfloat16()

    def time(most):
        run = lambda: B.kv8_attention(q, d.codes, d.scales, d.row0, d.starts, d.indptr, d.ids, 0.1, max_rows=most, max_len=600, mass=d.mass)  # noqa: E731
        a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        run()
        a.record()
        for _ in range(10):
            run()
        b.record()
        torch.cuda.synchronize()
        return a.elapsed_time(b)

    best = {most: min(time(most) for _ in range(3)) for most in (None, n)}
    assert best[None] < 12 * best[n], best


def test_a_budget_beyond_32_bits_is_refused():
    c = Cache([20], [4], 1, 64, "e4m3")
    d = c.device()
    for budget, first in [(2 ** 31, 0), (2 ** 32 + 8, 0), (2 ** 32 + 8, 2 ** 32)]:
        with pytest.raises(ValueError):
            B.kv8_evict(d.codes, d.scales, d.mass, d.lens, d.indptr, d.ids, d.indptr, d.ids, budget, first)


@pytest.mark.parametrize("rows", [[1, 1, 1], [40, 33, 3]])
def test_weights_behind_a_common_prompt(rows):
    """entries that share the pages of a prompt, one call each over weights that were scaled before: every page has the sum of all"""
    kv, H, dim, keep = 2, 6, 64, 0.5
    c = Cache([70, 64, 90], rows, kv, dim, "int8", seed=60, dirty=False)
    for e in (1, 2):
        c.ids[c.indptr[e]:c.indptr[e] + 4] = c.ids[:4]                   # 64 tokens
    d = c.device()
    d.mass *= keep
    q = torch.randn(c.row0[-1], H, dim, device="cuda").bfloat16()
    out = torch.zeros_like(q)
    for e in range(3):
        mine = slice(c.row0[e], c.row0[e + 1])
        B.kv8_attention(q[mine], d.codes, d.scales, i32(0, rows[e]), d.starts[e:e + 1], i32(0, c.indptr[e + 1] - c.indptr[e]), d.ids[c.indptr[e]:c.indptr[e + 1]], 0.125, out=out[mine],
                        mass=d.mass)
    answer, mass, spread, reach = R.attention(q.float().cpu().numpy(), c.codes, c.scales, c.fmt, c.row0, c.starts, c.tables, 0.125)
    assert (np.abs(out.double().cpu().numpy() - answer) <= attention_bound(spread, reach, answer, dim, 140, torch.bfloat16)).all()
    want, most = keep * c.mass.astype(np.float64), np.zeros(c.mass.shape)
    for e in range(3):
        for s in range(mass[e].shape[1]):
            p = c.ids[c.indptr[e] + s // 16]
            want[p, :, s % 16] += mass[e][:, s]
            most[p, :, s % 16] += mass_bound(mass[e][:, s], reach.max(), dim, 140, rows[e] * 3)
    assert (np.abs(d.mass.cpu().numpy() - want) <= most + 2.0 ** -22 * want).all()


@pytest.mark.parametrize("rows", [1, 8, 40])
@pytest.mark.parametrize("length", [64, 2000])
def test_a_row_without_a_score_above_minus_infinity(rows, length):
    """zeros, and no weight: by steps, two row tiles and prompts, whole and split"""
    c = Cache([200], [rows], 1, 64, "int8", seed=70, dirty=False)
    c.codes[:, 0] = 3                                                    # every key is above 0
    d = c.device()
    q = torch.randn(rows, 4, 64, device="cuda").bfloat16()
    q[0, 1] = -torch.inf
    out = B.kv8_attention(q, d.codes, d.scales, d.row0, d.starts, d.indptr, d.ids, 0.125, max_len=length, mass=d.mass, mass_keep=0.0)
    assert (out[0, 1] == 0).all() and torch.isfinite(out).all()
    total = sum(d.mass[c.ids[s // 16], 0, s % 16] for s in range(200 + rows)).item()
    assert abs(total - (4 * rows - 1)) <= 4 * rows * (200 + rows + 16) * 2.0 ** -22
