"""Small 8-bit paged caches for the tests: tables, pages in no order, what came before in them."""
import numpy as np
import torch

from oracle import kv8_ref as R

TORCH = {"e4m3": torch.float8_e4m3fn, "int8": torch.int8}


class Cache:
    """entries with `starts` tokens in front of `rows` rows; every byte of the pool is drawn (NaN codes too where `dirty`: behind an entry's last token)"""

    def __init__(self, starts, rows, kv, dim, fmt, seed=0, pages=None, dirty=True, layers=1, extra=0):
        rng = np.random.RandomState(seed)
        self.kv, self.dim, self.fmt, self.rng = kv, dim, fmt, rng
        self.starts, self.rows, self.B = list(starts), list(rows), len(starts)
        self.row0 = [int(x) for x in np.concatenate([[0], np.cumsum(rows)])]
        n = [(s + r + 15) // 16 + extra for s, r in zip(starts, rows)]
        self.indptr = [int(x) for x in np.concatenate([[0], np.cumsum(n)])]
        self.pages = (pages or sum(n) + 3)
        self.ids = [int(x) for x in rng.permutation(self.pages)[:sum(n)]]
        self.codes = rng.randint(0, 256, (self.pages, 2, kv, 16 * dim)).astype(np.uint8)
        self.scales = (2.0 ** rng.randint(-9, -4, (self.pages, 2, kv))).astype(np.float32)
        self.mass = np.exp(rng.randn(self.pages, kv, 16)).astype(np.float32)
        if fmt == "e4m3":
            nan = self.codes & 127 == 127
            keep = np.zeros_like(nan)
            if dirty:
                for e in range(self.B):
                    for t in range(16):
                        last = starts[e] + rows[e]
                        if last % 16 and t >= last % 16:
                            for side in (0, 1):
                                keep[self.ids[self.indptr[e] + last // 16], side][:, R.offsets(dim, side, t)] = True
            self.codes[nan & ~keep] &= 0xF0
        else:
            self.codes[self.codes == 128] = 127
        self.layers = layers

    @property
    def tables(self):
        return self.indptr, self.ids

    def device(self):
        """tensors on the device: the cache as one layer of a page-first pool where layers > 1"""
        i32 = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
        pool = torch.zeros(self.pages, self.layers, 2, self.kv, 16 * self.dim, dtype=torch.uint8, device="cuda")
        pool[:, -1] = torch.from_numpy(self.codes).cuda()
        sc = torch.zeros(self.pages, self.layers, 2, self.kv, device="cuda")
        sc[:, -1] = torch.from_numpy(self.scales).cuda()
        ms = torch.zeros(self.pages, self.layers, self.kv, 16, device="cuda")
        ms[:, -1] = torch.from_numpy(self.mass).cuda()
        d = type("Dev", (), {})()
        d.pool, d.codes, d.scales, d.mass = pool, pool.view(TORCH[self.fmt])[:, -1], sc[:, -1], ms[:, -1]
        d.row0, d.starts, d.indptr, d.ids = i32(self.row0), i32(self.starts), i32(self.indptr), i32(self.ids)
        d.lens = i32([s + r for s, r in zip(self.starts, self.rows)])
        return d


def codes_of(d):
    return d.codes.view(torch.uint8).cpu().numpy()


def attention_bound(spread, reach, out, dim, length, dtype):
    """How far an output may be off.  Scores: products are exact, sums of dim values and the two factors err by (dim + 4) 2^-24 of sum |q k| scale at most, the
    exponential and the fp32 sums by (length + 16) 2^-24 relative, numerator and denominator alike.  bf16 adds the weights' rounding, 2^-8 each, and the output's."""
    rel = 2 * (2 * (dim + 4) * 2.0 ** -24 * reach + (length + 16) * 2.0 ** -24)[..., None]
    half = torch.finfo(dtype).eps / 2
    return (rel + (half if dtype == torch.bfloat16 else 0.0)) * spread + half * (np.abs(out) + rel * spread) + 1e-30


def mass_bound(mass, reach, dim, length, rows):
    """a sum of `rows` weights, each off by the score's error and that of the log-sum (2 (dim + 4) + length + 16) 2^-24 as above"""
    return mass * (2 * (2 * (dim + 4) * reach + length + 16) + rows) * 2.0 ** -24 + 1e-12
