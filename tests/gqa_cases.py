"""Ragged GQA batches over the block-scaled 8-bit cache, shared by the CPU and GPU tests."""
import numpy as np

from oracle import gqa as G8


def bf16(x):
    """x rounded to bf16, as float32."""
    b = np.ascontiguousarray(x, np.float32).view(np.uint32)
    return ((b + 0x7FFF + ((b >> 16) & 1)) & 0xFFFF0000).astype(np.uint32).view(np.float32)


def rounded(x, dtype):
    return bf16(x) if dtype == "bf16" else np.asarray(x, np.float32).astype(np.float16).astype(np.float32)


class Batch:
    """`rows[b]` new rows of lane b behind `ctx[b]` cached ones.  Pages are handed out in random order from
    page 1; what no lane's row fills (page 0, spare pages, the ends of last pages) holds NaN codes,
    and scales of pages no lane owns are NaN."""

    def __init__(self, rows, ctx, heads, kv, dim, page, dtype="bf16", seed=0, spare=2, pow2=True, sharp=2.0):
        rng = np.random.default_rng(seed)
        self.rows, self.ctx, self.heads, self.kv, self.dim, self.page, self.dtype = list(rows), list(ctx), heads, kv, dim, page, dtype
        lanes = len(rows)
        need = [-(-(r + c) // page) if r else 0 for r, c in zip(rows, ctx)]
        self.pages = 1 + sum(need) + spare
        perm = 1 + rng.permutation(self.pages - 1)
        self.bt = np.zeros((lanes, max(need + [0]) + 1), np.int32)
        at = 0
        for b, n in enumerate(need):
            self.bt[b, :n] = perm[at:at + n]
            at += n
        self.cu = np.concatenate([[0], np.cumsum(rows)]).astype(np.int32)
        self.T = int(self.cu[-1])
        self.pos = np.concatenate([np.arange(c, c + r) for r, c in zip(rows, ctx)] + [[]]).astype(np.int32)
        lane = np.repeat(np.arange(lanes), rows)
        self.slots = (self.bt[lane, self.pos // page] * page + self.pos % page).astype(np.int32)
        self.max_rows = max(list(rows) + [0])
        self.max_kv = max([r + c for r, c in zip(rows, ctx) if r] + [0])
        shape = (self.pages, kv, page, dim)
        self.cache = dict(k=np.full(shape, 0x7F, np.uint8), v=np.full(shape, 0x7F, np.uint8),
                          ks=np.full(shape[:2], np.nan, np.float32), vs=np.full(shape[:2], np.nan, np.float32),
                          cen=np.zeros((self.pages, kv, dim), np.int8), cs=np.zeros((self.pages, kv), np.float32))
        for b, n in enumerate(need):
            left = rows[b] + ctx[b]
            for i in range(n):
                p, m = self.bt[b, i], min(page, left - i * page)
                for c, s, amp in (("k", "ks", 1.0), ("v", "vs", 1.0)):
                    x = rng.standard_normal((kv, m, dim)) + 0.4 * rng.standard_normal((kv, 1, dim))
                    f = 2.0 ** rng.integers(-9, -5, kv) if pow2 else 10.0 ** rng.uniform(-3, -1.5, kv)
                    self.cache[c][p, :, :m] = G8.to_e4m3(x * amp / f[:, None, None])
                    self.cache[s][p] = f
                if m == page:
                    G8.centroid(self.cache, p)
        self.q = rounded(rng.standard_normal((self.T, heads, dim)) * sharp, dtype)
        self.scale = float(np.float32(dim ** -0.5))

    def new_rows(self, seed=1, spread=True):
        """K and V rows to append, [T, kv, dim]; with `spread`, rows of very different size."""
        rng = np.random.default_rng(seed)
        out = []
        for _ in range(2):
            x = rng.standard_normal((self.T, self.kv, self.dim))
            if spread:
                x *= 2.0 ** rng.integers(-12, 12, (self.T, self.kv, 1))
            out.append(rounded(x, self.dtype))
        return out
