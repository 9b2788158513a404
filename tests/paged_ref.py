"""Plain 64-bit forms of the ops on a paged cache, and bounds on their errors.

A pool is a numpy array [blocks, n_kv, block_size, head_dim] of f32 / f16, or
for I8 pools a byte array [blocks, n_kv, page]: block_size * head_dim codes,
then one fp16 scale per 32 of them.
"""
import numpy as np

NONE = 0xFFFFFFFF  # a block table entry without a block
U = 2.0 ** -24     # half a step of f32
H = 2.0 ** -11     # half a step of f16


class Batch:
    """Sequences of (positions, rows): rows of the dense operands are each one's last positions."""

    def __init__(self, rng, seqs, block_size, width=0, spare=2, behind=0, before=0):
        self.seqs, self.bs = seqs, block_size
        pages = [-(-n // block_size) for n, _ in seqs]
        self.width = max([width, 1] + pages)
        self.blocks = sum(pages) + spare
        order = rng.permutation(self.blocks)
        self.table = np.full((len(seqs), self.width), NONE, np.uint32)
        at = 0
        for i, n in enumerate(pages):
            self.table[i, :n] = order[at:at + n]
            at += n
        self.starts = (before + np.concatenate([[0], np.cumsum([r for _, r in seqs])])).astype(np.int32)
        self.lens = np.array([n for n, _ in seqs], np.int32)
        self.rows = int(self.starts[-1]) + behind

    def each(self):
        """(row, sequence, position) of every row that belongs to a sequence."""
        for s in range(len(self.seqs)):
            for r in range(self.starts[s], self.starts[s + 1]):
                yield r, s, int(self.lens[s]) - int(self.starts[s + 1] - r)

    def where(self, s, pos):
        """(block, slot) of a position, or None without storage."""
        if pos < 0 or pos >= self.width * self.bs:
            return None
        b = int(self.table[s, pos // self.bs])
        return (b, pos % self.bs) if b < self.blocks else None


def quantise(x):
    """Codes and fp16 scales of groups of 32 of the last axis: scale = fp16(fp32(max / 127)), code = x / scale to even."""
    g = np.asarray(x, np.float64).reshape(*x.shape[:-1], -1, 32)
    d = (np.abs(g).max(-1).astype(np.float32) / np.float32(127)).astype(np.float16)
    step = np.where(d > 0, d, 1).astype(np.float64)[..., None]
    q = np.where(d[..., None] > 0, np.clip(np.rint(g / step), -127, 127), 0)
    return q.astype(np.int8).reshape(x.shape), d


def empty_pool(rng, kind, blocks, n_kv, bs, dim, garbage=False):
    """Finite values everywhere, or (garbage) NaN and infinities."""
    if kind == "i8":
        page = bs * dim + bs * dim // 16
        pool = rng.integers(0, 256, (blocks, n_kv, page), dtype=np.uint8)
        n = blocks * n_kv * bs * dim // 32
        d = np.full(n, np.nan, np.float16) if garbage else np.abs(rng.standard_normal(n) * 0.02).astype(np.float16)
        pool[:, :, bs * dim:] = d.view(np.uint8).reshape(blocks, n_kv, -1)
        return pool
    dt = np.float16 if kind == "f16" else np.float32
    if garbage:
        return rng.choice([np.nan, np.inf, -np.inf], (blocks, n_kv, bs, dim)).astype(dt)
    return rng.standard_normal((blocks, n_kv, bs, dim)).astype(dt)


def store(pool, kind, bs, dim, where, rows):
    """One position's rows [n_kv, dim] into a pool."""
    b, slot = where
    if kind != "i8":
        pool[b, :, slot] = rows
        return
    q, d = quantise(rows)
    pool[b, :, slot * dim:(slot + 1) * dim] = q.view(np.uint8)
    at = bs * dim + slot * dim // 16
    pool[b, :, at:at + dim // 16] = np.ascontiguousarray(d).view(np.uint8)


def load(pool, kind, bs, dim, where):
    """A position's values [n_kv, dim] in 64 bits."""
    b, slot = where
    if kind != "i8":
        return pool[b, :, slot].astype(np.float64)
    q = np.ascontiguousarray(pool[b, :, slot * dim:(slot + 1) * dim]).view(np.int8).astype(np.float64)
    at = bs * dim + slot * dim // 16
    d = np.ascontiguousarray(pool[b, :, at:at + dim // 16]).view(np.float16).astype(np.float64)
    return (q.reshape(len(q), -1, 32) * d[..., None]).reshape(len(q), dim)


def append(batch, kind, dim, pools, rows, limit=None):
    for r, s, pos in batch.each():
        w = batch.where(s, pos)
        if w is not None and (limit is None or pos < limit):
            for pool, x in zip(pools, rows):
                store(pool, kind, batch.bs, dim, w, x[r])


def attention(batch, kind, dim, heads, n_kv, pools, q, act, limit=None):
    """(output, bound on the kernel's error) in 64 bits; rows of no sequence are NaN in the output."""
    out = np.full((batch.rows, heads, dim), np.nan)
    err = np.zeros((batch.rows, heads, dim))
    cells = {}
    f16 = act == "f16"
    for r, s, pos in batch.each():
        cap = min(pos + 1, batch.width * batch.bs if limit is None else min(limit, batch.width * batch.bs))
        if s not in cells:
            n = int(batch.lens[s])
            cells[s] = [[load(p, kind, batch.bs, dim, w) if (w := batch.where(s, i)) else None for i in range(n)]
                        for p in pools]
        keys = [i for i in range(max(0, cap)) if cells[s][0][i] is not None]
        if not keys:
            out[r] = 0.0
            continue
        K, V = (np.stack([cells[s][j][i] for i in keys]) for j in (0, 1))
        for h in range(heads):
            g = h * n_kv // heads
            x = q[r, h].astype(np.float64)
            with np.errstate(all="ignore"):
                sc = K[:, g] @ x / np.sqrt(dim)
                w = np.exp(sc - sc.max())
                o = w @ V[:, g] / w.sum()
                out[r, h] = o
                # scores: dim products and sums in f32, the scale and the base-2 exponent's argument; an 8-bit
                # cache's values are rounded to f16 first beside f16 rows
                a = (np.abs(K[:, g]) @ np.abs(x)).max() / np.sqrt(dim)
                ds = (dim + 8) * U * a + (H * a if f16 and kind == "i8" else 0.0)
                top = np.abs(V[:, g]).max()
                # weights off by exp(ds), sums over the keys in f32; f16: weights, values of an 8-bit cache and the
                # output rounded to f16
                e = 2 * np.expm1(ds) + 2 * (len(keys) + 16) * U
                if f16:
                    e += H * (2 if kind == "i8" else 1)
                err[r, h] = 1.01 * e * top + (H * np.abs(o) + 2.0 ** -25 if f16 else U * np.abs(o))
    return out, err
