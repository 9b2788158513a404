"""Plain 64-bit forms of the operators for long contexts over the paged cache (flash_attention_paged_prefix, the
log-sum-exp of the chunk attention, paged_kv_weights, paged_kv_evict), and bounds on their errors."""
import numpy as np

from paged_ref import H, NONE, U, Batch


class Shared:
    """Groups of consecutive sequences that share positions: (first, one past the last, positions), in order."""

    def __init__(self, batch, groups, named=False):
        assert all(x[1] == y[0] for x, y in zip(groups, groups[1:]))
        self.groups = groups
        first = [a for a, _, _ in groups] + [groups[-1][1] if groups else 0]
        self.first = np.array(first, np.int32)
        self.len = np.array([p for _, _, p in groups], np.int32)
        if named:  # the tables of all the sequences of a group name the shared blocks
            for a, e, p in groups:
                batch.table[a:e, :p // batch.bs] = batch.table[a, :p // batch.bs]

    def of(self, s):
        for a, e, p in self.groups:
            if a <= s < e:
                return a, p
        return s, 0


def where(batch, shared, s, pos):
    """(block, slot) of a position; shared ones through the table of the group's first sequence."""
    if shared is not None:
        first, p = shared.of(s)
        if pos < p:
            s = first
    return batch.where(s, pos)


def cells(batch, shared, s, kind, dim, pools, limit, act):
    """[positions with storage], and their values [pool][position, kv, dim] as rows of type `act` see them."""
    n = min(int(batch.lens[s]), batch.width * batch.bs, limit or 1 << 30)
    at = [(i, w) for i in range(max(0, n)) if (w := where(batch, shared, s, i)) is not None]
    pos = np.array([i for i, _ in at], np.int64)
    b, slot = (np.array([w[j] for _, w in at], np.int64) for j in (0, 1))
    out = []
    for p in pools:
        if kind != "i8":
            out.append(p[b, :, slot].astype(np.float64))
            continue
        bs = batch.bs
        lane = slot[:, None] * dim + np.arange(dim)
        q = np.ascontiguousarray(p[b[:, None], :, lane].transpose(0, 2, 1)).view(np.int8).astype(np.float64)
        lane = bs * dim + slot[:, None] * (dim // 16) + np.arange(dim // 16)
        d = np.ascontiguousarray(p[b[:, None], :, lane].transpose(0, 2, 1)).view(np.float16).astype(np.float64)
        x = (q.reshape(len(at), p.shape[1], dim // 32, 32) * d[..., None]).reshape(len(at), p.shape[1], dim)
        with np.errstate(over="ignore"):
            out.append(x.astype(np.float16).astype(np.float64) if act == "f16" else x)
    return pos, out


def scores(batch, shared, s, kind, dim, heads, n_kv, pools, q, act, limit=None):
    """For each head: (head, KV head, positions, scores [rows, positions] with -inf where a row does not look, bound on a
    score's error [rows], values)."""
    pos, held = cells(batch, shared, s, kind, dim, pools, limit, act)
    a, e = int(batch.starts[s]), int(batch.starts[s + 1])
    last = int(batch.lens[s]) - (e - a) + np.arange(e - a)
    for h in range(heads):
        g = h * n_kv // heads
        x, k = q[a:e, h].astype(np.float64), held[0][:, g]
        with np.errstate(all="ignore"):
            sc = x @ k.T / np.sqrt(dim)
            sees = pos[None, :] <= last[:, None]
            size = np.where(sees, np.abs(x) @ np.abs(k).T / np.sqrt(dim), 0.0)
            # dim products and sums in 32 bits, the scale, the argument of the base-2 exponent
            ds = (dim + 8) * U * (size.max(1) if len(pos) else np.zeros(e - a))
        yield h, g, pos, np.where(sees, sc, -np.inf), ds, held[1][:, g] if len(held) > 1 else None


def attention(batch, shared, kind, dim, heads, n_kv, pools, q, act, limit=None):
    """(output, bound, log-sum-exp, bound); rows of no sequence are NaN."""
    out, err = np.full((batch.rows, heads, dim), np.nan), np.zeros((batch.rows, heads, dim))
    lse, lerr = np.full((batch.rows, heads), np.nan), np.zeros((batch.rows, heads))
    for s in range(len(batch.seqs)):
        a, e = int(batch.starts[s]), int(batch.starts[s + 1])
        if e <= a:
            continue
        for h, _, pos, sc, ds, vals in scores(batch, shared, s, kind, dim, heads, n_kv, pools, q, act, limit):
            with np.errstate(all="ignore"):
                m = sc.max(1) if len(pos) else np.full(e - a, -np.inf)
                w = np.where(np.isneginf(sc), 0.0, np.exp(sc - np.where(np.isneginf(m), 0.0, m)[:, None]))
                total = w.sum(1)
                none = total == 0
                if np.isfinite(vals).all():
                    o = w @ vals
                else:  # a row has nothing of the keys that it does not see
                    o = np.stack([w[i][w[i] != 0] @ vals[w[i] != 0] for i in range(e - a)])
                o = o / np.where(none, 1.0, total)[:, None] if len(pos) else np.zeros((e - a, dim))
                z = np.where(none, -np.inf, m + np.log(np.where(none, 1.0, total)))
                top = np.array([np.abs(vals[w[i] > 0]).max(initial=0.0) for i in range(e - a)])
                # weights off by exp(ds), sums over the keys; f16: weights and the output rounded to f16
                off = 2 * np.expm1(ds) + 2 * (len(pos) + 16) * U + (H if act == "f16" else 0.0)
                out[a:e, h] = o
                err[a:e, h] = (1.01 * off * top)[:, None] + (H * np.abs(o) + 2.0 ** -25 if act == "f16" else U * np.abs(o))
                lse[a:e, h] = z
                # scores off by ds, the sum by its additions, (m + log2 l) ln 2 by the rounding of its parts
                lerr[a:e, h] = np.where(none, 0.0, ds + (len(pos) + 16) * U + 6 * U * (np.abs(m) + np.abs(z) + 1))
    return out, err, lse, lerr


def weights(batch, kind, dim, heads, n_kv, pool, q, act, lse, held, theta, was, limit=None):
    """(weights [sequence, kv, width], bound): `was` where nothing is written."""
    out, err = was.astype(np.float64), np.zeros(was.shape)
    for s in range(len(batch.seqs)):
        a, e = int(batch.starts[s]), int(batch.starts[s + 1])
        n = min(int(batch.lens[s]), batch.width * batch.bs, limit or 1 << 30)
        if e <= a or n <= 0:
            continue
        old = max(0, min(n, int(batch.lens[s]) - (e - a)))
        out[s, :, :n] = 0.0
        if theta:
            out[s, :, :old] = np.float64(np.float32(theta)) * held[s, :, :old]
        err[s, :, :n] = 2 * U * np.abs(out[s, :, :n])
        for h, g, pos, sc, ds, _ in scores(batch, None, s, kind, dim, heads, n_kv, [pool], q, act, limit):
            by = lse[a:e, h].astype(np.float64)
            with np.errstate(all="ignore"):
                w = np.where(np.isneginf(sc) | np.isneginf(by)[:, None], 0.0, np.exp(sc - by[:, None]))
                # the score off by ds, the exponent's argument by the rounding of its parts; then the sum of the rows
                arg = ds + 4 * U * (np.abs(np.where(np.isfinite(sc), sc, 0)).max(1, initial=0) + np.abs(np.where(np.isfinite(by), by, 0)))
                e1 = w * (np.expm1(1.01 * arg) + 8 * U)[:, None]
                out[s, g, pos] += w.sum(0)
                err[s, g, pos] += e1.sum(0) + ((e - a) * heads // n_kv + 16) * U * w.sum(0)
        err[s, :, :n] += 2 * U * np.abs(out[s, :, :n])
    return out, err


def evict(batch, lens, weights, budget, top, limit=None):
    """[sequence] of (kept positions [kv, k])."""
    out = []
    n_kv = weights.shape[1]
    for s in range(len(lens)):
        n = max(0, min(int(lens[s]), batch.width * batch.bs, limit or 1 << 30))
        k = max(0, min(int(budget[s][0]), n, top))
        r = max(0, min(int(budget[s][1]), k))
        rows = np.zeros((n_kv, k), np.int64)
        none = np.array([batch.where(s, i) is None for i in range(n - r)], bool)
        for g in range(n_kv):
            w = weights[s, g, :n - r].astype(np.float64)
            # by class (storage and a number above), weight, then position
            low = none | np.isnan(w)
            order = np.lexsort((np.arange(n - r), -np.where(low, 0.0, w), low))
            rows[g] = np.sort(np.concatenate([order[:k - r], np.arange(n - r, n)]))
        out.append(rows)
    return out


def move(batch, kind, dim, pools, to_pools, kept, new_table):
    """Rows of the kept positions into the second pools, in place."""
    bs = batch.bs
    for s, rows in enumerate(kept):
        for g in range(len(rows)):
            for i, p in enumerate(rows[g]):
                t = int(new_table[s, i // bs])
                if t >= len(to_pools[0]):
                    continue
                w = batch.where(s, int(p))
                for src, dst in zip(pools, to_pools):
                    if kind != "i8":
                        dst[t, g, i % bs] = src[w[0], g, w[1]] if w else 0
                        continue
                    a, c = (i % bs) * dim, bs * dim + (i % bs) * dim // 16
                    dst[t, g, a:a + dim] = src[w[0], g, w[1] * dim:(w[1] + 1) * dim] if w else 0
                    x = bs * dim + (w[1] * dim // 16 if w else 0)
                    dst[t, g, c:c + dim // 16] = src[w[0], g, x:x + dim // 16] if w else 0


__all__ = ["Batch", "NONE", "Shared", "attention", "evict", "move", "weights", "where"]
