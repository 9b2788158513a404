"""The ops on a paged cache on the GPU: paged_kv_append, paged_kv_gather and
flash_attention_paged_chunk against their plain 64-bit forms (paged_ref.py).

Written and read values are bit-exact: an append copies, or rounds by a rule
that has one answer; a gather copies, or rounds code * scale once.  Attention
is held to the bound that paged_ref.attention derives for each row.  Every
place of the pools that no position of the batch names holds NaN and infinities.
"""
import numpy as np
import pytest

import paged_ref as ref
from neurofabric_amd import abi, hiprt
from neurofabric_amd.plugin import push_constants

pytestmark = [pytest.mark.gpu, pytest.mark.filterwarnings("ignore::RuntimeWarning")]

NP = {"f32": np.float32, "f16": np.float16}
NF = {"f32": abi.NF_DTYPE_F32, "f16": abi.NF_DTYPE_F16, "i8": abi.NF_DTYPE_I8}
ACT_POOL = [("f32", "f32"), ("f32", "i8"), ("f16", "f16"), ("f16", "i8")]


class Bufs:
    """Provider buffers that are released together."""

    def __init__(self, prov):
        self.prov, self.all = prov, []

    def __enter__(self):
        return self

    def __exit__(self, *_):
        self.prov.synchronize()
        for b in self.all:
            b.release()

    def put(self, a, dtype=None):
        dt = dtype if dtype is not None else {"f4": NF["f32"], "f2": NF["f16"], "u1": NF["i8"]}.get(
            a.dtype.str[1:], abi.NF_DTYPE_I32)
        b = self.prov.alloc(dt, max(a.nbytes, 4))
        if a.nbytes:
            b.write(a)
        self.all.append(b)
        return b

    def batch(self, b):
        return [self.put(b.table), self.put(b.starts), self.put(b.lens)]


def pc_of(batch, n_kv, dim, **more):
    return push_constants(M=n_kv, N=batch.width, K=len(batch.seqs), seq_len=batch.rows, head_dim=dim,
                          window_size=batch.bs, **more)


def rows_of(rng, act, n, kv, dim, scale=1.0):
    return (rng.standard_normal((n, kv, dim)) * scale).astype(NP[act])


def check(got, want, err, what):
    got = got.astype(np.float64)
    bad = ~(np.abs(got - want) <= err)
    assert not bad.any(), (what, int(bad.sum()), np.argwhere(bad)[:3].tolist(), got[bad][:3], want[bad][:3],
                           np.broadcast_to(err, got.shape)[bad][:3])


# ---- append and gather ----------------------------------------------------------

SHAPES = [  # sequences (positions, rows), KV heads, head_dim, block size
    ([(1, 1)], 1, 32, 1),
    ([(5, 5), (17, 1), (16, 16), (33, 7)], 2, 64, 16),
    ([(40, 3), (0, 0), (9, 9), (1, 1)], 4, 128, 8),
    ([(100, 64), (31, 31)], 8, 96, 32),
    ([(23, 11)], 3, 256, 5),
    ([(3, 1)] * 70, 1, 64, 2),
    ([(130, 130), (77, 76)], 8, 128, 16),
]


@pytest.mark.parametrize("act,pool", ACT_POOL)
@pytest.mark.parametrize("seqs,kv,dim,bs", SHAPES)
def test_append_and_gather(provider, act, pool, seqs, kv, dim, bs):
    rng = np.random.default_rng(len(seqs) * 1000 + dim)
    batch = ref.Batch(rng, seqs, bs, behind=3, before=2)
    pools = [ref.empty_pool(rng, pool, batch.blocks, kv, bs, dim, garbage=True) for _ in range(2)]
    rows = [rows_of(rng, act, batch.rows, kv, dim, s) for s in (1.0, 30.0)]
    rows[0][0] = 0.0
    rows[0][-4 if batch.rows > 4 else 0] = 0.0  # an all-zero group: scale 0
    was = [rows_of(rng, act, batch.rows, kv, dim) for _ in range(2)]
    with Bufs(provider) as m:
        desc = m.batch(batch)
        kb = [m.put(p) for p in pools]
        out = [m.put(w) for w in was]
        pc = pc_of(batch, kv, dim)
        provider.dispatch("paged_kv_append", [m.put(r) for r in rows] + desc, kb, pc=pc)
        provider.dispatch("paged_kv_gather", kb + desc, out, pc=pc)
        got = [b.read(np.uint8, p.nbytes).reshape(p.view(np.uint8).shape) for b, p in zip(kb, pools)]
        back = [b.read(NP[act], w.size).reshape(w.shape) for b, w in zip(out, was)]
    ref.append(batch, pool, dim, pools, rows)
    for g, p in zip(got, pools):
        assert np.array_equal(g, p.view(np.uint8))  # what no row names stays as it was
    for j in range(2):
        for r, s, pos in batch.each():
            was[j][r] = ref.load(pools[j], pool, bs, dim, batch.where(s, pos)).astype(NP[act])
        assert np.array_equal(back[j].view(np.uint8), was[j].view(np.uint8))


@pytest.mark.parametrize("act", ["f32", "f16"])
def test_append_rounds_next_to_borders(provider, act):
    """Values on, and one step beside, the borders between codes; subnormal and tiny scales; saturation, NaN, infinities."""
    rng = np.random.default_rng(7)
    groups = []
    for top in (1.0, 127.0, 100.3, 3e-5, 6e-6, 1e-7, 0.9, 60000.0):
        d = np.float16(np.float32(np.float16(top) if act == "f16" else np.float32(top)) / np.float32(127))
        k = rng.integers(-126, 126, 31) + 0.5
        x = (k * np.float64(d)).astype(NP[act])
        for step in (0, 1, -1):
            y = x.copy()
            for _ in range(abs(step)):
                y = np.nextafter(y, NP[act](step * np.inf))
            groups.append(np.concatenate([[NP[act](top)], np.clip(y, -top, top)]).astype(NP[act]))
    x = np.stack(groups).reshape(len(groups), 1, 32)
    batch = ref.Batch(rng, [(len(x), len(x))], 4)
    pools = [ref.empty_pool(rng, "i8", batch.blocks, 1, 4, 32) for _ in range(2)]
    special = x.copy()
    special[0, 0, 3] = np.nan
    special[1, 0, 4], special[1, 0, 5] = np.inf, -np.inf
    if act == "f32":
        special[2, 0, 6], special[2, 0, 7] = 3e38, -1e7
    with Bufs(provider) as m:
        kb = [m.put(p) for p in pools]
        provider.dispatch("paged_kv_append", [m.put(x), m.put(special)] + m.batch(batch), kb, pc=pc_of(batch, 1, 32))
        got = [b.read(np.uint8, p.nbytes).reshape(p.shape) for b, p in zip(kb, pools)]
    ref.append(batch, "i8", 32, pools[:1], [x])
    assert np.array_equal(got[0], pools[0])
    vals = [ref.load(got[1], "i8", 4, 32, batch.where(0, i))[0] for i in range(3)]
    clean = [ref.load(got[0], "i8", 4, 32, batch.where(0, i))[0] for i in range(3)]
    assert vals[0][3] == 0.0 and np.array_equal(np.delete(vals[0], 3), np.delete(clean[0], 3))
    assert vals[1][4] == 127 * 65504.0 and vals[1][5] == -127 * 65504.0
    if act == "f32":
        assert vals[2][6] == 127 * 65504.0 and vals[2][7] == -127 * 65504.0


def test_append_skips_what_has_no_storage(provider):
    """Positions below zero, past the table, past max_seq_len, and blocks past the pools: nothing is written; a gather gives zeros."""
    rng = np.random.default_rng(9)
    kv, dim, bs = 2, 64, 4
    batch = ref.Batch(rng, [(3, 3), (8, 8), (6, 6)], bs)
    batch.starts = np.array([0, 5, 13, 19], np.int32)  # five rows for three positions
    batch.rows = 19
    batch.table[1, 1] = batch.blocks + 5
    batch.table[2, 0] = 0x7FFFFFFF
    pools = [ref.empty_pool(rng, "f16", batch.blocks, kv, bs, dim) for _ in range(2)]
    rows = [rows_of(rng, "f16", batch.rows, kv, dim) for _ in range(2)]
    out = [np.ones_like(r) for r in rows]
    limit = 6
    with Bufs(provider) as m:
        desc, kb = m.batch(batch), [m.put(p) for p in pools]
        ob = [m.put(o) for o in out]
        pc = pc_of(batch, kv, dim, max_seq_len=limit)
        provider.dispatch("paged_kv_append", [m.put(r) for r in rows] + desc, kb, pc=pc)
        provider.dispatch("paged_kv_gather", kb + desc, ob, pc=pc)
        got = [b.read(np.float16, p.size).reshape(p.shape) for b, p in zip(kb, pools)]
        back = [b.read(np.float16, o.size).reshape(o.shape) for b, o in zip(ob, out)]
    ref.append(batch, "f16", dim, pools, rows, limit)
    for j in range(2):
        assert np.array_equal(got[j], pools[j])
        for r, s, pos in batch.each():
            w = batch.where(s, pos) if pos < limit else None
            assert np.array_equal(back[j][r], rows[j][r] if w else np.zeros((kv, dim), np.float16)), (r, s, pos)


def test_no_rows_or_sequences(provider):
    """Empty batches leave everything as it was."""
    rng = np.random.default_rng(1)
    for seqs in ([], [(5, 0), (0, 0)]):
        batch = ref.Batch(rng, seqs, 16, spare=2, behind=2)
        pool = ref.empty_pool(rng, "f32", batch.blocks, 2, 16, 64)
        x = rows_of(rng, "f32", batch.rows, 2, 64)
        with Bufs(provider) as m:
            desc, kb, xb = m.batch(batch), [m.put(pool), m.put(pool)], [m.put(x), m.put(x)]
            out = [m.put(x), m.put(x)]
            for rows in (batch.rows, 0):
                pc = push_constants(M=2, N=batch.width, K=len(seqs), seq_len=rows, head_dim=64, window_size=16, n_heads=2)
                provider.dispatch("paged_kv_append", xb + desc, kb, pc=pc)
                provider.dispatch("paged_kv_gather", kb + desc, out, pc=pc)
                provider.dispatch("flash_attention_paged_chunk", xb[:1] + kb + desc, out[:1], pc=pc)
            assert np.array_equal(kb[0].read(np.float32), pool.ravel()) and np.array_equal(kb[1].read(np.float32), pool.ravel())
            assert np.array_equal(out[0].read(np.float32), x.ravel()) and np.array_equal(out[1].read(np.float32), x.ravel())


# ---- attention ------------------------------------------------------------------

def run_attention(provider, rng, batch, act, pool, heads, kv, dim, scale=1.0, max_seq_len=0, edit=None, q_scale=1.0):
    """(got, want, bound, what the output held before)."""
    pools = [ref.empty_pool(rng, pool, batch.blocks, kv, batch.bs, dim, garbage=True) for _ in range(2)]
    for s, (n, _) in enumerate(batch.seqs):
        for pos in range(n):
            w = batch.where(s, pos)
            if w:
                for p in pools:
                    ref.store(p, pool, batch.bs, dim, w, (rng.standard_normal((kv, dim)) * scale).astype(NP[act]))
    if edit:
        edit(pools)
    q = rows_of(rng, act, batch.rows, heads, dim, q_scale)
    was = np.full_like(q, 7.5)
    with Bufs(provider) as m:
        out = m.put(was)
        provider.dispatch("flash_attention_paged_chunk", [m.put(q)] + [m.put(p) for p in pools] + m.batch(batch), [out],
                          pc=pc_of(batch, kv, dim, n_heads=heads, max_seq_len=max_seq_len))
        got = out.read(NP[act], q.size).reshape(q.shape)
    want, err = ref.attention(batch, pool, dim, heads, kv, pools, q, act, max_seq_len or None)
    return got, want, err, was


def check_attention(provider, rng, batch, act, pool, heads, kv, dim, **more):
    got, want, err, was = run_attention(provider, rng, batch, act, pool, heads, kv, dim, **more)
    mine = np.zeros(batch.rows, bool)
    for r, _, _ in batch.each():
        mine[r] = True
    check(got[mine], want[mine], err[mine], (act, pool, heads, kv, dim, batch.seqs))
    assert np.array_equal(got[~mine], was[~mine])


ATTENTION = [  # sequences (positions, rows), heads, KV heads, head_dim, block size
    ([(1, 1)], 1, 1, 64, 16),
    ([(1, 1), (2, 2), (300, 1)], 4, 4, 128, 16),
    ([(61, 1)], 32, 4, 64, 16),
    ([(700, 1), (3, 1), (129, 1), (256, 1)], 8, 1, 128, 16),
    ([(97, 5), (40, 2), (0, 0), (333, 4)], 8, 2, 64, 8),
    ([(200, 200)], 2, 1, 128, 16),
    ([(150, 70), (65, 64), (129, 1)], 6, 2, 64, 32),
    ([(260, 131)], 4, 4, 128, 4),
    ([(90, 33), (20, 20)], 6, 4, 64, 16),      # heads that do not divide evenly
    ([(90, 33), (20, 20)], 10, 1, 96, 16),
    ([(70, 9)], 16, 1, 128, 16),
    ([(70, 9), (64, 64)], 24, 1, 64, 64),
    ([(50, 50)], 3, 3, 256, 7),
    ([(50, 20)], 4, 2, 32, 3),
    ([(500, 3)] * 3, 8, 8, 96, 16),
]


@pytest.mark.parametrize("act,pool", ACT_POOL)
@pytest.mark.parametrize("seqs,heads,kv,dim,bs", ATTENTION)
def test_attention(provider, act, pool, seqs, heads, kv, dim, bs):
    rng = np.random.default_rng(heads * 100 + dim + len(seqs))
    batch = ref.Batch(rng, seqs, bs, behind=2, before=1)
    check_attention(provider, rng, batch, act, pool, heads, kv, dim)


MORE = [  # block sizes beside powers of two, KV heads beside divisors of 8, many sequences, few and many splits of the keys
    ([(200, 150), (90, 3)], 10, 5, 128, 48),
    ([(200, 150), (90, 3)], 6, 3, 64, 80),
    ([(300, 140)], 6, 6, 128, 128),
    ([(300, 140)], 16, 16, 64, 16),
    ([(130, 129), (40, 1)], 6, 3, 96, 8),
    ([(130, 129), (40, 1), (9, 9)], 8, 2, 96, 64),
    ([(i % 40 + 1, 1) for i in range(150)], 4, 2, 64, 16),
    ([(i + 5, i % 5) for i in range(80)] + [(200, 190)], 8, 2, 128, 16),
    ([(600 + 7 * i, 1) for i in range(20)], 4, 4, 64, 16),
    ([(1500, 2), (700, 3), (40, 1)], 32, 8, 128, 32),
    ([(1200, 120)], 2, 2, 128, 16),
    ([(256, 256)], 1, 1, 64, 16),
    ([(64, 1), (65, 1), (63, 1), (128, 32), (32, 32)], 1, 1, 128, 16),
]


@pytest.mark.parametrize("act,pool", ACT_POOL)
@pytest.mark.parametrize("seqs,heads,kv,dim,bs", MORE)
def test_attention_more(provider, act, pool, seqs, heads, kv, dim, bs):
    rng = np.random.default_rng(heads * 100 + dim + len(seqs) + bs)
    batch = ref.Batch(rng, seqs, bs, width=3, behind=1)
    check_attention(provider, rng, batch, act, pool, heads, kv, dim)


@pytest.mark.parametrize("act,pool", ACT_POOL)
@pytest.mark.parametrize("dim,bs", [(64, 16), (128, 24)])
def test_rows_of_no_sequence(provider, act, pool, dim, bs):
    """Starts below zero, past the rows, or decreasing make no sequence; lengths below zero or past the table no keys: the
    other sequences come out as they are, and no other row is touched."""
    rng = np.random.default_rng(21)
    heads, kv = 4, 2
    good = ref.Batch(rng, [(150, 60), (40, 2), (33, 33)], bs, behind=4)
    bad = ref.Batch(rng, [(10, 1)] * 7, bs)
    bad.blocks, bad.width = good.blocks, good.width
    bad.table = np.full((7, good.width), ref.NONE, np.uint32)
    bad.table[1], bad.table[3], bad.table[5] = good.table
    bad.starts = np.array([-5, 0, 60, 60, 62, 62, 95, 1 << 30], np.int32)
    bad.lens = np.array([100, 150, 3, 40, -7, 33, 1000], np.int32)
    bad.rows = good.rows
    pools = [ref.empty_pool(rng, pool, good.blocks, kv, bs, dim) for _ in range(2)]
    q, was = rows_of(rng, act, good.rows, heads, dim), np.full((good.rows, heads, dim), 3.25, NP[act])
    x = [rows_of(rng, act, good.rows, kv, dim) for _ in range(2)]
    with Bufs(provider) as m:
        kb, out, desc = [m.put(p) for p in pools], m.put(was), m.batch(bad)
        pc = pc_of(bad, kv, dim, n_heads=heads)
        provider.dispatch("paged_kv_append", [m.put(r) for r in x] + desc, kb, pc=pc)
        provider.dispatch("flash_attention_paged_chunk", [m.put(q)] + kb + desc, [out], pc=pc)
        got = out.read(NP[act], q.size).reshape(q.shape)
        held = [b.read(np.uint8, p.nbytes) for b, p in zip(kb, pools)]
        # decreasing starts, far lengths: nothing but ends in time
        wild = [m.put(bad.table), m.put(np.array([90, 80, 5, 70, 2, 2, 1, 0], np.int32)),
                m.put(np.array([2 ** 31 - 1, -2 ** 31, 2 ** 31 - 1, 7, 9, 2 ** 31 - 1, 0], np.int32))]
        provider.dispatch("flash_attention_paged_chunk", [m.put(q)] + kb + wild, [m.put(was)], pc=pc)
        provider.synchronize()
    ref.append(good, pool, dim, pools, x)
    for h, p in zip(held, pools):
        assert np.array_equal(h, p.reshape(-1).view(np.uint8))
    want, err = ref.attention(good, pool, dim, heads, kv, pools, q, act)
    mine = np.zeros(good.rows, bool)
    mine[:95] = True
    check(got[mine], want[mine], err[mine], (act, pool))
    assert np.array_equal(got[~mine], was[~mine])


@pytest.mark.parametrize("act,dim", [("f32", 40), ("f16", 40), ("f32", 33), ("f16", 1), ("f32", 200)])
def test_attention_odd_head_dims(provider, act, dim):
    rng = np.random.default_rng(dim)
    batch = ref.Batch(rng, [(77, 30), (5, 1)], 16)
    check_attention(provider, rng, batch, act, act, 4, 2, dim)


@pytest.mark.parametrize("act,pool", ACT_POOL)
def test_attention_long_context(provider, act, pool):
    """Keys split over many workgroups; sequences much shorter than the longest; a bound of max_seq_len above all."""
    rng = np.random.default_rng(5)
    batch = ref.Batch(rng, [(5000, 1), (17, 1), (1, 1), (2049, 1)], 16)
    check_attention(provider, rng, batch, act, pool, 4, 1, 64, max_seq_len=6000)
    batch = ref.Batch(rng, [(3000, 40)], 16)
    check_attention(provider, rng, batch, act, pool, 4, 2, 128)


@pytest.mark.parametrize("act,pool", ACT_POOL)
@pytest.mark.parametrize("dim", [64, 128])
def test_attention_large_scores(provider, act, pool, dim):
    """Weights that underflow and maxima that grow along the keys."""
    rng = np.random.default_rng(6)
    batch = ref.Batch(rng, [(400, 3), (130, 130)], 16)

    def edit(pools):
        for pos in range(400):
            b, slot = batch.where(0, pos)
            rows = (rng.standard_normal((2, dim)) * (0.02 * pos)).astype(NP[act])
            ref.store(pools[0], pool, 16, dim, (b, slot), rows)
    check_attention(provider, rng, batch, act, pool, 4, 2, dim, edit=edit, q_scale=2.0)


@pytest.mark.parametrize("act,pool", ACT_POOL)
@pytest.mark.parametrize("dim", [64, 128, 96])
def test_attention_rows_and_blocks_without_keys(provider, act, pool, dim):
    """More rows than positions, holes in the tables, a whole sequence without blocks, and positions past max_seq_len."""
    rng = np.random.default_rng(8)
    batch = ref.Batch(rng, [(3, 6), (100, 40), (40, 40), (200, 2)], 16)
    batch.table[1, 0] = ref.NONE
    batch.table[1, 3] = batch.blocks
    batch.table[2] = ref.NONE
    batch.table[3, 1:12] = ref.NONE
    check_attention(provider, rng, batch, act, pool, 8, 2, dim)
    check_attention(provider, rng, batch, act, pool, 8, 2, dim, max_seq_len=70)
    batch.table[:] = ref.NONE
    check_attention(provider, rng, batch, act, pool, 8, 2, dim)


@pytest.mark.parametrize("act,pool", ACT_POOL)
@pytest.mark.parametrize("dim", [64, 128, 96])
@pytest.mark.parametrize("rows", [3, 90])
def test_attention_masked_values_are_not_finite(provider, act, pool, dim, rows):
    """Keys and values of later rows of a chunk are NaN or infinite: earlier rows do not see them, the later ones do."""
    rng = np.random.default_rng(10)
    n = 150
    batch = ref.Batch(rng, [(n, rows), (64, 2)], 16)

    def edit(pools):
        for j, (pos, x) in enumerate([(n - 1, np.nan), (n - 2, np.inf)]):
            b, slot = batch.where(0, pos)
            for p in pools[1:] if j else pools:
                if pool == "i8":
                    at = 16 * dim + slot * dim // 16
                    p[b, :, at:at + dim // 16] = np.full((1, dim // 32), x, np.float16).view(np.uint8)
                else:
                    p[b, :, slot] = x
    got, want, err, _ = run_attention(provider, rng, batch, act, pool, 4, 2, dim, edit=edit)
    assert np.isnan(got[rows - 1]).all()
    assert not np.isfinite(got[rows - 2]).any()
    sound = [r for r in range(batch.rows) if r not in (rows - 1, rows - 2)]
    check(got[sound], want[sound], err[sound], (act, pool, dim))


@pytest.mark.parametrize("act,pool", ACT_POOL)
def test_attention_misaligned(provider, act, pool):
    """Imported operands at odd multiples of their element size."""
    import torch
    rng = np.random.default_rng(11)
    heads, kv, dim, bs = 4, 2, 64, 16
    batch = ref.Batch(rng, [(70, 70), (33, 1)], bs)
    pools = [ref.empty_pool(rng, pool, batch.blocks, kv, bs, dim) for _ in range(2)]
    rows = [rows_of(rng, act, batch.rows, kv, dim) for _ in range(2)]
    q = rows_of(rng, act, batch.rows, heads, dim)
    el = {"f32": 4, "f16": 2}[act]
    pel = 2 if pool == "i8" else el
    keep = []
    with Bufs(provider) as m:
        def odd(a, elt):
            t = torch.zeros(a.nbytes + 64, dtype=torch.uint8, device="cuda")
            t[elt:elt + a.nbytes] = torch.from_numpy(a.reshape(-1).view(np.uint8).copy()).cuda()
            keep.append(t)
            dt = {"f4": NF["f32"], "f2": NF["f16"], "u1": NF["i8"]}[a.dtype.str[1:]]
            import ctypes as C
            from neurofabric_amd import plugin
            desc, ops, h = abi.make_desc(dt, a.nbytes), abi.nf_buffer_ops(), C.c_void_p()
            provider.check(provider.mem.import_buffer(provider.handle, t.data_ptr() + elt, abi.NF_MEM_DOMAIN_DEVICE,
                                                      C.byref(desc), C.byref(ops), C.byref(h)), "import")
            m.all.append(plugin.Buffer(provider, h.value, ops, dt, a.nbytes))
            return m.all[-1]
        kb = [odd(p, pel) for p in pools]
        xb = [odd(r, el) for r in rows]
        qb, out = odd(q, el), odd(np.zeros_like(q), el)
        back = [odd(np.zeros_like(r), el) for r in rows]
        torch.cuda.synchronize()
        desc = m.batch(batch)
        pc = pc_of(batch, kv, dim, n_heads=heads)
        provider.dispatch("paged_kv_append", xb + desc, kb, pc=pc)
        provider.dispatch("paged_kv_gather", kb + desc, back, pc=pc)
        provider.dispatch("flash_attention_paged_chunk", [qb] + kb + desc, [out], pc=pc)
        got = out.read(NP[act], q.size).reshape(q.shape)
        gb = [b.read(NP[act], r.size).reshape(r.shape) for b, r in zip(back, rows)]
    ref.append(batch, pool, dim, pools, rows)
    for j in range(2):
        for r, s, pos in batch.each():
            assert np.array_equal(gb[j][r], ref.load(pools[j], pool, bs, dim, batch.where(s, pos)).astype(NP[act]))
    want, err = ref.attention(batch, pool, dim, heads, kv, pools, q, act)
    check(got, want, err, (act, pool))


@pytest.mark.parametrize("act,pool", [("f16", "f16"), ("f16", "i8")])
def test_offsets_past_32_bits(provider, act, pool):
    """The blocks that are used lie past 2^32 bytes and elements of the pools."""
    rng = np.random.default_rng(12)
    heads, kv, dim, bs = 8, 8, 128, 16
    page = ref.empty_pool(rng, pool, 1, 1, bs, dim).nbytes * kv
    blocks = (9 << 30) // page
    batch = ref.Batch(rng, [(40, 33)], bs)
    first = blocks - batch.blocks
    small = [ref.empty_pool(rng, pool, batch.blocks, kv, bs, dim) for _ in range(2)]
    rows = [rows_of(rng, act, batch.rows, kv, dim) for _ in range(2)]
    q = rows_of(rng, act, batch.rows, heads, dim)
    with Bufs(provider) as m:
        big = [provider.alloc(NF[pool], blocks * page) for _ in range(2)]
        m.all += big
        for b, p in zip(big, small):
            b.write(p, offset=first * page)
        at = ref.Batch(rng, batch.seqs, bs)
        at.table = np.where(batch.table == ref.NONE, batch.table, batch.table + np.uint32(first)).astype(np.uint32)
        desc = m.batch(at)
        pc = pc_of(batch, kv, dim, n_heads=heads)
        out = [m.put(np.zeros_like(q)), m.put(np.zeros_like(rows[0])), m.put(np.zeros_like(rows[0]))]
        provider.dispatch("paged_kv_append", [m.put(r) for r in rows] + desc, big, pc=pc)
        provider.dispatch("paged_kv_gather", big + desc, out[1:], pc=pc)
        provider.dispatch("flash_attention_paged_chunk", [m.put(q)] + big + desc, out[:1], pc=pc)
        got = [o.read(np.float16, a.size).reshape(a.shape) for o, a in zip(out, (q, rows[0], rows[0]))]
    ref.append(batch, pool, dim, small, rows)
    for j in range(2):
        for r, s, pos in batch.each():
            assert np.array_equal(got[1 + j][r], ref.load(small[j], pool, bs, dim, batch.where(s, pos)).astype(NP[act]))
    want, err = ref.attention(batch, pool, dim, heads, kv, small, q, act)
    check(got[0], want, err, pool)


# ---- a serving step ----------------------------------------------------------------

@pytest.mark.parametrize("act,pool", ACT_POOL)
def test_prefill_then_decode(provider, act, pool):
    """Chunks of a prompt, then single tokens, each appended and attended to in one run, as a model layer does; blocks are
    shared by two sequences with one prefix."""
    rng = np.random.default_rng(13)
    heads, kv, dim, bs = 8, 2, 64, 16
    total = 120
    whole = ref.Batch(rng, [(total, total), (total, total)], bs)
    whole.table[1, :3] = whole.table[0, :3]  # 48 positions in common
    pools = [ref.empty_pool(rng, pool, whole.blocks, kv, bs, dim, garbage=True) for _ in range(2)]
    shared = [rows_of(rng, act, 48, kv, dim) for _ in range(2)]
    done = [0, 48]
    with Bufs(provider) as m:
        kb = [m.put(p) for p in pools]
        for step in ([48, 0], [29, 1], [1, 40], [1, 1], [0, 1], [41, 28]):
            batch = ref.Batch(rng, [(done[i] + n, n) for i, n in enumerate(step)], bs)
            batch.table, batch.width, batch.blocks = whole.table, whole.width, whole.blocks
            rows = [rows_of(rng, act, batch.rows, kv, dim) for _ in range(2)]
            if step == [48, 0]:
                rows = shared
            q = rows_of(rng, act, batch.rows, heads, dim)
            desc, out = m.batch(batch), m.put(np.zeros_like(q))
            pc = pc_of(batch, kv, dim, n_heads=heads, max_seq_len=128)
            tasks = [provider.task("paged_kv_append", [m.put(r) for r in rows] + desc, kb, pc=pc),
                     provider.task("flash_attention_paged_chunk", [m.put(q)] + kb + desc, [out], pc=pc)]
            provider.run_tasks((abi.nf_task_desc * 2)(*tasks))
            got = out.read(NP[act], q.size).reshape(q.shape)
            ref.append(batch, pool, dim, pools, rows)
            want, err = ref.attention(batch, pool, dim, heads, kv, pools, q, act)
            check(got, want, err, (act, pool, step))
            done = [a + b for a, b in zip(done, step)]


@pytest.mark.parametrize("act,pool", [("f32", "f32"), ("f16", "i8")])
def test_captured_step_replays(provider, act, pool):
    """A captured step follows the lengths, tables and rows that its buffers hold at each replay."""
    rng = np.random.default_rng(14)
    heads, kv, dim, bs = 8, 2, 64, 16
    whole = ref.Batch(rng, [(300, 1), (300, 1), (300, 1)], bs)
    pools = [ref.empty_pool(rng, pool, whole.blocks, kv, bs, dim) for _ in range(2)]
    q = rows_of(rng, act, 3, heads, dim)
    with Bufs(provider) as m:
        kb, desc = [m.put(p) for p in pools], m.batch(whole)
        xb = [m.put(rows_of(rng, act, 3, kv, dim)) for _ in range(2)]
        qb, out = m.put(q), m.put(np.zeros_like(q))
        pc = pc_of(whole, kv, dim, n_heads=heads)
        tasks = (abi.nf_task_desc * 2)(provider.task("paged_kv_append", xb + desc, kb, pc=pc),
                                       provider.task("flash_attention_paged_chunk", [qb] + kb + desc, [out], pc=pc))
        graph = hiprt.Graph(provider.stream(), lambda: provider.run_tasks(tasks))
        for lens in ([300, 17, 1], [1, 300, 250], [64, 65, 66], [2, 2, 2]):
            rows = [rows_of(rng, act, 3, kv, dim) for _ in range(2)]
            batch = ref.Batch(rng, [(n, 1) for n in lens], bs)
            batch.table, batch.width, batch.blocks = whole.table, whole.width, whole.blocks
            desc[2].write(batch.lens)
            for b, r in zip(xb, rows):
                b.write(r)
            graph.launch()
            got = out.read(NP[act], q.size).reshape(q.shape)
            ref.append(batch, pool, dim, pools, rows)
            want, err = ref.attention(batch, pool, dim, heads, kv, pools, q, act)
            check(got, want, err, lens)
            provider.dispatch("flash_attention_paged_chunk", [qb] + kb + desc, [out], pc=pc)  # the eager call agrees
            assert np.array_equal(out.read(NP[act], q.size).reshape(q.shape), got)


def test_output_in_place_of_the_query(provider):
    """The output may be the query's own buffer."""
    rng = np.random.default_rng(15)
    for seqs, act, dim in (([(900, 1), (20, 1)], "f16", 128), ([(200, 90)], "f16", 64), ([(300, 30)], "f32", 64),
                           ([(100, 20)], "f16", 96)):
        batch = ref.Batch(rng, seqs, 16)
        pools = [ref.empty_pool(rng, act, batch.blocks, 2, 16, dim) for _ in range(2)]
        q = rows_of(rng, act, batch.rows, 8, dim)
        with Bufs(provider) as m:
            qb = m.put(q)
            provider.dispatch("flash_attention_paged_chunk", [qb] + [m.put(p) for p in pools] + m.batch(batch), [qb],
                              pc=pc_of(batch, 2, dim, n_heads=8))
            got = qb.read(NP[act], q.size).reshape(q.shape)
        want, err = ref.attention(batch, act, dim, 8, 2, pools, q, act)
        check(got, want, err, seqs)


def test_repeated_calls_give_the_same_bits(provider):
    rng = np.random.default_rng(16)
    batch = ref.Batch(rng, [(4000, 1), (100, 70), (31, 1)], 16)
    pools = [ref.empty_pool(rng, "i8", batch.blocks, 2, 16, 128) for _ in range(2)]
    q = rows_of(rng, "f16", batch.rows, 8, 128)
    with Bufs(provider) as m:
        args = [m.put(q)] + [m.put(p) for p in pools] + m.batch(batch)
        outs = [m.put(np.zeros_like(q)) for _ in range(6)]
        for o in outs:
            provider.dispatch("flash_attention_paged_chunk", args, [o], pc=pc_of(batch, 2, 128, n_heads=8))
        first = outs[0].read(np.uint16)
        assert all(np.array_equal(first, o.read(np.uint16)) for o in outs[1:])


MIDDLE = [  # around the counts of query rows at which another kernel takes the batch, alone and beside longer and shorter sequences
    ([(300, 16)], 8, 2, 128, 16),
    ([(300, 17)], 8, 2, 128, 16),
    ([(700, 24), (400, 24), (129, 24)], 4, 1, 128, 16),
    ([(700, 25), (400, 25), (129, 24)], 4, 1, 64, 24),
    ([(500, 64), (300, 96), (200, 32)], 1, 1, 128, 16),
    ([(520, 33), (300, 65), (200, 300), (90, 1)], 2, 2, 96, 16),
    ([(400, 21)] * 20, 3, 1, 64, 32),
]


@pytest.mark.parametrize("act,pool", ACT_POOL)
@pytest.mark.parametrize("seqs,heads,kv,dim,bs", MIDDLE)
def test_attention_between_kernels(provider, act, pool, seqs, heads, kv, dim, bs):
    rng = np.random.default_rng(heads * 100 + dim + len(seqs) + bs)
    batch = ref.Batch(rng, seqs, bs, width=2, behind=1)
    check_attention(provider, rng, batch, act, pool, heads, kv, dim)


@pytest.mark.parametrize("act,pool", ACT_POOL)
@pytest.mark.parametrize("dim", [64, 128, 96, 160])
@pytest.mark.parametrize("rows", [1, 12, 130])
def test_attention_scores_of_minus_infinity(provider, act, pool, dim, rows):
    """Keys that score -inf weigh nothing, as if they were not there, wherever they lie: in tiles and splits that hold
    nothing else, before finite keys and between them; a row with no other key gives zeros.  Elements of K are -inf, or
    (f32) finite with a product that is not."""
    rng = np.random.default_rng(dim + rows)
    heads, kv, bs = 4, 2, 16
    batch = ref.Batch(rng, [(600, rows), (200, min(rows, 70)), (400, 2), (7, 7)], bs)
    low = [range(320), range(200), range(64, 128), range(0)]
    pools = [ref.empty_pool(rng, pool, batch.blocks, kv, bs, dim) for _ in range(2)]
    q = rows_of(rng, act, batch.rows, heads, dim)
    q[..., :32] = np.abs(q[..., :32]) + NP[act](2)
    left = ref.Batch(rng, batch.seqs, bs)  # the same without those keys
    left.table = batch.table.copy()
    for s, positions in enumerate(low):
        for p in positions:
            b, slot = batch.where(s, p)
            if pool == "i8":
                pools[0][b, :, slot * dim:slot * dim + 32] = 0x81  # -127
                at = bs * dim + slot * dim // 16
                pools[0][b, :, at:at + 2] = np.full((1, 1), np.inf, np.float16).view(np.uint8)
            else:
                pools[0][b, 0, slot, :32] = -np.inf
                pools[0][b, 1, slot, :32] = -3e38 if pool == "f32" else -np.inf
            left.table[s, p // bs] = ref.NONE
    with Bufs(provider) as m:
        out = m.put(np.zeros_like(q))
        provider.dispatch("flash_attention_paged_chunk", [m.put(q)] + [m.put(p) for p in pools] + m.batch(batch), [out],
                          pc=pc_of(batch, kv, dim, n_heads=heads))
        got = out.read(NP[act], q.size).reshape(q.shape)
    want, err = ref.attention(left, pool, dim, heads, kv, pools, q, act)
    check(got, want, err, (act, pool, dim, rows))


@pytest.mark.parametrize("act,pool", ACT_POOL)
@pytest.mark.parametrize("rows", [1, 9, 300])
def test_append_of_one_slot_twice(provider, act, pool, rows):
    """What a slot holds that two rows of one append name is not defined; all other slots are as they would be."""
    rng = np.random.default_rng(rows)
    kv, dim, bs = 2, 64, 16
    batch = ref.Batch(rng, [(rows + 20, rows), (rows + 20, rows), (40, 5)], bs)
    last = (rows + 19) // bs
    batch.table[1, last] = batch.table[0, last]  # the last block of both
    pools = [ref.empty_pool(rng, pool, batch.blocks, kv, bs, dim) for _ in range(2)]
    x = [rows_of(rng, act, batch.rows, kv, dim) for _ in range(2)]
    with Bufs(provider) as m:
        kb = [m.put(p) for p in pools]
        provider.dispatch("paged_kv_append", [m.put(r) for r in x] + m.batch(batch), kb, pc=pc_of(batch, kv, dim))
        got = [b.read(np.uint8, p.nbytes).view(p.dtype).reshape(p.shape) for b, p in zip(kb, pools)]
    ref.append(batch, pool, dim, pools, x)
    shared = int(batch.table[0, last])
    first = max(20, bs * last) - bs * last  # the slots of that block that both write
    for g, p in zip(got, pools):
        for slot in range(first, (rows + 20) - bs * last):
            at = np.zeros(dim, np.float32)
            for a in (g, p):
                ref.store(a, pool, bs, dim, (shared, slot), np.broadcast_to(at, (kv, dim)))
        assert np.array_equal(g.view(np.uint8), p.view(np.uint8))


@pytest.mark.parametrize("dim", [64, 128, 96, 160])
@pytest.mark.parametrize("rows", [3, 150])
def test_largest_f16_values_in_an_i8_cache(provider, dim, rows):
    """Finite f16 rows stay finite in an I8 cache: read back within half a step of their scale (and the f16 rounding), and
    attended to, up to the largest value of the type."""
    rng = np.random.default_rng(dim + rows)
    heads, kv, bs = 4, 2, 16
    batch = ref.Batch(rng, [(rows, rows), (5, 5)], bs)
    x = [(rng.uniform(-6e4, 6e4, (batch.rows, kv, dim))).astype(np.float16) for _ in range(2)]
    for r in x:
        r[::2, :, 3::32] = 65504.0
        r[::2, :, 5::32] = -65504.0
        r[1::2, :, 7::32] = 65472.0
        r[0, :, :32] = [65504.0, -65504.0] * 16
    q = rows_of(rng, "f16", batch.rows, heads, dim, 1e-4)
    pools = [ref.empty_pool(rng, "i8", batch.blocks, kv, bs, dim) for _ in range(2)]
    with Bufs(provider) as m:
        kb, desc = [m.put(p) for p in pools], m.batch(batch)
        back, out = [m.put(np.zeros_like(r)) for r in x], m.put(np.zeros_like(q))
        pc = pc_of(batch, kv, dim, n_heads=heads)
        provider.dispatch("paged_kv_append", [m.put(r) for r in x] + desc, kb, pc=pc)
        provider.dispatch("paged_kv_gather", kb + desc, back, pc=pc)
        provider.dispatch("flash_attention_paged_chunk", [m.put(q)] + kb + desc, [out], pc=pc)
        held = [b.read(np.uint8, p.nbytes).reshape(p.shape) for b, p in zip(kb, pools)]
        got = [b.read(np.float16, r.size).reshape(r.shape) for b, r in zip(back, x)]
        o = out.read(np.float16, q.size).reshape(q.shape)
    for g, r in zip(got, x):
        top = np.abs(r.astype(np.float64)).reshape(batch.rows, kv, -1, 32).max(-1)
        # the scale is top / 127 within half a step of fp16; a code is off by half, and its product by half a step
        step = (top / 127 * (1 + 2.0 ** -11)).repeat(32, -1).reshape(r.shape)
        check(g, r.astype(np.float64), 0.5 * step + 2.0 ** -11 * 65504, (dim, rows))
    want, err = ref.attention(batch, "i8", dim, heads, kv, held, q, "f16")
    assert np.isfinite(want).all()
    check(o, want, err, (dim, rows))


MANY_ROWS = [  # rows around the count up to which they are spread over more waves, and past it; 16-byte pieces a row (f16, f32)
    ([(512, 512)], 0, 8, 128, 16),               # 128, 256
    ([(600, 507), (40, 1)], 5, 8, 128, 16),      # 513 rows in all
    ([(515, 515), (300, 290), (310, 300)], 2, 3, 96, 8),  # 36, 72
    ([(700, 650), (450, 450), (9, 3)], 1, 5, 256, 5),     # 160, 320
    ([(20, 9)] * 130, 3, 2, 32, 16),             # 8, 16; more sequences than a wave has lanes
]


@pytest.mark.parametrize("act,pool", ACT_POOL)
@pytest.mark.parametrize("seqs,behind,kv,dim,bs", MANY_ROWS)
def test_append_and_gather_many_rows(provider, act, pool, seqs, behind, kv, dim, bs):
    """As test_append_and_gather, for prompts: rows of no sequence, and blocks that are missing."""
    rng = np.random.default_rng(len(seqs) * 1000 + dim + behind)
    batch = ref.Batch(rng, seqs, bs, behind=behind)
    batch.table[0, 1] = ref.NONE
    batch.table[-1, 0] = batch.blocks
    pools = [ref.empty_pool(rng, pool, batch.blocks, kv, bs, dim, garbage=True) for _ in range(2)]
    rows = [rows_of(rng, act, batch.rows, kv, dim, s) for s in (1.0, 30.0)]
    was = [rows_of(rng, act, batch.rows, kv, dim) for _ in range(2)]
    with Bufs(provider) as m:
        desc = m.batch(batch)
        kb = [m.put(p) for p in pools]
        out = [m.put(w) for w in was]
        pc = pc_of(batch, kv, dim)
        provider.dispatch("paged_kv_append", [m.put(r) for r in rows] + desc, kb, pc=pc)
        provider.dispatch("paged_kv_gather", kb + desc, out, pc=pc)
        got = [b.read(np.uint8, p.nbytes).reshape(p.view(np.uint8).shape) for b, p in zip(kb, pools)]
        back = [b.read(NP[act], w.size).reshape(w.shape) for b, w in zip(out, was)]
    ref.append(batch, pool, dim, pools, rows)
    for g, p in zip(got, pools):
        assert np.array_equal(g, p.view(np.uint8))
    for j in range(2):
        for r, s, pos in batch.each():
            w = batch.where(s, pos)
            was[j][r] = ref.load(pools[j], pool, bs, dim, w).astype(NP[act]) if w else 0.0
        assert np.array_equal(back[j].view(np.uint8), was[j].view(np.uint8))


@pytest.mark.parametrize("act,pool", ACT_POOL)
def test_attention_more_splits_than_threads(provider, act, pool):
    """One head of one long sequence: its keys are split over more than 256 workgroups, whose partials one combines."""
    rng = np.random.default_rng(17)
    batch = ref.Batch(rng, [(40003, 1)], 16)
    check_attention(provider, rng, batch, act, pool, 1, 1, 64)


@pytest.mark.parametrize("kv,dim,bs", [(4, 64, 16), (2, 128, 8), (1, 96, 5)])
def test_flash_attention_paged_reads_the_cache(provider, kv, dim, bs):
    """An f32 cache written by paged_kv_append serves flash_attention_paged too: the last token of one sequence."""
    rng = np.random.default_rng(18)
    heads, n = 4, 77
    batch = ref.Batch(rng, [(n, n)], bs)
    pools = [ref.empty_pool(rng, "f32", batch.blocks, kv, bs, dim) for _ in range(2)]
    x = [rows_of(rng, "f32", n, kv, dim) for _ in range(2)]
    q = rows_of(rng, "f32", n, heads, dim)
    with Bufs(provider) as m:
        kb, desc = [m.put(p) for p in pools], m.batch(batch)
        provider.dispatch("paged_kv_append", [m.put(r) for r in x] + desc, kb, pc=pc_of(batch, kv, dim))
        out = m.put(np.zeros_like(q[-1:]))
        provider.dispatch("flash_attention_paged", [m.put(q[-1:])] + kb + desc[:1], [out],
                          pc=push_constants(seq_len=1, n_heads=heads, head_dim=dim, M=kv, N=batch.width, step_idx=n - 1,
                                            window_size=bs))
        got = out.read(np.float32, heads * dim).reshape(heads, dim)
    ref.append(batch, "f32", dim, pools, x)
    want = ref.attention(batch, "f32", dim, heads, kv, pools, q, "f32")[0][-1]
    check(got, want, 2e-5 * np.abs(want).max(), (kv, dim, bs))  # what that op's own test holds it to
