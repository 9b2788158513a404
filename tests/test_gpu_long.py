"""The operators for long contexts over the paged cache on the GPU, against their plain 64-bit forms (long_ref.py):
attention of sequences that share a prefix, the rows' log-sum-exp, gathered attention weights, and eviction by them.

Attention, log-sum-exp and weights are held to the bounds that long_ref derives; an eviction's choice and its moved rows are
equal.  Every place of the pools that no position of the batch names holds NaN and infinities.
"""
import numpy as np
import pytest

import long_ref as ref
import paged_ref
from neurofabric_amd import abi, hiprt
from neurofabric_amd.plugin import push_constants
from test_gpu_paged import ACT_POOL, NF, NP, Bufs, check, pc_of, rows_of

pytestmark = [pytest.mark.gpu, pytest.mark.filterwarnings("ignore::RuntimeWarning")]


def fill(rng, batch, shared, act, pool, kv, dim, scale=1.0):
    """Pools with values at the batch's positions, NaN and infinities elsewhere."""
    pools = [paged_ref.empty_pool(rng, pool, batch.blocks, kv, batch.bs, dim, garbage=True) for _ in range(2)]
    for s, (n, _) in enumerate(batch.seqs):
        at = sorted({w for i in range(n) if (w := ref.where(batch, shared, s, i)) is not None})
        for p in pools:
            x = (rng.standard_normal((max(1, len(at)), kv, dim)) * scale).astype(NP[act])
            for w, row in zip(at, x):
                paged_ref.store(p, pool, batch.bs, dim, w, row)
    return pools


def mine_of(batch):
    mine = np.zeros(batch.rows, bool)
    for r, _, _ in batch.each():
        mine[r] = True
    return mine


def run_attention(provider, rng, batch, shared, act, pool, heads, kv, dim, pools=None, max_seq_len=0, lse=True, q_scale=1.0,
                  chunk=False):
    """Checks output and log-sum-exp; (query, pools, log-sum-exp)."""
    pools = pools or fill(rng, batch, shared, act, pool, kv, dim)
    q = rows_of(rng, act, batch.rows, heads, dim, q_scale)
    was, wlse = np.full_like(q, 7.5), np.full((batch.rows, heads), -3.0, np.float32)
    with Bufs(provider) as m:
        out, lb = m.put(was), m.put(wlse)
        ins = [m.put(q)] + [m.put(p) for p in pools] + m.batch(batch)
        outs = [out, lb] if lse else [out]
        if chunk:
            pc = pc_of(batch, kv, dim, n_heads=heads, max_seq_len=max_seq_len)
            provider.dispatch("flash_attention_paged_chunk", ins, outs, pc=pc)
        else:
            pc = pc_of(batch, kv, dim, n_heads=heads, max_seq_len=max_seq_len, step_idx=len(shared.groups))
            provider.dispatch("flash_attention_paged_prefix", ins + [m.put(shared.first), m.put(shared.len)], outs, pc=pc)
        got, z = out.read(NP[act], q.size).reshape(q.shape), lb.read(np.float32, wlse.size).reshape(wlse.shape)
    want, err, wz, zerr = ref.attention(batch, shared, pool, dim, heads, kv, pools, q, act, max_seq_len or None)
    mine = mine_of(batch)
    what = (act, pool, heads, kv, dim, batch.seqs[:4], shared and shared.groups)
    check(got[mine], want[mine], err[mine], what)
    assert np.array_equal(got[~mine], was[~mine])
    if lse:
        none = np.isneginf(wz[mine])
        assert np.array_equal(np.isneginf(z[mine]), none)
        check(z[mine][~none], wz[mine][~none], zerr[mine][~none], ("lse",) + what)
        assert np.array_equal(z[~mine], wlse[~mine])
    else:
        assert np.array_equal(z, wlse)
    return q, pools, z


PREFIX = [  # sequences (positions, rows), groups (first, one past the last, shared positions), heads, KV heads, dim, block
    ([(1, 1)], [(0, 1, 1)], 1, 1, 64, 16),
    ([(40, 1), (33, 1), (50, 1)], [(0, 3, 32)], 8, 2, 128, 16),
    ([(40, 1), (33, 1), (50, 1)], [], 8, 2, 128, 16),
    ([(40, 5), (33, 1), (50, 9), (300, 2)], [(0, 2, 32), (2, 4, 17)], 8, 2, 64, 16),
    ([(200, 1)] * 20, [(0, 20, 160)], 8, 2, 128, 16),
    ([(200 + i, 1) for i in range(70)], [(0, 33, 191), (33, 33, 50), (33, 70, 128)], 4, 1, 64, 8),
    ([(200 + i, 1 + i % 3) for i in range(9)], [(1, 5, 100), (5, 8, 77)], 16, 2, 96, 32),
    ([(400, 100), (350, 66), (380, 90)], [(0, 3, 256)], 8, 4, 128, 16),
    ([(400, 100), (350, 66), (380, 90)], [(0, 3, 250)], 4, 4, 64, 16),
    ([(290, 17)] * 9, [(0, 9, 270)], 8, 2, 128, 16),
    ([(900, 1), (901, 2), (1000, 1)], [(0, 3, 880)], 32, 8, 128, 16),
    ([(90, 33), (120, 20)], [(0, 2, 64)], 6, 4, 64, 16),   # heads that do not divide evenly
    ([(90, 33), (120, 20)], [(0, 2, 70)], 3, 3, 80, 7),
    ([(600, 40)] + [(530 + i, 1) for i in range(30)], [(0, 31, 512)], 8, 2, 128, 16),
    ([(130, 1)] * 40, [(0, 40, 128)], 4, 4, 64, 64),
    ([(150, 1)] * 12, [(0, 12, 144)], 64, 8, 128, 48),
    ([(90, 1), (70, 2), (60, 1)], [(0, 2, 48)], 160, 1, 64, 16),   # many heads of one KV head
    ([(300, 1), (290, 3)], [(0, 2, 256)], 66, 2, 96, 16),
    ([(200 + i, 1) for i in range(6)], [(0, 4, 160), (4, 6, 96)], 40, 1, 128, 16),
    # more sequences, or groups, than a workgroup looks through by itself
    ([(140 + i % 9, 1 + i % 2) for i in range(150)], [(0, 70, 96), (70, 149, 130)], 4, 2, 64, 16),
    ([(60 + i % 7, 1) for i in range(160)], [(2 * i, 2 * i + 2, 16 + i % 33) for i in range(80)], 4, 1, 64, 16),
    ([(60 + i % 7, i % 3) for i in range(100)], [(i, i + 1, i % 40) for i in range(99)], 4, 2, 64, 8),
    ([(90, 70 if i % 40 == 3 else 1) for i in range(127)], [(0, 127, 17)], 2, 1, 128, 16),
    ([(90, 70 if i % 40 == 3 else 1) for i in range(128)], [(0, 128, 48)], 2, 1, 96, 16),
]


@pytest.mark.parametrize("act,pool", ACT_POOL)
@pytest.mark.parametrize("seqs,groups,heads,kv,dim,bs", PREFIX)
def test_prefix(provider, act, pool, seqs, groups, heads, kv, dim, bs):
    if pool == "i8" and dim % 32:
        pytest.skip("an 8-bit cache needs groups of 32")
    rng = np.random.default_rng(heads * 100 + dim + len(seqs))
    batch = ref.Batch(rng, seqs, bs, behind=2, before=1)
    shared = ref.Shared(batch, groups, named=len(seqs) % 2 == 0)
    run_attention(provider, rng, batch, shared, act, pool, heads, kv, dim, lse=len(seqs) % 3 != 0)


@pytest.mark.parametrize("act,pool", ACT_POOL)
@pytest.mark.parametrize("dim,bs", [(128, 16), (64, 8), (96, 32)])
def test_prefix_past_the_rows(provider, act, pool, dim, bs):
    """Prefixes that reach into the new rows, past a sequence's end and past the bound: a row looks no further than itself;
    rows before position 0, sequences without blocks, blocks past the pools."""
    rng = np.random.default_rng(31)
    batch = ref.Batch(rng, [(100, 60), (70, 10), (30, 30), (3, 6), (150, 1), (64, 64)], bs)
    shared = ref.Shared(batch, [(0, 4, 90), (4, 6, 5000)])
    run_attention(provider, rng, batch, shared, act, pool, 8, 2, dim)
    run_attention(provider, rng, batch, shared, act, pool, 8, 2, dim, max_seq_len=75)
    batch.table[1] = ref.NONE
    batch.table[0, 1] = batch.blocks + 3
    run_attention(provider, rng, batch, shared, act, pool, 8, 2, dim)
    batch.table[0] = ref.NONE
    run_attention(provider, rng, batch, shared, act, pool, 8, 2, dim)


@pytest.mark.parametrize("act,pool", ACT_POOL)
@pytest.mark.parametrize("dim,seqs,groups", [
    (128, [(290 + 7 * i, 120) for i in range(7)] + [(60, 33), (333, 131)], [(0, 5, 200), (5, 9, 31)]),
    (64, [(250 + i, 120) for i in range(16)] + [(70, 1), (0, 0), (310, 121)], [(0, 17, 100)]),
    (96, [(400, 330), (390, 330), (300, 255), (420, 403)], [(0, 3, 48)]),
])
def test_prefix_more_rows_than_partials(provider, act, pool, dim, seqs, groups):
    """So many query rows that the workspace does not hold two partials of each: the last sequences' keys alone are cut."""
    rng = np.random.default_rng(38)
    batch = ref.Batch(rng, seqs, 16, behind=3)
    run_attention(provider, rng, batch, ref.Shared(batch, groups), act, pool, 32, 8, dim)


@pytest.mark.parametrize("act,pool", ACT_POOL)
def test_prefix_bad_groups(provider, act, pool):
    """Groups below zero, past the sequences or decreasing, and negative prefixes end in time and touch no other row."""
    rng = np.random.default_rng(32)
    batch = ref.Batch(rng, [(80, 4)] * 6, 16, behind=3)
    kv, dim, heads = 2, 64, 8
    pools, q = fill(rng, batch, None, act, pool, kv, dim), rows_of(rng, act, batch.rows, heads, dim)
    was = np.full_like(q, 5.0)
    wild = [(np.array([-4, 3, 1 << 30], np.int32), np.array([64, 48], np.int32)),
            (np.array([5, 2, 4, 0], np.int32), np.array([64, -1, 2 ** 31 - 1], np.int32)),
            (np.array([-2 ** 31, 2 ** 31 - 1], np.int32), np.array([-2 ** 31], np.int32))]
    with Bufs(provider) as m:
        out, base, desc = m.put(was), [m.put(q)] + [m.put(p) for p in pools], m.batch(batch)
        for first, n in wild:
            pc = pc_of(batch, kv, dim, n_heads=heads, step_idx=len(n))
            provider.dispatch("flash_attention_paged_prefix", base + desc + [m.put(first), m.put(n)], [out], pc=pc)
            got = out.read(NP[act], q.size).reshape(q.shape)
            assert np.array_equal(got[24:], was[24:])
        # sequences before the first group and behind the last share nothing, a prefix below zero is none
        shared = ref.Shared(batch, [(1, 3, 64), (3, 4, 0)])
        neg = shared.len.copy()
        neg[1] = -7
        pc = pc_of(batch, kv, dim, n_heads=heads, step_idx=2)
        provider.dispatch("flash_attention_paged_prefix", base + desc + [m.put(shared.first), m.put(neg)], [out], pc=pc)
        got = out.read(NP[act], q.size).reshape(q.shape)
    want, err, _, _ = ref.attention(batch, shared, pool, dim, heads, kv, pools, q, act)
    check(got[:24], want[:24], err[:24], (act, pool))
    assert np.array_equal(got[24:], was[24:])


@pytest.mark.parametrize("act,pool", ACT_POOL)
@pytest.mark.parametrize("dim", [128, 64, 96])
def test_prefix_large_scores(provider, act, pool, dim):
    """Maxima that grow along the keys, in the shared part and behind it; weights that underflow."""
    rng = np.random.default_rng(33)
    batch = ref.Batch(rng, [(330, 2), (300, 1), (420, 3), (310, 1)] * 6, 16)
    shared = ref.Shared(batch, [(0, 12, 256), (12, 24, 288)])
    pools = fill(rng, batch, shared, act, pool, 2, dim)
    for s in range(24):
        for pos in range(0, int(batch.lens[s]), 7):
            w = ref.where(batch, shared, s, pos)
            paged_ref.store(pools[0], pool, 16, dim, w, (rng.standard_normal((2, dim)) * (0.02 * pos)).astype(NP[act]))
    run_attention(provider, rng, batch, shared, act, pool, 8, 2, dim, pools=pools, q_scale=2.0)


@pytest.mark.parametrize("act,pool", ACT_POOL)
@pytest.mark.parametrize("rows", [2, 60])
def test_prefix_masked_values_are_not_finite(provider, act, pool, rows):
    """Values of later rows of a chunk, inside and behind the shared part, are NaN: earlier rows do not see them."""
    rng = np.random.default_rng(34)
    dim, kv, heads = 64, 2, 8
    batch = ref.Batch(rng, [(128, rows), (130, rows), (128, 1), (200, 3)], 16)
    shared = ref.Shared(batch, [(0, 3, 128)])
    pools = fill(rng, batch, shared, act, pool, kv, dim)
    for s, pos in ((0, 127), (1, 129)):
        b, slot = ref.where(batch, shared, s, pos)
        for p in pools:
            if pool == "i8":
                at = 16 * dim + slot * dim // 16
                p[b, :, at:at + dim // 16] = np.full((1, dim // 32), np.nan, np.float16).view(np.uint8)
            else:
                p[b, :, slot] = np.nan
    q = rows_of(rng, act, batch.rows, heads, dim)
    with Bufs(provider) as m:
        out, lb = m.put(np.zeros_like(q)), m.put(np.zeros((batch.rows, heads), np.float32))
        provider.dispatch("flash_attention_paged_prefix", [m.put(q)] + [m.put(p) for p in pools] + m.batch(batch) +
                          [m.put(shared.first), m.put(shared.len)], [out, lb], pc=pc_of(batch, kv, dim, n_heads=heads, step_idx=1))
        got = out.read(NP[act], q.size).reshape(q.shape)
        z = lb.read(np.float32, batch.rows * heads).reshape(batch.rows, heads)
    want, err, wz, zerr = ref.attention(batch, shared, pool, dim, heads, kv, pools, q, act)
    last = [int(batch.lens[s]) - int(batch.starts[s + 1]) for s in range(4)]
    sees = np.zeros(batch.rows, bool)
    for r, s, pos in batch.each():
        sees[r] = s < 3 and pos >= 127
        assert last[s] + r == pos
    assert np.isnan(got[sees]).all() and np.isnan(z[sees]).all()
    check(got[~sees], want[~sees], err[~sees], (act, pool))
    check(z[~sees], wz[~sees], zerr[~sees], (act, pool))


@pytest.mark.parametrize("act,pool", ACT_POOL)
@pytest.mark.parametrize("dim,rows", [(64, 1), (128, 40), (96, 3)])
def test_prefix_scores_of_minus_infinity(provider, act, pool, dim, rows):
    """Keys that score -inf weigh nothing; a sequence that has nothing else gives zeros and -inf."""
    if pool == "i8":
        pytest.skip("an 8-bit cache holds no infinities of one sign")
    rng = np.random.default_rng(35)
    batch = ref.Batch(rng, [(100, rows), (90, rows), (200, rows)], 16)
    shared = ref.Shared(batch, [(0, 2, 48)])
    pools = fill(rng, batch, shared, act, pool, 2, dim)
    for s in range(3):
        for pos in range(int(batch.lens[s])):
            if s == 2 or pos < 48 or pos % 3 == 0:
                b, slot = ref.where(batch, shared, s, pos)
                pools[0][b, :, slot, 0] = -np.inf
    q = np.abs(rows_of(rng, act, batch.rows, 4, dim)) + NP[act](0.25)
    with Bufs(provider) as m:
        out, lb = m.put(np.zeros_like(q)), m.put(np.zeros((batch.rows, 4), np.float32))
        provider.dispatch("flash_attention_paged_prefix", [m.put(q)] + [m.put(p) for p in pools] + m.batch(batch) +
                          [m.put(shared.first), m.put(shared.len)], [out, lb], pc=pc_of(batch, 2, dim, n_heads=4, step_idx=1))
        got, z = out.read(NP[act], q.size).reshape(q.shape), lb.read(np.float32, batch.rows * 4).reshape(batch.rows, 4)
    want, _, wz, _ = ref.attention(batch, shared, pool, dim, 4, 2, pools, q, act)
    # bounds from the finite keys alone
    for p in pools:
        p[np.isinf(p)] = 0
    _, err, _, zerr = ref.attention(batch, shared, pool, dim, 4, 2, pools, q, act)
    check(got, want, err * 2, (act, dim))
    none = np.isneginf(wz)
    assert none[2 * rows:].all() and np.array_equal(np.isneginf(z), none)
    check(z[~none], wz[~none], 2 * zerr[~none], (act, dim))


def imported(provider, m, keep, a, elt):
    """A buffer at an odd multiple of `elt` bytes."""
    import ctypes as C

    import torch

    from neurofabric_amd import plugin
    t = torch.zeros(a.nbytes + 64, dtype=torch.uint8, device="cuda")
    t[elt:elt + a.nbytes] = torch.from_numpy(a.reshape(-1).view(np.uint8).copy()).cuda()
    torch.cuda.synchronize()
    keep.append(t)
    dt = {"f4": NF["f32"], "f2": NF["f16"], "u1": NF["i8"], "i4": abi.NF_DTYPE_I32}[a.dtype.str[1:]]
    desc, ops, h = abi.make_desc(dt, a.nbytes), abi.nf_buffer_ops(), C.c_void_p()
    provider.check(provider.mem.import_buffer(provider.handle, t.data_ptr() + elt, abi.NF_MEM_DOMAIN_DEVICE, C.byref(desc),
                                              C.byref(ops), C.byref(h)), "import")
    m.all.append(plugin.Buffer(provider, h.value, ops, dt, a.nbytes))
    return m.all[-1]


@pytest.mark.parametrize("act,pool", ACT_POOL)
def test_misaligned(provider, act, pool):
    """Imported operands at odd multiples of their element size, all three operators."""
    rng = np.random.default_rng(36)
    heads, kv, dim, bs = 4, 2, 64, 16
    batch = ref.Batch(rng, [(70, 20), (63, 1)], bs, spare=9)
    shared = ref.Shared(batch, [(0, 2, 48)], named=True)
    pools, q = fill(rng, batch, shared, act, pool, kv, dim), rows_of(rng, act, batch.rows, heads, dim)
    el = {"f32": 4, "f16": 2}[act]
    pel = 2 if pool == "i8" else el
    keep, width = [], batch.width * bs
    held = rng.random((2, kv, width)).astype(np.float32)
    lse = np.full((batch.rows, heads), 4.0, np.float32)
    top = 40
    new = np.array([[i for i in range(batch.blocks) if i not in batch.table][:3]] * 2, np.uint32)
    new[1] = [i for i in range(batch.blocks) if i not in batch.table][3:6]
    with Bufs(provider) as m:
        odd = lambda a, e: imported(provider, m, keep, a, e)  # noqa: E731
        kb, qb, out, desc = [odd(p, pel) for p in pools], odd(q, el), odd(np.zeros_like(q), el), m.batch(batch)
        hb, wb, lb = odd(held, 4), odd(np.zeros_like(held), 4), odd(lse, 4)
        kept, lens = odd(np.zeros((2, kv, top), np.int32), 4), odd(np.zeros(2, np.int32), 4)
        provider.dispatch("flash_attention_paged_prefix", [qb] + kb + desc + [m.put(shared.first), m.put(shared.len)], [out],
                          pc=pc_of(batch, kv, dim, n_heads=heads, step_idx=1))
        provider.dispatch("paged_kv_weights", [qb, kb[0]] + desc + [lb, hb], [wb],
                          pc=pc_of(batch, kv, dim, n_heads=heads, step_idx=width, theta=1.0))
        got, w = out.read(NP[act], q.size).reshape(q.shape), wb.read(np.float32, held.size).reshape(held.shape)
        pc = push_constants(M=kv, N=batch.width, K=2, seq_len=top, head_dim=dim, window_size=bs, step_idx=width)
        provider.dispatch("paged_kv_evict", kb + [hb, desc[0], desc[2], m.put(np.array([[40, 8], [33, 0]], np.int32)), m.put(new)],
                          kb + [wb, lens, kept], pc=pc)
        after = [b.read(np.uint8, p.nbytes).reshape(p.view(np.uint8).shape) for b, p in zip(kb, pools)]
        chosen = kept.read(np.int32, 2 * kv * top).reshape(2, kv, top)
    want, err, _, _ = ref.attention(batch, shared, pool, dim, heads, kv, pools, q, act)
    check(got, want, err, (act, pool))
    want, err = ref.weights(batch, pool, dim, heads, kv, pools[0], q, act, lse, held, 1.0, np.zeros_like(held))
    check(w, want, err, (act, pool))
    rows = ref.evict(batch, batch.lens, held, [[40, 8], [33, 0]], top)
    for s in range(2):
        assert np.array_equal(chosen[s, :, :rows[s].shape[1]], rows[s])
    ref.move(batch, pool, dim, [p.copy() for p in pools], pools, rows, new)
    for a, p in zip(after, pools):
        assert np.array_equal(a, p.view(np.uint8))


# ---- log-sum-exp and weights --------------------------------------------------------

CHUNK = [  # sequences (positions, rows), heads, KV heads, head_dim, block size
    ([(1, 1)], 1, 1, 64, 16),
    ([(1, 1), (2, 2), (300, 1)], 4, 4, 128, 16),
    ([(700, 1), (3, 1), (129, 1), (256, 1)], 8, 1, 128, 16),
    ([(97, 5), (40, 2), (0, 0), (333, 4)], 8, 2, 64, 8),
    ([(200, 200)], 2, 1, 128, 16),
    ([(150, 70), (65, 64), (129, 1)], 6, 2, 64, 32),
    ([(260, 131)], 4, 4, 128, 4),
    ([(90, 33), (20, 20)], 6, 4, 64, 16),      # heads that do not divide evenly
    ([(90, 33), (20, 20)], 10, 1, 96, 16),
    ([(50, 50)], 3, 3, 256, 7),
    ([(500, 3)] * 3, 8, 8, 96, 16),
    ([(i % 40 + 1, 1) for i in range(90)], 4, 2, 64, 16),
    ([(1500, 2), (700, 3), (40, 1)], 32, 8, 128, 32),
    ([(1200, 120)], 2, 2, 128, 16),
    ([(64, 1), (65, 1), (63, 1), (128, 32), (32, 32)], 1, 1, 128, 16),
    ([(300, 140)], 16, 16, 64, 16),
    ([(130, 129), (40, 1), (9, 9)], 8, 2, 96, 64),
    ([(90, 1), (70, 2), (200, 1)], 80, 2, 64, 16),       # many heads of one KV head
    ([(90, 1), (300, 7)], 130, 1, 128, 16),
    ([(600, 500), (90, 2), (300, 260)], 8, 1, 64, 16),   # rows cut as well
    ([(1100, 900)], 4, 1, 96, 8),
]


def run_weights(provider, rng, batch, act, pool, heads, kv, dim, lse, q, pools, theta=1.0, max_seq_len=0, width=None):
    width = width or max(batch.width * batch.bs if not max_seq_len else max_seq_len, 1)
    held = rng.random((len(batch.seqs), kv, width)).astype(np.float32)
    was = np.full_like(held, 9.0)
    pc = pc_of(batch, kv, dim, n_heads=heads, step_idx=width, theta=theta, max_seq_len=max_seq_len)
    with Bufs(provider) as m:
        wb, hb = m.put(was), m.put(held)
        ins = [m.put(q), m.put(pools[0])] + m.batch(batch) + [m.put(lse)]
        provider.dispatch("paged_kv_weights", ins + [hb], [wb], pc=pc)
        got = wb.read(np.float32, held.size).reshape(held.shape)
        provider.dispatch("paged_kv_weights", ins + [hb], [hb], pc=pc)  # in place
        again = hb.read(np.float32, held.size).reshape(held.shape)
    want, err = ref.weights(batch, pool, dim, heads, kv, pools[0], q, act, lse, held, theta, was, max_seq_len or None)
    check(got, want, err, (act, pool, heads, kv, dim, batch.seqs[:4], theta))
    wrote = np.zeros(was.shape, bool)
    for i in range(len(batch.seqs)):
        n = min(int(batch.lens[i]), batch.width * batch.bs, max_seq_len or 1 << 30)
        wrote[i, :, :max(0, n)] = batch.starts[i + 1] > batch.starts[i]
    assert np.array_equal(got[~wrote], was[~wrote])
    assert np.array_equal(again, np.where(wrote, got, held))
    return got


@pytest.mark.parametrize("act,pool", ACT_POOL)
@pytest.mark.parametrize("seqs,heads,kv,dim,bs", CHUNK)
def test_lse_and_weights(provider, act, pool, seqs, heads, kv, dim, bs):
    rng = np.random.default_rng(heads * 100 + dim + len(seqs) + bs)
    batch = ref.Batch(rng, seqs, bs, behind=2, before=1)
    q, pools, z = run_attention(provider, rng, batch, None, act, pool, heads, kv, dim, chunk=True)
    got = run_weights(provider, rng, batch, act, pool, heads, kv, dim, z, q, pools, theta=(0.0, 1.0, 0.75)[len(seqs) % 3],
                      width=batch.width * bs + len(seqs) % 4)
    assert np.isfinite(got).all()


@pytest.mark.parametrize("act,pool", ACT_POOL)
@pytest.mark.parametrize("dim", [128, 64, 96])
def test_weights_add_up_to_the_rows(provider, act, pool, dim):
    """With theta 0 a sequence's weights add up to its rows times the heads of a KV head; the output with a log-sum-exp is
    the one without."""
    rng = np.random.default_rng(41)
    heads, kv = 8, 2
    batch = ref.Batch(rng, [(300, 1), (150, 40), (90, 90), (33, 5)], 16)
    q, pools, z = run_attention(provider, rng, batch, None, act, pool, heads, kv, dim, chunk=True)
    got = run_weights(provider, rng, batch, act, pool, heads, kv, dim, z, q, pools, theta=0.0)
    for s, (n, r) in enumerate(batch.seqs):
        assert np.allclose(got[s, :, :n].astype(np.float64).sum(1), r * heads / kv, rtol=2e-5)
    outs = []
    with Bufs(provider) as m:
        ins = [m.put(q)] + [m.put(p) for p in pools] + m.batch(batch)
        for second in ([], [m.put(z)]):
            o = m.put(np.zeros_like(q))
            provider.dispatch("flash_attention_paged_chunk", ins, [o] + second, pc=pc_of(batch, kv, dim, n_heads=heads))
            outs.append(o.read(np.uint8, q.nbytes))
    assert np.array_equal(*outs)


@pytest.mark.parametrize("act,pool", ACT_POOL)
@pytest.mark.parametrize("dim,bs", [(128, 16), (64, 8), (96, 32), (40, 16)])
def test_lse_and_weights_without_keys(provider, act, pool, dim, bs):
    """Rows before position 0, holes in the tables, sequences without blocks or rows, positions past max_seq_len; rows whose
    log-sum-exp is -inf give nothing."""
    if pool == "i8" and dim % 32:
        pytest.skip("an 8-bit cache needs groups of 32")
    rng = np.random.default_rng(42)
    batch = ref.Batch(rng, [(3, 6), (100, 40), (40, 40), (200, 2), (50, 0), (-4, 3)], bs)
    batch.table[1, 0] = ref.NONE
    batch.table[1, 3] = batch.blocks
    batch.table[2] = ref.NONE
    batch.table[3, 1:5] = ref.NONE
    for limit in (0, 70):
        q, pools, z = run_attention(provider, rng, batch, None, act, pool, 8, 2, dim, chunk=True, max_seq_len=limit)
        got = run_weights(provider, rng, batch, act, pool, 8, 2, dim, z, q, pools, max_seq_len=limit)
        assert np.isfinite(got).all()


@pytest.mark.parametrize("act,pool", ACT_POOL)
@pytest.mark.parametrize("dim", [128, 64])
def test_weights_large_scores(provider, act, pool, dim):
    rng = np.random.default_rng(43)
    batch = ref.Batch(rng, [(400, 3), (130, 130)], 16)
    pools = fill(rng, batch, None, act, pool, 2, dim)
    for pos in range(400):
        paged_ref.store(pools[0], pool, 16, dim, batch.where(0, pos), (rng.standard_normal((2, dim)) * (0.02 * pos)).astype(NP[act]))
    q, _, z = run_attention(provider, rng, batch, None, act, pool, 8, 2, dim, pools=pools, chunk=True, q_scale=2.0)
    run_weights(provider, rng, batch, act, pool, 8, 2, dim, z, q, pools)


def test_weights_bad_batch(provider):
    """Starts below zero, past the rows, or decreasing, and wild lengths: other sequences come out, nothing else is written."""
    rng = np.random.default_rng(44)
    heads, kv, dim, bs = 8, 2, 64, 16
    good = ref.Batch(rng, [(150, 60), (40, 2), (33, 33)], bs, behind=4)
    pools, q = fill(rng, good, None, "f16", "f16", kv, dim), rows_of(rng, "f16", good.rows, heads, dim)
    lse = np.full((good.rows, heads), 5.0, np.float32)
    bad = ref.Batch(rng, [(10, 1)] * 7, bs)
    bad.blocks, bad.width, bad.rows = good.blocks, good.width, good.rows
    bad.table = np.full((7, good.width), ref.NONE, np.uint32)
    bad.table[1], bad.table[3], bad.table[5] = good.table
    bad.starts = np.array([-5, 0, 60, 60, 62, 62, 95, 1 << 30], np.int32)
    bad.lens = np.array([100, 150, 3, 40, -7, 33, 1000], np.int32)
    width = good.width * bs
    held, was = rng.random((7, kv, width)).astype(np.float32), np.full((7, kv, width), 2.0, np.float32)
    with Bufs(provider) as m:
        wb = m.put(was)
        base = [m.put(q), m.put(pools[0])]
        pc = pc_of(bad, kv, dim, n_heads=heads, step_idx=width, theta=1.0)
        provider.dispatch("paged_kv_weights", base + m.batch(bad) + [m.put(lse), m.put(held)], [wb], pc=pc)
        got = wb.read(np.float32, was.size).reshape(was.shape)
        wild = [m.put(bad.table), m.put(np.array([90, 80, 5, 70, 2, 2, 1, 0], np.int32)),
                m.put(np.array([2 ** 31 - 1, -2 ** 31, 2 ** 31 - 1, 7, 9, 2 ** 31 - 1, 0], np.int32))]
        provider.dispatch("paged_kv_weights", base + wild + [m.put(lse), m.put(held)], [m.put(was)], pc=pc)
        provider.synchronize()
    want, err = ref.weights(good, "f16", dim, heads, kv, pools[0], q, "f16", lse, held[[1, 3, 5]], 1.0, was[[1, 3, 5]])
    check(got[[1, 3, 5]], want, err, "good")
    assert np.array_equal(got[[0, 2, 4, 6]], was[[0, 2, 4, 6]])


# ---- eviction -------------------------------------------------------------------------

EVICT = [  # lengths, (keep, recent) of each, most kept, KV heads, head_dim, block size
    ([1], [(1, 1)], 1, 1, 64, 16),
    ([5, 0, 17], [(3, 1), (2, 2), (17, 4)], 20, 2, 64, 16),
    ([40, 100, 64], [(20, 0), (20, 20), (64, 10)], 64, 4, 128, 16),
    ([300, 257, 256], [(256, 64), (1, 0), (255, 255)], 256, 2, 96, 8),
    ([1000, 33], [(999, 100), (100, 50)], 999, 2, 64, 32),
    ([3000], [(700, 90)], 700, 3, 64, 16),
    ([50, 60], [(0, 0), (-3, 5)], 10, 2, 32, 5),
    ([90, 70], [(200, 300), (40, -1)], 60, 2, 64, 7),     # more than there are, more than `most`
    ([20000, 40000], [(5000, 500), (9000, 1)], 9000, 1, 32, 16),
    ([16500, 3, 0, 8192, 4097], [(2000, 30), (5, 1), (4, 4), (8192, 0), (4096, 4096)], 8192, 2, 32, 16),
    ([9000 - 60 * i for i in range(130)], [(90, 7)] * 130, 90, 2, 32, 16),
]


def run_evict(provider, rng, pool, lens, budget, top, kv, dim, bs, held=None, max_seq_len=0, edit=None, width=0):
    act = "f32" if pool == "f32" else "f16"
    batch = ref.Batch(rng, [(n, 0) for n in lens], bs, spare=1)
    pages = -(-top // bs)
    new = rng.permutation(len(lens) * pages).astype(np.uint32).reshape(len(lens), pages) + np.uint32(batch.blocks)
    from_blocks = batch.blocks
    total = from_blocks + len(lens) * pages
    pools = [paged_ref.empty_pool(rng, pool, total, kv, bs, dim) for _ in range(2)]
    del act
    batch.blocks = total
    if edit:
        edit(batch, new)
    width = width or max_seq_len or batch.width * bs
    if held is None:
        held = (rng.random((len(lens), kv, width)) ** 6).astype(np.float32)
        held[rng.random(held.shape) < 0.2] = 0.25  # ties
    was = np.full_like(held, -1.0)
    with Bufs(provider) as m:
        kb, desc = [m.put(p) for p in pools], m.batch(batch)
        wb, lb, jb = m.put(was), m.put(np.full(len(lens), -9, np.int32)), m.put(np.full((len(lens), kv, max(top, 1)), -5, np.int32))
        pc = push_constants(M=kv, N=batch.width, K=len(lens), seq_len=top, head_dim=dim, window_size=bs, step_idx=width,
                            max_seq_len=max_seq_len)
        ins = kb + [m.put(held), desc[0], desc[2], m.put(np.array(budget, np.int32)), m.put(new)]
        provider.dispatch("paged_kv_evict", ins, kb + [wb, lb, jb], pc=pc)
        got = [b.read(np.uint8, p.nbytes).reshape(p.view(np.uint8).shape) for b, p in zip(kb, pools)]
        w, n, kept = wb.read(np.float32, was.size).reshape(was.shape), lb.read(np.int32, len(lens)), jb.read(np.int32)
        kept = kept[:len(lens) * kv * top].reshape(len(lens), kv, top)
    rows = ref.evict(batch, batch.lens, held, budget, top, max_seq_len or None)
    for s, r in enumerate(rows):
        k = r.shape[1]
        assert n[s] == k
        assert np.array_equal(kept[s, :, :k], r), (s, lens[s], budget[s])
        assert (kept[s, :, k:] == -5).all()
        assert np.array_equal(w[s, :, :k].view(np.uint32), np.take_along_axis(held[s], r, 1).view(np.uint32))
        assert (w[s, :, k:] == -1.0).all()
    ref.move(batch, pool, dim, [p.copy() for p in pools], pools, rows, new)
    for g, p in zip(got, pools):
        assert np.array_equal(g, p.view(np.uint8))  # what no kept row goes to stays as it was
    return kept


@pytest.mark.parametrize("pool", ["f32", "f16", "i8"])
@pytest.mark.parametrize("lens,budget,top,kv,dim,bs", EVICT)
def test_evict(provider, pool, lens, budget, top, kv, dim, bs):
    run_evict(provider, np.random.default_rng(len(lens) * 100 + dim + top), pool, lens, budget, top, kv, dim, bs)


def test_evict_order_of_weights(provider):
    """Equal weights, both zeros, infinities, NaN, negative and subnormal ones."""
    rng = np.random.default_rng(51)
    kinds = np.array([0.0, -0.0, 1.0, 1.0, np.inf, -np.inf, np.nan, -np.nan, -2.0, 1e-40, -1e-40, 3e38, 0.5], np.float32)
    for n, keep, recent in ((700, 300, 20), (700, 80, 0), (700, 690, 5), (64, 1, 0), (1500, 700, 650)):
        held = kinds[rng.integers(0, len(kinds), (2, 2, 1504))]
        held[1] = 0.125 if keep != 80 else np.nan
        run_evict(provider, rng, "f16", [n, n], [(keep, recent)] * 2, keep, 2, 64, 16, held=held, width=1504)
    for keep, recent in ((4000, 300), (17000, 0), (30, 0)):  # a row of several workgroups
        held = kinds[rng.integers(0, len(kinds), (2, 1, 18003))]
        held[1] = 0.125 if keep != 30 else np.nan
        run_evict(provider, rng, "f16", [17003, 17999], [(keep, recent)] * 2, keep, 1, 32, 16, held=held, width=18003)


def test_evict_without_storage(provider):
    """Positions without blocks go first; the kept ones among them become zeros; new blocks past the pools are not written;
    lengths past the bound, below zero and past the table."""
    rng = np.random.default_rng(52)

    def holes(batch, new):
        batch.table[0, 1] = ref.NONE
        batch.table[1, :] = ref.NONE
        batch.table[2, 0] = batch.blocks
        new[0, 1] = batch.blocks
        new[2, 0] = 0xFFFFFFFF

    for pool in ("f32", "f16", "i8"):
        run_evict(provider, rng, pool, [60, 50, 40], [(50, 10), (20, 20), (40, 0)], 50, 2, 64, 16, edit=holes)
        run_evict(provider, rng, pool, [60, 50, 40], [(50, 10), (20, 20), (40, 0)], 50, 2, 64, 16, edit=holes, max_seq_len=45)

    def wild(batch, new):
        batch.lens[:] = [2 ** 31 - 1, -2 ** 31, -1]
    run_evict(provider, rng, "f16", [60, 50, 40], [(50, 10), (20, 20), (40, 0)], 50, 2, 64, 16, edit=wild)


@pytest.mark.parametrize("pool", ["f16", "i8"])
def test_evict_into_other_pools(provider, pool):
    """The rows go to pools of their own, of another number of blocks."""
    rng = np.random.default_rng(53)
    kv, dim, bs, top = 2, 64, 16, 24
    batch = ref.Batch(rng, [(100, 0), (37, 0)], bs)
    pools = [paged_ref.empty_pool(rng, pool, batch.blocks, kv, bs, dim) for _ in range(2)]
    to = [paged_ref.empty_pool(rng, pool, 4, kv, bs, dim) for _ in range(2)]
    new, budget = np.array([[3, 0], [2, 1]], np.uint32), np.array([[24, 4], [20, 20]], np.int32)
    held = rng.random((2, kv, batch.width * bs)).astype(np.float32)
    with Bufs(provider) as m:
        kb, tb, desc = [m.put(p) for p in pools], [m.put(p) for p in to], m.batch(batch)
        outs = tb + [m.put(np.zeros_like(held)), m.put(np.zeros(2, np.int32)), m.put(np.zeros((2, kv, top), np.int32))]
        pc = push_constants(M=kv, N=batch.width, K=2, seq_len=top, head_dim=dim, window_size=bs, step_idx=batch.width * bs)
        provider.dispatch("paged_kv_evict", kb + [m.put(held), desc[0], desc[2], m.put(budget), m.put(new)], outs, pc=pc)
        got = [b.read(np.uint8, p.nbytes).reshape(p.view(np.uint8).shape) for b, p in zip(tb, to)]
        left = [b.read(np.uint8, p.nbytes).reshape(p.view(np.uint8).shape) for b, p in zip(kb, pools)]
    ref.move(batch, pool, dim, pools, to, ref.evict(batch, batch.lens, held, budget, top), new)
    for g, p in zip(got + left, to + pools):
        assert np.array_equal(g, p.view(np.uint8))


# ---- together -------------------------------------------------------------------------

def test_no_rows_or_sequences(provider):
    """Empty batches leave everything as it was; an eviction of nothing writes lengths of 0."""
    rng = np.random.default_rng(61)
    for seqs in ([], [(5, 0), (0, 0)]):
        batch = ref.Batch(rng, seqs, 16, spare=2, behind=2)
        n = len(seqs)
        pool, x = paged_ref.empty_pool(rng, "f32", batch.blocks, 2, 16, 64), rows_of(rng, "f32", batch.rows, 2, 64)
        width = batch.width * 16
        held = rng.random((max(n, 1), 2, width)).astype(np.float32)
        with Bufs(provider) as m:
            desc, kb, xb = m.batch(batch), [m.put(pool), m.put(pool)], m.put(x)
            out, lb = m.put(x), m.put(np.zeros((batch.rows, 2), np.float32))
            hb, wb, nl, kept = m.put(held), m.put(held), m.put(np.full(2, 7, np.int32)), m.put(np.full(64, 7, np.int32))
            group = [m.put(np.array([0, n], np.int32)), m.put(np.array([3], np.int32))]
            budget, new = m.put(np.zeros((2, 2), np.int32)), m.put(np.zeros((2, 1), np.uint32))
            for rows in (batch.rows, 0):
                pc = dict(M=2, N=batch.width, K=n, head_dim=64, window_size=16)
                provider.dispatch("flash_attention_paged_prefix", [xb] + kb + desc + group, [out, lb],
                                  pc=push_constants(seq_len=rows, n_heads=2, step_idx=1, **pc))
                provider.dispatch("paged_kv_weights", [xb, kb[0]] + desc + [lb, hb], [wb],
                                  pc=push_constants(seq_len=rows, n_heads=2, step_idx=width, theta=1.0, **pc))
                provider.dispatch("paged_kv_evict", kb + [hb, desc[0], desc[2], budget, new], kb + [wb, nl, kept],
                                  pc=push_constants(seq_len=rows and 16, step_idx=width, **pc))
            for b, a in ((kb[0], pool), (kb[1], pool), (out, x), (wb, held)):
                assert np.array_equal(b.read(np.float32, a.size), a.ravel())
            assert (lb.read(np.float32) == 0).all() and (kept.read(np.int32) == 7).all()
            assert nl.read(np.int32, 2).tolist() == [0] * n + [7] * (2 - n)


@pytest.mark.parametrize("act,pool", ACT_POOL)
def test_decode_evict_decode(provider, act, pool):
    """A server's run: prompts behind a shared prefix, tokens one by one with their weights gathered, an eviction into new
    blocks (the shared ones stay), more tokens over what is left."""
    rng = np.random.default_rng(62)
    heads, kv, dim, bs, steps = 8, 2, 64, 16, 3
    n, prefix, tail, keep, recent = 3, 64, 20, 48, 12
    most = prefix + tail + 2 * steps
    batch = ref.Batch(rng, [(most, tail)] * n, bs, spare=n * -(-(keep + 16) // bs))
    shared = ref.Shared(batch, [(0, n, prefix)], named=True)
    free = [i for i in range(batch.blocks) if i not in batch.table]
    pools = fill(rng, batch, shared, act, pool, kv, dim)
    width = batch.width * bs
    held = np.zeros((n, kv, width), np.float32)

    def step(lens, rows, table, with_prefix):
        batch.seqs = [(m, rows) for m in lens]
        batch.lens = np.array(lens, np.int32)
        batch.starts = (np.arange(n + 1) * rows).astype(np.int32)
        batch.rows, batch.table = n * rows, table
        x = [rows_of(rng, act, n * rows, kv, dim) for _ in range(2)]
        q = rows_of(rng, act, n * rows, heads, dim)
        pc = pc_of(batch, kv, dim, n_heads=heads)
        desc = [m.put(table), m.put(batch.starts), m.put(batch.lens)]
        xb, qb, out, lb = [m.put(a) for a in x], m.put(q), m.put(np.zeros_like(q)), m.put(np.zeros((n * rows, heads), np.float32))
        tasks = [provider.task("paged_kv_append", xb + desc, kb, pc=pc)]
        if with_prefix:
            more = [m.put(shared.first), m.put(shared.len)]
            tasks.append(provider.task("flash_attention_paged_prefix", [qb] + kb + desc + more, [out, lb],
                                       pc=pc_of(batch, kv, dim, n_heads=heads, step_idx=1)))
        else:
            tasks.append(provider.task("flash_attention_paged_chunk", [qb] + kb + desc, [out, lb], pc=pc))
        tasks.append(provider.task("paged_kv_weights", [qb, kb[0]] + desc + [lb, wb], [wb],
                                   pc=pc_of(batch, kv, dim, n_heads=heads, step_idx=width, theta=1.0)))
        provider.run_tasks((abi.nf_task_desc * 3)(*tasks))
        paged_ref.append(batch, pool, dim, pools, x)
        got, z = out.read(NP[act], q.size).reshape(q.shape), lb.read(np.float32, q.shape[0] * heads).reshape(-1, heads)
        want, err, wz, zerr = ref.attention(batch, shared if with_prefix else None, pool, dim, heads, kv, pools, q, act)
        check(got, want, err, (lens, rows))
        check(z, wz, zerr, (lens, rows))
        was = held.copy()
        now = wb.read(np.float32, held.size).reshape(held.shape)
        want, err = ref.weights(batch, pool, dim, heads, kv, pools[0], q, act, z, was, 1.0, was)
        check(now, want, err, (lens, rows))
        held[:] = now

    with Bufs(provider) as m:
        kb, wb = [m.put(p) for p in pools], m.put(held)
        table = batch.table.copy()
        length = prefix + tail
        step([length] * n, tail, table, True)
        for _ in range(steps):
            length += 1
            step([length] * n, 1, table, True)
        # eviction, to blocks of their own
        new = np.full((n, batch.width), ref.NONE, np.uint32)
        per = -(-(keep + 16) // bs)
        for s in range(n):
            new[s, :per] = free[s * per:(s + 1) * per]
        pages = -(-keep // bs)
        w2, nl, kept = m.put(held), m.put(np.zeros(n, np.int32)), m.put(np.zeros((n, kv, keep), np.int32))
        pc = push_constants(M=kv, N=batch.width, K=n, seq_len=keep, head_dim=dim, window_size=bs, step_idx=width)
        provider.dispatch("paged_kv_evict", kb + [wb, m.put(table), m.put(batch.lens), m.put(np.array([[keep, recent]] * n, np.int32)),
                                                  m.put(np.ascontiguousarray(new[:, :pages]))], kb + [w2, nl, kept], pc=pc)
        rows = ref.evict(batch, batch.lens, held, [[keep, recent]] * n, keep)
        assert np.array_equal(kept.read(np.int32).reshape(n, kv, keep), np.stack(rows))
        ref.move(batch, pool, dim, [p.copy() for p in pools], pools, rows, new)
        for s in range(n):
            held[s, :, :keep] = np.take_along_axis(held[s], rows[s], 1)
        assert np.array_equal(w2.read(np.float32).reshape(held.shape)[:, :, :keep], held[:, :, :keep])
        wb.write(held)
        assert nl.read(np.int32).tolist() == [keep] * n
        length = keep
        for _ in range(steps):
            length += 1
            step([length] * n, 1, new, False)
        for b, p in zip(kb, pools):
            assert np.array_equal(b.read(np.uint8, p.nbytes), p.view(np.uint8).ravel())


@pytest.mark.parametrize("act,pool,rows", [("f16", "f16", 1), ("f16", "i8", 1), ("f32", "f32", 1), ("f16", "f16", 90)])
def test_offsets_past_32_bits(provider, act, pool, rows):
    """The blocks that are used lie past 2^32 bytes and elements of the pools, the last rows of the weights past as many."""
    rng = np.random.default_rng(63)
    heads, kv, dim, bs, top = 8, 8, 128, 16, 60
    width = 3 << 26
    batch = ref.Batch(rng, [(190, rows), (170, rows), (150, rows)], bs, spare=0)
    shared = ref.Shared(batch, [(0, 3, 64)], named=True)
    page = paged_ref.empty_pool(rng, pool, 1, 1, bs, dim).nbytes * kv
    used, pages = batch.blocks, -(-top // bs)
    batch.blocks += 3 * pages  # the evicted sequences' blocks
    new = (used + rng.permutation(3 * pages).reshape(3, pages)).astype(np.uint32)
    blocks = ((18 if pool == "f32" else 9) << 30) // page
    first = blocks - batch.blocks
    small = fill(rng, batch, shared, act, pool, kv, dim)
    q = rows_of(rng, act, batch.rows, heads, dim)
    limit = batch.width * bs
    held = rng.random((3, kv, limit)).astype(np.float32)
    budget = np.array([[60, 10], [50, 0], [33, 33]], np.int32)
    with Bufs(provider) as m:
        big = [provider.alloc(NF[pool], blocks * page) for _ in range(2)]
        wb = provider.alloc(NF["f32"], 3 * kv * width * 4)
        m.all += big + [wb]
        for b, p in zip(big, small):
            b.write(p, offset=first * page)
        for i in range(3 * kv):
            wb.write(held[i // kv, i % kv], offset=i * width * 4)
        at = ref.Batch(rng, batch.seqs, bs)
        far = lambda t: np.where(t == ref.NONE, t, t + np.uint32(first)).astype(np.uint32)  # noqa: E731
        at.table = far(batch.table)
        desc = m.batch(at)
        out, lb = m.put(np.zeros_like(q)), m.put(np.zeros((batch.rows, heads), np.float32))
        lens, kept = m.put(np.zeros(3, np.int32)), m.put(np.zeros((3, kv, top), np.int32))
        pc = pc_of(batch, kv, dim, n_heads=heads, step_idx=1)
        provider.dispatch("flash_attention_paged_prefix", [m.put(q)] + big + desc + [m.put(shared.first), m.put(shared.len)],
                          [out, lb], pc=pc)
        got = out.read(NP[act], q.size).reshape(q.shape)
        provider.dispatch("flash_attention_paged_chunk", [m.put(q)] + big + desc, [out, lb], pc=pc_of(batch, kv, dim, n_heads=heads))
        z = lb.read(np.float32, batch.rows * heads).reshape(batch.rows, heads)
        provider.dispatch("paged_kv_weights", [m.put(q), big[0]] + desc + [lb, wb], [wb],
                          pc=pc_of(batch, kv, dim, n_heads=heads, step_idx=width, theta=0.5))
        row = lambda i: wb.read(np.float32, limit, offset=i * width * 4)  # noqa: E731
        w = np.stack([row(i) for i in range(3 * kv)]).reshape(held.shape)
        pc = push_constants(M=kv, N=batch.width, K=3, seq_len=top, head_dim=dim, window_size=bs, step_idx=width)
        provider.dispatch("paged_kv_evict", big + [wb, desc[0], desc[2], m.put(budget), m.put(far(new))], big + [wb, lens, kept], pc=pc)
        chosen = kept.read(np.int32, 3 * kv * top).reshape(3, kv, top)
        after = [b.read(np.uint8, p.nbytes, offset=first * page).reshape(p.view(np.uint8).shape) for b, p in zip(big, small)]
        left = np.stack([row(i) for i in range(3 * kv)]).reshape(held.shape)
    want, err, wz, zerr = ref.attention(batch, shared, pool, dim, heads, kv, small, q, act)
    check(got, want, err, (act, pool))
    check(z, wz, zerr, (act, pool))
    want, err = ref.weights(batch, pool, dim, heads, kv, small[0], q, act, z, held, 0.5, held)
    check(w, want, err, (act, pool))
    rows = ref.evict(batch, batch.lens, w, budget, top)
    for s in range(3):
        k = rows[s].shape[1]
        assert np.array_equal(chosen[s, :, :k], rows[s])
        assert np.array_equal(left[s, :, :k].view(np.uint32), np.take_along_axis(w[s], rows[s], 1).view(np.uint32))
    ref.move(batch, pool, dim, [p.copy() for p in small], small, rows, new)
    for a, p in zip(after, small):
        assert np.array_equal(a, p.view(np.uint8))


@pytest.mark.parametrize("act,pool", [("f16", "f16"), ("f16", "i8"), ("f32", "f32")])
def test_captured_steps_replay(provider, act, pool):
    """Captured attention, weights and eviction follow lengths, groups and budgets that their buffers hold at each replay."""
    rng = np.random.default_rng(63)
    heads, kv, dim, bs, n = 8, 2, 64, 16, 6
    batch = ref.Batch(rng, [(300, 1)] * n, bs, spare=n * 4)
    free = [i for i in range(batch.blocks) if i not in batch.table]
    new = np.array(free[:n * 4], np.uint32).reshape(n, 4)
    pools = fill(rng, batch, None, act, pool, kv, dim)
    q, width, top = rows_of(rng, act, n, heads, dim), batch.width * bs, 64
    held = rng.random((n, kv, width)).astype(np.float32)
    z0 = np.zeros((n, heads), np.float32)
    with Bufs(provider) as m:
        kb, desc, qb = [m.put(p) for p in pools], m.batch(batch), m.put(q)
        out, lb, hb, wb = m.put(np.zeros_like(q)), m.put(z0), m.put(held), m.put(held)
        first, plen = m.put(np.zeros(3, np.int32)), m.put(np.zeros(2, np.int32))
        bb, nl, kept, we = m.put(np.zeros((n, 2), np.int32)), m.put(np.zeros(n, np.int32)), m.put(np.zeros((n, kv, top), np.int32)), m.put(held)
        tasks = (abi.nf_task_desc * 3)(
            provider.task("flash_attention_paged_prefix", [qb] + kb + desc + [first, plen], [out, lb],
                          pc=pc_of(batch, kv, dim, n_heads=heads, step_idx=2)),
            provider.task("paged_kv_weights", [qb, kb[0]] + desc + [lb, hb], [wb],
                          pc=pc_of(batch, kv, dim, n_heads=heads, step_idx=width, theta=0.5)),
            provider.task("paged_kv_evict", kb + [wb, desc[0], desc[2], bb, m.put(new)], kb + [we, nl, kept],
                          pc=push_constants(M=kv, N=batch.width, K=n, seq_len=top, head_dim=dim, window_size=bs, step_idx=width)))
        graph = hiprt.Graph(provider.stream(), lambda: provider.run_tasks(tasks))
        for lens, groups, budget in (([300] * n, [(0, 6, 256), (6, 6, 3)], (40, 8)), ([200, 17, 1, 300, 290, 299], [(0, 3, 16), (3, 6, 280)], (64, 64)),
                                     ([50, 60, 70, 300, 1, 2], [(0, 3, 40), (3, 4, 1)], (7, 0)), ([300] * n, [(0, 3, 250), (3, 6, 100)], (63, 5))):
            batch.seqs, batch.lens = [(x, 1) for x in lens], np.array(lens, np.int32)
            shared = ref.Shared(batch, groups)
            desc[2].write(batch.lens)
            first.write(shared.first)
            plen.write(shared.len)
            bb.write(np.array([budget] * n, np.int32))
            wb.write(held)
            graph.launch()
            got, z = out.read(NP[act], q.size).reshape(q.shape), lb.read(np.float32, z0.size).reshape(z0.shape)
            w, chosen = wb.read(np.float32, held.size).reshape(held.shape), kept.read(np.int32).reshape(n, kv, top)
            want, err, wz, zerr = ref.attention(batch, shared, pool, dim, heads, kv, pools, q, act)
            check(got, want, err, lens)
            check(z, wz, zerr, lens)
            want, err = ref.weights(batch, pool, dim, heads, kv, pools[0], q, act, z, held, 0.5, held)
            check(w, want, err, lens)
            rows = ref.evict(batch, batch.lens, w, [budget] * n, top)
            for s in range(n):
                assert np.array_equal(chosen[s, :, :rows[s].shape[1]], rows[s]), (lens, s)
            ref.move(batch, pool, dim, [p.copy() for p in pools], pools, rows, new)
            wb.write(held)
            provider.run_tasks(tasks)  # the eager calls agree
            assert np.array_equal(out.read(NP[act], q.size).reshape(q.shape).view(np.uint8), got.view(np.uint8))
            assert np.array_equal(wb.read(np.float32, held.size).reshape(held.shape), w)


@pytest.mark.parametrize("act,pool", ACT_POOL)
def test_captured_long_steps_share_the_workspace(provider, act, pool):
    """Two captured graphs of one prompt's attention, weights and eviction, whose kernels all keep partials in the workspace, are
    replayed in turn with new lengths, eager calls between them: every replay gives the eager calls' bits."""
    rng = np.random.default_rng(65)
    heads, kv, dim, bs, top, rows = 8, 1, 64, 16, 300, 200
    batch = ref.Batch(rng, [(17000, rows)], bs, spare=2 * -(-top // bs))
    free = [i for i in range(batch.blocks) if i not in batch.table]
    new = np.array(free, np.uint32).reshape(2, 1, -1)
    pools = fill(rng, batch, None, act, pool, kv, dim, 0.1)
    q, width = rows_of(rng, act, batch.rows, heads, dim), batch.width * bs
    held = rng.random((1, kv, width)).astype(np.float32)
    z0, k0 = np.zeros((batch.rows, heads), np.float32), np.zeros((1, kv, top), np.int32)
    with Bufs(provider) as m:
        desc, qb, hb = m.batch(batch), m.put(q), m.put(held)
        first, plen, budget = m.put(np.array([0, 1], np.int32)), m.put(np.array([9000], np.int32)), m.put(np.array([[top, 20]], np.int32))

        def steps(table):
            kb = [m.put(p) for p in pools]
            out = [m.put(np.zeros_like(q)), m.put(z0), m.put(np.zeros_like(held)), m.put(held), m.put(np.zeros(1, np.int32)), m.put(k0)]
            tasks = (abi.nf_task_desc * 3)(
                provider.task("flash_attention_paged_prefix", [qb] + kb + desc + [first, plen], out[:2],
                              pc=pc_of(batch, kv, dim, n_heads=heads, step_idx=1)),
                provider.task("paged_kv_weights", [qb, kb[0]] + desc + [out[1], hb], [out[2]],
                              pc=pc_of(batch, kv, dim, n_heads=heads, step_idx=width, theta=0.5)),
                provider.task("paged_kv_evict", kb + [out[2], desc[0], desc[2], budget, m.put(table)], kb + out[3:],
                              pc=push_constants(M=kv, N=batch.width, K=1, seq_len=top, head_dim=dim, window_size=bs, step_idx=width)))
            return tasks, kb + out

        all_steps = [steps(new[i]) for i in range(2)] + [steps(new[0])]
        read = lambda bufs: [b.read(np.uint8) for b in bufs]  # noqa: E731
        graphs = []
        for tasks, _ in all_steps[:2]:
            provider.run_tasks(tasks)
            graphs.append(hiprt.Graph(provider.stream(), lambda t=tasks: provider.run_tasks(t)))
        for n in (17000, 900, 16999, 300, 12345):
            desc[2].write(np.array([n], np.int32))
            plen.write(np.array([n // 2], np.int32))
            provider.run_tasks(all_steps[2][0])
            eager = read(all_steps[2][1][2:])
            for i in (0, 1, 0):
                graphs[i].launch()
            for i in range(2):
                got = read(all_steps[i][1][2:])
                for j, (a, b) in enumerate(zip(got, eager)):
                    assert np.array_equal(a, b), (n, i, j)
            kept = eager[5].view(np.int32)
            assert (np.diff(kept[:min(n, top)]) > 0).all() and kept[min(n, top) - 1] == n - 1


def test_output_in_place_of_the_query(provider):
    rng = np.random.default_rng(64)
    for seqs, group, act, dim in (([(900, 1), (820, 1)] * 4, 800, "f16", 128), ([(200, 90), (250, 80)], 96, "f16", 64),
                                  ([(300, 30), (330, 1)], 256, "f32", 64), ([(100, 20)] * 3, 70, "f16", 96), ([(40, 1)], 0, "f32", 64)):
        batch = ref.Batch(rng, seqs, 16)
        shared = ref.Shared(batch, [(0, len(seqs), group)])
        pools, q = fill(rng, batch, shared, act, act, 2, dim), rows_of(rng, act, batch.rows, 8, dim)
        with Bufs(provider) as m:
            qb = m.put(q)
            provider.dispatch("flash_attention_paged_prefix", [qb] + [m.put(p) for p in pools] + m.batch(batch) +
                              [m.put(shared.first), m.put(shared.len)], [qb], pc=pc_of(batch, 2, dim, n_heads=8, step_idx=1))
            got = qb.read(NP[act], q.size).reshape(q.shape)
        want, err, _, _ = ref.attention(batch, shared, act, dim, 8, 2, pools, q, act)
        check(got, want, err, seqs)


@pytest.mark.parametrize("act,pool", ACT_POOL)
def test_repeated_calls_give_the_same_bits(provider, act, pool):
    rng = np.random.default_rng(65)
    heads, kv, dim, bs = 16, 4, 128, 16
    batch = ref.Batch(rng, [(700 + 11 * i, 1 + i % 2) for i in range(12)], bs)
    shared = ref.Shared(batch, [(0, 7, 640), (7, 12, 512)])
    pools, q = fill(rng, batch, shared, act, pool, kv, dim), rows_of(rng, act, batch.rows, heads, dim)
    width = batch.width * bs
    held = rng.random((12, kv, width)).astype(np.float32)
    seen = set()
    with Bufs(provider) as m:
        base, desc = [m.put(q)] + [m.put(p) for p in pools], m.batch(batch)
        out, lb, hb, wb = m.put(np.zeros_like(q)), m.put(np.zeros((batch.rows, heads), np.float32)), m.put(held), m.put(held)
        group = [m.put(shared.first), m.put(shared.len)]
        for _ in range(4):
            provider.dispatch("flash_attention_paged_prefix", base + desc + group, [out, lb],
                              pc=pc_of(batch, kv, dim, n_heads=heads, step_idx=2))
            provider.dispatch("paged_kv_weights", base[:2] + desc + [lb, hb], [wb],
                              pc=pc_of(batch, kv, dim, n_heads=heads, step_idx=width, theta=1.0))
            seen.add(b"".join(b.read(np.uint8).tobytes() for b in (out, lb, wb)))
    assert len(seen) == 1


# ---- many sequences, padding, rows that count for nothing -------------------------------

RAGGED_HEADS = [  # types, sequences (positions, rows), positions that all share, heads, KV heads, head_dim
    ("f16", [(3 + i % 9, 3) for i in range(400)], 0, 96, 8, 64),
    ("f32", [(2 + i % 9, 2) for i in range(400)], 0, 96, 8, 64),
    ("f32", [(3 + i % 9, 3) for i in range(400)], 0, 48, 8, 64),
    ("f16", [(1000 if i < 30 else 10, 3) for i in range(100)], 0, 96, 8, 64),  # with splits, each workgroup finds its tile itself
    ("f16", [(35 + i % 3, 3) for i in range(700)], 32, 96, 8, 64),
    ("f16", [(5 + i % 3, 5) for i in range(1300)], 0, 28, 4, 64),
    ("f16", [(7 + i % 3, 7) for i in range(1400)], 0, 40, 8, 64),
    ("f16", [(11 + i % 3, 11) for i in range(1400)], 0, 24, 8, 64),
    ("f32", [(6 + i % 3, 6) for i in range(1400)], 0, 24, 8, 96),
]


@pytest.mark.parametrize("pool", ["rows", "i8"])
@pytest.mark.parametrize("act,seqs,share,heads,kv,dim", RAGGED_HEADS)
def test_prefix_heads_that_do_not_divide_a_tile(provider, act, pool, seqs, share, heads, kv, dim):
    """Many sequences whose query rows fill their tiles badly: every row is written; the first, the last and some others are
    held to the plain form."""
    pool = act if pool == "rows" else pool
    rng = np.random.default_rng(71)
    batch = ref.Batch(rng, seqs, 16, behind=3)
    shared = ref.Shared(batch, [(0, len(seqs), share)] if share else [])
    pools = fill(rng, batch, shared, act, pool, kv, dim)
    q = rows_of(rng, act, batch.rows, heads, dim)
    was = np.full_like(q, np.nan)
    with Bufs(provider) as m:
        out, lb = m.put(was), m.put(np.full((batch.rows, heads), np.nan, np.float32))
        provider.dispatch("flash_attention_paged_prefix", [m.put(q)] + [m.put(p) for p in pools] + m.batch(batch) +
                          [m.put(shared.first), m.put(shared.len)], [out, lb],
                          pc=pc_of(batch, kv, dim, n_heads=heads, step_idx=len(shared.groups)))
        got = out.read(NP[act], q.size).reshape(q.shape)
        z = lb.read(np.float32, batch.rows * heads).reshape(batch.rows, heads)
    mine = mine_of(batch)
    assert np.isfinite(got[mine]).all() and np.isfinite(z[mine]).all()
    assert np.isnan(got[~mine]).all() and np.isnan(z[~mine]).all()
    some = [0] + list(range(1, len(seqs) - 30, 37)) + list(range(len(seqs) - 30, len(seqs)))
    part = ref.Batch(rng, [(0, seqs[s][1]) for s in some], 16)
    part.lens, part.table, part.width, part.blocks = batch.lens[some], batch.table[some], batch.width, batch.blocks
    rows = np.concatenate([np.arange(batch.starts[s], batch.starts[s + 1]) for s in some])
    of = ref.Shared(part, [(0, len(some), share)] if share else [])
    want, err, wz, zerr = ref.attention(part, of, pool, dim, heads, kv, pools, q[rows], act)
    check(got[rows], want, err, (act, pool, heads, kv, seqs[:3]))
    check(z[rows], wz, zerr, ("lse", act, pool, heads, kv, seqs[:3]))


@pytest.mark.parametrize("act,pool", ACT_POOL)
@pytest.mark.parametrize("n,rows,heads,kv,dim,bs", [
    (200, 1, 8, 1, 64, 16), (77, 2, 8, 2, 128, 16), (700, 5, 4, 2, 96, 8), (33, 8, 4, 1, 64, 32), (1, 1, 16, 16, 128, 16),
    (5000, 3, 8, 1, 64, 16), (90, 0, 8, 2, 64, 16), (60, 4, 6, 4, 64, 16), (60, 2, 4, 2, 80, 16)])
def test_weights_of_one_padded_sequence(provider, act, pool, n, rows, heads, kv, dim, bs):
    """One sequence with few of the batch's rows, the others padding."""
    if pool == "i8" and dim % 32:
        pytest.skip("an 8-bit cache needs groups of 32")
    rng = np.random.default_rng(72)
    for behind in (7, 60, 300):
        batch = ref.Batch(rng, [(n, rows)], bs, behind=behind, before=behind % 2)
        q, pools, z = run_attention(provider, rng, batch, None, act, pool, heads, kv, dim, chunk=True)
        run_weights(provider, rng, batch, act, pool, heads, kv, dim, z, q, pools, theta=0.5)


@pytest.mark.parametrize("act,pool", ACT_POOL)
def test_captured_drafts_of_one_sequence(provider, act, pool):
    """A captured step of up to 16 drafts of one sequence is replayed with fewer of them, and with more again."""
    rng = np.random.default_rng(73)
    heads, kv, dim, bs, most = 8, 2, 64, 16, 16
    batch = ref.Batch(rng, [(400, most)], bs)
    pools, q, width = fill(rng, batch, None, act, pool, kv, dim), rows_of(rng, act, most, heads, dim), batch.width * bs
    held = rng.random((1, kv, width)).astype(np.float32)
    with Bufs(provider) as m:
        kb, desc, qb, hb = [m.put(p) for p in pools], m.batch(batch), m.put(q), m.put(held)
        out, lb, wb = m.put(np.zeros_like(q)), m.put(np.zeros((most, heads), np.float32)), m.put(held)
        tasks = (abi.nf_task_desc * 2)(
            provider.task("flash_attention_paged_chunk", [qb] + kb + desc, [out, lb], pc=pc_of(batch, kv, dim, n_heads=heads)),
            provider.task("paged_kv_weights", [qb, kb[0]] + desc + [lb, hb], [wb],
                          pc=pc_of(batch, kv, dim, n_heads=heads, step_idx=width, theta=0.5)))
        graph = hiprt.Graph(provider.stream(), lambda: provider.run_tasks(tasks))
        for n, rows in ((400, 16), (300, 1), (399, 8), (17, 9), (1, 1), (400, 16)):
            batch.seqs, batch.lens, batch.starts = [(n, rows)], np.array([n], np.int32), np.array([0, rows], np.int32)
            desc[1].write(batch.starts)
            desc[2].write(batch.lens)
            wb.write(np.full_like(held, 3.0))
            graph.launch()
            z, w = lb.read(np.float32, most * heads).reshape(most, heads), wb.read(np.float32, held.size).reshape(held.shape)
            want, err = ref.weights(batch, pool, dim, heads, kv, pools[0], q, act, z, held, 0.5, np.full_like(held, 3.0))
            check(w, want, err, (n, rows))
            wb.write(np.full_like(held, 3.0))
            provider.run_tasks(tasks)
            assert np.array_equal(wb.read(np.float32, held.size).reshape(held.shape), w)


@pytest.mark.parametrize("act,pool", ACT_POOL)
@pytest.mark.parametrize("n,dim,bs,width", [(4096, 64, 16, 8192), (4500, 128, 16, 8192), (4096, 96, 8, 16384), (4096, 80, 16, 300),
                                            (4096, 64, 16, 0)])
def test_weights_of_many_rows_keep_their_bits(provider, act, pool, n, dim, bs, width):
    """Each of 4096 rows gives the same weight, so that every rounding of a long sum may go the same way: a sum may be off by
    as many of them as there are tiles of 32 query rows, and some for what is within one, not by one for each row."""
    if pool == "i8" and dim % 32:
        pytest.skip("an 8-bit cache needs groups of 32")
    rng = np.random.default_rng(74)
    heads, kv, rows = 16, 2, 4096
    batch = ref.Batch(rng, [(n, rows)], bs, width=width)
    pools, q = fill(rng, batch, None, act, pool, kv, dim), np.zeros((rows, heads, dim), NP[act])  # all score 0
    lse = np.tile(np.repeat(np.array([3.4887, 0.5843], np.float32), 8), (rows, 1))
    held = np.zeros((1, kv, batch.width * bs), np.float32)
    with Bufs(provider) as m:
        wb = m.put(held)
        provider.dispatch("paged_kv_weights", [m.put(q), m.put(pools[0])] + m.batch(batch) + [m.put(lse), m.put(held)], [wb],
                          pc=pc_of(batch, kv, dim, n_heads=heads, step_idx=held.shape[2]))
        got = wb.read(np.float32, held.size).reshape(held.shape)[0, :, :n].astype(np.float64)
    # the weight as the kernel has it: the last position has one token's, a sum of 8, off by 8 roundings at most
    one = got[:, -1] / 8
    assert np.allclose(one, np.exp(-lse[0, ::8].astype(np.float64)), rtol=2e-6, atol=0)
    want = one[:, None] * (8.0 * np.minimum(n - np.arange(n), rows))
    check(got, want, (8 * rows / 32 + 32 + 8) * paged_ref.U * want, (act, pool, n, dim))


@pytest.mark.parametrize("act,pool", ACT_POOL)
@pytest.mark.parametrize("seqs,heads,kv,dim", [
    ([(300, 1), (90, 2), (64, 4)], 8, 2, 64), ([(300, 90), (200, 64), (33, 33)], 8, 2, 128), ([(400, 130)], 4, 1, 96),
    ([(700, 40), (90, 2)], 16, 2, 64), ([(90, 20), (60, 1)], 4, 2, 40), ([(600, 500)], 8, 1, 64)])
def test_weights_of_rows_that_count_for_nothing(provider, act, pool, seqs, heads, kv, dim):
    """Rows whose log-sum-exp is -inf give nothing, whatever their queries hold."""
    if pool == "i8" and dim % 32:
        pytest.skip("an 8-bit cache needs groups of 32")
    rng = np.random.default_rng(75)
    batch = ref.Batch(rng, seqs, 16, behind=2)
    q, pools, z = run_attention(provider, rng, batch, None, act, pool, heads, kv, dim, chunk=True)
    none = rng.random(z.shape) < 0.15
    none[batch.starts[1:] - 1] |= rng.random((len(seqs), heads)) < 0.5  # the last rows of the sequences among them
    z = np.where(none, -np.inf, z).astype(np.float32)
    bad = q.copy()
    bad[none] = rng.choice([np.nan, np.inf, -np.inf, 6e4], (int(none.sum()), dim)).astype(NP[act])
    plain = run_weights(provider, np.random.default_rng(5), batch, act, pool, heads, kv, dim, z, np.where(none[..., None], NP[act](0), q), pools)
    width = batch.width * batch.bs
    held = np.random.default_rng(5).random((len(seqs), kv, width)).astype(np.float32)
    with Bufs(provider) as m:
        wb = m.put(np.full_like(held, 9.0))
        provider.dispatch("paged_kv_weights", [m.put(bad), m.put(pools[0])] + m.batch(batch) + [m.put(z), m.put(held)], [wb],
                          pc=pc_of(batch, kv, dim, n_heads=heads, step_idx=width, theta=1.0))
        got = wb.read(np.float32, held.size).reshape(held.shape)
    assert np.isfinite(got).all()
    assert np.array_equal(got, plain)


@pytest.mark.parametrize("act,pool", [("f16", "f16"), ("f32", "f32"), ("f16", "i8")])
@pytest.mark.parametrize("op,lens,share", [("chunk", [0x7FFFF000], 0), ("chunk", [0x7FFFEF81], 0), ("prefix", [1 << 30, (1 << 30) - 77], (1 << 30) - 200),
                                           ("prefix", [1 << 30], (1 << 30) - 9)])
def test_as_many_positions_as_there_may_be(provider, act, pool, op, lens, share):
    """Sequences of the most positions, all in one block: keys of equal scores, of which none may be lost."""
    rng = np.random.default_rng(76)
    dim, bs, n = 64, 65536, len(lens)
    pages = -(-max(lens) // bs)
    batch = ref.Batch(rng, [(1, 1)] * n, bs)
    batch.blocks, batch.width, batch.table = 1, pages, np.zeros((n, pages), np.uint32)
    batch.lens = np.array(lens, np.int32)
    value = rng.choice([-1.0, 1.0], dim).astype(NP[act])
    pools = [paged_ref.empty_pool(rng, pool, 1, 1, bs, dim) for _ in range(2)]
    if pool == "i8":
        pools[1][0, 0, :bs * dim] = np.tile((64 * value).astype(np.int8).view(np.uint8), bs)
        pools[1][0, 0, bs * dim:] = np.full(bs * dim // 32, 2.0 ** -6, np.float16).view(np.uint8)
    else:
        pools[1][:] = value
    with Bufs(provider) as m:
        out, lb = m.put(np.zeros((n, 1, dim), NP[act])), m.put(np.zeros((n, 1), np.float32))
        ins = [m.put(np.zeros((n, 1, dim), NP[act]))] + [m.put(x) for x in pools] + m.batch(batch)
        more = {}
        if op == "prefix":
            ins += [m.put(np.array([0, n], np.int32)), m.put(np.array([share], np.int32))]
            more["step_idx"] = 1
        provider.dispatch("flash_attention_paged_" + op, ins, [out, lb],
                          pc=pc_of(batch, 1, dim, n_heads=1, max_seq_len=1 << 30 if op == "prefix" else 0, **more))
        got, z = out.read(NP[act], n * dim).reshape(n, dim), lb.read(np.float32, n)
    # Sums of weights of 1 or 2^7, 32 or more at a time, are exact; the combination of up to 512 splits may round each, and
    # the logarithm its parts, of up to 32.
    check(z, np.log(np.array(lens, np.float64)), (512 + 6 * 32 + 16) * paged_ref.U, (op, act, pool))
    check(got, np.tile(value.astype(np.float64), (n, 1)), 600 * paged_ref.U + (0 if act == "f32" else paged_ref.H), (op, act, pool))


@pytest.mark.parametrize("act,pool", ACT_POOL)
@pytest.mark.parametrize("seqs,heads,kv,dim", [([(300, 3), (90, 2)], 8, 2, 64), ([(300, 90), (200, 64), (33, 33)], 8, 2, 128),
                                               ([(90, 20), (60, 1)], 4, 2, 40), ([(600, 500)], 8, 1, 64)])
def test_weights_of_rows_without_a_number(provider, act, pool, seqs, heads, kv, dim):
    """A row whose log-sum-exp is NaN leaves NaN at the positions that it sees, and its KV head's others as they are without it."""
    if pool == "i8" and dim % 32:
        pytest.skip("an 8-bit cache needs groups of 32")
    rng = np.random.default_rng(77)
    batch = ref.Batch(rng, seqs, 16, behind=2)
    q, pools, z = run_attention(provider, rng, batch, None, act, pool, heads, kv, dim, chunk=True)
    r, h = int(batch.starts[0]) + seqs[0][1] // 2, heads - 1
    pos = seqs[0][0] - seqs[0][1] + seqs[0][1] // 2
    width = batch.width * batch.bs
    held = rng.random((len(seqs), kv, width)).astype(np.float32)
    got = []
    with Bufs(provider) as m:
        base, wb, hb = [m.put(q), m.put(pools[0])] + m.batch(batch), m.put(held), m.put(held)
        for x in (-np.inf, np.nan):
            lse = z.copy()
            lse[r, h] = x
            wb.write(held)
            provider.dispatch("paged_kv_weights", base + [m.put(lse), hb], [wb],
                              pc=pc_of(batch, kv, dim, n_heads=heads, step_idx=width, theta=1.0))
            got.append(wb.read(np.float32, held.size).reshape(held.shape))
    want = got[0].copy()
    want[0, kv - 1, :pos + 1] = np.nan
    assert np.isfinite(got[0]).all() and np.array_equal(got[1], want, equal_nan=True)
