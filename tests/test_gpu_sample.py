"""sample_token on the GPU against its definition: weights rint(2^40 exp((x - max) / T)) from 64-bit arithmetic, sums of
Python integers.  The tokens have to be the same; the probabilities are one rounding to f32 off (half a step, 2^-24, and
2^-40 / w for a weight whose last bit the two exponentials may round differently)."""
import math

import numpy as np
import pytest

from neurofabric_amd import abi
from neurofabric_amd.plugin import push_constants

pytestmark = [pytest.mark.gpu, pytest.mark.filterwarnings("ignore::RuntimeWarning")]

ONE = 1 << 40


def reference(x, u, temp, top_p, min_p, k):
    """(token, probability) of one row."""
    x = np.asarray(x, np.float64)
    x = np.where(np.isnan(x), -np.inf, np.minimum(x, np.finfo(np.float32).max))
    live = np.flatnonzero(x > -np.inf)
    if not len(live):
        return -1, 0.0
    top = x[live].max()
    temp = min(temp, np.float32(1e30))
    if not temp > 0:
        return int(live[np.argmax(x[live])]), 1.0
    order = live[np.argsort(-x[live], kind="stable")]
    w = [int(v) for v in np.rint(np.exp((x[order] - top) / np.float64(np.float32(temp))) * ONE)]
    if 0 < k < len(x):
        order, w = order[:k], w[:k]
    if top_p < 1:
        goal = float(np.float32(top_p)) * float(sum(w))
        n, run = 0, 0
        while n < len(w) and (n == 0 or float(run) < goal):
            run += w[n]
            n += 1
        order, w = order[:n], w[:n]
    kept = sorted((int(o), v) for o, v in zip(order, w) if not v < min(float(np.float32(min_p)), 1.0) * ONE)
    total = sum(v for _, v in kept)
    t = min(max(math.floor(float(np.float32(u)) * float(total)), 0), total - 1) if u == u else 0
    run = 0
    for o, v in kept:
        run += v
        if run > t:
            return o, v / total
    raise AssertionError


def draw(provider, x, u, params, k):
    rows, n = x.shape
    bufs = [provider.alloc_array(a, d) for a, d in
            ((x, abi.NF_DTYPE_F16 if x.dtype == np.float16 else abi.NF_DTYPE_F32), (u, abi.NF_DTYPE_F32),
             (params, abi.NF_DTYPE_F32), (k, abi.NF_DTYPE_I32))]
    outs = [provider.alloc(abi.NF_DTYPE_I32, rows * 4), provider.alloc(abi.NF_DTYPE_F32, rows * 4)]
    provider.dispatch("sample_token", bufs, outs, pc=push_constants(seq_len=rows, N=n))
    got = outs[0].read(np.int32), outs[1].read(np.float32)
    for b in bufs + outs:
        b.release()
    return got


def check(provider, x, u, params, k):
    u, params, k = np.asarray(u, np.float32), np.asarray(params, np.float32).reshape(-1, 3), np.asarray(k, np.int32)
    token, prob = draw(provider, x, u, params, k)
    for r in range(len(x)):
        want, p = reference(x[r], u[r], *params[r], int(k[r]))
        assert token[r] == want, (r, token[r], want, u[r], params[r], k[r])
        assert abs(float(prob[r]) - p) <= 2.0 ** -24 * p + 2.0 ** -39, (r, prob[r], p)


HOW = [(1.0, 1.0, 0.0, 0), (0.8, 0.95, 0.0, 40), (0.7, 0.9, 0.0, 0), (1.3, 1.0, 0.05, 0), (0.0, 0.5, 0.5, 3),
       (0.9, 0.97, 0.02, 200), (5.0, 0.999, 0.0, 0), (0.05, 0.3, 0.9, 1), (1.0, 0.0, 0.0, 7), (2.0, 0.6, 0.0, 5000)]


@pytest.mark.parametrize("dtype", [np.float32, np.float16])
@pytest.mark.parametrize("n", [1, 2, 63, 64, 65, 1000, 1025, 4097, 32000, 50257, 128256])
def test_sample(provider, n, dtype):
    rng = np.random.default_rng(n)
    rows = 20
    x = (rng.standard_normal((rows, n)) * rng.choice([0.1, 2.5, 8.0], (rows, 1))).astype(dtype)
    u = rng.random(rows).astype(np.float32)
    u[:3] = 0.0, np.nextafter(np.float32(1), np.float32(0)), 0.5
    how = [HOW[i % len(HOW)] for i in range(rows)]
    check(provider, x, u, [h[:3] for h in how], [h[3] for h in how])


@pytest.mark.parametrize("rows,n", [(3, 70000), (8, 131072), (300, 70001)])
def test_cuts_of_every_size(provider, rows, n):
    """top_k from one to nearly all with and without the other cuts, rows that are and are not spread over workgroups."""
    rng = np.random.default_rng(n)
    x = (rng.standard_normal((rows, n)) * 3).astype(np.float32)
    ks = [1, 2, 63, 64, 65, 255, 256, 257, 300, 1024, 2047, 2048, 2049, 5000, 40000, n - 1, n, n + 5, 0]
    ps = [1.0, 0.9, 0.5, 0.999999, 1e-6]
    how = [(ks[(7 * i + 3) % len(ks)], ps[i % 5], [0.0, 0.0, 1e-7, 0.2][i % 4], [0.6, 1.0, 3.0][i % 3]) for i in range(rows)]
    check(provider, x, rng.random(rows).astype(np.float32), [(t, p, m) for _, p, m, t in how], [h[0] for h in how])


def test_one_more_row_after_another(provider):
    """The same rows alone, together and again give the same tokens."""
    rng = np.random.default_rng(2)
    n = 66000
    x = (rng.standard_normal((5, n)) * 2).astype(np.float32)
    u = rng.random(5).astype(np.float32)
    params = np.array([[1.0, 0.99, 0.0], [0.7, 0.9, 0.0], [1.0, 1.0, 0.0], [1.0, 1.0, 0.1], [0.5, 0.8, 0.0]], np.float32)
    k = np.array([0, 50, 0, 0, 3000], np.int32)
    together = [draw(provider, x, u, params, k) for _ in range(3)]
    for t in together[1:]:
        assert np.array_equal(t[0], together[0][0]) and np.array_equal(t[1], together[0][1])
    for r in range(5):
        t, p = draw(provider, x[r:r + 1], u[r:r + 1], params[r:r + 1], k[r:r + 1])
        assert t[0] == together[0][0][r] and p[0] == together[0][1][r]


def test_captured(provider):
    """A captured draw follows its buffers at each replay."""
    from neurofabric_amd import hiprt
    rng = np.random.default_rng(4)
    rows, n = 3, 70000
    bufs = [provider.alloc(abi.NF_DTYPE_F32, rows * n * 4), provider.alloc(abi.NF_DTYPE_F32, rows * 4),
            provider.alloc(abi.NF_DTYPE_F32, rows * 12), provider.alloc(abi.NF_DTYPE_I32, rows * 4)]
    outs = [provider.alloc(abi.NF_DTYPE_I32, rows * 4), provider.alloc(abi.NF_DTYPE_F32, rows * 4)]
    pc = push_constants(seq_len=rows, N=n)
    tasks = (abi.nf_task_desc * 1)(provider.task("sample_token", bufs, outs, pc=pc))
    graph = hiprt.Graph(provider.stream(), lambda: provider.run_tasks(tasks))
    for i in range(4):
        x = (rng.standard_normal((rows, n)) * 2).astype(np.float32)
        u = rng.random(rows).astype(np.float32)
        params = np.array([[1.0, 0.9, 0.0], [0.8, 1.0, 0.01 * i], [0.9, 0.95, 0.0]], np.float32)
        k = np.array([0, 0, 40 * i], np.int32)
        for b, a in zip(bufs, (x, u, params, k)):
            b.write(a)
        graph.launch()
        token, prob = outs[0].read(np.int32), outs[1].read(np.float32)
        for r in range(rows):
            want, p = reference(x[r], u[r], *params[r], int(k[r]))
            assert token[r] == want and abs(float(prob[r]) - p) <= 2.0 ** -24 * p + 2.0 ** -39
        provider.dispatch("sample_token", bufs, outs, pc=pc)
        assert np.array_equal(outs[0].read(np.int32), token)
    for b in bufs + outs:
        b.release()


@pytest.mark.parametrize("n", [5, 3000, 40000, 70000])
def test_ties(provider, n):
    """Few distinct values: the lowest indices stay at every cut."""
    rng = np.random.default_rng(n)
    rows = 24
    x = rng.integers(-2, 3, (rows, n)).astype(np.float32)
    x[:6] = 1.5
    x[6:9, ::2] = -0.0
    x[6:9, 1::2] = 0.0
    u = rng.random(rows).astype(np.float32)
    how = [((1.0, 0.5, 0.0), 0), ((1.0, 1.0, 0.0), n // 3 + 1), ((0.7, 0.3, 0.1), n // 2), ((0.0, 1.0, 0.0), 0),
           ((1.0, 0.25, 0.0), 2), ((2.0, 0.9, 0.5), 0), ((1.0, 1e-9, 0.0), 0)]
    check(provider, x, u, [how[r % 7][0] for r in range(rows)], [how[r % 7][1] for r in range(rows)])


def test_borders_of_the_random_number(provider):
    """Two and four equal tokens split [0, 1) evenly; values outside it take the first or the last."""
    x = np.full((9, 4), -np.inf, np.float32)
    x[:, [1, 3]] = 3.0
    below = np.nextafter(np.float32(0.5), np.float32(0))
    u = [0.0, below, 0.5, 0.75, 1.0, 7.0, -1.0, np.nan, np.inf]
    token, prob = draw(provider, x, np.array(u, np.float32), np.tile(np.float32([1, 1, 0]), (9, 1)), np.zeros(9, np.int32))
    assert token.tolist() == [1, 1, 3, 3, 3, 3, 1, 1, 3] and np.all(prob == 0.5)


def test_not_finite(provider):
    """NaN and -inf are never drawn, +inf counts as the largest finite logit, and a row of nothing gives -1."""
    rng = np.random.default_rng(3)
    x = (rng.standard_normal((12, 700)) * 3).astype(np.float32)
    x[0] = np.nan
    x[1] = -np.inf
    x[2, ::3], x[2, 1::3] = np.nan, -np.inf
    x[3, [5, 9]] = np.inf
    x[4], x[4, 650] = -np.inf, -200.0
    x[5, 3] = np.nan
    x[6] = np.nan
    x[6, 1] = -3.4e38
    x[7, 8] = 3.4e38
    params = np.tile(np.float32([0.9, 0.9, 0.01]), (12, 1))
    params[8:] = [[np.nan, 0.9, 0.0], [-1, 1, 0], [1, np.nan, np.nan], [np.inf, 1, 2.0]]
    check(provider, x, rng.random(12).astype(np.float32), params, [0, 5, 10, 0, 3, 50, 0, 0, 0, 0, -4, 2000])


def test_extreme_temperatures_and_logits(provider):
    """Differences that overflow f32, temperatures whose products and quotients do."""
    big = np.finfo(np.float32).max
    base = np.array([big, -big, 0.0, np.nan, -np.inf, 1.0, big, -1.0, 1e-45, 3e38], np.float32)
    temps = [np.inf, 3.4e38, 1e30, 1e25, 1.0, 1e-30, 1e-45]
    x = np.stack([base] * len(temps) + [np.where(np.abs(base) > 2, np.float32(0.5), base)] * len(temps))
    x[len(temps):, [3, 4]] = np.nan, -np.inf
    u = np.linspace(0.05, 0.95, len(x)).astype(np.float32)
    for p, k in ((1.0, 0), (0.7, 0), (1.0, 3), (0.5, 5)):
        check(provider, x, u, [(t, p, 0.0) for t in temps * 2], [k] * len(x))


@pytest.mark.parametrize("dtype", [np.float32, np.float16])
def test_frequencies(provider, dtype):
    """4096 rows of the same logits at evenly spread random numbers: counts follow the weights to within one each."""
    n, rows = 50, 4096
    x = (np.random.default_rng(1).standard_normal(n) * 1.5).astype(dtype)
    u = ((np.arange(rows) + 0.5) / rows).astype(np.float32)
    token, _ = draw(provider, np.tile(x, (rows, 1)), u, np.tile(np.float32([1, 1, 0]), (rows, 1)), np.zeros(rows, np.int32))
    p = np.exp(x.astype(np.float64))
    assert np.abs(np.bincount(token, minlength=n) - rows * p / p.sum()).max() <= 1.0


@pytest.mark.parametrize("rows,n", [(3, 65536), (2, 40001), (4, 16384), (4, 16385), (5, 20011), (260, 16400)])
def test_cuts_of_short_rows(provider, rows, n):
    """Few and many rows on both sides of the lengths from which rows are spread over workgroups."""
    rng = np.random.default_rng(n + rows)
    x = (rng.standard_normal((rows, n)) * 3).astype(np.float32)
    ks = [0, 40, 300, 3000, 12000, 0, 1, 256]
    ps = [0.9, 1.0, 0.95, 0.999, 0.5]
    how = [(ks[(i + n) % len(ks)], ps[i % 5], [0.0, 0.05, 0.0][i % 3], [1.0, 0.7, 4.0, 0.0][i % 4]) for i in range(rows)]
    check(provider, x, rng.random(rows).astype(np.float32), [(t, p, m) for _, p, m, t in how], [h[0] for h in how])
