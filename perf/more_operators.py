"""Performance cases of the operators for long contexts over the paged cache: attention of sequences that share a prefix,
the attention weights that the cache's positions gather, and eviction by them.

Kinds of case:
  prefix   flash_attention_paged_prefix: sequences in groups, each group's first positions in the same blocks
  weights  paged_kv_weights: the rows' attention weights added up for each cached position, from their log-sum-exp
  score    flash_attention_paged_chunk with the log-sum-exp of its rows, then paged_kv_weights, as a layer runs them
  evict    paged_kv_evict: the positions of largest weight and the latest ones, moved to blocks of their own

A batch is `seqs` sequences; the last `chunk` positions (at most) of each are the new rows.  `ragged` spreads lengths over
the sequences by a fixed rule.  The pools' blocks are handed out in a random order.
"""
import math
import random

import numpy as np
import torch

own = False

TORCH = {"f32": torch.float32, "f16": torch.float16}
SIZE = {"f32": 4, "f16": 2}


def listed():
    llama = {"heads": 32, "kv": 8, "dim": 128, "block": 16}
    small = {"heads": 32, "kv": 4, "dim": 64, "block": 16}
    return [
        # Four answers to one short instruction, a token each, f32: the smallest call of the attention, latency counts.
        {"name": "prefix_f32_short", "kind": "prefix", "act": "f32", "pool": "f32", "seqs": 4, "groups": 1, "prefix": 96,
         "tail": 30, "chunk": 1, "ragged": True, **small},
        # A decode step of 64 conversations behind one system prompt of 8192 tokens.
        {"name": "prefix_decode_f16", "kind": "prefix", "act": "f16", "pool": "f16", "seqs": 64, "groups": 1,
         "prefix": 8192, "tail": 512, "chunk": 1, "ragged": True, **llama},
        # 32 questions about one long document in the 8-bit cache, a token each.
        {"name": "prefix_decode_i8_long", "kind": "prefix", "act": "f16", "pool": "i8", "seqs": 32, "groups": 1,
         "prefix": 32768, "tail": 1024, "chunk": 1, "ragged": True, **llama},
        # Five drafted tokens of each of 32 sequences behind four prompts.
        {"name": "prefix_verify_f16", "kind": "prefix", "act": "f16", "pool": "f16", "seqs": 32, "groups": 4,
         "prefix": 4096, "tail": 300, "chunk": 5, "ragged": True, **llama},
        # Questions of up to 200 tokens read in behind a document of 8192: the largest attention.
        {"name": "prefix_chunk_f16", "kind": "prefix", "act": "f16", "pool": "f16", "seqs": 16, "groups": 1,
         "prefix": 8192, "tail": 200, "chunk": 200, "ragged": True, **llama},
        # A decode step of one short sequence that also gathers its weights, f32: latency counts.
        {"name": "score_f32_short", "kind": "score", "act": "f32", "pool": "f32", "seqs": 1, "chunk": 1, "ctx": 100,
         "ragged": False, "theta": 1.0, **small},
        # The weights of a decode step of 64 sequences of up to 8192 tokens.
        {"name": "weights_decode_f16", "kind": "weights", "act": "f16", "pool": "f16", "seqs": 64, "chunk": 1, "ctx": 8192,
         "ragged": True, "theta": 1.0, **llama},
        # The same of 16 sequences of up to 32768 tokens in the 8-bit cache, older steps' weights fading.
        {"name": "weights_decode_i8", "kind": "weights", "act": "f16", "pool": "i8", "seqs": 16, "chunk": 1, "ctx": 32768,
         "ragged": True, "theta": 0.99, **llama},
        # The weights that the last 2048 tokens of two prompts of 8192 give all of their positions.
        {"name": "weights_prompt_f16", "kind": "weights", "act": "f16", "pool": "f16", "seqs": 2, "chunk": 2048,
         "ctx": 8192, "ragged": False, "theta": 0.0, **llama},
        # One short f32 sequence cut to 512 positions: the smallest eviction.
        {"name": "evict_f32_short", "kind": "evict", "act": "f32", "pool": "f32", "seqs": 1, "ctx": 600, "keep": 512,
         "recent": 64, "ragged": False, **small},
        # 32 sequences of up to 4096 positions cut to 1024 of them.
        {"name": "evict_f16_batch", "kind": "evict", "act": "f16", "pool": "f16", "seqs": 32, "ctx": 4096, "keep": 1024,
         "recent": 128, "ragged": True, **llama},
        # Two very long sequences in the 8-bit cache cut to a quarter.
        {"name": "evict_i8_long", "kind": "evict", "act": "f16", "pool": "i8", "seqs": 2, "ctx": 131072, "keep": 32768,
         "recent": 4096, "ragged": False, **llama},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(max(lo, hi))))))


def draw(rng):
    kind = rng.choice(["prefix", "prefix", "weights", "score", "evict", "evict"])
    act = rng.choice(["f32", "f16"])
    c = {"kind": kind, "act": act, "pool": rng.choice([act, "i8"]), "kv": rng.choice([1, 2, 4, 8]),
         "dim": rng.choice([64, 64, 128, 128, 96]), "block": rng.choice([8, 16, 16, 32]), "ragged": rng.random() < 0.7}
    c["heads"] = c["kv"] * rng.choice([1, 2, 4, 4, 8])
    if kind == "evict":
        c["seqs"] = _log(rng, 1, 32)
        c["ctx"] = _log(rng, 16, 131072 // c["seqs"])
        c["keep"] = max(1, int(c["ctx"] * rng.uniform(0.05, 0.9)))
        c["recent"] = int(c["keep"] * rng.uniform(0.0, 0.6))
        return c
    c["chunk"] = _log(rng, 1, 512)
    c["seqs"] = _log(rng, 1, max(1, min(64, 1024 // c["chunk"])))
    if kind == "prefix":
        c["groups"] = min(c["seqs"], rng.choice([1, 1, 1, 2, 3, 5]))
        c["prefix"] = _log(rng, 32, 8192)
        c["tail"] = max(c["chunk"], _log(rng, 1, 1024))
        return c
    c["ctx"] = max(c["chunk"], _log(rng, 16, 8192 if c["seqs"] > 1 or c["chunk"] > 1 else 65536))
    c["theta"] = rng.choice([0.0, 1.0, 1.0, 0.9])
    return c


# ---- batches -------------------------------------------------------------------

def _spread(case, i):
    return (i * 0.6180339887 + 0.25) % 1.0 if case["ragged"] and i else 0.0


def _groups(case):
    """[(first sequence, one past the last, shared positions)]: whole blocks of them."""
    n, k = case["seqs"], case["groups"]
    out = []
    for g in range(k):
        p = case["prefix"] - int(0.5 * _spread(case, g) * case["prefix"])
        out.append((n * g // k, n * (g + 1) // k, max(1, p // case["block"]) * case["block"]))
    return out


def _lens(case):
    """[(cached positions, new ones among them)] of the batch's sequences."""
    out = []
    if case["kind"] == "prefix":
        for first, last, p in _groups(case):
            for i in range(first, last):
                n = max(1, case["chunk"] - int(0.5 * _spread(case, i) * case["chunk"]))
                out.append((p + max(n, case["tail"] - int(0.75 * _spread(case, i) * case["tail"])), n))
        return out
    chunk = case.get("chunk", 1)
    for i in range(case["seqs"]):
        n = max(1, chunk - int(0.5 * _spread(case, i) * chunk))
        out.append((max(n, case["ctx"] - int(0.75 * _spread(case, i) * case["ctx"])), n))
    return out


def _budget(case):
    """[(positions, kept, latest among those)] of an eviction's sequences."""
    return [(n, min(n, case["keep"]), min(n, case["keep"], case["recent"])) for n, _ in _lens(case)]


class State:
    def __init__(self, case, seed):
        self.case = case
        self.gen = torch.Generator(device="cuda").manual_seed(seed)
        self.tasks = None
        self.handles = []

    def normal(self, act, *shape):
        return torch.randn(shape, generator=self.gen, device="cuda").to(TORCH[act])

    def __del__(self):
        for b in self.handles:
            b.release()


def _pool(s, blocks):
    case = s.case
    kv, d, bs = case["kv"], case["dim"], case["block"]
    if case["pool"] != "i8":
        return s.normal(case["pool"], blocks, kv, bs, d)
    codes = torch.randint(-127, 128, (blocks, kv, bs * d), generator=s.gen, device="cuda", dtype=torch.int8)
    scales = (0.02 + 0.01 * torch.rand(blocks, kv, bs * d // 32, generator=s.gen, device="cuda")).half()
    return torch.cat([codes.view(torch.uint8), scales.view(torch.uint8)], 2).contiguous()


def _gathered(s, *shape):
    """Weights as they gather: a few positions hold most, many hold next to nothing, some are equal."""
    w = torch.exp(2.0 * torch.randn(shape, generator=s.gen, device="cuda") - 4.0)
    return torch.where(w < 0.004, torch.round(w * 1000) / 1000, w)


def prepare(case, seed):
    s = State(case, seed)
    _prepare_batch(s, seed)
    if own:
        _bind(s)
    torch.cuda.synchronize()  # the provider's stream does not wait for torch's
    return s


def _prepare_batch(s, seed):
    case = s.case
    act, kv, d, bs, kind = case["act"], case["kv"], case["dim"], case["block"], case["kind"]
    lens = _lens(case)
    starts = [0]
    for _, n in lens:
        starts.append(starts[-1] + n)
    shared = [0] * len(lens)  # blocks that a sequence takes from its group's first
    if kind == "prefix":
        for first, last, p in _groups(case):
            for i in range(first + 1, last):
                shared[i] = p // bs
    pages = [-(-length // bs) for length, _ in lens]
    new = [-(-k // bs) for _, k, _ in _budget(case)] if kind == "evict" else []
    blocks = sum(pages) - sum(shared) + sum(new) + 3  # three that belong to no sequence
    order = list(range(blocks))
    random.Random(seed).shuffle(order)
    table = np.full((len(lens), max(pages)), -1, np.int32)
    at = 0
    for i, n in enumerate(pages):
        if shared[i]:
            table[i, :shared[i]] = table[i - 1, :shared[i]]
        table[i, shared[i]:n] = order[at:at + n - shared[i]]
        at += n - shared[i]
    dev = lambda a: torch.tensor(a, dtype=torch.int32, device="cuda")  # noqa: E731
    s.table, s.starts, s.lens = dev(table), dev(starts), dev([length for length, _ in lens])
    s.rows, s.most, s.longest = starts[-1], max(n for _, n in lens), max(length for length, _ in lens)
    s.kpool, s.vpool = _pool(s, blocks), _pool(s, blocks)
    zeros = lambda *shape: torch.zeros(shape, dtype=torch.float32, device="cuda")  # noqa: E731
    if kind == "evict":
        s.top = max(k for _, k, _ in _budget(case))
        moved = np.full((len(lens), -(-s.top // bs)), -1, np.int32)
        for i, n in enumerate(new):
            moved[i, :n] = order[at:at + n]
            at += n
        s.moved = dev(moved)
        s.budget = dev([[case["keep"], case["recent"]] for _ in lens])
        s.held = _gathered(s, len(lens), kv, s.longest)
        s.weights = zeros(len(lens), kv, s.longest)
        s.new_lens = dev([0] * len(lens))
        s.kept = torch.zeros(len(lens), kv, s.top, dtype=torch.int32, device="cuda")
        return
    s.q = s.normal(act, s.rows, case["heads"], d)
    s.out = torch.zeros_like(s.q)
    if kind == "prefix":
        s.groups = dev([first for first, _, _ in _groups(case)] + [len(lens)])
        s.prefixes = dev([p for _, _, p in _groups(case)])
        return
    s.held = _gathered(s, len(lens), kv, s.longest)
    s.weights = zeros(len(lens), kv, s.longest)
    s.lse = zeros(s.rows, case["heads"])
    if kind == "weights":  # the attention gave it
        s.lse = _plain_lse(s, _plain_scores(s))


def run(state):
    if own:
        return _run_own(state)
    kind = state.case["kind"]
    if kind == "evict":
        return _plain_evict(state)
    if kind == "weights":
        return [_plain_weights(state, _plain_scores(state), state.lse)]
    if kind == "prefix":
        return [_plain_attention(state, _plain_scores(state))]
    scores = _plain_scores(state)
    lse = _plain_lse(state, scores)
    return [_plain_attention(state, scores), lse, _plain_weights(state, scores, lse)]


# ---- the framework's operators ---------------------------------------------------

_provider = None


def _bind(s):
    """The provider's handles on the state's tensors, and its prepared tasks."""
    import ctypes

    from neurofabric_amd import abi, plugin

    global _provider
    if _provider is None:
        _provider = plugin.Provider()
        _provider.init()
    s.prov, case = _provider, s.case
    kinds = {torch.float32: abi.NF_DTYPE_F32, torch.float16: abi.NF_DTYPE_F16, torch.int32: abi.NF_DTYPE_I32,
             torch.uint8: abi.NF_DTYPE_I8}

    def h(t):
        desc = abi.make_desc(kinds[t.dtype], t.numel() * t.element_size())
        ops, handle = abi.nf_buffer_ops(), ctypes.c_void_p()
        s.prov.check(s.prov.mem.import_buffer(s.prov.handle, t.data_ptr(), abi.NF_MEM_DOMAIN_DEVICE, ctypes.byref(desc),
                                              ctypes.byref(ops), ctypes.byref(handle)), "import_buffer")
        s.handles.append(plugin.Buffer(s.prov, handle.value, ops, desc.dtype, desc.size_bytes))
        return s.handles[-1]

    pools = [h(s.kpool), h(s.vpool)]
    args = dict(M=case["kv"], N=s.table.shape[1], K=case["seqs"], head_dim=case["dim"], window_size=case["block"],
                max_seq_len=s.longest)
    tasks = []
    if case["kind"] == "evict":
        pc = plugin.push_constants(seq_len=s.top, step_idx=s.longest, **args)
        tasks.append(s.prov.task("paged_kv_evict", pools + [h(s.held), h(s.table), h(s.lens), h(s.budget), h(s.moved)],
                                 pools + [h(s.weights), h(s.new_lens), h(s.kept)], pc=pc))
    else:
        args.update(seq_len=s.rows, n_heads=case["heads"])
        q, out, batch = h(s.q), h(s.out), [h(s.table), h(s.starts), h(s.lens)]
        if case["kind"] == "prefix":
            pc = plugin.push_constants(step_idx=case["groups"], **args)
            tasks.append(s.prov.task("flash_attention_paged_prefix", [q] + pools + batch + [h(s.groups), h(s.prefixes)],
                                     [out], pc=pc))
        else:
            lse = h(s.lse)
            if case["kind"] == "score":
                tasks.append(s.prov.task("flash_attention_paged_chunk", [q] + pools + batch, [out, lse],
                                         pc=plugin.push_constants(**args)))
            pc = plugin.push_constants(step_idx=s.longest, theta=case["theta"], **args)
            tasks.append(s.prov.task("paged_kv_weights", [q, pools[0]] + batch + [lse, h(s.held)], [h(s.weights)], pc=pc))
    s.tasks = (abi.nf_task_desc * len(tasks))(*tasks)


def _run_own(s):
    if len(s.tasks) > 1:
        s.prov.run_tasks(s.tasks)
    else:
        s.prov.check(s.prov.dispatch_task(s.tasks[0]), "dispatch")
    kind = s.case["kind"]
    if kind == "evict":
        return [s.kpool, s.vpool, s.weights, s.new_lens, s.kept]
    if kind == "prefix":
        return [s.out]
    return [s.weights] if kind == "weights" else [s.out, s.lse, s.weights]


# ---- plain forms -----------------------------------------------------------------

def _rows(s):
    """Sequence, position, and place among the sequence's rows, of each of the batch's rows."""
    row = torch.arange(s.rows, device="cuda")
    seq = torch.searchsorted(s.starts.long(), row, right=True) - 1
    return seq, s.lens.long()[seq] - s.starts.long()[seq + 1] + row, row - s.starts.long()[seq]


def _values(s, pool):
    """[sequence, kv, position, dim] in 32 bits of every sequence, padded to the longest."""
    case = s.case
    bs, d = case["block"], case["dim"]
    pages = pool[s.table.long().clamp(min=0)]
    if case["pool"] != "i8":
        x = pages.float()
    else:
        codes = pages[..., :bs * d].contiguous().view(torch.int8).float()
        scale = pages[..., bs * d:].contiguous().view(torch.float16).float()
        x = (codes.reshape(scale.shape + (32,)) * scale[..., None]).reshape(pages.shape[:-1] + (bs, d))
        x = x.to(TORCH[case["act"]]).float()  # an 8-bit cache stands for what a gather into the rows' type gives
    return x.transpose(1, 2).reshape(case["seqs"], case["kv"], -1, d)


def _plain_scores(s):
    """[sequence, kv, row, head of the kv head, position]; -inf where a row does not look."""
    case = s.case
    kv, d, h, n, most = case["kv"], case["dim"], case["heads"], case["seqs"], s.most
    keys = _values(s, s.kpool)
    seq, pos, at = _rows(s)
    q = torch.zeros(n, most, h, d, device="cuda")
    q[seq, at] = s.q.float()
    last = torch.full((n, most), -1, dtype=torch.int64, device="cuda")
    last[seq, at] = pos
    q = q.reshape(n, most, kv, h // kv, d).permute(0, 2, 1, 3, 4).reshape(n, kv, most * (h // kv), d)
    w = torch.matmul(q, keys.transpose(2, 3).contiguous()) / math.sqrt(d)
    seen = torch.arange(keys.shape[2], device="cuda") <= last[..., None]
    return w.reshape(n, kv, most, h // kv, -1).masked_fill_(~seen[:, None, :, None], -math.inf)


def _take_rows(s, x):
    """[sequence, kv, row, head of the kv head, ...] as the batch's rows of heads."""
    seq, _, at = _rows(s)
    x = x.transpose(1, 2)[seq, at]
    return x.reshape((s.rows, s.case["heads"]) + x.shape[3:])


def _plain_lse(s, scores):
    m = scores.amax(-1, keepdim=True)
    m = torch.where(m == -math.inf, torch.zeros_like(m), m)
    return _take_rows(s, (m + (scores - m).exp_().sum(-1, keepdim=True).log())[..., 0])


def _plain_attention(s, scores):
    case = s.case
    kv, d, h, n, most = case["kv"], case["dim"], case["heads"], case["seqs"], s.most
    m = scores.amax(-1, keepdim=True)
    w = (scores - torch.where(m == -math.inf, torch.zeros_like(m), m)).exp_()
    total = w.sum(-1, keepdim=True)
    o = torch.matmul(w.reshape(n, kv, most * (h // kv), -1), _values(s, s.vpool)).reshape(n, kv, most, h // kv, d) / total
    return _take_rows(s, o).to(TORCH[case["act"]])


def _plain_weights(s, scores, lse):
    case = s.case
    kv, h, n, most = case["kv"], case["heads"], case["seqs"], s.most
    seq, _, at = _rows(s)
    shift = torch.zeros(n, most, kv, h // kv, device="cuda")
    shift[seq, at] = lse.reshape(s.rows, kv, h // kv)
    w = (scores - shift.transpose(1, 2)[..., None]).exp_().sum((2, 3))[..., :s.longest]
    place = torch.arange(s.longest, device="cuda")
    lens = s.lens.long()[:, None, None]
    old = place < lens - (s.starts[1:] - s.starts[:-1]).long()[:, None, None]
    w = torch.where(old, case["theta"] * s.held, torch.zeros_like(s.held)) + w
    s.weights.copy_(torch.where(place < lens, w, s.weights))
    return s.weights


def _plain_evict(s):
    case = s.case
    bs, d, kv, n = case["block"], case["dim"], case["kv"], case["seqs"]
    lens = s.lens.long()
    keep = torch.minimum(s.budget[:, 0].long(), lens).clamp(min=0)
    recent = torch.minimum(s.budget[:, 1].long().clamp(min=0), keep)
    place = torch.arange(s.longest, device="cuda")
    rank = s.held.clone()
    rank = rank.masked_fill((place >= (lens - recent)[:, None])[:, None], math.inf)  # the latest
    rank = rank.masked_fill((place >= lens[:, None])[:, None], -math.inf)
    order = torch.sort(rank, dim=2, descending=True, stable=True)[1][..., :s.top]
    kept = torch.arange(s.top, device="cuda") < keep[:, None]  # [sequence, place]
    far = torch.full_like(order, s.longest)
    order = torch.sort(torch.where(kept[:, None], order, far), dim=2)[0]
    seq, head, to = torch.nonzero(kept[:, None].expand(n, kv, s.top), as_tuple=True)
    src = order[seq, head, to]
    s.kept[seq, head, to] = src.int()
    s.weights[seq, head, to] = s.held[seq, head, src]
    a, b = s.table[seq, src // bs].long(), s.moved[seq, to // bs].long()
    x, y = src % bs, to % bs
    for pool in (s.kpool, s.vpool):
        if case["pool"] != "i8":
            pool[b, head, y] = pool[a, head, x]
            continue
        lane = torch.arange(d, device="cuda")
        pool[b[:, None], head[:, None], y[:, None] * d + lane] = pool[a[:, None], head[:, None], x[:, None] * d + lane]
        lane = bs * d + torch.arange(d // 16, device="cuda")
        step = d // 16
        pool[b[:, None], head[:, None], y[:, None] * step + lane] = pool[a[:, None], head[:, None], x[:, None] * step + lane]
    s.new_lens.copy_(keep)
    return [s.kpool, s.vpool, s.weights, s.new_lens, s.kept]


# ---- work ------------------------------------------------------------------------

def work(case):
    kv, d, e, kind = case["kv"], case["dim"], SIZE[case["act"]], case["kind"]
    row = kv * d * (34 / 32 if case["pool"] == "i8" else e)  # a position's keys in the pools
    if kind == "evict":
        total = sum(n * kv * 4 + k * (4 * row + kv * 8) for n, k, _ in _budget(case))
        return {"bytes": int(total), "flops": 0}
    lens = _lens(case)
    rows = sum(n for _, n in lens)
    pairs = sum(n * length - n * (n - 1) // 2 for length, n in lens)
    held = sum(length for length, _ in lens)
    if kind == "prefix":
        held -= sum((last - first - 1) * p for first, last, p in _groups(case))
    total = rows * case["heads"] * d * e
    flops = 2 * pairs * case["heads"] * d
    if kind in ("prefix", "score"):
        total += rows * case["heads"] * d * e + 2 * held * row
        flops *= 2
    else:
        total += held * row
    if kind in ("weights", "score"):
        total += rows * case["heads"] * 4 + held * kv * (8 if case["theta"] else 4)
    return {"bytes": int(total), "flops": flops}


# ---- 64-bit results ----------------------------------------------------------------

def exact(case, seed):
    """What run() returns, from the definitions in 64 bits, one sequence after the other."""
    global own
    was, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = was
    if case["kind"] == "evict":
        return _exact_evict(s)
    kv, d, h, kind = case["kv"], case["dim"], case["heads"], case["kind"]
    table, starts, lens = s.table.cpu().tolist(), s.starts.cpu().tolist(), s.lens.cpu().tolist()
    outs, lses = [], []
    weights = torch.zeros(len(lens), kv, s.longest, dtype=torch.float64, device="cuda")
    for i, length in enumerate(lens):
        n = starts[i + 1] - starts[i]
        pages = torch.tensor(table[i][:-(-length // case["block"])], device="cuda")
        mask = torch.arange(length, device="cuda")[None] > torch.arange(length - n, length, device="cuda")[:, None]
        o = torch.empty(n, h, d, dtype=torch.float64, device="cuda")
        z = torch.empty(n, h, dtype=torch.float64, device="cuda")
        for g in range(kv):
            keys = _exact_head(case, s.kpool, pages, g)[:length]
            vals = _exact_head(case, s.vpool, pages, g)[:length] if kind != "weights" else None
            for head in range(g * h // kv, (g + 1) * h // kv):
                x = (s.q[starts[i]:starts[i + 1], head].double() @ keys.T) * d ** -0.5
                x.masked_fill_(mask, -math.inf)
                z[:, head] = torch.logsumexp(x, 1)
                if kind != "weights":
                    o[:, head] = torch.softmax(x, 1) @ vals
                if kind != "prefix":
                    by = s.lse[starts[i]:starts[i + 1], head].double() if kind == "weights" else z[:, head]
                    weights[i, g, :length] += torch.exp(x - by[:, None]).sum(0)
        if kind != "prefix":
            weights[i, :, :length - n] += case["theta"] * s.held[i, :, :length - n].double()
        outs.append(o)
        lses.append(z)
    if kind == "prefix":
        return [torch.cat(outs)]
    return [weights] if kind == "weights" else [torch.cat(outs), torch.cat(lses), weights]


def _exact_head(case, pool, pages, g):
    """One KV head's rows of the blocks, in 64 bits."""
    bs, d = case["block"], case["dim"]
    x = pool[pages, g]
    if case["pool"] != "i8":
        return x.double().reshape(-1, d)
    c = x[:, :bs * d].contiguous().view(torch.int8).double().reshape(-1, d // 32, 32)
    c = (c * x[:, bs * d:].contiguous().view(torch.float16).double().reshape(-1, d // 32, 1)).reshape(-1, d)
    return c.to(TORCH[case["act"]]).double()  # by definition: rounded once to the rows' type


def _exact_evict(s):
    """Row by row in numpy: the latest positions, and the first of the others in the order of weight and position."""
    case = s.case
    bs, d = case["block"], case["dim"]
    held, table, moved = s.held.cpu().numpy(), s.table.cpu().numpy(), s.moved.cpu().numpy()
    weights = np.zeros(held.shape)
    kept = np.zeros((case["seqs"], case["kv"], s.top), np.int32)
    pools = [s.kpool.clone(), s.vpool.clone()]
    lens = []
    for i, (n, k, r) in enumerate(_budget(case)):
        lens.append(k)
        for g in range(case["kv"]):
            best = np.argsort(-held[i, g, :n - r].astype(np.float64), kind="stable")[:k - r]
            at = np.sort(np.concatenate([best, np.arange(n - r, n)]))
            kept[i, g, :k] = at
            weights[i, g, :k] = held[i, g, at]
            src = torch.tensor(table[i, at // bs] * bs + at % bs, device="cuda").long()
            dst = torch.tensor(moved[i, np.arange(k) // bs] * bs + np.arange(k) % bs, device="cuda").long()
            for pool in pools:
                if case["pool"] != "i8":
                    pool[dst // bs, g, dst % bs] = pool[src // bs, g, src % bs]
                    continue
                codes = pool[:, g, :bs * d].reshape(-1, d)
                scale = pool[:, g, bs * d:].reshape(-1, d // 16)
                codes[dst], scale[dst] = codes[src], scale[src]
                pool[:, g, :bs * d], pool[:, g, bs * d:] = codes.reshape(-1, bs * d), scale.reshape(-1, bs * d // 16)
    if case["pool"] != "i8":
        pools = [p.double() for p in pools]
    return pools + [torch.tensor(weights), torch.tensor(lens, dtype=torch.int32), torch.tensor(kept)]
