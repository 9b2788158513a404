"""Performance cases of the serving operators: the paged key/value cache (written, quantised to 8 bits or not, and
read back), attention of chunks of new tokens over it, and sampling of the next token.

Kinds of case:
  append     paged_kv_append: a batch's new key and value rows into f32 / f16 pools; the pools come back
  roundtrip  paged_kv_append and paged_kv_gather of the same rows; what the cache holds of them comes back
  gather     paged_kv_gather: whole sequences read back as dense rows
  attention  flash_attention_paged_chunk over what the cache holds
  step       paged_kv_append of the chunk's rows and flash_attention_paged_chunk, as a layer of a model runs them
  sample     sample_token for a batch of rows of logits

A batch is `seqs` sequences of up to `ctx` cached positions, the last `chunk` (at most) of them new. `ragged` spreads
both over the sequences by a fixed rule. The pools' blocks are handed out in a random order.
"""
import math
import random

import numpy as np
import torch

own = False

TORCH = {"f32": torch.float32, "f16": torch.float16}
SIZE = {"f32": 4, "f16": 2}
ONE = float(1 << 40)  # the largest sampling weight


def listed():
    return [
        # One token each of four sequences into an 8-bit cache and back: the smallest call of the cache operators.
        {"name": "kv_roundtrip_step", "kind": "roundtrip", "act": "f16", "pool": "i8", "seqs": 4, "chunk": 1, "ctx": 900,
         "ragged": True, "kv": 8, "dim": 128, "block": 16},
        # The rows of a prefill of four prompts of up to 2048 tokens, f16 cache.
        {"name": "kv_append_f16", "kind": "append", "act": "f16", "pool": "f16", "seqs": 4, "chunk": 2048, "ctx": 2048,
         "ragged": True, "kv": 8, "dim": 128, "block": 16},
        # A large batch of prompts in f32 activations, quantised as it is written, and read back.
        {"name": "kv_roundtrip_i8_f32", "kind": "roundtrip", "act": "f32", "pool": "i8", "seqs": 16, "chunk": 2048,
         "ctx": 2048, "ragged": True, "kv": 8, "dim": 128, "block": 32},
        # One long 8-bit sequence as dense f16 rows (a prefix handed to another engine).
        {"name": "kv_gather_i8", "kind": "gather", "act": "f16", "pool": "i8", "seqs": 1, "chunk": 65536, "ctx": 65536,
         "ragged": False, "kv": 8, "dim": 128, "block": 16},
        # A decode step of one short sequence, 32 heads over 4 KV heads of 64, f32: latency counts.
        {"name": "step_f32_short", "kind": "step", "act": "f32", "pool": "f32", "seqs": 1, "chunk": 1, "ctx": 100,
         "ragged": False, "heads": 32, "kv": 4, "dim": 64, "block": 16},
        # A decode step of 64 sequences of up to 8192 tokens, 32 heads over 8 KV heads of 128.
        {"name": "decode_f16_batch", "kind": "attention", "act": "f16", "pool": "f16", "seqs": 64, "chunk": 1, "ctx": 8192,
         "ragged": True, "heads": 32, "kv": 8, "dim": 128, "block": 16},
        # A decode step of four very long sequences in the 8-bit cache.
        {"name": "decode_i8_long", "kind": "attention", "act": "f16", "pool": "i8", "seqs": 4, "chunk": 1, "ctx": 131072,
         "ragged": True, "heads": 32, "kv": 8, "dim": 128, "block": 16},
        # Five drafted tokens of each of 16 sequences verified at once, 8-bit cache, rows appended first.
        {"name": "verify_i8", "kind": "step", "act": "f16", "pool": "i8", "seqs": 16, "chunk": 5, "ctx": 4096,
         "ragged": True, "heads": 32, "kv": 8, "dim": 128, "block": 16},
        # A chunk of 2048 prompt tokens of two sequences behind 6144 cached ones: the largest.
        {"name": "chunk_f16", "kind": "attention", "act": "f16", "pool": "f16", "seqs": 2, "chunk": 2048, "ctx": 8192,
         "ragged": False, "heads": 32, "kv": 8, "dim": 128, "block": 16},
        # Ragged chunks in f32, 32 heads over 4 KV heads of 64.
        {"name": "chunk_f32_ragged", "kind": "attention", "act": "f32", "pool": "f32", "seqs": 3, "chunk": 389, "ctx": 2000,
         "ragged": True, "heads": 32, "kv": 4, "dim": 64, "block": 16},
        # The next token of one conversation: top-k 40, then top-p 0.95, over 32000 logits.
        {"name": "sample_one", "kind": "sample", "act": "f32", "rows": 1, "vocab": 32000, "how": "top_k_p"},
        # A batch with every kind of request in it, over 128256 logits.
        {"name": "sample_batch", "kind": "sample", "act": "f32", "rows": 64, "vocab": 128256, "how": "mixed"},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["append", "roundtrip", "gather", "attention", "attention", "step", "sample"])
    act = rng.choice(["f32", "f16"])
    if kind == "sample":
        return {"kind": kind, "act": act, "rows": _log(rng, 1, 64), "vocab": _log(rng, 1000, 128256),
                "how": rng.choice(["temperature", "top_k_p", "top_p", "min_p", "mixed"])}
    c = {"kind": kind, "act": act, "pool": rng.choice([act, "i8"]), "kv": rng.choice([1, 2, 4, 8]),
         "dim": rng.choice([64, 64, 128, 128, 96]), "block": rng.choice([8, 16, 16, 32]), "ragged": rng.random() < 0.7}
    if kind in ("append", "roundtrip", "gather"):
        if kind == "append":
            c["pool"] = act
        c["seqs"] = _log(rng, 1, 16)
        c["ctx"] = _log(rng, 16, 32768 // c["seqs"])
        c["chunk"] = c["ctx"] if kind == "gather" or rng.random() < 0.5 else _log(rng, 1, c["ctx"])
        return c
    c["heads"] = c["kv"] * rng.choice([1, 2, 4, 4, 8])
    c["chunk"] = _log(rng, 1, 1024)
    c["seqs"] = _log(rng, 1, max(1, min(64, 2048 // c["chunk"])))
    c["ctx"] = max(c["chunk"], _log(rng, 16, 8192 if c["seqs"] > 1 or c["chunk"] > 1 else 131072))
    return c


# ---- batches -------------------------------------------------------------------

def _lens(case):
    """[(cached positions, new ones among them)] of the batch's sequences."""
    out = []
    for i in range(case["seqs"]):
        f = (i * 0.6180339887 + 0.25) % 1.0 if case["ragged"] and i else 0.0
        n = max(1, case["chunk"] - int(0.5 * f * case["chunk"]))
        out.append((max(n, case["ctx"] - int(0.75 * f * case["ctx"])), n))
    return out


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


def prepare(case, seed):
    s = State(case, seed)
    if case["kind"] == "sample":
        _prepare_sample(s)
    else:
        _prepare_batch(s, seed)
    if own:
        _bind(s)
    torch.cuda.synchronize()  # the provider's stream does not wait for torch's
    return s


def _prepare_batch(s, seed):
    case = s.case
    act, kv, d, bs = case["act"], case["kv"], case["dim"], case["block"]
    lens = _lens(case)
    starts = [0]
    for _, n in lens:
        starts.append(starts[-1] + n)
    pages = [-(-length // bs) for length, _ in lens]
    blocks = sum(pages) + 3  # three that belong to no sequence
    order = list(range(blocks))
    random.Random(seed).shuffle(order)
    table = np.full((len(lens), max(pages)), -1, np.int32)
    at = 0
    for i, n in enumerate(pages):
        table[i, :n] = order[at:at + n]
        at += n
    dev = lambda a: torch.tensor(a, dtype=torch.int32, device="cuda")  # noqa: E731
    s.table, s.starts, s.lens = dev(table), dev(starts), dev([length for length, _ in lens])
    s.rows, s.most = starts[-1], max(n for _, n in lens)
    s.kpool, s.vpool = _pool(s, blocks), _pool(s, blocks)
    if case["kind"] in ("append", "roundtrip", "step"):
        s.k, s.v = s.normal(act, s.rows, kv, d), s.normal(act, s.rows, kv, d)
    if case["kind"] in ("roundtrip", "gather"):
        s.ko, s.vo = (torch.zeros(s.rows, kv, d, dtype=TORCH[act], device="cuda") for _ in range(2))
    if case["kind"] in ("attention", "step"):
        s.q = s.normal(act, s.rows, case["heads"], d)
        s.out = torch.zeros_like(s.q)


_HOW = {  # temperature, top_p, min_p, top_k of the rows, in turn
    "temperature": [(1.0, 1.0, 0.0, 0)],
    "top_k_p": [(0.8, 0.95, 0.0, 40)],
    "top_p": [(0.7, 0.9, 0.0, 0)],
    "min_p": [(1.2, 1.0, 0.05, 0)],
    "mixed": [(0.8, 0.95, 0.0, 40), (0.7, 0.9, 0.0, 0), (1.0, 1.0, 0.0, 0), (1.2, 1.0, 0.05, 0), (0.0, 1.0, 0.0, 0),
              (0.9, 0.97, 0.02, 200), (1.0, 0.99, 0.0, 0), (0.6, 0.8, 0.1, 64)],
}


def _prepare_sample(s):
    case = s.case
    r, n = case["rows"], case["vocab"]
    x = torch.randn(r, n, generator=s.gen, device="cuda") * 2.5
    for _ in range(12):  # the few tokens that a model thinks likely
        at = torch.randint(0, n, (r, 1), generator=s.gen, device="cuda")
        x.scatter_add_(1, at, 4 + 6 * torch.rand(r, 1, generator=s.gen, device="cuda"))
    s.logits = x.to(TORCH[case["act"]])
    s.u = torch.rand(r, generator=s.gen, device="cuda")
    how = [_HOW[case["how"]][i % len(_HOW[case["how"]])] for i in range(r)]
    s.params = torch.tensor([h[:3] for h in how], dtype=torch.float32, device="cuda")
    s.top_k = torch.tensor([h[3] for h in how], dtype=torch.int32, device="cuda")
    s.token = torch.zeros(r, dtype=torch.int32, device="cuda")
    s.prob = torch.zeros(r, dtype=torch.float32, device="cuda")


def run(state):
    if own:
        return _run_own(state)
    case = state.case
    kind = case["kind"]
    if kind == "sample":
        return _plain_sample(state)
    if kind in ("append", "roundtrip", "step"):
        _plain_append(state)
    if kind == "append":
        return [state.kpool, state.vpool]
    if kind in ("roundtrip", "gather"):
        seq, pos = _rows(state)
        return [_plain_read(state, pool, seq, pos).to(TORCH[case["act"]]) for pool in (state.kpool, state.vpool)]
    return [_plain_attention(state)]


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
    kind = {torch.float32: abi.NF_DTYPE_F32, torch.float16: abi.NF_DTYPE_F16, torch.int32: abi.NF_DTYPE_I32,
            torch.uint8: abi.NF_DTYPE_I8}

    def h(t):
        desc = abi.make_desc(kind[t.dtype], t.numel() * t.element_size())
        ops, handle = abi.nf_buffer_ops(), ctypes.c_void_p()
        s.prov.check(s.prov.mem.import_buffer(s.prov.handle, t.data_ptr(), abi.NF_MEM_DOMAIN_DEVICE, ctypes.byref(desc),
                                              ctypes.byref(ops), ctypes.byref(handle)), "import_buffer")
        s.handles.append(plugin.Buffer(s.prov, handle.value, ops, desc.dtype, desc.size_bytes))
        return s.handles[-1]

    tasks = []
    if case["kind"] == "sample":
        pc = plugin.push_constants(N=case["vocab"], seq_len=case["rows"])
        tasks.append(s.prov.task("sample_token", [h(s.logits), h(s.u), h(s.params), h(s.top_k)], [h(s.token), h(s.prob)],
                                 pc=pc))
    else:
        batch = [h(s.table), h(s.starts), h(s.lens)]
        pools = [h(s.kpool), h(s.vpool)]
        args = dict(M=case["kv"], N=s.table.shape[1], K=case["seqs"], seq_len=s.rows, head_dim=case["dim"],
                    window_size=case["block"])
        if case["kind"] in ("append", "roundtrip", "step"):
            tasks.append(s.prov.task("paged_kv_append", [h(s.k), h(s.v)] + batch, pools, pc=plugin.push_constants(**args)))
        if case["kind"] in ("roundtrip", "gather"):
            tasks.append(s.prov.task("paged_kv_gather", pools + batch, [h(s.ko), h(s.vo)], pc=plugin.push_constants(**args)))
        if case["kind"] in ("attention", "step"):
            pc = plugin.push_constants(n_heads=case["heads"], max_seq_len=case["ctx"], **args)
            tasks.append(s.prov.task("flash_attention_paged_chunk", [h(s.q)] + pools + batch, [h(s.out)], pc=pc))
    s.tasks = (abi.nf_task_desc * len(tasks))(*tasks)


def _run_own(s):
    if len(s.tasks) > 1:
        s.prov.run_tasks(s.tasks)
    else:
        s.prov.check(s.prov.dispatch_task(s.tasks[0]), "dispatch")
    kind = s.case["kind"]
    if kind == "sample":
        return [s.token, s.prob]
    if kind == "append":
        return [s.kpool, s.vpool]
    if kind in ("roundtrip", "gather"):
        return [s.ko, s.vo]
    return [s.out]


# ---- plain forms -----------------------------------------------------------------

def _rows(s):
    """Sequence and position of each of the batch's rows."""
    row = torch.arange(s.rows, device="cuda")
    seq = torch.searchsorted(s.starts.long(), row, right=True) - 1
    return seq, s.lens.long()[seq] - s.starts.long()[seq + 1] + row


def _quantise(x):
    """Codes and fp16 scales of groups of 32; in 64 bits, as values lie next to the borders between codes."""
    g = x.double().reshape(*x.shape[:-1], -1, 32)
    d = (g.abs().amax(-1) / 127).float().half()
    step = torch.where(d > 0, d, torch.ones_like(d)).double()[..., None]
    codes = torch.where(d[..., None] > 0, torch.clamp(torch.round(g / step), -127, 127), torch.zeros_like(g))
    return codes.to(torch.int8).reshape(x.shape), d


def _plain_append(s):
    case = s.case
    bs, d = case["block"], case["dim"]
    seq, pos = _rows(s)
    block, slot = s.table[seq, pos // bs].long(), pos % bs
    for pool, x in ((s.kpool, s.k), (s.vpool, s.v)):
        if case["pool"] != "i8":
            pool[block, :, slot] = x
            continue
        codes, scale = _quantise(x)
        lo = slot[:, None] * d + torch.arange(d, device="cuda")
        pool[block[:, None], :, lo] = codes.view(torch.uint8).transpose(1, 2)
        hi = bs * d + slot[:, None] * (d // 16) + torch.arange(d // 16, device="cuda")
        pool[block[:, None], :, hi] = scale.view(torch.uint8).transpose(1, 2)


def _values(s, pages):
    """[..., kv, block, dim] in 32 bits of pages [..., kv, (page)]."""
    case = s.case
    bs, d = case["block"], case["dim"]
    if case["pool"] != "i8":
        return pages.float()
    codes = pages[..., :bs * d].contiguous().view(torch.int8).float()
    scale = pages[..., bs * d:].contiguous().view(torch.float16).float()
    shape = pages.shape[:-1] + (bs, d)
    return (codes.reshape(scale.shape + (32,)) * scale[..., None]).reshape(shape)


def _plain_read(s, pool, seq, pos):
    case = s.case
    bs, d = case["block"], case["dim"]
    block, slot = s.table[seq, pos // bs].long(), pos % bs
    if case["pool"] != "i8":
        return pool[block, :, slot].float()
    lo = slot[:, None] * d + torch.arange(d, device="cuda")
    codes = pool[block[:, None], :, lo].transpose(1, 2).contiguous().view(torch.int8).float()
    hi = bs * d + slot[:, None] * (d // 16) + torch.arange(d // 16, device="cuda")
    scale = pool[block[:, None], :, hi].transpose(1, 2).contiguous().view(torch.float16).float()
    return (codes.reshape(scale.shape + (32,)) * scale[..., None]).reshape(codes.shape)


def _plain_attention(s):
    """Every sequence padded to the longest, its rows padded to the longest chunk."""
    case = s.case
    kv, d, h, n, most = case["kv"], case["dim"], case["heads"], case["seqs"], s.most
    pages = s.table.long().clamp(min=0)
    keys, vals = (_values(s, pool[pages]).transpose(1, 2).reshape(n, kv, -1, d) for pool in (s.kpool, s.vpool))
    seq, pos = _rows(s)
    at = torch.arange(s.rows, device="cuda") - s.starts.long()[seq]
    q = torch.zeros(n, most, h, d, device="cuda")
    q[seq, at] = s.q.float()
    last = torch.full((n, most), -1, dtype=torch.int64, device="cuda")
    last[seq, at] = pos
    q = q.reshape(n, most, kv, h // kv, d).permute(0, 2, 1, 3, 4).reshape(n, kv, most * (h // kv), d)
    w = torch.matmul(q, keys.transpose(2, 3).contiguous()) / math.sqrt(d)
    seen = torch.arange(keys.shape[2], device="cuda") <= last[..., None]
    w = w.reshape(n, kv, most, h // kv, -1).masked_fill_(~seen[:, None, :, None], -math.inf)
    m = w.amax(-1, keepdim=True)
    w = w.sub_(torch.where(m == -math.inf, torch.zeros_like(m), m)).exp_()
    total = w.sum(-1, keepdim=True)
    o = torch.matmul(w.reshape(n, kv, most * (h // kv), -1), vals).reshape(n, kv, most, h // kv, d) / total
    return o.permute(0, 2, 1, 3, 4).reshape(n, most, h, d)[seq, at].to(TORCH[case["act"]])


def _plain_sample(s):
    """The weights in 64 bits, then whole numbers: their sums do not depend on the order."""
    x = s.logits.double()
    r, n = x.shape
    temp, top_p, min_p = s.params.double().unbind(1)
    greedy = temp <= 0
    x, order = torch.sort(x, dim=1, descending=True, stable=True)
    z = (x - x[:, :1]) / torch.where(greedy, torch.ones_like(temp), temp)[:, None]
    w = torch.round(torch.exp(z) * ONE).long()
    rank = torch.arange(n, device="cuda")
    k = torch.where((s.top_k <= 0) | (s.top_k > n), n, s.top_k).long()
    k = torch.where(greedy, torch.ones_like(k), k)
    w = torch.where(rank < k[:, None], w, torch.zeros_like(w))
    upto = torch.cumsum(w, 1)
    p = torch.where(top_p >= 1, torch.full_like(top_p, math.inf), top_p)
    keep = (upto - w).double() < p[:, None] * upto[:, -1:].double()
    keep = ((rank == 0) | keep) & (w.double() >= min_p[:, None] * ONE)
    kept = torch.zeros_like(w).scatter_(1, order, torch.where(keep, w, torch.zeros_like(w)))
    upto = torch.cumsum(kept, 1)
    total = upto[:, -1]
    t = torch.minimum(torch.floor(s.u.double() * total.double()).long(), total - 1)
    token = torch.searchsorted(upto, t[:, None], right=True)
    prob = kept.gather(1, token)[:, 0].double() / total.double()
    return [token[:, 0].to(torch.int32), prob.float()]


# ---- work ------------------------------------------------------------------------

def work(case):
    if case["kind"] == "sample":
        return {"bytes": case["rows"] * (case["vocab"] * SIZE[case["act"]] + 28), "flops": 8 * case["rows"] * case["vocab"]}
    kv, d, e, kind = case["kv"], case["dim"], SIZE[case["act"]], case["kind"]
    cell = 2 * kv * d * (34 / 32 if case["pool"] == "i8" else e)  # a position's key and value in the pools
    lens = _lens(case)
    rows = sum(n for _, n in lens)
    total = {"bytes": 0, "flops": 0}
    if kind in ("append", "roundtrip", "step"):
        total["bytes"] += rows * (2 * kv * d * e + cell)
        total["flops"] += 6 * rows * kv * d if case["pool"] == "i8" else 0
    if kind in ("roundtrip", "gather"):
        total["bytes"] += rows * (2 * kv * d * e + cell)
        total["flops"] += 2 * rows * kv * d
    if kind in ("attention", "step"):
        total["bytes"] += 2 * rows * case["heads"] * d * e + sum(length for length, _ in lens) * cell
        pairs = sum(n * length - n * (n - 1) // 2 for length, n in lens)
        total["flops"] += 4 * pairs * case["heads"] * d
    return total


# ---- 64-bit results ----------------------------------------------------------------

def exact(case, seed):
    """What run() returns, from the definitions in 64 bits, one sequence (or row) after the other."""
    global own
    was, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = was
    if case["kind"] == "sample":
        return _exact_sample(s)
    kv, d, bs, kind = case["kv"], case["dim"], case["block"], case["kind"]
    table, starts = s.table.cpu().tolist(), s.starts.cpu().tolist()
    lens = s.lens.cpu().tolist()
    if kind == "append":
        pools = [s.kpool.double(), s.vpool.double()]
    outs = [[], []] if kind != "attention" and kind != "step" else [[]]
    for i, length in enumerate(lens):
        n = starts[i + 1] - starts[i]
        blocks = torch.tensor(table[i][:-(-length // bs)], device="cuda")
        held = []
        for j, pool in enumerate((s.kpool, s.vpool)):
            x = _exact_pages(case, pool[blocks]).transpose(1, 2).reshape(-1, kv, d)[:length]
            if kind in ("append", "roundtrip", "step"):
                new = (s.k, s.v)[j][starts[i]:starts[i + 1]].double()
                x[length - n:] = _exact_held(new) if case["pool"] == "i8" else new
            held.append(x)
        if kind == "append":
            for pool, x in zip(pools, held):
                flat = torch.arange(length - n, length, device="cuda")
                pool[blocks[flat // bs], :, flat % bs] = x[length - n:]
            continue
        if kind in ("roundtrip", "gather"):
            for o, x in zip(outs, held):
                o.append(x[length - n:])
            continue
        o = torch.empty(n, case["heads"], d, dtype=torch.float64, device="cuda")
        mask = torch.arange(length, device="cuda")[None] > torch.arange(length - n, length, device="cuda")[:, None]
        for head in range(case["heads"]):
            g = head * kv // case["heads"]
            p = (s.q[starts[i]:starts[i + 1], head].double() @ held[0][:, g].T) * d ** -0.5
            o[:, head] = torch.softmax(p.masked_fill_(mask, -math.inf), 1) @ held[1][:, g]
        outs[0].append(o)
    return pools if kind == "append" else [torch.cat(o) for o in outs]


def _exact_pages(case, pages):
    bs, d = case["block"], case["dim"]
    if case["pool"] != "i8":
        return pages.double()
    blocks, kv = pages.shape[:2]
    c = pages[:, :, :bs * d].contiguous().view(torch.int8).double().reshape(blocks, kv, bs, d // 32, 32)
    sc = pages[:, :, bs * d:].contiguous().view(torch.float16).double().reshape(blocks, kv, bs, d // 32, 1)
    return (c * sc).reshape(blocks, kv, bs, d)


def _exact_held(x):
    """The values that an 8-bit cache holds of x: whole multiples, nearest and to even, of the rounded scale."""
    a = x.reshape(-1, 32)
    top = a.abs().max(1).values
    d = (top / 127.0).to(torch.float32).to(torch.float16).to(torch.float64)[:, None]
    q = torch.where(d == 0, torch.zeros_like(a), (a / d).round())
    return (q.clamp(-127, 127) * d).reshape(x.shape)


def _exact_sample(s):
    x = s.logits.double().cpu().numpy()
    params, top_k, u = s.params.double().cpu().numpy(), s.top_k.cpu().numpy(), s.u.double().cpu().numpy()
    tokens, probs = [], []
    for row, (temp, top_p, min_p), k, draw_at in zip(x, params, top_k, u):
        if temp <= 0:
            tokens.append(int(np.argmax(row)))
            probs.append(1.0)
            continue
        order = np.argsort(-row, kind="stable")
        w = np.rint(np.exp((row[order] - row.max()) / temp) * ONE).astype(np.int64)
        n = len(row) if k <= 0 or k > len(row) else int(k)
        order, w = order[:n], w[:n]
        if top_p < 1:
            before = np.cumsum(w) - w
            n = max(1, int(np.searchsorted(before.astype(np.float64), top_p * float(w.sum()), side="left")))
            order, w = order[:n], w[:n]
        ok = w.astype(np.float64) >= min_p * ONE
        order, w = order[ok], w[ok]
        by = np.argsort(order)
        order, w = order[by], w[by]
        upto = np.cumsum(w)
        t = min(int(math.floor(draw_at * float(upto[-1]))), int(upto[-1]) - 1)
        at = int(np.searchsorted(upto, t, side="right"))
        tokens.append(int(order[at]))
        probs.append(float(w[at]) / float(upto[-1]))
    return [torch.tensor(tokens, dtype=torch.int32), torch.tensor(probs, dtype=torch.float64)]
