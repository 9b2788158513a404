"""Refusals and plans of the operators for long contexts over the paged cache, without a GPU."""
import pytest

from neurofabric_amd import abi
from neurofabric_amd.plugin import load_library, plan
from test_serving_host import BF16, BS, D, F16, F32, H, I32, I8, KV, S, SIZE, T, W, args, batch, chunk, desc, pool, refused

GROUPS, TOP = 2, 20
WIDTH = W * BS


@pytest.fixture(scope="module")
def lib():
    return load_library()


def lse_of(n=T * H, dtype=F32):
    return desc(dtype, n * 4)


def prefix(lib, act=F16, pl=F16, q=None, out=None, pools=None, bat=None, groups=None, lens=None, lse=None, pc=None):
    q, out = q or desc(act, T * H * D * SIZE[act]), out or desc(act, T * H * D * SIZE[act])
    ins = [q] + (pools or [pool(pl)] * 2) + (bat or batch()) + [groups or desc(I32, (GROUPS + 1) * 4), lens or desc(I32, GROUPS * 4)]
    return plan(lib, "flash_attention_paged_prefix", ins, [out] + ([lse] if lse else []),
                pc=args(n_heads=H, step_idx=GROUPS) if pc is None else pc)


def weigh(lib, act=F16, pl=F16, q=None, pools=None, bat=None, lse=None, held=None, out=None, pc=None):
    rows = desc(F32, S * KV * WIDTH * 4)
    ins = [q or desc(act, T * H * D * SIZE[act])] + (pools or [pool(pl)])[:1] + (bat or batch()) + [lse or lse_of(), held or rows]
    return plan(lib, "paged_kv_weights", ins, [out or rows], pc=args(n_heads=H, step_idx=WIDTH, theta=1.0) if pc is None else pc)


def evict(lib, pl=F16, pools=None, rows=None, tables=None, lens=None, budget=None, new=None, to=None, rows_to=None,
          lens_to=None, kept=None, pc=None):
    r = desc(F32, S * KV * WIDTH * 4)
    ins = (pools or [pool(pl)] * 2) + [rows or r, tables or batch()[0], lens or desc(I32, S * 4), budget or desc(I32, S * 8),
                                       new or desc(I32, S * -(-TOP // BS) * 4)]
    outs = (to or [pool(pl)] * 2) + [rows_to or r, lens_to or desc(I32, S * 4), kept or desc(I32, S * KV * TOP * 4)]
    return plan(lib, "paged_kv_evict", ins, outs, pc=args(seq_len=TOP, step_idx=WIDTH) if pc is None else pc)


@pytest.mark.parametrize("act,pl,name", [(F32, F32, "f32_f32"), (F32, I8, "f32_i8"), (F16, F16, "f16_f16"), (F16, I8, "f16_i8")])
def test_plans(lib, act, pl, name):
    p = prefix(lib, act, pl)
    assert p["kernel"] == "attention_paged_prefix_" + name and p["count"] == T * H
    assert prefix(lib, act, pl, lse=lse_of())["out_bytes"] == p["out_bytes"] + T * H * 4
    assert weigh(lib, act, pl)["kernel"] == "paged_weights_" + name
    assert evict(lib, pl)["kernel"] == "paged_evict_" + name.split("_")[1]
    assert evict(lib, pl)["count"] == S * KV * TOP


@pytest.mark.parametrize("call", [prefix, weigh])
def test_batch_refusals(lib, call):
    more = {"n_heads": H, **({"step_idx": GROUPS} if call is prefix else {"step_idx": WIDTH, "theta": 1.0})}
    refused(call, lib, pc=b"", match="push constants")
    refused(call, lib, pc=args(head_dim=0, **more), match="head_dim")
    refused(call, lib, pc=args(head_dim=257, **more), match="head_dim")
    refused(call, lib, pc=args(K=S + 1, **more))
    refused(call, lib, pc=args(N=W + 1, **more))
    refused(call, lib, pc=args(K=65536, **more), match="65535")
    refused(call, lib, pc=args(window_size=65537, **more), match="65536")
    refused(call, lib, pc=args(seq_len=T + 1, **more), match="Q holds")
    refused(call, lib, pc=args(seq_len=(1 << 22) + 1, **more), match="rows")
    refused(call, lib, pc=args(**{**more, "n_heads": 1}), match="n_heads")
    refused(call, lib, pc=args(**{**more, "n_heads": 65536}), match="65535 heads")
    refused(call, lib, bat=[desc(I32, S * W * 4 - 4)] + batch()[1:], match="tables")
    refused(call, lib, bat=[batch()[0], desc(I32, S * 4), batch()[2]], match="starts")
    refused(call, lib, bat=batch()[:2] + [desc(I32, S * 4 - 4)], match="lengths")
    refused(call, lib, act=F32, pl=F16, match="dtype or I8")
    refused(call, lib, act=BF16, pl=BF16, match="F32 or F16")
    refused(call, lib, lse=lse_of(T * H - 1), match="log-sum-exp")
    refused(call, lib, lse=lse_of(dtype=F16), match="log-sum-exp")
    refused(call, lib, q=desc(F16, T * H * D * 2 - 2), match="Q holds")


def test_chunk_lse_refusals(lib):
    """The chunk attention's second output."""
    good = dict(q=desc(F16, T * H * D * 2), out=desc(F16, T * H * D * 2))
    ins = [good["q"]] + [pool(F16)] * 2 + batch()
    pc = args(n_heads=H)
    p = plan(lib, "flash_attention_paged_chunk", ins, [good["out"], lse_of()], pc=pc)
    assert p["kernel"] == chunk(lib)["kernel"] and p["out_bytes"] == chunk(lib)["out_bytes"] + T * H * 4
    refused(plan, lib, "flash_attention_paged_chunk", ins, [good["out"], lse_of(T * H - 1)], pc=pc, match="log-sum-exp")
    refused(plan, lib, "flash_attention_paged_chunk", ins, [good["out"], lse_of(dtype=I32)], pc=pc, match="log-sum-exp")


def test_prefix_refusals(lib):
    refused(prefix, lib, groups=desc(I32, GROUPS * 4), match="groups hold")
    refused(prefix, lib, lens=desc(I32, GROUPS * 4 - 4), match="prefixes hold")
    refused(prefix, lib, pc=args(n_heads=H, step_idx=65536), match="65535 groups")
    refused(prefix, lib, out=desc(F32, T * H * D * 4), match="one dtype")
    refused(prefix, lib, out=desc(F16, T * H * D * 2 - 2), match="output holds")
    assert prefix(lib, groups=desc(I32, 4), lens=desc(I32, 0), pc=args(n_heads=H))["count"] == T * H  # no groups


def test_weights_refusals(lib):
    more = dict(n_heads=H, step_idx=WIDTH)
    short, good = desc(F32, S * KV * WIDTH * 4 - 4), desc(F32, S * KV * WIDTH * 4)
    for theta in (-0.5, 1.5, float("nan"), float("inf")):
        refused(weigh, lib, pc=args(theta=theta, **more), match="theta")
    refused(weigh, lib, held=short, match="weights hold")
    refused(weigh, lib, out=short, match="weights hold")
    refused(weigh, lib, held=desc(F16, S * KV * WIDTH * 4), match="weights must be F32")
    refused(weigh, lib, pc=args(theta=1.0, n_heads=H, step_idx=WIDTH - 1), match="step_idx")
    refused(weigh, lib, pc=args(theta=1.0, n_heads=H, step_idx=0xFFFFFFFF), match="weights hold")
    # a bound on the lengths makes shorter rows enough
    few = desc(F32, S * KV * 10 * 4)
    assert weigh(lib, held=few, out=few, pc=args(theta=0.0, n_heads=H, step_idx=10, max_seq_len=10))["count"] == T * H
    refused(plan, lib, "paged_kv_weights", [desc(F16, T * H * D * 2), pool(F16)] + batch() + [lse_of()], [good], pc=args(theta=1.0, **more))


def test_evict_refusals(lib):
    more = dict(seq_len=TOP, step_idx=WIDTH)
    refused(evict, lib, pc=b"", match="push constants")
    refused(evict, lib, pc=args(**{**more, "head_dim": 257}), match="head_dim")
    refused(evict, lib, pc=args(**{**more, "M": 0}), match="KV heads")
    refused(evict, lib, pc=args(**{**more, "K": S + 1}))
    refused(evict, lib, pc=args(**{**more, "K": 65536}), match="65535")
    refused(evict, lib, pc=args(**{**more, "step_idx": WIDTH - 1}), match="step_idx")
    refused(evict, lib, pc=args(**{**more, "seq_len": TOP + 1}), match="kept positions")
    refused(evict, lib, pc=args(**{**more, "seq_len": 2 * BS + 1}), match="new block tables")
    refused(evict, lib, pc=args(**{**more, "seq_len": 0xFFFFFFFF}), match="rows")
    refused(evict, lib, pools=[pool(F16), pool(I8)], match="one dtype")
    refused(evict, lib, to=[pool(F16), pool(F32)], match="one dtype")
    refused(evict, lib, to=[pool(I8)] * 2, match="one dtype")
    refused(evict, lib, pl=BF16)
    refused(evict, lib, pl=I8, pc=args(**{**more, "head_dim": 48}), match="32")
    refused(evict, lib, rows=desc(F32, S * KV * WIDTH * 4 - 4), match="weights hold")
    refused(evict, lib, rows_to=desc(F16, S * KV * WIDTH * 4), match="weights must be F32")
    refused(evict, lib, tables=desc(I32, S * W * 4 - 4), match="tables")
    refused(evict, lib, lens=desc(I32, S * 4 - 4), match="lengths")
    refused(evict, lib, budget=desc(I32, S * 8 - 4), match="budgets")
    refused(evict, lib, new=desc(I32, S * 2 * 4 - 4), match="new block tables")
    refused(evict, lib, lens_to=desc(I32, S * 4 - 4), match="new lengths")
    refused(evict, lib, kept=desc(I32, S * KV * TOP * 4 - 4), match="kept positions")
    refused(plan, lib, "paged_kv_evict", [pool(F16)] * 2, [pool(F16)] * 2, pc=args(**more), match="7 inputs")
    assert evict(lib, pc=args(**{**more, "seq_len": 0}))["count"] == 0


def test_no_sizes_wrap(lib):
    """Products of sizes that pass 64 bits are refused, not taken for small."""
    big = dict(M=65535, K=65535, N=0xFFFFFFFF, window_size=65536, head_dim=256)
    refused(evict, lib, pc=args(**{**big, "seq_len": 1 << 22, "step_idx": 0xFFFFFFFF}))
    refused(weigh, lib, pc=args(**{**big, "seq_len": 1, "n_heads": 65535, "step_idx": 0xFFFFFFFF, "theta": 1.0}))


def test_prefix_of_too_many_positions(lib):
    """A sequence may hold 2^30 positions at most, by its table or by max_seq_len: a row of a group that sees all of its shared
    positions is at position 2^30 - 1 for the kernels."""
    wide = dict(n_heads=H, step_idx=GROUPS, N=16385, window_size=65536)
    sized = dict(pools=[desc(F16, 1 << 40)] * 2, bat=[desc(I32, S * 16385 * 4)] + batch()[1:])
    refused(prefix, lib, pc=args(**wide), match="2\\^30", **sized)
    refused(prefix, lib, pc=args(**wide, max_seq_len=(1 << 30) + 1), match="2\\^30", **sized)
    assert prefix(lib, pc=args(**wide, max_seq_len=1 << 30), **sized)["count"] == T * H
    assert prefix(lib, pc=args(**{**wide, "N": 16384}), **sized)["count"] == T * H


def test_evict_of_too_many_positions(lib):
    """A sequence may hold 2^30 positions at most, by its table or by max_seq_len."""
    wide = dict(seq_len=TOP, N=16385, window_size=65536)
    tables, blocks = desc(I32, S * 16385 * 4), [desc(F16, 1 << 40)] * 2
    sized = dict(pools=blocks, to=blocks, tables=tables, rows=desc(F32, 1 << 50), rows_to=desc(F32, 1 << 50))
    refused(evict, lib, pc=args(**wide, step_idx=0x7FFFFFFF), match="2\\^30", **sized)
    assert evict(lib, pc=args(**wide, step_idx=1 << 30, max_seq_len=1 << 30), **sized)["count"] == S * KV * TOP
