"""Refusals and plans of the serving ops (paged cache, chunk attention, sampling), without a GPU: the planner that
dispatch() uses, through nf_hip_plan_dispatch."""
import pytest

from neurofabric_amd import abi
from neurofabric_amd.plugin import NfError, load_library, plan, push_constants

F32, F16, BF16, I8, I32, Q8 = (abi.NF_DTYPE_F32, abi.NF_DTYPE_F16, abi.NF_DTYPE_BF16, abi.NF_DTYPE_I8, abi.NF_DTYPE_I32,
                               abi.NF_DTYPE_Q8_0)
SIZE = {F32: 4, F16: 2, BF16: 2, Q8: 4}
T, KV, H, D, BS, W, S, BLOCKS = 10, 2, 8, 64, 16, 3, 4, 6


@pytest.fixture(scope="module")
def lib():
    return load_library()


def desc(dtype, nbytes):
    return abi.make_desc(dtype, nbytes)


def pool(dtype, blocks=BLOCKS, bs=BS, d=D, kv=KV):
    n = blocks * kv * bs * d
    return desc(dtype, n + n // 16 if dtype == I8 else n * SIZE[dtype])


def args(**over):
    a = dict(M=KV, N=W, K=S, seq_len=T, head_dim=D, window_size=BS)
    a.update(over)
    return push_constants(**a)


def batch(seqs=S, width=W):
    return [desc(I32, seqs * width * 4), desc(I32, (seqs + 1) * 4), desc(I32, seqs * 4)]


def append(lib, act=F16, pl=F16, rows=None, pools=None, bat=None, pc=None):
    rows = rows or [desc(act, T * KV * D * SIZE[act])] * 2
    return plan(lib, "paged_kv_append", rows + (bat or batch()), pools or [pool(pl)] * 2, pc=args() if pc is None else pc)


def gather(lib, act=F16, pl=F16, rows=None, pools=None, bat=None, pc=None):
    rows = rows or [desc(act, T * KV * D * SIZE[act])] * 2
    return plan(lib, "paged_kv_gather", (pools or [pool(pl)] * 2) + (bat or batch()), rows, pc=args() if pc is None else pc)


def chunk(lib, act=F16, pl=F16, q=None, out=None, pools=None, bat=None, pc=None):
    q, out = q or desc(act, T * H * D * SIZE[act]), out or desc(act, T * H * D * SIZE[act])
    return plan(lib, "flash_attention_paged_chunk", [q] + (pools or [pool(pl)] * 2) + (bat or batch()), [out],
                pc=args(n_heads=H) if pc is None else pc)


def refused(call, *a, match=None, **k):
    with pytest.raises(NfError, match=match) as e:
        call(*a, **k)
    assert e.value.status == 1  # NF_ERROR_INVALID_ARG


@pytest.mark.parametrize("act,pl,name", [(F32, F32, "f32_f32"), (F32, I8, "f32_i8"), (F16, F16, "f16_f16"),
                                         (F16, I8, "f16_i8")])
def test_plans(lib, act, pl, name):
    p = append(lib, act, pl)
    assert p["kernel"] == "paged_append_" + name and p["count"] == T * KV * D
    cells = 2 * (T * KV * D * 17 // 16 if pl == I8 else T * KV * D * SIZE[act])
    assert p["act_bytes"] == 2 * T * KV * D * SIZE[act] and p["out_bytes"] == cells
    p = gather(lib, act, pl)
    assert p["kernel"] == "paged_gather_" + name and p["act_bytes"] == cells
    assert chunk(lib, act, pl)["kernel"] == "attention_paged_chunk_" + name


@pytest.mark.parametrize("call", [append, gather, chunk])
def test_batch_refusals(lib, call):
    heads = {"n_heads": H} if call is chunk else {}
    refused(call, lib, pc=b"", match="push constants")
    refused(call, lib, pc=args(head_dim=0, **heads), match="head_dim")
    refused(call, lib, pc=args(head_dim=257, **heads), match="head_dim")
    refused(call, lib, pc=args(K=S + 1, **heads))
    refused(call, lib, pc=args(N=W + 1, **heads), match="tables")
    refused(call, lib, pc=args(K=65536, **heads), match="65535")
    refused(call, lib, pc=args(window_size=65537, **heads), match="65536")
    refused(call, lib, pc=args(seq_len=T + 1, **heads))
    refused(call, lib, pc=args(seq_len=0xFFFFFFFF, **heads))
    refused(call, lib, pc=args(seq_len=(1 << 22) + 1, **heads), match="rows")
    refused(call, lib, bat=[desc(I32, S * W * 4 - 4)] + batch()[1:], match="tables")
    refused(call, lib, bat=[batch()[0], desc(I32, S * 4), batch()[2]], match="starts")
    refused(call, lib, bat=batch()[:2] + [desc(I32, S * 4 - 4)], match="lengths")
    refused(call, lib, pools=[pool(F16), pool(I8)], match="one dtype")
    refused(call, lib, act=F32, pl=F16, match="dtype or I8")
    refused(call, lib, act=F16, pl=F32, match="dtype or I8")
    refused(call, lib, act=BF16, pl=BF16, match="F32 or F16")
    refused(call, lib, pl=Q8, match="dtype or I8")
    n = T * (H if call is chunk else KV) * 48 * 2
    over = dict(q=desc(F16, n), out=desc(F16, n)) if call is chunk else dict(rows=[desc(F16, n)] * 2)
    refused(call, lib, pl=I8, pc=args(head_dim=48, **heads), match="32", **over)


def test_row_refusals(lib):
    good, short = desc(F16, T * KV * D * 2), desc(F16, T * KV * D * 2 - 2)
    for call in (append, gather):
        refused(call, lib, pc=args(M=0), match="KV heads")
        refused(call, lib, rows=[short, good], match="hold fewer")
        refused(call, lib, rows=[good, short], match="hold fewer")
        refused(call, lib, rows=[good, desc(F32, T * KV * D * 4)], match="one dtype")
    refused(chunk, lib, q=desc(F16, T * H * D * 2 - 2), match="Q holds")
    refused(chunk, lib, out=desc(F16, T * H * D * 2 - 2), match="output holds")
    refused(chunk, lib, out=desc(F32, T * H * D * 4), match="one dtype")
    refused(chunk, lib, pc=args(n_heads=1), match="n_heads")
    refused(chunk, lib, pc=args(n_heads=0, M=0), match="KV heads")


def test_arity(lib):
    rows, pools = [desc(F16, T * KV * D * 2)] * 2, [pool(F16)] * 2
    refused(plan, lib, "paged_kv_append", rows + batch()[:2], pools, pc=args())
    refused(plan, lib, "paged_kv_append", rows + batch(), pools[:1], pc=args())
    refused(plan, lib, "paged_kv_gather", pools + batch()[:2], rows, pc=args())
    refused(plan, lib, "flash_attention_paged_chunk", rows[:1] + pools + batch()[:2], rows[:1], pc=args(n_heads=H))
    refused(plan, lib, "flash_attention_paged_chunk", rows[:1] + pools + batch(), [], pc=args(n_heads=H))


def test_defaults(lib):
    """Block size 16 without one; every query head has its own KV head without M."""
    assert append(lib, pc=args(window_size=0))["count"] == T * KV * D
    assert chunk(lib, pc=args(n_heads=H, M=0), pools=[pool(F16, kv=H)] * 2)["count"] == T * H


def sample(lib, rows=3, n=100, act=F32, logits=None, u=None, par=None, k=None, tok=None, prob=None, pc=None):
    ins = [logits or desc(act, rows * n * SIZE[act]), u or desc(F32, rows * 4), par or desc(F32, rows * 12),
           k or desc(I32, rows * 4)]
    return plan(lib, "sample_token", ins, [tok or desc(I32, rows * 4), prob or desc(F32, rows * 4)],
                pc=push_constants(seq_len=rows, N=n) if pc is None else pc)


def test_sample(lib):
    assert sample(lib)["kernel"] == "sample_token_f32" and sample(lib, act=F16)["kernel"] == "sample_token_f16"
    assert sample(lib, rows=0)["count"] == 0
    refused(sample, lib, pc=b"", match="push constants")
    refused(sample, lib, n=0, match="2\\^22")
    refused(sample, lib, n=(1 << 22) + 1, match="2\\^22")
    refused(sample, lib, rows=65536, match="65535")
    refused(sample, lib, act=BF16, match="F32 or F16")
    refused(sample, lib, logits=desc(F32, 3 * 100 * 4 - 4), match="logits")
    refused(sample, lib, u=desc(F32, 8), match="random numbers")
    refused(sample, lib, par=desc(F32, 32), match="parameters")
    refused(sample, lib, k=desc(I32, 8), match="top_k")
    refused(sample, lib, tok=desc(I32, 8), match="outputs")
    refused(sample, lib, prob=desc(F32, 8), match="outputs")
    refused(plan, lib, "sample_token", [desc(F32, 400)] * 3, [desc(I32, 4)] * 2, pc=push_constants(seq_len=1, N=100))
    refused(plan, lib, "sample_token", [desc(F32, 400)] * 4, [desc(I32, 4)], pc=push_constants(seq_len=1, N=100))


@pytest.mark.parametrize("call", [append, gather])
def test_most_elements(lib, call):
    """A thread per element where rows are not whole pieces: rounded up to workgroups they stay below 2^32."""
    def rows(t, kv, d):
        dense, pl = [desc(F16, t * kv * d * 2)] * 2, [pool(F16, kv=kv, d=d)] * 2
        return dict(rows=dense, pools=pl, pc=args(seq_len=t, M=kv, head_dim=d))
    assert call(lib, **rows(4095, 4097, 256))["count"] == 2 ** 32 - 256
    refused(call, lib, **rows(8191, 8193, 64), match="too many rows")  # 2^32 - 64
