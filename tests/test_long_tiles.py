"""The bound on the tiles of a batch's query rows that flash_attention_paged_prefix sizes its launch by, against a count."""
import ctypes
import random
import subprocess
from pathlib import Path

import pytest

SOURCE = """
#include "paged_tiles.hpp"
extern "C" unsigned long long bound(unsigned long long rows, unsigned long long parts, unsigned long long group,
                                    unsigned long long few, unsigned long long narrow, unsigned long long wide) {
  return nfhip::most_tiles(rows, parts, group, few, narrow, wide);
}
"""
# (few, narrow, wide) of the f16 kernels with 16 and 32 rows a narrow tile, and of the f32 kernel
HEIGHTS = [(64, 16, 128), (64, 32, 128), (32, 16, 64)]


@pytest.fixture(scope="module")
def bound(tmp_path_factory):
    at = tmp_path_factory.mktemp("tiles")
    (at / "tiles.cpp").write_text(SOURCE)
    csrc = Path(__file__).resolve().parents[1] / "neurofabric_amd" / "csrc"
    subprocess.run(["g++", "-std=c++17", "-O1", "-shared", "-fPIC", f"-I{csrc}", str(at / "tiles.cpp"), "-o", str(at / "tiles.so")],
                   check=True)
    f = ctypes.CDLL(str(at / "tiles.so")).bound
    f.restype, f.argtypes = ctypes.c_uint64, [ctypes.c_uint64] * 6
    return f


def count(tokens, group, few, narrow, wide):
    """The tiles of parts of so many tokens each."""
    return sum(-(-n * group // (narrow if n * group <= few else wide)) for n in tokens)


@pytest.mark.parametrize("few,narrow,wide", HEIGHTS)
@pytest.mark.parametrize("group,tokens", [(12, [3] * 400), (12, [2] * 400), (6, [3] * 400), (7, [5] * 1300), (5, [7] * 1400),
                                          (3, [11] * 1400), (3, [6] * 1400), (12, [3] * 100), (33, [1] * 500), (71, [1] * 500)])
def test_heads_that_do_not_divide_a_tile(bound, few, narrow, wide, group, tokens):
    assert bound(sum(tokens) * group, len(tokens), group, few, narrow, wide) >= count(tokens, group, few, narrow, wide)


@pytest.mark.parametrize("few,narrow,wide", HEIGHTS)
def test_random_batches(bound, few, narrow, wide):
    rng = random.Random(narrow * wide)
    for _ in range(20000):
        group = rng.choice([1, 2, 3, 4, 5, 6, 7, 8, 12, 14, 16, 20, 33, 40, 71, 160, rng.randint(1, 300)])
        most = rng.choice([1, 3, 9, 90])
        tokens = [rng.randint(0, most) for _ in range(rng.randint(1, 40))] + [1]
        pad = rng.choice([0, 0, 3])  # rows of no sequence
        n = bound((sum(tokens) + pad) * group, len(tokens), group, few, narrow, wide)
        assert n >= count(tokens, group, few, narrow, wide), (group, tokens, pad)


@pytest.mark.parametrize("few,narrow,wide", HEIGHTS)
def test_like_parts_are_counted_exactly(bound, few, narrow, wide):
    """Single tokens, and parts whose rows are full tiles, have no more than they need."""
    for group in (1, 2, 4, 8, 16):
        assert bound(500 * group, 500, group, few, narrow, wide) == 500
        assert bound(50 * wide, 50, group, few, narrow, wide) <= 50 * (wide // narrow)
