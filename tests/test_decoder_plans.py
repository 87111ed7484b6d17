"""How the decoder block's calls choose to run a geometry: host arithmetic, no GPU (256 compute units are assumed without one)."""
import ctypes
import random
import re

import pytest

from deep_learning_framework_amd import kai
from deep_learning_framework_amd.kai import KaiError, VMath


@pytest.mark.parametrize("geometry,expected", [
    ((32, 1, 32, 8, 128, 64, 65), "tiles of 16 rows, 4 parts, scratch 2129920"),
    ((3, 61, 12, 12, 64, 48, 33), "tiles of 32 rows, 7 parts, scratch 4058208"),
    ((1, 16, 32, 8, 128, 256, 513), "tiles of 64 rows, 32 parts, scratch 8519680"),
    ((1, 1, 4, 2, 64, 16, 1), "tiles of 16 rows, 1 part, scratch 0"),
    ((2, 4, 3, 1, 20, 5, 8), "a wave a row, 1 part, scratch 0"),
    ((2, 4, 3, 1, 256, 64, 80), "a wave a row, 40 parts, scratch 990720"),
    ((2, 4, 3, 1, 64, 64, 0), "tiles of 16 rows, 1 part, scratch 0"),
    ((0, 4, 3, 1, 64, 64, 2), "nothing"),
    ((2, 0, 3, 1, 64, 64, 2), "nothing"),
])
def test_cache_attention_plans(geometry, expected):
    assert VMath.cache_attention_plan(*geometry) == expected


@pytest.mark.parametrize("which,yvec,ndat,xvec,expected", [
    ("forward", 512, 16, 256, "rows"),
    ("forward", 11008, 1, 4096, "separate"),
    ("forward", 3, 4, 0, "separate"),
    ("forward", 333, 1000, 777, "tiles 64 x 128, 0 whole, 96 in 2 parts, scratch 6291456"),
    ("x", 4096, 2048, 1024, "tiles 256 x 128, 0 whole, 64 in 4 parts, scratch 33554432"),
    ("weights", 4096, 2048, 1024, "tiles 256 x 128, 256 whole, scratch 0"),
    ("x", 40, 70, 72, "separate"),
    ("weights", 40, 70, 72, "separate"),
    ("forward", 0, 4, 8, "nothing"),
    ("x", 8, 0, 8, "nothing"),
])
def test_gated_plans(which, yvec, ndat, xvec, expected):
    assert VMath.gated_plan(which, yvec, ndat, xvec) == expected


def test_scratch_stays_below_what_a_product_may_ask():
    """Callers reserve 64 MiB for a product's parts before they record a graph."""
    rng = random.Random(5)
    size = lambda low, high: int(round(2 ** rng.uniform(low, high)))
    shapes = [(11008, 4096, 4096), (18371, 4849, 14840), (193, 193, 4096)]
    for yvec, ndat, xvec in shapes + [(size(6, 15), size(6, 14), size(6, 15)) for _ in range(4000)]:
        for which in ("forward", "x", "weights"):
            text = VMath.gated_plan(which, yvec, ndat, xvec)
            if text.startswith("tiles"):
                tile = re.match(r"tiles (\d+) x (\d+), (\d+) whole(?:, (\d+) in (\d+) parts)?, scratch (\d+)$", text)
                rows, columns, whole, cut, parts, scratch = (int(v or 0) for v in tile.groups())
                assert scratch == 4 * rows * columns * cut * parts <= 64 << 20, (which, yvec, ndat, xvec, text)
    for _ in range(4000):
        nkv, group = rng.choice([1, 2, 3, 8, 12, 64]), rng.choice([1, 2, 5, 8])
        geometry = (size(0, 8), size(0, 8), nkv * group, nkv, rng.choice([32, 64, 80, 96, 128, 20, 256, 1]), size(0, 10), size(0, 14))
        text = VMath.cache_attention_plan(*geometry)
        assert int(text.rsplit(" ", 1)[1]) < 64 << 20, (geometry, text)


def test_plans_check_their_arguments():
    for bad in ((-1, 1, 4, 2, 64, 16, 2), (1, 1, 4, 3, 64, 16, 2), (1, 1, 4, 0, 64, 16, 2), (1, 1, 4, 2, 257, 16, 2),
                (1, 1, 4, 2, 64, -1, 2), (1, 1, 4, 2, 64, 2 ** 16, 2 ** 16), (2 ** 22, 8, 4, 2, 64, 16, 2)):
        with pytest.raises(KaiError) as e:
            VMath.cache_attention_plan(*bad)
        assert e.value.code == 510
    for bad in ((-1, 4, 8), (4, 2 ** 31, 8), (4, 4, -2)):
        with pytest.raises(KaiError) as e:
            VMath.gated_plan("x", *bad)
        assert e.value.code == 510
    L = kai.load()
    buf = ctypes.create_string_buffer(64)
    assert L.kai_gated_plan(3, 4, 4, 4, buf, 64) == 510
    assert L.kai_gated_plan(0, 4, 4, 4, None, 64) == 523 and L.kai_gated_plan(0, 4, 4, 4, buf, 0) == 510
    assert L.kai_cache_attention_plan(1, 1, 4, 2, 64, 16, 2, None, 64) == 523
    assert L.kai_cache_attention_plan(1, 1, 4, 2, 64, 16, 2, buf, 0) == 510
    assert L.kai_cache_attention_plan(1, 1, 4, 2, 64, 16, 2, buf, 6) == 0 and buf.value == b"tiles"    # truncated, terminated
