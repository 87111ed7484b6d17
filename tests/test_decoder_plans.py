"""How the decoder block's calls choose to run a geometry: host arithmetic, no GPU (256 compute units are assumed without one)."""
import ctypes

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
