"""What the tensor-level callers of a decoder block's operators refuse before an address reaches a kernel.  Tensors of device -1
live in host memory, and the library refuses that device itself (510), so a call that passes its own checks ends there and none
of this needs a GPU."""
import numpy as np
import pytest

from deep_learning_framework_amd import kai
from deep_learning_framework_amd.kai import DeviceBuffer, KaiError
from deep_learning_framework_amd.tensor_ops import KeyValueCache, Tensor, gated, gated_backprop, rotate

HOST = -1
SHAPE, LIBRARY = 10003, 510


def refused(code, call, *args, **kwargs):
    with pytest.raises(KaiError) as e:
        call(*args, **kwargs)
    assert e.value.code == code, e.value.message


def ints(a, device=HOST):
    return DeviceBuffer.from_numpy(np.asarray(a, np.int32), device)


def tensor(*shape):
    return Tensor(shape, HOST)


def test_counts_positions_and_masks_are_no_addresses():
    cache = KeyValueCache(2, 1, 8, 4, 4, device=HOST)
    k, q = tensor(2, 3, 8), tensor(2, 3, 16)
    append = lambda **a: cache.append(k, k, **a)
    attend = lambda **a: cache.attend(q, 2, **a)
    d = kai.rotary_desc(8)
    turn = lambda positions: rotate(q, 2, d, positions=positions)
    freed = ints([1, 1])
    freed.free()
    for call in (append, attend):
        for counts in (3.0, [1], [1, 2, 3], [1.5, 2.0], [[1, 2]], 2 ** 31, [True, False], "2", ints([1]), freed):
            refused(SHAPE, call, counts=counts)
        for counts in (None, 3, np.int64(2), [1, 3], np.array([0, 2]), ints([1, 1])):      # past their checks
            refused(LIBRARY, call, counts=counts)
    for positions in (4096, [0, 1, 2], np.zeros((2, 3)), np.full((2, 3), 2 ** 31), ints(np.zeros(5))):
        refused(SHAPE, append, positions=positions)
        refused(SHAPE, turn, positions)
    for positions in (None, np.zeros((2, 3), np.int64), ints(np.zeros(6))):
        refused(LIBRARY, append, positions=positions)
        refused(LIBRARY, turn, positions)
    for mask in (4096, np.zeros((2, 3), np.int32), np.zeros((2, 3, 2), np.int32), ints(np.zeros(5))):
        refused(SHAPE, attend, mask=mask)
    for mask in (None, np.full((2, 3, 1), 2 ** 32 - 1, np.uint32), np.zeros((2, 3, 1), np.int32), ints(np.zeros(6))):
        refused(LIBRARY, attend, mask=mask)
    other = ints([1, 1])
    other.device = 0              # a buffer of another device than the cache's
    refused(SHAPE, append, counts=other)
    other.device = HOST


def test_rotate_writes_into_its_own_shape_only():
    x, d = tensor(2, 3, 16), kai.rotary_desc(8)
    for out in (tensor(2, 3, 8), tensor(1, 3, 16), tensor(6, 16), tensor(2, 16, 3)):
        refused(SHAPE, rotate, x, 2, d, out=out)
    elsewhere = tensor(2, 3, 16)
    elsewhere.device = 0
    refused(SHAPE, rotate, x, 2, d, out=elsewhere)
    for heads in (0, -2, 3):
        refused(SHAPE, rotate, x, heads, d)
    for out in (None, x, tensor(2, 3, 16)):
        refused(LIBRARY, rotate, x, 2, d, out=out)


def test_a_rotary_description_is_no_address():
    x = tensor(2, 3, 16)
    for desc in (4096, 1.0, {"nrot": 8}, "halves"):
        refused(SHAPE, rotate, x, 2, desc)
        refused(SHAPE, KeyValueCache, 2, 1, 8, 4, 4, rotary=desc, device=HOST)
    refused(LIBRARY, KeyValueCache(2, 1, 8, 4, 4, rotary=kai.rotary_desc(8), device=HOST).append, tensor(2, 3, 8), tensor(2, 3, 8))


def test_gated_backprop_takes_a_gradient_of_the_result():
    y = tensor(5, 4)
    y.saved = {"op": "gated", "x": tensor(5, 3), "wg": tensor(4, 3), "wu": tensor(4, 3), "bg": None, "bu": None, "gate": tensor(5, 4),
               "up": tensor(5, 4), "actfunc": 8, "leaky_alpha": None}
    for shape in ((5, 3), (4, 4), (5,), (4, 5), (20,)):
        refused(SHAPE, gated_backprop, y, tensor(*shape))
    refused(LIBRARY, gated_backprop, y, tensor(5, 4))
    refused(SHAPE, gated_backprop, tensor(5, 4), tensor(5, 4))       # of a result that kept nothing
    x, w = tensor(5, 3), tensor(4, 3)
    refused(SHAPE, gated, x, w, tensor(3, 3))
    refused(SHAPE, gated, tensor(5, 4), w, w)
    refused(SHAPE, gated, x, w, w, tensor(3))


def test_accept_takes_whole_numbers(monkeypatch):
    monkeypatch.setattr(kai, "synchronize", lambda: None)
    cache = KeyValueCache(2, 1, 8, 4, 4, device=HOST)
    cache.accept(3)
    for counts in (1.7, [0.5, 1.0], [True, True], 2 ** 32 + 1, [2 ** 32, 0], -2 ** 32, 14, [-4, 0], [1, 1, 1], [[1, 1]]):
        with pytest.raises((KaiError, ValueError, OverflowError)):
            cache.accept(counts)
        assert list(cache.lengths) == [3, 3] and list(cache._len.to_numpy(2, np.int32)) == [3, 3]
    cache.accept([13, -3])
    assert list(cache._len.to_numpy(2, np.int32)) == [16, 0] and cache.lengths.dtype == np.int32


def test_append_refuses_what_finds_no_room(monkeypatch):
    monkeypatch.setattr(kai, "synchronize", lambda: None)
    cache, k = KeyValueCache(2, 1, 8, 4, 4, device=HOST), tensor(2, 3, 8)
    cache.accept([14, 0])
    for counts in (None, 3, 4, [3, 0], np.array([3, 1])):
        refused(SHAPE, cache.append, k, k, counts=counts)
    for counts in (2, [2, 3], [-1, 5], ints([3, 3])):        # the last is the device's to clip
        refused(LIBRARY, cache.append, k, k, counts=counts)
    refused(SHAPE, KeyValueCache(2, 1, 8, 1, 2, device=HOST).append, k, k)


def test_rotary_descriptions_whose_angles_are_no_numbers():
    """Each field is a number by itself, but not what is computed from it: cosines of infinity were written as NaN."""
    nothing = lambda d: kai.VMath.rotary(0, None, None, None, 0, 3, 512, 1, 512, d)      # no rows: the description alone counts
    parts = dict(scaling="parts", factor=2.0, trained=10.0)
    for d in (kai.rotary_desc(8, magnitude=1e39), kai.rotary_desc(8, magnitude=-1e300), kai.rotary_desc(512, base=1e-305), kai.rotary_desc(8, base=1e-300, scaling="linear", factor=1e-200),
              kai.rotary_desc(8, scaling="linear", factor=5e-324), kai.rotary_desc(8, scaling="linear", factor=1e-300),
              kai.rotary_desc(4, scaling="base", factor=1e-308), kai.rotary_desc(8, **dict(parts, factor=1e-300)),
              kai.rotary_desc(8, low_turns=0.0, high_turns=5e-324, **parts),
              kai.rotary_desc(8, low_turns=-1.7e308, high_turns=1.7e308, **parts)):
        refused(LIBRARY, nothing, d)
    for d in (kai.rotary_desc(8, base=0.5), kai.rotary_desc(8, base=1e-300), kai.rotary_desc(8, base=1e300), kai.rotary_desc(8, magnitude=3e38),
              kai.rotary_desc(8, scaling="linear", factor=1e-3), kai.rotary_desc(8, scaling="base", factor=1e300),
              kai.rotary_desc(8, low_turns=1.0, high_turns=1.0 + 2.0 ** -40, **parts)):
        nothing(d)


@pytest.mark.gpu
def test_host_values_reach_the_calls():
    """Counts, positions and masks from the host give what the same values on the device give."""
    rng = np.random.default_rng(5)
    r = lambda *s: Tensor.from_numpy(rng.standard_normal(s).astype(np.float32))
    k, v, q = r(2, 5, 16), r(2, 5, 16), r(2, 5, 32)
    counts, positions = np.array([5, 2]), rng.integers(0, 9, (2, 5))
    mask = np.zeros((2, 5, 1), np.uint32)
    mask[:, :, 0] = [1, 3, 5, 0x8000000B, 31]
    out = []
    for put in (lambda a: a, lambda a: DeviceBuffer.from_numpy(a.astype(np.uint32).view(np.int32))):
        cache = KeyValueCache(2, 1, 16, 4, 4, rotary=kai.rotary_desc(16))
        cache.append(k, v, counts=put(counts), positions=put(positions))
        turned = rotate(q, 2, cache.rotary, positions=put(positions))
        out.append([turned.numpy(), cache.attend(turned, 2, counts=put(counts), mask=put(mask)).numpy()])
    for a, b in zip(*out):
        assert np.array_equal(a, b)
    cache.append(k, v, counts=2)
    assert np.all(cache.attend(q, 2, counts=2).numpy()[:, 2:] == 0)
