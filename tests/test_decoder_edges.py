"""Calls of the decoder block's operators at the edge of what they allow: a cache of no pages, keys that are NaN where rows see
them, inputs of no columns, lengths that move while a recorded call names them."""
import numpy as np
import pytest

from deep_learning_framework_amd import kai
from deep_learning_framework_amd.kai import DeviceBuffer, KaiError, VMath
from deep_learning_framework_amd.tensor_ops import KeyValueCache, Tensor, gated, gated_backprop

from test_decoder_ops import ACTS, REL_FRO_TOL, _attend, _attention_case, _expected, dev_int, rel_fro


@pytest.mark.gpu
@pytest.mark.parametrize("npiece", [64, 20])
def test_cache_of_no_pages(npiece):
    """A table and lengths, but no page: nothing is read or written, and every new token sees nothing."""
    q = np.ones((2, 3, 4 * npiece), np.float32)
    y = DeviceBuffer.from_numpy(np.full(q.shape, 5.0, np.float32))
    table, lens = dev_int([[0, 1], [2, 0]]), dev_int([20, 3])
    k = DeviceBuffer.from_numpy(np.ones((2, 3, 2 * npiece), np.float32))
    VMath.cache_append(0, None, None, k, k, table, lens, None, None, 2, 3, 2 * npiece, 2, npiece, 0, 16, 2, None)
    VMath.cache_attention(0, y, DeviceBuffer.from_numpy(q), None, None, table, lens, None, None, 2, 3, 4 * npiece, 4, 2, npiece,
                          0, 16, 2, kai.hyper(0.1))
    assert np.all(y.to_numpy(q.shape) == 0)


@pytest.mark.gpu
@pytest.mark.parametrize("npiece", [64, 20])
@pytest.mark.parametrize("where", ["keys", "values"])
def test_nan_that_a_row_sees_reaches_it(npiece, where):
    """Some hundred keys (whole parts of the sequence) or values are NaN: every row that sees them is NaN, where their weight
    has vanished too, and the sequence beside it is as before."""
    rng = np.random.default_rng(40)
    c = _attention_case(rng, 2, 3, 4, 2, npiece, 32, [3000, 2900], None, False)
    c["q"][0] = 1.0
    c["ck"][c["table"][0, 5]] = -40.0            # scores of about -320 (64) and -179 (20) against some tens
    clean = _attend(c)
    want, room = _expected(c)
    assert np.all(np.abs(clean - want) <= room)
    if where == "keys":
        c["ck"][c["table"][0, 20:40]] = np.nan
    else:
        c["cv"][c["table"][0, 5]] = np.nan
    got = _attend(c)
    assert np.all(np.isnan(got[0]))
    assert np.array_equal(got[1], clean[1])


@pytest.mark.gpu
def test_gated_without_columns():
    """x of no columns: the projections are their biases."""
    x, w = Tensor((3, 2, 0)), Tensor((4, 0))
    bg, bu = np.arange(4, dtype=np.float32), np.ones(4, np.float32) * 3
    y = gated(x, w, w, Tensor.from_numpy(bg), Tensor.from_numpy(bu), actfunc="relu", keep=True)
    assert y.shape == (3, 2, 4)
    assert np.array_equal(y.numpy(), np.broadcast_to(bg * bu, y.shape))
    g = gated_backprop(y, Tensor.from_numpy(np.ones(y.shape, np.float32)))
    assert np.array_equal(g["bu"].numpy(), 6 * bg)
    assert np.array_equal(g["bg"].numpy(), [0, 18, 18, 18])


@pytest.mark.gpu
def test_accepted_lengths_stand_where_they_stood():
    cache = KeyValueCache(2, 1, 16, 4, 2)
    place = cache._len.ptr
    cache.accept([3, 1])
    cache.accept(2)
    assert cache._len.ptr == place and np.array_equal(cache._len.to_numpy(2, np.int32), [5, 3])
    for counts in (4, [-6, 0], [[1, 1]], [1, 1, 1]):
        with pytest.raises((KaiError, ValueError)):
            cache.accept(counts)
    assert np.array_equal(cache._len.to_numpy(2, np.int32), [5, 3])


@pytest.mark.gpu
@pytest.mark.parametrize("ndat,xvec,yvec", [(2, 4096, 260), (24, 4096, 260), (32, 4096, 97), (32, 512, 1030), (16, 1025, 2049)])
def test_gated_few_rows_both_ways(ndat, xvec, yvec):
    """Up to 32 rows: long reductions with few outputs run as the dense layer's products, the others in one launch."""
    rng = np.random.default_rng(ndat + yvec)
    x = rng.standard_normal((ndat, xvec)).astype(np.float32)
    wg, wu = ((rng.uniform(-1, 1, (yvec, xvec)) * xvec ** -0.5).astype(np.float32) for _ in range(2))
    bu = rng.standard_normal(yvec).astype(np.float32)
    T = Tensor.from_numpy
    y = gated(T(x), T(wg), T(wu), None, T(bu), actfunc="swish", keep=True)
    gate, up = x.astype(np.float64) @ wg.T, x.astype(np.float64) @ wu.T + bu
    assert rel_fro(y.saved["gate"].numpy(), gate) <= REL_FRO_TOL
    assert rel_fro(y.saved["up"].numpy(), up) <= REL_FRO_TOL
    assert rel_fro(y.numpy(), ACTS["swish"][0](gate) * up) <= REL_FRO_TOL
    assert np.array_equal(gated(T(x), T(wg), T(wu), None, T(bu), actfunc="swish").numpy(), y.numpy())


@pytest.mark.gpu
@pytest.mark.parametrize("ndat,xvec,yvec", [(1500, 1003, 3001), (1100, 4350, 1001)])
@pytest.mark.parametrize("acc", [False, True])
def test_gated_more_tiles_than_compute_units(ndat, xvec, yvec, acc):
    """Whole rounds of tiles over the chip and a cut rest, with edges in both directions: every output is written once."""
    rng = np.random.default_rng(ndat)
    x = rng.standard_normal((ndat, xvec)).astype(np.float32)
    wg, wu = ((rng.uniform(-1, 1, (yvec, xvec)) * xvec ** -0.5).astype(np.float32) for _ in range(2))
    gy = rng.standard_normal((ndat, yvec)).astype(np.float32)
    T = Tensor.from_numpy
    tx, twg, twu, tgy = T(x), T(wg), T(wu), T(gy)
    y = gated(tx, twg, twu, actfunc="swish", keep=True)
    gate, up = x.astype(np.float64) @ wg.T, x.astype(np.float64) @ wu.T
    act, slope = ACTS["swish"]
    assert rel_fro(y.saved["gate"].numpy(), gate) <= REL_FRO_TOL
    assert rel_fro(y.saved["up"].numpy(), up) <= REL_FRO_TOL
    assert rel_fro(y.numpy(), act(gate) * up) <= REL_FRO_TOL
    g32, u32 = (y.saved[n].numpy().astype(np.float64) for n in ("gate", "up"))
    gg, gu = gy * u32 * slope(g32), gy * act(g32)
    start = 2.0 if acc else np.nan                # a gradient that is not added to is not read
    out = {"x": T(np.full(x.shape, start)), "wg": T(np.full(wg.shape, start)), "wu": T(np.full(wu.shape, start))}
    VMath.gated_backward(0, out["x"].ptr, out["wg"].ptr, out["wu"].ptr, None, None, None, tgy.ptr, twg.ptr, twu.ptr, tx.ptr,
                         y.saved["gate"].ptr, y.saved["up"].ptr, yvec, ndat, xvec, y.saved["actfunc"], None, acc)
    want = {"x": gg @ wg + gu @ wu, "wg": gg.T @ x, "wu": gu.T @ x}
    for n, t in out.items():
        assert rel_fro(t.numpy(), want[n] + (2.0 if acc else 0.0)) <= REL_FRO_TOL, n
