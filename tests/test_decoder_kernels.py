"""Every tile of the attention over the cache and of the gated projection, by name: each case asserts the plan that it is there for
and then the results, against 64 bits, with what that kernel can get wrong (edges in both directions, cut and whole tiles side
by side, drafted trees, keys that are NaN and not seen, infinities, odd addresses).

Tolerances as in test_decoder_ops.py: the repository's relative Frobenius 1e-5 for sums in another order, and for the attention
the bound that is computed beside the result."""
import re

import numpy as np
import pytest

from util import REL_FRO_TOL, rel_fro

from deep_learning_framework_amd import kai
from deep_learning_framework_amd.kai import ACT, DeviceBuffer, VMath
from deep_learning_framework_amd.tensor_ops import Tensor, gated, gated_backprop

from test_decoder_ops import ACTS, _attend, _attention_case, _check_attention, _expected

pytestmark = pytest.mark.gpu

ALL_ACTS = dict(ACTS)
_L, _A = float(np.float32(1.0507009)), float(np.float32(1.6732632))
_soft = lambda g: np.log1p(np.exp(g))
ALL_ACTS["selu"] = (lambda g: np.where(g > 0, _L * g, _L * _A * np.expm1(np.minimum(g, 0))),
                    lambda g: np.where(g > 0, _L, _L * _A * np.exp(np.minimum(g, 0))))
ALL_ACTS["mish"] = (lambda g: g * np.tanh(_soft(g)),
                    lambda g: np.tanh(_soft(g)) + g * (1 - np.tanh(_soft(g)) ** 2) / (1 + np.exp(-g)))


# ---- attention over the cache ------------------------------------------------------------------------------------------

def wide_table(c, most):
    """The same cache behind a table of ``most`` pages a sequence, those that it does not use unassigned."""
    table = np.full((c["nbat"], most), -1, np.int32)
    table[:, :c["table"].shape[1]] = c["table"]
    c["table"], c["most"] = table, most
    return c


def plan_of(c):
    return VMath.cache_attention_plan(c["nbat"], c["ntimes"], c["nhead"], c["nkv"], c["npiece"], c["page"], c["most"])


TILES = [
    # rows, nbat, ntimes, nhead, nkv, page, pages a sequence, lens, counts, tree
    (16, 2, 5, 6, 2, 48, 40, [700, 33], [5, 3], True),
    (32, 2, 23, 8, 8, 48, 64, [700, 1201], [23, 11], True),
    (32, 1, 7, 32, 8, 100, 80, [1500], None, False),            # 28 rows of 32
    (64, 2, 23, 16, 4, 48, 256, [1100, 333], [23, 9], True),     # 92 rows: a whole tile and a part of one
    (64, 1, 45, 64, 64, 64, 80, [1400], None, True),             # two parts: a wave takes several tiles; two mask words
    (64, 3, 16, 32, 8, 100, 200, [0, 40, 900], [16, 0, 13], False),
    (64, 1, 130, 8, 2, 256, 128, [200], None, False),            # a run of 130 tokens, 520 rows of a key head
]


@pytest.mark.parametrize("npiece", [32, 64, 80, 96, 128])
@pytest.mark.parametrize("case", range(len(TILES)))
def test_attention_tiles(case, npiece):
    rows, nbat, ntimes, nhead, nkv, page, most, lens, counts, tree = TILES[case]
    rng = np.random.default_rng(1000 * case + npiece)
    c = wide_table(_attention_case(rng, nbat, ntimes, nhead, nkv, npiece, page, lens, counts, tree), most)
    assert plan_of(c).startswith("tiles of %d rows, " % rows), plan_of(c)
    got = _check_attention(c)
    assert np.array_equal(got, _attend(c)), "the same call twice gives the same bits"


@pytest.mark.parametrize("npiece", [32, 64, 80, 96, 128])
@pytest.mark.parametrize("case", [1, 3, 4])
def test_attention_tiles_unseen_keys_and_missing_pages(case, npiece):
    """Keys that no row sees, keys that some rows see, what stands behind the sequences, all NaN or infinite; a page in the middle
    is missing; strides and addresses off 16 bytes."""
    rows, nbat, ntimes, nhead, nkv, page, most, lens, counts, tree = TILES[case]
    rng = np.random.default_rng(77 * case + npiece)
    c = wide_table(_attention_case(rng, nbat, ntimes, nhead, nkv, npiece, page, lens, counts, tree, extra=9), most)
    c["table"][0, 3] = c["npage"]
    c["see_new"][:, :, 2] = False               # nobody sees new token 2, itself neither
    c["see_new"][0, 1] = False                  # and token 1 of the first sequence no new one
    assert plan_of(c).startswith("tiles of %d rows, " % rows)
    clean = _check_attention(c, q_off=1, c_off=3)
    want, room = _expected(c)
    used = {}
    for b in range(nbat):
        count = ntimes if c["counts"] is None else c["counts"][b]
        used[b] = c["lens"][b] + count
        for at in [c["lens"][b] + 2] + list(range(used[b], -(-used[b] // page) * page)):
            for name in ("ck", "cv"):
                c[name][c["table"][b, at // page], at % page] = rng.choice([np.nan, np.inf, -np.inf])
    spare = sorted(set(range(c["npage"])) - {int(c["table"][b, k]) for b in range(nbat) for k in range(-(-used[b] // page))})
    c["ck"][spare], c["cv"][spare] = np.nan, np.inf
    assert np.array_equal(_attend(c, q_off=1, c_off=3), clean)
    # token 4 of the first sequence turns into NaN: those that do not see it are as before, those that do are NaN
    n = c["lens"][0] + 4
    c["ck"][c["table"][0, n // page], n % page] = np.nan
    got = _attend(c)
    count = ntimes if c["counts"] is None else c["counts"][0]
    sees = c["see_new"][0][:count, 4]
    assert sees.any() and not sees.all()
    assert np.all(np.isnan(got[0, :count][sees]))
    assert np.all(np.abs(got[0, :count][~sees] - want[0, :count][~sees]) <= room[0, :count][~sees])
    if nbat > 1:
        rest = 1 if c["counts"] is None else c["counts"][1]
        assert np.all(np.abs(got[1, :rest] - want[1, :rest]) <= room[1, :rest])


LARGE = [
    # npiece, ntimes, nhead, nkv, page, pages a sequence, lens, plan
    (64, 3, 4, 2, 64, 3, [150], "tiles of 16 rows, 2 parts"), (64, 3, 4, 2, 128, 1, [100], "tiles of 16 rows, 1 part,"),
    (128, 23, 16, 4, 128, 128, [1100], "tiles of 64 rows"), (32, 7, 32, 8, 100, 80, [1500], "tiles of 32 rows"),
    (20, 3, 4, 2, 64, 20, [900], "a wave a row, 10 parts"), (20, 3, 4, 2, 128, 1, [100], "a wave a row, 1 part,"),
    (256, 2, 2, 1, 64, 20, [900], "a wave a row, 10 parts"),
]


@pytest.mark.parametrize("case", range(len(LARGE)))
def test_attention_of_large_values(case):
    """Values whose sum passes the largest float: their weighted mean does not, and small ones beside them keep their bits."""
    npiece, ntimes, nhead, nkv, page, most, lens, plan = LARGE[case]
    rng = np.random.default_rng(500 + case)
    c = wide_table(_attention_case(rng, 1, ntimes, nhead, nkv, npiece, page, lens, None, False), most)
    assert plan_of(c).startswith(plan), plan_of(c)
    c["cv"] = (rng.uniform(0.5, 1.0, c["cv"].shape) * 2e38).astype(np.float32)
    c["cv"][..., 1::2] *= np.float32(1e-38)
    c["cv"][..., 3::4] *= np.float32(1e-24)
    c["cv"][..., 2::8] *= -1
    got = _attend(c)
    want, _ = _expected(c)
    room = 0 * want
    for d in range(npiece):                      # the bound of each column by its own values
        room[..., d] = np.abs(c["cv"].reshape(-1, nkv, npiece)[:, :, d]).max()
    # relative to the largest value: the scores' errors as in test_decoder_ops.py (coef sum |q k| is below 30), and a rounding a key
    keys = lens[0] + ntimes
    off = (npiece + 2) * 2.0 ** -24 * 30
    assert np.all(np.abs(got - want) <= room * (2 * np.expm1(off) + (keys + 24) * 2.0 ** -24))
    assert np.abs(got).max() > 1e38


# ---- the gated projection's tiles -------------------------------------------------------------------------------------------

GATED_TILES = [
    # product, tile, which tiles are cut, yvec, ndat, xvec
    ("forward", "64 x 128", "cut", 40, 40, 260), ("forward", "64 x 128", "mixed", 700, 1500, 260), ("forward", "64 x 128", "whole", 40, 40, 17),
    ("forward", "128 x 128", "cut", 5001, 65, 1500), ("forward", "128 x 128", "mixed", 1500, 1500, 700),
    ("forward", "128 x 128", "whole", 5001, 260, 513),
    ("forward", "256 x 128", "cut", 5001, 200, 2049), ("forward", "256 x 128", "mixed", 3001, 1500, 513),
    ("forward", "256 x 128", "whole", 5001, 2049, 130),
    ("forward", "256 x 256", "mixed", 3001, 3001, 1500), ("forward", "256 x 256", "whole", 5001, 1500, 513),
    ("weights", "64 x 128", "cut", 300, 700, 700), ("weights", "64 x 128", "mixed", 3001, 513, 260), ("weights", "64 x 128", "whole", 40, 40, 17),
    ("weights", "128 x 128", "cut", 700, 2049, 260), ("weights", "128 x 128", "mixed", 2049, 513, 1003),
    ("weights", "128 x 128", "whole", 3001, 200, 260),
    ("weights", "256 x 128", "cut", 5001, 3001, 64), ("weights", "256 x 128", "mixed", 1500, 513, 3001),
    ("weights", "256 x 128", "whole", 5001, 200, 513),
    ("weights", "256 x 256", "mixed", 3001, 1500, 3001), ("weights", "256 x 256", "whole", 5001, 700, 1500),
    ("x", "64 x 128", "cut", 300, 300, 1500), ("x", "64 x 128", "mixed", 200, 2049, 1003), ("x", "64 x 128", "whole", 40, 200, 1500),
    ("x", "128 x 128", "cut", 700, 2049, 260), ("x", "128 x 128", "mixed", 200, 2049, 2049), ("x", "128 x 128", "whole", 65, 2049, 1003),
    ("x", "256 x 128", "cut", 1500, 3001, 260), ("x", "256 x 128", "mixed", 260, 3001, 3001), ("x", "256 x 128", "whole", 130, 2049, 3001),
    ("x", "256 x 256", "cut", 3001, 1500, 2049),
]


def assert_plan(which, tile, cuts, yvec, ndat, xvec):
    text = VMath.gated_plan(which, yvec, ndat, xvec)
    found = re.match(r"tiles (\d+ x \d+), (\d+) whole(, \d+ in \d+ parts)?, scratch \d+$", text)
    assert found and found.group(1) == tile, text
    assert ("whole" if not found.group(3) else "mixed" if int(found.group(2)) else "cut") == cuts, text


def offset_buffers(off):
    put = lambda a: DeviceBuffer.from_numpy(np.concatenate([np.full(off, 3.0, np.float32), np.ravel(a), np.full(9, 3.0, np.float32)]))
    at = lambda b: b.offset(4 * off)

    def get(b, shape):
        n = int(np.prod(shape))
        a = b.to_numpy(off + n + 9)
        assert np.all(a[:off] == 3.0) and np.all(a[off + n:] == 3.0), "nothing beside the outputs is written"
        return a[off:off + n].reshape(shape)
    return put, at, get


@pytest.mark.parametrize("off", [0, 1])
@pytest.mark.parametrize("case", range(len(GATED_TILES)))
def test_gated_tiles(case, off):
    which, tile, cuts, yvec, ndat, xvec = GATED_TILES[case]
    assert_plan(which, tile, cuts, yvec, ndat, xvec)
    rng = np.random.default_rng(case)
    r = lambda *s: rng.standard_normal(s, dtype=np.float32)
    x, wg, wu = r(ndat, xvec), r(yvec, xvec) * np.float32(xvec ** -0.5), r(yvec, xvec) * np.float32(xvec ** -0.5)
    put, at, get = offset_buffers(off)
    dx, dwg, dwu = put(x), put(wg), put(wu)      # addresses are taken of buffers that live as long as the call
    x8, wg8, wu8 = (a.astype(np.float64) for a in (x, wg, wu))
    if which == "forward":
        name = list(ALL_ACTS)[case % len(ALL_ACTS)]
        act = ALL_ACTS[name][0]
        bg, bu = r(yvec), r(yvec)
        gate, up = x8 @ wg8.T + bg, x8 @ wu8.T + bu
        outs = [put(np.full((ndat, yvec), np.nan, np.float32)) for _ in range(3)]
        dbg, dbu = put(bg), put(bu)
        VMath.gated_forward(0, *(at(o) for o in outs), at(dwg), at(dwu), at(dbg), at(dbu), at(dx), yvec, ndat, xvec, ACT[name],
                            kai.hyper(0.25))
        y, got_gate, got_up = (get(o, (ndat, yvec)) for o in outs)
        assert rel_fro(got_gate, gate) <= REL_FRO_TOL and rel_fro(got_up, up) <= REL_FRO_TOL
        # the activation's own slope (below 1.1) and the product pass the sums' errors on
        assert rel_fro(y, act(gate) * up) <= 2 * REL_FRO_TOL
        return
    gate, up, gy = r(ndat, yvec), r(ndat, yvec), r(ndat, yvec)
    act, slope = ALL_ACTS["swish"]
    g8, u8 = gate.astype(np.float64), up.astype(np.float64)
    gg, gu = gy * u8 * slope(g8), gy * act(g8)
    want = (gg @ wg8 + gu @ wu8,) if which == "x" else (gg.T @ x8, gu.T @ x8)
    dgy, dgate, dup = put(gy), put(gate), put(up)
    for acc in (False, True):
        start = [r(*w.shape) if acc else np.full(w.shape, np.nan, np.float32) for w in want]
        outs = [put(s) for s in start]
        addresses = [at(o) for o in outs]
        gradients = addresses + [None, None] if which == "x" else [None] + addresses
        VMath.gated_backward(0, *gradients, None, None, None, at(dgy), at(dwg), at(dwu), at(dx), at(dgate), at(dup), yvec, ndat, xvec,
                             ACT["swish"], None, acc)
        for o, s, w in zip(outs, start, want):
            assert rel_fro(get(o, w.shape), w + s if acc else w) <= REL_FRO_TOL


@pytest.mark.parametrize("off", [0, 1])
@pytest.mark.parametrize("yvec,ndat,xvec", [(700, 2049, 260), (1500, 513, 700)])
def test_gated_gradients_one_weight_missing(yvec, ndat, xvec, off):
    """One product in a launch that is made for two, added to what is there; bias sums alone."""
    rng = np.random.default_rng(ndat)
    r = lambda *s: rng.standard_normal(s, dtype=np.float32)
    assert VMath.gated_plan("weights", yvec, ndat, xvec).startswith("tiles") and VMath.gated_plan("x", yvec, ndat, xvec).startswith("tiles")
    put, at, get = offset_buffers(off)
    x, wg, wu, gate, up, gy = r(ndat, xvec), r(yvec, xvec), r(yvec, xvec), r(ndat, yvec), r(ndat, yvec), r(ndat, yvec)
    keep = list(map(put, (gy, wg, wu, x, gate, up)))
    ins = [at(b) for b in keep]
    act, slope = ALL_ACTS["swish"]
    g8, u8 = gate.astype(np.float64), up.astype(np.float64)
    gg, gu = gy * u8 * slope(g8), gy * act(g8)
    want = {"gx": gg @ wg + gu @ wu, "gwg": gg.T @ x, "gwu": gu.T @ x, "gbg": gg.sum(0), "gbu": gu.sum(0)}
    names = list(want)
    for wanted in (["gwg"], ["gwu"], ["gx", "gwu", "gbg"], ["gbg", "gbu"], ["gwg", "gbu"]):
        for acc in (False, True):
            start = {n: r(*want[n].shape) if acc else np.full(want[n].shape, np.nan, np.float32) for n in wanted}
            outs = {n: put(start[n]) for n in wanted}
            VMath.gated_backward(0, *(at(outs[n]) if n in outs else None for n in names), None, *ins, yvec, ndat, xvec, ACT["swish"],
                                 None, acc)
            for n in wanted:
                assert rel_fro(get(outs[n], want[n].shape), want[n] + start[n] if acc else want[n]) <= REL_FRO_TOL, (n, wanted)


@pytest.mark.parametrize("yvec,ndat,xvec", [(300, 300, 1500), (700, 2049, 260), (300, 700, 700), (40, 40, 17), (1500, 513, 700)])
def test_gated_gradients_infinities(yvec, ndat, xvec):
    """An infinity or a NaN in a weight, in x or in a gradient reaches exactly the sums that it enters, in whole tiles and in
    parts, in the last partial step and in either half of x's gradient."""
    rng = np.random.default_rng(yvec + xvec)
    r = lambda *s: rng.standard_normal(s, dtype=np.float32)
    x, wg, wu, gate, up, gy = r(ndat, xvec), r(yvec, xvec), r(yvec, xvec), r(ndat, yvec), r(ndat, yvec), r(ndat, yvec)
    wg[5, 7], wu[9, 7], wu[yvec - 1, 3], wg[2, 11] = np.inf, -np.inf, np.inf, np.nan
    x[4, 2], x[ndat - 1, 1], x[6, 13] = np.inf, -np.inf, np.nan
    gy[3, 11], x[3, 9], wg[11, 5] = np.inf, 0.0, 0.0
    gate[8, 1] = np.float32(-np.inf)
    f8 = lambda a: a.astype(np.float64)
    with np.errstate(all="ignore"):
        gg, gu = f8(gy * up), f8(gy * gate)                        # in 32 bits, as the kernel's first launch leaves them
        want = {"gx": gg @ f8(wg) + gu @ f8(wu), "gwg": gg.T @ f8(x), "gwu": gu.T @ f8(x)}
    out = {n: DeviceBuffer.from_numpy(np.zeros(w.shape, np.float32)) for n, w in want.items()}
    put = DeviceBuffer.from_numpy
    VMath.gated_backward(0, out["gx"], out["gwg"], out["gwu"], None, None, None, put(gy), put(wg), put(wu), put(x), put(gate), put(up),
                         yvec, ndat, xvec, ACT["none"], None, False)
    for n, w in want.items():
        got = out[n].to_numpy(w.shape)
        assert np.array_equal(np.isnan(got), np.isnan(w)), n
        over = np.isinf(w)
        assert over.any() and np.array_equal(got[over], w[over]), n
        fine = np.isfinite(w)
        assert rel_fro(got[fine], w[fine]) <= REL_FRO_TOL, n


@pytest.mark.parametrize("name", list(ALL_ACTS))
@pytest.mark.parametrize("ndat,xvec,yvec,way", [(1500, 260, 700, "tiles 64 x 128, 256 whole, 8 in"), (16, 256, 512, "rows"),
                                                (24, 4096, 260, "separate"), (40, 17, 40, "tiles 64 x 128, 1 whole")])
def test_every_activation_every_way(name, ndat, xvec, yvec, way):
    assert VMath.gated_plan("forward", yvec, ndat, xvec).startswith(way)
    rng = np.random.default_rng(ndat)
    r = lambda *s: rng.standard_normal(s, dtype=np.float32)
    x, wg, wu, gy = r(ndat, xvec), r(yvec, xvec) * np.float32(2 * xvec ** -0.5), r(yvec, xvec) * np.float32(xvec ** -0.5), r(ndat, yvec)
    act, slope = ALL_ACTS[name]
    T = Tensor.from_numpy
    tb = T(np.full(yvec, 0.125, np.float32))
    y = gated(T(x), T(wg), T(wu), tb, tb, actfunc=name, leaky_alpha=0.25, keep=True)
    f8 = lambda a: a.astype(np.float64)
    gate, up = f8(x) @ f8(wg).T + 0.125, f8(x) @ f8(wu).T + 0.125
    assert rel_fro(y.numpy(), act(gate) * up) <= 2 * REL_FRO_TOL
    g = gated_backprop(y, T(gy))
    g32, u32 = f8(y.saved["gate"].numpy()), f8(y.saved["up"].numpy())
    gg, gu = gy * u32 * slope(g32), gy * act(g32)
    want = {"x": gg @ f8(wg) + gu @ f8(wu), "wg": gg.T @ f8(x), "wu": gu.T @ f8(x), "bg": gg.sum(0), "bu": gu.sum(0)}
    for n, w in want.items():
        assert rel_fro(g[n].numpy(), w) <= REL_FRO_TOL, n
