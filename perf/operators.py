"""The operators of a decoder block, as cases that can be measured and checked.

Rotary positions (and their gradient), the cache of keys and values (written, and read by the attention of a tree of
drafted tokens), and the gated feed-forward projection (and its gradients), each in a plain form of elementary torch
operations and, where ``own`` is true, as the calls of ``deep_learning_framework_amd.kai`` that a user makes.
"""
import math

import torch

own = False

DEV = "cuda"
F4 = 4


# ---- the cases -------------------------------------------------------------------------------------------------

def listed():
    rot = {"kind": "rotary", "rows_given": True, "nrot": 0, "layout": "halves", "scaling": "none", "factor": 1.0,
           "backward": False, "far": 0}
    att = {"kind": "attention", "tree": True, "ragged": True, "page": 64}
    gated = {"kind": "gated", "backward": False, "keep": False, "bias": False, "act": "swish"}
    app = {"kind": "append", "page": 64, "nrot": 0, "layout": "halves", "ragged": False}
    return [
        # the queries of a small training batch of the 12-head attention block, positions 0 .. ntimes - 1
        dict(rot, name="rotary 2x384 12x64", nbat=2, ntimes=384, nhead=12, npiece=64, rows_given=False),
        # the gradient of a long-context training batch: half of each head rotated, pair layout, stretched positions
        dict(rot, name="rotary backward 4x4096 32x128", nbat=4, ntimes=4096, nhead=32, npiece=128, nrot=64,
             layout="pairs", scaling="parts", factor=8.0, backward=True, far=100000),
        # one step of a served batch: each sequence's token goes behind its own last one
        dict(app, name="append 64x1 8x128", nbat=64, ntimes=1, nkvhead=8, npiece=128, maxlen=640),
        # prompts entering the cache at once, of different lengths, pages of an odd size
        dict(app, name="append 4x2000 8x128", nbat=4, ntimes=2000, nkvhead=8, npiece=128, maxlen=300, ragged=True,
             page=48),
        # one token for each of many sequences: plain decoding
        dict(att, name="attention 32x1 over 4096", nbat=32, ntimes=1, nhead=32, nkvhead=8, npiece=128, maxlen=4096,
             tree=False),
        # drafted trees of an uneven batch, every head with keys of its own, heads of 64
        dict(att, name="attention tree 3x61 over 1500", nbat=3, ntimes=61, nhead=12, nkvhead=12, npiece=64,
             maxlen=1500, page=48),
        # one long context and a short draft
        dict(att, name="attention tree 1x16 over 131072", nbat=1, ntimes=16, nhead=32, nkvhead=8, npiece=128,
             maxlen=131072, page=256),
        # a single served token through both projections
        dict(gated, name="gated 1 4096-11008", ndat=1, xvec=4096, yvec=11008),
        # a drafted tree's rows, or a served batch's
        dict(gated, name="gated 24 4096-11008", ndat=24, xvec=4096, yvec=11008),
        # sizes off every tile, with biases, the error-function activation and what training keeps
        dict(gated, name="gated 1000 777-333", ndat=1000, xvec=777, yvec=333, bias=True, act="gelu", keep=True),
        # a training step's tokens, forward
        dict(gated, name="gated 4096 4096-11008", ndat=4096, xvec=4096, yvec=11008, keep=True),
        # all gradients of a training step
        dict(gated, name="gated backward 2048 1024-4096", ndat=2048, xvec=1024, yvec=4096, bias=True, backward=True),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    kind = rng.choice(["rotary", "append", "attention", "gated"])
    npiece = rng.choice([32, 64, 64, 80, 96, 128, 128])
    if kind == "rotary":
        nhead = rng.choice([1, 4, 8, 12, 32])
        ntok = _log(rng, 1, 16384 * 4096 // (nhead * npiece) // 2)
        nbat = rng.choice([1, 2, 3, 8])
        scaling = rng.choice(["none", "linear", "base", "parts"])
        return {"kind": "rotary", "nbat": nbat, "ntimes": max(1, min(ntok, 65536) // nbat), "nhead": nhead,
                "npiece": npiece, "rows_given": rng.random() < 0.7, "nrot": rng.choice([0, npiece // 2]),
                "layout": rng.choice(["halves", "pairs"]), "scaling": scaling,
                "factor": 1.0 if scaling == "none" else rng.choice([2.0, 4.0, 8.0]), "backward": rng.random() < 0.5,
                "far": rng.choice([0, 1000, 500000])}
    if kind == "append":
        nbat = _log(rng, 1, 96)
        ntimes = 1 if rng.random() < 0.4 else _log(rng, 2, 6000 // nbat + 2)
        return {"kind": "append", "nbat": nbat, "ntimes": ntimes, "nkvhead": rng.choice([1, 2, 8, 12]),
                "npiece": npiece, "maxlen": _log(rng, 1, 1000), "page": rng.choice([16, 48, 64, 100]),
                "nrot": rng.choice([0, npiece // 2]), "layout": rng.choice(["halves", "pairs"]),
                "ragged": rng.random() < 0.5}
    if kind == "attention":
        nkv = rng.choice([1, 2, 8, 12])
        group = rng.choice([1, 1, 2, 4, 8])
        ntimes = 1 if rng.random() < 0.3 else _log(rng, 2, 80)
        maxlen = _log(rng, 1, 100000)
        # no more keys and no more rows times keys than the long listed case
        nbat = max(1, min(_log(rng, 1, 32), 131072 * 8 * 128 // (maxlen * nkv * npiece),
                          131072 * 512 * 128 // (maxlen * ntimes * nkv * group * npiece)))
        while ntimes > 1 and nbat * maxlen * ntimes * nkv * group * npiece > 131072 * 512 * 128:
            ntimes = ntimes // 2
        return {"kind": "attention", "nbat": nbat, "ntimes": ntimes, "nhead": nkv * group, "nkvhead": nkv,
                "npiece": npiece, "maxlen": maxlen, "page": rng.choice([16, 48, 64, 100, 256]),
                "tree": ntimes > 1 and rng.random() < 0.7, "ragged": rng.random() < 0.6}
    ndat = _log(rng, 1, 4096)
    xvec, yvec = _log(rng, 64, 4096), _log(rng, 64, 8192)
    return {"kind": "gated", "ndat": ndat, "xvec": xvec, "yvec": yvec, "bias": rng.random() < 0.5,
            "act": rng.choice(["swish", "swish", "gelu", "sigmoid", "relu"]), "keep": rng.random() < 0.5,
            "backward": rng.random() < 0.4}


def work(case):
    if case["kind"] == "rotary":
        n = case["nbat"] * case["ntimes"] * case["nhead"]
        nrot = case["nrot"] or case["npiece"]
        return {"bytes": 2 * F4 * n * case["npiece"], "flops": 3 * n * nrot}
    if case["kind"] == "append":
        n = sum(_counts(case)) * case["nkvhead"] * case["npiece"]
        return {"bytes": 4 * F4 * n, "flops": 3 * n}
    if case["kind"] == "attention":
        lens, counts = _lengths(case), _counts(case)
        keys = sum(n + c for n, c in zip(lens, counts))
        rows_keys = sum(c * (n + (c + 1) / 2) for n, c in zip(lens, counts))
        rows = sum(counts) * case["nhead"]
        return {"bytes": F4 * case["npiece"] * (2 * keys * case["nkvhead"] + 2 * rows),
                "flops": 4 * rows_keys * case["nhead"] * case["npiece"]}
    m, k, n = case["ndat"], case["xvec"], case["yvec"]
    if case["backward"]:
        return {"bytes": F4 * (2 * m * k + 3 * m * n + 4 * k * n), "flops": 8 * m * n * k}
    return {"bytes": F4 * (m * k + 2 * n * k + (3 if case["keep"] else 1) * m * n), "flops": 4 * m * n * k}


# ---- what a user's program has in hand -------------------------------------------------------------------------

def _counts(case):
    """New tokens of each sequence: all of them, or spread between one and all."""
    b, t = case["nbat"], case["ntimes"]
    return [t if not case["ragged"] else max(1, t - (t * i * 3) // (4 * b)) for i in range(b)]


def _lengths(case):
    """Keys of each sequence that the cache holds already."""
    b, n = case["nbat"], case["maxlen"]
    return [n if not case["ragged"] else n - (n * i * 2) // (3 * b) for i in range(b)]


def _rand(gen, *shape):
    return torch.randn(*shape, device=DEV, generator=gen)


def _xavier(gen, rows, cols):
    return (torch.rand(rows, cols, device=DEV, generator=gen) * 2 - 1) * math.sqrt(1.0 / cols)


def _tree(nbat, ntimes, gen_cpu):
    """Drafted trees: a random earlier parent for each node (the first is the root); a node sees its ancestors."""
    parent = (torch.rand(nbat, ntimes, generator=gen_cpu) * torch.arange(ntimes)).floor().to(torch.int64)
    see = torch.zeros(nbat, ntimes, ntimes, dtype=torch.bool)
    rows = torch.arange(nbat)
    for t in range(ntimes):
        if t > 0:
            see[:, t] = see[rows, parent[:, t]]
        see[:, t, t] = True
    return see


def _words(see):
    """Bits of the visibility matrix, 32 to a word."""
    b, t, _ = see.shape
    nword = (t + 31) // 32
    full = torch.zeros(b, t, nword * 32, dtype=torch.int64)
    full[:, :, :t] = see.to(torch.int64)
    words = (full.view(b, t, nword, 32) << torch.arange(32)).sum(-1)
    return torch.where(words >= 2 ** 31, words - 2 ** 32, words).to(torch.int32)


def _cache(case, gen, gen_cpu, reach):
    """Pages in an order of their own, and the table that finds them."""
    page = case["page"]
    per = (reach + page - 1) // page
    npage = per * case["nbat"]
    table = torch.randperm(npage, generator=gen_cpu).view(case["nbat"], per).to(torch.int32).to(DEV)
    width = case["nkvhead"] * case["npiece"]
    return {"ck": _rand(gen, npage, page, width), "cv": _rand(gen, npage, page, width), "table": table,
            "npage": npage, "nmaxpage": per}


def prepare(case, seed):
    gen = torch.Generator(device=DEV)
    gen.manual_seed(seed)
    cpu = torch.Generator()
    cpu.manual_seed(seed)
    s = {"case": case}
    if case["kind"] == "rotary":
        b, t, width = case["nbat"], case["ntimes"], case["nhead"] * case["npiece"]
        s["x"] = _rand(gen, b, t, width)
        s["pos"] = None
        if case["rows_given"]:
            first = torch.randint(0, case["far"] + 1, (b, 1), generator=cpu)
            s["pos"] = (first + torch.arange(t)).to(torch.int32).to(DEV)
        s["y"] = torch.empty_like(s["x"])
    elif case["kind"] == "append":
        b, t, width = case["nbat"], case["ntimes"], case["nkvhead"] * case["npiece"]
        s["k"], s["v"] = _rand(gen, b, t, width), _rand(gen, b, t, width)
        s.update(_cache(case, gen, cpu, case["maxlen"] + t))
        s["len"] = torch.tensor(_lengths(case), dtype=torch.int32, device=DEV)
        s["count"] = torch.tensor(_counts(case), dtype=torch.int32, device=DEV)
    elif case["kind"] == "attention":
        b, t = case["nbat"], case["ntimes"]
        s["q"] = _rand(gen, b, t, case["nhead"] * case["npiece"])
        s.update(_cache(case, gen, cpu, case["maxlen"] + t))
        s["len"] = torch.tensor(_lengths(case), dtype=torch.int32, device=DEV)
        s["count"] = torch.tensor(_counts(case), dtype=torch.int32, device=DEV)
        s["words"] = None
        if case["tree"]:
            s["words"] = _words(_tree(b, t, cpu)).to(DEV)
        s["coef"] = torch.full((1,), 1.0 / math.sqrt(case["npiece"]), device=DEV)
        s["y"] = torch.zeros(b, t, case["nhead"] * case["npiece"], device=DEV)
    else:
        m, k, n = case["ndat"], case["xvec"], case["yvec"]
        s["x"] = _rand(gen, m, k)
        s["wg"], s["wu"] = _xavier(gen, n, k), _xavier(gen, n, k)
        s["bg"], s["bu"] = (_rand(gen, n) * 0.1, _rand(gen, n) * 0.1) if case["bias"] else (None, None)
        if case["backward"]:
            s["gate"], s["up"] = _rand(gen, m, n) * 0.6, _rand(gen, m, n) * 0.6
            s["gy"] = _rand(gen, m, n) * 0.01
    return s


# ---- one pass ----------------------------------------------------------------------------------------------------

TRAINED, LOW_TURNS, HIGH_TURNS, BASE = 8192.0, 1.0, 4.0, 10000.0


def _magnitude(case):
    return 1.0 + 0.1 * math.log(case["factor"]) if case["scaling"] == "parts" else 1.0


def run(s):
    kind = s["case"]["kind"]
    if kind == "rotary":
        return _own_rotary(s) if own else _plain_rotary(s)
    if kind == "append":
        return _own_append(s) if own else _plain_append(s)
    if kind == "attention":
        return _own_attention(s) if own else _plain_attention(s)
    if s["case"]["backward"]:
        return _own_gated_backward(s) if own else _plain_gated_backward(s)
    return _own_gated(s) if own else _plain_gated(s)


def _ptr(t):
    return None if t is None else t.data_ptr()


def _own_desc(s, nrot, layout, scaling="none", factor=1.0, magnitude=1.0):
    from deep_learning_framework_amd import kai
    if "desc" not in s:
        s["desc"] = kai.rotary_desc(nrot, layout=layout, base=BASE, scaling=scaling, factor=factor, trained=TRAINED,
                                    low_turns=LOW_TURNS, high_turns=HIGH_TURNS, magnitude=magnitude)
    return s["desc"]


def _own_rotary(s):
    from deep_learning_framework_amd import kai
    c = s["case"]
    desc = _own_desc(s, c["nrot"] or c["npiece"], c["layout"], c["scaling"], c["factor"], _magnitude(c))
    call = kai.VMath.rotary_backward if c["backward"] else kai.VMath.rotary
    call(0, _ptr(s["y"]), _ptr(s["x"]), _ptr(s["pos"]), c["nbat"], c["ntimes"], c["nhead"] * c["npiece"], c["nhead"],
         c["npiece"], desc)
    return s["y"]


def _own_append(s):
    from deep_learning_framework_amd import kai
    c = s["case"]
    desc = _own_desc(s, c["nrot"] or c["npiece"], c["layout"])
    kai.VMath.cache_append(0, _ptr(s["ck"]), _ptr(s["cv"]), _ptr(s["k"]), _ptr(s["v"]), _ptr(s["table"]),
                           _ptr(s["len"]), _ptr(s["count"]), None, c["nbat"], c["ntimes"],
                           c["nkvhead"] * c["npiece"], c["nkvhead"], c["npiece"], s["npage"], c["page"],
                           s["nmaxpage"], desc)
    return s["ck"], s["cv"]


def _own_attention(s):
    from deep_learning_framework_amd import kai
    c = s["case"]
    kai.VMath.cache_attention(0, _ptr(s["y"]), _ptr(s["q"]), _ptr(s["ck"]), _ptr(s["cv"]), _ptr(s["table"]),
                              _ptr(s["len"]), _ptr(s["count"]), _ptr(s["words"]), c["nbat"], c["ntimes"],
                              c["nhead"] * c["npiece"], c["nhead"], c["nkvhead"], c["npiece"], s["npage"], c["page"],
                              s["nmaxpage"], _ptr(s["coef"]))
    return s["y"]


def _own_gated(s):
    from deep_learning_framework_amd import kai
    c = s["case"]
    m, k, n = c["ndat"], c["xvec"], c["yvec"]
    y = torch.empty(m, n, device=DEV)
    gate, up = (torch.empty(m, n, device=DEV), torch.empty(m, n, device=DEV)) if c["keep"] else (None, None)
    kai.VMath.gated_forward(0, _ptr(y), _ptr(gate), _ptr(up), _ptr(s["wg"]), _ptr(s["wu"]), _ptr(s["bg"]),
                            _ptr(s["bu"]), _ptr(s["x"]), n, m, k, kai.ACT[c["act"]], None)
    return {"y": y, "gate": gate, "up": up}


def _own_gated_backward(s):
    from deep_learning_framework_amd import kai
    c = s["case"]
    m, k, n = c["ndat"], c["xvec"], c["yvec"]
    gx, gwg, gwu = torch.empty(m, k, device=DEV), torch.empty(n, k, device=DEV), torch.empty(n, k, device=DEV)
    gbg, gbu = (torch.empty(n, device=DEV), torch.empty(n, device=DEV)) if c["bias"] else (None, None)
    work_buffer = torch.empty(2, m, n, device=DEV)
    kai.VMath.gated_backward(0, _ptr(gx), _ptr(gwg), _ptr(gwu), _ptr(gbg), _ptr(gbu), _ptr(work_buffer), _ptr(s["gy"]),
                             _ptr(s["wg"]), _ptr(s["wu"]), _ptr(s["x"]), _ptr(s["gate"]), _ptr(s["up"]), n, m, k,
                             kai.ACT[c["act"]], None, False)
    return {"gx": gx, "gwg": gwg, "gwu": gwu, "gbg": gbg, "gbu": gbu}


# ---- the plain forms ---------------------------------------------------------------------------------------------

def _plain_frequencies(nrot, scaling, factor):
    """Radians a position, in 64 bits."""
    i = torch.arange(nrot // 2, device=DEV, dtype=torch.float64)
    base = BASE * factor ** (nrot / (nrot - 2.0)) if scaling == "base" and nrot > 2 else BASE
    f = torch.exp(i * (-2.0 / nrot * math.log(base)))
    if scaling == "linear":
        return f / factor
    if scaling == "parts":
        turns = TRAINED * f / (2 * math.pi)
        keep = ((turns - LOW_TURNS) / (HIGH_TURNS - LOW_TURNS)).clamp(0, 1)
        return f * keep + f / factor * (1 - keep)
    return f


def _plain_rotate(x, pos, nrot, layout, freq, magnitude, sign):
    """x[b, t, h, d] by the angles of pos[b, t]; sign -1 turns back, which is the gradient."""
    angle = pos.to(torch.float64)[..., None] * freq
    c, si = (magnitude * torch.cos(angle)).float(), (magnitude * torch.sin(angle) * sign).float()
    c, si = c[:, :, None], si[:, :, None]
    y = x.clone()
    if layout == "halves":
        x1, x2 = x[..., :nrot // 2], x[..., nrot // 2:nrot]
        y[..., :nrot // 2], y[..., nrot // 2:nrot] = x1 * c - x2 * si, x2 * c + x1 * si
    else:
        x1, x2 = x[..., 0:nrot:2], x[..., 1:nrot:2]
        y[..., 0:nrot:2], y[..., 1:nrot:2] = x1 * c - x2 * si, x2 * c + x1 * si
    return y


def _plain_rotary(s):
    c = s["case"]
    b, t, h, d = c["nbat"], c["ntimes"], c["nhead"], c["npiece"]
    nrot = c["nrot"] or d
    pos = s["pos"] if s["pos"] is not None else torch.arange(t, device=DEV).expand(b, t)
    freq = _plain_frequencies(nrot, c["scaling"], c["factor"])
    y = _plain_rotate(s["x"].view(b, t, h, d), pos, nrot, c["layout"], freq, _magnitude(c),
                      -1.0 if c["backward"] else 1.0)
    return y.view(b, t, h * d)


def _plain_append(s):
    c = s["case"]
    b, t, h, d = c["nbat"], c["ntimes"], c["nkvhead"], c["npiece"]
    nrot = c["nrot"] or d
    pos = s["len"].to(torch.int64)[:, None] + torch.arange(t, device=DEV)
    k = _plain_rotate(s["k"].view(b, t, h, d), pos, nrot, c["layout"], _plain_frequencies(nrot, "none", 1.0), 1.0, 1.0)
    # rows behind a sequence's count write its last row once more
    row = torch.minimum(torch.arange(t, device=DEV)[None, :], s["count"].to(torch.int64)[:, None] - 1)
    at = s["len"].to(torch.int64)[:, None] + row
    page = s["table"].to(torch.int64).gather(1, at // c["page"])
    slot = page * c["page"] + at % c["page"]
    pick = row[..., None].expand(b, t, h * d)
    s["ck"].view(-1, h * d)[slot.view(-1)] = k.view(b, t, h * d).gather(1, pick).view(-1, h * d)
    s["cv"].view(-1, h * d)[slot.view(-1)] = s["v"].gather(1, pick).view(-1, h * d)
    return s["ck"], s["cv"]


def _plain_see(s, reach):
    """[b, t, key]: whether a new token sees a key of the cache."""
    c = s["case"]
    b, t = c["nbat"], c["ntimes"]
    key = torch.arange(reach, device=DEV)[None, None, :]
    start = s["len"].to(torch.int64)[:, None, None]
    new = key - start
    if s["words"] is None:
        seen = new <= torch.arange(t, device=DEV)[None, :, None]
    else:
        at = new.clamp(0, t - 1).expand(b, t, reach)
        seen = (s["words"].to(torch.int64).gather(2, at // 32) >> (at % 32)) & 1 == 1
    return (new < 0) | (seen & (new >= 0) & (new < s["count"].to(torch.int64)[:, None, None]))


def _plain_attention(s):
    c = s["case"]
    b, t, h, kv, d = c["nbat"], c["ntimes"], c["nhead"], c["nkvhead"], c["npiece"]
    group = h // kv
    reach = c["maxlen"] + t
    at = torch.arange(reach, device=DEV)
    page = s["table"].to(torch.int64)[:, at // c["page"]]
    slot = (page * c["page"] + at % c["page"]).view(-1)
    k = s["ck"].view(-1, kv * d)[slot].view(b, reach, kv, d).permute(0, 2, 3, 1)
    v = s["cv"].view(-1, kv * d)[slot].view(b, reach, kv, d).permute(0, 2, 1, 3)
    q = s["q"].view(b, t, kv, group, d).permute(0, 2, 1, 3, 4).reshape(b, kv, t * group, d)
    score = torch.matmul(q, k.contiguous()).view(b, kv, t, group, reach) * s["coef"]
    see = _plain_see(s, reach)[:, None, :, None, :]
    score = score.masked_fill(~see, float("-inf"))
    p = torch.exp(score - score.amax(-1, keepdim=True))
    p = (p / p.sum(-1, keepdim=True)).view(b, kv, t * group, reach)
    y = torch.matmul(p, v.contiguous()).view(b, kv, t, group, d).permute(0, 2, 1, 3, 4).reshape(b, t, h * d)
    given = torch.arange(t, device=DEV)[None, :, None] < s["count"][:, None, None]
    s["y"].copy_(torch.where(given, y, s["y"]))
    return s["y"]


def _plain_act(g, act):
    if act == "swish":
        return g / (1 + torch.exp(-g))
    if act == "gelu":
        return g * 0.5 * (1 + torch.erf(g / math.sqrt(2.0)))
    if act == "sigmoid":
        return 1 / (1 + torch.exp(-g))
    return g.clamp_min(0)


def _plain_act_slope(g, act):
    if act == "gelu":
        return 0.5 * (1 + torch.erf(g / math.sqrt(2.0))) + g * torch.exp(-g * g / 2) / math.sqrt(2 * math.pi)
    if act == "relu":
        return (g > 0).to(g.dtype)
    p = 1 / (1 + torch.exp(-g))
    return p * (1 - p) if act == "sigmoid" else p + g * p * (1 - p)


def _plain_gated(s):
    c = s["case"]
    gate, up = torch.matmul(s["x"], s["wg"].t()), torch.matmul(s["x"], s["wu"].t())
    if c["bias"]:
        gate, up = gate + s["bg"], up + s["bu"]
    y = _plain_act(gate, c["act"]) * up
    return {"y": y, "gate": gate if c["keep"] else None, "up": up if c["keep"] else None}


def _plain_gated_backward(s):
    c = s["case"]
    gup = s["gy"] * _plain_act(s["gate"], c["act"])
    ggate = s["gy"] * s["up"] * _plain_act_slope(s["gate"], c["act"])
    gx = torch.matmul(ggate, s["wg"]) + torch.matmul(gup, s["wu"])
    out = {"gx": gx, "gwg": torch.matmul(ggate.t(), s["x"]), "gwu": torch.matmul(gup.t(), s["x"])}
    out["gbg"], out["gbu"] = (ggate.sum(0), gup.sum(0)) if c["bias"] else (None, None)
    return out


# ---- the definitions in 64 bits ----------------------------------------------------------------------------------

def _exact_turn(x, pos, nrot, layout, scaling, factor, magnitude, back):
    """x [tokens, heads, npiece] as complex numbers times e^(i angle), the angles from their definition."""
    half = nrot // 2
    freq = []
    for i in range(half):
        f = BASE ** (-2.0 * i / nrot)
        if scaling == "base" and nrot > 2:
            f = (BASE * factor ** (nrot / (nrot - 2.0))) ** (-2.0 * i / nrot)
        elif scaling == "linear":
            f = f / factor
        elif scaling == "parts":
            turns = TRAINED * f / (2 * math.pi)
            if turns < LOW_TURNS:
                f = f / factor
            elif turns < HIGH_TURNS:
                mix = (turns - LOW_TURNS) / (HIGH_TURNS - LOW_TURNS)
                f = (1 - mix) * f / factor + mix * f
        freq.append(f)
    angle = pos.double().view(-1, 1, 1) * torch.tensor(freq, dtype=torch.float64, device=x.device)
    turn = torch.polar(torch.full_like(angle, magnitude), -angle if back else angle)
    y = x.double().clone()
    if layout == "halves":
        z = torch.complex(y[..., :half].contiguous(), y[..., half:nrot].contiguous()) * turn
        y[..., :half], y[..., half:nrot] = z.real, z.imag
    else:
        z = torch.view_as_complex(y[..., :nrot].reshape(y.shape[0], y.shape[1], half, 2).contiguous()) * turn
        y[..., :nrot] = torch.view_as_real(z).reshape(y.shape[0], y.shape[1], nrot)
    return y


def _exact_rotary(s, c):
    b, t, h, d = c["nbat"], c["ntimes"], c["nhead"], c["npiece"]
    pos = s["pos"].view(-1) if s["pos"] is not None else torch.arange(t, device=DEV).repeat(b)
    y = _exact_turn(s["x"].view(b * t, h, d), pos, c["nrot"] or d, c["layout"], c["scaling"], c["factor"],
                    _magnitude(c), c["backward"])
    return y.view(b, t, h * d)


def _exact_append(s, c):
    h, d, page = c["nkvhead"], c["npiece"], c["page"]
    ck, cv = s["ck"].double(), s["cv"].double()
    for i, (n, count) in enumerate(zip(_lengths(c), _counts(c))):
        at = torch.arange(n, n + count, device=DEV)
        k = _exact_turn(s["k"][i, :count].view(count, h, d), at, c["nrot"] or d, c["layout"], "none", 1.0, 1.0, False)
        where = s["table"][i].long()[at // page]
        ck[where, at % page] = k.view(count, h * d)
        cv[where, at % page] = s["v"][i, :count].double()
    return ck, cv


def _exact_attention(s, c):
    h, kv, d, page = c["nhead"], c["nkvhead"], c["npiece"], c["page"]
    y = s["y"].double()
    words = None if s["words"] is None else s["words"].cpu()
    for i, (n, count) in enumerate(zip(_lengths(c), _counts(c))):
        at = torch.arange(n + count, device=DEV)
        where = s["table"][i].long()[at // page]
        k, v = (s[name][where, at % page].double().view(n + count, kv, d) for name in ("ck", "cv"))
        see = torch.ones(count, n + count, dtype=torch.bool)
        if words is None:
            see[:, n:] = torch.ones(count, count).tril().bool()
        else:
            bits = torch.arange(count)
            see[:, n:] = (words[i, :count].long()[:, bits // 32] >> (bits % 32)) % 2 == 1
        see = see.to(DEV)
        for j in range(h):
            q = s["q"][i, :count, j * d:(j + 1) * d].double()
            z = q @ k[:, j * kv // h].t().contiguous() * float(s["coef"])
            z[~see] = -math.inf
            y[i, :count, j * d:(j + 1) * d] = torch.softmax(z, 1) @ v[:, j * kv // h]
    return y


def _exact_gated(s, c):
    x, wg, wu = s["x"].double(), s["wg"].double(), s["wu"].double()
    name = {"swish": torch.nn.functional.silu, "gelu": torch.nn.functional.gelu, "sigmoid": torch.sigmoid,
            "relu": torch.relu}[c["act"]]
    if not c["backward"]:
        gate, up = x @ wg.t(), x @ wu.t()
        if c["bias"]:
            gate, up = gate + s["bg"].double(), up + s["bu"].double()
        y = name(gate) * up
        return {"y": y, "gate": gate if c["keep"] else None, "up": up if c["keep"] else None}
    gate, up = s["gate"].double().requires_grad_(), s["up"].double().requires_grad_()
    with torch.enable_grad():
        y = name(gate) * up
    ggate, gup = torch.autograd.grad(y, (gate, up), s["gy"].double())
    both = torch.cat([ggate, gup], 1)
    gw = both.t().contiguous() @ x
    n = c["yvec"]
    sums = both.sum(0)
    return {"gx": both @ torch.cat([wg, wu], 0), "gwg": gw[:n], "gwu": gw[n:], "gbg": sums[:n] if c["bias"] else None,
            "gbu": sums[n:] if c["bias"] else None}


def exact(case, seed):
    s = prepare(case, seed)
    of = {"rotary": _exact_rotary, "append": _exact_append, "attention": _exact_attention, "gated": _exact_gated}
    return of[case["kind"]](s, case)
