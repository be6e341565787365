"""Operators of a token path that gets its views one after another.

A program that follows a video keeps the K and V of earlier frames in a cache
of 8-bit codes, gives Q and K rotary positions with a time axis, and lets the
rows of a new frame (or a single row: a camera token) attend to all that is
kept.  Four operators: Q/K LayerNorm with rotary positions of several axes,
the cache's write and its read, and attention over the cache with capped
scores, a bias by distance, and causal, prefix and document masks.

Sizes are those of the depth model's views (a 504x336 image: a 24 x 36 patch
grid and two special tokens, 866 rows; twelve views: 10,392 rows; 12 or 16
heads of 64); `draw` spreads around them.

`run` computes the operators in plain torch, or calls the library where `own`
is true.  The library's handles name the same torch tensors, without a copy.
"""
import ctypes
import math
import os
import sys

import torch

own = False

HD = 64
PAIRS = HD // 2
EPS, FREQ = 1e-5, 100.0
N_SPECIAL = 2  # class token and one register
TOP = {"q8": 127.0, "f8": 448.0}


# ------------------------------------------------------------------ the cases
def listed():
    return [
        # Q and K of one new frame: latency
        dict(name="rope_frame", kind="rope", gh=24, gw=36, frames=1, time=11, heads=12, kv=12,
             convention="blocks", interleaved=False, pt=8, ph=12, norm=True, f16=False),
        # Q and K of a whole clip, frequencies over the whole head
        dict(name="rope_clip", kind="rope", gh=24, gw=36, frames=12, time=0, heads=12, kv=12,
             convention="sections", interleaved=False, pt=8, ph=12, norm=True, f16=False),
        # one new frame into a cache of twelve, and what was written read back
        dict(name="write_frame", kind="write", sequences=1, kv=12, capacity=10392, n=866, start=9526,
             step=0, cut=0, format="q8", heads_outer=True),
        # eight streams' first frames, the streams of different lengths
        dict(name="write_streams", kind="write", sequences=8, kv=16, capacity=1732, n=866, start=800,
             step=100, cut=33, format="f8", heads_outer=True),
        # one frame read back to f32
        dict(name="read_frame", kind="read", sequences=1, kv=12, capacity=10392, n=866, start=866,
             step=0, cut=0, format="f8", heads_outer=True),
        # a whole cache read back to f32
        dict(name="read_all", kind="read", sequences=1, kv=12, capacity=10392, n=10392, start=0,
             step=0, cut=0, format="q8", heads_outer=True),
        # one row over one frame: launches count
        dict(name="token_frame", kind="attend", sequences=1, heads=12, kv=12, capacity=866, n=1,
             start=865, step=0, cut=0, format="q8", cap=0.0, bias=False, mask="none", unit=866,
             heads_outer=True),
        # one row over a long history: the cache's bytes count
        dict(name="token_history", kind="attend", sequences=1, heads=16, kv=16, capacity=124704, n=1,
             start=124703, step=0, cut=0, format="f8", cap=0.0, bias=False, mask="none", unit=866,
             heads_outer=True),
        # a new frame over twelve
        dict(name="attend_frame", kind="attend", sequences=1, heads=12, kv=12, capacity=10392, n=866,
             start=9526, step=0, cut=0, format="q8", cap=0.0, bias=False, mask="none", unit=866,
             heads_outer=True),
        # causal rows after a prefix that sees itself whole, capped scores, heads that share K and
        # V, streams of different lengths
        dict(name="attend_prefix", kind="attend", sequences=3, heads=16, kv=8, capacity=2600, n=1301,
             start=1201, step=400, cut=77, format="f8", cap=30.0, bias=False, mask="prefix", unit=866,
             heads_outer=False),
        # twelve scenes packed in one sequence, each by itself, nearer rows preferred
        dict(name="attend_scenes", kind="attend", sequences=1, heads=12, kv=12, capacity=10392,
             n=10392, start=0, step=0, cut=0, format="q8", cap=0.0, bias=True, mask="documents",
             unit=866, heads_outer=True),
        # twelve frames at once, each over itself and the earlier ones
        dict(name="attend_clip", kind="attend", sequences=1, heads=12, kv=12, capacity=10392,
             n=10392, start=0, step=0, cut=0, format="q8", cap=0.0, bias=False, mask="frames",
             unit=866, heads_outer=True),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _draw(rng):
    kind = rng.choice(["rope", "rope", "write", "write", "read", "read", "token", "token", "attend",
                       "attend", "attend", "attend"])
    heads = rng.choice([12, 12, 16])
    if kind == "rope":
        pt = rng.choice([4, 8, 10, 16])
        return dict(kind=kind, gh=_log_int(rng, 3, 48), gw=_log_int(rng, 3, 72),
                    frames=_log_int(rng, 1, 12), time=_log_int(rng, 1, 100000) - 1, heads=heads,
                    kv=rng.choice([heads, heads, heads // 2]),
                    convention=rng.choice(["blocks", "sections"]),
                    interleaved=rng.random() < 0.4, pt=pt, ph=(PAIRS - pt) // 2,
                    norm=rng.random() < 0.8, f16=rng.random() < 0.4)
    c = dict(kind=kind, sequences=1 if rng.random() < 0.5 else _log_int(rng, 2, 8))
    if kind in ("write", "read"):
        c["kv"] = heads
    else:
        c.update(heads=heads, kv=heads // rng.choice([1, 1, 2, 4]))
    c["n"] = 1 if kind == "token" else _log_int(rng, 1, 10392)
    past = _log_int(rng, 1, 130000 if kind == "token" else 10392) - 1
    c.update(capacity=past + c["n"] + rng.choice([0, 0, 1, 77]), start=past,
             step=rng.randrange(past // c["sequences"] + 1),
             cut=rng.choice([0, rng.randrange(c["n"] // c["sequences"] + 1)]),
             format=rng.choice(["q8", "f8"]), heads_outer=rng.random() < 0.6)
    if kind in ("token", "attend"):
        c.update(kind="attend", cap=rng.choice([0.0, 0.0, 0.0, 20.0, 50.0]), bias=rng.random() < 0.3,
                 mask=rng.choice(["none", "none", "causal", "prefix", "documents", "frames"]),
                 unit=_log_int(rng, 38, 3458))
    return c


def draw(rng):
    most = max(_cost(c) for c in listed())
    while True:
        c = _draw(rng)
        if _cost(c) <= most and all({k: v for k, v in x.items() if k != "name"} != c
                                    for x in listed()):
            return c


# ------------------------------------------------------------------ work
def _spans(c):
    """(start, count) of each sequence."""
    return [(max(c["start"] - s * c["step"], 0), max(c["n"] - s * c["cut"], 0))
            for s in range(c["sequences"])]


def _prefix(c, s):
    """The rows of sequence s that every row of it may see."""
    return c["unit"] // (1 + s)


def _sum_to(n):
    return n * (n + 1) // 2


def _visible(c, s, start, count):
    """(pairs of a query and a key, keys that some query sees) of one sequence."""
    end, unit = start + count, c["unit"]
    if count == 0:
        return 0, 0
    if c["mask"] == "none":
        return count * end, end
    if c["mask"] in ("causal", "prefix"):
        pre = min(_prefix(c, s), end) if c["mask"] == "prefix" else 0
        low = min(max(pre - 1, start - 1), end - 1) + 1  # rows below see the prefix whole
        return (low - start) * pre + _sum_to(end) - _sum_to(low), end
    pairs = 0
    for d in range(start // unit, (end - 1) // unit + 1):
        rows = min((d + 1) * unit, end) - max(d * unit, start)
        seen = min((d + 1) * unit, end)
        pairs += rows * (seen - d * unit if c["mask"] == "documents" else seen)
    return pairs, end - (start // unit * unit if c["mask"] == "documents" else 0)


def work(case):
    c, kind = case, case["kind"]
    if kind == "rope":
        rows = c["frames"] * (N_SPECIAL + c["gh"] * c["gw"])
        values = rows * (c["heads"] + c["kv"]) * HD
        return {"bytes": 8 * values + 12 * rows, "flops": (11 if c["norm"] else 3) * values}
    rows = sum(n for _, n in _spans(c))
    held, wide = 2 * c.get("kv", 0) * (HD + 4), 2 * c.get("kv", 0) * 4 * HD
    if kind == "write":  # written, then read back
        return {"bytes": rows * 2 * (wide + held), "flops": 0}
    if kind == "read":
        return {"bytes": rows * (wide + held), "flops": 0}
    seen = [_visible(c, s, *x) for s, x in enumerate(_spans(c))]
    return {"bytes": 2 * 4 * HD * c["heads"] * rows + held * sum(k for _, k in seen),
            "flops": 4 * HD * c["heads"] * sum(p for p, _ in seen)}


def _cost(c):
    w = work(c)
    if c["kind"] == "attend":  # the plain form's scores
        return max(w["bytes"], 50 * c["sequences"] * c["heads"] * c["n"] * c["capacity"])
    return w["bytes"]


# ------------------------------------------------------------------ inputs
_RT = None


def _library():
    sys.path.insert(0, os.path.join(os.getcwd(), "vestra-engine_amd"))
    import vestra_hip as vh
    global _RT
    if _RT is None:
        _RT = vh.Runtime(0)  # one runtime serves every state, as in a program
    return vh, _RT


def _wrap(vh, rt, t):
    """A library tensor over a torch tensor's memory, which it keeps alive."""
    kind = {torch.float32: vh.VK_F32, torch.float16: vh.VK_F16, torch.uint8: vh.VK_U8,
            torch.int32: vh.VK_I32}[t.dtype]
    h = ctypes.c_void_p()
    status = vh.lib.vk_tensor_wrap(rt.handle, kind, t.data_ptr(), t.numel(), ctypes.byref(h))
    if status != vh.VK_OK:
        raise vh.VestraError(status, vh.lib.vk_last_error().decode())
    w = vh.Tensor(rt, h)
    w.torch = t
    return w


def _pairs(c):
    """Both elements, the axis and the frequency of each of the 32 pairs."""
    p = (c["pt"], c["ph"], PAIRS - c["pt"] - c["ph"])
    axis = [a for a in range(3) for _ in range(p[a])]
    if c["convention"] == "sections":
        inside, half, base = list(range(PAIRS)), [PAIRS] * PAIRS, [0] * PAIRS
    else:
        inside = [i for a in range(3) for i in range(p[a])]
        half = [p[a] for a in axis]
        base = [2 * sum(p[:a]) for a in axis]
    if c["interleaved"]:
        first = [b + 2 * i for b, i in zip(base, inside)]
        second = [f + 1 for f in first]
    else:
        first = [b + i for b, i in zip(base, inside)]
        second = [f + h for f, h in zip(first, half)]
    inv = [FREQ ** (-2.0 * i / (2 * h)) for i, h in zip(inside, half)]
    return first, second, axis, inv


def _ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def _quantised(x, fmt):
    """Codes (as bytes) and scales of rows of 64."""
    d = x.abs().amax(-1)
    d = d / torch.full_like(d, TOP[fmt])  # a quotient: by a number, torch takes its reciprocal
    y = x / torch.where(d > 0, d, 1.0)[..., None]
    if fmt == "q8":
        return torch.round(y).to(torch.int8).view(torch.uint8), d
    return y.to(torch.float8_e4m3fn).view(torch.uint8), d


def _values(codes, fmt):
    return codes.view(torch.int8 if fmt == "q8" else torch.float8_e4m3fn).float()


def _data(case, seed):
    """The inputs of a case as torch tensors."""
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    c, kind = case, case["kind"]

    def normal(*shape, scale=1.0, shift=0.0):
        return torch.randn(*shape, generator=g, device="cuda") * scale + shift

    if kind == "rope":
        n = N_SPECIAL + c["gh"] * c["gw"]
        i = torch.arange(n, device="cuda") - N_SPECIAL
        grid = torch.stack([torch.zeros_like(i), i // c["gw"] + 1, i % c["gw"] + 1], 1)
        grid[:N_SPECIAL] = 0
        pos = grid.repeat(c["frames"], 1)
        pos[:, 0] = c["time"] + torch.arange(c["frames"], device="cuda").repeat_interleave(n)
        rows = n * c["frames"]
        t = {"q": normal(c["heads"], rows, HD, scale=1.5), "k": normal(c["kv"], rows, HD, scale=1.5),
             "pos": pos.int().contiguous()}
        if c["norm"]:
            for name in ("qg", "qb", "kg", "kb"):
                p = normal(HD, scale=0.02, shift=float(name[1] == "g"))
                t[name] = p.half() if c["f16"] else p
        return t
    S, kv, n, cap = c["sequences"], c["kv"], c["n"], c["capacity"]
    spans = _spans(c)
    t = {"starts": _ints([s for s, _ in spans]), "counts": _ints([k for _, k in spans])}
    if kind == "write":
        shape = (kv, S, n, HD) if c["heads_outer"] else (S, kv, n, HD)
        t.update(k=normal(*shape, scale=1.5), v=normal(*shape))
    # what the cache holds: normalised keys, values of unit size
    for name, scale in (("k", 1.5), ("v", 1.0)):
        t[name + "_codes"], t[name + "_scale"] = _quantised(normal(S, kv, cap, HD, scale=scale),
                                                            c["format"])
    if kind == "attend":
        H = c["heads"]
        t["q"] = normal(*((H, S, n, HD) if c["heads_outer"] else (S, H, n, HD)), scale=1.5)
        if c["bias"]:
            t["slopes"] = 2.0 ** (-8.0 * torch.arange(1, H + 1, device="cuda") / H)
        if c["mask"] == "prefix":
            t["prefix"] = _ints([_prefix(c, s) for s in range(S)])
        if c["mask"] in ("documents", "frames"):
            t["q_docs"] = ((t["starts"][:, None] + torch.arange(n, device="cuda")) // c["unit"]).int()
            t["k_docs"] = (torch.arange(cap, device="cuda") // c["unit"]).int().repeat(S, 1)
    return t


def prepare(case, seed):
    c, t, kind = case, _data(case, seed), case["kind"]
    s = {"case": c, "t": t}
    if kind == "rope":
        s["pairs"] = [torch.tensor(x, device="cuda",
                                   dtype=torch.float64 if i == 3 else torch.long)
                      for i, x in enumerate(_pairs(c))]
        t["q_out"], t["k_out"] = torch.empty_like(t["q"]), torch.empty_like(t["k"])
    elif kind == "attend":
        t["out"] = torch.zeros_like(t["q"])
    else:
        S, kv, n = c["sequences"], c["kv"], c["n"]
        shape = (kv, S, n, HD) if c["heads_outer"] else (S, kv, n, HD)
        t["k_out"], t["v_out"] = (torch.zeros(*shape, device="cuda") for _ in "kv")
    if own:  # a program holds its tensors and its cache as the library's handles
        vh, rt = _library()
        s["rt"] = rt
        h = s["h"] = {name: _wrap(vh, rt, x) for name, x in t.items()}
        if kind == "rope":
            s["axes"] = vh.RopeAxes((c["pt"], c["ph"], PAIRS - c["pt"] - c["ph"]), FREQ,
                                    sections=c["convention"] == "sections",
                                    interleaved=c["interleaved"])
        else:
            s["layout"] = vh.VK_QK_HEADS_OUTER if c["heads_outer"] else vh.VK_QK_VIEWS_OUTER
            s["cache"] = vh.KvCache(vh.VK_CACHE_Q8 if c["format"] == "q8" else vh.VK_CACHE_F8,
                                    c["sequences"], c["kv"], c["capacity"], h["k_codes"],
                                    h["v_codes"], h["k_scale"], h["v_scale"])
        if kind == "attend":
            s["rules"] = vh.AttentionRules(cap=c["cap"], slopes=h.get("slopes"),
                                           causal=c["mask"] in ("causal", "prefix"),
                                           prefix=h.get("prefix"), q_docs=h.get("q_docs"),
                                           k_docs=h.get("k_docs"),
                                           docs_ordered=c["mask"] == "frames")
    torch.cuda.synchronize()  # the library's stream is its own
    return s


# ------------------------------------------------------------------ one pass
def _plain_norm(x, g, b):
    m = x.mean(-1, keepdim=True)
    var = ((x - m) ** 2).mean(-1, keepdim=True)
    return (x - m) / torch.sqrt(var + EPS) * g.float() + b.float()


def _plain_rotate(x, pairs, cos, sin):
    first, second = pairs
    a, b = x[..., first], x[..., second]
    out = torch.empty_like(x)
    out[..., first] = a * cos - b * sin
    out[..., second] = b * cos + a * sin
    return out


def _plain_rope(s):
    t = s["t"]
    first, second, axis, inv = s["pairs"]
    angle = t["pos"].double()[:, axis] * inv  # far positions: angles in 64 bits
    cos, sin = torch.cos(angle).float(), torch.sin(angle).float()
    q, k = t["q"], t["k"]
    if s["case"]["norm"]:
        q, k = _plain_norm(q, t["qg"], t["qb"]), _plain_norm(k, t["kg"], t["kb"])
    return {"q": _plain_rotate(q, (first, second), cos, sin),
            "k": _plain_rotate(k, (first, second), cos, sin)}


def _slots(t, n, cap):
    """The cache slot of every row [sequences, n], and which rows count."""
    i = torch.arange(n, device="cuda")
    slot = t["starts"][:, None] + i
    return slot.clamp(max=cap - 1).long(), (i < t["counts"][:, None]) & (slot < cap)


def _by_sequence(x, c):
    return x.transpose(0, 1) if c["heads_outer"] else x


def _plain_read(s):
    c, t = s["case"], s["t"]
    slot, valid = _slots(t, c["n"], c["capacity"])
    index = slot[:, None, :].expand(-1, c["kv"], -1)

    def values(name):
        codes = torch.gather(t[name + "_codes"], 2, index[..., None].expand(-1, -1, -1, HD))
        x = _values(codes, c["format"]) * torch.gather(t[name + "_scale"], 2, index)[..., None]
        out = t[name + "_out"]
        return torch.where(valid[:, None, :, None], x, _by_sequence(out, c))

    return {name: _by_sequence(values(name), c).contiguous() for name in "kv"}


def _plain_write(s):
    c, t = s["case"], s["t"]
    slot, valid = _slots(t, c["n"], c["capacity"])
    seq = torch.arange(c["sequences"], device="cuda")[:, None].expand_as(slot)[valid]
    at = slot[valid]

    def write(name):
        codes, d = _quantised(_by_sequence(t[name], c).transpose(1, 2)[valid], c["format"])
        t[name + "_codes"][seq, :, at] = codes
        t[name + "_scale"][seq, :, at] = d

    write("k")
    write("v")
    return dict(_plain_read(s), k_scale=t["k_scale"], v_scale=t["v_scale"])


def _plain_attend(s):
    c, t = s["case"], s["t"]
    S, H, kv, n, cap = c["sequences"], c["heads"], c["kv"], c["n"], c["capacity"]
    q = _by_sequence(t["q"], c).reshape(S, kv, H // kv * n, HD)
    k = _values(t["k_codes"], c["format"]) * t["k_scale"][..., None]
    v = _values(t["v_codes"], c["format"]) * t["v_scale"][..., None]
    u = torch.matmul(q * HD ** -0.5, k.transpose(2, 3).contiguous()).reshape(S, H, n, cap)
    if c["cap"]:
        u = c["cap"] * torch.tanh(u / c["cap"])
    j = torch.arange(cap, device="cuda")
    pos = (t["starts"][:, None] + torch.arange(n, device="cuda"))[:, :, None]
    if c["bias"]:
        u = u - t["slopes"][:, None, None] * (pos - j).abs().float()[:, None]
    seen = (j < (t["starts"] + t["counts"])[:, None, None]).expand(S, n, cap)
    if c["mask"] == "causal":
        seen = seen & (j <= pos)
    elif c["mask"] == "prefix":
        seen = seen & ((j <= pos) | (j < t["prefix"][:, None, None]))
    elif c["mask"] == "documents":
        seen = seen & (t["q_docs"][:, :, None] == t["k_docs"][:, None, :])
    elif c["mask"] == "frames":
        seen = seen & (t["q_docs"][:, :, None] >= t["k_docs"][:, None, :])
    seen = seen[:, None]
    u = u.masked_fill(~seen, -math.inf)
    top = u.amax(-1, keepdim=True)
    p = torch.exp(u - torch.where(top > -math.inf, top, 0.0))
    total = p.sum(-1, keepdim=True)
    p = p / torch.where(total > 0, total, 1.0)
    o = torch.matmul(p.reshape(S, kv, H // kv * n, cap), v).reshape(S, H, n, HD)
    valid = torch.arange(n, device="cuda") < t["counts"][:, None]
    o = torch.where(valid[:, None, :, None], o, 0.0)
    return _by_sequence(o, c).contiguous()


def run(s):
    c, kind = s["case"], s["case"]["kind"]
    if not own:
        return {"rope": _plain_rope, "write": _plain_write, "read": _plain_read,
                "attend": _plain_attend}[kind](s)
    t, h, rt = s["t"], s["h"], s["rt"]
    if kind == "rope":
        rows = c["frames"] * (N_SPECIAL + c["gh"] * c["gw"])
        rt.qk_norm_rope_axes_f32(h["q"], h["k"], h.get("qg"), h.get("qb"), h.get("kg"), h.get("kb"),
                                 h["pos"], c["heads"], c["kv"], rows, s["axes"], EPS, h["q_out"],
                                 h["k_out"])
        return {"q": t["q_out"], "k": t["k_out"]}
    if kind == "attend":
        # the longest sequence's rows: what the program knows of the lengths on the host
        rt.attention_cached_f32(s["cache"], h["q"], c["heads"], c["n"], h["starts"], h["counts"],
                                c["start"] + c["n"], s["rules"], h["out"], s["layout"])
        return t["out"]
    if kind == "write":
        rt.kv_cache_write_f32(s["cache"], h["k"], h["v"], c["n"], h["starts"], h["counts"],
                              s["layout"])
    rt.kv_cache_read_f32(s["cache"], c["n"], h["starts"], h["counts"], h["k_out"], h["v_out"],
                         s["layout"])
    got = {"k": t["k_out"], "v": t["v_out"]}
    return dict(got, k_scale=t["k_scale"], v_scale=t["v_scale"]) if kind == "write" else got


# ------------------------------------------------------------------ in 64 bits
def _exact_rope(c, t):
    first, second, axis, inv = _pairs(c)
    out = {}
    for name in "qk":
        x = t[name].double()
        if c["norm"]:
            mean = x.sum(-1, keepdim=True) / HD
            var = (x * x).sum(-1, keepdim=True) / HD - mean * mean
            x = (x - mean) * torch.rsqrt(var + EPS)
            x = x * t[name + "g"].double() + t[name + "b"].double()
        y = torch.empty_like(x)
        for f, e, a, w in zip(first, second, axis, inv):
            turn = torch.polar(torch.ones_like(t["pos"][:, a], dtype=torch.float64),
                               t["pos"][:, a].double() * w)
            z = torch.complex(x[..., f], x[..., e]) * turn
            y[..., f], y[..., e] = z.real, z.imag
        out[name] = y
    return out


def _exact_codes(x, fmt):
    """Scales and held values: the scale is rounded to 32 bits, the quotient
    to 32 bits and then to the code, as the operator defines them."""
    d = (x.double().abs().amax(-1) / TOP[fmt]).float().double()
    y = (x.double() / torch.where(d > 0, d, 1.0)[..., None]).float()
    y = torch.round(y) if fmt == "q8" else y.to(torch.float8_e4m3fn)
    return d, y.double() * d[..., None]


def _exact_cache(c, t):
    S, n = c["sequences"], c["n"]
    out = {}
    for name in "kv":
        held = _values(t[name + "_codes"], c["format"]).double()
        scale = t[name + "_scale"].double()
        values = held * scale[..., None]
        if c["kind"] == "write":
            d, x = _exact_codes(_by_sequence(t[name], c), c["format"])
        back = torch.zeros(S, c["kv"], n, HD, dtype=torch.float64, device="cuda")
        for s, (start, count) in enumerate(_spans(c)):
            rows = min(count, c["capacity"] - start)
            if c["kind"] == "write":
                scale[s, :, start:start + rows] = d[s, :, :rows]
                values[s, :, start:start + rows] = x[s, :, :rows]
            back[s, :, :rows] = values[s, :, start:start + rows]
        out[name] = _by_sequence(back, c).contiguous()
        if c["kind"] == "write":
            out[name + "_scale"] = scale
    return out


def _exact_attend(c, t):
    q = _by_sequence(t["q"], c)
    out = torch.zeros(q.shape, dtype=torch.float64, device="cuda")
    step = max(1, int(2e8 // c["capacity"]))
    for s, (start, count) in enumerate(_spans(c)):
        end = min(start + count, c["capacity"])
        j = torch.arange(end, device="cuda")
        for h in range(c["heads"]):
            kh = h * c["kv"] // c["heads"]
            k, v = (_values(t[m + "_codes"][s, kh, :end], c["format"]).double()
                    * t[m + "_scale"][s, kh, :end].double()[:, None] for m in "kv")
            for i in range(0, count, step):
                p = start + torch.arange(i, min(i + step, count), device="cuda")[:, None]
                u = q[s, h, i:i + step][:p.shape[0]].double() @ k.T.contiguous() / 8.0
                if c["cap"]:
                    u = c["cap"] * torch.tanh(u / c["cap"])
                if c["bias"]:
                    u = u - t["slopes"][h].double() * (p - j).abs()
                hidden = {"none": j < 0, "causal": j > p,
                          "prefix": (j > p) & (j >= _prefix(c, s)),
                          "documents": j // c["unit"] != p // c["unit"],
                          "frames": j // c["unit"] > p // c["unit"]}[c["mask"]]
                w = torch.softmax(u.masked_fill(hidden, -math.inf), -1)
                out[s, h, i:i + p.shape[0]] = w @ v
    return _by_sequence(out, c).contiguous()


def exact(case, seed):
    t = _data(case, seed)
    if case["kind"] == "rope":
        return _exact_rope(case, t)
    return (_exact_attend if case["kind"] == "attend" else _exact_cache)(case, t)
