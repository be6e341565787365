"""Operators of a token path's feed-forward in fewer bits.

A program that serves the block in 8 bits holds a linear's weights as int8
codes with a scale for each output channel, quantises each token's row as it
comes and multiplies in integers; the result takes the epilogues of the F32
linear (GELU, LayerScale + residual) or is gated: the columns are a gate and
its partner, and act(gate) * partner is what leaves.  A program that trains
the gated feed-forward does so in 16 bits, forward and backward.

Sizes are those of the depth model's views (a 504x336 image: 866 rows; twelve
views: 10,392 rows), of its widths (384, 768, 1024, and 1536 of its larger
sibling) and of gated hidden layers two thirds of the plain ones; `draw`
spreads around them, odd ones among them.

`run` computes the operators in plain torch, or calls the library where `own`
is true.  The library's handles name the same torch tensors, without a copy.
"""
import ctypes
import math
import os
import sys

import torch

own = False

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


# ------------------------------------------------------------------ the cases
def listed():
    return [
        # one token's hidden layer in 8 bits: latency
        dict(name="i8_token", kind="i8", rows=1, width=1024, out=4096, end="gelu", act="", x="f32",
             y="f32", bias=True),
        # one image's rows back to the residual stream, with LayerScale
        dict(name="i8_image_residual", kind="i8", rows=866, width=4096, out=1024, end="residual",
             act="", x="f32", y="f32", bias=True),
        # a clip's Q, K and V, activations kept in 16 bits
        dict(name="i8_clip", kind="i8", rows=10392, width=768, out=2304, end="store", act="",
             x="bf16", y="bf16", bias=True),
        # sizes that no tile divides
        dict(name="i8_ragged", kind="i8", rows=1301, width=770, out=1999, end="store", act="",
             x="f16", y="f32", bias=False),
        # one token's gated layer in 8 bits
        dict(name="i8_gated_token", kind="i8", rows=1, width=1536, out=2 * 4096, end="gated",
             act="silu", x="f32", y="f32", bias=True),
        # a clip's gated layer, from the F32 stream to what the next product quantises
        dict(name="i8_gated_clip", kind="i8", rows=10392, width=1536, out=2 * 4096, end="gated",
             act="silu", x="f32", y="bf16", bias=True),
        # a handful of tokens in 16 bits
        dict(name="gated_tokens", kind="gated", rows=5, width=1024, hidden=2736, act="silu",
             t="bf16", bias=True),
        # one image
        dict(name="gated_image", kind="gated", rows=866, width=1024, hidden=2736, act="silu",
             t="f16", bias=True),
        # a clip, the larger width
        dict(name="gated_clip", kind="gated", rows=10392, width=1536, hidden=4096, act="gelu",
             t="bf16", bias=False),
        # a training step on a few rows of a small model, odd hidden layer
        dict(name="train_small", kind="train", rows=257, width=384, hidden=1023, act="silu",
             t="bf16", bias=True),
        # one image
        dict(name="train_image", kind="train", rows=866, width=768, hidden=2048, act="gelu",
             t="bf16", bias=True),
        # a clip, the larger width
        dict(name="train_clip", kind="train", rows=10392, width=1536, hidden=4096, act="silu",
             t="bf16", bias=True),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _size(rng, lo, hi):
    n = _log_int(rng, lo, hi)
    return rng.choice([n, n, max(8, n // 8 * 8), max(64, n // 64 * 64)])


def _draw(rng):
    kind = rng.choice(["i8", "i8", "i8 gated", "i8 gated", "gated", "gated", "train", "train"])
    rows = rng.choice([1, _log_int(rng, 2, 64)]) if rng.random() < 0.25 else _log_int(rng, 1, 10392)
    c = dict(kind=kind.split()[0], rows=rows, width=_size(rng, 64, 4096),
             act=rng.choice(["silu", "silu", "gelu"]), bias=rng.random() < 0.7)
    if kind == "i8":
        c.update(out=_size(rng, 64, 8192), end=rng.choice(["store", "gelu", "residual"]), act="",
                 x=rng.choice(["f32", "f32", "f16", "bf16"]))
        c["y"] = "f32" if c["end"] == "residual" else rng.choice(["f32", "f32", "f16", "bf16"])
    elif kind == "i8 gated":
        c.update(out=2 * _size(rng, 64, 4096), end="gated", x=rng.choice(["f32", "f32", "f16", "bf16"]),
                 y=rng.choice(["f32", "f16", "bf16"]))
    else:
        c.update(hidden=_size(rng, 64, 4096),
                 t=rng.choice(["bf16", "bf16", "f16"]) if kind == "gated" else "bf16")
    return c


def draw(rng):
    most = max(work(c)["flops"] for c in listed())
    while True:
        c = _draw(rng)
        if work(c)["flops"] <= most and all({k: v for k, v in x.items() if k != "name"} != c
                                            for x in listed()):
            return c


# ------------------------------------------------------------------ work
def work(case):
    c = case
    m, k = c["rows"], c["width"]
    if c["kind"] == "i8":
        n = c["out"]
        size = {"f32": 4, "f16": 2, "bf16": 2}
        wide = m * (n // 2 if c["end"] == "gated" else n) * size[c["y"]]
        wide *= 2 if c["end"] == "residual" else 1
        return {"bytes": m * k * size[c["x"]] + n * k + 8 * n + wide, "flops": 2 * m * n * k}
    h = c["hidden"]
    weights = 2 * h * k * 2 + (4 * h if c["bias"] else 0)
    forward = m * k * 2 + weights + m * h * 2
    product = 4 * m * h * k
    if c["kind"] == "gated":
        return {"bytes": forward, "flops": product}
    return {"bytes": forward + m * h * 2 + m * k * 2 + weights, "flops": 3 * product}


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
    kind = {torch.float32: vh.VK_F32, torch.float16: vh.VK_F16, torch.bfloat16: vh.VK_BF16}[t.dtype]
    h = ctypes.c_void_p()
    status = vh.lib.vk_tensor_wrap(rt.handle, kind, t.data_ptr(), t.numel(), ctypes.byref(h))
    if status != vh.VK_OK:
        raise vh.VestraError(status, vh.lib.vk_last_error().decode())
    w = vh.Tensor(rt, h)
    w.torch = t
    return w


def _data(case, seed):
    """The inputs of a case as torch tensors."""
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    c = case
    m, k = c["rows"], c["width"]

    def normal(*shape, scale=1.0):
        return torch.randn(*shape, generator=g, device="cuda") * scale

    # layer-normalised rows: unit size, a few channels much larger
    x = normal(m, k) * (1.0 + 7.0 * (torch.rand(k, generator=g, device="cuda") < 0.01))
    if c["kind"] == "i8":
        n = c["out"]
        w = normal(n, k, scale=k ** -0.5)
        scale = w.abs().amax(1)
        scale = scale / torch.full_like(scale, 127.0)
        t = {"x": x.to(TYPES[c["x"]]), "scale": scale,
             "codes": torch.round(w / scale[:, None]).to(torch.int8)}
        if c["bias"]:
            t["bias"] = normal(n, scale=0.1)
        if c["end"] == "residual":
            t["ls"] = normal(n, scale=0.1)
            t["y"] = normal(m, n)
        return t
    kind, h = TYPES[c["t"]], c["hidden"]
    t = {"x": x.to(kind), "w": normal(2 * h, k, scale=1.5 * k ** -0.5).to(kind)}
    if c["bias"]:
        t["bias"] = normal(2 * h, scale=0.1).to(kind)
    if c["kind"] == "train":
        t["grad"] = normal(m, h, scale=0.01).to(kind)
    return t


def prepare(case, seed):
    c, t = case, _data(case, seed)
    s = {"case": c, "t": t}
    m, k = c["rows"], c["width"]
    if c["kind"] == "i8":
        if c["end"] != "residual":
            n = c["out"] // 2 if c["end"] == "gated" else c["out"]
            t["y"] = torch.empty(m, n, device="cuda", dtype=TYPES[c["y"]])
    else:
        t["h"] = torch.empty(m, c["hidden"], device="cuda", dtype=TYPES[c["t"]])
        if c["kind"] == "train":
            t["dx"], t["dw"] = torch.empty_like(t["x"]), torch.empty_like(t["w"])
            if c["bias"]:
                t["db"] = torch.empty_like(t["bias"])
    if own:  # a program holds its weights laid out and its tensors as the library's handles
        vh, rt = _library()
        s["rt"] = rt
        s["act"] = {"": 0, "silu": vh.VK_GATE_SILU, "gelu": vh.VK_GATE_GELU}[c["act"]]
        if c["kind"] == "i8":
            host = {n: t[n].cpu().numpy() for n in ("codes", "scale", "bias", "ls") if n in t}
            s["linear"] = rt.prepare_linear_i8(k, c["out"], host["codes"], host["scale"],
                                               host.get("bias"), host.get("ls"))
        s["h"] = {n: _wrap(vh, rt, v) for n, v in t.items()
                  if n not in ("codes", "scale", "ls") and not (c["kind"] == "i8" and n == "bias")}
    torch.cuda.synchronize()  # the library's stream is its own
    return s


# ------------------------------------------------------------------ one pass
def _plain_act(g, act):
    if act == "silu":
        return g / (1.0 + torch.exp(-g))
    return 0.5 * g * (1.0 + torch.erf(g * 2 ** -0.5))


def _plain_slope(g, act):
    if act == "silu":
        s = 1.0 / (1.0 + torch.exp(-g))
        return s * (1.0 + g * (1.0 - s))
    return 0.5 * (1.0 + torch.erf(g * 2 ** -0.5)) + g * torch.exp(-0.5 * g * g) * (2 * math.pi) ** -0.5


def _plain_i8(s):
    c, t = s["case"], s["t"]
    x = t["x"].float()
    d = x.abs().amax(1)
    d = d / torch.full_like(d, 127.0)  # a quotient: by a number, torch takes its reciprocal
    codes = torch.round(x / torch.where(d > 0, d, 1.0)[:, None])
    y = torch.matmul(codes, t["codes"].float().T) * d[:, None] * t["scale"]
    if c["bias"]:
        y = y + t["bias"]
    if c["end"] == "gelu":
        y = _plain_act(y, "gelu")
    elif c["end"] == "residual":
        t["y"] += y * t["ls"]
        return t["y"]
    elif c["end"] == "gated":
        h = c["out"] // 2
        y = _plain_act(y[:, :h], c["act"]) * y[:, h:]
    return y.to(TYPES[c["y"]])


def _plain_gated(s):
    c, t = s["case"], s["t"]
    h = c["hidden"]
    x, w = t["x"].float(), t["w"].float()
    y = torch.matmul(x, w.T)
    if c["bias"]:
        y = y + t["bias"].float()
    g, u = y[:, :h], y[:, h:]
    a = _plain_act(g, c["act"])
    out = {"h": (a * u).to(TYPES[c["t"]])}
    if c["kind"] == "train":
        grad = t["grad"].float()
        d = torch.cat([grad * u * _plain_slope(g, c["act"]), grad * a], 1)
        out["dx"] = torch.matmul(d, w).to(TYPES[c["t"]])
        out["dw"] = torch.matmul(d.T, x).to(TYPES[c["t"]])
        if c["bias"]:
            out["db"] = d.sum(0).to(TYPES[c["t"]])
    return out


def run(s):
    c = s["case"]
    if not own:
        return (_plain_i8 if c["kind"] == "i8" else _plain_gated)(s)
    t, h, rt = s["t"], s["h"], s["rt"]
    m, k = c["rows"], c["width"]
    if c["kind"] == "i8":
        lin = s["linear"]
        if c["end"] == "gelu":
            lin.run_gelu(h["x"], m, h["y"])
        elif c["end"] == "residual":
            lin.run_residual(h["x"], m, h["y"])
        elif c["end"] == "gated":
            lin.run_gated(h["x"], m, h["y"], s["act"])
        else:
            lin.run_into(h["x"], m, h["y"])
        return t["y"]
    n = c["hidden"]
    rt.gated_forward(h["x"], h["w"], h.get("bias"), m, k, n, h["h"], s["act"])
    if c["kind"] == "train":
        rt.gated_backward(h["x"], h["w"], h.get("bias"), h["grad"], m, k, n, h["dx"], h["dw"],
                          h.get("db"), s["act"])
    return {name: t[name] for name in ("h", "dx", "dw", "db") if name in t}


# ------------------------------------------------------------------ in 64 bits
def _phi(g):
    return 0.5 * torch.special.erfc(-g / math.sqrt(2.0))


def _exact_act(g, act):
    """The activation and its derivative."""
    if act == "silu":
        p = torch.sigmoid(g)
        return g * p, p + g * p * (1 - p)
    return g * _phi(g), _phi(g) + g * torch.exp(-g * g / 2) / math.sqrt(2 * math.pi)


def _exact_i8(c, t):
    """The scale is rounded to 32 bits, the quotient to 32 bits and then to
    the code, as the operator defines them."""
    x = t["x"].double()
    d = (x.abs().amax(1, keepdim=True) / 127.0).float().double()
    codes = torch.round((x / torch.where(d > 0, d, 1.0)).float()).double()
    y = (codes * d) @ (t["codes"].double() * t["scale"].double()[:, None]).T.contiguous()
    if c["bias"]:
        y = y + t["bias"].double()
    if c["end"] == "gelu":
        return _exact_act(y, "gelu")[0]
    if c["end"] == "residual":
        return t["y"].double() + t["ls"].double() * y
    if c["end"] == "gated":
        g, u = y.split(c["out"] // 2, 1)
        return _exact_act(g, c["act"])[0] * u
    return y


def exact(case, seed):
    c, t = case, _data(case, seed)
    if c["kind"] == "i8":
        return _exact_i8(c, t)
    x, w = t["x"].double(), t["w"].double()
    n = c["hidden"]
    b = t["bias"].double() if c["bias"] else torch.zeros(2 * n, dtype=torch.float64, device="cuda")
    g, u = (x @ w[i:i + n].T.contiguous() + b[i:i + n] for i in (0, n))
    a, slope = _exact_act(g, c["act"])
    out = {"h": a * u}
    if c["kind"] == "train":
        grad = t["grad"].double()
        dg, du = grad * u * slope, grad * a
        out["dx"] = dg @ w[:n] + du @ w[n:]
        out["dw"] = torch.cat([dg.T.contiguous() @ x, du.T.contiguous() @ x])
        if c["bias"]:
            out["db"] = torch.cat([dg.sum(0), du.sum(0)])
    return out
