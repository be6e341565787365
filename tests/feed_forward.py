"""Plain 64-bit forms of the feed-forward in fewer bits, with the error that the
kernels' arithmetic may add, derived step by step: every f32 step is off by at most
2^-24 of its result, a sum of K products held in f32 by K 2^-23 of the sum of their
sizes (the matrix cores may cut where they could round)."""
import math

import numpy as np

import vestra_hip as vh

U = 2.0 ** -24
HALF = {"f32": U, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}  # half a step, of the value
LEAST = {"f32": 2.0 ** -149, "f16": 2.0 ** -25, "bf16": 2.0 ** -134}  # and below the normals
DTYPE = {"f32": vh.VK_F32, "f16": vh.VK_F16, "bf16": vh.VK_BF16}


def erf(x):
    return np.vectorize(math.erf, otypes=[np.float64])(x)


def rounded(x, t):
    """x as the type holds it, in f32."""
    x = np.asarray(x, np.float32)
    if t == "f16":
        return x.astype(np.float16).astype(np.float32)
    if t == "bf16":
        b = x.view(np.uint32)
        r = ((b + (0x7fff + ((b >> 16) & 1))) >> 16) << 16
        return np.where(np.isnan(x), x, r.view(np.float32))
    return x


def upload(rt, x, t):
    return {"f32": rt.upload_f32, "f16": rt.upload_f16, "bf16": rt.upload_bf16}[t](x)


def download(rt, t):
    return t.numpy() if t.dtype == vh.VK_F32 else rt.download_16(t)


def activation(g, act):
    """act(g), its derivative, and how far the kernel's act may be off."""
    if act == vh.VK_GATE_SILU:
        s = 1 / (1 + np.exp(-np.clip(g, -700, 700)))
        # e^-g: its exponent in base 2 is off by 2^-23 of itself; v_exp, the sum, v_rcp, the product
        return g * s, s * (1 + g * (1 - s)), np.abs(g * s) * (8 + 2 * np.abs(g)) * U
    p = 0.5 * (1 + erf(g / math.sqrt(2)))
    # erff within 2 ulp of 1, its argument within 2^-23, half of g
    return g * p, p + g * np.exp(-g * g / 2) / math.sqrt(2 * math.pi), np.abs(g) * 8 * U


def quantised(x):
    """Codes and scales of rows, in the f32 steps that define them."""
    x = np.asarray(x, np.float32)
    with np.errstate(invalid="ignore", over="ignore", divide="ignore"):
        top = np.max(np.abs(x), axis=1, initial=0)
        d = top / np.float32(127)
        odd = ~np.isfinite(x).all(axis=1)
        none = odd | (d < np.float32(2.0 ** -100))
        codes = np.rint(x / np.where(none, np.float32(1), d)[:, None])
    codes[none] = 0
    return codes, np.where(odd, np.float32(np.nan), np.where(none, np.float32(0), d))


def linear(x, w, t, bias, gamma):
    """(y, tolerance) of the 8-bit linear: codes w [out, in], scales t."""
    c, s = quantised(x)
    p = (c.astype(np.float64) @ w.astype(np.float64).T) * t.astype(np.float64) * \
        s.astype(np.float64)[:, None]
    y = p + (0 if bias is None else bias.astype(np.float64))
    tol = 3.01 * U * np.abs(p) + (0 if bias is None else 1.01 * U * np.abs(y))
    if gamma is not None:
        g = gamma.astype(np.float64)
        y, tol = y * g, tol * np.abs(g) + 1.01 * U * np.abs(y * g)
    return y, tol + 2.0 ** -140


def gelu_tolerance(y, tol):
    """GELU by Abramowitz & Stegun 7.1.26: the kernel's is within 3.7e-7 of the exact one."""
    return 1.13 * tol + 3.7e-7 + 2 * U * np.abs(y)


def gated(g, u, tg, tu, act):
    """(act(g) u, tolerance) from g and u that may be off by tg and tu; act' <= 1.13."""
    a, _, ta = activation(g, act)
    ta = ta + 1.13 * tg
    return a * u, ta * np.abs(u) + np.abs(a) * tu + ta * tu + 1.01 * U * np.abs(a * u)


def held(y, tol, t):
    """The tolerance of y once it is rounded to the type."""
    return tol + HALF[t] * (np.abs(y) + tol) + LEAST[t] if t != "f32" else tol


def products(x, w, bias):
    """x w^T + bias and its tolerance."""
    k = x.shape[1]
    y = x @ w.T
    tol = k * 2 * U * (np.abs(x) @ np.abs(w).T)
    if bias is not None:
        y = y + bias
        tol = tol + U * (np.abs(y) + tol)
    return y, tol


def forward(x, w, bias, act, t):
    x, w = x.astype(np.float64), w.astype(np.float64)
    n = w.shape[0] // 2
    y, tol = products(x, w, None if bias is None else bias.astype(np.float64))
    h, th = gated(y[:, :n], y[:, n:], tol[:, :n], tol[:, n:], act)
    return h, held(h, th, t)


def backward(x, w, bias, grad, act, t):
    """{name: (gradient, tolerance)}."""
    x, w, dh = (v.astype(np.float64) for v in (x, w, grad))
    n = w.shape[0] // 2
    y, tol = products(x, w, None if bias is None else bias.astype(np.float64))
    g, u, tg, tu = y[:, :n], y[:, n:], tol[:, :n], tol[:, n:]
    a, slope, ta = activation(g, act)
    # act'' <= 1.13 / sqrt 2 < 0.8; act' itself takes a few f32 steps more than act
    ts = 0.8 * tg + (np.abs(g) + 2) * 12 * U
    d = np.concatenate([dh * u * slope, dh * a], 1)
    td = np.concatenate([np.abs(dh) * (tu * np.abs(slope) + np.abs(u) * ts + tu * ts),
                         np.abs(dh) * (ta + 1.13 * tg)], 1) + 3 * U * np.abs(d)
    th = held(d, td, t)  # as operands of the products
    rows = x.shape[0]
    out = {"dx": (d @ w, th @ np.abs(w) + 2 * n * 2 * U * (np.abs(d) @ np.abs(w))),
           "dw": (d.T @ x, th.T @ np.abs(x) + rows * 2 * U * (np.abs(d).T @ np.abs(x))),
           "dbias": (d.sum(0), td.sum(0) + rows * U * np.abs(d).sum(0))}
    return {k: (v, held(v, e, t)) for k, (v, e) in out.items()}


def slope(f, step=2.0 ** -7):
    """f'(0) of f(s) by differences of the fourth order, and a bound on their error: halving the
    step takes it to a sixteenth, so that what the two differ by is above it; and f's own
    rounding, 2^-50 of its size, over the step."""
    def difference(e):
        return (8 * (f(e) - f(-e)) - (f(2 * e) - f(-2 * e))) / (12 * e)
    a, b = difference(step), difference(step / 2)
    return b, abs(a - b) + abs(f(0.0)) * 2.0 ** -40


def assert_within(got, want, tol, label):
    got = np.asarray(got, np.float64).reshape(want.shape)
    odd = np.isnan(want)
    assert np.array_equal(np.isnan(got), odd), (label, "NaN where the plain form has none, or none")
    off = np.abs(got - want) - tol
    off[odd] = 0
    if off.size and off.max() > 0:
        at = np.unravel_index(int(np.argmax(off)), want.shape)
        raise AssertionError(f"{label}: at {at} got {got[at]!r}, want {want[at]!r} "
                             f"+- {tol[at]:.3e}")
