"""act(g) and act'(g) of the gated feed-forward alone: products that are exact (one term each), so
that what is left of a tolerance is the activation's own f32 steps and the result's rounding,
both relative: gates far out keep their value."""
import math

import numpy as np
import pytest

import feed_forward as ff
import vestra_hip as vh

pytestmark = pytest.mark.gpu
ACTS = [vh.VK_GATE_SILU, vh.VK_GATE_GELU]


def phi(g):
    return 0.5 * np.vectorize(math.erfc, otypes=[np.float64])(-g / math.sqrt(2))


def act_of(g, act):
    """(act(g), its tolerance, act'(g), its tolerance), in 64 bits.

    GELU: Phi's tail is off by 1.4 u of its fit, 9 u of t (its fma 1 u and v_rcp_f32 2 u, times
    2.7, by which t P(t) moves), 3 u of the Horner steps, 4 u of v_exp_f32 and two products: 17.4 u,
    and the exponent a^2 / 2 log2(e) by three roundings, 1.25 a^2 u of the power: (19 + 1.3 a^2) u
    of itself together; 1 - tail that much of the tail and 1 u.  The slope adds g phi(g): the same
    power and 5 u, and the sum's rounding.
    SiLU: the exponent by two roundings, 2 |g| u of e^-g and so, at most, of s; v_exp_f32, the sum,
    v_rcp_f32, the product: 8 u.  1 - s by s's error and u; the slope by those and four more."""
    u = ff.U
    if act == vh.VK_GATE_SILU:
        s = 1 / (1 + np.exp(-g))
        es = s * np.where(g < 0, 8 + 2 * np.abs(g), 8 + 2 * np.abs(g) * (1 - s)) * u
        one = es + u
        slope = s * (1 + g * (1 - s))
        return (g * s, np.abs(g) * (es + s * u), slope,
                es * np.abs(1 + g * (1 - s)) + s * np.abs(g) * one + 4 * u * s * (1 + np.abs(g)))
    p, tail = phi(g), phi(-np.abs(g))
    part = (19 + 1.3 * g * g) * u
    ep = tail * part + p * u
    density = np.abs(g) * np.exp(-g * g / 2) / math.sqrt(2 * math.pi)
    slope = p + np.sign(g) * density
    return (g * p, np.abs(g) * (ep + p * u), slope, ep + density * (part + 5 * u) + np.abs(slope) * u)


def gates(t, low, high):
    return np.unique(ff.rounded(np.linspace(low, high, 1501), t)).astype(np.float64)


# as far out as the results are normal numbers of the type
RANGES = {("bf16", 0): (-80, 80), ("bf16", 1): (-12.7, 12.7), ("f16", 0): (-11, 40),
          ("f16", 1): (-3.9, 40)}


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("t", ["bf16", "f16"])
@pytest.mark.parametrize("rows", [True, False])
def test_forward_and_backward(rt, t, act, rows):
    """One gate a row (few rows and tiles), partners and gradients of 1 or powers of two."""
    g = gates(t, *RANGES[t, act])
    want, tol, slope, tol_slope = act_of(g, act)
    k, h = 8, 40
    calls = [g[i:i + 17] for i in range(0, len(g), 170)] if rows else [g]
    for part in calls:
        m = len(part)
        x = np.zeros((m, k), np.float32)
        x[:, 0], x[:, 1] = part, 1
        w = np.zeros((2 * h, k), np.float32)
        w[:h, 0], w[h:, 1] = 1, 2.0 ** np.arange(h) if t == "bf16" else 2.0 ** (np.arange(h) % 8)
        dx, dw = ff.upload(rt, x, t), ff.upload(rt, w, t)
        out = rt.alloc(ff.DTYPE[t], m * h)
        rt.gated_forward(dx, dw, None, m, k, h, out, act)
        at = np.searchsorted(g, part)
        up = w[h:, 1].astype(np.float64)
        v = want[at][:, None] * up
        ff.assert_within(rt.download_16(out), v, ff.held(v, tol[at][:, None] * up, t), "forward")


@pytest.mark.parametrize("act", ACTS)
def test_slopes(rt, act):
    """dbias of one row: the gradients of g and u themselves, rounded once."""
    t, m, k = "bf16", 1, 8
    g = gates(t, *RANGES[t, act])
    h = len(g)
    x = np.zeros((m, k), np.float32)
    x[0, 0] = 1
    w = np.zeros((2 * h, k), np.float32)
    w[:h, 0], w[h:, 0] = g, 4
    grad = np.full((m, h), 0.5, np.float32)
    db = rt.alloc(vh.VK_BF16, 2 * h)
    rt.gated_backward(*(ff.upload(rt, v, t) for v in (x, w)), None, ff.upload(rt, grad, t), m, k, h,
                      None, None, db, act)
    a, ta, s, ts = act_of(g, act)
    want = np.concatenate([2 * s, 0.5 * a])
    tol = np.concatenate([2 * ts, 0.5 * ta]) + 2 * ff.U * np.abs(want)
    ff.assert_within(rt.download_16(db), want, ff.held(want, tol, t), "dg, du")


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("m", [9, 120])
def test_eight_bits(rt, m, act):
    """f32 results, whose partners are large: g = code / 16 (SiLU: code / 2), u = 127 2^20."""
    k, h = 40, 30
    step = 2.0 ** (-4 if act == vh.VK_GATE_GELU else -1)
    rng = np.random.default_rng(3)
    codes = rng.integers(-127, 128, (m, h))
    x = np.zeros((m, k), np.float32)
    x[:, :h], x[:, h] = codes, 127  # each row's scale is 1
    w = np.zeros((2 * h, k), np.int8)
    w[:h, :h], w[h:, h] = np.eye(h), 1
    scale = np.r_[np.full(h, step), np.full(h, 2.0 ** 20)].astype(np.float32)
    out = rt.alloc_f32(m * h)
    rt.prepare_linear_i8(k, 2 * h, w, scale).run_gated(rt.upload_f32(x), m, out, act)
    v, tol, _, _ = act_of(codes * step, act)
    u = 127 * 2.0 ** 20
    ff.assert_within(out.numpy(), v * u, (tol + ff.U * np.abs(v)) * u, (m, act))
