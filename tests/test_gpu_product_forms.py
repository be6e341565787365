"""Every form of the products of the feed-forward in fewer bits against 64 bits: each tile, whole
and with its k shared out over workgroups, alone and beside another product."""
import numpy as np
import pytest

import feed_forward as ff
import product_forms as forms
import vestra_hip as vh

pytestmark = pytest.mark.gpu


def inputs(rng, m, k, h, t):
    x = ff.rounded(rng.standard_normal((m, k), np.float32), t)
    w = ff.rounded(rng.standard_normal((2 * h, k), np.float32) * np.float32(1.5 * k ** -0.5), t)
    return x, w, ff.rounded(rng.standard_normal(2 * h, np.float32) * np.float32(0.3), t)


@pytest.mark.parametrize("t", ["f16", "bf16"])
@pytest.mark.parametrize("m,k,h", forms.FORWARD)
def test_forward(rt, rng, m, k, h, t):
    x, w, b = inputs(rng, m, k, h, t)
    out = rt.alloc(ff.DTYPE[t], m * h)
    rt.gated_forward(*(ff.upload(rt, v, t) for v in (x, w, b)), m, k, h, out)
    ff.assert_within(rt.download_16(out), *ff.forward(x, w, b, vh.VK_GATE_SILU, t), (m, k, h))


@pytest.mark.parametrize("t,m,k,h", [(t, *s) for t in forms.BACKWARD for s in forms.BACKWARD[t]])
def test_backward(rt, rng, t, m, k, h):
    x, w, b = inputs(rng, m, k, h, t)
    grad = ff.rounded(rng.standard_normal((m, h), np.float32) * np.float32(0.1), t)
    out = {n: rt.alloc(ff.DTYPE[t], s) for n, s in
           (("dx", m * k), ("dw", 2 * h * k), ("dbias", 2 * h))}
    rt.gated_backward(*(ff.upload(rt, v, t) for v in (x, w, b, grad)), m, k, h, out["dx"],
                      out["dw"], out["dbias"])
    for n, (want, tol) in ff.backward(x, w, b, grad, vh.VK_GATE_SILU, t).items():
        ff.assert_within(rt.download_16(out[n]), want, tol, (n, m, k, h))


def linear(rng, m, k, n):
    """x, codes, scales that make results of unit size, a bias."""
    x = rng.standard_normal((m, k), np.float32)
    w = rng.integers(-127, 128, (n, k)).astype(np.int8)
    t = (rng.uniform(0.5, 1, n) * k ** -0.5 / 73).astype(np.float32)
    return x, w, t, rng.standard_normal(n).astype(np.float32)


@pytest.mark.parametrize("m,k,n", forms.LINEAR_I8)
def test_linear_i8(rt, rng, m, k, n):
    x, w, t, b = linear(rng, m, k, n)
    lin, dx = rt.prepare_linear_i8(k, n, w, t, b), rt.upload_f32(x)
    y, tol = ff.linear(x, w, t, b, None)
    for out in ("f32", "bf16", "f16"):
        got = rt.alloc(ff.DTYPE[out], m * n)
        lin.run_into(dx, m, got)
        ff.assert_within(ff.download(rt, got), y, ff.held(y, tol, out), (m, k, n, out))
    r = rng.standard_normal((m, n), np.float32)
    got = rt.upload_f32(r)
    lin.run_residual(dx, m, got)
    ff.assert_within(got.numpy(), r + y, tol + 1.01 * ff.U * np.abs(r + y), (m, k, n, "residual"))


@pytest.mark.parametrize("m,k,h", forms.GATED_I8)
def test_gated_i8(rt, rng, m, k, h):
    x, w, t, b = linear(rng, m, k, 2 * h)
    lin, dx = rt.prepare_linear_i8(k, 2 * h, w, t, b), rt.upload_f32(x)
    y, tol = ff.linear(x, w, t, b, None)
    want, tol = ff.gated(y[:, :h], y[:, h:], tol[:, :h], tol[:, h:], vh.VK_GATE_SILU)
    for out in ("f32", "bf16", "f16"):
        got = rt.alloc(ff.DTYPE[out], m * h)
        lin.run_gated(dx, m, got)
        ff.assert_within(ff.download(rt, got), want, ff.held(want, tol, out), (m, k, h, out))
