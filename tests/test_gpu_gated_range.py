"""Gradients of the gated feed-forward in f16 whose dg and du f16 does not hold as they are, while
it holds dx and dw: past 65,504, and below the normal numbers."""
import numpy as np
import pytest

import cached
import feed_forward as ff
import vestra_hip as vh

pytestmark = pytest.mark.gpu


def exact(x, w, grad, act):
    """{name: (gradient, tolerance)} as ff.backward has them, but for the operands' rounding: d times
    a power of two is rounded to 11 bits, or where it then lies below f16's normal numbers, to a
    multiple of 2^-24: the largest |d| times that power is at least 2^14 (or the power 1 and |d| at
    least 2^-8), so that this is off by 2^-39 (2^-17) of the largest at most."""
    x, w, dh = (v.astype(np.float64) for v in (x, w, grad))
    n = w.shape[0] // 2
    y, tol = ff.products(x, w, None)
    g, u, tg, tu = y[:, :n], y[:, n:], tol[:, :n], tol[:, n:]
    a, slope, ta = ff.activation(g, act)
    ts = 0.8 * tg + (np.abs(g) + 2) * 12 * ff.U
    d = np.concatenate([dh * u * slope, dh * a], 1)
    td = np.concatenate([np.abs(dh) * (tu * np.abs(slope) + np.abs(u) * ts + tu * ts),
                         np.abs(dh) * (ta + 1.13 * tg)], 1) + 3 * ff.U * np.abs(d)
    top = np.abs(d).max()
    floor = top * 2.0 ** (-17 if 2.0 ** -8 <= top <= 65504 else -39)
    th = td + 2.0 ** -11 * (np.abs(d) + td) + floor
    rows = x.shape[0]
    out = {"dx": (d @ w, th @ np.abs(w) + 2 * n * 2 * ff.U * (np.abs(d) @ np.abs(w))),
           "dw": (d.T @ x, th.T @ np.abs(x) + rows * 2 * ff.U * (np.abs(d).T @ np.abs(x))),
           "dbias": (d.sum(0), td.sum(0) + rows * ff.U * np.abs(d).sum(0))}
    return {k: (v, ff.held(v, e, "f16")) for k, (v, e) in out.items()}


def inputs(rng, m, k, h, size, large):
    """Rows of x of `size`, weights small enough for dx; gradients up to `large`."""
    x = ff.rounded(rng.standard_normal((m, k)) * size, "f16")
    w = ff.rounded(rng.standard_normal((2 * h, k)) * 2.0 * k ** -0.5 / size, "f16")
    grad = ff.rounded(rng.uniform(-1, 1, (m, h)) * large, "f16")
    return x, w, grad


def call(rt, x, w, grad, act, want, m, k, h):
    o = {n: rt.alloc(vh.VK_F16, s) for n, s in (("dx", m * k), ("dw", 2 * h * k), ("dbias", 2 * h))}
    a = [ff.upload(rt, v, "f16") for v in (x, w)]
    rt.gated_backward(*a, None, ff.upload(rt, grad, "f16"), m, k, h, o["dx"], o["dw"], o["dbias"],
                      act)
    for n, (v, tol) in want.items():
        got = rt.download_16(o[n]).astype(np.float64).reshape(v.shape)
        fine = np.abs(v) + tol < 65504
        assert np.isinf(got[np.abs(v) - tol > 65520]).all(), n
        ff.assert_within(np.where(fine, got, 0), np.where(fine, v, 0), tol, (n, m, k, h, act))


# few tiles whose k is shared out, whole tiles of each size, rows and widths that no tile divides
SIZES = [(1, 64, 64), (5, 40, 33), (40, 2881, 65), (130, 384, 129), (257, 384, 300),
         (1300, 96, 1000)]


@pytest.mark.parametrize("act", [vh.VK_GATE_SILU, vh.VK_GATE_GELU])
@pytest.mark.parametrize("m,k,h", SIZES)
def test_past_the_largest_number(rt, rng, m, k, h, act):
    """du and dg some times 65,504; x and w small, so that dx and dw are held."""
    x, w, grad = inputs(rng, m, k, h, 2.0 ** -4, 60000)
    w[h:] *= np.float32(4)
    w = ff.rounded(w, "f16")
    x[:, 0], w[:h, 0] = 1, 0  # one partner of every row is 8 or more
    w[h, 0] = 9
    want = exact(x, w, grad, act)
    call(rt, x, w, grad, act, want, m, k, h)


@pytest.mark.parametrize("act", [vh.VK_GATE_SILU, vh.VK_GATE_GELU])
@pytest.mark.parametrize("m,k,h", SIZES)
def test_below_the_normal_numbers(rt, rng, m, k, h, act):
    """Gradients of 2^-24 to 2^-18 and partners of some 2^-7, rows of x of 2^6: dg and du are
    below what f16 holds, dw is not."""
    x, w, grad = inputs(rng, m, k, h, 2.0 ** 6, 2.0 ** -18)
    w[h:] = ff.rounded(w[h:] * 2.0 ** -8, "f16")
    want = exact(x, w, grad, act)
    call(rt, x, w, grad, act, want, m, k, h)


def test_it_is_held_and_not_all_zeros(rng):
    """That the two above look at what they say (no GPU in it): f16's own d has infinities or is
    half zeros, the results are numbers."""
    m, k, h = 257, 384, 300
    x, w, grad = inputs(rng, m, k, h, 2.0 ** 6, 2.0 ** -18)
    w[h:] = ff.rounded(w[h:] * 2.0 ** -8, "f16")
    y = x.astype(np.float64) @ w.astype(np.float64).T
    dg = grad * y[:, h:] * ff.activation(y[:, :h], 0)[1]
    assert (ff.rounded(dg, "f16") == 0).mean() > 0.5
    assert (ff.rounded(exact(x, w, grad, 0)["dw"][0], "f16") == 0).mean() < 0.1


@pytest.mark.parametrize("size", [2.0 ** -16, 30000])
def test_a_row_that_is_no_number(rt, rng, size):
    """It chooses no power: the others' dx stands."""
    m, k, h = 90, 40, 24
    x, w, grad = inputs(rng, m, k, h, 1.0, size)
    w[h:] = ff.rounded(w[h:] * 2.0 ** (-8 if size < 1 else 4), "f16")
    w[:h] = ff.rounded(w[:h] * 2.0 ** -4, "f16")
    w[h:, 1:] *= np.float32(2.0 ** -9 if size > 1 else 1)
    x[33] = np.nan
    dx = rt.alloc(vh.VK_F16, m * k)
    rt.gated_backward(*(ff.upload(rt, v, "f16") for v in (x, w)), None, ff.upload(rt, grad, "f16"),
                      m, k, h, dx, None, None)
    got = rt.download_16(dx).reshape(m, k).astype(np.float64)
    rest = np.r_[0:33, 34:90]
    v, tol = exact(x[rest], w, grad[rest], vh.VK_GATE_SILU)["dx"]
    fine = np.abs(v) + tol < 65504
    ff.assert_within(np.where(fine, got[rest], 0), np.where(fine, v, 0), tol, "dx")
    assert np.isnan(got[33]).all()


def test_an_infinity_leaves_d_as_it_is(rt, rng):
    """As at ordinary sizes: the other rows' dx has the bits that it has without that row."""
    m, k, h = 90, 40, 24
    x, w, grad = inputs(rng, m, k, h, 1.0, 1.0)
    a = [ff.upload(rt, v, "f16") for v in (x, w)]
    got = []
    for g in (grad, np.where(np.arange(m)[:, None] == 44, np.float32(np.inf), grad)):
        dx = rt.alloc(vh.VK_F16, m * k)
        rt.gated_backward(*a, None, ff.upload(rt, g, "f16"), m, k, h, dx, None, None)
        got.append(rt.download_16(dx).reshape(m, k))
    assert not np.isfinite(got[1][44]).all()
    got[1][44] = got[0][44]
    np.testing.assert_array_equal(*got)


def test_one_at_a_time_and_captured(rt, rng):
    """Each gradient alone gives the bits of all together; replays of one graph follow the
    gradients' size, whichever side of f16 they are on."""
    m, k, h = 130, 384, 129
    x, w, _ = inputs(rng, m, k, h, 2.0 ** -2, 1)
    a = [ff.upload(rt, v, "f16") for v in (x, w)]
    grads = [ff.upload(rt, ff.rounded(rng.uniform(-1, 1, (m, h)) * s, "f16"), "f16")
             for s in (1, 60000, 2.0 ** -18, 30, 60000)]
    o = [rt.alloc(vh.VK_F16, s) for s in (m * k, 2 * h * k, 2 * h)]
    alone = [rt.alloc(vh.VK_F16, len(v)) for v in o]

    def step(grad, out=o):
        rt.gated_backward(*a, None, grad, m, k, h, *out)

    step(grads[0])
    graphs = [cached.captured(rt, lambda grad=grad: step(grad)) for grad in grads]
    for _ in range(2):
        for grad, graph in zip(grads, graphs):
            for i in range(3):
                step(grad, [alone[j] if j == i else None for j in range(3)])
            step(grads[3])  # other values in the outputs
            graph.launch()
            for p, q in zip(o, alone):
                np.testing.assert_array_equal(rt.download_16(p), rt.download_16(q))
