"""The 8-bit linear where the scales of rows and channels are far apart: what one of them takes out
of f32, the other brings back."""
import numpy as np
import pytest

import feed_forward as ff
import vestra_hip as vh

pytestmark = pytest.mark.gpu

MOST = float(np.finfo(np.float32).max)


@pytest.mark.parametrize("m", [7, 20, 100])
@pytest.mark.parametrize("end", ["plain", "gated"])
def test_scales_far_apart(rt, rng, m, end):
    """Few rows that each workgroup quantises, few rows, tiles.  Channel scales of 2^-140 to 2^127,
    row scales of 2^-97 to 2^120."""
    k, n = 300, 60
    c = rng.integers(-127, 128, (n, k)).astype(np.int8)
    t = (rng.uniform(1, 2, n) * 2.0 ** np.linspace(-140, 126, n)).astype(np.float32)
    x = rng.standard_normal((m, k)).astype(np.float32)
    x *= (2.0 ** np.linspace(-92, 118, m)).astype(np.float32)[:, None]
    if end == "gated":  # partners of 1: the gate's columns are what is looked at, where they are large
        c[n // 2:], t[n // 2:] = 0, 1
        bias = np.r_[np.zeros(n // 2), np.ones(n // 2)].astype(np.float32)
        t[:n // 2] = (rng.uniform(1, 2, n // 2) * 2.0 ** np.linspace(-40, 126, n // 2)).astype(np.float32)
        out = rt.alloc_f32(m * n // 2)
        rt.prepare_linear_i8(k, n, c, t, bias).run_gated(rt.upload_f32(x), m, out, vh.VK_GATE_SILU)
        got = out.numpy().reshape(m, n // 2).astype(np.float64)
        y, tol = ff.linear(x, c[:n // 2], t[:n // 2], None, None)
        fine = (np.abs(y) < 0.99 * MOST) & (y > 100)  # there SiLU is the gate itself
        off = np.abs(got - y) - tol - 12 * ff.U * np.abs(y)
        assert fine.sum() > 30 and (off[fine] <= 0).all()
        assert (got[y > 1.01 * MOST] == np.inf).all()
        return
    out = rt.alloc_f32(m * n)
    rt.prepare_linear_i8(k, n, c, t).run_into(rt.upload_f32(x), m, out)
    got = out.numpy().reshape(m, n).astype(np.float64)
    y, tol = ff.linear(x, c, t, None, None)
    fine = np.abs(y) < 0.99 * MOST
    assert fine.sum() > m * n // 2
    ff.assert_within(np.where(fine, got, 0), np.where(fine, y, 0), tol, (m, end))
    past = np.abs(y) > 1.01 * MOST
    assert past.any() and np.isinf(got[past]).all()
