"""The attention over the 8-bit cache at the ends of f32: the same meaning whichever form a call
takes (one query, few, tiles of 128), and nothing of what a query does not see."""
import numpy as np
import pytest

import cached
from test_gpu_attention_cached import Case

pytestmark = pytest.mark.gpu

vh = pytest.importorskip("vestra_hip")

ROWS = [1, 9, 70]


@pytest.mark.parametrize("n", ROWS)
@pytest.mark.parametrize("keys", [300, 3000])
@pytest.mark.parametrize("code", [0x7f, 0xff])
def test_hidden_codes_change_no_bit_of_small_queries(rt, rng, n, keys, code):
    """Slots of another document whose codes are no number, beside queries whose products with a
    code are near f32's smallest numbers."""
    c = Case(rt, rng, 1, 1, 2, 2, keys, n, [keys - n], qs=1e-37, ks=1e37).fill()
    hidden = np.arange(5, keys - n, 16)
    docs = {"q_docs": np.zeros((1, n), np.int32), "k_docs": np.zeros((1, keys), np.int32)}
    docs["k_docs"][:, hidden] = 1
    want = c.check(docs, pick=[0, n // 2, n - 1])
    codes = cached.quantise(c.k, 1)[0]
    codes[:, :, hidden, ::7] = code
    c.cache.k.write(codes.reshape(-1))
    assert np.array_equal(c.run(docs), want)


@pytest.mark.parametrize("n", ROWS)
@pytest.mark.parametrize("fmt", [0, 1])
@pytest.mark.parametrize("qs,ks,rule", [
    (1e27, 1e-27, {"scale": 0.125, "cap": 2e-13}),         # q scale / cap past f32's largest
    (3e37, 1e-30, {"scale": 2.0 ** 30, "cap": 2.0 ** 32}),
    (1e30, 1e-28, {"scale": 2.0 ** 39}),                   # q scale past it
    (1e-36, 1e25, {"scale": 2.0 ** 39, "cap": 2.0 ** 79}),  # q scale / cap below its smallest
    (1e-38, 3e37, {"scale": 2.0 ** -39}), (1e-42, 1e35, {"scale": 2.0 ** 25}),
    (1e-38, 3e37, {"scale": -0.125}), (3e37, 1e-38, {"scale": 0.25, "cap": 1.0}),
])
def test_scaled_queries_outside_f32(rt, rng, fmt, n, qs, ks, rule):
    """Scores in range, of a query times the scale (over the cap) that is not."""
    c = Case(rt, rng, fmt, 1, 2, 2, 330, n, [330 - n], qs=qs, ks=ks).fill()
    c.check(rule, label=f"{qs} {ks} {rule}")


@pytest.mark.parametrize("n", ROWS)
@pytest.mark.parametrize("qs,ks", [(1e22, 1e22), (1e30, 1e10), (1e10, 1e30)])
def test_products_that_a_small_scale_brings_back(rt, rng, n, qs, ks):
    """q . k past f32's largest, the score far inside: one key has all the weight."""
    c = Case(rt, rng, 0, 1, 2, 2, 330, n, [330 - n], qs=qs, ks=ks).fill()
    got = c.check({"scale": 2.0 ** -40})
    assert np.isfinite(got).all()
    q, k = c.q.astype(np.float64), c.kh
    best = np.argmax(np.einsum("shid,shjd->shij", q, k), -1)
    assert np.allclose(got[0, 1, 0], c.vheld[0, 1, best[0, 1, 0]], rtol=1e-6, atol=1e-12)


@pytest.mark.parametrize("n", ROWS)
@pytest.mark.parametrize("fmt", [0, 1])
@pytest.mark.parametrize("which", ["k_scale", "v_scale"])
@pytest.mark.parametrize("scale", [np.inf, -np.inf, np.nan])
def test_scales_that_are_no_number(rt, rng, n, fmt, which, scale):
    """An infinite or NaN scale, put there by hand: NaN to every query that sees the key, in
    every column, whatever its codes and its score are."""
    keys = 200
    c = Case(rt, rng, fmt, 1, 2, 2, keys, n, [keys - n]).fill()
    bad = 77
    c.k[:, :, bad], c.v[:, :, bad, ::2] = 0.5 * c.k[:, :, bad], 0.0
    c.fill()
    want = c.run()
    t = getattr(c.cache, which)
    scales = t.numpy().reshape(1, 2, keys)
    scales[0, 1, bad] = scale
    t.write(scales.reshape(-1))
    got = c.run()
    assert np.array_equal(got[:, 0], want[:, 0]) and np.isnan(got[:, 1]).all()
    # a score of -inf beside it
    c.q[0, 1, 0] = -1e30 * np.sign(c.kh[0, 1, bad])
    assert np.isnan(c.run()[0, 1, 0]).all()
