"""The linear in 8-bit integers against its 64-bit form: codes, sums, epilogues and the
gated form, over sizes that no tile divides, types, and rows that hold what a row may."""
import numpy as np
import pytest

import cached
import feed_forward as ff
import vestra_hip as vh

pytestmark = pytest.mark.gpu


def weights(rng, k, n):
    w = rng.standard_normal((n, k)).astype(np.float32)
    codes, scale = ff.quantised(w)
    return codes.astype(np.int8), scale


def rows_of(rng, m, k, t="f32"):
    x = rng.standard_normal((m, k)).astype(np.float32) * (1 + 7 * (rng.random(k) < 0.02))
    return ff.rounded(x, t)


def run(rt, lin, x, t, n, out, call, start=None):
    m = x.shape[0]
    dx = ff.upload(rt, x, t)
    y = rt.upload_f32(start) if start is not None else rt.alloc(ff.DTYPE[out], m * n)
    call(lin, dx, m, y)
    return ff.download(rt, y).reshape(m, n)


SIZES = [(1, 64, 64), (1, 1024, 4096), (2, 130, 33), (3, 5000, 40), (4, 4096, 20), (4, 4097, 17),
         (5, 900, 70), (7, 1, 5), (16, 257, 96), (17, 512, 48),
         (31, 1031, 200), (32, 4096, 64), (33, 127, 65), (64, 128, 64), (65, 129, 127),
         (130, 768, 300), (257, 384, 257), (866, 768, 640), (1301, 770, 1999), (300, 5000, 96),
         (40, 20000, 70), (129, 9000, 33), (17, 9000, 50), (32, 20001, 130), (2, 20000, 96),
         (2600, 512, 2304)]


@pytest.mark.parametrize("m,k,n", SIZES)
def test_sums_of_every_size(rt, rng, m, k, n):
    w, t = weights(rng, k, n)
    b = rng.standard_normal(n).astype(np.float32)
    x = rows_of(rng, m, k)
    got = run(rt, rt.prepare_linear_i8(k, n, w, t, b), x, "f32", n, "f32",
              lambda lin, *a: lin.run_into(*a))
    want, tol = ff.linear(x, w, t, b, None)
    ff.assert_within(got, want, tol, (m, k, n))


@pytest.mark.parametrize("m,k,n", [(1, 300, 70), (20, 256, 100), (200, 520, 130),
                                   (3000, 128, 2050)])
@pytest.mark.parametrize("t,out", [("f32", "bf16"), ("f16", "f32"), ("bf16", "f16"), ("f16", "f16"),
                                   ("bf16", "bf16")])
def test_types(rt, rng, m, k, n, t, out):
    w, s = weights(rng, k, n)
    x = rows_of(rng, m, k, t)
    got = run(rt, rt.prepare_linear_i8(k, n, w, s), x, t, n, out, lambda lin, *a: lin.run_into(*a))
    want, tol = ff.linear(x, w, s, None, None)
    ff.assert_within(got, want, ff.held(want, tol, out), (m, k, n, t, out))


@pytest.mark.parametrize("m,k,n", [(1, 256, 64), (19, 130, 70), (257, 384, 260), (2600, 256, 2300)])
def test_epilogues(rt, rng, m, k, n):
    w, s = weights(rng, k, n)
    b, g = (rng.standard_normal(n).astype(np.float32) for _ in "bg")
    x = rows_of(rng, m, k)
    plain = rt.prepare_linear_i8(k, n, w, s, b)
    scaled = rt.prepare_linear_i8(k, n, w, s, b, g)
    y, tol = ff.linear(x, w, s, b, None)
    got = run(rt, plain, x, "f32", n, "f32", lambda lin, *a: lin.run_gelu(*a))
    ff.assert_within(got, ff.activation(y, vh.VK_GATE_GELU)[0], ff.gelu_tolerance(y, tol), "gelu")
    r = rng.standard_normal((m, n)).astype(np.float32)
    got = run(rt, plain, x, "f32", n, "f32", lambda lin, *a: lin.run_residual(*a), r)
    ff.assert_within(got, r + y, tol + 1.01 * ff.U * np.abs(r + y), "residual")
    y, tol = ff.linear(x, w, s, b, g)
    got = run(rt, scaled, x, "f32", n, "f32", lambda lin, *a: lin.run_into(*a))
    ff.assert_within(got, y, tol, "LayerScale")
    got = run(rt, scaled, x, "f32", n, "f32", lambda lin, *a: lin.run_residual(*a), r)
    ff.assert_within(got, r + y, tol + 1.01 * ff.U * np.abs(r + y), "LayerScale, residual")


@pytest.mark.parametrize("act", [vh.VK_GATE_SILU, vh.VK_GATE_GELU])
@pytest.mark.parametrize("m,k,h,out", [(1, 1536, 4096, "f32"), (1, 7, 1, "f32"),
                                       (15, 130, 31, "bf16"), (32, 384, 96, "f16"),
                                       (33, 384, 33, "f32"), (130, 257, 191, "f32"), (866, 256, 683, "bf16"),
                                       (2700, 200, 1365, "f32")])
def test_gated(rt, rng, m, k, h, out, act):
    w, s = weights(rng, k, 2 * h)
    s = s * np.float32(2 * k ** -0.5)
    b = rng.standard_normal(2 * h).astype(np.float32)
    x = rows_of(rng, m, k)
    lin = rt.prepare_linear_i8(k, 2 * h, w, s, b)
    got = run(rt, lin, x, "f32", h, out, lambda lin, *a: lin.run_gated(*a, act))
    y, tol = ff.linear(x, w, s, b, None)
    want, tol = ff.gated(y[:, :h], y[:, h:], tol[:, :h], tol[:, h:], act)
    ff.assert_within(got, want, ff.held(want, tol, out), (m, k, h))


@pytest.mark.parametrize("m,k,n", [(9, 200, 40), (150, 200, 70)])
def test_rows_that_hold_anything(rt, rng, m, k, n):
    w, s = weights(rng, k, n)
    b = rng.standard_normal(n).astype(np.float32)
    x = rows_of(rng, m, k)
    x[0] = 0
    x[1, 7], x[2, 3], x[3, k - 1] = np.nan, np.inf, -np.inf
    x[4] *= np.float32(2.0 ** -110)  # a scale below the least: zeros
    x[5] *= np.float32(1e36)
    x[6] = np.finfo(np.float32).max
    x[7] *= np.float32(2.0 ** -90)
    x[8, 1:] = 0
    got = run(rt, rt.prepare_linear_i8(k, n, w, s, b), x, "f32", n, "f32",
              lambda lin, *a: lin.run_into(*a))
    want, tol = ff.linear(x, w, s, b, None)
    assert np.isnan(got[1:4]).all() and np.array_equal(got[0], b) and np.array_equal(got[4], b)
    fine = np.abs(want) < 3.4e38  # what f32 holds
    assert np.isinf(got[~fine & ~np.isnan(want)]).all()
    want[~fine], got[~fine] = 0, 0
    ff.assert_within(got, want, tol, "rows")


def test_ties_and_borders_of_codes(rt):
    """Quotients at and next to half a step, rounded to f32 and then to even."""
    k, n = 254, 254
    x = np.zeros((300, k), np.float32)
    rng = np.random.default_rng(5)
    for i in range(300):
        top = np.float32(rng.uniform(0.5, 2) * 2.0 ** rng.integers(-8, 8))
        d = top / np.float32(127)
        half = (np.arange(-126, 127) + 0.5).astype(np.float32) * d
        x[i, 1:] = np.nextafter(half, np.float32([np.inf, -np.inf, 0])[i % 3]) if i % 4 else half
        x[i, 0] = top
    w = np.eye(k, dtype=np.int8)  # each column copies a code
    lin = rt.prepare_linear_i8(k, n, w, np.ones(n, np.float32))
    got = run(rt, lin, x, "f32", n, "f32", lambda lin, *a: lin.run_into(*a))
    c, s = ff.quantised(x)
    np.testing.assert_array_equal(got, (c * s[:, None]).astype(np.float32))


@pytest.mark.parametrize("k", [1, 130, 131072])
def test_largest_sums(rt, k):
    """All codes at their ends: the int32 sum at its largest."""
    x = np.full((40, k), 3.0, np.float32)
    w = np.full((33, k), -128, np.int8)
    got = run(rt, rt.prepare_linear_i8(k, 33, w, np.ones(33, np.float32)), x, "f32", 33, "f32",
              lambda lin, *a: lin.run_into(*a))
    want, tol = ff.linear(x, w, np.ones(33, np.float32), None, None)
    ff.assert_within(got, want, tol, k)


def test_weights_quantised_here(rt, rng):
    k, n = 140, 50
    w = rng.standard_normal((k, n)).astype(np.float32)
    w[:, 3], w[5, 4] = 0, np.inf
    x = rows_of(rng, 70, k)
    codes, s = ff.quantised(w.T.copy())
    got = [run(rt, lin, x, "f32", n, "f32", lambda lin, *a: lin.run_into(*a)) for lin in
           (rt.prepare_linear_i8_f32(k, n, w),
            rt.prepare_linear_i8(k, n, codes.astype(np.int8), s))]
    np.testing.assert_array_equal(*got)
    assert np.isnan(got[0][:, 4]).all() and (got[0][:, 3] == 0).all()


def test_no_rows(rt, rng):
    w, s = weights(rng, 64, 32)
    lin = rt.prepare_linear_i8(64, 32, w, s)
    lin.run_into(rt.alloc_f32(0), 0, rt.alloc_f32(0))
    rt.synchronize()


def test_guard_values_stay(rt, rng):
    """Nothing past the rows of the output is written."""
    for m, n in ((1, 33), (30, 65), (100, 67), (300, 2050)):
        w, s = weights(rng, 96, n)
        lin = rt.prepare_linear_i8(96, n, w, s)
        room = rt.upload_f32(np.full(m * n + 512, 7.0, np.float32))
        lin.run_into(rt.upload_f32(rows_of(rng, m, 96)), m, room.view(256, m * n))
        got = room.numpy()
        assert (got[:256] == 7).all() and (got[256 + m * n:] == 7).all()
        assert (got[256:-256] != 7).all()


@pytest.mark.parametrize("m", [1, 40, 1000])
def test_captured(rt, rng, m):
    k, n = 256, 320
    w, s = weights(rng, k, n)
    lin = rt.prepare_linear_i8(k, n, w, s)
    x, y = rt.upload_f32(rows_of(rng, m, k)), rt.alloc_f32(m * n)
    lin.run_into(x, m, y)
    g = cached.captured(rt, lambda: lin.run_into(x, m, y))
    for _ in range(3):
        h = rows_of(rng, m, k)
        x.write(h)
        g.launch()
        got = y.numpy().reshape(m, n)
        lin.run_into(x, m, y)  # the program's own work between replays
        np.testing.assert_array_equal(got, y.numpy().reshape(m, n))
        want, tol = ff.linear(h, w, s, None, None)
        ff.assert_within(got, want, tol, m)


def test_two_runtimes_share_a_linear(rng):
    """Queued together, each with its own codes of x, sums and counters; few tiles of a long k."""
    a, b = vh.Runtime(0), vh.Runtime(0)
    calls = []
    for m, k, n in ((40, 20000, 70), (866, 768, 640), (8, 300, 90)):
        w, s = weights(rng, k, n)
        lin = a.prepare_linear_i8(k, n, w, s)
        for r in (a, b):
            x, y = rows_of(rng, m, k), r.alloc_f32(m * n)
            calls.append((r, lin, r.upload_f32(x), m, y, ff.linear(x, w, s, None, None)))
    for _ in range(4):
        for r, lin, x, m, y, _ in calls:
            assert vh.lib.vk_linear_i8_run_into(r.handle, lin.handle, x.handle, m, y.handle) == 0
    for r, _, _, m, y, (want, tol) in calls:
        r.synchronize()
        ff.assert_within(y.numpy(), want, tol, m)


def test_refusals(rt, rng):
    w, s = weights(rng, 64, 33)
    g = np.ones(33, np.float32)
    lin, scaled = rt.prepare_linear_i8(64, 33, w, s), rt.prepare_linear_i8(64, 33, w, s, None, g)
    x, y = rt.alloc_f32(2 * 64), rt.alloc_f32(2 * 33)
    room = rt.alloc_f32(1024)

    def refused(code, call, *a):
        with pytest.raises(vh.VestraError) as e:
            call(*a)
        assert e.value.code == code, e.value

    bad = vh.VK_ERR_INVALID
    refused(bad, lin.run_into, x, 3, y)
    refused(vh.VK_ERR_UNSUPPORTED, lin.run_into, x, 1 << 24, y)
    refused(bad, lin.run_into, x, 2, rt.alloc_f32(2 * 32))
    refused(bad, lin.run_into, rt.alloc_u8(128), 2, y)
    refused(bad, lin.run_into, room.view(0, 128), 2, room.view(64, 66))
    refused(bad, lin.run_into, room.view(1, 128), 2, y)
    refused(bad, lin.run_residual, x, 2, rt.alloc(vh.VK_BF16, 66))
    refused(bad, lin.run_gated, x, 2, rt.alloc_f32(33))  # an odd number of columns
    refused(bad, scaled.run_gelu, x, 2, y)
    even = rt.prepare_linear_i8(64, 32, w[:32], s[:32])
    refused(bad, even.run_gated, x, 2, rt.alloc_f32(32), 5)
    refused(vh.VK_ERR_UNSUPPORTED, rt.prepare_linear_i8, 131073, 1, np.zeros(131073, np.int8),
            np.ones(1, np.float32))
    refused(bad, rt.prepare_linear_i8, 64, 33, w, s[:32])
    lin.run_into(x, 2, y)  # and still runs
    rt.synchronize()
