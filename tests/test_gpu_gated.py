"""The gated feed-forward in 16 bits, forward and backward, against its 64-bit form."""
import numpy as np
import pytest

import cached
import feed_forward as ff
import vestra_hip as vh

pytestmark = pytest.mark.gpu
ACTS = [vh.VK_GATE_SILU, vh.VK_GATE_GELU]


def inputs(rng, m, k, h, t, bias=True):
    x = ff.rounded(rng.standard_normal((m, k)), t)
    w = ff.rounded(rng.standard_normal((2 * h, k)) * 1.5 * k ** -0.5, t)
    b = ff.rounded(rng.standard_normal(2 * h) * 0.3, t) if bias else None
    return x, w, b


def up(rt, t, *arrays):
    return [None if a is None else ff.upload(rt, a, t) for a in arrays]


SIZES = [(1, 64, 64), (1, 8, 1), (48, 2881, 173), (70, 4000, 64), (33, 2000, 7), (2, 136, 33),
         (5, 1024, 300), (16, 7, 40), (17, 513, 70), (32, 384, 96), (33, 100, 31),
         (64, 64, 32), (70, 257, 65), (17, 8192, 70), (20, 9001, 33),
         (257, 384, 1023), (866, 768, 700), (1300, 96, 2050), (2100, 130, 1030)]


@pytest.mark.parametrize("t", ["f16", "bf16"])
@pytest.mark.parametrize("m,k,h", SIZES)
def test_forward(rt, rng, m, k, h, t):
    for act, bias in ((vh.VK_GATE_SILU, True), (vh.VK_GATE_GELU, False)):
        x, w, b = inputs(rng, m, k, h, t, bias)
        dx, dw, db = up(rt, t, x, w, b)
        out = rt.alloc(ff.DTYPE[t], m * h)
        rt.gated_forward(dx, dw, db, m, k, h, out, act)
        want, tol = ff.forward(x, w, b, act, t)
        ff.assert_within(rt.download_16(out), want, tol, (m, k, h, act))


BACK = [(1, 64, 64), (1, 8, 1), (2, 1344, 688), (8651, 64, 64), (40, 2881, 65), (281, 241, 3330),
        (3, 17, 5), (31, 136, 33), (64, 64, 32), (65, 96, 63), (70, 257, 65),
        (130, 384, 129), (257, 384, 1023), (866, 256, 300), (1300, 96, 2050), (2100, 520, 130)]


@pytest.mark.parametrize("t", ["f16", "bf16"])
@pytest.mark.parametrize("m,k,h", BACK)
def test_backward(rt, rng, m, k, h, t):
    for act, bias in ((vh.VK_GATE_SILU, True), (vh.VK_GATE_GELU, False)):
        x, w, b = inputs(rng, m, k, h, t, bias)
        grad = ff.rounded(rng.standard_normal((m, h)) * 0.1, t)
        dx, dw, db, dg = up(rt, t, x, w, b, grad)
        out = {n: rt.alloc(ff.DTYPE[t], s) for n, s in
               (("dx", m * k), ("dw", 2 * h * k), ("dbias", 2 * h))}
        rt.gated_backward(dx, dw, db, dg, m, k, h, out["dx"], out["dw"], out["dbias"], act)
        for n, (want, tol) in ff.backward(x, w, b, grad, act, t).items():
            ff.assert_within(rt.download_16(out[n]), want, tol, (n, m, k, h, act))


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("m,k,h,t", [(3, 24, 9, "f16"), (90, 40, 50, "bf16"), (65, 2100, 3, "f16")])
def test_gradients_are_slopes(rt, rng, m, k, h, t, act):
    """Against differences of the 64-bit forward, value by value of each input."""
    x, w, b = inputs(rng, m, k, h, t)
    grad = ff.rounded(rng.standard_normal((m, h)), t)
    o = {"dx": rt.alloc(ff.DTYPE[t], m * k), "dw": rt.alloc(ff.DTYPE[t], 2 * h * k),
         "dbias": rt.alloc(ff.DTYPE[t], 2 * h)}
    rt.gated_backward(*up(rt, t, x, w, b, grad), m, k, h, o["dx"], o["dw"], o["dbias"], act)
    tol = {n: e for n, (_, e) in ff.backward(x, w, b, grad, act, t).items()}
    at = {"dx": x, "dw": w, "dbias": b}
    for name, got in o.items():
        got = rt.download_16(got).reshape(at[name].shape)
        for i in rng.choice(got.size, min(got.size, 12), replace=False):
            def loss(s):
                v = {n: a.astype(np.float64) for n, a in at.items()}
                v[name].flat[i] += s
                y = v["dx"] @ v["dw"].T + v["dbias"]
                return float((grad * ff.activation(y[:, :h], act)[0] * y[:, h:]).sum())

            want, off = ff.slope(loss)
            assert abs(got.flat[i] - want) <= tol[name].flat[i] + off, (name, i)


def steps(rt, rng, sizes, t="bf16"):
    """Forward and backward of each size: [(what enqueues it, its outputs)]; step(True) takes other
    inputs, for outputs that hold something else."""
    out = []
    for m, k, h in sizes:
        a, other = (up(rt, t, *inputs(rng, m, k, h, t),
                       ff.rounded(rng.standard_normal((m, h)), t)) for _ in "ab")
        o = [rt.alloc(ff.DTYPE[t], s) for s in (m * h, m * k, 2 * h * k, 2 * h)]

        def step(dirty=False, a=a, other=other, o=o, m=m, k=k, h=h):
            v = other if dirty else a
            rt.gated_forward(*v[:3], m, k, h, o[0])
            rt.gated_backward(*v, m, k, h, *o[1:])
        out.append((step, o))
    return out


def bits(rt, o):
    rt.synchronize()
    return [rt.download_16(v) for v in o]


# products whose k several workgroups share, among others
SHARED = [(70, 4000, 64), (2048, 72, 40), (40, 2881, 65), (130, 384, 129)]


def test_the_same_bits_from_shared_products(rt, rng):
    """Whoever arrives last adds the parts in their order, and leaves the counters as they were."""
    calls = steps(rt, rng, SHARED)
    for step, _ in calls:
        step()
    want = [bits(rt, o) for _, o in calls]
    for i in range(12):
        for step, _ in calls[i % 2::2] if i % 3 else calls:
            step(True)
            step()
        for (_, o), w in zip(calls, want):
            for p, q in zip(bits(rt, o), w):
                np.testing.assert_array_equal(p, q)


def test_two_runtimes_side_by_side(rng):
    """Each its stream, work buffer and counters; their calls queued together."""
    a, b = vh.Runtime(0), vh.Runtime(0)
    calls = [(r, *c) for pair in zip(steps(a, rng, SHARED), steps(b, rng, SHARED))
             for r, c in zip((a, b), pair)]
    for _, step, _ in calls:
        step()
    want = [bits(r, o) for r, _, o in calls]
    for _ in range(4):
        for _, step, _ in calls:
            step()
    for (r, _, o), w in zip(calls, want):
        for p, q in zip(bits(r, o), w):
            np.testing.assert_array_equal(p, q)


def test_graphs_outlive_a_larger_work_buffer(rng):
    """A capture that would have to grow the work buffer is refused; captured after an eager call,
    graphs give the same bits while eager calls grow and fill the buffer."""
    rt = vh.Runtime(0)
    calls = steps(rt, rng, SHARED)
    big, out = steps(rt, rng, [(4000, 1031, 2048)])[0]  # more than the first buffer's 32 MiB

    def refused():
        with pytest.raises(vh.VestraError):
            big()

    for step, _ in calls:
        step()
    want = [bits(rt, o) for _, o in calls]
    graphs = [cached.captured(rt, step) for step, _ in calls]
    cached.captured(rt, refused)
    big()
    first = bits(rt, out)
    for _ in range(3):
        for step, _ in calls:
            step(True)
        for g in graphs:
            g.launch()
        big()
        for (_, o), w in zip(calls, want):
            for p, q in zip(bits(rt, o), w):
                np.testing.assert_array_equal(p, q)
        for p, q in zip(bits(rt, out), first):
            np.testing.assert_array_equal(p, q)


def test_gradients_one_at_a_time(rt, rng):
    """Each alone gives the bits of all together, and the same call the same bits."""
    m, k, h, t = 200, 130, 70, "bf16"
    x, w, b = inputs(rng, m, k, h, t)
    grad = ff.rounded(rng.standard_normal((m, h)), t)
    a = up(rt, t, x, w, b, grad)
    sizes = (m * k, 2 * h * k, 2 * h)

    def call(wanted):
        o = [rt.alloc(vh.VK_BF16, s) if i in wanted else None for i, s in enumerate(sizes)]
        rt.gated_backward(*a, m, k, h, *o)
        return [None if v is None else rt.download_16(v) for v in o]

    every = call((0, 1, 2))
    for i in range(3):
        np.testing.assert_array_equal(call((i,))[i], every[i])
    for p, q in zip(every, call((0, 1, 2))):
        np.testing.assert_array_equal(p, q)


@pytest.mark.parametrize("act", ACTS)
def test_extremes_of_the_gate(rt, act):
    """Gates far out on both sides, infinities and NaN in one row alone."""
    k, h, t = 8, 40, "bf16"
    x = np.zeros((50, k), np.float32)
    x[:, 0] = ff.rounded(np.linspace(-300, 300, 50), t)
    x[:, 1] = 1
    x[10, 2], x[11, 2], x[12, 2] = np.inf, -np.inf, np.nan
    w = np.zeros((2 * h, k), np.float32)
    w[:h, 0], w[h:, 1], w[:, 2] = 1, 1, 1
    dx, dw = up(rt, t, x, w)
    out = rt.alloc(vh.VK_BF16, 50 * h)
    rt.gated_forward(dx, dw, None, 50, k, h, out, act)
    got = rt.download_16(out).reshape(50, h)
    assert np.isnan(got[11:13]).all() and (got[10] == np.inf).all()
    fine = np.r_[0:10, 13:50]
    want, tol = ff.forward(x[fine], w, None, act, t)
    ff.assert_within(got[fine], want, tol, "rows")


def test_a_row_of_nan_stays_in_its_row_of_dx(rt, rng):
    m, k, h, t = 90, 40, 24, "bf16"
    x, w, b = inputs(rng, m, k, h, t)
    grad = ff.rounded(rng.standard_normal((m, h)), t)
    a = up(rt, t, x, w, b, grad)
    clean, dirty = rt.alloc(vh.VK_BF16, m * k), rt.alloc(vh.VK_BF16, m * k)
    rt.gated_backward(*a, m, k, h, clean, None, None)
    x[33] = np.nan
    a[0] = ff.upload(rt, x, t)
    rt.gated_backward(*a, m, k, h, dirty, None, None)
    p, q = (rt.download_16(v).reshape(m, k) for v in (clean, dirty))
    assert np.isnan(q[33]).all()
    q[33] = p[33]
    np.testing.assert_array_equal(p, q)


def test_what_the_work_buffer_held_does_not_show(rt, rng):
    """The buffer full of NaN before the call: padding is written, not assumed."""
    m, k, h, t = 77, 37, 21, "bf16"
    x, w, b = inputs(rng, m, k, h, t)
    grad = ff.rounded(rng.standard_normal((m, h)), t)
    a = up(rt, t, x, w, b, grad)
    o = [rt.alloc(vh.VK_BF16, s) for s in (m * k, 2 * h * k, 2 * h)]
    big = [np.full((400, 300), np.nan, np.float32), np.full((600, 300), np.nan, np.float32)]
    bx, bw = up(rt, t, *big)
    bg = ff.upload(rt, np.full((400, 300), np.nan, np.float32), t)
    bo = [rt.alloc(vh.VK_BF16, s) for s in (400 * 300, 600 * 300, 600)]
    rt.gated_backward(bx, bw, None, bg, 400, 300, 300, *bo)
    rt.gated_backward(*a, m, k, h, *o)
    for (n, (want, tol)), got in zip(ff.backward(x, w, b, grad, vh.VK_GATE_SILU, t).items(), o):
        ff.assert_within(rt.download_16(got), want, tol, n)


def test_no_rows(rt, rng):
    _, w, b = inputs(rng, 1, 16, 8, "bf16")
    dw, db = up(rt, "bf16", w, b)
    none = rt.alloc(vh.VK_BF16, 0)
    rt.gated_forward(none, dw, db, 0, 16, 8, none)
    gw, gb = up(rt, "bf16", w, b)
    rt.gated_backward(none, dw, db, none, 0, 16, 8, none, gw, gb)
    assert not rt.download_16(gw).any() and not rt.download_16(gb).any()


def test_guard_values_stay(rt, rng):
    for m, k, h in ((3, 24, 17), (70, 40, 33), (300, 72, 1030)):
        x, w, b = inputs(rng, m, k, h, "bf16")
        grad = ff.rounded(rng.standard_normal((m, h)), "bf16")
        a = up(rt, "bf16", x, w, b, grad)
        rooms = [ff.upload(rt, np.full(s + 512, 7.0), "bf16")
                 for s in (m * h, m * k, 2 * h * k, 2 * h)]
        o = [r.view(256, len(r) - 512) for r in rooms]
        rt.gated_forward(*a[:3], m, k, h, o[0])
        rt.gated_backward(*a, m, k, h, *o[1:])
        for r in rooms:
            got = rt.download_16(r)
            assert (got[:256] == 7).all() and (got[-256:] == 7).all()


@pytest.mark.parametrize("m", [4, 300])
def test_captured(rt, rng, m):
    k, h, t = 136, 100, "bf16"
    x, w, b = inputs(rng, m, k, h, t)
    grad = ff.rounded(rng.standard_normal((m, h)), t)
    a = up(rt, t, x, w, b, grad)
    o = [rt.alloc(vh.VK_BF16, s) for s in (m * h, m * k, 2 * h * k, 2 * h)]

    def step():
        rt.gated_forward(*a[:3], m, k, h, o[0])
        rt.gated_backward(*a, m, k, h, *o[1:])

    step()
    want = [rt.download_16(v) for v in o]
    g = cached.captured(rt, step)
    for _ in range(3):
        for v in o:
            rt.gated_forward(*a[:3], m, k, h, o[0])
        g.launch()
        for v, e in zip(o, want):
            np.testing.assert_array_equal(rt.download_16(v), e)


def test_refusals(rt, rng):
    m, k, h = 4, 16, 8
    x, w, b = up(rt, "bf16", *inputs(rng, m, k, h, "bf16"))
    out, grad = rt.alloc(vh.VK_BF16, m * h), rt.alloc(vh.VK_BF16, m * h)
    room = rt.alloc(vh.VK_BF16, 4096)

    def refused(call, *a, code=vh.VK_ERR_INVALID):
        with pytest.raises(vh.VestraError) as e:
            call(*a)
        assert e.value.code == code, e.value

    refused(rt.gated_forward, rt.alloc_f32(m * k), w, b, m, k, h, out)
    refused(rt.gated_forward, rt.alloc(vh.VK_F16, m * k), w, b, m, k, h, out)  # two types
    refused(rt.gated_forward, x, w, b, m + 1, k, h, out)
    refused(rt.gated_forward, x, w, b, m, k, h + 1, out)
    refused(rt.gated_forward, x, w, b, m, k, h, out, 9)
    refused(rt.gated_forward, x, w, rt.alloc(vh.VK_BF16, h), m, k, h, out)
    refused(rt.gated_forward, room.view(0, m * k), w, b, m, k, h, room.view(32, m * h))
    refused(rt.gated_forward, room.view(1, m * k), w, b, m, k, h, out)
    refused(rt.gated_backward, x, w, b, grad, m, k, h, None, None, None)
    refused(rt.gated_backward, x, w, b, grad, m, k, h, rt.alloc(vh.VK_BF16, 1), None, None)
    refused(rt.gated_backward, x, w, b, grad, m, k, h, None, None, room.view(0, 2 * h + 1))
    refused(rt.gated_backward, x, w, b, grad, m, k, h, x, None, None)
    refused(rt.gated_backward, x, w, b, grad, m, k, h, room.view(0, m * k),
            room.view(32, 2 * h * k), None)
    rt.gated_forward(x, w, b, m, k, h, out)  # and still runs
    rt.synchronize()


@pytest.mark.parametrize("act", ACTS)
def test_the_feed_forward_of_a_block(rt, rng, act):
    """LayerNorm, the gated layer and the way back to the residual stream, in 8 bits and in
    16, from the same weights: each step from what the step before gave."""
    m, d, h = 140, 96, 250
    tok = rng.standard_normal((m, d)).astype(np.float32)
    w12 = rng.standard_normal((2 * h, d)).astype(np.float32) * np.float32(1.5 * d ** -0.5)
    w3 = rng.standard_normal((d, h)).astype(np.float32) * np.float32(h ** -0.5)
    b12, b3, ls = (rng.standard_normal(n).astype(np.float32) * np.float32(0.1)
                   for n in (2 * h, d, d))
    gamma, beta = np.ones(d, np.float32), np.zeros(d, np.float32)
    tokens, ln = rt.upload_f32(tok), rt.alloc_f32(m * d)
    rt.layernorm_into_f32(tokens, rt.upload_f32(gamma), rt.upload_f32(beta), m, d, 1e-6, ln)
    x = ln.numpy().reshape(m, d)

    # 8 bits
    up8, down8 = (rt.prepare_linear_i8_f32(k, n, wt.T.copy(), bias, g) for k, n, wt, bias, g in
                  ((d, 2 * h, w12, b12, None), (h, d, w3, b3, ls)))
    hid = rt.alloc(vh.VK_BF16, m * h)
    up8.run_gated(ln, m, hid, act)
    down8.run_residual(hid, m, tokens)
    codes, s = ff.quantised(w12)
    y, tol = ff.linear(x, codes, s, b12, None)
    want, tol = ff.gated(y[:, :h], y[:, h:], tol[:, :h], tol[:, h:], act)
    mid = rt.download_16(hid).reshape(m, h)
    ff.assert_within(mid, want, ff.held(want, tol, "bf16"), "gated")
    codes, s = ff.quantised(w3)
    y, tol = ff.linear(mid, codes, s, b3, ls)
    ff.assert_within(tokens.numpy(), tok + y, tol + 1.01 * ff.U * np.abs(tok + y), "residual")

    # 16 bits, the gated layer's step of training after it
    x16, w16, b16 = (ff.rounded(v, "bf16") for v in (x, w12, b12))
    dx, dw, db = up(rt, "bf16", x16, w16, b16)
    rt.gated_forward(dx, dw, db, m, d, h, hid, act)
    h16, th = ff.forward(x16, w16, b16, act, "bf16")
    ff.assert_within(rt.download_16(hid), h16, th, "16 bits")
    # and the two agree as far as 8 bits go: a code is off by at most half a scale
    c, sx = ff.quantised(x)
    assert np.linalg.norm(mid - h16) < 0.03 * np.linalg.norm(h16)
    grad = ff.rounded(rng.standard_normal((m, h)), "bf16")
    o = [rt.alloc(vh.VK_BF16, n) for n in (m * d, 2 * h * d, 2 * h)]
    rt.gated_backward(dx, dw, db, ff.upload(rt, grad, "bf16"), m, d, h, *o, act)
    for (n, (want, tol)), got in zip(ff.backward(x16, w16, b16, grad, act, "bf16").items(), o):
        ff.assert_within(rt.download_16(got), want, tol, n)
