"""Rotary positions of several axes with the Q/K LayerNorm, vk_qk_norm_rope_axes_f32,
against the formula in 64 bits and against the 2D entry points.

Bound: a rotated value is x c + y s of LayerNorm'd values x, y: each is off by 8 u of
its LayerNorm terms |gamma| (|x| + |mean|) inv + |beta| (mean and variance of 64 values:
a tree of 10 roundings, rms below 4 u; v_rsq_f32 1 ulp; three roundings) and cos and sin
by 2 u; two products and a sum: 16 u of both values' terms covers them.  To it comes the
angle's own error, |p f| 2^-50 (both sides' powers, products and the quotient by 2 pi).
"""
import numpy as np
import pytest

import cached
from test_gpu_patch_block import normals

pytestmark = pytest.mark.gpu

vh = pytest.importorskip("vestra_hip")

U = cached.U


def pairs_of(pairs, freq, sections, interleaved, exp_head):
    """(first, second, axis, frequency) of the 32 pairs, from the header's words."""
    out, base, j = [], 0, 0
    for a, p in enumerate(pairs):
        for i in range(p):
            if sections:
                e = (2 * j, 2 * j + 1) if interleaved else (j, j + 32)
                f = float(freq) ** (-2.0 * j / 64)
            else:
                e = (base + 2 * i, base + 2 * i + 1) if interleaved else (base + i, base + i + p)
                f = float(freq) ** (-2.0 * i / (64 if exp_head else 2 * p))
            out.append((*e, a, f))
            j += 1
        base += 2 * p
    return out


def reference(x, g, b, eps, pos, spec):
    """x [..., rows, 64] in 64 bits, and the bound."""
    x = x.astype(np.float64)
    size = np.abs(x)
    if g is not None:
        m = x.mean(-1, keepdims=True)
        inv = 1 / np.sqrt(((x - m) ** 2).mean(-1, keepdims=True) + eps)
        size = (np.abs(x) + np.abs(m)) * inv * np.abs(g.astype(np.float64)) + np.abs(b.astype(np.float64))
        x = (x - m) * inv * g.astype(np.float64) + b.astype(np.float64)
    y, tol = np.empty_like(x), np.empty_like(x)
    for e0, e1, a, f in spec:
        p = pos[:, a].astype(np.float64)
        c, s = np.cos(p * f), np.sin(p * f)
        y[..., e0] = x[..., e0] * c - x[..., e1] * s
        y[..., e1] = x[..., e1] * c + x[..., e0] * s
        both = size[..., e0] + size[..., e1]
        tol[..., e0] = tol[..., e1] = both * (16 * U + np.abs(p * f) * 2.0 ** -50)
    return y, tol + 1e-40


def run(rt, q, k, params, pos, axes, eps=1e-5, sequences=1, layout=0, in_place=False):
    H, KV = q.shape[1], 0 if k is None else k.shape[1]
    n = q.shape[2]
    lay = cached.heads_outer if layout == vh.VK_QK_HEADS_OUTER else (lambda x: x)
    up = {np.dtype(np.float32): rt.upload_f32, np.dtype(np.float16): rt.upload_f16,
          np.dtype(np.int32): rt.upload_i32, np.dtype(np.int64): rt.upload_i64}
    qd, kd = rt.upload_f32(lay(q)), None if k is None else rt.upload_f32(lay(k))
    qo = qd if in_place else rt.alloc_f32(q.size)
    ko = kd if in_place or k is None else rt.alloc_f32(k.size)
    pd = [None if p is None else up[p.dtype](p) for p in params]
    rt.qk_norm_rope_axes_f32(qd, kd, *pd, up[pos.dtype](pos), H, KV, n, axes, eps, qo, ko, sequences,
                             layout)
    back = [None if t is None else lay(t.numpy().reshape(lay(x).shape)) for t, x in ((qo, q), (ko, k))]
    return back


def params_of(rng, kind):
    if kind is None:
        return [None] * 4
    g = [normals(rng, 64, scale=0.3, shift=1), normals(rng, 64, scale=0.3),
         normals(rng, 64, scale=0.3, shift=1), normals(rng, 64, scale=0.3)]
    return [x.astype(kind) for x in g]


def check(got, x, g, b, pos, spec, eps=1e-5):
    S, H, n, _ = x.shape
    for s in range(S):
        want, tol = reference(x[s], g, b, eps, pos[s * n:(s + 1) * n], spec)
        off = np.abs(got[s] - want)
        assert np.all(off <= tol), (np.max(off / tol), s)


CONVENTIONS = [(False, False, False), (False, True, False), (False, False, True),
               (False, True, True), (True, False, False), (True, True, False)]


@pytest.mark.parametrize("sections,interleaved,exp_head", CONVENTIONS)
@pytest.mark.parametrize("pairs", [(32,), (16, 16), (8, 12, 12), (5, 0, 27), (1, 2, 3, 26)])
def test_conventions(rt, rng, sections, interleaved, exp_head, pairs):
    S, H, KV, n = 1, 3, 2, 21
    q, k = normals(rng, S, H, n, 64), normals(rng, S, KV, n, 64)
    pos = rng.integers(-40, 1000, (n, len(pairs))).astype(np.int32)
    p = params_of(rng, np.float32)
    spec = pairs_of(pairs, 100.0, sections, interleaved, exp_head)
    axes = vh.RopeAxes(pairs, 100.0, sections, interleaved, exp_head)
    qo, ko = run(rt, q, k, p, pos, axes)
    check(qo, q, p[0], p[1], pos, spec)
    check(ko, k, p[2], p[3], pos, spec)


@pytest.mark.parametrize("S,H,KV,n", [(1, 1, 0, 1), (1, 12, 12, 15), (1, 16, 4, 17), (3, 5, 7, 33),
                                      (7, 2, 1, 1), (2, 12, 12, 866)])
@pytest.mark.parametrize("layout", [0, 1])
@pytest.mark.parametrize("kind", [None, np.float32, np.float16])
@pytest.mark.parametrize("in_place", [False, True])
def test_shapes(rt, rng, S, H, KV, n, layout, kind, in_place):
    q, k = normals(rng, S, H, n, 64), normals(rng, S, KV, n, 64) if KV else None
    pos = rng.integers(0, 60, (S * n, 3)).astype(np.int64)
    p = params_of(rng, kind)
    if not KV:
        p = p[:2] + [None, None]
    spec = pairs_of((8, 12, 12), 100.0, False, False, False)
    qo, ko = run(rt, q, k, p, pos, vh.RopeAxes((8, 12, 12)), sequences=S, layout=layout,
                 in_place=in_place)
    check(qo, q, p[0], p[1], pos, spec)
    if KV:
        check(ko, k, p[2], p[3], pos, spec)


@pytest.mark.parametrize("dtype", [np.int32, np.int64, np.float32])
def test_far_positions(rt, rng, dtype):
    n = 40
    far = np.array([0, 1, -1, 1023, 1024, 2 ** 20 + 3, 2 ** 30 + 7, 2 ** 31 - 1, -2 ** 31, 12345678])
    pos = rng.choice(far, (n, 3))
    pos = pos.astype(dtype)
    if dtype == np.int64:
        pos[0] = 2 ** 40 + 12345
    if dtype == np.float32:
        pos[:8] = normals(rng, 8, 3, scale=30)  # fractions count
    q = normals(rng, 1, 4, n, 64)
    spec = pairs_of((8, 12, 12), 10000.0, True, False, False)
    qo, _ = run(rt, q, None, [None] * 4, pos, vh.RopeAxes((8, 12, 12), 10000.0, sections=True))
    check(qo, q, None, None, pos, spec)


@pytest.mark.parametrize("interleaved", [False, True])
def test_two_axes_are_the_2d_form(rt, rng, interleaved):
    """Equal to vk_qk_norm_rope_mode_f32 within twice the bound (its angle is an f32
    product: positions up to 60, where that is off by 60 u a turn)."""
    H, n = 4, 50
    q, k = normals(rng, 1, H, n, 64), normals(rng, 1, H, n, 64)
    pos = rng.integers(0, 60, (n, 2)).astype(np.int32)
    p = params_of(rng, np.float32)
    qo, ko = run(rt, q, k, p, pos, vh.RopeAxes((16, 16), 100.0, interleaved=interleaved))
    qd, kd = rt.upload_f32(q), rt.upload_f32(k)
    rt.qk_norm_rope_mode_f32(qd, kd, *[rt.upload_f32(x) for x in p], rt.upload_i32(pos), H, n, 100.0,
                             1e-5, vh.VK_ROPE_INTERLEAVED if interleaved else 0)
    spec = pairs_of((16, 16), 100.0, False, interleaved, False)
    for got, old, x, g, b in ((qo, qd, q, p[0], p[1]), (ko, kd, k, p[2], p[3])):
        _, tol = reference(x, g, b, 1e-5, pos, spec)
        assert np.all(np.abs(got - old.numpy().reshape(got.shape)) <= 2 * tol + 128 * U * np.abs(x).max())


def test_the_sequential_order_gives_the_cpu_sums(rt, rng):
    """With no rotation (positions 0) the rows are the runtime's LayerNorm in either order:
    the sequential one bit for bit the left-to-right sums in f32."""
    H, n = 3, 19
    q, k = normals(rng, 1, H, n, 64, scale=3, shift=1), normals(rng, 1, H, n, 64)
    p = params_of(rng, np.float32)
    pos = np.zeros((n, 3), np.int32)
    rt.set_layernorm_order(vh.VK_LN_ORDER_SEQUENTIAL)
    try:
        got = run(rt, q, k, p, pos, vh.RopeAxes((8, 12, 12)))
    finally:
        rt.set_layernorm_order(vh.VK_LN_ORDER_TREE)
    f = np.float32
    for y, x, g, b in ((got[0], q, p[0], p[1]), (got[1], k, p[2], p[3])):
        for h in range(H):
            for i in range(n):
                s = f(0)
                for e in x[0, h, i]:
                    s = f(s + e)
                mean = f(s / f(64))
                d = (x[0, h, i] - mean).astype(f)
                s = f(0)
                for e in (d * d).astype(f):
                    s = f(s + e)
                inv = f(f(1) / np.sqrt(f(f(s / f(64)) + f(1e-5))))
                want = ((d * inv).astype(f) * g).astype(f) + b
                assert np.array_equal(y[0, h, i], want.astype(f))


@pytest.mark.parametrize("S,H,KV,n", [(2, 3, 2, 17), (1, 12, 12, 50), (3, 1, 0, 1)])
@pytest.mark.parametrize("layout", [0, 1])
@pytest.mark.parametrize("kind", [np.float32, np.float16])
def test_the_sequential_order_at_real_positions(rt, rng, S, H, KV, n, layout, kind):
    """The rotation of rows whose LayerNorm is the left-to-right sums in f32.  Beside those,
    which are the kernel's own bits, cos and sin are off by 2 u and half a u of the reduced
    angle, each product and the sum by u: 5 u of both values, and the angle's own error."""
    f = np.float32
    pairs, freq = (8, 12, 12), 100.0
    q, k = normals(rng, S, H, n, 64, scale=3, shift=1), normals(rng, S, KV, n, 64) if KV else None
    p = params_of(rng, kind)
    if not KV:
        p = p[:2] + [None, None]
    pos = rng.integers(-30, 3000, (S * n, 3)).astype(np.int32)
    spec = pairs_of(pairs, freq, False, False, False)
    rt.set_layernorm_order(vh.VK_LN_ORDER_SEQUENTIAL)
    try:
        got = run(rt, q, k, p, pos, vh.RopeAxes(pairs, freq), sequences=S, layout=layout)
    finally:
        rt.set_layernorm_order(vh.VK_LN_ORDER_TREE)
    for y, x, g, b in ((got[0], q, p[0], p[1]), (got[1], k, p[2], p[3])):
        if x is None:
            continue
        mean = np.add.accumulate(x, -1, f)[..., -1:] / f(64)
        d = x - mean
        var = np.add.accumulate(d * d, -1, f)[..., -1:] / f(64)
        x = (d * (f(1) / np.sqrt(var + f(1e-5)))) * g.astype(f) + b.astype(f)
        assert x.dtype == f
        for s in range(S):
            at = pos[s * n:(s + 1) * n]
            want, _ = reference(x[s], None, None, 0.0, at, spec)
            for e0, e1, a, w in spec:
                both = np.abs(x[s, ..., e0].astype(np.float64)) + np.abs(x[s, ..., e1])
                tol = both * (5 * U + np.abs(at[:, a] * w) * 2.0 ** -50) + 1e-40
                for e in (e0, e1):
                    assert np.all(np.abs(y[s, ..., e] - want[..., e]) <= tol)


def test_refusals(rt):
    n = 4
    q, k, o = (rt.alloc_f32(2 * n * 64) for _ in range(3))
    o2 = rt.alloc_f32(len(q))
    pos = rt.upload_i32(np.zeros(3 * n, np.int32))
    g = [rt.upload_f32(np.ones(64)) for _ in range(4)]
    axes = vh.RopeAxes((8, 12, 12))

    def call(q=q, k=k, g=g, pos=pos, heads=2, kv=2, n=n, axes=axes, qo=o, ko=o2, layout=0):
        rt.qk_norm_rope_axes_f32(q, k, *g, pos, heads, kv, n, axes, 1e-5, qo, ko, 1, layout)

    call()
    call(qo=q, ko=k)
    both = rt.alloc_f32(3 * n * 64)
    bad = [dict(axes=vh.RopeAxes((8, 12, 11))), dict(axes=vh.RopeAxes((8, 12, 12), -1.0)),
           dict(axes=vh.RopeAxes((8, 12, 12), float("nan"))), dict(layout=2), dict(kv=0),
           dict(k=None), dict(ko=None), dict(heads=0), dict(heads=3), dict(n=5),
           dict(pos=rt.upload_f32(np.zeros(2 * n))), dict(g=[None] + g[1:]), dict(g=g[:3] + [None]),
           dict(g=g[:3] + [rt.upload_f16(np.ones(64))]), dict(g=g[:3] + [rt.upload_f32(np.ones(63))]),
           dict(qo=o, ko=o), dict(qo=k), dict(qo=q, k=q, ko=o2), dict(ko=q),
           dict(q=both.view(0, len(q)), qo=both.view(64, len(q)))]
    for args in bad:
        with pytest.raises(vh.VestraError) as e:
            call(**args)
        assert e.value.code == vh.VK_ERR_INVALID, args
    flags = vh.RopeAxes((8, 12, 12))
    flags.struct.mode = 8
    with pytest.raises(vh.VestraError):
        call(axes=flags)
    with pytest.raises(vh.VestraError):
        vh.RopeAxes((8, 8, 8, 4, 4))
    rt.synchronize()
