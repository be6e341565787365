"""The 8-bit cache of K and V rows through the C ABI, against its definition in
numpy: the codes and scales bit for bit (both divisions are correctly rounded), and
what is read back (code * scale, one rounding)."""
import numpy as np
import pytest

import cached
from test_gpu_patch_block import normals

pytestmark = pytest.mark.gpu

vh = pytest.importorskip("vestra_hip")


def make(rt, fmt, S, H, cap, fill=0):
    c = rt.kv_cache(fmt, S, H, cap)
    n = S * H * cap
    c.k.write(np.full(n * 64, fill, np.uint8))
    c.v.write(np.full(n * 64, fill + 1, np.uint8))
    c.k_scale.write(np.full(n, 3, np.float32))
    c.v_scale.write(np.full(n, 5, np.float32))
    return c


def download(rt, c):
    def u8(t):
        out = np.empty(len(t), np.uint8)
        assert vh.lib.vk_download_u8(rt.handle, t.handle, out.ctypes.data, out.size) == 0
        return out
    shape = (c.sequences, c.heads, c.capacity)
    return (u8(c.k).reshape(*shape, 64), u8(c.v).reshape(*shape, 64),
            c.k_scale.numpy().reshape(shape), c.v_scale.numpy().reshape(shape))


def expect(c, before, k, v, n, starts, counts):
    """The cache after the write, k and v [S, H, n, 64]."""
    kc, vc, ks, vs = (x.copy() for x in before)
    for s in range(c.sequences):
        start, count = cached.spans(n, c.capacity, starts, counts, s)
        for i in range(count):
            if 0 <= start + i < c.capacity:
                kc[s, :, start + i], ks[s, :, start + i] = cached.quantise(k[s, :, i], c.format)
                vc[s, :, start + i], vs[s, :, start + i] = cached.quantise(v[s, :, i], c.format)
    return kc, vc, ks, vs


def same(got, want):
    for g, w, name in zip(got, want, ("k", "v", "k_scale", "v_scale")):
        assert np.array_equal(g, w, equal_nan=name.endswith("scale")), name


SHAPES = [  # S, H, cap, n, starts, counts
    (1, 1, 1, 1, None, None), (1, 12, 40, 37, [3], None), (3, 2, 65, 5, [0, 60, 31], [5, 5, 0]),
    (2, 16, 130, 129, None, [129, 17]), (5, 3, 7, 9, [0, -4, 6, 7, 2 ** 31 - 3], [9, 9, 3, 9, 9]),
    (2, 1, 4, 4, [-2 ** 31, 2], [4, -7]),
]


@pytest.mark.parametrize("fmt", [0, 1])
@pytest.mark.parametrize("outer", [0, 1])
@pytest.mark.parametrize("S,H,cap,n,starts,counts", SHAPES)
def test_write_and_read(rt, rng, fmt, outer, S, H, cap, n, starts, counts):
    k, v = normals(rng, S, H, n, 64, scale=1.5), normals(rng, S, H, n, 64)
    c = make(rt, fmt, S, H, cap)
    before = download(rt, c)
    lay = cached.heads_outer if outer == vh.VK_QK_HEADS_OUTER else (lambda x: x)
    st = None if starts is None else rt.upload_i32(np.array(starts, np.int32))
    ct = None if counts is None else rt.upload_i32(np.array(counts, np.int32))
    rt.kv_cache_write_f32(c, rt.upload_f32(lay(k)), rt.upload_f32(lay(v)), n, st, ct, outer)
    want = expect(c, before, k, v, n, starts, counts)
    same(download(rt, c), want)
    ko, vo = rt.upload_f32(np.full(k.size, 7)), rt.upload_f32(np.full(k.size, 9))
    rt.kv_cache_read_f32(c, n, st, ct, ko, vo, outer)
    for got, codes, scales, fill in ((ko, want[0], want[2], 7), (vo, want[1], want[3], 9)):
        held = cached.values(codes, scales, fmt).astype(np.float32)
        w = np.full(k.shape, fill, np.float32)
        for s in range(S):
            start, count = cached.spans(n, cap, starts, counts, s)
            for i in range(count):
                if 0 <= start + i < cap:
                    w[s, :, i] = held[s, :, start + i]
        assert np.array_equal(got.numpy(), lay(w).reshape(-1))


@pytest.mark.parametrize("fmt", [0, 1])
def test_rows_of_every_size(rt, rng, fmt):
    """Rows from the smallest numbers to the largest, zeros, borders between two codes,
    infinities and NaN."""
    sizes = 2.0 ** np.arange(-149, 128, 4.0)
    k = (normals(rng, len(sizes), 64).astype(np.float64) * sizes[:, None])
    k = np.clip(k, -3.4e38, 3.4e38).astype(np.float32)
    v = np.zeros_like(k)
    v[0, 3], v[1, 7], v[2, 9] = np.inf, -np.inf, np.nan
    v[3, 5], v[4] = -0.0, np.float32(2.0 ** -94)
    v[5] = np.float32(127 * 2.0 ** -100) if fmt == 0 else np.float32(448 * 2.0 ** -100)
    v[6] = np.nextafter(v[5], np.float32(0))
    v[7] = 3.4028235e38
    v[8] = np.arange(64) + 0.5  # with the largest below: ties between int8 codes
    v[8, 63] = 127.0
    v[9] = np.arange(64) * 0.4375 + 0.03125
    v[9, 0] = 448.0
    v[10:] = np.where(rng.random((len(sizes) - 10, 64)) < 0.5, k[10:], 0)
    n = len(sizes)
    c = make(rt, fmt, 1, 1, n)
    before = download(rt, c)
    rt.kv_cache_write_f32(c, rt.upload_f32(k), rt.upload_f32(v), n)
    want = expect(c, before, k[None, None], v[None, None], n, None, None)
    same(download(rt, c), want)
    vo = rt.alloc_f32(v.size)
    rt.kv_cache_read_f32(c, n, None, None, None, vo)
    got = vo.numpy().reshape(v.shape)
    assert np.isnan(got[:3]).all() and not np.isnan(got[3:]).any()
    # half a step of the row's scale (int8), or half a step of the value (e4m3: 2^-4; its
    # smallest step is 2^-9 of the scale)
    d = want[3][0, 0].astype(np.float64)[3:, None]
    off = np.abs(got[3:].astype(np.float64) - v[3:])
    step = 0.5 * d if fmt == 0 else np.maximum(2.0 ** -4 * np.abs(v[3:]), 2.0 ** -10 * d)
    assert np.all((off <= step * (1 + 2.0 ** -20)) | ((d == 0) & (np.abs(v[3:]) < 448 * 2.0 ** -99)))


def test_every_code_reads_back(rt):
    for fmt in (0, 1):
        c = make(rt, fmt, 1, 4, 1)
        codes = np.arange(256, dtype=np.uint8)
        c.k.write(codes)
        c.v.write(codes[::-1].copy())
        ko, vo = rt.alloc_f32(256), rt.alloc_f32(256)
        rt.kv_cache_read_f32(c, 1, None, None, ko, vo)
        for got, cc, d in ((ko, codes, 3.0), (vo, codes[::-1], 5.0)):
            want = cached.values(cc.reshape(4, 64), np.full(4, d, np.float32), fmt)
            assert np.array_equal(got.numpy(), want.astype(np.float32).reshape(-1), equal_nan=True)


def test_a_captured_step_follows_starts(rt, rng):
    """A captured write and read, replayed with other starts and inputs between."""
    S, H, cap, n = 2, 3, 20, 4
    c = make(rt, 0, S, H, cap)
    k, v = (rt.upload_f32(normals(rng, H, S, n, 64)) for _ in range(2))
    st = rt.upload_i32(np.zeros(S, np.int32))
    ko, vo = rt.alloc_f32(len(k)), rt.alloc_f32(len(k))
    rt.kv_cache_write_f32(c, k, v, n, st)
    rt.synchronize()
    graph = cached.captured(rt, lambda: (rt.kv_cache_write_f32(c, k, v, n, st),
                                         rt.kv_cache_read_f32(c, n, st, None, ko, vo)))
    want = download(rt, c)
    for step in range(4):
        starts = np.array([4 * step, 16 - 4 * step], np.int32)
        cached.set_i32(rt, st, starts)
        kh, vhost = normals(rng, S, H, n, 64), normals(rng, S, H, n, 64)
        k.write(cached.heads_outer(kh))
        v.write(cached.heads_outer(vhost))
        graph.launch()
        rt.synchronize()
        want = expect(c, want, kh, vhost, n, starts, None)
        same(download(rt, c), want)
        slots = np.stack([cached.values(want[0][s, :, a:a + n], want[2][s, :, a:a + n], 0)
                          for s, a in enumerate(starts)]).astype(np.float32)
        assert np.array_equal(ko.numpy(), cached.heads_outer(slots).reshape(-1))


def test_refusals(rt):
    c = rt.kv_cache(0, 2, 3, 8)
    k = rt.alloc_f32(2 * 3 * 4 * 64)
    v, out = rt.alloc_f32(len(k)), rt.alloc_f32(len(k))
    i2, i3 = rt.upload_i32(np.zeros(2, np.int32)), rt.upload_i32(np.zeros(3, np.int32))
    ok = dict(cache=c, k=k, v=v, n=4)
    rt.kv_cache_write_f32(**ok, starts=i2, counts=i2)
    bad = [dict(ok, n=3), dict(ok, starts=i3), dict(ok, counts=i3), dict(ok, layout=2),
           dict(ok, starts=c.k_scale.view(0, 2)), dict(ok, v=v.view(0, len(v) - 64)),
           dict(ok, k=rt.alloc_f32(len(k) + 1).view(1, len(k))),
           dict(ok, cache=vh.KvCache(2, 2, 3, 8, c.k, c.v, c.k_scale, c.v_scale)),
           dict(ok, cache=vh.KvCache(0, 2, 3, 8, c.k, c.k, c.k_scale, c.v_scale)),
           dict(ok, cache=vh.KvCache(0, 2, 3, 9, c.k, c.v, c.k_scale, c.v_scale)),
           dict(ok, cache=vh.KvCache(0, 2, 3, 8, c.k, c.v, c.v_scale, c.v_scale)),
           dict(ok, cache=vh.KvCache(0, 2, 3, 8, c.k, k, c.k_scale, c.v_scale)),
           dict(ok, cache=vh.KvCache(0, 0, 3, 8, c.k, c.v, c.k_scale, c.v_scale))]
    for args in bad:
        with pytest.raises(vh.VestraError) as e:
            rt.kv_cache_write_f32(**args)
        assert e.value.code == vh.VK_ERR_INVALID and e.value.message
    c.struct.head_dim = 128
    with pytest.raises(vh.UnsupportedShape):
        rt.kv_cache_write_f32(**ok)
    c.struct.head_dim = 64
    with pytest.raises(vh.VestraError):
        rt.kv_cache_read_f32(c, 4, None, None, None, None)
    with pytest.raises(vh.VestraError):
        rt.kv_cache_read_f32(c, 4, None, None, out, out)
    with pytest.raises(vh.VestraError):
        rt.kv_cache_read_f32(c, 3, None, None, out, v)
    # nothing to do
    rt.kv_cache_write_f32(c, rt.alloc_f32(0), rt.alloc_f32(0), 0)
    rt.synchronize()
