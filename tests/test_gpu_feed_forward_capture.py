"""The feed-forward in fewer bits captured: replays on other inputs than the eager call's, into
outputs that hold something else; and which calls need the work buffer, which a capture cannot
grow."""
import ctypes

import numpy as np
import pytest

import cached
import feed_forward as ff
import product_forms as forms
import vestra_hip as vh

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("t", ["f16", "bf16"])
@pytest.mark.parametrize("m,k,h", [(4, 136, 100), (70, 4000, 64), (300, 131, 100), (1300, 96, 1000)])
def test_replays_compute(rt, rng, m, k, h, t):
    """The inputs change between replays; what a replay leaves is what an eager call on them leaves,
    and not what the outputs held."""
    dtype = ff.DTYPE[t]
    sizes = (m * k, 2 * h * k, 2 * h, m * h)
    held = [rt.alloc(dtype, n) for n in sizes]  # x, w, bias, grad: what the graph names
    o, eager = ([rt.alloc(dtype, n) for n in (m * h, m * k, 2 * h * k, 2 * h)] for _ in "oe")

    def put(scale):
        for v, n, s in zip(held, sizes, (1, k ** -0.5, 0.3, scale)):
            new = ff.upload(rt, ff.rounded(rng.standard_normal(n) * s, t), t)
            copy16(rt, v, new)

    def step(a, out):
        rt.gated_forward(*a[:3], m, k, h, out[0])
        rt.gated_backward(*a, m, k, h, *out[1:])

    put(0.1)
    step(held, o)
    graph = cached.captured(rt, lambda: step(held, o))
    for scale in (0.1, 1.0, 0.02):
        put(scale)
        junk = [ff.upload(rt, np.full(len(v), 3.0, np.float32), t) for v in o]
        for v, j in zip(o, junk):
            copy16(rt, v, j)
        graph.launch()
        step(held, eager)
        for p, q in zip(o, eager):
            p, q = rt.download_16(p), rt.download_16(q)
            np.testing.assert_array_equal(p, q)
            assert not (p == 3).all()


def copy16(rt, dst, src):
    """An even number of 16-bit values, as half as many f32."""
    n = len(dst) // 2
    assert len(dst) == 2 * n == len(src)
    views = []
    for v in (dst, src):
        handle = ctypes.c_void_p()
        assert vh.lib.vk_tensor_wrap(rt.handle, vh.VK_F32, v.device_ptr, n,
                                     ctypes.byref(handle)) == vh.VK_OK
        views.append(vh.Tensor(rt, handle))
    rt.copy_segment_into_f32(views[0], 0, views[1], 0, n)


@pytest.mark.parametrize("rows,k", [(15, 1090), (16, 1024), (16, 1025), (17, 64), (1, 16384),
                                    (1, 16385), (8, 2048), (8, 2000), (9, 1793)])
def test_which_rows_need_the_work_buffer(rng, rows, k):
    """16,384 bytes of codes, each row's rounded up to 128: up to there a first call may be a
    captured one; past it that is refused, and runs after an eager one."""
    rt = vh.Runtime(0)
    n = 40
    w, s = ff.quantised(rng.standard_normal((n, k)).astype(np.float32))
    lin = rt.prepare_linear_i8(k, n, w.astype(np.int8), s)
    x = rng.standard_normal((rows, k)).astype(np.float32)
    dx, y = rt.upload_f32(x), rt.alloc_f32(rows * n)
    needs = rows * -(-k // 128) * 128 > 16384 or rows > 16
    assert needs == (forms.linear_i8(rows, k, n) != {("own rows",)})

    def refused():
        with pytest.raises(vh.VestraError):
            lin.run_into(dx, rows, y)

    if needs:
        cached.captured(rt, refused)
        lin.run_into(dx, rows, y)
    graph = cached.captured(rt, lambda: lin.run_into(dx, rows, y))
    y.write(np.zeros(rows * n, np.float32))
    graph.launch()
    ff.assert_within(y.numpy(), *ff.linear(x, w, s, None, None), (rows, k))
