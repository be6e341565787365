"""The counters of sums that workgroups share: there once they are needed, and not before."""
import numpy as np
import pytest

import cached
import feed_forward as ff
import vestra_hip as vh

pytestmark = pytest.mark.gpu


def test_a_runtime_is_created_while_another_captures(rng):
    """Creating one allocates nothing, which a capturing thread could not."""
    a = vh.Runtime(0)
    x, y = a.upload_f32(rng.standard_normal(4096).astype(np.float32)), a.alloc_f32(4096)
    made = []

    def step():
        a.copy_segment_into_f32(y, 0, x, 0, 4096)
        made.append(vh.Runtime(0))

    g = cached.captured(a, step)
    for _ in range(2):
        x.write(rng.standard_normal(4096).astype(np.float32))
        g.launch()
        np.testing.assert_array_equal(y.numpy(), x.numpy())
    b = made[0]  # and it is one like any other
    w, t = ff.quantised(rng.standard_normal((70, 20000)).astype(np.float32))
    rows = rng.standard_normal((40, 20000)).astype(np.float32)
    out = b.alloc_f32(40 * 70)
    b.prepare_linear_i8(20000, 70, w.astype(np.int8), t).run_into(b.upload_f32(rows), 40, out)
    ff.assert_within(out.numpy(), *ff.linear(rows, w, t, None, None), "shared sums")


@pytest.mark.parametrize("first", ["work", "shared"])
def test_shared_sums_from_the_first_call_on(rng, first):
    """A fresh runtime whose work buffer comes with this call, or with another operation's."""
    rt = vh.Runtime(0)
    if first == "work":
        w, t = ff.quantised(rng.standard_normal((64, 64)).astype(np.float32))
        rt.prepare_linear_i8(64, 64, w.astype(np.int8), t).run_into(
            rt.upload_f32(np.zeros(200 * 64, np.float32)), 200, rt.alloc_f32(200 * 64))
    m, k, h, kind = 70, 4000, 64, "bf16"
    x, w = (ff.rounded(rng.standard_normal(s) * k ** -0.25, kind) for s in ((m, k), (2 * h, k)))
    out = rt.alloc(vh.VK_BF16, m * h)
    up = [ff.upload(rt, v, kind) for v in (x, w)]
    for _ in range(3):
        rt.gated_forward(*up, None, m, k, h, out)
        ff.assert_within(rt.download_16(out), *ff.forward(x, w, None, vh.VK_GATE_SILU, kind), first)
