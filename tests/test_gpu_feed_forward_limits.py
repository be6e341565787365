"""Sizes past what a launch holds are refused before anything is allocated or looked at."""
import pytest

import vestra_hip as vh

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("m,k,h", [(1 << 24, 16, 1024), (1 << 23, 16, 2017), ((1 << 24) + 1, 16, 8),
                                   (4, (1 << 20) + 8, 8), (4, 8, (1 << 20) + 1),
                                   (4, 1 << 16, 1 << 13), (1 << 24, 1025, 8),
                                   (1 << 20, 16385, 8)])
def test_gated(rt, m, k, h):
    t = rt.alloc(vh.VK_BF16, 64)
    for call in (lambda: rt.gated_forward(t, t, None, m, k, h, t),
                 lambda: rt.gated_backward(t, t, None, t, m, k, h, t, None, None)):
        with pytest.raises(vh.VestraError) as e:
            call()
        assert e.value.code == vh.VK_ERR_UNSUPPORTED, e.value


def test_linear_i8(rt):
    """Less than 2^24 rows; as many outputs as a launch's tiles hold, of a wide linear."""
    import numpy as np
    n = 1 << 14
    lin = rt.prepare_linear_i8(8, n, np.ones((n, 8), np.int8), np.ones(n, np.float32))
    t = rt.alloc_f32(64)
    for rows in (1 << 24, (1 << 20) + 1, (1 << 64) - 1):
        with pytest.raises(vh.VestraError) as e:
            lin.run_into(t, rows, t)
        assert e.value.code in (vh.VK_ERR_UNSUPPORTED, vh.VK_ERR_INVALID), e.value
