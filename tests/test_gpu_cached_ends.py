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
