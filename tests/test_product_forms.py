"""The sizes whose values are checked take every form that the plan has for a card of 256 CUs."""
import random

import pytest

import product_forms as forms


def sizes(n, seed, top):
    rng = random.Random(seed)
    return [[int(2 ** rng.uniform(0, t)) for t in top] for _ in range(n)]


def union(form, tuples):
    return set().union(*(form(*s) for s in tuples))


def test_forward():
    assert union(forms.forward, sizes(20000, 1, (13.5, 13, 13))) <= \
        union(forms.forward, forms.FORWARD)


@pytest.mark.parametrize("t", ["bf16", "f16"])
def test_backward(t):
    def form(m, k, h):
        return forms.backward(m, k, h, t)

    assert union(form, sizes(30000, 2, (13.5, 12.6, 13))) <= union(form, forms.BACKWARD[t])
    assert all(m % 64 and h % 64 for m, _, h in forms.BACKWARD[t])


@pytest.mark.parametrize("gated", [False, True])
def test_linear_i8(gated):
    def form(m, k, n):
        return forms.linear_i8(m, k, n * (2 if gated else 1), gated)

    assert union(form, sizes(30000, 3, (13.5, 16, 13))) <= \
        union(form, forms.GATED_I8 if gated else forms.LINEAR_I8)
