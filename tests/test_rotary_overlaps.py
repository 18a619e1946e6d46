"""Rotary positions in place refuse views whose elements are written twice, by themselves or as q and k, and take those that only
lie between each other's rows. Checked at the C ABI against a count of the elements, without a GPU: calls that pass
the checks fail at the launch."""
import ctypes
import itertools
import random

import numpy as np
import pytest
import torch

from sffft_amd import mixers

NULL = ctypes.c_void_p(0)
EINVAL = 1
BASE = 1 << 40
pytestmark = pytest.mark.skipif(torch.cuda.is_available(), reason="addresses that no kernel may follow")


def apply(B, T, H, Hk, D, sq, sk, gap, qo=None, ko=None):
    """Whether the call passes: q at BASE, k `gap` elements behind it, in place unless qo or ko (elements, strides) say otherwise."""
    p = mixers.Rotary(0, B, T, H, Hk, D, 2, 0, 0, 10, 32)
    qo, ko = qo or (0, sq), ko or (gap, sk)
    for n, s in (("q", sq), ("k", sk), ("qo", qo[1]), ("ko", ko[1])):
        setattr(p, n, (ctypes.c_longlong * 3)(*s))
    at = [ctypes.c_void_p(BASE + 4 * e) for e in (0, gap, qo[0], ko[0])]
    if not Hk:
        at[1] = at[3] = NULL
    return mixers.lib().sffft_rotary_apply(p, at[0], at[1], ctypes.c_void_p(1 << 50), NULL, at[2], at[3], NULL) != EINVAL


def elements(B, T, H, D, s, at=0):
    """Every element that a view touches, twice if it is touched twice."""
    n = np.arange
    return (at + n(B)[:, None, None, None] * s[0] + n(T)[:, None, None] * s[1] + n(H)[:, None] * s[2] + n(D)).ravel()


def twice(*views):
    e = np.concatenate(views)
    return len(np.unique(e)) != len(e)


USUAL = [  # B, T, H, Hk, D, q's strides, k's, k's place: what models have
    (2, 5, 4, 2, 8, (5 * 8 * 8, 64, 8), (5 * 8 * 8, 64, 8), 32),           # parts of a fused projection, fewer key heads
    (2, 5, 4, 4, 8, (5 * 96, 96, 8), (5 * 96, 96, 8), 32),
    (2, 5, 4, 4, 8, (320, 8, 40), (320, 8, 40), 160),                       # head-major halves
    (2, 5, 1, 1, 8, (320, 8, 3), (320, 8, 5), 160),                         # one head: its stride does not count
    (1, 1, 4, 2, 8, (1, 1, 8), (7, 9, 8), 32),
    (2, 5, 4, 4, 8, (5 * 64, 64, 16), (5 * 64, 64, 16), 8),                 # heads of q and k by turns
    (2, 5, 4, 2, 8, (160, 32, 8), (80, 16, 8), 1000),                       # arrays of their own
    (2, 5, 4, 2, 8, (5 * 64, 64, 8), (5 * 64, 64, 16), 32),                 # keys and values by turns behind the queries
    (2, 5, 4, 2, 8, (5 * 64, 64, 8), (5 * 64, 64, 16), 40),
    (2, 1, 4, 1, 8, (64, 3, 8), (64, 7, 3), 32),                            # one token of each
]


@pytest.mark.parametrize("case", USUAL, ids=str)
def test_usual_views_pass(case):
    B, T, H, Hk, D, sq, sk, gap = case
    assert not twice(elements(B, T, H, D, sq), elements(B, T, Hk, D, sk, gap))
    assert apply(*case)


ALIASED = [
    (2, 5, 1, 0, 8, (8, 8, 8), (0, 0, 0), 0),                               # batches at the tokens' stride
    (1, 5, 3, 0, 8, (0, 8, 8), (0, 0, 0), 0),                               # heads at the tokens'
    (1, 5, 3, 0, 8, (0, 16, 8), (0, 0, 0), 0),                              # windows
    (1, 5, 3, 0, 8, (0, 4, 100), (0, 0, 0), 0),
    (2, 5, 4, 3, 8, (160, 32, 8), (160, 32, 8), 8),                         # k: q's heads from the second on
    (2, 5, 4, 4, 8, (160, 32, 8), (160, 32, 8), 4),
    (2, 5, 4, 2, 8, (5 * 64, 64, 8), (5 * 64, 64, 8), 24),                  # one head shared
    (2, 5, 4, 4, 8, (320, 64, 8), (160, 32, 8), 32),                        # between the rows, at other strides
    (2, 5, 4, 4, 8, (160, 32, 8), (160, 32, 8), 0),
]


@pytest.mark.parametrize("case", ALIASED, ids=str)
def test_aliased_views_are_refused(case):
    B, T, H, Hk, D, sq, sk, gap = case
    assert twice(elements(B, T, H, D, sq), elements(B, T, Hk, D, sk, gap))
    assert not apply(*case)


def test_no_aliased_view_passes():
    """Random small strides and places: whatever passes touches no element twice, and much does pass."""
    rng, passed = random.Random(1), 0
    for _ in range(20000):
        B, T, H, Hk, D = (rng.randint(1, 3), rng.randint(1, 4), rng.randint(1, 3), rng.randint(0, 3), rng.choice((2, 4)))
        sq = tuple(rng.choice((0, 1, 2, 4, 6, 8, 12, 16, 24, 32, 48, 64)) for _ in range(3))
        sk = sq if rng.random() < 0.8 else tuple(rng.choice((2, 4, 8, 16, 24, 48)) for _ in range(3))
        gap = rng.randint(0, 70)
        if apply(B, T, H, Hk, D, sq, sk, gap):
            passed += 1
            assert not twice(elements(B, T, H, D, sq), elements(B, T, Hk, D, sk, gap)), (B, T, H, Hk, D, sq, sk, gap)
    assert passed > 2000


def test_outputs_elsewhere():
    s = (160, 32, 8)
    assert apply(2, 5, 4, 4, 8, s, s, 1000, (5000, s), (9000, s))
    assert not apply(2, 5, 4, 4, 8, s, s, 1000, (5000, (160, 8, 8)), (9000, s))      # written twice
    assert not apply(2, 5, 4, 4, 8, s, s, 1000, (5000, s), (5016, s))                # over each other
    assert apply(2, 5, 4, 4, 8, s, s, 1000, (5000, (320, 64, 8)), (5032, (320, 64, 8)))  # halves of one array
    assert not apply(2, 5, 4, 3, 8, s, s, 8, None, (9000, s))                        # q in place over k, which is read
    assert not apply(2, 5, 4, 3, 8, s, s, 8, (9000, s), None)
    assert apply(2, 5, 4, 4, 8, (320, 64, 8), (320, 64, 8), 32, None, (9000, s))


def test_permutations_of_the_dimensions():
    for order in itertools.permutations(range(3)):
        n, s, span = (2, 3, 4), [0, 0, 0], 8
        for i in order:
            s[i], span = span, span * n[i]
        assert apply(2, 3, 4, 4, 8, tuple(s), tuple(s), span)
        s = [2 * x for x in s]
        assert apply(2, 3, 4, 4, 8, tuple(s), tuple(s), 8)
