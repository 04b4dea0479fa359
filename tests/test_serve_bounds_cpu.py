"""What the GPU tests of batched serving can see (serve_bounds.py), on the CPU: their bounds hold the two f16 terms of
an f16 cache and do not hold one."""
import numpy as np
import pytest

import serve_bounds as B


@pytest.mark.parametrize("scale", [1.0, 4.0])
@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("kernel", list(B.KERNELS))
def test_each_of_two_terms_is_needed(hd, kernel, scale):
    c, q, heads, floor = B.one_each(np.random.default_rng(hd), hd, kernel)
    want, bound = B.attention(c, q, heads, scale, roundings=8, floor=floor)
    hold = 14 if floor == B.FEW_FLOOR else 8
    for terms, inside in (((2, 2), True), ((1, 2), False), ((2, 1), False)):
        got = B.attention_in_terms(c, q, heads, scale, *terms, hold=hold)
        worst = np.max(np.abs(got - want) / bound)
        assert worst <= 1 if inside else worst > 3, (terms, worst)


@pytest.mark.parametrize("kernel", list(B.KERNELS))
def test_small_terms_are_off_by_a_part_of_the_largest(kernel):
    """A value far below its row's largest, and a weight far below its row's, are rounded to a step of the largest: by
    more than 2^-22 of themselves, by less than the floors."""
    c, q, heads, floor = B.one_large(np.random.default_rng(3), 64, kernel)
    want, bound = B.attention(c, q, heads, 1.0, floor=floor)
    hold = 14 if floor == B.FEW_FLOOR else 8
    assert np.all(np.abs(B.attention_in_terms(c, q, heads, 1.0, hold=hold) - want) <= bound)
    x = np.array([1.0, 1e-9 * 1.37])
    assert abs(B.terms(x * 2.0 ** 13, 2) / 2.0 ** 13 - x)[1] > 2.0 ** -22 * x[1]
    assert np.all(abs(B.terms(x * 2.0 ** 13, 2) / 2.0 ** 13 - x) <= 2.0 ** -22 * x + B.QUERY_FLOOR)
    w = 1.37 * 2.0 ** -16  # of the largest
    off = abs(B.terms(np.array([w * 2.0 ** hold]), 2)[0] / 2.0 ** hold - w)
    assert off <= 2.0 ** -22 * w + floor
    assert (off > 2.0 ** -22 * w) == (hold == 8)
