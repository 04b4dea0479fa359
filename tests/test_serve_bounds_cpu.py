"""What the GPU tests of batched serving can see (serve_bounds.py), on the CPU: their bounds hold the two f16 terms of
an f16 cache and do not hold one, and no tile of positions can be left out or taken twice within them."""
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


@pytest.mark.parametrize("dtype,rows,heads", [("f16", [2], 4), ("f32", [2], 4), ("f16", [40], 4)])
def test_no_tile_can_be_left_out_or_taken_twice(dtype, rows, heads):
    """Every tile of 16 positions, and every position by itself, for the first row of the long cache."""
    c, q, value, want, tolerance = B.every_position(np.random.default_rng(1), dtype, rows, heads, 70001)
    n = c.row_positions()[0][1] + 1
    whole = np.stack([value[t:min(t + 16, n)].sum(0) for t in range(0, n, 16)])
    for part, size in ((whole, 16.0), (value[:n], 1.0)):
        for sign in (-1, 1):
            got = (value[:n].sum(0) + sign * part) / (n + sign * size)
            outside = np.abs(got - want[0, 0]) > tolerance[0, 0]
            assert outside.any(1).all()
