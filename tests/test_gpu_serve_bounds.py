"""GPU tests of batched serving with inputs whose bounds are tight (serve_bounds.py; what they can see is shown in
test_serve_bounds_cpu.py)."""
import numpy as np
import pytest

import serve_bounds as B
from test_gpu_serve import attend

pytestmark = pytest.mark.gpu


def inside(got, want, bound, what):
    err = np.abs(got - want)
    bad = ~(err <= bound)
    print(f"{what}: {np.max(err / bound):.3g} of the bound", flush=True)
    assert not bad.any(), f"{what}: {bad.sum()} of {bad.size} outside, up to {np.nanmax(err / bound):.3g} times the bound"


# ------------------------------------------------------------------------- the two terms of an f16 cache

@pytest.mark.parametrize("scale", [1.0, 4.0])
@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("kernel", list(B.KERNELS))
def test_queries_and_weights_have_two_terms(hd, kernel, scale):
    """Scores of one product and results of one weight: nothing hides a term's rounding."""
    c, q, heads, floor = B.one_each(np.random.default_rng(hd), hd, kernel)
    want, bound = B.attention(c, q, heads, scale, roundings=8, floor=floor)
    inside(attend(c, q, heads, scale), want, bound, f"{kernel} queries of {hd}, scale {scale}")


@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("kernel", list(B.KERNELS))
def test_queries_with_one_large_value(hd, kernel):
    """The others are held as steps of the largest: off by 2^-39 of it."""
    c, q, heads, floor = B.one_large(np.random.default_rng(hd), hd, kernel)
    want, bound = B.attention(c, q, heads, 1.0, floor=floor)
    inside(attend(c, q, heads, 1.0), want, bound, f"{kernel} queries of {hd}")


@pytest.mark.parametrize("hd", [64, 256])
@pytest.mark.parametrize("kernel", list(B.KERNELS))
def test_keys_and_values_below_the_least_normal_f16(hd, kernel):
    """An f16 cache's subnormal numbers count as what they are."""
    c, q, heads, floor = B.one_each(np.random.default_rng(hd + 1), hd, kernel)
    for a, by in ((c.k, 2.0 ** -18), (c.v, 2.0 ** -20)):
        a[:] = (a.astype(np.float64) * by).astype(np.float16)
    assert 0 < np.abs(c.k[c.k != 0]).max() < 2.0 ** -14
    want, bound = B.attention(c, q, heads, 2.0 ** 18, roundings=8, floor=floor)
    inside(attend(c, q, heads, 2.0 ** 18), want, bound, f"{kernel} queries of {hd}")


# ------------------------------------------------------------------------- every tile of a long cache

@pytest.mark.parametrize("dtype,rows,heads,shared", [("f16", [2], 4, 0), ("f32", [2], 4, 0), ("f16", [40], 4, 0), ("f16", [10], 4, 0),
                                                     ("f32", [40], 4, 0), ("f16", [1] * 3, 4, 69500), ("f32", [1] * 3, 4, 69500),
                                                     ("f16", [2] * 20, 4, 69632)])
def test_every_position_of_a_long_cache_counts_once(dtype, rows, heads, shared):
    c, q, _, want, tolerance = B.every_position(np.random.default_rng(len(rows)), dtype, rows, heads, 70001, shared=shared)
    inside(attend(c, q, heads, 0.125, shared), want, tolerance + 1e-30, f"{dtype} {rows} shared {shared}")
