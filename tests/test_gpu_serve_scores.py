"""GPU tests of the paged attention with scores of any size (include/uq_serve.h): finite queries, keys and scales give
finite results, the softmax's limit where scores lie far apart."""
import numpy as np
import pytest

import serve_model as M
from test_gpu_serve import attend

pytestmark = pytest.mark.gpu

# heads of one KV head, rows, positions of the page table: 16, 32, 64 and 128 queries a block, and a block a workgroup
KERNELS = [(4, [1], 1 << 18), (24, [1], 1 << 18), (12, [4], 1 << 18), (20, [7], 1 << 18), (4, [3], 0)]


def largest_of(c, q, heads, scale):
    """The mean of the values of each row's positions of largest score, and its bound: weights equal where scores are,
    and n + 64 roundings of the sums."""
    out, bound = np.zeros((c.n_rows, heads, c.hd)), np.zeros((c.n_rows, heads, c.hd))
    for r, (b, pos) in enumerate(c.row_positions()):
        page, slot, ok = c.slots(b, pos + 1)
        k, v = (a[page[ok], 0, slot[ok]].astype(np.float64) for a in (c.k, c.v))
        for h in range(heads):
            s = scale * (k @ q[r, h].astype(np.float64))
            top = s == s.max()
            out[r, h] = v[top].mean(0)
            bound[r, h] = (8 + 2 * (len(s) + 64)) * M.U32 * np.abs(v[top]).mean(0) + 1e-30
    return out, bound


def steps(rng, dtype, heads, rows, room, order, hd=64, n=300):
    """Keys of one value, -4 .. 4 in steps of a quarter, so that scores are one product and the largest are ties."""
    c = M.Cache(rng, dtype, 1, hd, 16, rows, [n], room=room)
    c.k[:] = 0
    page, slot, _ = c.slots(0, n)
    x = rng.integers(-16, 17, n) / 4
    if order:
        x = np.sort(x)[::order]
    c.k[page, 0, slot, 3] = x
    return c, rng.standard_normal((c.n_rows, heads, hd)).astype(np.float32)


@pytest.mark.parametrize("hd,order", [(64, 0), (64, 1), (64, -1), (128, 0), (256, 1), (512, -1)])
@pytest.mark.parametrize("kernel", range(len(KERNELS)))
@pytest.mark.parametrize("dtype,powers", [("f16", (12, 20, 21, 22, 23, 24, 25, 26, 28, 30, 40, 60)),
                                          ("f32", (12, 21, 22, 24, 26, 30, 31, 32, 40, 60, 100))])
def test_scores_far_from_zero(dtype, powers, kernel, hd, order):
    """Scores of 2^12 to 2^100, above and below zero (all of them below: keys of one sign), next to ordinary rows."""
    heads, rows, room = KERNELS[kernel]
    rng = np.random.default_rng(kernel)
    c, q = steps(rng, dtype, heads, rows, room, order, hd)
    plain = q.copy()
    for below in (False, True):
        if below:
            c.k = -np.abs(c.k) - np.where(c.k != 0, 1, 0).astype(c.k.dtype)
            c.k[..., 3] = np.where(c.k[..., 3] == 0, -1, c.k[..., 3])
        for e in powers:
            q = plain.copy()
            far = rng.random(q.shape[:2]) < 0.7
            far[0, 0] = True
            sign = 1.0 if below else rng.choice([-1.0, 1.0], q.shape[:2])
            q[..., 3] = np.where(far, 1.37 * 2.0 ** e * sign, q[..., 3])
            got = attend(c, q, heads, 0.5)
            want, bound = largest_of(c, q, heads, 0.5)
            near, near_bound = M.attention(c, q, heads, 0.5)
            want[~far], bound[~far] = near[~far], near_bound[~far]
            bad = ~(np.abs(got - want) <= bound)
            assert not bad.any(), (f"2^{e}, below {below}: {bad.any(-1).sum()} of {far.sum()} + {(~far).sum()} rows and heads, "
                                   f"not finite {(~np.isfinite(got)).any(-1).sum()}")


@pytest.mark.parametrize("order", [0, 1])
@pytest.mark.parametrize("dtype", ["f16", "f32"])
@pytest.mark.parametrize("kernel", range(len(KERNELS)))
def test_scores_far_and_near_in_one_row(dtype, kernel, order):
    """Scores near 2^24 that differ by little: weights of all sizes, none of them lost or infinite. The scores are exact
    (whole numbers), so a weight is off by the rounding of its exponent, half a step of f32 at 2^24 times log2 e: 2^1,
    and as much for the largest."""
    heads, rows, room = KERNELS[kernel]
    rng = np.random.default_rng(kernel + 9)
    c, q = steps(rng, dtype, heads, rows, room, order)
    page, slot, _ = c.slots(0, 300)
    c.k[page, 0, slot, 3] = 1
    c.k[page, 0, slot, 5] = (rng.integers(0, 3, 300) if not order else np.arange(300) // 100) * 8
    c.v[:] = np.abs(c.v) + 1
    q[:] = 0
    q[..., 3], q[..., 5] = 2.0 ** 24, 1
    got = attend(c, q, heads, 1.0)
    assert np.isfinite(got).all()
    for r, (b, pos) in enumerate(c.row_positions()):
        pg, sl, _ = c.slots(b, pos + 1)
        s = c.k[pg, 0, sl, 5].astype(np.float64)
        v = c.v[pg, 0, sl].astype(np.float64)
        w = np.exp(s - s.max())
        low, high = w * 2.0 ** -4, np.minimum(w * 2.0 ** 4, 1.0)
        top = s == s.max()
        low[top] = high[top] = 1.0
        # a mean with weights between low and high lies between the means of the extreme choices
        least = (low @ v) / (high.sum())
        most = (high @ v) / (low.sum())
        assert np.all(got[r] >= 0.999 * least) and np.all(got[r] <= 1.001 * most)


@pytest.mark.parametrize("dtype", ["f16", "f32"])
@pytest.mark.parametrize("kernel", range(len(KERNELS)))
def test_scores_of_zero_under_any_scale(dtype, kernel):
    """Keys of zero: the mean of the values, whatever the queries and the scale."""
    heads, rows, room = KERNELS[kernel]
    rng = np.random.default_rng(kernel + 5)
    c, q = steps(rng, dtype, heads, rows, room, 0)
    c.k[:] = 0
    for size, scale in ((1e30, 1e30), (3e38, -1e38), (1e-38, 1.7e38), (1.0, -1.7e38), (1e-30, 1e-38)):
        got = attend(c, (q * 0.2 * size).astype(np.float32), heads, scale)
        want, bound = largest_of(c, np.ones_like(q), heads, 1.0)
        assert np.all(np.abs(got - want) <= bound), (size, scale)


@pytest.mark.parametrize("kernel", range(len(KERNELS)))
def test_scales_that_meet_small_queries(kernel):
    """A scale of 2^126 and queries of 2^-126 times ordinary ones are the ordinary attention, bit for bit; an f16
    cache (an f32 cache's products would lie below the least normal number)."""
    heads, rows, room = KERNELS[kernel]
    rng = np.random.default_rng(kernel + 6)
    c = M.Cache(rng, "f16", 1, 64, 16, rows, [300], room=room)
    q = (8 * rng.integers(-2 ** 12, 2 ** 12, (c.n_rows, heads, 64)) * 2.0 ** -12).astype(np.float32)
    want = attend(c, q, heads, 0.125)
    for x in (40, 100, 120):
        got = attend(c, (q * 2.0 ** -x).astype(np.float32), heads, 0.125 * 2.0 ** x)
        assert np.array_equal(got.view(np.int32), want.view(np.int32)), x
