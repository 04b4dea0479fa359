"""GPU tests of silu in the GatedDeltaNet layers' batched operators
(include/uq_serve.h), whose value is small far below 0, relative to that value."""
import numpy as np
import pytest

import gdn_model as M
from test_gpu_gdn_serve import Conv, Rule

pytestmark = pytest.mark.gpu

U = M.U
FLOOR = 2.0 ** -119  # results below it may be 0: reciprocals below 2^-126 are, of x to -89


def conv(c):
    """Results and their bound as gdn_model.conv's, with silu's own slope: of t within e of s at most
    sigmoid(s) exp(e) (1 + |s| + e), and 1.1. Its own roundings: 2 of the power of 2, one each of its correction, of 1 + it,
    and of the product, 2 of the reciprocal: 8 U with those of the correction's terms."""
    out = np.full((c.n_rows, c.ch), np.nan)
    tol = out.copy()
    w = c.conv1d.astype(np.float64).T
    for b, r, f, t in c.seqs():
        old = c.win[f, :c.taps - 1].astype(np.float64) if f is not None else np.zeros((c.taps - 1, c.ch))
        x = np.concatenate([old, c.qkv[r].astype(np.float64)])
        n = r.stop - r.start
        parts = [x[k:k + n] * w[k] for k in range(c.taps)]
        s, e = sum(parts), (c.taps + 1) * U * sum(np.abs(p) for p in parts)
        y = M.silu(s)
        slope = np.minimum(1.1, np.exp(e) * (1 + np.abs(s) + e) / (1 + np.exp(-s)))
        ye = slope * e + 8 * U * np.abs(y) + FLOOR
        h, he = (a.reshape(n, -1, c.hd) for a in (y, ye))
        q, qe = h[:, :2 * c.nqk], he[:, :2 * c.nqk]
        norm, ne = (np.linalg.norm(a, axis=-1, keepdims=True) for a in (q, qe))
        big = np.maximum(norm, M.EPS)
        he[:, :2 * c.nqk] = qe / big + np.abs(q) / big * (ne / big + 16 * U)
        h[:, :2 * c.nqk] = q / big
        out[r], tol[r] = y, ye
    return out, tol


@pytest.mark.parametrize("size", [1, 8, 30])
@pytest.mark.parametrize("taps,hd", [(4, 64), (4, 128), (3, 64)])
def test_convolution_far_below_zero(taps, hd, size):
    """Sums from -4 to -120 and on: each result within its own size."""
    c = M.Case(140 + size, 2, 4, hd, taps, [1, 40, 3], frm=[0, -1, 2])
    c.qkv *= np.float32(size)
    c.win *= np.float32(size)
    d = Conv(c)
    d.run()
    got = d.results()[0]
    with np.errstate(over="ignore"):
        want, tol = conv(c)
    assert np.all(np.abs(got - want) <= tol), np.max(np.abs(got - want) / tol)


def test_silu_of_single_values():
    """One tap of 1, so that the sum is the input: from the lowest value of the type to the highest."""
    c = M.Case(150, 1, 6, 64, 4, [9])
    c.conv1d[:] = 0
    c.conv1d[:, 3] = 1
    c.qkv[:, 128:] = np.linspace(-100, 100, 9 * 6 * 64).reshape(9, -1)
    c.qkv[8, 128:140] = [-3.4e38, -1e38, -1e30, -1e4, -1e-30, 0, 1e-30, 1e4, 1e30, 1e38, 2.5e38, 3.4e38]
    d = Conv(c)
    d.run()
    got = d.results()[0][:, 128:]
    x = c.qkv[:, 128:].astype(np.float64)
    with np.errstate(over="ignore"):
        want = M.silu(x)
    err = np.abs(got - want)
    assert np.all(err <= 8 * U * np.abs(want) + FLOOR), x[err > 8 * U * np.abs(want) + FLOOR]


@pytest.mark.parametrize("rows", [[9], [70]])
def test_the_rules_gate_far_below_zero(rows):
    """Results with the gate beside those without: the product's rounding and silu's 8."""
    c = M.Case(151, 1, 2, 64, 4, rows)
    c.z[:] = np.linspace(-100, 100, c.z.size).reshape(c.z.shape)
    runs = [Rule(c, 0, (True, gated)) for gated in (False, True)]
    for r in runs:
        r.run()
    plain, gated = (r.results()[0].astype(np.float64) for r in runs)
    with np.errstate(over="ignore"):
        want = plain * M.silu(c.z.astype(np.float64))
    assert np.all(np.abs(gated - want) <= 9 * U * np.abs(want) + FLOOR * np.maximum(1, np.abs(plain)))
