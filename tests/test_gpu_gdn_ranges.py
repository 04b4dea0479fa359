"""GPU tests of the batched gated delta rule (include/uq_serve.h) near the end of
f32's range, and of values that are not finite beside values far from 1."""
import numpy as np
import pytest

import gdn_model as M
from test_gpu_gdn_layer import plain
from test_gpu_gdn_serve import Rule, bits

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("power", [112, 116, 120, 122])
def test_values_and_states_near_the_end_of_the_range(power, hd):
    """Values to 2^125 and states to 2^124, whose results f32 holds: by powers of 2 bit for bit."""
    def change(c):
        c.v *= np.float32(2.0 ** power)
        c.state *= np.float32(2.0 ** power)

    want, ws = plain(hd=hd)
    got, gs = plain(change, hd)
    assert np.array_equal(bits(got), bits(np.ldexp(want, power))) and np.array_equal(bits(gs), bits(np.ldexp(ws, power)))


@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf])
@pytest.mark.parametrize("at", [40, 100])
@pytest.mark.parametrize("power,frm", [(116, 0), (116, -1), (-60, 0), (-60, -1)])
def test_a_value_that_is_not_finite_beside_others_of_any_size(power, frm, at, bad):
    """Rows before it, other heads and the other sequence are as without it, within the model's bound."""
    c = M.Case(121, 2, 4, 64, 4, [150, 70], frm=[frm, 1], to=[0, 1])
    c.v *= np.float32(2.0 ** power)
    c.state *= np.float32(2.0 ** power)
    (want, tol), _ = M.rule(c, False)
    c.v[at, 1, 7] = bad
    r = Rule(c, 0, (False, False))
    r.run()
    out, _ = r.results()
    seen = np.ones(out.shape, bool)
    seen[at:150, 1] = False
    assert np.all((np.abs(out - want) <= tol) | ~seen), np.nonzero(~(np.abs(out - want) <= tol) & seen)
    assert not np.isfinite(out[at:150, 1, 7]).any()


@pytest.mark.parametrize("bad", [np.nan, np.inf])
@pytest.mark.parametrize("at", [66, 100])
@pytest.mark.parametrize("power", [-30, 30])
def test_a_key_that_is_not_finite_beside_keys_of_any_size(power, at, bad):
    """Keys 2^p times larger, betas 4^-p and states 2^-p times: results 2^-p; a key that is not finite is seen from its
    row on alone."""
    c = M.Case(122, 2, 4, 64, 4, [150, 70], decay=(-9, -5))
    (want, tol), _ = M.rule(c, False)
    want, tol = np.ldexp(want, -power), np.ldexp(tol, -power)
    c.k *= np.float32(2.0 ** power)
    c.beta *= np.float32(4.0 ** -power)
    c.state *= np.float32(2.0 ** -power)
    c.k[at, 1, 7] = bad
    r = Rule(c, 0, (False, False))
    r.run()
    out, _ = r.results()
    seen = np.ones(out.shape, bool)
    seen[at:150, 1::2] = False
    assert np.all((np.abs(out - want) <= tol) | ~seen), np.nonzero(~(np.abs(out - want) <= tol) & seen)
