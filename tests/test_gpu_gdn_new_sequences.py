"""GPU tests of the batched gated delta rule (include/uq_serve.h) where a state,
or a column of one, is 0: new sequences and what they compute from values of any
size, by rows and by chunks."""
import numpy as np
import pytest

import gdn_model as M
from test_gpu_gdn_layer import ROWS
from test_gpu_gdn_serve import Rule, bits

pytestmark = pytest.mark.gpu


def plain(change=None, hd=64, frm=(-1, -1, -1, -1), decay=(-6, 0)):
    """Results without norm and gate, and states, of a case whose arrays `change` has scaled."""
    c = M.Case(101, 2, 4, hd, 4, ROWS, frm=frm, to=[0, 1, 2, 3], decay=decay)
    if change:
        change(c)
    r = Rule(c, 0, (False, False))
    r.run()
    return r.results()


def scaled(got, want, power):
    return all(np.array_equal(bits(g), bits(np.ldexp(w, power))) for g, w in zip(got, want))


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("power", [-70, -45, -20, 20, 90])
def test_new_sequences_are_linear_in_values(power, hd):
    """By powers of 2 bit for bit, as every scale is one."""
    def change(c):
        c.v *= np.float32(2.0 ** power)
        c.state[4] *= np.float32(2.0 ** power)  # the slot that no sequence has

    assert scaled(plain(change, hd), plain(hd=hd), power)


def test_new_sequences_have_a_scale_for_each_column():
    power = (np.arange(64) * 37 % 101 - 50).astype(np.int32)

    def change(c):
        c.v[:] = np.ldexp(c.v, power)
        c.state[4] = np.ldexp(c.state[4], power)

    assert scaled(plain(change), plain(), power)


@pytest.mark.parametrize("power", [-70, -20, 60])
def test_columns_of_zeros(power):
    """Sequences that go on from states of which single columns are 0."""
    def zeros(c):
        c.state[..., 1::3] = 0

    def change(c):
        zeros(c)
        c.v *= np.float32(2.0 ** power)
        c.state *= np.float32(2.0 ** power)

    own = (0, 1, 2, 3)
    assert scaled(plain(change, frm=own), plain(zeros, frm=own), power)


@pytest.mark.parametrize("power", [-30, -12, 20])
def test_keys_of_zeros_among_others(power):
    """Keys 2^p times larger, betas 4^-p and states 2^-p times: results 2^-p, whatever keys of zeros lie between."""
    def zeros(c):
        c.k[3::7] = 0

    def change(c):
        zeros(c)
        c.k *= np.float32(2.0 ** power)
        c.beta *= np.float32(4.0 ** -power)
        c.state *= np.float32(2.0 ** -power)

    own = (0, 1, 2, 3)
    assert scaled(plain(change, frm=own), plain(zeros, frm=own), -power)


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("power", [-70, -45, -30, -20, -13])
def test_new_sequences_of_small_values(power, hd):
    """Against 64 bits: with a state of 0 the model's bound holds nothing but the values' own sizes."""
    c = M.Case(102, 2, 4, hd, 4, ROWS, frm=[-1] * 4, to=[0, 1, 2, 3])
    c.v *= np.float32(2.0 ** power)
    r = Rule(c, 0, (False, False))
    r.run()
    r.check(False)


def test_corrections_of_zeros_beside_a_small_state():
    """Betas of 0 leave a state of 2^-110 to its decay, whatever the values are."""
    c = M.Case(103, 2, 4, 64, 4, ROWS, decay=(-12, -5))
    c.beta[:] = 0
    c.v *= np.float32(2.0 ** 60)
    c.state *= np.float32(2.0 ** -110)
    r = Rule(c, 0, (False, False))
    r.run()
    r.check(False)
