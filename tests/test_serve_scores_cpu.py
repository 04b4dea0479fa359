"""The running reference of the paged attention's softmax (uq_attn_ref.h) on the CPU: weights stay within what their
type holds, and the largest is not lost, for scores of any size."""
import ctypes as C

import numpy as np
import pytest

import uq

# shift, move (below 0: with every larger score), the largest exponent that may be held (f16: 65504; f32: far below 2^127)
KINDS = {"f16 few": (14.0, -1.0, 15.9), "f16 many": (8.0, 15.0, 15.9), "f32": (0.0, -1.0, 1.0)}


def softmax(z, exp, kind, tile):
    E = uq.emu()
    E.uq_emu_softmax.argtypes = [C.c_void_p, C.c_int, C.c_int, C.c_int, C.c_float, C.c_float, C.c_void_p]
    E.uq_emu_softmax.restype = C.c_double
    z = np.ascontiguousarray(z, np.float32)
    largest = np.zeros(1)
    l = E.uq_emu_softmax(z.ctypes.data, z.size, tile, exp, *KINDS[kind][:2], largest.ctypes.data)
    return l, largest[0]


@pytest.mark.parametrize("order", [0, 1, -1])
@pytest.mark.parametrize("kind", list(KINDS))
@pytest.mark.parametrize("e", [0, 4, 10, 19, 20, 21, 22, 23, 24, 25, 27, 30, 31, 33, 40, 60, 90])
def test_weights_are_held_within_their_type(kind, e, order):
    rng = np.random.default_rng(e)
    for sign in (0, 1, -1):
        z = rng.uniform(-1, 1, 500).astype(np.float32) * np.float32(1.37 * 2.0 ** e)
        z = np.abs(z) * sign if sign else z
        z = np.sort(z)[::order] if order else z
        z[100:110] = z.max()  # ties
        for tile, exp in ((16, 0), (128, 0), (16, -30), (128, 30)):
            l, largest = softmax(np.ldexp(z, -exp), exp, kind, tile)
            assert largest <= KINDS[kind][2], (sign, tile)
            # the largest is 2^0 at least, and the ten ties all count
            assert 10 <= l <= 500 * 2.0 ** KINDS[kind][2], (sign, tile, l)


@pytest.mark.parametrize("kind", list(KINDS))
def test_scores_about_the_border_of_both_forms(kind):
    """Scores that rise or fall through +-2^22, a power of two or two a step."""
    for at in (2.0 ** 22, -2.0 ** 22):
        for step in (0.5, 2.0, -0.5, -2.0):
            z = (at + step * np.arange(-40, 41)).astype(np.float32)
            for tile in (1, 16):
                l, largest = softmax(z, 0, kind, tile)
                want = np.exp2(z.astype(np.float64) - z.max()).sum()
                assert largest <= KINDS[kind][2]
                shifts = l / want  # 2^(largest + a)
                assert 1 - 1e-12 <= shifts <= 2.0 ** KINDS[kind][2]


@pytest.mark.parametrize("kind", list(KINDS))
def test_nothing_seen_leaves_no_weight(kind):
    l, _ = softmax(np.full(40, -np.inf), 0, kind, 16)
    assert l == 0
    l, _ = softmax(np.concatenate([np.full(40, -np.inf), [3.0]]), 0, kind, 16)
    assert np.isfinite(l) and l >= 0.9
