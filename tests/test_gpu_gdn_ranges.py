"""GPU tests of the batched gated delta rule (include/uq_serve.h) near the end of
f32's range."""
import numpy as np
import pytest

from test_gpu_gdn_layer import plain
from test_gpu_gdn_serve import bits

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
