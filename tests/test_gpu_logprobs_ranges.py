"""GPU tests of uq_logprobs_d (include/uq_serve.h) where logits lie further apart
than f32's range, at scales that bring them back into it."""
import numpy as np
import pytest

import gdn_model as M
from test_gpu_logprobs import Run, close

pytestmark = pytest.mark.gpu

LOW, HIGH = np.finfo(np.float32).min, np.finfo(np.float32).max


def check(x, tokens, scale, n_top):
    got = Run(x, tokens, scale, n_top, 1).run().results()
    want = M.logprobs(x, tokens, scale, n_top)
    for k in ("logprob", "top_logprob"):  # what is below f32's range
        want[k] = np.where(want[k] < LOW, -np.inf, want[k])
    close(got["logprob"], want["logprob"], want["tol_logprob"])
    close(got["entropy"], want["entropy"], want["tol_entropy"])
    close(got["top_logprob"], want["top_logprob"], want["tol_top"])
    assert np.array_equal(got["rank"], want["rank"]) and np.array_equal(got["top_id"], want["top_id"])


@pytest.mark.parametrize("scale", [2.0, 1.0, 0.3, 0.1, 1e-3, 1e-30, 1e-37, 1e-38, 1e-39, 1e-45])
@pytest.mark.parametrize("vocab", [40, 3000])
def test_logits_further_apart_than_the_range(vocab, scale):
    """Every alternative of 40 tokens, and the far tokens of 3000, whose parts are joined across the range. The kernel's
    factor is that of a logit's difference: with 24 bits, and where it is denormal of at most 2^-20 of the difference's
    range, within 2 roundings of the sums' 112."""
    rng = np.random.default_rng(vocab)
    x = rng.standard_normal((7, vocab)).astype(np.float32) * np.float32(1e37)
    x[0, :], x[0, 5], x[0, 6] = 3e38, -3e38, LOW
    x[1, 7], x[1, 8], x[1, vocab - 1] = LOW, HIGH, -3e38
    x[2, :20], x[2, 20:] = LOW, HIGH
    x[3, :-3], x[3, -3:] = LOW, 0.0
    x[4, 1:], x[4, 0] = LOW, HIGH
    x[5, ::2], x[5, 1] = -np.inf, LOW
    x[6] = np.linspace(-3.3e38, 3.3e38, vocab)
    check(x, [5, 7, 3, 9, 11, 1, 0], scale, 64)
