"""GPU tests of batched serving with inputs whose bounds are tight (serve_bounds.py; what they can see is shown in
test_serve_bounds_cpu.py), and at sizes that take the branches of long work lists."""
import numpy as np
import pytest

import serve_bounds as B
import serve_model as M
from test_gpu_serve import attend, run_verify

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


# ------------------------------------------------------------------------- long work lists

@pytest.mark.parametrize("dtype,heads,hd,rows,lens,room", [
    ("f16", 64, 64, [3, 520, 1], [9, 600, 70], 1 << 16),  # 260 blocks of 128 queries
    ("f16", 64, 64, [130], [200], 1 << 16),               # 65 of them
    ("f32", 64, 64, [2, 520], [40, 530], 1 << 16),        # 1040 of 32
    ("f32", 64, 64, [520], [48], 0),                      # 2080 of 16
    ("f16", 64, 512, [1, 80, 2], [4, 1000, 90], 1 << 14),  # 320 of 16
    ("f32", 64, 512, [80], [300], 1 << 14),
    ("f16", 48, 64, [100, 1], [400, 30], 0),              # 300 of 16, a workgroup each
    ("f32", 48, 64, [100], [400], 0),
    ("f16", 64, 64, [17] * 70, [20 + i for i in range(70)], 1 << 12)])  # many sequences of many blocks
def test_attention_of_many_blocks(dtype, heads, hd, rows, lens, room):
    """Sequences of more blocks than a wave's lanes and than a workgroup's threads, which look for theirs together."""
    rng = np.random.default_rng(len(rows) + hd)
    c = M.Cache(rng, dtype, 1, hd, 16, rows, lens, room=room)
    q = rng.standard_normal((c.n_rows, heads, hd)).astype(np.float32)
    want, bound = B.attention(c, q, heads, hd ** -0.5)
    inside(attend(c, q, heads, hd ** -0.5), want, bound + 1e-30, f"{dtype} {rows[:3]} rows of {heads} heads")


@pytest.mark.parametrize("seqs,vocab,draft", [(2048, 8200, True), (2731, 6145, False), (8300, 8200, False), (4200, 20000, False)])
def test_verify_of_many_chunks(seqs, vocab, draft):
    """Sequences times chunks of the vocabulary beyond what is a wave each: 2 to 8 chunks a wave, the last wave fewer."""
    rng = np.random.default_rng(seqs)
    p = rng.random((seqs, vocab), np.float32)
    q = rng.random((seqs, vocab), np.float32) if draft else None
    rows = np.ones(seqs, np.int64)
    rows[::7], rows[1::7] = 2, 0
    rows = rows[:np.searchsorted(np.cumsum(rows), seqs, side="right")].tolist()  # no more rows than there are
    n = sum(rows)
    tokens, u = rng.integers(0, vocab, n), rng.random(n).astype(np.float32)
    p, q = p[:n], None if q is None else q[:n]
    got, want = run_verify(p, q, tokens, u, rows), M.verify(p, q, tokens, u, rows)
    assert np.array_equal(got[0], want[0]) and np.array_equal(got[1], want[1])
