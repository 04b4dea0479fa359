"""GPU tests of uq_logprobs_d (include/uq_serve.h) against 64 bits
(gdn_model.logprobs): vocabularies, strides, alternatives, ties, masks, rows
without a possible token, values that are not finite, streams and graphs."""
import numpy as np
import pytest

import gdn_model as M
import uq
from test_gpu_gdn_serve import bits, dev, hip_of_bench, host
from uq import serve

pytestmark = pytest.mark.gpu


class Run:
    def __init__(self, x, tokens, scale=1.0, n_top=5, pad=0, want=("logprob", "rank", "entropy", "top_id", "top_logprob")):
        n, vocab = x.shape
        wide = np.full((n, vocab + pad), 1e30, np.float32)
        wide[:, :vocab] = x
        self.n, self.vocab, self.scale, self.n_top, self.pad = n, vocab, scale, n_top, pad
        self.x, self.tokens = dev(wide), dev(np.asarray(tokens, np.int32)) if tokens is not None else None
        like = {"logprob": np.float32, "rank": np.int32, "entropy": np.float32, "top_id": np.int32, "top_logprob": np.float32}
        self.like = {k: np.full((n, n_top) if k.startswith("top") else n, 77, t) for k, t in like.items()}
        self.d = {k: dev(a) if k in want and a.size else None for k, a in self.like.items()}
        self.out = serve.LogProbs(*(self.d[k] for k in like), n_top)
        self.ws = uq.DeviceArray(serve.logprobs_ws_bytes(n, vocab, n_top))
        self.ws.upload(np.full(self.ws.nbytes, 0xFF, np.uint8))

    def run(self, stream=None):
        serve.logprobs_d(self.out, self.x, self.tokens, self.n, self.vocab, self.ws, self.scale, self.vocab + self.pad, stream)
        return self

    def results(self):
        return {k: host(d, self.like[k]) for k, d in self.d.items() if d is not None}


def close(got, want, tol):
    nan = np.isnan(want)
    assert np.array_equal(np.isnan(got), nan)
    low = np.isneginf(want)
    assert np.array_equal(np.isneginf(got), low)
    ok = ~nan & ~low
    assert np.all(np.abs(got[ok] - want[ok]) <= tol[ok]), np.max(np.abs(got[ok] - want[ok]) / tol[ok])


def check(x, tokens, scale=1.0, n_top=5, pad=0):
    got = Run(x, tokens, scale, n_top, pad).run().results()
    want = M.logprobs(x, tokens, scale, n_top)
    close(got["logprob"], want["logprob"], want["tol_logprob"])
    close(got["entropy"], want["entropy"], want["tol_entropy"])
    assert np.array_equal(got["rank"], want["rank"])
    if n_top:
        assert np.array_equal(got["top_id"], want["top_id"])
        close(got["top_logprob"], want["top_logprob"], want["tol_top"])
    return got


@pytest.mark.parametrize("n,vocab,n_top,pad,scale", [
    (1, 1, 1, 0, 1.0), (3, 2, 5, 0, 2.0), (2, 63, 64, 1, 1.0), (5, 64, 64, 0, 0.1), (4, 1023, 20, 2, 1.0), (4, 1024, 20, 0, 1.3), (3, 1025, 1, 3, 1.0),
    (7, 32003, 5, 1, 0.7), (2, 152064, 20, 0, 1.25), (130, 20011, 3, 0, 1.0), (2, 600001, 64, 0, 1.0), (300, 999, 0, 0, 1.0), (70, 152064, 20, 0, 1.0)])
def test_against_64_bits(n, vocab, n_top, pad, scale):
    rng = np.random.default_rng(vocab + n)
    x = (3 * rng.standard_normal((n, vocab))).astype(np.float32)
    check(x, rng.integers(0, vocab, n), scale, n_top, pad)


@pytest.mark.parametrize("n_top", [1, 5, 64])
def test_ties_go_to_the_lower_number(n_top):
    """Few distinct logits over many tiles, one value alone, zeros of both signs."""
    rng = np.random.default_rng(n_top)
    x = rng.integers(-3, 3, (6, 9000)).astype(np.float32)
    x[1] = 2.5
    x[2] = np.where(rng.random(9000) < 0.5, 0.0, -0.0)
    x[3, 1024:] = -1e30
    x[4] = np.repeat(np.arange(9), 1000)
    x[5] = np.repeat(np.arange(9)[::-1], 1000)
    check(x, [8999, 4097, 8, 0, 1500, 1023], 1.0, n_top)


@pytest.mark.parametrize("n_top", [3, 64])
def test_orders(n_top):
    """Ascending rows bring a larger logit with every token, descending ones none after the first; the largest in one
    lane's places or in the last tile's end."""
    vocab = 70001
    up = np.linspace(-9, 9, vocab).astype(np.float32)
    lane = np.zeros(vocab, np.float32)
    lane[5::256] = np.linspace(1, 2, len(lane[5::256]))
    last = np.zeros(vocab, np.float32)
    last[-3:] = [7, 6, 8]
    x = np.stack([up, up[::-1], lane, last])
    check(x, [0, 0, 5, vocab - 1], 1.0, n_top)
    check(np.repeat(x, 40, 0), np.arange(160) * 400, 1.0, n_top)  # runs of several tiles


def test_masks():
    """Tokens that cannot follow: minus infinity is no alternative, the type's lowest value is one; rows of nothing."""
    rng = np.random.default_rng(3)
    vocab, low = 5000, np.float32(np.finfo(np.float32).min)
    x = rng.standard_normal((9, vocab)).astype(np.float32)
    x[0, rng.permutation(vocab)[:4990]] = -np.inf
    x[1] = -np.inf
    x[2] = low
    x[3, 2:] = low
    x[4, :4999] = -np.inf
    x[5] = low
    x[5, 17] = -3e38
    x[6] = 3e38
    x[6, 9] = low
    x[7, 100:] = -np.inf
    x[8] = np.where(np.arange(vocab) % 2, low, -np.inf)
    with np.errstate(over="ignore"):
        for scale in (1.0, 0.3):
            check(x, [3, 3, 3, 3, 4999, 17, 8, 200, 0], scale, 20)


def test_values_that_are_not_finite():
    rng = np.random.default_rng(4)
    x = rng.standard_normal((6, 3000)).astype(np.float32)
    x[0, 2999], x[2, 0], x[3, 1500], x[5] = np.nan, np.inf, -np.nan, np.nan
    check(x, [1, 2, 0, 4, 5, 6], 1.0, 7)


def test_tokens_that_are_none():
    x = np.random.default_rng(5).standard_normal((4, 500)).astype(np.float32)
    check(x, [-1, 500, 2 ** 31 - 1, -2 ** 31], 1.0, 2)


def test_peaked_and_flat():
    x = np.zeros((5, 4000), np.float32)
    x[0, 77], x[1, 77], x[2], x[3] = 1000.0, 30.0, 1e4, -1e4
    x[4] = np.linspace(-1e4, 1e4, 4000)
    check(x, [77, 0, 5, 6, 3998], 1.0, 4)


def test_only_what_is_wanted():
    rng = np.random.default_rng(6)
    x = rng.standard_normal((3, 2000)).astype(np.float32)
    tokens = [1, 2, 3]
    full = Run(x, tokens).run().results()
    for want in (("logprob",), ("rank",), ("entropy",), ("top_id",), ("top_logprob",), ("entropy", "top_id")):
        r = Run(x, tokens if {"logprob", "rank"} & set(want) else None, want=want).run().results()
        assert set(r) == set(want) and all(np.array_equal(r[k].view(np.int32), full[k].view(np.int32)) for k in want)


def test_far_rows():
    """Rows whose offsets pass 2^32 bytes."""
    n, vocab, row = 3, 1000, 600_000_000
    x = np.random.default_rng(7).standard_normal((n, vocab)).astype(np.float32)
    big = uq.DeviceArray(4 * (2 * row + vocab))
    L = uq.lib()
    for i in range(n):
        assert L.uq_memcpy_htod(big.ptr.value + 4 * i * row, x[i].ctypes.data, x[i].nbytes, None) == 0
        uq.synchronize()
    near = Run(x, [1, 2, 3]).run()
    want = near.results()
    serve.logprobs_d(near.out, big, near.tokens, n, vocab, near.ws, row=row)
    got = near.results()
    assert all(np.array_equal(got[k].view(np.int32), want[k].view(np.int32)) for k in want)
    big.free()


def test_replays_and_streams():
    """A captured call follows the logits and tokens of the time; two graphs share a workspace in turn."""
    hip = hip_of_bench()
    s = hip.stream()
    rng = np.random.default_rng(8)
    runs = [Run(np.zeros((n, vocab), np.float32), np.zeros(n), 1.1, top) for n, vocab, top in ((40, 3001, 5), (2, 90000, 20))]
    runs[0].ws = runs[1].ws = max((r.ws for r in runs), key=lambda w: w.nbytes)
    hip.sync()
    graphs = [hip.capture(s, lambda r=r: r.run(s)) for r in runs]
    for i in range(6):
        r = runs[i % 2]
        x = (2 * rng.standard_normal((r.n, r.vocab))).astype(np.float32)
        tokens = rng.integers(0, r.vocab, r.n)
        r.x.upload(x)
        r.tokens.upload(tokens.astype(np.int32))
        hip.sync()
        hip.launch_graph(graphs[i % 2], s)
        hip.sync()
        got = r.results()
        eager = Run(x, tokens, 1.1, r.n_top).run().results()
        assert all(np.array_equal(got[k].view(np.int32), eager[k].view(np.int32)) for k in eager), f"replay {i}"


@pytest.mark.parametrize("n_top", [20, 33, 64])
def test_more_candidates_than_are_kept(n_top):
    """Rows whose tiles hold more that may be among the first than a wave keeps: the type's lowest value but for a few
    tokens, one value but for larger and smaller ones among it, two values in turn, and tiles that end in ties."""
    rng = np.random.default_rng(n_top)
    vocab = 9 * 1024 + 77
    low = np.float32(np.finfo(np.float32).min)
    x = np.full((6, vocab), low, np.float32)
    x[0, rng.permutation(vocab)[:11]] = rng.standard_normal(11)
    x[1] = 1.0
    x[1, rng.permutation(vocab)[:15]] = 2.0
    x[1, rng.permutation(vocab)[:4000]] = -3.0
    x[2] = np.where(np.arange(vocab) % 2, 5.0, 4.0)
    x[3] = np.repeat(rng.permutation(vocab // 7 + 1), 7)[:vocab] // 9
    x[4] = np.minimum(np.arange(vocab), 3000)
    x[5] = rng.standard_normal(vocab)
    x[5, 1024:2048] = 0.5
    tokens = [5, 4000, 1, 77, 9000, 1500]
    with np.errstate(over="ignore"):
        check(x, tokens, 1.0, n_top)
        check(np.repeat(x, 300, 0)[:, :6000], np.minimum(np.repeat(tokens, 300), 5999), 1.0, n_top)  # runs of several tiles


@pytest.mark.parametrize("n_top", [0, 20, 64])
def test_many_rows(n_top):
    """So many rows that a wave takes more than one tile: ascending and descending ones, ties within and between tiles,
    masks of the type's lowest value and of minus infinity, the same rows again and again."""
    rng = np.random.default_rng(9)
    vocab, n = 2100, 22001
    x = rng.standard_normal((9, vocab)).astype(np.float32)
    x[1], x[2] = np.sort(x[1]), np.sort(x[2])[::-1]
    x[3] = 1.5
    x[4] = np.arange(vocab) // 700
    x[5], x[6] = np.finfo(np.float32).min, -np.inf
    x[5, rng.permutation(vocab)[:9]] = 0.0
    x[6, rng.permutation(vocab)[:30]] = rng.integers(0, 3, 30)
    x[7, 1500:] = 7.0
    tokens = np.array([3, 2000, 1, 1024, 700, 1999, 4, 1501, 1023])
    which = np.arange(n) % 9
    with np.errstate(over="ignore"):
        want = M.logprobs(x, tokens, 1.25, n_top)
        for k in ("logprob", "top_logprob"):  # 1.25 times the lowest value is nearest to -infinity among f32's
            want[k] = np.where(want[k] < np.finfo(np.float32).min, -np.inf, want[k])
    got = Run(x[which], tokens[which], 1.25, n_top).run().results()
    close(got["logprob"], want["logprob"][which], want["tol_logprob"][which])
    close(got["entropy"], want["entropy"][which], want["tol_entropy"][which])
    assert np.array_equal(got["rank"], want["rank"][which])
    if n_top:
        assert np.array_equal(got["top_id"], want["top_id"][which])
        close(got["top_logprob"], want["top_logprob"][which], want["tol_top"][which])
