"""The GatedDeltaNet operators of batched serving and the log probabilities
(include/uq_serve.h) without a GPU: what is refused before any launch,
workspace sizes, and the 64-bit models against plain loops."""
import numpy as np
import pytest

import gdn_model as M
import uq
from test_serve_cpu import A, At, refused
from uq import serve


def states(**over):
    s = dict(d_conv=A, d_state=A, n_slots=8, n_qk_heads=2, n_v_heads=4, head_dim=64, conv_kernel=4, d_from=A, d_to=A)
    return serve.GdnStates(**dict(s, **over))


def batch(**over):
    return serve.SeqBatch(**dict(dict(n_seqs=3, n_rows=7, d_row_start=A), **over))


def rows(**over):
    s = dict(d_qkv=A, qkv_row=512, d_conv1d=A, eps=1e-6, d_out=At(8192), d_beta_raw=A, d_alpha=A, d_dt_bias=A, d_a=A, d_beta=A, d_gate=A)
    return serve.GdnRows(**dict(s, **over))


def heads(**over):
    s = dict(d_q=A, q_row=128, d_k=A, k_row=128, d_v=A, v_row=256, d_gate=A, d_beta=A, scale=0.125, d_norm=A, d_z=A, z_row=256)
    return serve.GdnHeads(**dict(s, **over))


BAD_STATES = [("ARG", dict(n_qk_heads=0)), ("ARG", dict(n_v_heads=0)), ("ARG", dict(n_v_heads=1026)), ("LEN", dict(n_v_heads=3)),
              ("ARG", dict(head_dim=32)), ("ARG", dict(head_dim=256)), ("ARG", dict(conv_kernel=1)), ("ARG", dict(conv_kernel=10)),
              ("ARG", dict(n_slots=1 << 30)), ("ARG", dict(d_from=None)), ("ARG", dict(d_to=None))]
BAD_BATCH = [("ARG", dict(n_seqs=65536)), ("ARG", dict(n_rows=(1 << 23) + 1)), ("ARG", dict(d_row_start=None))]


@pytest.mark.parametrize("kind,over", BAD_STATES)
def test_bad_states_are_refused(kind, over):
    refused(kind, serve.gdn_conv_d, states(**over), batch(), rows())
    refused(kind, serve.gdn_rule_d, A, states(**over), batch(), heads(), A)
    assert serve.gdn_rule_ws_bytes(states(**over), batch()) == 0


@pytest.mark.parametrize("kind,over", BAD_BATCH)
def test_bad_batches_are_refused(kind, over):
    refused(kind, serve.gdn_conv_d, states(), batch(**over), rows())
    refused(kind, serve.gdn_rule_d, A, states(), batch(**over), heads(), A)
    assert serve.gdn_rule_ws_bytes(states(), batch(**over)) == 0


def test_each_call_needs_its_own_states():
    refused("ARG", serve.gdn_conv_d, states(d_conv=None), batch(), rows())
    refused("ARG", serve.gdn_rule_d, A, states(d_state=None), batch(), heads(), A)
    refused("ARG", serve.gdn_rule_d, A, states(d_state=At(4104)), batch(), heads(), A, text="aligned")
    assert serve.gdn_rule_ws_bytes(states(d_conv=None), batch()) > 0


@pytest.mark.parametrize("kind,over", [
    ("LEN", dict(qkv_row=511)), ("ARG", dict(d_qkv=None)), ("ARG", dict(d_conv1d=None)), ("ARG", dict(d_out=None)), ("ARG", dict(d_out=A)),
    ("ARG", dict(d_alpha=None)), ("ARG", dict(d_beta_raw=None)), ("ARG", dict(d_dt_bias=None)), ("ARG", dict(d_a=None)), ("ARG", dict(d_beta=None)),
    ("ARG", dict(d_gate=None)), ("LEN", dict(raw_row=3))])
def test_bad_rows_are_refused(kind, over):
    refused(kind, serve.gdn_conv_d, states(), batch(), rows(**over))


@pytest.mark.parametrize("kind,over", [
    ("ARG", dict(d_q=None)), ("ARG", dict(d_k=None)), ("ARG", dict(d_v=None)), ("ARG", dict(d_gate=None)), ("ARG", dict(d_beta=None)),
    ("LEN", dict(q_row=127)), ("LEN", dict(k_row=127)), ("LEN", dict(v_row=255)), ("LEN", dict(v_row=(1 << 24) + 1)), ("LEN", dict(z_row=255)), ("ARG", dict(scale=float("nan"))),
    ("ARG", dict(scale=float("inf")))])
def test_bad_heads_are_refused(kind, over):
    refused(kind, serve.gdn_rule_d, A, states(), batch(), heads(**over), A)


def test_rule_workspace():
    for n_rows, most in ((7, 0), (7, 1), (5000, 0), (5000, 5000), (64, 1)):
        b = batch(n_rows=n_rows)
        need = serve.gdn_rule_ws_bytes(states(), b, most)
        assert need > 0
        refused("ARG", serve.gdn_rule_d, A, states(), b, heads(), At(nbytes=need - 1), most_rows=most, text="workspace")
    refused("ARG", serve.gdn_rule_d, A, states(), batch(), heads(), At(4104), text="aligned")
    refused("ARG", serve.gdn_rule_d, A, states(), batch(), heads(), At(None))
    refused("ARG", serve.gdn_rule_d, At(None), states(), batch(), heads(), A)
    L = uq.lib()
    s, b, h, r = states(), batch(), heads(), rows()
    assert L.uq_gdn_rule_d(A.ptr, None, b._at, h._at, 0, A.ptr, 1 << 40, None) == 4
    assert L.uq_gdn_rule_d(A.ptr, s._at, None, h._at, 0, A.ptr, 1 << 40, None) == 4
    assert L.uq_gdn_rule_d(A.ptr, s._at, b._at, None, 0, A.ptr, 1 << 40, None) == 4
    assert L.uq_gdn_conv_d(s._at, b._at, None, None) == 4 and L.uq_gdn_conv_d(None, b._at, r._at, None) == 4


def probs(**over):
    s = dict(d_logprob=A, d_rank=A, d_entropy=A, d_top_id=A, d_top_logprob=A, n_top=5)
    return serve.LogProbs(**dict(s, **over))


def test_logprobs_refusals():
    ok = dict(out=probs(), d_x=A, d_tokens=A, n_rows=3, vocab=100, ws=A)
    refused("ARG", serve.logprobs_d, **dict(ok, vocab=0), row=100)
    refused("ARG", serve.logprobs_d, **dict(ok, vocab=(1 << 24) + 1))
    refused("ARG", serve.logprobs_d, **dict(ok, n_rows=(1 << 23) + 1))
    refused("ARG", serve.logprobs_d, **dict(ok, n_rows=1 << 20, vocab=(1 << 19) + 1))
    refused("ARG", serve.logprobs_d, **dict(ok, out=probs(n_top=65)))
    refused("LEN", serve.logprobs_d, **ok, row=99)
    refused("ARG", serve.logprobs_d, **dict(ok, d_x=At(None)))
    refused("ARG", serve.logprobs_d, **dict(ok, d_tokens=None))
    for scale in (0.0, -1.0, float("nan"), float("inf"), 3e38):
        refused("ARG", serve.logprobs_d, **ok, scale=scale, text="scale")
    need = serve.logprobs_ws_bytes(3, 100, 5)
    assert need > 0
    refused("ARG", serve.logprobs_d, **dict(ok, ws=At(nbytes=need - 1)), text="workspace")
    refused("ARG", serve.logprobs_d, **dict(ok, ws=At(4104)), text="aligned")
    refused("ARG", serve.logprobs_d, **dict(ok, ws=At(None)))
    for a in ((3, 0, 5), (3, 1 << 25, 0), (1 << 24, 10, 0), (3, 100, 65)):
        assert serve.logprobs_ws_bytes(*a) == 0
    assert uq.lib().uq_logprobs_d(None, A.ptr, 100, A.ptr, 3, 100, 1.0, A.ptr, 1 << 40, None) == 4


def test_empty_batches_need_no_device():
    for b in (batch(n_seqs=0, n_rows=0, d_row_start=None), batch(n_rows=0)):
        serve.gdn_conv_d(states(), b, rows())
        serve.gdn_rule_d(A, states(), b, heads(), A)
    serve.gdn_conv_d(states(n_slots=0, d_conv=None), batch(n_rows=0), rows())
    serve.logprobs_d(probs(), A, A, 0, 100, A)


# ------------------------------------------------------------------------- the models

def test_the_rules_model_is_the_step():
    c = M.Case(3, 2, 4, 64, 4, [5, 0, 70], frm=[1, 0, -1], to=[1, 2, 0])
    (out, tol), (st, _) = M.rule(c, finish=False)
    for b, r, f, t in c.seqs():
        S = c.state[f].astype(np.float64) if f is not None else np.zeros((4, 64, 64))
        for i in range(r.start, r.stop):
            for h in range(4):
                S[h] *= np.exp(np.float64(c.gate[i, h]))
                d = (c.v[i, h].astype(np.float64) - c.k[i, h % 2].astype(np.float64) @ S[h]) * c.beta[i, h]
                S[h] += np.outer(c.k[i, h % 2], d)
                assert np.allclose(out[i, h], c.scale * (c.q[i, h % 2].astype(np.float64) @ S[h]), rtol=1e-12, atol=1e-14)
        assert np.allclose(st[t], S, rtol=1e-12, atol=1e-14)
    assert np.array_equal(st[3], c.state[3]) and np.nanmax(tol) < 1e-2


def test_the_convolutions_model_is_the_loop():
    c = M.Case(4, 1, 2, 64, 3, [4, 1], frm=[0, -1], to=[2, 1], pad=1)
    (out, _), (beta, _), (gate, _), win = M.conv(c)
    x = np.concatenate([c.win[0, :2], c.qkv[:4]]).astype(np.float64)
    for i in range(4):
        y = sum(x[i + k] * c.conv1d[:, k] for k in range(3))
        y = (y / (1 + np.exp(-y))).reshape(-1, 64)
        y[:2] /= np.linalg.norm(y[:2], axis=1, keepdims=True)
        assert np.allclose(out[i], y.reshape(-1), rtol=1e-12)
    assert np.array_equal(win[2, :2], x[4:]) and np.array_equal(win[1, :2], [np.zeros(c.ch), c.qkv[4]])
    assert np.array_equal(win[2, 2], c.win[2, 2]) and np.isnan(out[5]).all()


def test_the_log_probabilities_model():
    x = np.array([[1, 3, 3, -np.inf], [-np.inf] * 4, [0, np.nan, 1, 2], [-3.4e38] * 4], np.float32)
    r = M.logprobs(x, [2, 1, 0, 9], 0.5, 3)
    p = np.exp([0.5, 1.5, 1.5]) / np.exp([0.5, 1.5, 1.5]).sum()
    assert np.isclose(r["logprob"][0], np.log(p[2])) and r["rank"].tolist() == [1, 1, -1, -1]
    assert np.isclose(r["entropy"][0], -(p * np.log(p)).sum()) and r["top_id"][0].tolist() == [1, 2, 0]
    assert r["entropy"][1] == 0 and r["top_id"][1].tolist() == [-1] * 3 and np.isnan(r["logprob"][2])
    assert np.isclose(r["entropy"][3], np.log(4)) and r["logprob"][3] == -np.inf and r["top_id"][3].tolist() == [0, 1, 2]
