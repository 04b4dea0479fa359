"""Performance cases of batched serving's recurrent layers and of the log probabilities of its answers.

`uq.serve` takes the new rows of several sequences through a GatedDeltaNet layer's recurrent part (the
causal convolution with its windows, the gated delta rule with its states, token by token for a few
rows and by chunks for many) and reports, from a row's logits, the log probability and rank of a given
token, the entropy and the likeliest alternatives. A case is a dict of plain values; `prepare` makes
what a serving program holds, `run` is one pass through one operator: in elementary torch operations
where `own` is false, by the library's entry points where it is true. `exact` is the operator's
definition in 64 bits.

Head counts and widths are those of the synthetic hybrid model of bench.py (16 query/key and 32 value
heads of 128, four taps, vocabulary 152064) and of the tests (heads of 64).
"""
import ctypes
import math
import os
import random
import sys

import torch

own = False

EPS = 1e-6


# ---------------------------------------------------------------------- cases
def listed():
    model = {"nqk": 16, "nv": 32, "hd": 128, "taps": 4}
    return [
        # sequences that verify up to four drafted tokens each: a small convolution, all latency
        {"name": "conv 29 drafts", "kind": "conv", "seqs": 29, "first": 5, "most": 5, "mix": 1, **model},
        # the prompts of three requests in one batch
        {"name": "conv prompts", "kind": "conv", "seqs": 3, "first": 2048, "most": 2048, "mix": 2, **model},
        # one decoded token of one conversation: the smallest call of the rule
        {"name": "rule 1", "kind": "rule", "seqs": 1, "first": 1, "most": 1, "gated": True, "mix": 3, **model},
        # an ordinary decode batch: the states themselves are the work
        {"name": "rule 64", "kind": "rule", "seqs": 64, "first": 1, "most": 1, "gated": True, "mix": 4, **model},
        # a batch of sequences with up to four drafted tokens each, narrower heads, no gate
        {"name": "rule 29 drafts", "kind": "rule", "seqs": 29, "first": 5, "most": 5, "gated": False, "mix": 5,
         "nqk": 4, "nv": 12, "hd": 64, "taps": 4},
        # one short prompt
        {"name": "rule prompt 509", "kind": "rule", "seqs": 1, "first": 509, "most": 509, "gated": True, "mix": 6, **model},
        # a chunk of one prompt beside the decoded tokens of other conversations
        {"name": "rule 1021 beside 40", "kind": "rule", "seqs": 41, "first": 1021, "most": 1, "gated": True, "mix": 7, **model},
        # the prompts of three requests in one batch
        {"name": "rule prompts", "kind": "rule", "seqs": 3, "first": 2048, "most": 2048, "gated": True, "mix": 8, **model},
        # one decoded token's report
        {"name": "logprobs 1 top 20", "kind": "logprobs", "rows": 1, "vocab": 152064, "top": 20, "pad": 0},
        # a decode batch's
        {"name": "logprobs 64 top 20", "kind": "logprobs", "rows": 64, "vocab": 152064, "top": 20, "pad": 0},
        # a smaller vocabulary, rows that start at any float
        {"name": "logprobs 13 odd", "kind": "logprobs", "rows": 13, "vocab": 32003, "top": 5, "pad": 2},
        # a given text's tokens scored, without alternatives
        {"name": "logprobs 1021 scored", "kind": "logprobs", "rows": 1021, "vocab": 152064, "top": 0, "pad": 0},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """A case of the same ranges, no larger than the largest listed one of its kind."""
    kind = rng.choice(["conv", "rule", "rule", "prompt", "prompt", "beside", "logprobs", "logprobs"])
    if kind == "logprobs":
        rows = _log(rng, 1, 1021)
        top = rng.choice([0, 1, 5, 20, 64])
        return {"kind": kind, "rows": rows, "vocab": _log(rng, 500, min(152064, 152064 * (1021 if top == 0 else 200) // rows)), "top": top,
                "pad": rng.choice([0, 0, 1, 6])}
    hd = rng.choice([64, 128, 128])
    nqk = rng.choice([2, 4, 8, 16])
    c = {"kind": "conv" if kind == "conv" else "rule", "nqk": nqk, "nv": nqk * rng.choice([1, 2, 2, 3] if nqk < 16 else [1, 2]), "hd": hd,
         "taps": rng.choice([2, 4, 4, 4, 5]), "mix": rng.randrange(1 << 30)}
    if kind != "conv":
        c["gated"] = rng.random() < 0.7
    if kind == "rule" or (kind == "conv" and rng.random() < 0.5):
        most = rng.choice([1, 1, 5, 9])
        return dict(c, seqs=_log(rng, 1, 64 // (1 if most == 1 else 2)), first=most, most=most)
    if kind == "beside":
        return dict(c, seqs=_log(rng, 2, 41), first=_log(rng, 10, 1021), most=rng.choice([1, 4]))
    n = rng.randint(1, 3)
    first = _log(rng, 17, 4096 // n)
    return dict(c, seqs=n, first=first, most=first)


def _rows(case):
    """New rows of each sequence: the first as many as the case says, the others spread."""
    rng = random.Random(case["mix"])
    lo = max(1, case["most"] // 2) if case["most"] > 16 else 1
    return [case["first"] if i == 0 else _log(rng, lo, case["most"]) for i in range(case["seqs"])]


# ---------------------------------------------------------------------- inputs
class Buf:
    """A torch tensor where the binding takes a device array."""

    def __init__(self, t):
        self.t, self.ptr, self.nbytes = t, ctypes.c_void_p(t.data_ptr()), t.numel() * t.element_size()


def _serve():
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "unltd-inference_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    from uq import serve

    return serve


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)

    def normal(*shape):
        return torch.randn(*shape, generator=g, device="cuda")

    def uniform(*shape):
        return torch.rand(*shape, generator=g, device="cuda")

    def whole(v):
        return torch.tensor(v, dtype=torch.int32, device="cuda")

    s = {"case": case}
    if case["kind"] == "logprobs":
        n, v, top = case["rows"], case["vocab"], case["top"]
        s["logits"] = 2.5 * normal(n, v + case["pad"])
        # a text's own tokens are likelier than others
        s["tokens"] = torch.randint(0, v, (n,), generator=g, device="cuda", dtype=torch.int32)
        s["logits"][torch.arange(n, device="cuda"), s["tokens"].long()] += 8.0 * uniform(n)
        s["scale"] = 1.25
        s["out"] = {"logprob": torch.empty(n, device="cuda"), "rank": torch.empty(n, dtype=torch.int32, device="cuda"),
                    "entropy": torch.empty(n, device="cuda"), "top_id": torch.empty(n, top, dtype=torch.int32, device="cuda"),
                    "top_logprob": torch.empty(n, top, device="cuda")}
        if own:
            serve = _serve()
            o = s["out"]
            s["probs"] = serve.LogProbs(Buf(o["logprob"]), Buf(o["rank"]), Buf(o["entropy"]), Buf(o["top_id"]) if top else None,
                                        Buf(o["top_logprob"]) if top else None, top)
            s["ws"] = Buf(torch.empty(serve.logprobs_ws_bytes(n, v, top), dtype=torch.uint8, device="cuda"))
            s["bufs"] = [Buf(s["logits"]), Buf(s["tokens"])]
        return s

    nqk, nv, hd, taps = case["nqk"], case["nv"], case["hd"], case["taps"]
    channels, rows = (2 * nqk + nv) * hd, _rows(case)
    n, slots = sum(rows), len(rows) + 1
    start = [sum(rows[:i]) for i in range(len(rows) + 1)]
    s["rows"], s["start"], s["d_start"] = rows, start, whole(start)
    s["slots"] = torch.randperm(slots, generator=g, device="cuda")[:len(rows)].int()
    if case["kind"] == "conv":
        s["win"] = normal(slots, taps, channels)
        s["qkv"] = normal(n, channels)
        s["conv1d"] = 0.5 * normal(channels, taps)
        s["beta_raw"], s["alpha"] = normal(n, nv), 2.0 * normal(n, nv) - 3.0
        s["dt_bias"], s["a"] = normal(nv), -torch.exp(2.7 * uniform(nv))
        s["out"], s["beta"], s["gate"] = torch.empty(n, channels, device="cuda"), torch.empty(n, nv, device="cuda"), torch.empty(n, nv, device="cuda")
    else:
        # rows as the convolution leaves them: unit queries and keys, values, decays from none to nearly all
        x = normal(n, channels)
        qk = x[:, :2 * nqk * hd].view(n, 2 * nqk, hd)
        qk /= torch.linalg.vector_norm(qk, dim=-1, keepdim=True)
        s["qkv"] = x
        s["gate"] = -torch.exp(8.0 * uniform(n, nv) - 6.5)
        s["beta"] = torch.sigmoid(1.5 * normal(n, nv))
        s["z"], s["norm"] = normal(n, nv * hd), 1.0 + 0.1 * normal(hd)
        s["state"] = 0.3 * normal(slots, nv, hd, hd)
        s["out"] = torch.empty(n, nv, hd, device="cuda")
        s["scale"] = 1.0 / math.sqrt(hd)
    if own:
        serve = _serve()
        s["batch"] = serve.SeqBatch(n_seqs=len(rows), n_rows=n, d_row_start=Buf(s["d_start"]))
        s["states"] = serve.GdnStates(d_conv=Buf(s["win"]) if "win" in s else None, d_state=Buf(s["state"]) if "state" in s else None,
                                      n_slots=slots, n_qk_heads=nqk, n_v_heads=nv, head_dim=hd, conv_kernel=taps, d_from=Buf(s["slots"]),
                                      d_to=Buf(s["slots"]))
        if case["kind"] == "conv":
            s["in"] = serve.GdnRows(d_qkv=Buf(s["qkv"]), qkv_row=channels, d_conv1d=Buf(s["conv1d"]), eps=EPS, d_out=Buf(s["out"]),
                                    d_beta_raw=Buf(s["beta_raw"]), d_alpha=Buf(s["alpha"]), d_dt_bias=Buf(s["dt_bias"]), d_a=Buf(s["a"]),
                                    d_beta=Buf(s["beta"]), d_gate=Buf(s["gate"]))
        else:
            q, k, v = s["qkv"][:, :nqk * hd], s["qkv"][:, nqk * hd:2 * nqk * hd], s["qkv"][:, 2 * nqk * hd:]
            s["in"] = serve.GdnHeads(d_q=Buf(q), q_row=channels, d_k=Buf(k), k_row=channels, d_v=Buf(v), v_row=channels, d_gate=Buf(s["gate"]),
                                     d_beta=Buf(s["beta"]), scale=s["scale"], d_norm=Buf(s["norm"]) if case["gated"] else None, eps=EPS,
                                     d_z=Buf(s["z"]) if case["gated"] else None, z_row=nv * hd)
            s["o"] = Buf(s["out"])
            s["ws"] = Buf(torch.empty(serve.gdn_rule_ws_bytes(s["states"], s["batch"], max(rows)), dtype=torch.uint8, device="cuda"))
    return s


# ---------------------------------------------------------------------- one pass
def run(s):
    c = s["case"]
    if own:
        serve = _serve()
        if c["kind"] == "conv":
            serve.gdn_conv_d(s["states"], s["batch"], s["in"])
            return [s["out"], s["beta"], s["gate"], s["win"]]
        if c["kind"] == "rule":
            serve.gdn_rule_d(s["o"], s["states"], s["batch"], s["in"], s["ws"], most_rows=max(s["rows"]))
            return [s["out"], s["state"]]
        serve.logprobs_d(s["probs"], *s["bufs"], c["rows"], c["vocab"], s["ws"], scale=s["scale"], row=c["vocab"] + c["pad"])
        return s["out"]
    return {"conv": _conv, "rule": _rule, "logprobs": _logprobs}[c["kind"]](s)


def _conv(s):
    c = s["case"]
    nqk, nv, hd, taps = c["nqk"], c["nv"], c["hd"], c["taps"]
    x, n, slots = s["qkv"], s["qkv"].shape[0], s["slots"].long()
    rows = s["d_start"].diff().long()
    seq = torch.repeat_interleave(torch.arange(len(rows), device="cuda"), rows, output_size=n)
    at = torch.arange(n, device="cuda") - s["d_start"][:-1].long()[seq]  # a row's place in its sequence
    # the sequence [the window's rows; the new rows], by places: place p of sequence b
    old = s["win"][slots, :taps - 1]

    def entry(b, place):
        inside = place >= taps - 1
        new = x[(s["d_start"][b].long() + place - (taps - 1)).clamp(min=0, max=n - 1)]
        return torch.where(inside[:, None], new, old[b, place.clamp(max=max(taps - 2, 0))])

    y = sum(entry(seq, at + t) * s["conv1d"][:, t] for t in range(taps))
    y = y / (1.0 + torch.exp(-y))
    qk = y[:, :2 * nqk * hd].view(n, 2 * nqk, hd)
    qk = qk / torch.sqrt((qk * qk).sum(-1, keepdim=True)).clamp(min=EPS)
    s["out"] = torch.cat([qk.reshape(n, -1), y[:, 2 * nqk * hd:]], 1)
    s["beta"] = 1.0 / (1.0 + torch.exp(-s["beta_raw"]))
    t = (s["alpha"] + s["dt_bias"]).double()
    s["gate"] = (torch.log1p(torch.exp(-t.abs())) + t.clamp(min=0.0)).float() * s["a"]
    every = torch.arange(len(rows), device="cuda")
    s["win"][slots, :taps - 1] = torch.stack([entry(every, rows + t) for t in range(taps - 1)], 1)
    return [s["out"], s["beta"], s["gate"], s["win"]]


def _rule(s):
    c = s["case"]
    nqk, nv, hd = c["nqk"], c["nv"], c["hd"]
    rows, n = s["d_start"].diff().long(), s["qkv"].shape[0]
    most = max(s["rows"])
    size = min(64, 1 << (most - 1).bit_length())  # rows of a chunk, a power of two
    order = torch.argsort(rows, descending=True)  # long sequences first: those with rows left are the first few
    x = s["qkv"].view(n, 2 * nqk + nv, hd)
    S = s["state"][s["slots"].long()[order]]
    out = torch.empty(n, nv, hd, device="cuda")
    lower = torch.tril(torch.ones(size, size, device="cuda", dtype=torch.bool))
    of = torch.arange(nv, device="cuda") % nqk  # a value head's query and key head
    lengths = sorted(s["rows"], reverse=True)
    for c0 in range(0, most, size):
        live = sum(1 for r in lengths if r > c0)
        b = order[:live]
        place = c0 + torch.arange(size, device="cuda")
        has = place[None, :] < rows[b][:, None]
        r = (s["d_start"][:-1].long()[b][:, None] + place).clamp(max=n - 1)

        def heads(t):  # [sequences, rows, heads, ..] as [sequences, heads, rows, ..], zero where there is no row
            t = t[r] * has.view(*has.shape, *([1] * (t.dim() - 1)))
            return t.transpose(1, 2).contiguous()

        q, k, v = heads(x[:, :nqk])[:, of], heads(x[:, nqk:2 * nqk])[:, of], heads(x[:, 2 * nqk:])
        beta = heads(s["beta"])
        g = torch.cumsum(heads(s["gate"]).double(), -1)
        decay = torch.exp(torch.where(lower, g[..., :, None] - g[..., None, :], -math.inf)).float()
        eg = torch.exp(g).float()[..., None]
        kk = (k @ k.transpose(-1, -2)) * decay * beta[..., None]
        # the inverse of I + the part of kk below the diagonal, blocks of 1, 2, 4, .. joined two and two
        t = torch.eye(size, device="cuda").expand_as(kk).clone()
        w = 1
        while w < size:
            m = size // (2 * w)
            i = torch.arange(m, device="cuda")[:, None] * 2 * w + torch.arange(w, device="cuda")
            lo, hi = i[:, :, None], i[:, :, None] + w
            lo2, hi2 = i[:, None, :], i[:, None, :] + w
            t[..., hi, lo2] = -(t[..., hi, hi2] @ kk[..., hi, lo2] @ t[..., lo, lo2])
            w *= 2
        Sl = S[:live]
        u = t @ (beta[..., None] * (v - eg * (k @ Sl)))
        o = s["scale"] * (eg * (q @ Sl) + ((q @ k.transpose(-1, -2)) * decay) @ u)
        S[:live] = eg[..., -1:, :] * Sl + (k * decay[..., -1, :, None]).transpose(-1, -2) @ u
        out[r[has]] = o.transpose(1, 2)[has]
    if c["gated"]:
        z = s["z"].view(n, nv, hd)
        out = out * torch.rsqrt((out * out).mean(-1, keepdim=True) + EPS) * s["norm"] * (z / (1.0 + torch.exp(-z)))
    s["state"][s["slots"].long()[order]] = S
    return [out, s["state"]]


def _logprobs(s):
    c = s["case"]
    raw, tok = s["logits"][:, :c["vocab"]], s["tokens"].long()[:, None]
    x = raw * s["scale"]
    x = x - x.amax(-1, keepdim=True)
    e = torch.exp(x)
    total = e.sum(-1, keepdim=True)
    lse = torch.log(total)
    mine = raw.gather(1, tok)
    first = torch.arange(c["vocab"], device="cuda") < tok
    out = {"logprob": (x.gather(1, tok) - lse)[:, 0], "entropy": (lse - (e * x).sum(-1, keepdim=True) / total)[:, 0],
           "rank": ((raw > mine) | ((raw == mine) & first)).sum(-1, dtype=torch.int32)}
    if c["top"]:
        at = torch.sort(raw, dim=-1, descending=True, stable=True)[1][:, :c["top"]]
        out["top_id"], out["top_logprob"] = at.int(), x.gather(1, at) - lse
    else:
        out["top_id"], out["top_logprob"] = s["out"]["top_id"], s["out"]["top_logprob"]
    return out


# ---------------------------------------------------------------------- work
def work(case):
    if case["kind"] == "logprobs":
        n, v, top = case["rows"], case["vocab"], case["top"]
        return {"bytes": 4 * n * (v + 4 + 2 * top), "flops": 5 * n * v}
    nqk, nv, hd, taps = case["nqk"], case["nv"], case["hd"], case["taps"]
    rows, channels = _rows(case), (2 * nqk + nv) * hd
    n = sum(rows)
    if case["kind"] == "conv":
        return {"bytes": 4 * (n * (2 * channels + 4 * nv) + channels * (taps + 2 * len(rows) * (taps - 1))), "flops": n * channels * (2 * taps + 6)}
    io = channels + nv * hd * (2 if case["gated"] else 1) + 2 * nv
    return {"bytes": 4 * (n * io + 2 * len(rows) * nv * hd * hd), "flops": 6 * n * nv * hd * hd}


# ---------------------------------------------------------------------- in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    return {"conv": _exact_conv, "rule": _exact_rule, "logprobs": _exact_logprobs}[case["kind"]](s)


def _exact_conv(s):
    c = s["case"]
    nqk, hd, taps = c["nqk"], c["hd"], c["taps"]
    win, outs = s["win"].double(), []
    w = s["conv1d"].double().T[:, None]  # [tap][1][channel]
    for b, slot in enumerate(s["slots"].tolist()):
        whole = torch.cat([win[slot, :taps - 1], s["qkv"][s["start"][b]:s["start"][b + 1]].double()])
        n = whole.shape[0] - (taps - 1)
        y = (torch.stack([whole[t:t + n] for t in range(taps)]) * w).sum(0)
        y = y * torch.sigmoid(y)
        heads = y.view(n, -1, hd)
        heads[:, :2 * nqk] /= torch.linalg.vector_norm(heads[:, :2 * nqk], dim=-1, keepdim=True).clamp(min=EPS)
        outs.append(y)
        win[slot, :taps - 1] = whole[n:]
    gate = torch.nn.functional.softplus(s["alpha"].double() + s["dt_bias"].double(), threshold=1e9) * s["a"].double()
    return [torch.cat(outs), torch.sigmoid(s["beta_raw"].double()), gate, win]


def _exact_rule(s):
    c = s["case"]
    nqk, nv, hd = c["nqk"], c["nv"], c["hd"]
    n = s["qkv"].shape[0]
    x = s["qkv"].double().view(n, -1, hd)
    times = -(-nv // nqk)
    q, k, v = x[:, :nqk].repeat(1, times, 1)[:, :nv], x[:, nqk:2 * nqk].repeat(1, times, 1)[:, :nv], x[:, 2 * nqk:]
    decay, beta = torch.exp(s["gate"].double()), s["beta"].double()
    states = s["state"].double()
    out = torch.empty(n, nv, hd, dtype=torch.float64, device="cuda")
    slots, starts = s["slots"].tolist(), s["start"]
    for i in range(max(s["rows"])):
        alive = [b for b, m in enumerate(s["rows"]) if m > i]
        r = torch.tensor([starts[b] + i for b in alive], device="cuda")
        at = torch.tensor([slots[b] for b in alive], device="cuda")
        S = states[at] * decay[r][:, :, None, None]
        error = beta[r][:, :, None] * (v[r] - (k[r][:, :, :, None] * S).sum(2))
        S += k[r][:, :, :, None] * error[:, :, None, :]
        out[r] = s["scale"] * (q[r][:, :, :, None] * S).sum(2)
        states[at] = S
    if c["gated"]:
        z = s["z"].double().view(n, nv, hd)
        out = out / torch.sqrt(out.square().mean(-1, keepdim=True) + EPS) * s["norm"].double() * (z * torch.sigmoid(z))
    return [out, states]


def _exact_logprobs(s):
    c = s["case"]
    v, top = c["vocab"], c["top"]
    outs = {"logprob": [], "entropy": [], "rank": None, "top_id": [], "top_logprob": []}
    for x, t in zip(s["logits"][:, :v], s["tokens"].tolist()):
        lp = torch.log_softmax(x.double() * s["scale"], 0)
        outs["logprob"].append(lp[t])
        outs["entropy"].append(-(lp.exp() * lp).sum())
        if top:
            ids = torch.topk(x, top)[1]
            outs["top_logprob"].append(lp[ids])
    return {"logprob": torch.stack(outs["logprob"]), "entropy": torch.stack(outs["entropy"]), "rank": None, "top_id": None,
            "top_logprob": torch.stack(outs["top_logprob"]) if top else None}
