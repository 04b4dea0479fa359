"""Performance cases of the batched serving operators: rows of several sequences over a paged cache.

`uq.serve` prepares the heads of a batch's new rows and appends them to the cache's pages, attends over
the pages (with the positions that all sequences share read once) and verifies drafted tokens. A case
is a dict of plain values; `prepare` makes what a serving program holds, `run` is one pass through one
operator: in elementary torch operations where `own` is false, by the library's entry points where it
is true. `exact` is the operator's definition in 64 bits.

Head counts and widths are those of the synthetic hybrid model of bench.py (16 query heads of 256 over
4, rotation over 64 values, vocabulary 152064) and of the tests (heads of 64 and 128).
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
    model = {"heads": 16, "kv": 4, "hd": 256}
    return [
        # one decoded token of one conversation: the smallest append, all latency
        {"name": "append 1", "kind": "append", "seqs": 1, "least": 1, "most": 1, "longest": 3071, "mix": 1, **model,
         "rot": 64, "rope": "imrope", "gate": True, "type": "f16", "page": 64},
        # a batch of sequences that verify up to four drafted tokens each, plain rotation over the whole head
        {"name": "append 29 drafts", "kind": "append", "seqs": 29, "least": 1, "most": 5, "longest": 9000, "mix": 2,
         "heads": 32, "kv": 8, "hd": 128, "rot": 128, "rope": "neox", "gate": False, "type": "f16", "page": 16},
        # the prompts of three requests prefilled in one batch, into a cache of the activations' own type
        {"name": "append prompts", "kind": "append", "seqs": 3, "least": 1024, "most": 2048, "longest": 5000, "mix": 3, **model,
         "rot": 64, "rope": "imrope", "gate": True, "type": "f32", "page": 64},
        # one decoded token of a short conversation: the smallest attention
        {"name": "attn 1 x 700", "kind": "attn", "seqs": 1, "least": 1, "most": 1, "longest": 700, "shared": 0, "mix": 4, **model,
         "gate": True, "type": "f16", "page": 64},
        # an ordinary decode batch: conversations of all lengths up to 8k
        {"name": "attn 32 ragged", "kind": "attn", "seqs": 32, "least": 1, "most": 1, "longest": 8192, "shared": 0, "mix": 5, **model,
         "gate": True, "type": "f16", "page": 64},
        # one token over a whole long document, cache of the activations' own type
        {"name": "attn 1 x 64k f32", "kind": "attn", "seqs": 1, "least": 1, "most": 1, "longest": 65537, "shared": 0, "mix": 6, **model,
         "gate": True, "type": "f32", "page": 256},
        # the last chunk of a prompt of 4k tokens
        {"name": "attn chunk 509", "kind": "attn", "seqs": 1, "least": 509, "most": 509, "longest": 4096, "shared": 0, "mix": 7, **model,
         "gate": True, "type": "f16", "page": 64},
        # conversations that begin with one long document
        {"name": "prefix 48 x 16k", "kind": "attn", "seqs": 48, "least": 1, "most": 1, "longest": 700, "shared": 16384, "mix": 8, **model,
         "gate": False, "type": "f16", "page": 64},
        # continuations of one system prompt with up to three drafted tokens each, narrower heads
        {"name": "prefix 7 drafts f32", "kind": "attn", "seqs": 7, "least": 1, "most": 4, "longest": 300, "shared": 2011, "mix": 9,
         "heads": 12, "kv": 2, "hd": 128, "gate": False, "type": "f32", "page": 32},
        # four drafted tokens of one conversation
        {"name": "verify 1 x 5", "kind": "verify", "seqs": 1, "least": 5, "most": 5, "mix": 10, "vocab": 152064, "draft": True},
        # a batch of them
        {"name": "verify 64 x 5", "kind": "verify", "seqs": 64, "least": 5, "most": 5, "mix": 11, "vocab": 152064, "draft": True},
        # drafts without probabilities (taken from the text so far), a smaller vocabulary, ragged
        {"name": "verify 13 ragged", "kind": "verify", "seqs": 13, "least": 1, "most": 8, "mix": 12, "vocab": 32003, "draft": False},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """A case of the same ranges, no larger than the largest listed one of its kind."""
    kind = rng.choice(["append", "append", "attn", "attn", "attn", "chunk", "prefix", "prefix", "verify", "verify"])
    c = {"kind": kind if kind in ("append", "verify") else "attn", "mix": rng.randrange(1 << 30)}
    if kind == "verify":
        most = rng.randint(1, 8)
        n = _log(rng, 1, 64)
        return dict(c, seqs=n, least=rng.randint(1, most), most=most, vocab=_log(rng, 500, 152064 * 320 // max(320, n * most)),
                    draft=rng.random() < 0.7)
    hd = rng.choice([64, 128, 256])
    kv = rng.choice([1, 2, 4, 8][:4 if hd < 256 else 3])  # at most 1024 values a cached position, 4096 a row of queries
    group = rng.choice([g for g in (1, 2, 3, 4, 6, 8) if kv * g * hd <= 4096])
    c.update(heads=kv * group, kv=kv, hd=hd, gate=rng.random() < 0.5, type=rng.choice(["f16", "f16", "f32"]),
             page=rng.choice([16, 32, 64, 128, 256]))
    if kind == "append":
        if rng.random() < 0.4:
            n = rng.randint(1, 3)
            most = _log(rng, 1, 4093 // n)
        else:
            n, most = _log(rng, 1, 64), rng.randint(1, 5)
        return dict(c, seqs=n, least=1, most=most, longest=most + _log(rng, 1, 4000), rope=rng.choice(["imrope", "neox", "llama", "none"]),
                    rot=rng.choice([hd // 4, hd // 2, hd]))
    if kind == "chunk":
        n = rng.choice([1, 1, 2])
        most = _log(rng, 17, 509 // n)
        return dict(c, seqs=n, least=17, most=most, shared=0, longest=most + _log(rng, 1, 3586))
    most = rng.choice([1, 1, 1, 5])
    n = _log(rng, 1, 48 // most)
    if kind == "attn":
        return dict(c, seqs=n, least=1, most=most, shared=0, longest=max(most, _log(rng, 8, 65537 // n)))
    return dict(c, seqs=n, least=1, most=most, shared=_log(rng, 64, 16384), longest=_log(rng, 5, 700))


def _rows(case):
    """New rows of each sequence."""
    rng = random.Random(case["mix"])
    return [_log(rng, case["least"], case["most"]) for _ in range(case["seqs"])]


def _lens(case):
    """Positions of each sequence, its new rows among them: the first as long as the case says, the others spread."""
    rng = random.Random(case["mix"] + 1)
    return [case.get("shared", 0) + max(n, case["longest"] if i == 0 else _log(rng, 1, case["longest"])) for i, n in enumerate(_rows(case))]


# ---------------------------------------------------------------------- inputs
class Buf:
    """A torch tensor where the binding takes a device array."""

    def __init__(self, t):
        self.t, self.ptr, self.nbytes = t, ctypes.c_void_p(t.data_ptr()), t.numel() * t.element_size()


def _serve():
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "unltd-inference_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    import uq
    from uq import serve

    return uq, serve


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)

    def normal(*shape):
        return torch.randn(*shape, generator=g, device="cuda")

    def whole(v):
        return torch.tensor(v, dtype=torch.int32, device="cuda")

    rows = _rows(case)
    n = sum(rows)
    start = [sum(rows[:i]) for i in range(len(rows) + 1)]
    s = {"case": case, "rows": rows, "start": start, "d_start": whole(start)}
    if case["kind"] == "verify":
        v = case["vocab"]
        logits = 3.0 * normal(n, v)
        s["p"] = torch.softmax(logits, -1)
        if case["draft"]:  # a smaller model's view of the same text
            s["q"] = torch.softmax(logits + 0.7 * normal(n, v), -1)
            del logits
            drawn = torch.cat([torch.multinomial(r, 1, generator=g) for r in s["q"].split(64)]).view(-1)
        else:
            s["q"], drawn = None, s["p"].argmax(-1)
        s["tokens"] = torch.cat([drawn[:1], drawn[:-1]]).int()  # row r's token: what row r - 1 was continued with
        s["u"] = torch.rand(n, generator=g, device="cuda")
        if own:
            _, serve = _serve()
            s["batch"] = serve.SeqBatch(n_seqs=len(rows), n_rows=n, d_row_start=Buf(s["d_start"]))
            s["accepted"], s["next"] = (torch.empty(len(rows), dtype=torch.int32, device="cuda") for _ in range(2))
            s["ws"] = torch.empty(serve.draft_verify_ws_bytes(s["batch"], v), dtype=torch.uint8, device="cuda")
            s["args"] = [Buf(s["accepted"]), Buf(s["next"]), Buf(s["p"]), Buf(s["q"]) if case["draft"] else None, Buf(s["tokens"]),
                         Buf(s["u"]), s["batch"], v, Buf(s["ws"])]
        return s

    heads, kv, hd, page, shared = case["heads"], case["kv"], case["hd"], case["page"], case.get("shared", 0)
    lens = s["lens"] = _lens(case)
    s["d_len"] = whole(lens)
    # pages in any order; those of the shared positions are every sequence's first, a page that they end in is copied
    whole_shared = shared // page
    need = [-(-x // page) - whole_shared for x in lens]
    most = whole_shared + max(need)
    total = whole_shared + sum(need) + 3
    order = torch.randperm(total, generator=g, device="cuda").tolist()
    common, rest, table = order[:whole_shared], order[whole_shared:], []
    for k in need:
        table.append(common + rest[:k] + [-1] * (most - whole_shared - k))
        rest = rest[k:]
    s["table"], s["d_table"] = table, whole(table)
    dtype = torch.float16 if case["type"] == "f16" else torch.float32
    s["k"], s["v"] = (normal(total, kv, page, hd).to(dtype) for _ in range(2))
    if shared % page:
        for t in table[1:]:
            for c in (s["k"], s["v"]):
                c[t[whole_shared], :, :shared % page] = c[table[0][whole_shared], :, :shared % page]
    wide = 2 * hd if case["gate"] else hd  # a head's query, its gate behind it
    s["qg"] = normal(n, heads, wide)
    if case["kind"] == "append":
        s["kin"], s["vin"] = normal(n, kv * hd), normal(n, kv * hd)
        s["wq"], s["wk"] = (1.0 + 0.1 * normal(hd) for _ in range(2))
        s["theta"] = 1.0e7 ** (-2.0 / case["rot"])
        s["freqs"] = (s["theta"] ** torch.arange(case["rot"] // 2, device="cuda", dtype=torch.float64)).float()
        s["q_out"] = torch.empty(n, heads, hd, device="cuda")
    else:
        s["q"] = 2.0 * normal(n, heads, hd)
        s["out"] = torch.empty(n, heads, hd, device="cuda")
        s["scale"] = 1.0 / math.sqrt(hd)
    if own:
        uq, serve = _serve()
        f = uq.DType.F16 if case["type"] == "f16" else uq.DType.F32
        s["kv"] = serve.KvPages(Buf(s["k"]), Buf(s["v"]), f, total, page, kv, hd)
        s["batch"] = serve.SeqBatch(n_seqs=len(rows), n_rows=n, d_row_start=Buf(s["d_start"]), d_len=Buf(s["d_len"]), d_pages=Buf(s["d_table"]), max_pages=most)
        if case["kind"] == "append":
            s["heads"] = serve.HeadRows(n_head=heads, d_q=Buf(s["qg"]), q_row=heads * wide, q_head=wide, d_k=Buf(s["kin"]), k_row=kv * hd,
                                        d_v=Buf(s["vin"]), v_row=kv * hd, d_q_norm=Buf(s["wq"]), d_k_norm=Buf(s["wk"]), eps=EPS,
                                        rope=case["rope"], n_rot=case["rot"], theta_scale=s["theta"], d_freqs=Buf(s["freqs"]), d_q_out=Buf(s["q_out"]))
        else:
            s["ws"] = Buf(torch.empty(serve.attn_paged_ws_bytes(s["kv"], s["batch"], heads, shared), dtype=torch.uint8, device="cuda"))
            s["bufs"] = [Buf(s["out"]), Buf(s["q"])]
            s["gate"] = dict(d_gate=Buf(s["qg"][:, :, hd:]), gate_row=heads * wide, gate_head=wide) if case["gate"] else {}
    return s


# ---------------------------------------------------------------------- one pass
def run(s):
    c = s["case"]
    if own:
        _, serve = _serve()
        if c["kind"] == "append":
            serve.kv_append_d(s["kv"], s["batch"], s["heads"])
            return [s["q_out"], s["k"], s["v"]]
        if c["kind"] == "attn":
            serve.attn_paged_d(*s["bufs"], s["kv"], s["batch"], c["heads"], s["scale"], s["ws"], shared_len=c["shared"], **s["gate"])
            return s["out"]
        serve.draft_verify_d(*s["args"])
        return [s["accepted"], s["next"]]
    return {"append": _append, "attn": _attend, "verify": _verify}[c["kind"]](s)


def _append(s):
    c = s["case"]
    hd, kv, page = c["hd"], c["kv"], c["page"]
    rows = s["d_start"].diff().long()
    n = s["qg"].shape[0]
    seq = torch.repeat_interleave(torch.arange(len(rows), device="cuda"), rows, output_size=n)
    at = (s["d_len"].long() - rows - s["d_start"][:-1])[seq] + torch.arange(n, device="cuda")
    ang, mine = None, None
    if c["rope"] != "none":
        half = c["rot"] // 2
        i = torch.arange(0, half, 3 if c["rope"] == "imrope" else 1, device="cuda")
        f = s["theta"] ** i.double() if c["rope"] == "imrope" else s["freqs"].double()
        ang = at.double()[:, None, None] * f
        mine = (2 * i, 2 * i + 1) if c["rope"] == "llama" else (i, i + half)

    def prep(x, w):
        x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * w
        if ang is not None:
            cos, sin, a, b = torch.cos(ang).float(), torch.sin(ang).float(), x[..., mine[0]], x[..., mine[1]]
            x[..., mine[0]], x[..., mine[1]] = a * cos - b * sin, a * sin + b * cos
        return x

    q = prep(s["qg"][:, :, :hd], s["wq"])
    pg = s["d_table"][seq, at // page].long()
    s["k"][pg, :, at % page] = prep(s["kin"].view(n, kv, hd), s["wk"]).to(s["k"].dtype)
    s["v"][pg, :, at % page] = s["vin"].view(n, kv, hd).to(s["v"].dtype)
    return [q, s["k"], s["v"]]


def _attend(s):
    c = s["case"]
    hd, kv = c["hd"], c["kv"]
    group, out = c["heads"] // kv, []
    for b, (n, ln) in enumerate(zip(s["rows"], s["lens"])):
        t = s["d_table"][b, :-(-ln // c["page"])].long()
        k, v = (x[t].float().transpose(0, 1).reshape(kv, -1, hd)[:, :ln] for x in (s["k"], s["v"]))
        q = s["q"][s["start"][b]:s["start"][b + 1]].view(n, kv, group, hd).permute(1, 0, 2, 3).reshape(kv, n * group, hd)
        sc = (q @ k.transpose(1, 2).contiguous() * s["scale"]).view(kv, n, group, ln)
        hide = torch.arange(ln, device="cuda")[None, :] > ln - n + torch.arange(n, device="cuda")[:, None]
        sc = sc.masked_fill(hide[None, :, None], -math.inf)
        p = torch.exp(sc - sc.amax(-1, keepdim=True))
        p = (p / p.sum(-1, keepdim=True)).view(kv, n * group, ln)
        out.append((p @ v.contiguous()).view(kv, n, group, hd).permute(1, 0, 2, 3).reshape(n, kv * group, hd))
    out = torch.cat(out)
    return out / (1.0 + torch.exp(-s["qg"][:, :, hd:])) if c["gate"] else out


def _verify(s):
    p, q, tok, u, rows = s["p"], s["q"], s["tokens"].long(), s["u"].double(), s["d_start"].diff().long()
    n, first, last = p.shape[0], s["d_start"][:-1].long(), s["d_start"][1:].long() - 1
    nxt = torch.cat([tok[1:], tok[:1]])  # what row r's drafted continuation is
    at = torch.arange(n, device="cuda")
    qx = q[at, nxt].double() if q is not None else 1.0
    no = ~(u * qx < p[at, nxt].double())
    no[last] = True  # a sequence's last row has no continuation to test
    # the first refused row of each sequence
    before = torch.cat([no.new_zeros(1, dtype=torch.long), torch.cumsum(no.long(), 0)])
    refused = torch.nonzero(no).view(-1)
    row = refused[before[first]]
    ended = row == last
    w = p[row].double()
    if q is not None:
        w = torch.where(ended[:, None], w, (w - q[row].double()).clamp(min=0.0))
    else:
        w[torch.arange(len(row), device="cuda")[~ended], nxt[row][~ended]] = 0.0
    w = torch.where(w.sum(-1, keepdim=True) > 0, w, p[row].double())
    acc = torch.cumsum(w, -1)
    token = (acc > u[last][:, None] * acc[:, -1:]).int().argmax(-1)
    return [(row - first).int(), token.int()]


# ---------------------------------------------------------------------- work
def work(case):
    rows = _rows(case)
    n = sum(rows)
    if case["kind"] == "verify":  # the row that is drawn from, a number or two of each other
        reads = (2 if case["draft"] else 1) * case["vocab"] * len(rows) + 4 * n
        return {"bytes": 4 * reads + 8 * len(rows), "flops": 3 * case["vocab"] * len(rows)}
    heads, kv, hd = case["heads"], case["kv"], case["hd"]
    size = 2 if case["type"] == "f16" else 4
    if case["kind"] == "append":
        per = hd * (4 * (2 * heads + 2 * kv) + 2 * kv * size)
        return {"bytes": n * per, "flops": n * (heads + kv) * (4 * hd + 3 * case["rot"])}
    lens, shared = _lens(case), case["shared"]
    held = shared + sum(x - shared for x in lens)
    seen = sum(k * x - k * (k - 1) // 2 for k, x in zip(rows, lens))
    return {"bytes": 2 * held * kv * hd * size + n * heads * hd * 4 * (3 if case["gate"] else 2), "flops": 4 * seen * heads * hd}


# ---------------------------------------------------------------------- in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "verify":
        return _exact_verify(s)
    if case["kind"] == "append":
        return _exact_append(s)
    return _exact_attention(s)


def _exact_verify(s):
    accepted, tokens = [], []
    u, tok = s["u"].double().tolist(), s["tokens"].tolist()
    for a, b in zip(s["start"], s["start"][1:]):
        r = a
        while r + 1 < b and u[r] * (1.0 if s["q"] is None else float(s["q"][r, tok[r + 1]])) < float(s["p"][r, tok[r + 1]]):
            r += 1
        w = p = s["p"][r].double().cpu()
        if r + 1 < b:
            w = p.clone()
            if s["q"] is None:
                w[tok[r + 1]] = 0.0
            else:
                w = torch.relu(w - s["q"][r].double().cpu())
            w = w if float(w.sum()) > 0 else p
        c = torch.cumsum(w, 0)
        accepted.append(r - a)
        tokens.append(int(torch.searchsorted(c, u[b - 1] * c[-1], right=True)))
    return [torch.tensor(x, dtype=torch.int32) for x in (accepted, tokens)]


def _exact_append(s):
    c, out = s["case"], []
    hd, page, half = c["hd"], c["page"], c["rot"] // 2
    k, v = s["k"].double(), s["v"].double()

    def turned(x, w, pos):
        x = x.double()
        x = x / torch.sqrt(torch.linalg.vector_norm(x, dim=-1, keepdim=True) ** 2 / hd + EPS) * w.double()
        y = x.clone()
        for i in range(0, half if c["rope"] != "none" else 0, 3 if c["rope"] == "imrope" else 1):
            f = s["theta"] ** i if c["rope"] == "imrope" else float(s["freqs"][i])
            z = torch.polar(torch.ones_like(pos), pos * f)[:, None]
            a, b = (2 * i, 2 * i + 1) if c["rope"] == "llama" else (i, half + i)
            z = z * torch.complex(x[..., a], x[..., b])
            y[..., a], y[..., b] = z.real, z.imag
        return y

    for b, ln in enumerate(s["lens"]):
        r = slice(s["start"][b], s["start"][b + 1])
        n = r.stop - r.start
        at = torch.arange(ln - n, ln, device="cuda")
        pg = torch.tensor(s["table"][b], device="cuda")[at // page]
        out.append(turned(s["qg"][r, :, :hd], s["wq"], at.double()))
        k[pg, :, at % page] = turned(s["kin"][r].view(n, -1, hd), s["wk"], at.double())
        v[pg, :, at % page] = s["vin"][r].view(n, -1, hd).double()
    return [torch.cat(out), k, v]


def _exact_attention(s):
    c = s["case"]
    hd, page, group = c["hd"], c["page"], c["heads"] // c["kv"]
    out = torch.empty(s["q"].shape, dtype=torch.float64, device="cuda")
    for b, ln in enumerate(s["lens"]):
        a, e = s["start"][b], s["start"][b + 1]
        slots = torch.arange(ln, device="cuda")
        pages = torch.tensor(s["table"][b], device="cuda")[slots // page]
        last = torch.arange(ln - (e - a), ln, device="cuda")
        for h in range(c["kv"]):
            keys, values = (x[pages, h, slots % page].double() for x in (s["k"], s["v"]))
            for j in range(group):
                score = s["q"][a:e, h * group + j].double() @ keys.T * s["scale"]
                score[slots[None] > last[:, None]] = -math.inf
                out[a:e, h * group + j] = torch.softmax(score, 1) @ values
    return out * torch.sigmoid(s["qg"][:, :, hd:].double()) if c["gate"] else out
