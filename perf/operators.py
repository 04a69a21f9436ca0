"""Decoding several continuations of one prompt: the operators' cases, their plain forms and their 64-bit values.

A program that answers a prompt with several sequences (beam search, samples side by side, drafts that
are verified) keeps the prompt's keys and values once, in pages, and each sequence's own ones in pages of
its own. A step of it is

* append   the new tokens' queries, keys and values: per-head norms, position rotation, keys and values
           into the pages (`qmh_paged_append`);
* attend   the queries over the shared prefix, computed for all sequences of a group together, and over
           each sequence's own pages (`qmh_paged_attention`);
* select   the best continuations over beams and vocabulary (`qmh_beam_select`);
* reorder  the states of the beams that survive: dense caches (`qmh_beam_reorder`) or pages
           (`qmh_paged_reorder`).

Head shapes are those of the workloads c1 to c5 (`quillm_amd.WORKLOADS`), and some odd ones; the
vocabularies those of the framework's tests. Where `own` is false the passes are elementary torch
operations in 32 bits (64 for angles and for the scores that decide a choice); where it is true they are
the calls that a user of the library makes.
"""
import ctypes
import math

import torch

own = False

# query heads, kv heads, head_dim: c1, c2, c3, c4, c5, and two with remainders
HEADS = {"c1": (6, 6, 48), "c2": (6, 2, 48), "c3": (12, 12, 64), "c4": (32, 4, 64), "c5": (32, 32, 128),
         "o1": (5, 1, 80), "o2": (14, 2, 96)}
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
EPS = 1e-5
MAX_POS = 131072


def listed():
    return [
        # one token of a small model's single conversation: nothing but latency
        {"name": "append one", "kind": "append", "heads": "c2", "dtype": "f32", "tokens": 1, "seqs": 1, "page": 16, "far": 200,
         "layout": "pairs", "scaling": "none", "rot": 48, "norm": False},
        # a server's step: 96 sequences of a grouped-query model, normed heads, half the head rotated, a stretched context
        {"name": "append step", "kind": "append", "heads": "c4", "dtype": "bf16", "tokens": 96, "seqs": 96, "page": 32,
         "far": 100000, "layout": "halves", "scaling": "bands", "rot": 32, "norm": True},
        # three ragged prompts into the pages of a 7B-shaped model
        {"name": "append prompt", "kind": "append", "heads": "c5", "dtype": "f16", "tokens": 4001, "seqs": 3, "page": 64,
         "far": 9000, "layout": "halves", "scaling": "yarn", "rot": 128, "norm": False},
        # four beams of a small model, a few tokens into the answer
        {"name": "attend small", "kind": "attend", "heads": "c2", "dtype": "f32", "groups": 1, "beams": 4, "q": 1, "page": 16,
         "prefix": 37, "len": 9},
        # drafts of three tokens verified for three prompts of four sequences, full precision
        {"name": "attend drafts", "kind": "attend", "heads": "c3", "dtype": "f32", "groups": 3, "beams": 4, "q": 3, "page": 16,
         "prefix": 1023, "len": 130},
        # 64 answers to one long document on a grouped-query model
        {"name": "attend document", "kind": "attend", "heads": "c4", "dtype": "f16", "groups": 1, "beams": 64, "q": 1, "page": 32,
         "prefix": 16380, "len": 300},
        # two prompts of 16 answers each, well into the answers, 7B-shaped heads
        {"name": "attend answers", "kind": "attend", "heads": "c5", "dtype": "bf16", "groups": 2, "beams": 16, "q": 1, "page": 64,
         "prefix": 4096, "len": 700},
        # a step of one four-beam search over the workloads' vocabulary
        {"name": "select small", "kind": "select", "dtype": "f32", "groups": 1, "beams": 4, "vocab": 32000, "out": 8, "done": False},
        # a batch of searches, 16-bit logits (ties are common), finished beams among them
        {"name": "select batch", "kind": "select", "dtype": "bf16", "groups": 16, "beams": 5, "vocab": 32003, "out": 10, "done": True},
        # the largest: 24 prompts of 8 beams over a large vocabulary
        {"name": "select wide", "kind": "select", "dtype": "f32", "groups": 24, "beams": 8, "vocab": 128256, "out": 16, "done": False},
        # a beam search's dense key caches ([kv width][max_seq] per sequence) into the other of two buffers
        {"name": "reorder dense", "kind": "reorder", "form": "dense", "inplace": False, "heads": "c1", "layers": 6, "groups": 2,
         "beams": 4, "live": 131, "max_seq": 256},
        # the pages of 8 prompts' 6 beams after a step, in place
        {"name": "reorder pages", "kind": "reorder", "form": "pages", "inplace": True, "heads": "c5", "dtype": "f16", "groups": 8,
         "beams": 6, "page": 32, "len": 451, "moved": 3},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["append", "append", "attend", "attend", "attend", "select", "select", "reorder", "reorder"])
    most = {}
    for c in listed():
        if c["kind"] == kind:
            w = work(c)
            most = {k: max(w[k], most.get(k, 0)) for k in w}
    while True:
        c = _draw(rng, kind)
        w = work(c)
        if w["bytes"] <= most["bytes"] and w["flops"] <= most["flops"]:
            return c


def _draw(rng, kind):
    heads = rng.choice(sorted(HEADS))
    hd = HEADS[heads][2]
    dtype = rng.choice(sorted(TYPES))
    if kind == "append":
        n = _log(rng, 1, 4001)
        return {"kind": kind, "heads": heads, "dtype": dtype, "tokens": n, "seqs": rng.choice([1, n, rng.randint(1, n)]),
                "page": rng.choice([16, 32, 64, 128]), "far": _log(rng, 2, MAX_POS - 4096),
                "layout": rng.choice(["pairs", "halves"]), "scaling": rng.choice(["none", "linear", "ntk", "bands", "yarn"]),
                "rot": rng.choice([hd, hd, hd // 2, hd // 4]), "norm": rng.choice([False, True])}
    if kind == "attend":
        return {"kind": kind, "heads": heads, "dtype": dtype, "groups": rng.randint(1, 6), "beams": _log(rng, 1, 64),
                "q": rng.choice([1, 1, 1, 2, 3, 5, 8]), "page": rng.choice([16, 32, 64, 128]),
                "prefix": rng.choice([0, _log(rng, 1, 16380), _log(rng, 1, 16380), _log(rng, 1, 16380)]), "len": _log(rng, 8, 1500)}
    if kind == "select":
        beams = _log(rng, 1, 16)
        return {"kind": kind, "dtype": dtype, "groups": _log(rng, 1, 64), "beams": beams, "vocab": _log(rng, 300, 128256),
                "out": beams * rng.choice([1, 2]), "done": rng.choice([False, True])}
    beams = _log(rng, 1, 16)
    if rng.random() < 0.5:
        live = _log(rng, 1, 1500)
        return {"kind": kind, "form": "dense", "inplace": rng.choice([False, True]), "heads": heads, "layers": rng.randint(1, 8),
                "groups": rng.randint(1, 8), "beams": beams, "live": live, "max_seq": live + rng.randint(0, 300),
                "moved": rng.randint(0, beams - 1)}
    return {"kind": kind, "form": "pages", "inplace": True, "heads": heads, "dtype": dtype, "groups": rng.randint(1, 8),
            "beams": beams, "page": rng.choice([16, 32, 64, 128]), "len": _log(rng, 1, 1500), "moved": rng.randint(0, beams - 1)}


# ------------------------------------------------------------------------------------- inputs

def _gen(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed) * 1000003 + sum(ord(c) * (i + 1) for i, c in enumerate(repr(sorted(case.items(), key=str)))))
    return g


def _randn(g, dtype, *size):
    return torch.randn(*size, device="cuda", generator=g).to(dtype)


def _randint(g, lo, hi, *size):
    """Whole numbers in [lo, hi]."""
    return torch.randint(lo, hi + 1, size, device="cuda", generator=g, dtype=torch.int32)


def _pages_for(g, counts, width, n_pages):
    """Tables [len(counts), width] of distinct pages of a pool of n_pages, in random order: counts[i] of them in row i
    and -1 behind. The pool is as large as the longest sequences would need, so some pages belong to nobody."""
    perm = torch.randperm(n_pages, device="cuda", generator=g).to(torch.int32)
    t = torch.full((max(1, len(counts)), max(1, width)), -1, dtype=torch.int32, device="cuda")
    at = 0
    for i, c in enumerate(counts):
        t[i, :c] = perm[at:at + c]
        at += c
    return t


def _append_layout(case):
    """Tokens of each sequence: ragged runs that add up to the case's tokens."""
    n, s = case["tokens"], case["seqs"]
    runs = [n // s] * s
    for i in range(n - sum(runs)):
        runs[i] += 1
    for i in range(0, s - 1, 2):  # every other boundary moves by a third of a run
        d = runs[i] // 3
        runs[i] -= d
        runs[i + 1] += d
    return runs


def _append_inputs(case, seed):
    H, KV, hd = HEADS[case["heads"]]
    dt, ps, g = TYPES[case["dtype"]], case["page"], _gen(case, seed)
    runs = _append_layout(case)
    n = case["tokens"]
    # what a sequence holds already: pages that are part full
    start = [int(v) for v in _randint(g, 0, 2 * ps, len(runs)).tolist()]
    counts = [(st + r + ps - 1) // ps for st, r in zip(start, runs)]
    n_pages = sum((r + 3 * ps - 1) // ps for r in runs)
    table = _pages_for(g, counts, (max(runs) + 3 * ps - 1) // ps, n_pages)
    seq = torch.repeat_interleave(torch.arange(len(runs), device="cuda"), torch.tensor(runs, device="cuda")).to(torch.int32)
    first = torch.tensor(start, device="cuda", dtype=torch.int32)
    base = torch.cumsum(torch.tensor([0] + runs[:-1], device="cuda"), 0).to(torch.int32)
    slot = (torch.arange(n, device="cuda", dtype=torch.int32) - base[seq.long()] + first[seq.long()]).contiguous()
    # the shared prefix lies before the sequence's own pages: positions are far beyond the slots
    pos = (slot + case["far"]).to(torch.int32)
    qkv = _randn(g, dt, n, (H + 2 * KV) * hd)  # one fused projection's rows
    gain = [1.0 + 0.1 * torch.randn(hd, device="cuda", generator=g) for _ in range(2)]
    k = _randn(g, dt, n_pages, KV, ps, hd)
    v = _randn(g, dt, n_pages, KV, ps, hd)
    return {"qkv": qkv, "gain": gain if case["norm"] else None, "k": k, "v": v, "table": table, "seq": seq, "slot": slot,
            "pos": pos}


def _attend_inputs(case, seed):
    H, KV, hd = HEADS[case["heads"]]
    dt, ps, g = TYPES[case["dtype"]], case["page"], _gen(case, seed)
    G, B = case["groups"], case["groups"] * case["beams"]
    P, L = case["prefix"], max(case["len"], case["q"])
    plen = _randint(g, (P + 1) // 2, P, G) if P else torch.zeros(G, dtype=torch.int32, device="cuda")
    plen[0] = P
    olen = _randint(g, max(case["q"], (L + 1) // 2), L, B)
    olen[-1] = L
    pc, oc = [(int(x) + ps - 1) // ps for x in plen.tolist()], [(int(x) + ps - 1) // ps for x in olen.tolist()]
    n_pages = G * ((P + ps - 1) // ps) + B * ((L + ps - 1) // ps)
    tables = _pages_for(g, pc + oc, max(pc + oc), n_pages)
    k, v = _randn(g, dt, n_pages, KV, ps, hd), _randn(g, dt, n_pages, KV, ps, hd)
    q = _randn(g, dt, B * case["q"], H * hd) * 1.5
    return {"q": q, "k": k, "v": v, "ptable": tables[:G].contiguous(), "table": tables[G:].contiguous(), "plen": plen, "len": olen,
            "P": P, "L": L}


def _select_inputs(case, seed):
    g = _gen(case, seed)
    rows = case["groups"] * case["beams"]
    x = torch.randn(rows, case["vocab"], device="cuda", generator=g) * 2.5
    x[:, 3] = -math.inf  # a token that the grammar or a stop list rules out
    score = -5.0 * torch.rand(rows, device="cuda", generator=g)
    done = (torch.rand(rows, device="cuda", generator=g) < 0.3).to(torch.int32) if case["done"] else None
    return {"logits": x.to(TYPES[case["dtype"]]), "score": score, "done": done}


def _parents(case, g):
    G, K = case["groups"], case["beams"]
    if not case["inplace"]:
        return _randint(g, 0, K - 1, G * K)
    # survivors keep their places, `moved` others take a survivor's state
    out = torch.empty(G, K, dtype=torch.int32, device="cuda")
    for i in range(G):
        perm = torch.randperm(K, device="cuda", generator=g)
        gone, stay = perm[:case["moved"]], perm[case["moved"]:]
        out[i, stay] = stay.to(torch.int32)
        if len(gone):
            out[i, gone] = stay[torch.randint(0, len(stay), (len(gone),), device="cuda", generator=g)].to(torch.int32)
    return out.flatten().contiguous()


def _reorder_inputs(case, seed):
    _, KV, hd = HEADS[case["heads"]]
    g = _gen(case, seed)
    s = {"parent": _parents(case, g)}
    G, K = case["groups"], case["beams"]
    if case["form"] == "dense":
        size = (case["layers"], G * K, KV * hd, case["max_seq"])
        s["src"] = _randn(g, torch.float32, *size)
        s["dst"] = s["src"] if case["inplace"] else _randn(g, torch.float32, *size)
        return s
    ps, n = case["page"], case["len"]
    # the beams of a prompt are equally long
    length = _randint(g, (n + 1) // 2, n, G)
    length[0] = n
    s["len"] = length.repeat_interleave(K).contiguous()
    counts = [(int(x) + ps - 1) // ps for x in s["len"].tolist()]
    n_pages = G * K * ((n + ps - 1) // ps)
    s["table"] = _pages_for(g, counts, max(counts), n_pages)
    dt = TYPES[case["dtype"]]
    s["k"], s["v"] = _randn(g, dt, n_pages, KV, ps, hd), _randn(g, dt, n_pages, KV, ps, hd)
    return s


_INPUTS = {"append": _append_inputs, "attend": _attend_inputs, "select": _select_inputs, "reorder": _reorder_inputs}

# a stretched context's parameters: factor, low and high (rotations over the first context), its length, magnitude
THETA, FACTOR, LOW, HIGH, FIRST = 10000.0, 8.0, 1.0, 4.0, 8192
YARN_LOW, YARN_HIGH = 1.0, 32.0


def _magnitude(case):
    return 0.1 * math.log(FACTOR) + 1.0 if case["scaling"] == "yarn" else 1.0


def _f32(x):
    """x as a float holds it: the library takes its parameters so."""
    return ctypes.c_float(x).value


def prepare(case, seed):
    s = _INPUTS[case["kind"]](case, seed)
    s["case"], kind = case, case["kind"]
    if kind == "append":
        H, KV, hd = HEADS[case["heads"]]
        s["q_out"] = torch.zeros(case["tokens"], H * hd, device="cuda", dtype=TYPES[case["dtype"]])
        s["freq"] = _freqs(case)
    elif kind == "attend":
        s["out"] = torch.zeros_like(s["q"])
    elif kind == "select":
        n = (case["groups"], case["out"])
        s["score_out"] = torch.zeros(n, device="cuda")
        s["parent_out"], s["token_out"] = (torch.zeros(n, device="cuda", dtype=torch.int32) for _ in range(2))
    if own:
        _prepare_own(case, s)
    torch.cuda.synchronize()  # the library has a stream of its own
    return s


# ------------------------------------------------------------------------------------- the plain forms

def _freqs(case):
    """Radians per position of each rotated pair, in 64 bits."""
    r, kind = case["rot"], case["scaling"]
    i = torch.arange(r // 2, device="cuda", dtype=torch.float64)
    theta = THETA * FACTOR ** (r / (r - 2)) if kind == "ntk" else THETA
    f = theta ** (-2.0 * i / r)
    if kind == "linear":
        f = f / FACTOR
    elif kind == "bands":  # pairs that turn often stay, those that turn rarely are slowed, a ramp between
        keep = ((f * FIRST / (2 * math.pi) - LOW) / (HIGH - LOW)).clamp(0, 1)
        f = f * keep + f / FACTOR * (1 - keep)
    elif kind == "yarn":  # the ramp runs over the pairs' numbers

        def pair(turns):
            return r * math.log(FIRST / (turns * 2 * math.pi)) / (2 * math.log(THETA))

        lo, hi = max(math.floor(pair(YARN_HIGH)), 0), min(math.ceil(pair(YARN_LOW)), r - 1)
        keep = 1 - ((i - lo) / max(hi - lo, 0.001)).clamp(0, 1)
        f = f * keep + f / FACTOR * (1 - keep)
    return f


def _plain_append(s):
    case = s["case"]
    H, KV, hd = HEADS[case["heads"]]
    n, r, ps = case["tokens"], case["rot"], case["page"]
    x = s["qkv"].float().view(n, H + 2 * KV, hd)
    q, k, v = x[:, :H], x[:, H:H + KV], x[:, H + KV:]
    if s["gain"] is not None:
        q = q * torch.rsqrt((q * q).mean(-1, keepdim=True) + EPS) * s["gain"][0]
        k = k * torch.rsqrt((k * k).mean(-1, keepdim=True) + EPS) * s["gain"][1]
    ang = s["pos"].double()[:, None] * s["freq"]
    mag = _f32(_magnitude(case))
    c, w = (torch.cos(ang) * mag).float()[:, None], (torch.sin(ang) * mag).float()[:, None]

    def rotate(y):
        a, b = (y[..., :r // 2], y[..., r // 2:r]) if case["layout"] == "halves" else (y[..., 0:r:2], y[..., 1:r:2])
        both = [a * c - b * w, a * w + b * c]
        turned = torch.cat(both, -1) if case["layout"] == "halves" else torch.stack(both, -1).flatten(-2)
        return torch.cat([turned, y[..., r:]], -1)

    dt = s["k"].dtype
    page = s["table"][s["seq"].long(), (s["slot"] // ps).long()].long()
    off = (s["slot"] % ps).long()
    s["q_out"].copy_(rotate(q).flatten(1))
    s["k"][page, :, off] = rotate(k).to(dt)
    s["v"][page, :, off] = v.to(dt)
    return {"q": s["q_out"], "k": s["k"], "v": s["v"]}


def _gather(pages, table, n):
    """[rows, kv heads, n, head_dim] in 32 bits of the tables' first n positions."""
    x = pages[table[:, :(n + pages.shape[2] - 1) // pages.shape[2]].clamp(min=0).long()]
    return x.permute(0, 2, 1, 3, 4).flatten(2, 3)[:, :, :n].float()


def _plain_attend(s):
    case = s["case"]
    H, KV, hd = HEADS[case["heads"]]
    G, K, Q, P, L = case["groups"], case["beams"], case["q"], s["P"], s["L"]
    B, M, scale = G * K, H // KV, 1.0 / math.sqrt(hd)
    q = s["q"].float().view(B, Q, KV, M, hd).permute(0, 2, 1, 3, 4).contiguous()  # [B, KV, Q, M, hd]
    ko, vo = _gather(s["k"], s["table"], L), _gather(s["v"], s["table"], L)
    so = torch.bmm(q.view(B * KV, Q * M, hd), ko.flatten(0, 1).transpose(1, 2).contiguous()).view(B, KV, Q, M, L) * scale
    last = s["len"][:, None] - Q + 1 + torch.arange(Q, device="cuda")  # positions each query sees
    so.masked_fill_((torch.arange(L, device="cuda") >= last[..., None])[:, None, :, None], -math.inf)
    m = so.amax(-1, keepdim=True)
    if P:
        kp, vp = _gather(s["k"], s["ptable"], P), _gather(s["v"], s["ptable"], P)
        qg = q.view(G, K, KV, Q * M, hd).transpose(1, 2).reshape(G * KV, K * Q * M, hd)
        sp = torch.bmm(qg, kp.flatten(0, 1).transpose(1, 2).contiguous()).view(G, KV, K * Q * M, P) * scale
        sp.masked_fill_((torch.arange(P, device="cuda") >= s["plen"][:, None])[:, None, None], -math.inf)
        mp = sp.amax(-1, keepdim=True).view(G, KV, K, Q, M, 1).transpose(1, 2).reshape(B, KV, Q, M, 1)
        m = torch.maximum(m, mp)
    m = torch.where(m == -math.inf, torch.zeros_like(m), m)
    eo = torch.exp(so - m)
    total = eo.sum(-1, keepdim=True)
    acc = torch.bmm(eo.view(B * KV, Q * M, L), vo.flatten(0, 1).contiguous()).view(B, KV, Q, M, hd)
    if P:
        ep = torch.exp(sp - m.view(G, K, KV, Q * M, 1).transpose(1, 2).reshape(G, KV, K * Q * M, 1))
        t = ep.sum(-1, keepdim=True).view(G, KV, K, Q, M, 1).transpose(1, 2).reshape(B, KV, Q, M, 1)
        a = torch.bmm(ep.view(G * KV, K * Q * M, P), vp.flatten(0, 1).contiguous())
        total = total + t
        acc = acc + a.view(G, KV, K, Q, M, hd).transpose(1, 2).reshape(B, KV, Q, M, hd)
    s["out"].copy_((acc / total).permute(0, 2, 1, 3, 4).reshape(B * Q, H * hd))
    return s["out"]


def _plain_select(s):
    case = s["case"]
    G, K, V, n = case["groups"], case["beams"], case["vocab"], case["out"]
    x = s["logits"].float() + 0.0
    # the scores decide a choice: 64 bits. Within a beam the logits' order decides, the lower token where they tie
    m = x.amax(-1, keepdim=True).double()
    lse = m + torch.log(torch.exp(x.double() - m).sum(-1, keepdim=True))
    bits = x.view(torch.int32)
    key = torch.where(bits < 0, bits ^ 0x7FFFFFFF, bits).long() * (1 << 32) + (V - 1 - torch.arange(V, device="cuda"))
    take = min(n, V)
    token = torch.topk(key, take, -1)[1]
    total = s["score"].double()[:, None] + (torch.gather(x, 1, token).double() - lse)
    if s["done"] is not None:  # a finished beam stands as it is: its one continuation is the end token
        fin = s["done"][:, None] != 0
        first = torch.arange(take, device="cuda") == 0
        total = torch.where(fin, torch.where(first, s["score"].double()[:, None], -math.inf), total)
        token = torch.where(fin, torch.full_like(token, EOS), token)
    flat = token + V * torch.arange(K, device="cuda").repeat(G)[:, None]
    flat, total = flat.view(G, K * take), total.view(G, K * take)
    order = torch.argsort(flat, dim=-1, stable=True)
    flat, total = torch.gather(flat, 1, order), torch.gather(total, 1, order)
    best, order = torch.sort(total, dim=-1, descending=True, stable=True)
    best, flat = best[:, :n], torch.gather(flat, 1, order)[:, :n]
    got = best > -math.inf
    s["score_out"].copy_(best)
    s["parent_out"].copy_(torch.where(got, flat // V, -1))
    s["token_out"].copy_(torch.where(got, flat % V, -1))
    return {"score": s["score_out"], "parent": s["parent_out"], "token": s["token_out"]}


EOS = 2


def _plain_reorder(s):
    case = s["case"]
    G, K = case["groups"], case["beams"]
    first = torch.arange(G, device="cuda").repeat_interleave(K) * K
    src = first + s["parent"].long()
    if case["form"] == "dense":
        n = case["live"]
        s["dst"][:, :, :, :n] = s["src"][:, :, :, :n][:, src]
        return s["dst"]
    ps, n = case["page"], case["len"]
    t = torch.arange(n, device="cuda")
    live = t < s["len"][:, None]
    to = s["table"].long()[:, t // ps][live]
    frm = s["table"].long()[src][:, t // ps][live]
    off = (t % ps).expand(G * K, n)[live]
    s["k"][to, :, off] = s["k"][frm, :, off]
    s["v"][to, :, off] = s["v"][frm, :, off]
    return {"k": s["k"], "v": s["v"]}


_PLAIN = {"append": _plain_append, "attend": _plain_attend, "select": _plain_select, "reorder": _plain_reorder}


# ------------------------------------------------------------------------------------- the library's calls

def _prepare_own(case, s):
    import quillm_amd as q

    q.init(0)
    lib, kind = q.load_library(), case["kind"]
    dt = {"f32": q.F32, "f16": q.F16, "bf16": q.BF16}[case.get("dtype", "f32")]

    def pages():
        p = q.Pages(dtype=dt, n_kv_heads=s["k"].shape[1], head_dim=s["k"].shape[3], page_size=s["k"].shape[2],
                    n_pages=s["k"].shape[0], k=s["k"].data_ptr(), v=s["v"].data_ptr())
        s["pages"] = p
        return ctypes.pointer(p)

    if kind == "append":
        H, KV, hd = HEADS[case["heads"]]
        yarn = case["scaling"] == "yarn"
        s["rotary"] = q.Rotary(case["rot"], case["layout"], case["scaling"], MAX_POS, theta=THETA, factor=FACTOR,
                               low=YARN_LOW if yarn else LOW, high=YARN_HIGH if yarn else HIGH, first_len=FIRST,
                               magnitude=_magnitude(case))
        x, step, size = s["qkv"].data_ptr(), s["qkv"].shape[1], s["qkv"].element_size()
        gains = [t.data_ptr() for t in s["gain"]] if s["gain"] else [None, None]
        a = q.AppendArgs(pages=pages(), rotary=s["rotary"].handle, n_tokens=case["tokens"], n_heads=H, q=x, q_stride=step,
                         q_out=s["q_out"].data_ptr(), q_out_stride=H * hd, k=x + H * hd * size, k_stride=step,
                         v=x + (H + KV) * hd * size, v_stride=step, q_gain=gains[0], k_gain=gains[1], eps=EPS,
                         n_seq=case["seqs"], table=s["table"].data_ptr(), table_stride=s["table"].shape[1],
                         seq=s["seq"].data_ptr(), slot=s["slot"].data_ptr(), pos=s["pos"].data_ptr())
        s["call"] = lib.qmh_paged_append, ctypes.byref(a), None
        s["keep"], s["got"] = a, {"q": s["q_out"], "k": s["k"], "v": s["v"]}
    elif kind == "attend":
        H, KV, hd = HEADS[case["heads"]]
        a = q.AttentionArgs(pages=pages(), n_heads=H, n_seq=case["groups"] * case["beams"], q_len=case["q"],
                            n_groups=case["groups"], q=s["q"].data_ptr(), q_stride=H * hd, out=s["out"].data_ptr(),
                            out_stride=H * hd, table=s["table"].data_ptr(), len=s["len"].data_ptr(),
                            table_stride=s["table"].shape[1], max_len=s["L"], prefix_table=s["ptable"].data_ptr(),
                            prefix_len=s["plen"].data_ptr(), prefix_stride=s["ptable"].shape[1], max_prefix=s["P"],
                            scale=1.0 / math.sqrt(hd))
        n = lib.qmh_paged_attention_ws(ctypes.byref(a))
        s["ws"] = torch.empty(max(n, 1), dtype=torch.uint8, device="cuda")
        s["call"] = lib.qmh_paged_attention, ctypes.byref(a), s["ws"].data_ptr(), n, None
        s["keep"], s["got"] = a, s["out"]
    elif kind == "select":
        a = q.BeamArgs(dtype=dt, n_groups=case["groups"], n_beams=case["beams"], vocab=case["vocab"], n_out=case["out"], eos=EOS,
                       logits=s["logits"].data_ptr(), stride=case["vocab"], score=s["score"].data_ptr(),
                       done=s["done"].data_ptr() if case["done"] else None, out_score=s["score_out"].data_ptr(),
                       out_parent=s["parent_out"].data_ptr(), out_token=s["token_out"].data_ptr())
        n = lib.qmh_beam_select_ws(ctypes.byref(a))
        s["ws"] = torch.empty(max(n, 1), dtype=torch.uint8, device="cuda")
        s["call"] = lib.qmh_beam_select, ctypes.byref(a), s["ws"].data_ptr(), n, None
        s["keep"], s["got"] = a, {"score": s["score_out"], "parent": s["parent_out"], "token": s["token_out"]}
    elif case["form"] == "dense":
        x = s["src"]
        a = q.BeamState(n_outer=x.shape[0], outer_stride=4 * x.stride(0), seq_stride=4 * x.stride(1), n_rows=x.shape[2],
                        row_stride=4 * x.stride(2), live=4 * case["live"])
        s["call"] = (lib.qmh_beam_reorder, ctypes.byref(a), s["dst"].data_ptr(), x.data_ptr(), s["parent"].data_ptr(),
                     case["groups"], case["beams"], None)
        s["keep"], s["got"] = a, s["dst"]
    else:
        s["call"] = (lib.qmh_paged_reorder, pages(), s["table"].data_ptr(), s["table"].shape[1], s["len"].data_ptr(),
                     case["len"], s["parent"].data_ptr(), case["groups"], case["beams"], None)
        s["got"] = {"k": s["k"], "v": s["v"]}


def run(s):
    if not own:
        return _PLAIN[s["case"]["kind"]](s)
    call = s["call"]
    if call[0](*call[1:]):
        import quillm_amd as q

        raise q.QmhError(q.last_error())
    return s["got"]


# ------------------------------------------------------------------------------------- work

def work(case):
    kind = case["kind"]
    if kind == "select":
        rows = case["groups"] * case["beams"]
        e = 4 if case["dtype"] == "f32" else 2
        # an exponential and a sum for each logit
        return {"bytes": rows * (case["vocab"] * e + 4) + 12 * case["groups"] * case["out"], "flops": 2 * rows * case["vocab"]}
    H, KV, hd = HEADS[case["heads"]]
    e = 2 if case.get("dtype", "f32") != "f32" else 4
    if kind == "append":
        n = case["tokens"]
        row = (H + 2 * KV) * hd
        return {"bytes": n * (2 * row * e + 12), "flops": n * (H + KV) * (3 * case["rot"] + (4 * hd if case["norm"] else 0))}
    if kind == "attend":
        # lengths are uniform between a half and the whole, the first group's and the last sequence's whole
        P, L, Q = case["prefix"], max(case["len"], case["q"]), case["q"]
        B = case["groups"] * case["beams"]
        pre = P + 0.75 * P * (case["groups"] - 1)
        mine = L + 0.75 * L * (B - 1)
        rows = B * Q * H * hd
        seen = case["beams"] * Q * H * pre + Q * H * max(mine - B * (Q - 1) / 2, B)
        return {"bytes": 2 * rows * e + 2 * KV * hd * e * (pre + mine), "flops": 4 * hd * seen}
    G, K = case["groups"], case["beams"]
    if not case["inplace"]:
        writes, stay = K, K
    else:
        writes, stay = case["moved"], K - case["moved"]
    reads = stay * (1 - (1 - 1 / stay) ** writes)  # distinct parents, as drawn
    if case["form"] == "dense":
        one = case["layers"] * KV * hd * case["live"] * 4
        per = G
    else:
        one = 2 * KV * hd * e
        per = case["len"] * (1 + 0.75 * (G - 1))
    return {"bytes": (reads + writes) * one * per + 4 * G * K, "flops": 0}


# ------------------------------------------------------------------------------------- 64-bit values

def _exact_append(case, seed):
    s = _append_inputs(case, seed)
    H, KV, hd = HEADS[case["heads"]]
    r = case["rot"]
    f = _freqs(case)
    turn = torch.polar(torch.full_like(f, _f32(_magnitude(case))).expand(case["tokens"], -1).contiguous(),
                       s["pos"].double()[:, None] * f[None])

    def one(x, gain):
        x = x.double().unflatten(-1, (-1, hd))
        if gain is not None:
            x = x / torch.sqrt(x.square().mean(-1, keepdim=True) + _f32(EPS)) * gain.double()
        head = x[..., :r]
        if case["layout"] == "halves":
            head = head.unflatten(-1, (2, r // 2)).transpose(-1, -2)
        else:
            head = head.unflatten(-1, (r // 2, 2))
        z = torch.view_as_real(torch.view_as_complex(head.contiguous()) * turn[:, None])
        z = (z.transpose(-1, -2) if case["layout"] == "halves" else z).flatten(-2)
        return torch.cat([z, x[..., r:]], -1)

    gq, gk = s["gain"] if s["gain"] is not None else (None, None)
    q, k, v = s["qkv"].split([H * hd, KV * hd, KV * hd], -1)
    kk, vv = s["k"].double(), s["v"].double()
    where = s["table"][s["seq"].long()].gather(1, (s["slot"] // case["page"]).long()[:, None])[:, 0].long()
    at = (s["slot"] % case["page"]).long()
    kk[where, :, at] = one(k, gk)
    vv[where, :, at] = v.double().unflatten(-1, (KV, hd))
    return {"q": one(q, gq).flatten(1), "k": kk, "v": vv}


def _exact_attend(case, seed):
    s = _attend_inputs(case, seed)
    H, KV, hd = HEADS[case["heads"]]
    Q, ps = case["q"], case["page"]
    q = s["q"].double().view(-1, Q, H, hd)
    plen, olen = s["plen"].tolist(), s["len"].tolist()

    def rows(pages, table, n):
        t = torch.arange(n, device="cuda")
        return pages[table[t // ps].long(), :, t % ps].double().transpose(0, 1)  # [kv head, position, head_dim]

    out = []
    for b in range(q.shape[0]):
        g = b // case["beams"]
        if b % case["beams"] == 0:
            pk, pv = rows(s["k"], s["ptable"][g], plen[g]), rows(s["v"], s["ptable"][g], plen[g])
        k, v = (torch.cat([p, rows(x, s["table"][b], olen[b])], 1) for p, x in ((pk, s["k"]), (pv, s["v"])))
        one = torch.empty(Q, H, hd, device="cuda", dtype=torch.float64)
        for j in range(Q):
            n = plen[g] + olen[b] - Q + 1 + j
            w = torch.bmm(q[b, j].view(KV, H // KV, hd), k[:, :n].transpose(1, 2).contiguous()) / math.sqrt(hd)
            one[j] = torch.bmm(torch.softmax(w, -1), v[:, :n].contiguous()).view(H, hd)
        out.append(one.flatten(1))
    return torch.cat(out)


def _exact_select(case, seed):
    s = _select_inputs(case, seed)
    G, K, V, n = case["groups"], case["beams"], case["vocab"], case["out"]
    x = s["logits"].double()
    done = s["done"].tolist() if s["done"] is not None else [0] * (G * K)
    sc = s["score"].double().tolist()
    lse = torch.logsumexp(x, -1).tolist()
    best = torch.topk(x, min(V, n), -1)[0][:, -1].tolist()
    score, parent, token = [], [], []
    for g in range(G):
        cand = []
        for b in range(K):
            i = g * K + b
            if done[i]:
                cand.append((-sc[i], b, 0, EOS))
                continue
            at = torch.nonzero(x[i] >= best[i])[:, 0].tolist()
            vals = x[i][at].tolist()
            cand += [(-(sc[i] + (val - lse[i])), b, t, t) for val, t in zip(vals, at) if val > -math.inf]
        cand = sorted(cand)[:n]
        cand += [(math.inf, -1, -1, -1)] * (n - len(cand))
        score.append([-c[0] for c in cand])
        parent.append([c[1] for c in cand])
        token.append([c[3] for c in cand])
    return {"score": torch.tensor(score, dtype=torch.float64), "parent": torch.tensor(parent, dtype=torch.int32),
            "token": torch.tensor(token, dtype=torch.int32)}


def _exact_reorder(case, seed):
    s = _reorder_inputs(case, seed)
    K, par = case["beams"], s["parent"].tolist()
    if case["form"] == "dense":
        out, n = s["dst"].double().clone(), case["live"]
        for b, p in enumerate(par):
            out[:, b, :, :n] = s["src"][:, b - b % K + p, :, :n].double()
        return out
    out = {}
    for name in "kv":
        x = s[name].double()
        y = x.clone()
        for b, p in enumerate(par):
            t = torch.arange(int(s["len"][b]), device="cuda")
            here, there = (s["table"][i][t // case["page"]].long() for i in (b, b - b % K + p))
            y[here, :, t % case["page"]] = x[there, :, t % case["page"]]
        out[name] = y
    return out


def exact(case, seed):
    return {"append": _exact_append, "attend": _exact_attend, "select": _exact_select, "reorder": _exact_reorder}[case["kind"]](
        case, seed)
