"""Verifying drafted trees over a paged cache: the operators' cases, their plain forms and their 64-bit values.

A server whose sequences are drafted ahead checks in one pass a tree of guessed tokens for each. Its step is

* plan     pages for the new tokens, taken from and given back to a list of free ones, and for each token its sequence,
           slot and position, for trees the ancestors too (`qmh_paged_plan`);
* attend   each node over its sequence's context (a shared prefix, its own pages) and its ancestors (`qmh_tree_attention`);
* logits   penalties for repeated tokens, biases and grammar masks, and each row's best token (`qmh_logits_edit`);
* accept   the longest path that the model agrees with: its keys and values moved to follow the context, in all
           layers (`qmh_tree_accept`).

Head shapes are those of the workloads c1 to c5 (`quillm_amd.WORKLOADS`), and some odd ones; the vocabularies those of the
framework's tests. Where `own` is false the passes are elementary torch operations in 32 bits; where it is true they are the
calls that a user of the library makes.
"""
import ctypes
import math

import torch

own = False

# query heads, kv heads, head_dim: c1, c2, c3, c4, c5, and two with remainders
HEADS = {"c1": (6, 6, 48), "c2": (6, 2, 48), "c3": (12, 12, 64), "c4": (32, 4, 64), "c5": (32, 32, 128),
         "o1": (5, 1, 80), "o2": (14, 2, 96)}
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
PAD = 3  # rows that a batch has behind its last sequence's


def listed():
    return [
        # 48 drafted sequences of a server: a step's trees get pages, positions and masks; then what was not accepted goes back
        {"name": "plan step", "kind": "plan", "seqs": 48, "page": 16, "tree": 24, "add": 24, "len": 900, "tight": True},
        # a batch of long prompts comes and goes
        {"name": "plan prompts", "kind": "plan", "seqs": 201, "page": 32, "tree": 0, "add": 1200, "len": 0, "tight": False},
        # one conversation of a small model, five drafted tokens: nothing but latency
        {"name": "attend small", "kind": "attend", "heads": "c2", "dtype": "f32", "groups": 1, "beams": 1, "nodes": 5, "ragged": False,
         "static": True, "page": 16, "prefix": 0, "len": 43},
        # three prompts of four sequences each, full precision, ragged trees
        {"name": "attend prefix", "kind": "attend", "heads": "c3", "dtype": "f32", "groups": 3, "beams": 4, "nodes": 17, "ragged": True,
         "static": False, "page": 16, "prefix": 515, "len": 190},
        # a server of 7B-shaped sequences, each with its own tree
        {"name": "attend server", "kind": "attend", "heads": "c5", "dtype": "bf16", "groups": 8, "beams": 1, "nodes": 32, "ragged": True,
         "static": False, "page": 64, "prefix": 0, "len": 4100},
        # a grouped-query model with large trees of one shape
        {"name": "attend grouped", "kind": "attend", "heads": "c4", "dtype": "f16", "groups": 12, "beams": 1, "nodes": 64, "ragged": False,
         "static": True, "page": 32, "prefix": 0, "len": 6000},
        # one long conversation
        {"name": "attend long", "kind": "attend", "heads": "c4", "dtype": "bf16", "groups": 1, "beams": 1, "nodes": 48, "ragged": False,
         "static": False, "page": 128, "prefix": 0, "len": 30011},
        # one conversation's next token before it is sampled: a row edited in place
        {"name": "logits one", "kind": "logits", "dtype": "f32", "seqs": 1, "nodes": 1, "vocab": 32000, "history": 700, "biases": 12,
         "grammar": False, "out": "inplace", "best": False},
        # trees checked under grammars by a greedy server: only the best tokens are wanted
        {"name": "logits trees", "kind": "logits", "dtype": "bf16", "seqs": 16, "nodes": 24, "vocab": 32003, "history": 1500, "biases": 5,
         "grammar": True, "out": "none", "best": True},
        # the largest: everything at once over a large vocabulary, edited logits kept for a sampler
        {"name": "logits wide", "kind": "logits", "dtype": "f32", "seqs": 40, "nodes": 4, "vocab": 128256, "history": 4000, "biases": 300,
         "grammar": True, "out": "other", "best": True},
        # four sequences of a small model, all its layers
        {"name": "accept small", "kind": "accept", "heads": "c2", "dtype": "f32", "layers": 6, "seqs": 4, "nodes": 16, "page": 16, "len": 300},
        # 64 sequences with large trees, 7B-shaped heads, four layers in one call
        {"name": "accept server", "kind": "accept", "heads": "c5", "dtype": "f16", "layers": 4, "seqs": 64, "nodes": 61, "page": 32, "len": 2000},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["plan", "attend", "attend", "attend", "logits", "logits", "accept"])
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
    heads, dtype, page = rng.choice(sorted(HEADS)), rng.choice(sorted(TYPES)), rng.choice([16, 32, 64, 128])
    if kind == "plan":
        tree = rng.choice([0, _log(rng, 1, 120)])
        return {"kind": kind, "seqs": _log(rng, 1, 2000), "page": page, "tree": tree, "add": tree or _log(rng, 1, 3000),
                "len": rng.choice([0, _log(rng, 1, 6000)]), "tight": rng.choice([False, True])}
    if kind == "attend":
        nodes = _log(rng, 1, 130)
        return {"kind": kind, "heads": heads, "dtype": dtype, "groups": rng.randint(1, 8), "beams": rng.choice([1, 1, _log(rng, 1, 12)]),
                "nodes": nodes, "ragged": rng.choice([False, True]), "static": rng.choice([False, True]), "page": page,
                "prefix": rng.choice([0, 0, _log(rng, 1, 6000)]), "len": nodes + _log(rng, 1, 30000)}
    if kind == "logits":
        out = rng.choice(["inplace", "none", "other"])
        return {"kind": kind, "dtype": dtype, "seqs": _log(rng, 1, 64), "nodes": rng.choice([1, _log(rng, 1, 40)]),
                "vocab": _log(rng, 300, 128256), "history": _log(rng, 1, 4000), "biases": rng.choice([0, _log(rng, 1, 300)]),
                "grammar": rng.choice([False, True]), "out": out, "best": out == "none" or rng.choice([False, True])}
    return {"kind": kind, "heads": heads, "dtype": dtype, "layers": rng.randint(1, 8), "seqs": _log(rng, 1, 64), "nodes": _log(rng, 1, 130),
            "page": page, "len": 200 + _log(rng, 1, 3000)}


# ------------------------------------------------------------------------------------- inputs

def _gen(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed) * 1000003 + sum(ord(c) * (i + 1) for i, c in enumerate(repr(sorted(case.items(), key=str)))))
    return g


def _rand(g, *size):
    return torch.rand(*size, device="cuda", generator=g)


def _randn(g, dtype, *size):
    return torch.randn(*size, device="cuda", generator=g, dtype=dtype)


def _randint(g, lo, hi, *size):
    """Whole numbers in [lo, hi]."""
    return torch.randint(lo, hi + 1, size, device="cuda", generator=g, dtype=torch.int32)


def _spread(g, lo, hi, n):
    """n whole numbers spread evenly over [lo, hi], in an order of the seed's: their sum is the case's."""
    x = lo + (torch.arange(n, device="cuda") * (hi - lo) + (n - 1) // 2) // max(n - 1, 1) if n > 1 else torch.full((1,), hi, device="cuda")
    return x[torch.randperm(n, device="cuda", generator=g)].to(torch.int32)


def _trees(g, seqs, nodes):
    """Parents [seqs, nodes]: node 0 is the root, half of the others follow the one before, half any earlier one."""
    j = torch.arange(nodes, device="cuda")
    some = (_rand(g, seqs, nodes) * j).long()
    p = torch.where(_rand(g, seqs, nodes) < 0.5, j - 1, some)
    p[:, 0] = -1
    return p.to(torch.int32).contiguous()


def _ancestors(parent):
    """Truth values [seqs, nodes, nodes]: row j has its ancestors and itself."""
    S, N = parent.shape
    see = torch.eye(N, dtype=torch.bool, device=parent.device).repeat(S, 1, 1)
    p, left = parent.long(), N
    while left > 1:  # each round doubles the steps upward
        up = torch.gather(see, 1, p.clamp(min=0)[..., None].expand(S, N, N))
        see = see | (up & (p >= 0)[..., None])
        p = torch.where(p >= 0, torch.gather(p, 1, p.clamp(min=0)), -1)
        left = (left + 1) // 2
    return see


def _pack(see):
    """Truth values to words of 32 bits, bit k of word w for column 32 w + k."""
    n = see.shape[-1]
    see = torch.nn.functional.pad(see, (0, -n % 32)).unflatten(-1, (-1, 32))
    w = (see.long() << torch.arange(32, device=see.device)).sum(-1)
    return torch.where(w >= 1 << 31, w - (1 << 32), w).to(torch.int32).contiguous()


def _unpack(words, n):
    return ((words[..., None] >> torch.arange(32, device=words.device)) & 1).bool().flatten(-2)[..., :n]


def _tables(g, counts, width, n_pages):
    """Tables [len(counts), width] of distinct pages in random order, -1 behind; and the pages that are left."""
    perm = torch.randperm(n_pages, device="cuda", generator=g).to(torch.int32)
    c = torch.tensor(counts, device="cuda")
    at = torch.cumsum(c, 0) - c
    j = torch.arange(max(1, width), device="cuda")
    t = torch.where(j < c[:, None], perm[(at[:, None] + j).clamp(max=n_pages - 1)], -1)
    return t.contiguous(), perm[sum(counts):]


def _plan_inputs(case, seed):
    g = _gen(case, seed)
    S, ps, A, L = case["seqs"], case["page"], case["add"], case["len"]
    start = _randint(g, (L + 1) // 2, L, S)
    add = _spread(g, (A + 1) // 2, A, S)
    keep = start + (_rand(g, S) * (add // 3 + 1)).to(torch.int32) if L else torch.zeros_like(start)  # what stays after the step
    have = [-(-x // ps) for x in start.tolist()]
    need = [-(-(x + y) // ps) for x, y in zip(start.tolist(), add.tolist())]
    stride = -(-(L + A) // ps) + 1
    grow = sum(need) - sum(have)
    spare = max(1, grow - 2 if case["tight"] else grow + grow // 8)  # too few: the last sequences that need one go without
    size = S * stride  # of the ring, which has been round some times
    table, free = _tables(g, have, stride, sum(have) + spare)
    turn = int(_randint(g, 0, size - 1, 1))
    ring = torch.full((size,), -1, dtype=torch.int32, device="cuda")
    ring[(turn + torch.arange(spare, device="cuda")) % size] = free
    tokens = sum(add.tolist()) + PAD
    s = {"start": start, "add": add, "keep": keep, "len": start.clone(), "table": table, "ring": ring, "base": _randint(g, 0, 4000, S),
         "ring_state": torch.tensor([turn, spare], dtype=torch.int32, device="cuda"), "tokens": tokens}
    s["parent"] = _trees(g, S, case["tree"]) if case["tree"] else None
    return s


def _attend_inputs(case, seed):
    H, KV, hd = HEADS[case["heads"]]
    dt, ps, g = TYPES[case["dtype"]], case["page"], _gen(case, seed)
    G, B, N, P, L = case["groups"], case["groups"] * case["beams"], case["nodes"], case["prefix"], case["len"]
    nodes = _spread(g, N // 2, N, B) if case["ragged"] else torch.full((B,), N, dtype=torch.int32, device="cuda")
    olen = torch.maximum(_randint(g, (L + 1) // 2, L, B), nodes)
    olen[-1] = L
    plen = _randint(g, (P + 1) // 2, P, G)
    plen[0] = P
    pc, oc = [-(-x // ps) for x in plen.tolist()], [-(-x // ps) for x in olen.tolist()]
    n_pages = G * -(-P // ps) + B * -(-L // ps)
    tables, _ = _tables(g, pc + oc, max(pc + oc), n_pages)
    first = torch.nn.functional.pad(torch.cumsum(nodes, 0), (1, 0)).to(torch.int32)
    rows = int(first[-1]) + (PAD if case["ragged"] else 0)
    k, v = _randn(g, dt, n_pages, KV, ps, hd), _randn(g, dt, n_pages, KV, ps, hd)
    parent = _trees(g, 1 if case["static"] else B, N)
    return {"q": _randn(g, dt, rows, H * hd) * 1.5, "k": k, "v": v, "ptable": tables[:G].contiguous(), "table": tables[G:].contiguous(),
            "plen": plen, "len": olen, "first": first if case["ragged"] else None, "nodes": nodes, "rows": rows, "parent": parent,
            "mask": _pack(_ancestors(parent))}


def _logits_inputs(case, seed):
    g = _gen(case, seed)
    S, N, V, h = case["seqs"], case["nodes"], case["vocab"], case["history"]
    rows = S * N

    def tokens(*size):  # some tokens are far more common than others
        return (_rand(g, *size) ** 3 * V).to(torch.int32).clamp(max=V - 1)

    hlen = _randint(g, (h + 1) // 2, h, S)
    hlen[-1] = h
    s = {"logits": (_randn(g, torch.float32, rows, V) * 2.5).to(TYPES[case["dtype"]]), "history": tokens(S, h), "hlen": hlen,
         "plen": (_rand(g, S) * hlen).to(torch.int32), "rep": 1 + 0.5 * _rand(g, S), "pres": 0.5 * _rand(g, S), "freq": 0.3 * _rand(g, S)}
    s["rep"][0] = 1.0
    if case["biases"]:
        n = min(case["biases"], V)
        s["btoken"] = torch.stack([torch.randperm(V, device="cuda", generator=g)[:n] for _ in range(S)]).to(torch.int32)
        s["bias"] = _randn(g, torch.float32, S, n) * 3
        s["blen"] = _randint(g, 0, n, S)
    if case["grammar"]:
        # states of a grammar: some allow a word or two, some nearly everything; a quarter of the rows has none
        m = max(2, rows // 3)
        share = _rand(g, m, 1) ** 4
        ok = _rand(g, m, V) < share
        ok[:, 7] = True
        s["allow"] = _pack(ok)
        s["allow_row"] = torch.where(_rand(g, rows) < 0.25, -1, _randint(g, 0, m - 1, rows)).to(torch.int32)
    if N > 1:
        s["token"] = tokens(S, N)
        s["see"] = _ancestors(_trees(g, S, N))
        s["mask"] = _pack(s["see"])
    return s


def _accept_inputs(case, seed):
    H, KV, hd = HEADS[case["heads"]]
    dt, ps, g = TYPES[case["dtype"]], case["page"], _gen(case, seed)
    S, N, V = case["seqs"], case["nodes"], 32000
    parent, token = _trees(g, S, N), _randint(g, 0, V - 1, S, N)
    # the model agrees with a drafted child of most nodes
    choice = _randint(g, 0, V - 1, S, N)
    child = torch.randint(0, N, (S, N), device="cuda", generator=g)
    for c in (torch.arange(N, device="cuda").expand(S, N), child):
        p = torch.gather(parent, 1, c).long()
        use = (_rand(g, S, N) < 0.9) & (p >= 0)
        to = torch.where(use, p, N)
        wide = torch.cat([choice, choice[:, :1]], 1)
        # of several children the one with the largest number, whatever order they are written in
        last = torch.full((S, N + 1), -1, device="cuda").scatter_reduce(1, to, c.contiguous(), "amax")
        took = torch.gather(token, 1, last.clamp(min=0))
        choice = torch.where(last >= 0, took, wide)[:, :N].contiguous()
    length = _randint(g, max(N, case["len"] // 2), max(N, case["len"]), S)
    # pages of the tree only: what lies before is not looked at
    stride = -(-max(N, case["len"]) // ps)
    lo, hi = (length - N) // ps, (length + ps - 1) // ps
    counts = (hi - lo).tolist()
    n_pages = S * ((N + ps - 2) // ps + 1)
    dense, _ = _tables(g, counts, max(counts), n_pages)
    j = torch.arange(stride, device="cuda") - lo[:, None]
    inside = (j >= 0) & (j < (hi - lo)[:, None])
    table = torch.where(inside, torch.gather(dense, 1, j.clamp(0, dense.shape[1] - 1).long()), -1).to(torch.int32).contiguous()
    size = (case["layers"], n_pages, KV, ps, hd)
    room = 64 + case["nodes"]
    return {"parent": parent, "token": token, "choice": choice.flatten(), "len": length, "table": table, "k": _randn(g, dt, *size),
            "v": _randn(g, dt, *size), "history": _randint(g, 0, V - 1, S, room), "hlen": _randint(g, 0, 63, S)}


_INPUTS = {"plan": _plan_inputs, "attend": _attend_inputs, "logits": _logits_inputs, "accept": _accept_inputs}


def prepare(case, seed):
    s = _INPUTS[case["kind"]](case, seed)
    s["case"], kind = case, case["kind"]

    def ints(*size):
        return torch.full(size, -1, dtype=torch.int32, device="cuda")

    if kind == "plan":
        n = case["seqs"]
        s["got"] = {"table": s["table"], "len": s["len"], "ring": s["ring"], "state": s["ring_state"], "first": ints(n + 1), "seq": ints(s["tokens"]),
                    "slot": ints(s["tokens"]), "pos": ints(s["tokens"]), "refused": ints(n), "late": ints(n)}
        if case["tree"]:
            s["got"]["mask"] = torch.zeros(n, case["tree"], -(-case["tree"] // 32), dtype=torch.int32, device="cuda")
    elif kind == "attend":
        s["got"] = torch.zeros_like(s["q"])
    elif kind == "logits":
        s["got"] = {}
        if case["out"] != "none":
            s["got"]["out"] = s["logits"] if case["out"] == "inplace" else torch.zeros_like(s["logits"])
        if case["best"]:
            s["got"]["best"] = ints(s["logits"].shape[0])
    else:
        S, N = s["parent"].shape
        s["got"] = {"count": ints(S), "path": ints(S, N), "next": ints(S), "keep": ints(S), "history": s["history"], "hlen": s["hlen"], "k": s["k"],
                    "v": s["v"]}
    if own:
        _prepare_own(case, s)
    torch.cuda.synchronize()  # the library has a stream of its own
    return s


# ------------------------------------------------------------------------------------- the plain forms

def _plain_plan_call(s, keep, add, refused, trees):
    """One plan: tables, lengths and the ring after it; the tokens where there are some."""
    case, got = s["case"], s["got"]
    ps, cap, R = case["page"], s["table"].shape[1] * case["page"], s["ring"].shape[0]
    length, state = s["len"].long(), s["ring_state"].long()
    keep = keep.long()
    no_tokens = add is None
    add = torch.zeros_like(keep) if no_tokens else add.long()
    new = keep + add
    fine = (length >= 0) & (length <= cap) & (keep >= 0) & (keep <= length) & (add >= 0) & (new <= cap)
    if trees:
        fine &= add <= case["tree"]
    have, need = (length + ps - 1) // ps, (new + ps - 1) // ps
    take = torch.where(fine, (need - have).clamp(min=0), 0)
    give = torch.where(fine, (have - need).clamp(min=0), 0)
    paged = fine & ((take == 0) | (torch.cumsum(take, 0) <= state[1])) & ((give == 0) | (torch.cumsum(give, 0) <= R - state[1]))
    more = torch.where(paged, add, 0)
    served = paged & ((more == 0) | (torch.cumsum(more, 0) <= s["tokens"]))
    take, give, more = (torch.where(served, x, 0) for x in (take, give, more))
    j = torch.arange(s["table"].shape[1], device="cuda")
    gains = (j >= have[:, None]) & (j < (have + take)[:, None])
    from_ring = (state[0] + (torch.cumsum(take, 0) - take)[:, None] + j - have[:, None]) % R
    gone = served[:, None] & (j >= need[:, None]) & (j < have[:, None])
    to_ring = (state[0] + state[1] + (torch.cumsum(give, 0) - give)[:, None] + j - need[:, None]) % R
    ring = torch.cat([s["ring"], s["ring"][:1]])
    wide = torch.where(gone, to_ring, R)
    ring = ring.scatter(0, wide.flatten(), s["table"].flatten())
    s["table"].copy_(torch.where(gains, s["ring"][from_ring], torch.where(gone, -1, s["table"])))
    s["ring"].copy_(ring[:R])
    s["ring_state"].copy_(torch.stack([(state[0] + take.sum()) % R, state[1] - take.sum() + give.sum()]))
    s["len"].copy_(torch.where(served, new, length))
    refused.copy_(torch.where(served, 0, torch.where(paged, 2, torch.where(fine, 1, 3))))
    if no_tokens:
        return
    first = torch.nn.functional.pad(torch.cumsum(more, 0), (1, 0))
    t = torch.arange(s["tokens"], device="cuda")
    live = t < first[-1]
    i = torch.searchsorted(first[1:].contiguous(), t, right=True).clamp(max=len(keep) - 1)
    j = t - first[i]
    slot, depth = keep[i] + j, j
    if trees:
        see = _ancestors(s["parent"])
        depth = see.sum(-1)[i, j.clamp(0, case["tree"] - 1)] - 1
        row = torch.arange(case["tree"], device="cuda") < more[:, None]
        got["mask"].copy_(torch.where(row[..., None], _pack(see), got["mask"]))
    got["first"].copy_(first)
    got["seq"].copy_(torch.where(live, i, -1))
    got["slot"].copy_(torch.where(live, slot, -1))
    got["pos"].copy_(torch.where(live, s["base"].long()[i] + keep[i] + depth, -1))


def _plain_plan(s):
    _plain_plan_call(s, s["start"], s["add"], s["got"]["refused"], bool(s["case"]["tree"]))
    _plain_plan_call(s, s["keep"], None, s["got"]["late"], False)
    return s["got"]


def _gather_pages(pages, table, n):
    """[rows, kv heads, n, head_dim] in 32 bits of the tables' first n positions."""
    x = pages[table[:, :(n + pages.shape[2] - 1) // pages.shape[2]].clamp(min=0).long()]
    return x.permute(0, 2, 1, 3, 4).flatten(2, 3)[:, :, :n].float()


def _plain_attend(s):
    case = s["case"]
    H, KV, hd = HEADS[case["heads"]]
    G, K, N, P, L = case["groups"], case["beams"], case["nodes"], case["prefix"], case["len"]
    B, M, scale = G * K, H // KV, 1.0 / math.sqrt(hd)
    j = torch.arange(N, device="cuda")
    n = s["nodes"].long()
    first = torch.cumsum(n, 0) - n
    live = j < n[:, None]
    row = torch.where(live, first[:, None] + j, s["rows"])  # one row more takes what is nobody's
    q = torch.cat([s["q"], s["q"][:1]])[row].float().view(B, N, KV, M, hd).permute(0, 2, 1, 3, 4).contiguous()  # [B, KV, N, M, hd]
    see = _unpack(s["mask"], N).expand(B, N, N)
    ko, vo = _gather_pages(s["k"], s["table"], L), _gather_pages(s["v"], s["table"], L)
    so = torch.bmm(q.view(B * KV, N * M, hd), ko.flatten(0, 1).transpose(1, 2).contiguous()).view(B, KV, N, M, L) * scale
    t = torch.arange(L, device="cuda") - (s["len"].long() - n)[:, None]  # positions by node number, the context below 0
    seen = torch.gather(see, 2, t.clamp(0, N - 1)[:, None].expand(B, N, L)) & (t < n[:, None])[:, None]
    seen = seen | (t < 0)[:, None]
    so.masked_fill_(~seen[:, None, :, None], -math.inf)
    m = so.amax(-1, keepdim=True)
    if P:
        kp, vp = _gather_pages(s["k"], s["ptable"], P), _gather_pages(s["v"], s["ptable"], P)
        qg = q.view(G, K, KV, N * M, hd).transpose(1, 2).reshape(G * KV, K * N * M, hd)
        sp = torch.bmm(qg, kp.flatten(0, 1).transpose(1, 2).contiguous()).view(G, KV, K * N * M, P) * scale
        sp.masked_fill_((torch.arange(P, device="cuda") >= s["plen"][:, None])[:, None, None], -math.inf)
        mp = sp.amax(-1, keepdim=True).view(G, KV, K, N, M, 1).transpose(1, 2).reshape(B, KV, N, M, 1)
        m = torch.maximum(m, mp)
    m = torch.where(m == -math.inf, torch.zeros_like(m), m)
    eo = torch.exp(so - m)
    total = eo.sum(-1, keepdim=True)
    acc = torch.bmm(eo.view(B * KV, N * M, L), vo.flatten(0, 1).contiguous()).view(B, KV, N, M, hd)
    if P:
        ep = torch.exp(sp - m.view(G, K, KV, N * M, 1).transpose(1, 2).reshape(G, KV, K * N * M, 1))
        total = total + ep.sum(-1, keepdim=True).view(G, KV, K, N, M, 1).transpose(1, 2).reshape(B, KV, N, M, 1)
        a = torch.bmm(ep.view(G * KV, K * N * M, P), vp.flatten(0, 1).contiguous())
        acc = acc + a.view(G, KV, K, N, M, hd).transpose(1, 2).reshape(B, KV, N, M, hd)
    y = (acc / total).permute(0, 2, 1, 3, 4).reshape(B * N, H * hd).to(s["got"].dtype)
    s["got"].copy_(torch.cat([s["got"], y[:1]]).index_copy(0, row.flatten(), y)[:-1])
    return s["got"]


def _plain_logits(s):
    case, got = s["case"], s["got"]
    S, N, V = case["seqs"], case["nodes"], case["vocab"]
    x = s["logits"].float()
    at = torch.arange(case["history"], device="cuda")
    live = at < s["hlen"][:, None]
    output = live & (at >= s["plen"][:, None])
    tok = s["history"].long()
    count = torch.zeros(S, V, device="cuda").scatter_add_(1, tok, output.float()).repeat_interleave(N, 0)
    prompt = torch.zeros(S, V, device="cuda").scatter_add_(1, tok, (live & ~output).float()).repeat_interleave(N, 0)
    if N > 1:
        path = s["token"].long()[:, None].expand(S, N, N).reshape(S * N, N)
        count.scatter_add_(1, path, s["see"].reshape(S * N, N).float())
    r, p, f = (s[k].repeat_interleave(N)[:, None] for k in ("rep", "pres", "freq"))
    x = torch.where((count > 0) | (prompt > 0), torch.where(x > 0, x / r, x * r), x)
    x = x - (f * count + p * (count > 0))
    if case["biases"]:
        on = torch.arange(s["bias"].shape[1], device="cuda") < s["blen"][:, None]
        b = torch.zeros(S, V, device="cuda").scatter_add_(1, s["btoken"].long(), torch.where(on, s["bias"], 0.0))
        x = x + b.repeat_interleave(N, 0)
    if case["grammar"]:
        ok = _unpack(s["allow"], V)[s["allow_row"].clamp(min=0).long()] | (s["allow_row"] < 0)[:, None]
        x = torch.where(ok, x, -math.inf)
    if case["best"]:
        got["best"].copy_(torch.where(x == x.amax(-1, keepdim=True), torch.arange(V, device="cuda"), V).amin(-1))
    if case["out"] != "none":
        got["out"].copy_(x)
    return got


def _plain_accept(s):
    case, got = s["case"], s["got"]
    S, N = s["parent"].shape
    p, tok, choice = s["parent"].long(), s["token"], s["choice"].view(S, N)
    node = torch.arange(N, device="cuda").expand(S, N)
    fits = (p >= 0) & (tok == torch.gather(choice, 1, p.clamp(min=0)))
    follow = torch.full((S, N + 1), N, device="cuda").scatter_reduce(1, torch.where(fits, p, N), node, "amin")
    follow[:, N] = N
    cur, path = torch.zeros(S, 1, dtype=torch.long, device="cuda"), []
    for _ in range(N):
        path.append(cur)
        cur = torch.gather(follow, 1, cur)
    path = torch.cat(path, 1)
    on = path < N
    count = on.sum(1)
    begin = s["len"].long() - N
    last = torch.gather(path, 1, (count - 1)[:, None])
    got["count"].copy_(count)
    got["path"].copy_(torch.where(on, path, -1))
    got["next"].copy_(torch.gather(choice, 1, last)[:, 0])
    got["keep"].copy_(begin + count)
    room = s["history"].shape[1]
    to = s["hlen"].long()[:, None] + node
    wide = torch.cat([s["history"], s["history"][:, :1]], 1)
    wide = wide.scatter(1, torch.where(on & (to < room), to, room), torch.gather(tok, 1, path.clamp(max=N - 1)))
    s["history"].copy_(wide[:, :room])
    s["hlen"].copy_((s["hlen"] + count).clamp(max=room))
    src, dst, ps = begin[:, None] + path.clamp(max=N - 1), begin[:, None] + node, case["page"]
    moves = on & (path != node)
    i = node.new_zeros(S, N) + torch.arange(S, device="cuda")[:, None]
    src, dst, i = src[moves], dst[moves], i[moves]
    here, there = s["table"][i, dst // ps].long(), s["table"][i, src // ps].long()
    for x in (s["k"], s["v"]):
        x[:, here, :, dst % ps] = x[:, there, :, src % ps]
    return got


_PLAIN = {"plan": _plain_plan, "attend": _plain_attend, "logits": _plain_logits, "accept": _plain_accept}


# ------------------------------------------------------------------------------------- the library's calls

def _ptr(x):
    return x.data_ptr() if x is not None else None


def _prepare_own(case, s):
    import quillm_amd as q

    q.init(0)
    lib, kind, got = q.load_library(), case["kind"], s["got"]
    dt = {"f32": q.F32, "f16": q.F16, "bf16": q.BF16}[case.get("dtype", "f32")]

    def pages(k, v):
        s["pages"] = q.Pages(dtype=dt, n_kv_heads=k.shape[1], head_dim=k.shape[3], page_size=k.shape[2], n_pages=k.shape[0], k=k.data_ptr(),
                             v=v.data_ptr())
        return ctypes.pointer(s["pages"])

    def call(fn, a, need):
        ws = torch.empty(max(need, 1), dtype=torch.uint8, device="cuda")
        s.setdefault("keep_alive", []).append((a, ws))
        s.setdefault("calls", []).append((fn, ctypes.byref(a), ws.data_ptr(), need, None))

    if kind == "plan":
        d = dict(n_seq=case["seqs"], page_size=case["page"], table=_ptr(s["table"]), table_stride=s["table"].shape[1], len=_ptr(s["len"]),
                 free_pages=_ptr(s["ring"]), free_size=s["ring"].shape[0], free_state=_ptr(s["ring_state"]))
        a = q.PlanArgs(keep=_ptr(s["start"]), add=_ptr(s["add"]), base=_ptr(s["base"]), n_tokens=s["tokens"], first=_ptr(got["first"]),
                       seq=_ptr(got["seq"]), slot=_ptr(got["slot"]), pos=_ptr(got["pos"]), refused=_ptr(got["refused"]), parent=_ptr(s["parent"]),
                       parent_stride=case["tree"], tree_size=case["tree"], mask=_ptr(got.get("mask")), **d)
        call(lib.qmh_paged_plan, a, lib.qmh_paged_plan_ws(ctypes.byref(a)))
        a = q.PlanArgs(keep=_ptr(s["keep"]), refused=_ptr(got["late"]), **d)
        call(lib.qmh_paged_plan, a, lib.qmh_paged_plan_ws(ctypes.byref(a)))
    elif kind == "attend":
        H, KV, hd = HEADS[case["heads"]]
        words = s["mask"].shape[2]
        base = q.AttentionArgs(pages=pages(s["k"], s["v"]), n_heads=H, n_seq=case["groups"] * case["beams"], q_len=case["nodes"],
                               n_groups=case["groups"], q=_ptr(s["q"]), q_stride=H * hd, out=_ptr(got), out_stride=H * hd, table=_ptr(s["table"]),
                               len=_ptr(s["len"]), table_stride=s["table"].shape[1], max_len=case["len"], prefix_table=_ptr(s["ptable"]),
                               prefix_len=_ptr(s["plen"]), prefix_stride=s["ptable"].shape[1], max_prefix=case["prefix"],
                               scale=1.0 / math.sqrt(hd))
        a = q.TreeArgs(base=base, n_rows=s["rows"], first=_ptr(s["first"]), mask=_ptr(s["mask"]), mask_words=words,
                       mask_stride=0 if case["static"] else case["nodes"] * words)
        call(lib.qmh_tree_attention, a, lib.qmh_tree_attention_ws(ctypes.byref(a)))
    elif kind == "logits":
        N, V = case["nodes"], case["vocab"]
        a = q.LogitsArgs(dtype=dt, n_rows=s["logits"].shape[0], vocab=V, logits=_ptr(s["logits"]), stride=V, out=_ptr(got.get("out")), out_stride=V,
                         best=_ptr(got.get("best")), n_seq=case["seqs"], rows_per_seq=N, history=_ptr(s["history"]),
                         history_stride=case["history"], history_len=_ptr(s["hlen"]), prompt_len=_ptr(s["plen"]), repetition=_ptr(s["rep"]),
                         presence=_ptr(s["pres"]), frequency=_ptr(s["freq"]))
        if case["biases"]:
            a.bias_token, a.bias, a.bias_len, a.bias_stride = _ptr(s["btoken"]), _ptr(s["bias"]), _ptr(s["blen"]), s["bias"].shape[1]
        if case["grammar"]:
            a.allow, a.allow_stride, a.n_allow, a.allow_row = _ptr(s["allow"]), s["allow"].shape[1], s["allow"].shape[0], _ptr(s["allow_row"])
        if N > 1:
            a.node_token, a.node_stride, a.mask, a.mask_words = _ptr(s["token"]), N, _ptr(s["mask"]), s["mask"].shape[2]
            a.mask_stride = N * s["mask"].shape[2]
        call(lib.qmh_logits_edit, a, lib.qmh_logits_edit_ws(ctypes.byref(a)))
    else:
        S, N = s["parent"].shape
        k, v = s["k"], s["v"]
        a = q.AcceptArgs(n_seq=S, tree_size=N, parent=_ptr(s["parent"]), parent_stride=N, token=_ptr(s["token"]), token_stride=N, n_rows=S * N,
                         choice=_ptr(s["choice"]), len=_ptr(s["len"]), count=_ptr(got["count"]), path=_ptr(got["path"]), next=_ptr(got["next"]),
                         keep=_ptr(got["keep"]), history=_ptr(s["history"]), history_stride=s["history"].shape[1],
                         history_len=_ptr(s["hlen"]), pages=pages(k[0], v[0]), n_layers=case["layers"], layer_stride=k.stride(0),
                         table=_ptr(s["table"]), table_stride=s["table"].shape[1])
        s["keep_alive"] = a
        s["calls"] = [(lib.qmh_tree_accept, ctypes.byref(a), None)]


def run(s):
    if not own:
        return _PLAIN[s["case"]["kind"]](s)
    for fn, *args in s["calls"]:
        if fn(*args):
            import quillm_amd as q

            raise q.QmhError(q.last_error())
    return s["got"]


# ------------------------------------------------------------------------------------- work

def work(case):
    kind = case["kind"]
    if kind == "plan":  # additions and lengths are uniform between a half and the whole
        S, ps = case["seqs"], case["page"]
        tokens = 0.75 * S * case["add"]
        words = -(-case["tree"] // 32)
        # the tokens' three numbers, masks and parents; pages there and back; numbers of a sequence
        return {"bytes": int(tokens * (12 + (4 * words + 4 if case["tree"] else 0)) + 2 * 8 * tokens / ps + 40 * S), "flops": 0}
    e = 4 if case.get("dtype", "f32") == "f32" else 2
    if kind == "logits":
        S, N, V = case["seqs"], case["nodes"], case["vocab"]
        rows, masks = S * N, max(2, S * N // 3)
        hist = 0.75 * case["history"] * S
        sparse = 4 * hist + 8 * 0.5 * case["biases"] * S
        grammar = masks * V / 8 if case["grammar"] else 0
        if case["out"] == "inplace" and not case["best"]:
            # only what changes: the tokens that were seen, and under a grammar most of the rows
            touch = min(V, hist / S + 0.5 * case["biases"] + N / 2) * rows * 2 * e
            return {"bytes": int(sparse + grammar + touch + (0.6 * rows * V * e if case["grammar"] else 0)), "flops": int(touch)}
        return {"bytes": int(rows * V * e * (2 if case["out"] != "none" else 1) + sparse + grammar), "flops": 2 * rows * V}
    H, KV, hd = HEADS[case["heads"]]
    if kind == "attend":
        # lengths are uniform between a half and the whole, the first group's and the last sequence's whole
        P, L, N, B = case["prefix"], case["len"], case["nodes"], case["groups"] * case["beams"]
        n = 0.75 * N if case["ragged"] else N
        pre = P + 0.75 * P * (case["groups"] - 1)
        mine = L + 0.75 * L * (B - 1)
        rows = B * n * H * hd
        seen = case["beams"] * n * H * pre + n * H * max(mine - B * n / 2, B)
        return {"bytes": int(2 * rows * e + 2 * KV * hd * e * (pre + mine)), "flops": int(4 * hd * seen)}
    S, N = case["seqs"], case["nodes"]
    moved = S * 0.4 * min(N - 1, 8)  # about: a path goes on with three of four, half of the steps skip a number
    return {"bytes": int(S * N * 16 + 2 * moved * 2 * case["layers"] * KV * hd * e), "flops": 0}


# ------------------------------------------------------------------------------------- 64-bit values

def _exact_plan(case, seed):
    s = _plan_inputs(case, seed)
    ps, S, T = case["page"], case["seqs"], case["tree"]
    table, ring, length, base = (s[k].tolist() for k in ("table", "ring", "len", "base"))
    at, count = s["ring_state"].tolist()
    parent = s["parent"].tolist() if T else None
    cap, R = len(table[0]) * ps, len(ring)

    def one(keep, add, trees):
        """What each sequence gets, in their order, from the ring as it stood before."""
        nonlocal at, count
        why, tokens, freed = [], [], []
        took = asked = spent = back = 0
        first = [0]
        for i in range(S):
            new = keep[i] + add[i]
            n = 0
            if not (0 <= length[i] <= cap and 0 <= keep[i] <= length[i] and add[i] >= 0 and new <= cap and not (trees and add[i] > T)):
                why.append(3)
            else:
                have, need = -(-length[i] // ps), -(-new // ps)
                asked += max(need - have, 0)
                back += max(have - need, 0)
                if (need > have and asked > count) or (need < have and back > R - count):
                    why.append(1)
                else:
                    spent += add[i]
                    if add[i] and spent > s["tokens"]:
                        why.append(2)
                    else:
                        why.append(0)
                        for j in range(have, need):
                            table[i][j] = ring[(at + took) % R]
                            took += 1
                        for j in range(need, have):
                            freed.append(table[i][j])
                            table[i][j] = -1
                        n, length[i] = add[i], new
                        up = []
                        for j in range(n):
                            up.append(up[parent[i][j]] + 1 if trees and parent[i][j] >= 0 else 0 if trees else j)
                            tokens.append((i, keep[i] + j, base[i] + keep[i] + up[j]))
            first.append(first[-1] + n)
        for j, page in enumerate(freed):
            ring[(at + count + j) % R] = page
        at, count = (at + took) % R, count - took + len(freed)
        return why, tokens, first

    add = s["add"].tolist()
    why, tokens, first = one(s["start"].tolist(), add, bool(T))
    late, _, _ = one(s["keep"].tolist(), [0] * S, False)
    tokens += [(-1, -1, -1)] * (s["tokens"] - len(tokens))
    cols = list(zip(*tokens))
    i32 = torch.int32
    out = {"table": torch.tensor(table, dtype=i32), "len": torch.tensor(length, dtype=i32), "ring": torch.tensor(ring, dtype=i32),
           "state": torch.tensor([at, count], dtype=i32), "first": torch.tensor(first, dtype=i32), "seq": torch.tensor(cols[0], dtype=i32),
           "slot": torch.tensor(cols[1], dtype=i32), "pos": torch.tensor(cols[2], dtype=i32), "refused": torch.tensor(why, dtype=i32),
           "late": torch.tensor(late, dtype=i32)}
    if T:
        words = -(-T // 32)
        mask = torch.zeros(S, T, words, dtype=i32)
        for i in range(S):
            if why[i]:
                continue
            bits = []
            for j in range(add[i]):
                bits.append((bits[parent[i][j]] if parent[i][j] >= 0 else 0) | 1 << j)
            for j, b in enumerate(bits):
                w = [(b >> (32 * x)) & 0xFFFFFFFF for x in range(words)]
                mask[i, j] = torch.tensor([x - (1 << 32) if x >> 31 else x for x in w], dtype=i32)
        out["mask"] = mask
    return out


def _exact_attend(case, seed):
    s = _attend_inputs(case, seed)
    H, KV, hd = HEADS[case["heads"]]
    ps, M = case["page"], H // KV
    q = s["q"].double().view(-1, KV, M, hd)
    plen, olen, nodes, parent = (s[k].tolist() for k in ("plen", "len", "nodes", "parent"))

    def rows(pages, table, n):
        t = torch.arange(n, device="cuda")
        return pages[table[t // ps].long(), :, t % ps].double().transpose(0, 1)  # [kv head, position, head_dim]

    out = torch.zeros(s["rows"], KV, M, hd, device="cuda", dtype=torch.float64)
    r = 0
    for b, n in enumerate(nodes):
        g = b // case["beams"]
        if b % case["beams"] == 0:
            pk, pv = rows(s["k"], s["ptable"][g], plen[g]), rows(s["v"], s["ptable"][g], plen[g])
        if n == 0:
            continue
        k, v = (torch.cat([p, rows(x, s["table"][b], olen[b])], 1) for p, x in ((pk, s["k"]), (pv, s["v"])))
        ctx = plen[g] + olen[b] - n
        hide = torch.zeros(n, ctx + n, dtype=torch.bool)
        for j in range(n):
            line, x = set(), j
            while x >= 0:
                line.add(x)
                x = parent[b if len(parent) > 1 else 0][x]
            hide[j, ctx:] = torch.tensor([x not in line for x in range(n)])
        hide = hide.cuda()
        for h in range(KV):  # a kv head at a time: the scores of one are large enough
            w = torch.matmul(q[r:r + n, h].reshape(n * M, hd), k[h].t().contiguous()).view(n, M, -1) / math.sqrt(hd)
            w = torch.softmax(w.masked_fill(hide[:, None], -math.inf), -1)
            out[r:r + n, h] = torch.matmul(w.view(n * M, -1), v[h]).view(n, M, hd)
        r += n
    return out.flatten(1)


def _exact_logits(case, seed):
    s = _logits_inputs(case, seed)
    N, V = case["nodes"], case["vocab"]
    out, best = [], []
    hist, hlen, plen = s["history"].tolist(), s["hlen"].tolist(), s["plen"].tolist()
    for r in range(case["seqs"] * N):
        i, x = r // N, s["logits"][r].double()
        if r % N == 0:
            said = torch.bincount(torch.tensor(hist[i][plen[i]:hlen[i]], dtype=torch.long), minlength=V)
            told = torch.bincount(torch.tensor(hist[i][:plen[i]], dtype=torch.long), minlength=V).cuda()
        c = said.clone()
        if N > 1:
            for t in s["token"][i][s["see"][i, r % N]].tolist():
                c[t] += 1
        c = c.double().cuda()
        rep, pres, freq = (s[k][i].double() for k in ("rep", "pres", "freq"))
        at = torch.nonzero(c + told)[:, 0]
        x[at] = torch.minimum(x[at] / rep, x[at] * rep)  # a factor of at least 1 lowers both signs
        x = x - freq * c - pres * c.sign()
        if case["biases"]:
            n = int(s["blen"][i])
            x[s["btoken"][i, :n].long()] += s["bias"][i, :n].double()
        if case["grammar"] and int(s["allow_row"][r]) >= 0:
            word = s["allow"][int(s["allow_row"][r])].long() & 0xFFFFFFFF
            t = torch.arange(V, device="cuda")
            x[(word[t // 32] // 2 ** (t % 32)) % 2 == 0] = -math.inf
        best.append(int(torch.nonzero(x == x.max())[0, 0]))
        if case["out"] != "none":
            out.append(x)
    got = {}
    if case["out"] != "none":
        got["out"] = torch.stack(out)
    if case["best"]:
        got["best"] = torch.tensor(best, dtype=torch.int32)
    return got


def _exact_accept(case, seed):
    s = _accept_inputs(case, seed)
    S, N = s["parent"].shape
    parent, token, choice = s["parent"].tolist(), s["token"].tolist(), s["choice"].view(S, N).tolist()
    history, hlen, length, table, ps = s["history"].tolist(), s["hlen"].tolist(), s["len"].tolist(), s["table"].tolist(), case["page"]
    got = {k: [] for k in ("count", "path", "next", "keep")}
    k, v = s["k"].double(), s["v"].double()
    for i in range(S):
        line = [0]
        while True:
            c = [c for c in range(N) if parent[i][c] == line[-1] and token[i][c] == choice[i][line[-1]]]
            if not c:
                break
            line.append(c[0])
        begin = length[i] - N
        for to, frm in enumerate(line):
            a, b = begin + to, begin + frm
            if hlen[i] < len(history[i]):
                history[i][hlen[i]] = token[i][frm]
                hlen[i] += 1
            if to != frm:  # in this order no place is written before it is read
                for x in (k, v):
                    x[:, table[i][a // ps], :, a % ps] = x[:, table[i][b // ps], :, b % ps]
        got["count"].append(len(line))
        got["path"].append(line + [-1] * (N - len(line)))
        got["next"].append(choice[i][line[-1]])
        got["keep"].append(begin + len(line))
    got.update(history=history, hlen=hlen)
    return {**{n: torch.tensor(x, dtype=torch.int32) for n, x in got.items()}, "k": k, "v": v}


def exact(case, seed):
    return {"plan": _exact_plan, "attend": _exact_attend, "logits": _exact_logits, "accept": _exact_accept}[case["kind"]](case, seed)
