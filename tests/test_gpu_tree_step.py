"""The ops for drafted trees run together, as a server uses them: a one-layer model with random weights continues several prompts
greedily under penalties, biases and grammars; a drafter that is right most of the time proposes a tree for each step. Pages are
taken and given back on the device, lengths, masks, histories and choices never leave it. What comes out must be, token for token,
what the model says one token at a time; that statement, in 64 bits, keeps no cache."""
import ctypes

import numpy as np
import pytest

import _ops as o
import _trees as tr

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("H,KV,hd,rot,layout,most", [(4, 2, 32, 32, "halves", 9), (6, 1, 64, 16, "pairs", 36)])
def test_greedy_with_drafts(gpu, H, KV, hd, rot, layout, most):
    q, L, V, B, ps, eps, goal = gpu, gpu.load_library(), 211, 3, 16, 1e-5, 40
    rs = np.random.default_rng(hd)
    dim, words = H * hd, -(-most // 32)
    emb = rs.standard_normal((V, dim)).astype(np.float32)
    wqkv = (rs.standard_normal((dim, (H + 2 * KV) * hd)) * dim ** -0.5 * 1.5).astype(np.float32)
    wo = (rs.standard_normal((dim, V)) * dim ** -0.5 * 3).astype(np.float32)
    gains = (1 + 0.2 * rs.standard_normal((2, hd))).astype(np.float32)
    prompts = [list(map(int, rs.integers(0, V, n))) for n in (37, 64, 5)]
    rep, pres, freq = (np.array(x, np.float32) for x in ([1.0, 1.3, 1.1], [0.0, 0.2, 0.4], [0.1, 0.0, 0.3]))
    bias_token, bias = rs.integers(0, V, (B, 4)).astype(np.int32), rs.standard_normal((B, 4)).astype(np.float32)
    allow = rs.random((2, V)) < 0.7
    grammar = [-1, 0, 1]
    scale = float(np.float32(hd ** -0.5))
    f = o.freqs(rot, "none")

    # ---- the model one token at a time, in 64 bits
    def choice(i, tokens):
        x = (emb[tokens].astype(np.float64) @ wqkv.astype(np.float64)).reshape(len(tokens), H + 2 * KV, hd)
        at = np.arange(len(tokens))
        qq = o.rotate(o.norm(x[:, :H], gains[0].astype(np.float64), eps), at, f, layout)
        kk = o.rotate(o.norm(x[:, H:H + KV], gains[1].astype(np.float64), eps), at, f, layout)
        out, _, _ = o.attention(qq[-1], kk, x[:, H + KV:], scale)
        y = (out.reshape(-1) + emb[tokens[-1]].astype(np.float64)) @ wo.astype(np.float64)
        told = prompts[i][:-1]  # the prompt's last token is the first tree's root
        said = np.bincount(tokens[len(told):], minlength=V)
        seen = (said > 0) | (np.bincount(told, minlength=V) > 0)
        y = np.where(seen, np.where(y > 0, y / rep[i], y * rep[i]), y) - freq[i] * said - pres[i] * (said > 0)
        for t, b in {int(t): b for t, b in zip(bias_token[i], bias[i])}.items():
            y[t] += b
        if grammar[i] >= 0:
            y = np.where(allow[grammar[i]], y, -np.inf)
        return int(np.argmax(y))

    truth = [list(p) for p in prompts]
    for i in range(B):
        for _ in range(goal + most + 1):
            truth[i].append(choice(i, truth[i]))

    # ---- the server
    dev = q.DeviceBuffer.from_array
    stride, n_pages = 12, 26  # fewer pages than three full rows of the table
    pool = [q.DeviceBuffer(n_pages * KV * ps * hd * 4) for _ in range(2)]
    nan = np.full(n_pages * KV * ps * hd, np.nan, np.float32)
    for b in pool:
        L.qmh_memcpy_h2d(b.ptr, nan.ctypes.data, nan.nbytes)
    pages = q.Pages(dtype=o.F32, n_kv_heads=KV, head_dim=hd, page_size=ps, n_pages=n_pages, k=pool[0].ptr, v=pool[1].ptr)
    rotary = q.Rotary(rot, layout, max_pos=4096)
    i32 = lambda *n: dev(np.full(n, -1, np.int32))  # noqa: E731
    table, length, ring, state = i32(B, stride), dev(np.zeros(B, np.int32)), dev(rs.permutation(n_pages).astype(np.int32)), dev(np.array([0, n_pages], np.int32))
    keep, count, nxt, path, refused, best = i32(B), i32(B), i32(B), i32(B, most), i32(B), i32(B * most)
    hist = np.zeros((B, 200), np.int32)
    for i, p in enumerate(prompts):
        hist[i, :len(p) - 1] = p[:-1]
    dhist, dhlen, dplen = dev(hist), dev(np.array([len(p) - 1 for p in prompts], np.int32)), dev(np.array([len(p) - 1 for p in prompts], np.int32))
    dg, dedit = [dev(g) for g in gains], [dev(x) for x in (rep, pres, freq, bias_token, bias, np.full(B, 4, np.int32), tr.pack(allow, -(-V // 32)))]

    def step(tokens, add, kept, parent=None):
        """Plan and append: tokens of all sequences, in their rows. Returns the rows' places and queries."""
        n = len(tokens) + 2  # padding rows
        first, seq, slot, pos, mask = i32(B + 1), i32(n), i32(n), i32(n), i32(B, most, words)
        hold = [dev(np.array(add, np.int32)), dev(parent) if parent is not None else None]
        a = q.PlanArgs(n_seq=B, page_size=ps, table=table.ptr, table_stride=stride, len=length.ptr, keep=kept, add=hold[0].ptr, free_pages=ring.ptr,
                       free_size=n_pages, free_state=state.ptr, n_tokens=n, first=first.ptr, seq=seq.ptr, slot=slot.ptr, pos=pos.ptr,
                       refused=refused.ptr, parent=o.ptr(hold[1]), parent_stride=most, tree_size=most, mask=mask.ptr if parent is not None else None)
        q._check(L.qmh_paged_plan(ctypes.byref(a), None, 0, None), "plan")
        x, width, queries = np.zeros((n, (H + 2 * KV) * hd), np.float32), (H + 2 * KV) * hd, q.DeviceBuffer(n * dim * 4)
        x[:len(tokens)] = emb[tokens] @ wqkv
        dx = dev(x)
        a = q.AppendArgs(pages=ctypes.pointer(pages), rotary=rotary.handle, n_tokens=n, n_heads=H, q=dx.ptr, q_stride=width, q_out=queries.ptr,
                         q_out_stride=dim, k=dx.ptr + 4 * dim, k_stride=width, v=dx.ptr + 4 * (dim + KV * hd), v_stride=width, q_gain=dg[0].ptr,
                         k_gain=dg[1].ptr, eps=eps, n_seq=B, table=table.ptr, table_stride=stride, seq=seq.ptr, slot=slot.ptr, pos=pos.ptr)
        q._check(L.qmh_paged_append(ctypes.byref(a), None), "append")
        q.sync()
        assert (refused.to_array(np.int32) == 0).all()
        return n, first, mask, queries

    step(sum((p[:-1] for p in prompts), []), [len(p) - 1 for p in prompts], None)
    q._check(L.qmh_memcpy_h2d(keep.ptr, np.array([len(p) - 1 for p in prompts], np.int32).ctypes.data, 4 * B), "keep")
    told = [list(p) for p in prompts]  # all tokens so far; the last is the next root
    steps = long = 0
    while min(len(t) - len(p) for t, p in zip(told, prompts)) < goal:
        # trees: most nodes guess the model's next token, some anything
        nodes = [int(rs.integers(1, most + 1)) if len(t) - len(p) < goal else 1 for t, p in zip(told, prompts)]
        nodes = [min(n, 1 + len(truth[i]) - len(told[i])) for i, n in enumerate(nodes)]
        parent, token = np.full((B, most), -1, np.int32), np.zeros((B, most), np.int32)
        for i, n in enumerate(nodes):
            parent[i, :n] = tr.tree(rs, n)
            token[i, 0] = told[i][-1]
            d = tr.depths(parent[i, :n])
            for j in range(1, n):
                token[i, j] = truth[i][len(told[i]) - 1 + d[j]] if rs.random() < 0.75 else rs.integers(0, V)
        rows = np.concatenate([token[i, :n] for i, n in enumerate(nodes)])
        n, first, mask, queries = step(rows, nodes, keep.ptr, parent)
        dout = dev(np.zeros((n, dim), np.float32))
        base = q.AttentionArgs(pages=ctypes.pointer(pages), n_heads=H, n_seq=B, q_len=most, n_groups=B, q=queries.ptr, q_stride=dim, out=dout.ptr,
                               out_stride=dim, table=table.ptr, len=length.ptr, table_stride=stride, max_len=stride * ps, scale=scale)
        a = q.TreeArgs(base=base, n_rows=n, first=first.ptr, mask=mask.ptr, mask_stride=most * words, mask_words=words)
        need = L.qmh_tree_attention_ws(ctypes.byref(a))
        ws = q.DeviceBuffer(max(need, 16))
        q._check(L.qmh_tree_attention(ctypes.byref(a), ws.ptr, need, None), "attention")
        q.sync()
        logits = dev(((dout.to_array(np.float32).reshape(n, dim)[:len(rows)] + emb[rows]) @ wo).astype(np.float32))
        dtoken, dparent = dev(token), dev(parent)
        row_grammar = dev(np.repeat(grammar, nodes).astype(np.int32))
        a = q.LogitsArgs(dtype=o.F32, n_rows=len(rows), vocab=V, logits=logits.ptr, stride=V, best=best.ptr, n_seq=B, rows_per_seq=most,
                         first=first.ptr, history=dhist.ptr, history_stride=200, history_len=dhlen.ptr, prompt_len=dplen.ptr,
                         repetition=dedit[0].ptr, presence=dedit[1].ptr, frequency=dedit[2].ptr, bias_token=dedit[3].ptr, bias=dedit[4].ptr,
                         bias_len=dedit[5].ptr, bias_stride=4, allow=dedit[6].ptr, allow_stride=-(-V // 32), n_allow=2, allow_row=row_grammar.ptr,
                         node_token=dtoken.ptr, node_stride=most, mask=mask.ptr, mask_stride=most * words, mask_words=words)
        q._check(L.qmh_logits_edit(ctypes.byref(a), None, 0, None), "logits")
        a = q.AcceptArgs(n_seq=B, tree_size=most, parent=dparent.ptr, parent_stride=most, token=dtoken.ptr, token_stride=most, n_rows=len(rows),
                         first=first.ptr, choice=best.ptr, len=length.ptr, count=count.ptr, path=path.ptr, next=nxt.ptr, keep=keep.ptr,
                         history=dhist.ptr, history_stride=200, history_len=dhlen.ptr, pages=ctypes.pointer(pages), n_layers=1,
                         table=table.ptr, table_stride=stride)
        q._check(L.qmh_tree_accept(ctypes.byref(a), None), "accept")
        q.sync()
        c, p, x = count.to_array(np.int32), path.to_array(np.int32).reshape(B, most), nxt.to_array(np.int32)
        for i in range(B):
            told[i] += [int(token[i, k]) for k in p[i, 1:c[i]]] + [int(x[i])]
            assert told[i] == truth[i][:len(told[i])], (steps, i)
            long += c[i] > 2
        steps += 1
    assert long > 5, "no path of drafts was accepted"
    kept = keep.to_array(np.int32)
    assert list(kept) == [len(t) - 1 for t in told]
    h = dhist.to_array(np.int32).reshape(B, 200)
    for i in range(B):
        assert list(h[i, :kept[i]]) == told[i][:-1]
    # the sequences end: every page is free again
    zero = dev(np.zeros(B, np.int32))
    a = q.PlanArgs(n_seq=B, page_size=ps, table=table.ptr, table_stride=stride, len=length.ptr, keep=zero.ptr, free_pages=ring.ptr, free_size=n_pages,
                   free_state=state.ptr, refused=refused.ptr)
    q._check(L.qmh_paged_plan(ctypes.byref(a), None, 0, None), "plan")
    q.sync()
    assert sorted(ring.to_array(np.int32)) == list(range(n_pages)) and state.to_array(np.int32)[1] == n_pages
    rotary.close()
