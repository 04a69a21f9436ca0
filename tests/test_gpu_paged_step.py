"""The ops for several continuations of one prompt run together, as a program uses them: a one-layer model with random
weights answers two prompts by beam search. The prompt's keys and values go to shared pages once; each step appends the
beams' tokens, attends, selects and reorders the beams' own pages. The same search in 64 bits keeps no cache: it
recomputes every hypothesis from its tokens."""
import ctypes

import numpy as np
import pytest

import _ops as o
from test_gpu_beam import best_of

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("reorder", ["pages", "tables"])
@pytest.mark.parametrize("H,KV,hd,rot,layout,K", [(4, 2, 32, 32, "halves", 3), (6, 1, 64, 16, "pairs", 5)])
def test_beam_search_over_pages(gpu, H, KV, hd, rot, layout, K, reorder):
    q, L, V, G, ps, steps, eps = gpu, gpu.load_library(), 300, 2, 16, 22, 1e-5
    rs = np.random.default_rng(hd)
    dim, B = H * hd, G * K
    emb = rs.standard_normal((V, dim)).astype(np.float32)
    wqkv = (rs.standard_normal((dim, (H + 2 * KV) * hd)) * dim ** -0.5 * 1.5).astype(np.float32)
    wo = (rs.standard_normal((dim, V)) * dim ** -0.5 * 3).astype(np.float32)
    gains = (1 + 0.2 * rs.standard_normal((2, hd))).astype(np.float32)
    prompts = [rs.integers(0, V, n) for n in (37, 64)]
    first = [int(p[-1]) for p in prompts]
    plen = [len(p) - 1 for p in prompts]  # the last token is the first step's
    scale = float(np.float32(hd ** -0.5))

    # ---- the search in 64 bits, from the tokens alone
    f = o.freqs(rot, "none")

    def logits_of(tokens):
        x = emb[tokens].astype(np.float64) @ wqkv.astype(np.float64)
        x = x.reshape(len(tokens), H + 2 * KV, hd)
        at = np.arange(len(tokens))
        qq = o.rotate(o.norm(x[:, :H], gains[0].astype(np.float64), eps), at, f, layout)
        kk = o.rotate(o.norm(x[:, H:H + KV], gains[1].astype(np.float64), eps), at, f, layout)
        out, _, _ = o.attention(qq[-1], kk, x[:, H + KV:], scale)
        return out, (out.reshape(-1) + emb[tokens[-1]].astype(np.float64)) @ wo.astype(np.float64)

    # ---- the pages: prompts' ones shared, own ones of each beam
    own_pages = -(-steps // ps)
    tables, n_pages = o.make_tables(rs, [-(-n // ps) for n in plen] + [own_pages] * B, 6)
    table, ptable = tables[G:].copy(), tables[:G].copy()
    pool = [q.DeviceBuffer(n_pages * KV * ps * hd * 4) for _ in range(2)]
    nan = np.full(n_pages * KV * ps * hd, np.nan, np.float32)
    for b in pool:
        L.qmh_memcpy_h2d(b.ptr, nan.ctypes.data, nan.nbytes)
    pages = q.Pages(dtype=o.F32, n_kv_heads=KV, head_dim=hd, page_size=ps, n_pages=n_pages, k=pool[0].ptr, v=pool[1].ptr)
    rotary = q.Rotary(rot, layout, max_pos=4096)
    dev = q.DeviceBuffer.from_array
    dg = [dev(g) for g in gains]

    def append(tokens, seq, slot, pos, tab, n_seq):
        n, width = len(tokens), (H + 2 * KV) * hd
        x = dev((emb[tokens] @ wqkv).astype(np.float32))
        out, keep = q.DeviceBuffer(n * dim * 4), [dev(np.array(a, np.int32)) for a in (seq, slot, pos)]
        dtab = dev(tab)
        a = q.AppendArgs(pages=ctypes.pointer(pages), rotary=rotary.handle, n_tokens=n, n_heads=H, q=x.ptr, q_stride=width, q_out=out.ptr,
                         q_out_stride=dim, k=x.ptr + 4 * dim, k_stride=width, v=x.ptr + 4 * (dim + KV * hd), v_stride=width, q_gain=dg[0].ptr,
                         k_gain=dg[1].ptr, eps=eps, n_seq=n_seq, table=dtab.ptr, table_stride=tab.shape[1], seq=keep[0].ptr,
                         slot=keep[1].ptr, pos=keep[2].ptr)
        q._check(L.qmh_paged_append(ctypes.byref(a), None), "append")
        q.sync()
        return out

    tok = np.concatenate([p[:-1] for p in prompts])
    append(tok, np.repeat([0, 1], plen), np.concatenate([np.arange(n) for n in plen]), np.concatenate([np.arange(n) for n in plen]), ptable, G)

    hyps = [[[]] * K for _ in range(G)]
    score = np.where(np.arange(B) % K == 0, 0.0, -np.inf).astype(np.float32)
    dscore, dparent, dtoken = dev(score), q.DeviceBuffer(4 * B), q.DeviceBuffer(4 * B)
    dptab, dplen = dev(ptable), dev(np.array(plen, np.int32))
    now = np.repeat(first, K)
    for step in range(steps):
        dq = append(now, np.arange(B), [step] * B, np.repeat(plen, K) + step, table, B)
        dtab, dlen, dout = dev(table), dev(np.full(B, step + 1, np.int32)), q.DeviceBuffer(B * dim * 4)
        a = q.AttentionArgs(pages=ctypes.pointer(pages), n_heads=H, n_seq=B, q_len=1, n_groups=G, q=dq.ptr, q_stride=dim, out=dout.ptr,
                            out_stride=dim, table=dtab.ptr, len=dlen.ptr, table_stride=table.shape[1], max_len=steps, prefix_table=dptab.ptr,
                            prefix_len=dplen.ptr, prefix_stride=ptable.shape[1], max_prefix=max(plen), scale=scale)
        need = L.qmh_paged_attention_ws(ctypes.byref(a))
        ws = q.DeviceBuffer(max(need, 1))
        q._check(L.qmh_paged_attention(ctypes.byref(a), ws.ptr, need, None), "attention")
        q.sync()
        out = dout.to_array(np.float32).reshape(B, H, hd)
        lg = ((out.reshape(B, dim) + emb[now]) @ wo).astype(np.float32)
        dlg = dev(lg)
        s = q.BeamArgs(dtype=o.F32, n_groups=G, n_beams=K, vocab=V, n_out=K, eos=0, logits=dlg.ptr, stride=V, score=dscore.ptr,
                       out_score=dscore.ptr, out_parent=dparent.ptr, out_token=dtoken.ptr)
        need = L.qmh_beam_select_ws(ctypes.byref(s))
        ws2 = q.DeviceBuffer(need)
        q._check(L.qmh_beam_select(ctypes.byref(s), ws2.ptr, need, None), "select")
        q.sync()
        parent, token = dparent.to_array(np.int32).reshape(G, K), dtoken.to_array(np.int32).reshape(G, K)
        for g in range(G):
            x = np.zeros((K, V))
            for j in range(K):
                if score[g * K + j] > -np.inf:
                    want, x[j] = logits_of(list(prompts[g]) + hyps[g][j])
                    # 32-bit projections of `dim` terms on both sides of an attention over tens of positions
                    o.close(out[g * K + j], want, 2e-4 * np.abs(want).max(), f"step {step} beam {j}")
            got = best_of(x, score[g * K:(g + 1) * K].astype(np.float64), None, K, 0)
            assert list(parent[g]) == [w[1] for w in got] and list(token[g]) == [w[2] for w in got], step
            hyps[g] = [hyps[g][b] + [t] for _, b, t in got]
            score[g * K:(g + 1) * K] = [w[0] for w in got]
        now = token.reshape(-1)
        if reorder == "pages":
            q._check(L.qmh_paged_reorder(ctypes.byref(pages), dtab.ptr, table.shape[1], dlen.ptr, step + 1, dparent.ptr, G, K, None), "reorder")
            q.sync()
        else:
            # whole pages are shared by their numbers: the tables' rows move, and the page in use is copied to one of one's own
            part = (step + 1) % ps
            st = q.BeamState(n_outer=1, seq_stride=table.shape[1] * 4, n_rows=1, row_stride=0, live=4 * ((step + 1) // ps))
            q._check(L.qmh_beam_reorder(ctypes.byref(st), dtab.ptr, dtab.ptr, dparent.ptr, G, K, None), "tables")
            if part:
                sub = dev(np.ascontiguousarray(table[:, (step + 1) // ps:(step + 1) // ps + 1]))
                plive = dev(np.full(B, part, np.int32))
                q._check(L.qmh_paged_reorder(ctypes.byref(pages), sub.ptr, 1, plive.ptr, part, dparent.ptr, G, K, None), "page")
            q.sync()
            table = dtab.to_array(np.int32).reshape(table.shape)
    rotary.close()
