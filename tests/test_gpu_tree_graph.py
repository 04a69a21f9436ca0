"""A step of the ops for drafted trees on a stream of the caller's and captured into a graph: plan, attention, edits and acceptance,
replayed several times with other contents, with eager work and synchronizations between, each replay held to eager calls on copies
of the same state."""
import ctypes

import numpy as np
import pytest

import _ops as o
import _trees as tr
from test_gpu_paged import _hip

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["f16", "f32"])
def test_step_in_a_graph(gpu, dtype):
    q, L, hip, dt = gpu, gpu.load_library(), _hip(), o.TYPES[dtype]
    B, H, KV, hd, ps, stride, T, V, layers = 5, 4, 2, 64, 16, 90, 12, 5000, 2
    rs = np.random.default_rng(1)
    pool = 5 * 90
    stream, graph, exe = ctypes.c_void_p(), ctypes.c_void_p(), ctypes.c_void_p()
    assert hip.hipStreamCreate(ctypes.byref(stream)) == 0

    class Side:
        """The state and buffers of one program."""

        def __init__(self):
            sizes = dict(table=B * stride, len=B, keep=B, add=B, ring=pool, state=2, first=B + 1, seq=B * T, slot=B * T, pos=B * T, refused=B,
                         parent=B * T, token=B * T, mask=B * T, best=B * T, count=B, path=B * T, next=B, back=B, hist=B * 400, hlen=B)
            self.i = {k: q.DeviceBuffer.from_array(np.full(n, -1, np.int32)) for k, n in sizes.items()}
            es = o.BYTES[dt]
            self.k, self.v = (q.DeviceBuffer(layers * pool * KV * ps * hd * es) for _ in range(2))
            self.x, self.out = q.DeviceBuffer(B * T * H * hd * es), q.DeviceBuffer(B * T * H * hd * es)
            self.logits, self.edited, self.f = q.DeviceBuffer(B * T * V * es), q.DeviceBuffer(B * T * V * es), q.DeviceBuffer(4 * B)
            self.pages = q.Pages(dtype=dt, n_kv_heads=KV, head_dim=hd, page_size=ps, n_pages=pool, k=self.k.ptr, v=self.v.ptr)
            self.ws = []

        def put(self, name, a):
            b = self.i[name] if name in self.i else getattr(self, name)
            a = np.ascontiguousarray(a)
            assert a.nbytes <= b.nbytes
            assert L.qmh_memcpy_h2d(b.ptr, a.ctypes.data, a.nbytes) == 0

        def step(self, s):
            """The calls of a step on stream s; the arguments stay alive with the side."""
            i = {k: b.ptr for k, b in self.i.items()}
            plan = q.PlanArgs(n_seq=B, page_size=ps, table=i["table"], table_stride=stride, len=i["len"], keep=i["keep"], add=i["add"],
                              free_pages=i["ring"], free_size=pool, free_state=i["state"], n_tokens=B * T, first=i["first"], seq=i["seq"],
                              slot=i["slot"], pos=i["pos"], refused=i["refused"], parent=i["parent"], parent_stride=T, tree_size=T, mask=i["mask"])
            base = q.AttentionArgs(pages=ctypes.pointer(self.pages), n_heads=H, n_seq=B, q_len=T, n_groups=B, q=self.x.ptr, q_stride=H * hd,
                                   out=self.out.ptr, out_stride=H * hd, table=i["table"], len=i["len"], table_stride=stride, max_len=stride * ps,
                                   scale=0.125)
            tree = q.TreeArgs(base=base, n_rows=B * T, first=i["first"], mask=i["mask"], mask_stride=T, mask_words=1)
            edit = q.LogitsArgs(dtype=dt, n_rows=B * T, vocab=V, logits=self.logits.ptr, stride=V, out=self.edited.ptr, out_stride=V, best=i["best"],
                                n_seq=B, rows_per_seq=T, first=i["first"], history=i["hist"], history_stride=400, history_len=i["hlen"],
                                repetition=self.f.ptr, presence=self.f.ptr, node_token=i["token"], node_stride=T, mask=i["mask"], mask_stride=T,
                                mask_words=1)
            acc = q.AcceptArgs(n_seq=B, tree_size=T, parent=i["parent"], parent_stride=T, token=i["token"], token_stride=T, n_rows=B * T,
                               first=i["first"], choice=i["best"], len=i["len"], count=i["count"], path=i["path"], next=i["next"],
                               keep=i["back"], history=i["hist"], history_stride=400, history_len=i["hlen"],
                               pages=ctypes.pointer(self.pages), n_layers=layers, layer_stride=pool * KV * ps * hd, table=i["table"],
                               table_stride=stride)
            if not self.ws:
                self.ws = [(n, q.DeviceBuffer(max(n, 16))) for n in (L.qmh_paged_plan_ws(ctypes.byref(plan)), L.qmh_tree_attention_ws(ctypes.byref(tree)),
                                                                     L.qmh_logits_edit_ws(ctypes.byref(edit)))]
                assert self.ws[1][0] and self.ws[2][0], "parts to join in both"
            w = self.ws
            q._check(L.qmh_paged_plan(ctypes.byref(plan), w[0][1].ptr, w[0][0], s), "plan")
            q._check(L.qmh_tree_attention(ctypes.byref(tree), w[1][1].ptr, w[1][0], s), "attention")
            q._check(L.qmh_logits_edit(ctypes.byref(edit), w[2][1].ptr, w[2][0], s), "logits")
            q._check(L.qmh_tree_accept(ctypes.byref(acc), s), "accept")

        def everything(self):
            return [b.to_array(np.uint8).tobytes() for b in (*self.i.values(), self.k, self.v, self.out, self.edited)]

    a, b = Side(), Side()
    ring, table = rs.permutation(pool).astype(np.int32), np.full((B, stride), -1, np.int32)
    kv = [o.encode(rs.standard_normal((layers, pool, KV, ps, hd)), dt) for _ in range(2)]
    for x in (a, b):
        for name, v in dict(ring=ring, state=np.array([3, pool], np.int32), table=table, len=np.zeros(B, np.int32), hlen=np.zeros(B, np.int32),
                            hist=np.zeros(B * 400, np.int32), k=kv[0], v=kv[1], f=np.full(B, 1.25, np.float32)).items():
            x.put(name, v)
        zero = np.zeros(x.out.nbytes, np.uint8)
        x.put("out", zero)
        x.put("edited", np.zeros(x.edited.nbytes, np.uint8))
    keep, ok = np.zeros(B, np.int32), False  # by the bounds, attention and edits run in parts whatever the lengths
    for replay in range(6):
        add = rs.integers(0, T + 1, B).astype(np.int32)
        parent = np.stack([tr.tree(rs, T) for _ in range(B)])
        token = rs.integers(0, V, (B, T)).astype(np.int32)
        x = o.encode(rs.standard_normal((B * T, H * hd)), dt)
        logits = rs.standard_normal((B * T, V))
        first = tr.starts(add)
        for i in range(B):
            for c in range(1, add[i]):
                logits[first[i] + parent[i, c], token[i, c]] = 9.0  # the model agrees with some child of every node
        for side in (a, b):
            for name, v in dict(keep=keep, add=add, parent=parent, token=token, x=x, logits=o.encode(logits, dt)).items():
                side.put(name, v)
        q.sync()
        if replay == 0:
            a.step(stream)
            assert hip.hipStreamSynchronize(stream) == 0
        else:
            if replay == 1:
                assert hip.hipStreamBeginCapture(stream, 0) == 0
                a.step(stream)
                assert hip.hipStreamEndCapture(stream, ctypes.byref(graph)) == 0
                assert hip.hipGraphInstantiate(ctypes.byref(exe), graph, None, None, ctypes.c_size_t(0)) == 0
            assert hip.hipGraphLaunch(exe, stream) == 0
            assert hip.hipStreamSynchronize(stream) == 0
        b.step(None)
        q.sync()
        assert a.everything() == b.everything(), replay
        got = a.i["back"].to_array(np.int32)
        assert (a.i["refused"].to_array(np.int32) == 0).all()
        ok |= bool((a.i["count"].to_array(np.int32) > 2).any())
        keep = got
    assert ok, "no path was longer than two nodes"
    hip.hipGraphExecDestroy(exe)
    hip.hipGraphDestroy(graph)
    hip.hipStreamDestroy(stream)
