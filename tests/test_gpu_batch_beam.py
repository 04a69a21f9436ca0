"""Beam search over a batch (qmh_batch_beam, qmh_batch_reorder) against a search on the CPU over the oracle's logits: the
forward is bitwise the oracle's, so hypotheses are equal token for token."""
import numpy as np
import pytest

from _ops import U32
from test_gpu_beam import best_of

pytestmark = pytest.mark.gpu


def bits(a):
    return np.ascontiguousarray(a).view(np.uint32)


def search(oracle, path, prompt, n_beams, n_steps, eos):
    """[(score, tokens)] best first: each step's totals in 64 bits, rounded to float as the scores kept."""
    hyps = [(np.float32(0.0), [], False)] + [(np.float32(-np.inf), [], False)] * (n_beams - 1)
    for _ in range(n_steps):
        x, score, done = [], [], []
        V = None
        for s, toks, fin in hyps:
            if s > -np.inf and not fin:
                lg, _ = oracle.run_model(path, list(prompt) + toks, 0)
                V = lg.shape[1]
                x.append(lg[-1].astype(np.float64))
            else:
                x.append(None)
            score.append(float(s))
            done.append(fin)
        V = V or 1 + max(eos, max(max(t) for _, t, _ in hyps if t))
        x = np.stack([np.zeros(V) if r is None else r for r in x])
        got = best_of(x, np.array(score), done if eos >= 0 else None, n_beams, max(eos, 0))
        hyps = [(np.float32(t), hyps[b][1] + [tok], b >= 0 and (hyps[b][2] or tok == eos)) if b >= 0 else (np.float32(-np.inf), [-1], False)
                for t, b, tok in got]
    return hyps


@pytest.mark.parametrize("shape,wt,groups,beams,steps", [("small", "q4_0", 2, 4, 6), ("gqa48", "q8_0", 1, 3, 5), ("odd", "q4_0", 3, 1, 4),
                                                         ("mha", "q4_0", 1, 17, 3)])
@pytest.mark.parametrize("end", [False, True])
def test_batch_beam_matches_a_search_on_the_oracle(gpu, oracle, small_models, shape, wt, groups, beams, steps, end):
    path = small_models[(shape, wt)]
    rs = np.random.default_rng(beams)
    with gpu.Model.load(path) as m:
        lens = [5 + 3 * g for g in range(groups)]
        prompts = [rs.integers(0, m.vocab, n).astype(np.int32) for n in lens]
        eos = -1
        if end:  # a token that some hypothesis takes early: the best second one of the first prompt
            eos = int(search(oracle, path, prompts[0], beams, 1, -1)[min(1, beams - 1)][1][0])
        with gpu.Batch(m, groups * beams) as bt:
            for k in range(max(lens) - 1):
                p = [min(k, lens[g] - 2) for g in range(groups) for _ in range(beams)]
                bt.forward([prompts[i // beams][p[i]] for i in range(groups * beams)], p, want_logits=False)
            ids, scores, ms = bt.beam([p[-1] for p in prompts], [n - 1 for n in lens], beams, steps, eos)
            assert ms > 0
            for g in range(groups):
                want = search(oracle, path, prompts[g], beams, steps, eos)
                for j in range(beams):
                    i = g * beams + j
                    assert list(ids[i]) == want[j][1], (g, j)
                    # one float per step; the log sums' 64-bit difference may tip each rounding
                    assert abs(scores[i] - want[j][0]) <= steps * 2 * U32 * abs(want[j][0])
            # the caches are the hypotheses' own: each goes on as the oracle does from its tokens
            tail = [int(r[-1]) for r in ids]
            lg = bt.forward([max(t, 0) for t in tail], [lens[i // beams] - 1 + steps for i in range(groups * beams)])
            for i in range(groups * beams):
                toks = [int(t) for t in ids[i]]
                if eos in toks[:-1]:
                    continue  # a finished one repeats eos
                want, _ = oracle.run_model(path, list(prompts[i // beams]) + toks, 0)
                assert np.array_equal(bits(lg[i]), bits(want[-1])), i


def test_batch_beam_of_one_is_greedy(gpu, small_models):
    path = small_models[("small", "q8_0")]
    with gpu.Model.load(path) as m, gpu.Batch(m, 3) as a, gpu.Batch(m, 3) as b:
        ids, _, _ = a.beam([3, 4, 5], [0, 0, 0], 1, 20)
        want, _ = b.greedy([3, 4, 5], [0, 0, 0], 20)
        assert np.array_equal(ids.T, want)


def test_batch_reorder_moves_the_caches(gpu, small_models):
    path = small_models[("gqa", "q4_0")]
    rs = np.random.default_rng(1)
    with gpu.Model.load(path) as m, gpu.Batch(m, 6) as a, gpu.Batch(m, 6) as b:
        toks = rs.integers(0, m.vocab, (6, 40)).astype(np.int32)
        parent = np.array([2, 0, 1, -1, 0, 2], np.int32)  # two groups of three: a ring, and one's state to another
        src = [2, 0, 1, 3, 3, 5]
        for k in range(39):
            a.forward(toks[:, k], [k] * 6, want_logits=False)
            b.forward(toks[src, k], [k] * 6, want_logits=False)
        a.reorder(parent, 3, 39)
        assert np.array_equal(bits(a.forward(toks[:, 39], [39] * 6)), bits(b.forward(toks[:, 39], [39] * 6)))


def test_batch_beam_refusals(gpu, small_models):
    path = small_models[("small", "q4_0")]
    L = gpu.load_library()
    with gpu.Model.load(path) as m, gpu.Batch(m, 6) as b:
        t, p = np.array([1, 2], np.int32), np.array([0, 0], np.int32)

        def call(n_beams=3, steps=2, eos=-1, tok=t, pos=p):
            return L.qmh_batch_beam(b._h, n_beams, tok.ctypes.data, pos.ctypes.data, steps, eos, None, None, None)
        assert call() == 0
        for kw in (dict(n_beams=0), dict(n_beams=4), dict(n_beams=65), dict(steps=-1), dict(eos=m.vocab), dict(tok=np.array([1, m.vocab], np.int32)),
                   dict(pos=np.array([0, m.cfg.max_seq - 1], np.int32))):
            assert call(**kw) == -1 and "batch" in gpu.last_error(), kw
        par = np.zeros(6, np.int32)
        for args in ((None, 3, 4), (par.ctypes.data, 4, 4), (par.ctypes.data, 3, -1), (par.ctypes.data, 3, m.cfg.max_seq + 1)):
            assert L.qmh_batch_reorder(b._h, *args) == -1 and "batch_reorder" in gpu.last_error()
        assert L.qmh_batch_reorder(None, par.ctypes.data, 3, 4) == -1 and L.qmh_batch_beam(None, 3, t.ctypes.data, p.ctypes.data, 1, -1, None, None, None) == -1


def test_batch_beam_again_and_with_other_group_sizes(gpu, small_models):
    """One batch used for searches of every group size and other calls in between gives what fresh ones give."""
    path = small_models[("gqa", "q4_0")]
    with gpu.Model.load(path) as m, gpu.Batch(m, 6) as a:
        for n_beams, steps in ((6, 9), (3, 12), (1, 5), (2, 7), (6, 9)):
            groups = 6 // n_beams
            tok, pos = list(range(2, 2 + groups)), [0] * groups
            got = a.beam(tok, pos, n_beams, steps, 1)
            a.greedy([7] * 6, [0] * 6, 4)
            with gpu.Batch(m, 6) as b:
                want = b.beam(tok, pos, n_beams, steps, 1)
            assert np.array_equal(got[0], want[0]) and np.array_equal(bits(got[1]), bits(want[1])), n_beams
