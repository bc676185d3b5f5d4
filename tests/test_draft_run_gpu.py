"""The draft-verification operators as they are used together, and the log
probabilities of a loaded model.

The run: a tree of drafted tokens attends the cache and votes on its rows, its
logits are scored, an accepted path's rows are moved behind the cache, and when
the cache is full the rows with the smallest totals leave it; a later token
attends what is left.  Every step is compared with the same steps in 64 bits on
the host, from the definitions.  Tolerances: the attention's error is bounded
by 2 (hd + 8) u D + (2 n + 64) u relative to the weighted values (u = 2^-24, D
the largest score by magnitude of its terms, below 64 here, n below 256), so
2 * 72 * 64 u + 576 u < 6e-4; values are moved, not computed, so caches are
compared for equality."""
import os
import subprocess
import sys

import numpy as np
import pytest
import torch

from smallm_engine_b200 import CudaModel, Generator, GreedySampler, SmallmError, TopKSampler, synth
from test_attention_tree_gpu import random_parents, tree_bits, words_of

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


def attend(q, k, v, n, seen, G):
    """64-bit reference: outputs [T][H][hd] and weights [kv][n + T]."""
    T, H, hd = q.shape
    N = n + T
    vis = np.ones((T, N), bool)
    vis[:, n:] = seen
    out = np.zeros((T, H, hd))
    tot = np.zeros((k.shape[0], N))
    for h in range(H):
        g = h // G
        s = q[:, h].astype(np.float64) @ k[g, :N].astype(np.float64).T / np.sqrt(hd)
        s[~vis] = -np.inf
        e = np.exp(s - s.max(1, keepdims=True))
        p = e / e.sum(1, keepdims=True)
        out[:, h] = p @ v[g, :N].astype(np.float64)
        tot[g] += p.sum(0)
    return out, tot


def test_verify_commit_evict(be):
    H, kv, hd, max_ctx, vocab, budget = 8, 2, 64, 160, 997, 96
    G = H // kv
    rng = np.random.default_rng(3)
    k, v = (rng.standard_normal((kv, max_ctx, hd), dtype=np.float32) for _ in range(2))
    w = np.zeros((kv, max_ctx), np.float32)
    kd, vd, wd = (torch.from_numpy(x).cuda() for x in (k, v, w))
    k, v, w = k.copy(), v.copy(), w.astype(np.float64)
    proj = torch.from_numpy(0.1 * rng.standard_normal((H * hd, vocab), dtype=np.float32)).cuda()
    n = 100
    be.device_errors()
    s = torch.cuda.Stream()
    for step in range(4):
        # a drafted tree: its rows are appended, it attends, and is scored
        T = 11 + step
        parents = random_parents(T, rng)
        seen = tree_bits(parents)
        rows = rng.standard_normal((2, kv, T, hd), dtype=np.float32)
        q = rng.standard_normal((T, H, hd), dtype=np.float32)
        tokens = rng.integers(0, vocab, T)
        need = be.attention_tree_workspace(H, kv, hd, n, T, True)
        with torch.cuda.stream(s):
            kd[:, n:n + T], vd[:, n:n + T] = (torch.from_numpy(x).cuda() for x in rows)
            wd[:, n:n + T] = 0
            work = torch.empty(max(need, 16), dtype=torch.uint8, device="cuda")
            out = torch.empty(T, H, hd, device="cuda")
            qd, mask, tok = torch.from_numpy(q).cuda(), words_of(seen), torch.from_numpy(tokens.astype(np.int32)).cuda()
            lp, ent = torch.empty(T, device="cuda"), torch.empty(T, device="cuda")
            ids, tlp = torch.empty(T, 3, dtype=torch.int32, device="cuda"), torch.empty(T, 3, device="cuda")
            be.attention_tree(qd.data_ptr(), kd.data_ptr(), vd.data_ptr(), out.data_ptr(), H, kv, hd, max_ctx, n, T,
                              work.data_ptr(), need, mask=mask.data_ptr(), weights=wd.data_ptr(), stream=s.cuda_stream)
            logits = out.view(T, H * hd) @ proj
            be.logprobs(logits.data_ptr(), T, vocab, tok.data_ptr(), lp.data_ptr(), ent.data_ptr(), 3, ids.data_ptr(),
                        tlp.data_ptr(), stream=s.cuda_stream)
        s.synchronize()
        k[:, n:n + T], v[:, n:n + T], w[:, n:n + T] = rows[0], rows[1], 0
        want, tot = attend(q, k, v, n, seen, G)
        scale = np.abs(v[:, :n + T]).max()
        assert np.abs(out.cpu().numpy() - want).max() <= 6e-4 * scale
        w[:, :n + T] += tot
        assert np.abs(wd[:, :n + T].cpu().numpy() - w[:, :n + T]).max() <= 6e-4 * H * T
        ref = torch.log_softmax(logits.double(), 1)
        assert float((lp.double() - ref[range(T), tokens]).abs().max()) <= 700 * U
        assert ids.cpu().numpy().tolist() == torch.sort(logits, dim=1, descending=True, stable=True).indices[:, :3].tolist()
        # accept the path to one of the last tokens; its rows close up
        path, u = [], T - 1
        while u >= 0:
            path.append(u)
            u = parents[u]
        path = n + np.array(path[::-1])
        be.cache_move(kd.data_ptr(), vd.data_ptr(), kv, hd, max_ctx,
                      (lst := torch.from_numpy(path.astype(np.int32)).cuda()).data_ptr(), path.size, n,
                      weights=wd.data_ptr())
        be.synchronize()
        for x in (k, v, w):
            x[:, n:n + path.size] = x[:, path]
        n += path.size
        # over budget: the least attended rows leave
        if n > budget:
            first, last = 4, 16
            kept = torch.empty(kv, budget, dtype=torch.int32, device="cuda")
            torch.cuda.synchronize()
            be.cache_select(wd.data_ptr(), kv, max_ctx, n, budget, first, last, kept.data_ptr())
            be.cache_move(kd.data_ptr(), vd.data_ptr(), kv, hd, max_ctx, kept.data_ptr(), budget, 0, per_head=True,
                          weights=wd.data_ptr())
            be.synchronize()
            rows_kept = kept.cpu().numpy()
            totals = wd.cpu().numpy()
            for g in range(kv):
                assert np.all(np.diff(rows_kept[g]) > 0)
                assert rows_kept[g, :first].tolist() == list(range(first))
                assert rows_kept[g, -last:].tolist() == list(range(n - last, n))
                gone = np.setdiff1d(np.arange(first, n - last), rows_kept[g])
                mid = rows_kept[g, first:-last]
                # by the totals in 64 bits, within their tolerance
                assert w[g, mid].min() >= w[g, gone].max() - 2 * 6e-4 * H * T * (step + 1)
                for x in (k, v, w):
                    x[g, :budget] = x[g, rows_kept[g]]
            assert np.abs(totals[:, :budget] - w[:, :budget]).max() <= 6e-4 * H * T * (step + 1)
            n = budget
        np.testing.assert_array_equal(kd[:, :n].cpu().numpy(), k[:, :n])
        np.testing.assert_array_equal(vd[:, :n].cpu().numpy(), v[:, :n])
        wd[:, :n] = torch.from_numpy(w[:, :n].astype(np.float32)).cuda()
    # a single token over what is left
    q = rng.standard_normal((1, H, hd), dtype=np.float32)
    need = be.attention_tree_workspace(H, kv, hd, n, 1)
    work, out = torch.empty(max(need, 16), dtype=torch.uint8, device="cuda"), torch.empty(1, H, hd, device="cuda")
    qd = torch.from_numpy(q).cuda()
    torch.cuda.synchronize()
    be.attention_tree(qd.data_ptr(), kd.data_ptr(), vd.data_ptr(), out.data_ptr(), H, kv, hd, max_ctx, n, 1,
                      work.data_ptr(), need)
    be.synchronize()
    want, _ = attend(q, kd.cpu().numpy(), vd.cpu().numpy(), n, np.ones((1, 1), bool), G)
    assert np.abs(out.cpu().numpy() - want).max() <= 6e-4 * np.abs(v).max()
    assert be.device_errors() == 0


def test_two_calls_at_once(be):
    """Two streams, a workspace each: the same bits as one after the other."""
    H, kv, hd, n, T = 32, 8, 128, 3000, 8
    sets = []
    for seed in (1, 2):
        g = torch.Generator(device="cuda").manual_seed(seed)
        q = torch.randn(T, H * hd, device="cuda", generator=g)
        k, v = (torch.randn(kv, n + T, hd, device="cuda", generator=g) for _ in range(2))
        need = be.attention_tree_workspace(H, kv, hd, n, T, True)
        sets.append((q, k, v, torch.empty(need, dtype=torch.uint8, device="cuda"), need))

    def call(i, stream, out, w):
        q, k, v, work, need = sets[i]
        be.attention_tree(q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), H, kv, hd, n + T, n, T,
                          work.data_ptr(), need, weights=w.data_ptr(), stream=stream)
    alone, both = [], []
    for dst in (alone, both):
        dst += [(torch.zeros(T, H * hd, device="cuda"), torch.zeros(kv, n + T, device="cuda")) for _ in sets]
    streams = [torch.cuda.Stream() for _ in sets]
    torch.cuda.synchronize()
    for i, st in enumerate(streams):
        call(i, st.cuda_stream, *alone[i])
        torch.cuda.synchronize()
    for rep in range(5):
        for _, w in both:
            w.zero_()
        torch.cuda.synchronize()
        for i, st in enumerate(streams):
            call(i, st.cuda_stream, *both[i])
        torch.cuda.synchronize()
        for a, b in zip(alone, both):
            assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def chain_of_calls(be, st):
    """attention with totals, select, move, logprobs of the output, on stream st."""
    H, kv, hd, n, T = 8, 2, 64, 700, 5
    g = torch.Generator(device="cuda").manual_seed(11)
    q = torch.randn(T, H * hd, device="cuda", generator=g)
    k0, v0 = (torch.randn(kv, n + T, hd, device="cuda", generator=g) for _ in range(2))
    k, v, w = k0.clone(), v0.clone(), torch.zeros(kv, n + T, device="cuda")
    need = be.attention_tree_workspace(H, kv, hd, n, T, True)
    work = torch.empty(need, dtype=torch.uint8, device="cuda")
    out, rows = torch.empty(T, H * hd, device="cuda"), torch.empty(kv, 300, dtype=torch.int32, device="cuda")
    ent = torch.empty(T, device="cuda")
    torch.cuda.synchronize()

    def reset():
        k.copy_(k0), v.copy_(v0), w.zero_()

    def attend_(s):
        be.attention_tree(q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), H, kv, hd, n + T, n, T,
                          work.data_ptr(), need, weights=w.data_ptr(), stream=s.cuda_stream)

    def evict(s):
        be.cache_select(w.data_ptr(), kv, n + T, n + T, 300, 4, 16, rows.data_ptr(), stream=s.cuda_stream)
        be.cache_move(k.data_ptr(), v.data_ptr(), kv, hd, n + T, rows.data_ptr(), 300, 0, per_head=True,
                      weights=w.data_ptr(), stream=s.cuda_stream)

    def score(s):
        be.logprobs(out.data_ptr(), T, H * hd, None, None, ent.data_ptr(), 0, None, None, stream=s.cuda_stream)
    return reset, attend_, evict, score, (k, v, w, out, rows, ent, q, work)


def test_captured_with_other_streams(be):
    """One graph over two streams: scoring beside the eviction, both after the
    attention, replayed: the same bits as one call after the other."""
    st, side = torch.cuda.Stream(), torch.cuda.Stream()
    reset, attend_, evict, score, t = chain_of_calls(be, st)
    with torch.cuda.stream(st):
        reset()
        attend_(st), evict(st), score(st)
    st.synchronize()
    want = [x.clone() for x in t[:6]]
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=st):
        reset()
        attend_(st)
        side.wait_stream(st)
        score(side)
        evict(st)
        st.wait_stream(side)
        t[5].add_(1)
    for _ in range(3):
        for x in (t[3], t[4], t[5]):
            x.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(want[:5], t)) and torch.equal(want[5] + 1, t[5])
    assert be.device_errors() == 0


FIRST = """
import sys, torch
sys.path.insert(0, {tests!r})
from smallm_engine_b200 import CUDABackend
from test_draft_run_gpu import chain_of_calls
be = CUDABackend()
st = torch.cuda.Stream()
reset, attend_, evict, score, t = chain_of_calls(be, st)
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph, stream=st):
    reset()
    attend_(st), evict(st), score(st)
graph.replay()
torch.cuda.synchronize()
got = [x.clone() for x in t[:6]]
with torch.cuda.stream(st):
    reset()
    attend_(st), evict(st), score(st)
st.synchronize()
assert all(torch.equal(a, b) for a, b in zip(got, t))
print("same")
"""


def test_first_calls_captured():
    """The very first calls of a process may be captured ones."""
    here = os.path.dirname(os.path.abspath(__file__))
    r = subprocess.run([sys.executable, "-c", FIRST.format(tests=here)], capture_output=True, text=True, timeout=300,
                       cwd=os.path.dirname(here))
    assert r.returncode == 0 and r.stdout.strip().endswith("same"), r.stderr[-2000:]


def test_bad_list_is_not_a_steps_error(be, gguf_dir):
    """Bit 7 stays for the caller of cache_move to read; a model steps on."""
    m = CudaModel(synth.write_gguf(synth.tiny_spec("llama-q4_0"), 8, gguf_dir / "lp-llama2.gguf"))
    want = m.forward(5, 0)
    k, v = torch.zeros(2, 1, 64, 32, device="cuda")
    rows = torch.tensor([3, 3], dtype=torch.int32, device="cuda")
    torch.cuda.synchronize()
    be.device_errors()
    be.cache_move(k.data_ptr(), v.data_ptr(), 1, 32, 64, rows.data_ptr(), 2, 0)
    be.synchronize()
    m.reset_cache()
    np.testing.assert_array_equal(m.forward(5, 0), want)
    assert m.logprobs(1).token == 1
    assert be.device_errors() == 128 and be.device_errors() == 0
    m.close()


def test_model_logprobs_and_generator(gguf_dir):
    spec = synth.tiny_spec("llama-q4_0")
    m = CudaModel(synth.write_gguf(spec, 8, gguf_dir / "lp-llama.gguf"))
    for pos, tok in enumerate([5, 9, 200]):
        logits = m.forward(tok, pos).astype(np.float64)
        d = logits - logits.max()
        ref = d - np.log(np.exp(d).sum())
        r = m.logprobs(17, 8)
        assert r.token == 17 and abs(r.logprob - ref[17]) <= 700 * U
        assert abs(r.entropy + (np.exp(ref) * ref).sum()) <= 2 * 516 * U * 8
        order = np.argsort(-logits, kind="stable")[:8]
        assert [i for i, _ in r.top] == order.tolist()
        assert np.abs(np.array([p for _, p in r.top]) - ref[order]).max() <= 700 * U
        assert m.logprobs().logprob is None and m.logprobs().entropy == r.entropy
    with pytest.raises(SmallmError):
        m.logprobs(spec.vocab)
    with pytest.raises(SmallmError):
        m.logprobs(0, 65)
    # the generator's tokens do not depend on asking, and each is scored in the
    # distribution it was taken from
    m.reset_cache()
    plain = Generator(m, GreedySampler()).generate([5, 9, 200, 31], 8)
    m.reset_cache()
    g = Generator(m, GreedySampler(), logprobs=2)
    assert g.generate([5, 9, 200, 31], 8) == plain
    assert [r.token for r in g.logprobs] == plain
    for r in g.logprobs:
        assert r.top[0] == (r.token, r.logprob) and r.top[0][1] >= r.top[1][1]
    m.reset_cache()
    g = Generator(m, TopKSampler(5, 1.0, 3), logprobs=5)
    out = g.generate([5, 9, 200, 31], 6)
    assert all(r.token in [i for i, _ in r.top] for r in g.logprobs) and [r.token for r in g.logprobs] == out
    m.close()
