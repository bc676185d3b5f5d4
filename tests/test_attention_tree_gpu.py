"""Attention of drafted tokens over the KV cache (smallm_attention_tree)
against its definition in 64 bits.

Tolerance.  With u = 2^-24, a score is a sum of hd products: its error is at
most E = (hd + 8) u D, D the largest sum of |q_d k_d| / sqrt(hd) over the
token's seen rows (the 8: operands held to 2^-22 in two halves, the scale).
That changes a weight by the factor e^{+-E}, the softmax by twice that.  The
sums over n rows add at most n u each for the weights' sum and the output, and
the exponential, the joins and the division a few u more:
    |out - exact| <= (2 E + (2 n + 64) u) sum_k p_k |v_k|
    |totals - exact| <= (2 E + (n + T G + 64) u) sum p   (+ u |total|)
"""
import numpy as np
import pytest
import torch

from smallm_engine_b200 import SmallmError, _lib

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


def tree_bits(parents):
    T = len(parents)
    m = np.zeros((T, T), bool)
    for t in range(T):
        u = t
        while u >= 0:
            m[t, u] = True
            u = parents[u]
    return m


def words_of(seen):
    """bool [T][T] -> int32 words [T][ceil(T / 32)] on the GPU"""
    T = seen.shape[0]
    W = (T + 31) // 32
    pad = np.zeros((T, W * 32), bool)
    pad[:, :T] = seen
    w = np.packbits(pad, axis=1, bitorder="little").view(np.uint32)
    return torch.from_numpy(w.astype(np.int64).astype(np.uint32).view(np.int32).copy()).cuda()


def random_parents(T, rng):
    return [int(rng.integers(-1, t)) for t in range(T)]


def inputs(H, kv, hd, n, T, max_ctx, seed, pad=0, q_scale=2.5):
    g = torch.Generator(device="cuda").manual_seed(seed)
    q = q_scale * torch.randn(T, H * hd + pad, device="cuda", generator=g)
    k = torch.randn(kv, max_ctx, hd, device="cuda", generator=g)
    v = torch.randn(kv, max_ctx, hd, device="cuda", generator=g)
    return q, k, v


def run(be, q, k, v, H, n, T, mask=None, weights=None, out=None, stream=None, work=None):
    kv, max_ctx, hd = k.shape
    need = be.attention_tree_workspace(H, kv, hd, n, T, weights is not None)
    if work is None:
        work = torch.full((max(need, 16),), 0xFF, dtype=torch.uint8, device="cuda")
    if out is None:
        out = torch.full((T, H * hd), float("nan"), device="cuda")
    torch.cuda.synchronize()
    be.attention_tree(q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), H, kv, hd, max_ctx, n, T,
                      work.data_ptr(), need, mask=None if mask is None else mask.data_ptr(),
                      weights=None if weights is None else weights.data_ptr(), q_stride=q.stride(0),
                      out_stride=out.stride(0), stream=stream)
    torch.cuda.synchronize()
    return out


def check(out, q, k, v, H, n, T, seen, totals=None, before=None):
    """seen: bool [T][T] over the drafted rows."""
    kv, _, hd = k.shape
    G, N = H // kv, n + T
    vis = torch.ones(T, N, dtype=torch.bool, device="cuda")
    vis[:, n:] = torch.from_numpy(np.asarray(seen)).cuda()
    want_tot = torch.zeros(kv, N, dtype=torch.float64, device="cuda")
    tol_tot = torch.zeros_like(want_tot)
    for h in range(H):
        g = h // G
        qh = q[:, h * hd:(h + 1) * hd].double()
        kh = torch.where(vis.any(0)[:, None], k[g, :N].double(), 0.0)
        vh = torch.where(vis.any(0)[:, None], v[g, :N].double(), 0.0)
        s = (qh @ kh.T) / hd ** 0.5
        s = torch.where(vis, s, -torch.inf)
        D = torch.where(vis, (qh.abs() @ kh.abs().T) / hd ** 0.5, 0.0).amax(1)
        top = s.amax(1, keepdim=True)
        e = torch.where(vis, torch.exp(s - torch.where(top == -torch.inf, 0.0, top)), 0.0)
        L = e.sum(1, keepdim=True)
        p = torch.where(L > 0, e / L, 0.0)
        rel = 2 * (hd + 8) * U * D
        want = p @ vh
        tol = (rel + (2 * N + 64) * U)[:, None] * (p @ vh.abs()) + 1e-37
        got = out[:, h * hd:(h + 1) * hd].double()
        assert bool(((got - want).abs() <= tol).all()), (h, float(((got - want).abs() / tol).max()))
        want_tot[g] += p.sum(0)
        tol_tot[g] += ((rel + (N + T * G + 64) * U)[:, None] * p).sum(0)
    if totals is not None:
        want_tot += before[:, :N].double()
        err = (totals[:, :N].double() - want_tot).abs()
        assert bool((err <= tol_tot + 2 * U * want_tot.abs() + 1e-37).all()), float((err / tol_tot).max())
        assert torch.equal(totals[:, N:], before[:, N:])  # rows behind the last are left alone


SHAPES = [(14, 2, 64), (32, 8, 128), (4, 4, 32), (6, 1, 128), (3, 3, 64), (64, 1, 32)]


@pytest.mark.parametrize("H,kv,hd", SHAPES)
@pytest.mark.parametrize("n,T", [(0, 1), (1, 1), (31, 1), (32, 2), (0, 5), (255, 1), (257, 3), (1000, 7), (2500, 1)])
def test_chain(be, H, kv, hd, n, T):
    q, k, v = inputs(H, kv, hd, n, T, n + T + 3, 1 + n + T)
    out = run(be, q, k, v, H, n, T)
    check(out, q, k, v, H, n, T, np.tril(np.ones((T, T), bool)))


@pytest.mark.parametrize("H,kv,hd", SHAPES)
@pytest.mark.parametrize("n,T", [(0, 33), (40, 16), (63, 65), (700, 31), (3001, 64), (129, 128), (50, 200)])
def test_tree(be, H, kv, hd, n, T):
    rng = np.random.default_rng(T)
    seen = tree_bits(random_parents(T, rng))
    q, k, v = inputs(H, kv, hd, n, T, n + T, 7 + n + T, pad=64)
    w = torch.rand(kv, n + T, device="cuda")
    before = w.clone()
    out = run(be, q, k, v, H, n, T, mask=words_of(seen), weights=w)
    check(out, q, k, v, H, n, T, seen, w, before)


@pytest.mark.parametrize("H,kv,hd,n,T", [(32, 8, 128, 20011, 1), (32, 8, 128, 9000, 64), (14, 2, 64, 30000, 9),
                                         (8, 2, 32, 12345, 40), (12, 2, 128, 5000, 31), (16, 1, 128, 777, 1024)])
def test_long(be, H, kv, hd, n, T):
    q, k, v = inputs(H, kv, hd, n, T, n + T + 77, 3)
    w = torch.rand(kv, n + T + 77, device="cuda")
    before = w.clone()
    out = run(be, q, k, v, H, n, T, weights=w)
    check(out, q, k, v, H, n, T, np.tril(np.ones((T, T), bool)), w, before)


@pytest.mark.parametrize("n", [0, 5, 100])
@pytest.mark.parametrize("T", [3, 40, 130])
def test_arbitrary_masks_and_empty_rows(be, n, T):
    H, kv, hd = 8, 2, 64
    rng = np.random.default_rng(n + T)
    seen = rng.random((T, T)) < 0.3
    seen[0] = False
    seen[T - 1] = False
    mask = words_of(seen)
    if T % 32:  # bits at n_tokens and above are ignored
        mask[:, -1] |= torch.tensor(-1 << (T % 32), dtype=torch.int32, device="cuda")
    q, k, v = inputs(H, kv, hd, n, T, n + T, 11)
    w = torch.zeros(kv, n + T, device="cuda")
    out = run(be, q, k, v, H, n, T, mask=mask, weights=w)
    check(out, q, k, v, H, n, T, seen, w, torch.zeros_like(w))
    if n == 0:
        assert float(out[0].abs().max()) == 0.0 and float(out[T - 1].abs().max()) == 0.0


@pytest.mark.parametrize("T", [6, 70])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
def test_unseen_rows_may_hold_anything(be, T, bad):
    """Drafted row 2 and everything behind the last row hold NaN or infinities;
    only tokens that see row 2 may notice."""
    H, kv, hd, n = 8, 2, 128, 61
    seen = np.tril(np.ones((T, T), bool))
    seen[:, 2] = False
    seen[4, 2] = True
    q, k, v = inputs(H, kv, hd, n, T, n + T + 40, 5)
    kb, vb = k.clone(), v.clone()
    for x in (kb, vb):
        x[:, n + 2] = bad
        x[:, n + T:] = bad
    w = torch.zeros(kv, n + T + 40, device="cuda")
    out = run(be, q, kb, vb, H, n, T, mask=words_of(seen), weights=None)
    ok = [t for t in range(T) if t != 4]
    assert bool(torch.isfinite(out[ok]).all())
    assert not bool(torch.isfinite(out[4]).all())
    # the others answer as if the row were not there
    seen[4, 2] = False
    k[:, n + 2] = 0
    v[:, n + 2] = 0
    ref = run(be, q, k, v, H, n, T, mask=words_of(seen))
    check(ref, q, k, v, H, n, T, seen)
    out[4] = ref[4]
    check(out, q, k, v, H, n, T, seen)
    # q of one token: the others do not notice either
    q[1] = bad
    out = run(be, q, k, v, H, n, T, mask=words_of(seen), weights=w)
    assert torch.equal(out[[t for t in range(T) if t != 1]], ref[[t for t in range(T) if t != 1]])


@pytest.mark.parametrize("T", [1, 40])
@pytest.mark.parametrize("ks,vs", [(1e-12, 1e12), (1e10, 1e-20), (1e-30, 1e30), (0.0, 1.0), (1.0, 0.0)])
def test_magnitudes(be, T, ks, vs):
    """Scores near zero or spread over thousands, values of any size."""
    H, kv, hd, n = 8, 2, 128, 300
    q, k, v = inputs(H, kv, hd, n, T, n + T, 9, q_scale=1e-8 if ks == 1e10 else 1.0)
    k *= ks
    v *= vs
    out = run(be, q, k, v, H, n, T)
    check(out, q, k, v, H, n, T, np.tril(np.ones((T, T), bool)))


def test_one_large_row(be):
    """One row's key and value are a million times the others'."""
    H, kv, hd, n, T = 8, 2, 128, 500, 32
    q, k, v = inputs(H, kv, hd, n, T, n + T, 21)
    k[:, 77] *= 1e-3
    v[:, 77] *= 1e6
    out = run(be, q, k, v, H, n, T)
    check(out, q, k, v, H, n, T, np.tril(np.ones((T, T), bool)))


@pytest.mark.parametrize("n,T", [(4000, 1), (4000, 32)])
def test_same_bits_again_and_from_a_graph(be, n, T):
    """A replayed graph and a second call give the first call's bits; the
    workspace's contents do not matter; another stream's does its own work."""
    H, kv, hd = 32, 8, 128
    q, k, v = inputs(H, kv, hd, n, T, n + T, 4)
    w0, w1, w2 = (torch.zeros(kv, n + T, device="cuda") for _ in range(3))
    first = run(be, q, k, v, H, n, T, weights=w0)
    again = run(be, q, k, v, H, n, T, weights=w1)
    assert torch.equal(first, again) and torch.equal(w0, w1)
    need = be.attention_tree_workspace(H, kv, hd, n, T, True)
    work = torch.empty(need, dtype=torch.uint8, device="cuda")
    out = torch.zeros_like(first)
    s = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=s):
        be.attention_tree(q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), H, kv, hd, n + T, n, T,
                          work.data_ptr(), need, weights=w2.data_ptr(), stream=s.cuda_stream)
    for i in range(3):
        work.fill_(0xFF - i)
        out.zero_()
        w2.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, first) and torch.equal(w2, w0)


def test_strided_output_leaves_the_gaps(be):
    H, kv, hd, n, T = 6, 2, 64, 90, 5
    q, k, v = inputs(H, kv, hd, n, T, n + T, 2, pad=128)
    out = torch.full((T, H * hd + 32), 7.0, device="cuda")
    run(be, q, k, v, H, n, T, out=out)
    check(out[:, :H * hd], q, k, v, H, n, T, np.tril(np.ones((T, T), bool)))
    assert float((out[:, H * hd:] - 7.0).abs().max()) == 0.0


def test_large_offsets(be):
    """A cache whose last rows lie beyond 2^31 elements."""
    H, kv, hd, n, T = 2, 2, 128, 8_600_000, 2
    k = torch.zeros(kv, n + T, hd, device="cuda")
    v = torch.zeros(kv, n + T, hd, device="cuda")
    g = torch.Generator(device="cuda").manual_seed(1)
    tail = 500
    k[:, -tail:] = torch.randn(kv, tail, hd, device="cuda", generator=g)
    v[:, -tail:] = torch.randn(kv, tail, hd, device="cuda", generator=g)
    # keys far below the tail score -1e4 and vanish
    q = torch.randn(T, H * hd, device="cuda", generator=g)
    q[:, 0::hd] = 120.0
    k[:, :-tail, 0] = -1000.0
    out = run(be, q, k, v, H, n, T)
    start = n + T - tail
    check(out, q, k[:, start:].contiguous(), v[:, start:].contiguous(), H, tail - T, T, np.tril(np.ones((T, T), bool)))


def test_refusals(be):
    H, kv, hd, n, T = 8, 2, 64, 100, 4
    q, k, v = inputs(H, kv, hd, n, T, 128, 2)
    out = torch.full((T, H * hd), 3.0, device="cuda")
    need = be.attention_tree_workspace(H, kv, hd, n, T)
    work = torch.empty(max(need, 16) + 16, dtype=torch.uint8, device="cuda")
    L = _lib.lib()
    P = dict(q=q.data_ptr(), qs=H * hd, k=k.data_ptr(), v=v.data_ptr(), H=H, kv=kv, hd=hd, max_ctx=128, n=n, T=T,
             mask=None, out=out.data_ptr(), os=H * hd, w=None, work=work.data_ptr(), nb=work.numel())

    def rc(**kw):
        a = {**P, **kw}
        return L.smallm_attention_tree(be.h, a["q"], a["qs"], a["k"], a["v"], a["H"], a["kv"], a["hd"], a["max_ctx"],
                                       a["n"], a["T"], a["mask"], a["out"], a["os"], a["w"], a["work"], a["nb"], None)

    torch.cuda.synchronize()
    for kw in (dict(q=None), dict(k=None), dict(v=None), dict(out=None), dict(H=7), dict(H=0), dict(kv=0),
               dict(hd=96), dict(hd=0), dict(qs=H * hd - 4), dict(qs=H * hd + 1), dict(os=H * hd - 4),
               dict(os=H * hd + 2), dict(q=P["q"] + 4), dict(k=P["k"] + 8), dict(v=P["v"] + 4),
               dict(out=P["out"] + 4), dict(mask=P["q"] + 2), dict(w=P["q"] + 1)):
        assert rc(**kw) == _lib.ERR_INVALID, kw
    for kw in (dict(n=125), dict(max_ctx=103), dict(n=2**32 - 2), dict(T=1025, n=0, max_ctx=4096),
               dict(H=65 * 2, qs=130 * hd, os=130 * hd)):
        assert rc(**kw) == _lib.ERR_RANGE, kw
    w = torch.zeros(kv, 128, device="cuda")
    need_w = be.attention_tree_workspace(H, kv, hd, n, T, True)
    assert need_w > need
    assert rc(w=w.data_ptr(), nb=need_w - 1) == _lib.ERR_INVALID
    assert b"workspace" in L.smallm_last_error()
    assert rc(w=w.data_ptr(), work=None, nb=need_w) == _lib.ERR_INVALID
    assert rc(w=w.data_ptr(), work=P["work"] + 4, nb=need_w) == _lib.ERR_INVALID
    torch.cuda.synchronize()
    assert float((out - 3.0).abs().max()) == 0.0 and float(w.abs().max()) == 0.0  # nothing was launched
    assert rc(T=0, q=None) == _lib.OK
    with pytest.raises(SmallmError):
        be.attention_tree_workspace(7, 2, 64, 0, 1)
