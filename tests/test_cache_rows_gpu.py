"""Keeping a KV cache within its budget: smallm_cache_select and
smallm_cache_move against numpy.  Both are exact: selections and moved rows
are compared for equality."""
import numpy as np
import pytest
import torch

from smallm_engine_b200 import _lib

pytestmark = pytest.mark.gpu


def select_reference(w, n, keep, first, last):
    """Stable order by total, largest first, NaN last; then ascending rows."""
    out = []
    for head in w:
        mid = head[first:n - last].astype(np.float64)
        mid = np.where(np.isnan(mid), -np.inf, mid)
        nan = np.isnan(head[first:n - last])
        order = np.lexsort((np.arange(mid.size), -mid, nan))
        best = np.sort(order[:keep - first - last]) + first
        out.append(np.concatenate([np.arange(first), best, np.arange(n - last, n)]))
    return np.array(out, np.int64)


def select(be, w, n, keep, first, last, stream=None):
    kv, max_ctx = w.shape
    rows = torch.full((kv, max(keep, 1)), -1, dtype=torch.int32, device="cuda")
    torch.cuda.synchronize()
    be.cache_select(w.data_ptr(), kv, max_ctx, n, keep, first, last, rows.data_ptr(), stream=stream)
    torch.cuda.synchronize()
    return rows


@pytest.mark.parametrize("kv,n,keep,first,last", [
    (1, 1, 1, 0, 0), (2, 5, 3, 1, 1), (2, 40, 40, 0, 0), (3, 1000, 1, 0, 0), (2, 1021, 512, 4, 32),
    (8, 4096, 4095, 0, 0), (4, 5000, 300, 16, 284), (2, 70000, 33333, 7, 13), (8, 131072, 65536, 16, 256),
    (1, 300001, 150000, 3, 0), (130, 500, 77, 5, 5), (3, 2048, 2000, 2000, 0), (3, 2049, 1025, 0, 1025),
    (1, 400001, 200000, 5, 9), (150, 30001, 12345, 1, 2)])  # the last two: keys that do not fit shared memory
@pytest.mark.parametrize("kind", ["lognormal", "ties", "equal", "special"])
def test_select(be, kv, n, keep, first, last, kind):
    rng = np.random.default_rng(n + keep)
    w = np.exp(2 * rng.standard_normal((kv, n + 3))).astype(np.float32)
    if kind == "ties":
        w = np.floor(rng.random((kv, n + 3)) * 7).astype(np.float32)
    elif kind == "equal":
        w[:] = 0.5
    elif kind == "special":
        w[rng.random(w.shape) < 0.2] = np.nan
        w[rng.random(w.shape) < 0.1] = np.inf
        w[rng.random(w.shape) < 0.1] = -np.inf
        w[rng.random(w.shape) < 0.2] = 0.0
        w[rng.random(w.shape) < 0.2] = -0.0
        w[rng.random(w.shape) < 0.1] *= -1
        w[rng.random(w.shape) < 0.1] = 1e-42
    rows = select(be, torch.from_numpy(w).cuda(), n, keep, first, last)
    np.testing.assert_array_equal(rows.cpu().numpy(), select_reference(w, n, keep, first, last))


def move_reference(x, rows, dst):
    y = x.copy()
    for g in range(x.shape[0]):
        r = rows[g if rows.shape[0] > 1 else 0]
        y[g, dst:dst + r.size] = x[g, r]
    return y


def lists(rng, heads, span, c, dst):
    return np.stack([np.sort(rng.choice(span, c, replace=False)) + dst for _ in range(heads)]).astype(np.int64)


@pytest.mark.parametrize("kv,hd,span,c,dst,per_head", [
    (2, 64, 1, 1, 0, False), (2, 64, 10, 1, 5, False), (8, 128, 64, 6, 4001, False), (3, 32, 300, 299, 17, True),
    (8, 128, 5000, 2500, 0, True), (1, 64, 20000, 19000, 3, True), (2, 128, 4096, 4096, 0, False),
    (16, 32, 3000, 1025, 1, True), (70, 64, 500, 250, 2, True), (8, 128, 32768, 16384, 0, True)])
@pytest.mark.parametrize("with_weights", [False, True])
def test_move(be, kv, hd, span, c, dst, per_head, with_weights):
    rng = np.random.default_rng(span + c)
    max_ctx = dst + span + 5
    k = rng.standard_normal((kv, max_ctx, hd), dtype=np.float32)
    v = rng.standard_normal((kv, max_ctx, hd), dtype=np.float32)
    w = rng.random((kv, max_ctx), dtype=np.float32)
    k[0, 0, 0], v[0, -1, 0] = np.nan, np.inf  # rows are moved, not computed with
    rows = lists(rng, kv if per_head else 1, span, c, dst)
    kd, vd, wd = (torch.from_numpy(x).cuda() for x in (k, v, w))
    rd = torch.from_numpy(rows.astype(np.int32)).cuda()
    torch.cuda.synchronize()
    be.device_errors()
    be.cache_move(kd.data_ptr(), vd.data_ptr(), kv, hd, max_ctx, rd.data_ptr(), c, dst, per_head=per_head,
                  weights=wd.data_ptr() if with_weights else None)
    assert be.device_errors() == 0
    np.testing.assert_array_equal(kd.cpu().numpy(), move_reference(k, rows, dst))
    np.testing.assert_array_equal(vd.cpu().numpy(), move_reference(v, rows, dst))
    np.testing.assert_array_equal(wd.cpu().numpy(), move_reference(w, rows, dst) if with_weights else w)


@pytest.mark.parametrize("entry,value", [(0, 2), (5, 9), (5, 15), (6, 21), (7, 64), (7, 2**32 - 1), (3, 2**31)])
def test_bad_lists_raise_the_error_bit(be, entry, value):
    """A list that is not ascending, reaches below its destination or past the
    cache: reported, and nothing before the destination or behind the largest
    row that a list may name is touched."""
    kv, hd, max_ctx, dst = 2, 64, 64, 8
    rows = np.array([9, 10, 13, 14, 16, 17, 22, 30], np.int64)
    rows[entry] = value
    k = torch.randn(kv + 2, max_ctx, hd, device="cuda")
    v = torch.randn(kv + 2, max_ctx, hd, device="cuda")
    kb, vb = k.clone(), v.clone()
    rd = torch.from_numpy(rows.astype(np.uint32).view(np.int32).copy()).cuda()
    torch.cuda.synchronize()
    be.device_errors()
    be.cache_move(k[1].data_ptr(), v[1].data_ptr(), kv, hd, max_ctx, rd.data_ptr(), 8, dst)
    # entry 5 = 15 breaks the order but not the bound, entry 6 = 21 is legal
    assert be.device_errors() == (0 if (entry, value) == (6, 21) else 128)
    for x, b in ((k, kb), (v, vb)):
        assert torch.equal(x[0], b[0]) and torch.equal(x[-1], b[-1])
        assert torch.equal(x[1:-1, :dst], b[1:-1, :dst]) and torch.equal(x[1:-1, dst + 8:], b[1:-1, dst + 8:])


def test_select_then_move_from_a_graph(be):
    """The two calls of an eviction captured together and replayed on fresh data."""
    kv, hd, max_ctx, n, keep, first, last = 4, 64, 3000, 2900, 1000, 4, 64
    k, v, w = (torch.empty(s, device="cuda") for s in ((kv, max_ctx, hd), (kv, max_ctx, hd), (kv, max_ctx)))
    rows = torch.empty(kv, keep, dtype=torch.int32, device="cuda")
    s = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    be.device_errors()
    with torch.cuda.graph(graph, stream=s):
        be.cache_select(w.data_ptr(), kv, max_ctx, n, keep, first, last, rows.data_ptr(), stream=s.cuda_stream)
        be.cache_move(k.data_ptr(), v.data_ptr(), kv, hd, max_ctx, rows.data_ptr(), keep, 0, per_head=True,
                      weights=w.data_ptr(), stream=s.cuda_stream)
    for seed in range(3):
        rng = np.random.default_rng(seed)
        kn, vn = (rng.standard_normal((kv, max_ctx, hd), dtype=np.float32) for _ in range(2))
        wn = rng.random((kv, max_ctx), dtype=np.float32)
        for d, h in ((k, kn), (v, vn), (w, wn)):
            d.copy_(torch.from_numpy(h))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        want = select_reference(wn, n, keep, first, last)
        np.testing.assert_array_equal(rows.cpu().numpy(), want)
        for d, h in ((k, kn), (v, vn), (w, wn)):
            np.testing.assert_array_equal(d.cpu().numpy(), move_reference(h, want, 0))
    assert be.device_errors() == 0


def test_refusals(be):
    L = _lib.lib()
    x = torch.zeros(2, 64, 32, device="cuda")
    w = torch.zeros(2, 64, device="cuda")
    r = torch.zeros(2, 64, dtype=torch.int32, device="cuda")
    p, wp, rp = x.data_ptr(), w.data_ptr(), r.data_ptr()
    sel = lambda *a: L.smallm_cache_select(be.h, *a, None)  # noqa: E731
    assert sel(None, 2, 64, 64, 8, 0, 0, rp) == _lib.ERR_INVALID
    assert sel(wp, 2, 64, 64, 8, 0, 0, None) == _lib.ERR_INVALID
    assert sel(wp, 2, 64, 65, 8, 0, 0, rp) == _lib.ERR_RANGE
    assert sel(wp, 2, 64, 64, 65, 0, 0, rp) == _lib.ERR_INVALID
    assert sel(wp, 2, 64, 64, 8, 5, 4, rp) == _lib.ERR_INVALID
    assert sel(wp, 2, 64, 64, 8, 2**32 - 1, 2, rp) == _lib.ERR_INVALID
    assert sel(wp, 2, 2**31, 2**30 + 1, 8, 0, 0, rp) == _lib.ERR_RANGE
    assert sel(wp, 65536, 64, 64, 8, 0, 0, rp) == _lib.ERR_RANGE
    assert sel(wp + 2, 2, 64, 64, 8, 0, 0, rp) == _lib.ERR_INVALID
    assert sel(wp, 2, 64, 64, 8, 0, 0, rp + 1) == _lib.ERR_INVALID
    assert sel(wp, 0, 64, 64, 8, 0, 0, rp) == _lib.OK
    assert sel(wp, 2, 64, 64, 0, 0, 0, rp) == _lib.OK
    mv = lambda *a: L.smallm_cache_move(be.h, *a, None)  # noqa: E731
    assert mv(None, p, None, 2, 32, 64, rp, 0, 4, 0) == _lib.ERR_INVALID
    assert mv(p, None, None, 2, 32, 64, rp, 0, 4, 0) == _lib.ERR_INVALID
    assert mv(p, p, None, 2, 32, 64, None, 0, 4, 0) == _lib.ERR_INVALID
    assert mv(p, p, None, 2, 48, 64, rp, 0, 4, 0) == _lib.ERR_INVALID
    assert mv(p + 4, p, None, 2, 32, 64, rp, 0, 4, 0) == _lib.ERR_INVALID
    assert mv(p, p, None, 2, 32, 64, rp, 0, 4, 61) == _lib.ERR_RANGE
    assert mv(p, p, None, 2, 32, 64, rp, 0, 4, 2**32 - 2) == _lib.ERR_RANGE
    assert mv(p, p, None, 2, 32, 2**31, rp, 0, 2**30 + 1, 0) == _lib.ERR_RANGE
    assert mv(p, p, None, 65536, 32, 64, rp, 0, 4, 0) == _lib.ERR_RANGE
    assert mv(p, p, wp + 2, 2, 32, 64, rp, 0, 4, 0) == _lib.ERR_INVALID
    assert mv(p, p, None, 2, 32, 64, rp + 2, 0, 4, 0) == _lib.ERR_INVALID
    assert mv(p, p, None, 2, 32, 64, rp, 0, 0, 0) == _lib.OK
    torch.cuda.synchronize()
    assert float(x.abs().max()) == 0.0 and int(r.abs().max()) == 0
