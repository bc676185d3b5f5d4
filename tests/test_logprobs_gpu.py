"""Log probabilities, entropy and top alternatives (smallm_logprobs) against
their definition in 64 bits.

Tolerance, u = 2^-24.  x - m is one rounding of a value of at most R, R the
row's range above the point where e^(x-m) no longer counts (at most 104 in
f32); e^. adds 2 units, the sum of V positive terms in chunks at most V u but,
with every thread's chain at most 256 long and the joins 20 deep, 300 u here:
    |log p - exact| <= (|x - m| + |lse - m| + 2 * 104 + 300 + 8) u
    |H - exact|     <= (2 * 104 + 300 + 8) u (1 + |H|) * 2
(the entropy divides a sum of e^d d by a sum of e^d: both errors, each
relative to a quantity of at most 1 + H).
Ids are exact: order by value, equal values by id."""
import numpy as np
import pytest
import torch

from smallm_engine_b200 import _lib

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


def run(be, x, tokens, top, stride=None, stream=None):
    rows, V = x.shape
    lp = torch.full((rows,), 5.0, device="cuda")
    ent = torch.full((rows,), 5.0, device="cuda")
    ids = torch.full((rows, max(top, 1)), -1, dtype=torch.int32, device="cuda")
    tlp = torch.full((rows, max(top, 1)), 5.0, device="cuda")
    torch.cuda.synchronize()
    be.logprobs(x.data_ptr(), rows, V, tokens.data_ptr(), lp.data_ptr(), ent.data_ptr(), top, ids.data_ptr(),
                tlp.data_ptr(), stride=x.stride(0) if stride is None else stride, stream=stream)
    torch.cuda.synchronize()
    return lp, ent, ids[:, :top], tlp[:, :top]


def check(got, x, tokens, top):
    lp, ent, ids, tlp = got
    xd = x.double()
    m = xd.amax(1, keepdim=True)
    d = xd - m  # around the maximum: beside 3e38 even 64 bits lose the logarithm of the sum
    ls = torch.log(torch.exp(d).sum(1, keepdim=True))
    want = d - ls
    p = torch.exp(want)
    H = -torch.where(p > 0, p * want, 0.0).sum(1)
    tol = lambda v: ((v - m).abs() + ls.abs() + 516) * U  # noqa: E731
    t = tokens.long()[:, None]

    def near(a, b, bound):
        same = (a == b) | ((a - b).abs() <= bound)
        assert bool(same.all()), float(((a - b).abs() / bound).nan_to_num().max())
    near(lp.double()[:, None], want.gather(1, t), tol(xd.gather(1, t)))
    near(ent.double(), H, 2 * 516 * U * (1 + H))
    order = torch.sort(x + 0.0, dim=1, descending=True, stable=True).indices[:, :top]
    assert torch.equal(ids.long(), order)
    near(tlp.double(), want.gather(1, order), tol(xd.gather(1, order)))


@pytest.mark.parametrize("rows,V,top", [(1, 1, 1), (3, 2, 2), (1, 31, 5), (2, 1000, 64), (1, 32000, 1), (5, 50257, 20),
                                        (1, 128256, 20), (9, 151936, 5), (300, 151936, 0), (700, 4099, 33),
                                        (2, 600001, 64), (148, 65, 64), (33, 16385, 7)])
@pytest.mark.parametrize("kind", ["normal", "peaked", "ties", "masked", "sorted"])
def test_logprobs(be, rows, V, top, kind):
    g = torch.Generator(device="cuda").manual_seed(V + rows)
    x = 2.5 * torch.randn(rows, V + 5, device="cuda", generator=g)
    if kind == "peaked":
        x[:, V // 2] += 40.0
    elif kind == "ties":
        x = torch.round(x)
        x[0] = 0.25
    elif kind == "masked":  # a grammar leaves few tokens; one row leaves one
        x[torch.rand(x.shape, device="cuda", generator=g) < 0.97] = -torch.inf
        x[:, V // 3] = -3.0
        x[0, :V] = -torch.inf
        x[0, V - 1] = 17.0
    elif kind == "sorted":  # every alternative in one thread's reach
        x = torch.sort(x, dim=1, descending=rows % 2 == 0).values.contiguous()
    x = x[:, :V]
    tokens = torch.randint(0, V, (rows,), device="cuda", generator=g).to(torch.int32)
    check(run(be, x, tokens, top), x, tokens, top)


@pytest.mark.parametrize("V", [40, 70001])
def test_offsets_and_extremes(be, V):
    """Logits far from zero, -0 beside +0, the type's lowest value."""
    x = torch.randn(6, V, device="cuda")
    x[0] += 1e4
    x[1] -= 1e6
    x[2, :] = torch.finfo(torch.float32).min
    x[3, :] = torch.finfo(torch.float32).min
    x[3, 7] = 1.0
    x[4, 1::2], x[4, ::2] = 0.0, -0.0
    x[5] *= 1e-30
    tokens = torch.tensor([3, 4, 5, 7, 6, V - 1], dtype=torch.int32, device="cuda")
    check(run(be, x, tokens, 6), x, tokens, 6)


@pytest.mark.parametrize("V", [17, 128256])
def test_rows_without_a_distribution(be, V):
    x = torch.randn(6, V, device="cuda")
    x[0, 3] = torch.nan
    x[1, 4] = torch.inf
    x[2, :] = -torch.inf
    x[3, :] = torch.nan
    x[4, 5], x[4, 6] = torch.inf, torch.nan
    tokens = torch.tensor([0, 4, 2, 3, 5, V], dtype=torch.int32, device="cuda")
    lp, ent, ids, tlp = run(be, x, tokens, 8)
    for r in range(5):
        assert bool(torch.isnan(lp[r])) and bool(torch.isnan(ent[r])) and bool(torch.isnan(tlp[r]).all()), r
    assert bool(torch.isnan(lp[5])) and bool(torch.isfinite(ent[5]))  # a token outside the vocabulary
    key = torch.where(torch.isnan(x), -torch.inf, x)
    for r in (0, 1, 5):
        assert ids[r].tolist() == torch.sort(key[r], descending=True, stable=True).indices[:8].tolist()
    assert ids[2].tolist() == list(range(8)) and ids[3].tolist() == list(range(8))
    assert ids[4, 0] == 5


def test_optional_outputs_and_strides(be):
    x = torch.randn(4, 1003, device="cuda")[:, :1000]
    lp, ent = torch.zeros(4, device="cuda"), torch.zeros(4, device="cuda")
    tok = torch.arange(4, dtype=torch.int32, device="cuda")
    torch.cuda.synchronize()
    be.logprobs(x.data_ptr(), 4, 1000, tok.data_ptr(), lp.data_ptr(), None, 0, None, None, stride=1003)
    be.logprobs(x.data_ptr(), 4, 1000, None, None, ent.data_ptr(), 0, None, None, stride=1003)
    torch.cuda.synchronize()
    want = torch.log_softmax(x.double(), 1)
    assert bool(((lp.double() - want[range(4), range(4)]).abs() < 600 * U).all())
    assert bool(((ent.double() + (want.exp() * want).sum(1)).abs() < 9000 * U).all())
    # rows at any 4-byte alignment
    y = torch.randn(3 * 1000 + 1, device="cuda")[1:].view(3, 1000)
    tok = torch.tensor([1, 2, 3], dtype=torch.int32, device="cuda")
    check(run(be, y, tok, 10), y, tok, 10)


def test_same_bits_again_and_from_a_graph(be):
    x = torch.randn(3, 128256, device="cuda")
    tok = torch.tensor([1, 2, 3], dtype=torch.int32, device="cuda")
    first = run(be, x, tok, 20)
    again = run(be, x, tok, 20)
    assert all(torch.equal(a, b) for a, b in zip(first, again))
    outs = [torch.zeros_like(t) for t in first]
    s = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=s):
        be.logprobs(x.data_ptr(), 3, 128256, tok.data_ptr(), outs[0].data_ptr(), outs[1].data_ptr(), 20,
                    outs[2].data_ptr(), outs[3].data_ptr(), stream=s.cuda_stream)
    for _ in range(2):
        for t in outs:
            t.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(first, outs))


def test_refusals(be):
    L = _lib.lib()
    x = torch.zeros(2, 100, device="cuda")
    o = torch.zeros(2, 100, device="cuda")
    p, q = x.data_ptr(), o.data_ptr()
    f = lambda *a: L.smallm_logprobs(be.h, *a, None)  # noqa: E731
    assert f(None, 2, 100, 100, None, None, q, 0, None, None) == _lib.ERR_INVALID
    assert f(p, 2, 0, 100, None, None, q, 0, None, None) == _lib.ERR_INVALID
    assert f(p, 2, 100, 99, None, None, q, 0, None, None) == _lib.ERR_INVALID
    assert f(p, 2, 100, 100, p, None, q, 0, None, None) == _lib.ERR_INVALID
    assert f(p, 2, 100, 100, None, q, q, 0, None, None) == _lib.ERR_INVALID
    assert f(p, 2, 100, 100, None, None, q, 3, None, q) == _lib.ERR_INVALID
    assert f(p, 2, 100, 100, None, None, q, 3, q, None) == _lib.ERR_INVALID
    assert f(p, 2, 100, 100, None, None, q, 65, q, q) == _lib.ERR_RANGE
    assert f(p, 2, 10, 10, None, None, q, 11, q, q) == _lib.ERR_RANGE
    assert f(p, 2**26 + 1, 1, 1, None, None, q, 0, None, None) == _lib.ERR_RANGE
    assert f(p, 1, 2**30 + 1, 2**30 + 1, None, None, q, 0, None, None) == _lib.ERR_RANGE
    assert f(p + 2, 2, 10, 10, None, None, q, 0, None, None) == _lib.ERR_INVALID
    assert f(p, 2, 10, 10, p + 1, q, None, 0, None, None) == _lib.ERR_INVALID
    assert f(p, 2, 10, 10, p, q + 1, None, 0, None, None) == _lib.ERR_INVALID
    assert f(p, 2, 10, 10, None, None, q + 2, 0, None, None) == _lib.ERR_INVALID
    assert f(p, 2, 10, 10, None, None, q, 1, q + 3, q) == _lib.ERR_INVALID
    assert f(p, 2, 10, 10, None, None, q, 1, q, q + 3) == _lib.ERR_INVALID
    assert f(p, 0, 100, 100, None, None, q, 0, None, None) == _lib.OK
    torch.cuda.synchronize()
    assert float(o.abs().max()) == 0.0
