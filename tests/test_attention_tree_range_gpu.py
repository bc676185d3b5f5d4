"""Attention of drafted tokens where magnitudes differ widely: large finite rows
that a token does not see or gives no weight, scores beyond f32's range or too
large for a weight to be told from its neighbour's, sums of values beyond f32's
range, and totals of rows that a token whose result is not finite does not see.

Against the definition in 64 bits with the tolerance derived in
test_attention_tree_gpu.py, unless a test says otherwise.  That tolerance also
covers how rows enter: an element is off by at most 2^-22 of itself or 2^-25 of
its row's largest magnitude, and a weight's product with its row by 2^-24 of
the token's largest such product among 64 keys."""
import numpy as np
import pytest
import torch

from test_attention_tree_gpu import U, check, inputs, run, words_of

pytestmark = pytest.mark.gpu

BIG = [1e6, 1e9, 1e12, 1e20, 3e38]


def chain(T):
    return np.tril(np.ones((T, T), bool))


def unit_rows(shape, seed):
    """Values in (-1, 1), so that a multiple up to f32's largest stays finite."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    return 2 * torch.rand(shape, device="cuda", generator=g) - 1


@pytest.mark.parametrize("H,kv,hd", [(8, 2, 128), (6, 3, 64), (4, 1, 32)])
@pytest.mark.parametrize("T", [6, 70])
@pytest.mark.parametrize("which", ["k", "v", "kv"])
@pytest.mark.parametrize("f", BIG)
def test_large_unseen_row(be, H, kv, hd, T, which, f):
    """A drafted row that only one token sees holds large finite values, as an
    unwritten slot may: the other tokens answer as if it were not there."""
    n = 61
    seen = chain(T)
    seen[:, 2] = False
    seen[4, 2] = True
    q, k, v = inputs(H, kv, hd, n, T, n + T, 5)
    for x, name in ((k, "k"), (v, "v")):
        if name in which:
            x[:, n + 2] = f * unit_rows((kv, hd), 3)
    w = torch.zeros(kv, n + T, device="cuda")
    out = run(be, q, k, v, H, n, T, mask=words_of(seen))
    seen[4, 2] = False
    k[:, n + 2] = 0
    v[:, n + 2] = 0
    ref = run(be, q, k, v, H, n, T, mask=words_of(seen), weights=w)
    check(ref, q, k, v, H, n, T, seen, w, torch.zeros_like(w))
    out[4] = ref[4]
    check(out, q, k, v, H, n, T, seen)


@pytest.mark.parametrize("T", [1, 33])
@pytest.mark.parametrize("f", BIG)
@pytest.mark.parametrize("drop", [0.0, 1e-13, 1e-25, 0.03])
def test_large_value_of_small_weight(be, T, f, drop):
    """A seen row whose V is large: what its weight makes of it is the result,
    and where that is nothing the other rows are.  Its key takes the score down
    (or, at `drop` 0, far below what f32 can weigh)."""
    H, kv, hd, n = 8, 2, 128, 300
    q, k, v = inputs(H, kv, hd, n, T, n + T, 13)
    q[:, 0::hd] = 8.0
    k[:, :, 0] = 0.0
    down = 1000.0 if drop == 0.0 else -np.log(drop)
    k[:, 77, 0] = -down * hd ** 0.5 / 8.0
    v[:, 77] = f * unit_rows((kv, hd), 2)
    w = torch.zeros(kv, n + T, device="cuda")
    out = run(be, q, k, v, H, n, T, weights=w)
    check(out, q, k, v, H, n, T, chain(T), w, torch.zeros_like(w))


@pytest.mark.parametrize("T", [1, 33])
@pytest.mark.parametrize("n", [190, 5000])
@pytest.mark.parametrize("f,drop", [(1e12, 1e-9), (1e20, 1e-15), (1e30, 1e-25)])
def test_tile_of_large_values_with_small_weights(be, T, n, f, drop):
    """64 neighbouring rows are all large and have small weights."""
    H, kv, hd = 8, 2, 64
    q, k, v = inputs(H, kv, hd, n, T, n + T, 17)
    q[:, 0::hd] = 8.0
    k[:, :, 0] = 0.0
    k[:, 64:128, 0] = np.log(drop) * hd ** 0.5 / 8.0
    v[:, 64:128] *= f
    out = run(be, q, k, v, H, n, T)
    check(out, q, k, v, H, n, T, chain(T))


@pytest.mark.parametrize("T", [1, 33])
@pytest.mark.parametrize("f", BIG[1:])
def test_large_key_far_below(be, T, f):
    """A seen row with a large key that every token scores far below the others
    (beyond f32's range for the largest) has no weight and changes nothing."""
    H, kv, hd, n = 8, 2, 128, 300
    q, k, v = inputs(H, kv, hd, n, T, n + T, 19)
    q[:, 0::hd] = 8.0
    k[:, 77] = 0.0
    k[:, 77, 0] = -f
    w = torch.zeros(kv, n + T, device="cuda")
    out = run(be, q, k, v, H, n, T, weights=w)
    assert float(w[:, 77].abs().max()) == 0.0
    rows = [r for r in range(n + T) if r != 77]
    check(out, q, k[:, rows], v[:, rows], H, n - 1, T, chain(T), w[:, rows], torch.zeros_like(w[:, rows]))


@pytest.mark.parametrize("T", [1, 33])
def test_rows_of_every_size(be, T):
    """Every row of K and V has a size of its own, over fifty powers of ten; the
    scores stay ordinary, since q is small where K is large."""
    H, kv, hd, n = 8, 2, 64, 500
    q, k, v = inputs(H, kv, hd, n, T, n + T, 23)
    g = torch.Generator(device="cuda").manual_seed(4)
    k *= torch.pow(10.0, -30.0 * torch.rand(kv, n + T, 1, device="cuda", generator=g))
    v *= torch.pow(10.0, 50.0 * torch.rand(kv, n + T, 1, device="cuda", generator=g) - 25.0)
    w = torch.zeros(kv, n + T, device="cuda")
    out = run(be, q, k, v, H, n, T, weights=w)
    check(out, q, k, v, H, n, T, chain(T), w, torch.zeros_like(w))


@pytest.mark.parametrize("T", [1, 33])
def test_scales_beyond_f32_with_scores_of_zero(be, T):
    """q and K of 1e30, orthogonal: every score is 0, the output V's mean."""
    H, kv, hd, n = 8, 2, 64, 100
    q, k, v = inputs(H, kv, hd, n, T, n + T, 29)
    q.zero_()
    q[:, 0::hd] = 1e30
    k[:, :, 0] = 0.0
    k *= 1e30
    out = run(be, q, k, v, H, n, T)
    check(out, torch.zeros_like(q), torch.zeros_like(k), v, H, n, T, chain(T))


# ------------------------------------------------------------ large scores --

@pytest.mark.parametrize("n,T", [(20, 2), (100, 2), (300, 30), (4000, 2), (4000, 30)])
@pytest.mark.parametrize("where", ["first", "middle", "last"])
def test_a_score_above_f32s_range_is_not_a_zero(be, n, T, where):
    """One seen row scores beyond f32's largest value for token 0 alone: its
    output is not finite.  (For the others that row's other elements lie more
    than 2^-25 below its largest, so their scores of it are not known.)"""
    H, kv, hd = 8, 2, 64
    q, k, v = inputs(H, kv, hd, n, T, n + T, 31)
    at = {"first": 0, "middle": n // 2, "last": n - 1}[where]
    q[:, 0::hd] = 0.0
    k[:, :, 0] = 0.0
    k[:, at, 0] = 1e20
    q[0, 0::hd] = 1e20
    w = torch.zeros(kv, n + T, device="cuda")
    out = run(be, q, k, v, H, n, T, weights=w)
    assert not bool(torch.isfinite(out[0]).any()) and bool(torch.isfinite(out[1:]).all())
    assert not bool(torch.isfinite(w[:, :n + 1]).any())


@pytest.mark.parametrize("n,T", [(20, 2), (300, 30), (4000, 2), (4000, 30)])
def test_a_score_above_f32s_range_of_a_row_of_ones_own(be, n, T):
    """The same of a drafted row that token 0 alone sees: the others are right."""
    H, kv, hd = 8, 2, 64
    seen = np.eye(T, dtype=bool)
    q, k, v = inputs(H, kv, hd, n, T, n + T, 31)
    q[0, 0::hd] = 1e20
    k[:, :, 0] = 0.0
    k[:, n, 0] = 1e20
    out = run(be, q, k, v, H, n, T, mask=words_of(seen))
    assert not bool(torch.isfinite(out[0]).any())
    q[0, 0::hd] = 0.0
    k[:, n, 0] = 0.0
    ref = run(be, q, k, v, H, n, T, mask=words_of(seen))
    check(ref, q, k, v, H, n, T, seen)
    out[0] = ref[0]
    check(out, q, k, v, H, n, T, seen)


@pytest.mark.parametrize("n", [3, 100, 4000])
def test_all_scores_below_f32s_range_are_not_an_empty_row(be, n):
    """Not finite, as the header says, rather than the zeros of a token that
    sees nothing."""
    H, kv, hd, T = 8, 2, 64, 1
    q, k, v = inputs(H, kv, hd, n, T, n + T, 37)
    q[:, 0::hd] = 1e20
    k[:, :, 0] = -1e20
    out = run(be, q, k, v, H, n, T)
    assert not bool(torch.isfinite(out).any())


@pytest.mark.parametrize("e", range(10, 16))
@pytest.mark.parametrize("n,T", [(60, 1), (700, 1), (700, 33)])
@pytest.mark.parametrize("winners", [1, 2])
def test_large_scores(be, e, n, T, winners):
    """Scores up to 2^27 whose gaps (2^13 at least) are far above their error
    (2^-22 of them, 2^5): the largest takes everything, two equal ones half
    each, and the output is one row or the mean of two: V's and the weights'
    2^-22 each, and 8 u for two sums, the reciprocal and the products."""
    H, kv, hd = 4, 2, 64
    for shift in range(3):
        q, k, v = inputs(H, kv, hd, n, T, n + T, 41 + shift)
        q.zero_()
        q[:, 0::hd] = 2.0 ** e + shift
        k.zero_()
        k[:, :, 0] = 2.0 ** e - 64 - (torch.arange(n + T, device="cuda") % 53)
        best = [5, n - 3][:winners]
        k[:, best, 0] = 2.0 ** e + 3 * shift
        w = torch.zeros(kv, n + T, device="cuda")
        out = run(be, q, k, v, H, n, T, weights=w)
        want = v[:, best].double().mean(1).repeat_interleave(H // kv, 0).reshape(1, H * hd)
        tol = (4 * U + 4 * U + 8 * U) * v[:, best].abs().amax().double()
        assert bool(((out.double() - want).abs() <= tol).all()), float((out.double() - want).abs().max())
        total = torch.zeros_like(w)
        total[:, best] = T * (H // kv) / winners
        assert bool(((w - total).abs() <= 4 * T * H * U * total).all())


# ------------------------------------------------------------ large values --

@pytest.mark.parametrize("n,T", [(60, 1), (4000, 1), (4000, 33), (20000, 2)])
@pytest.mark.parametrize("f", [1e36, 3.3e38])
def test_mean_of_values_whose_sum_passes_f32(be, n, T, f):
    """Equal scores: a mean of V near f32's largest value is finite."""
    H, kv, hd = 8, 2, 64
    q, k, v = inputs(H, kv, hd, n, T, n + T, 43)
    k.zero_()
    v = f * (0.5 + 0.5 * unit_rows(v.shape, 6).abs())
    out = run(be, q, k, v, H, n, T)
    assert bool(torch.isfinite(out).all())
    check(out, q, k, v, H, n, T, chain(T))


@pytest.mark.parametrize("n,T", [(60, 1), (4000, 1), (4000, 33), (20000, 2)])
@pytest.mark.parametrize("f", [1e-34, 1e-30, 1e-26])
def test_tiny_values_keep_their_bits(be, n, T, f):
    """The same bound without its absolute part: the result's scale is f, each
    element of it within (2 n + 64) u of the mean of |V|, and the last rounding
    within half of f32's smallest step."""
    H, kv, hd = 8, 2, 64
    q, k, v = inputs(H, kv, hd, n, T, n + T, 47)
    k.zero_()
    v = f * (0.5 + 0.5 * unit_rows(v.shape, 6).abs())
    out = run(be, q, k, v, H, n, T).view(T, kv, H // kv, hd).double()
    for t in range(T):
        mean = v[:, :n + t + 1].double().mean(1)
        # (every partial sum is rounded to f32's smallest step at most n times)
        tol = (2 * (n + T) + 64) * U * mean + (n + T) * 2.0 ** -149
        assert bool(((out[t] - mean[:, None]).abs() <= tol[:, None]).all()), float(((out[t] - mean[:, None]).abs() / tol[:, None]).max())


# ------------------------------------------------------------------ totals --

@pytest.mark.parametrize("T", [3, 6, 70])
@pytest.mark.parametrize("n", [40, 3000])
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_totals_of_rows_that_a_spoiled_token_does_not_see(be, T, n, bad):
    """Token 1's q is not finite: the rows that it sees have no total any more,
    the others get the other tokens' weight."""
    H, kv, hd = 4, 2, 64
    seen = chain(T)
    q, k, v = inputs(H, kv, hd, n, T, n + T, 53)
    w0, w = (torch.zeros(kv, n + T, device="cuda") for _ in range(2))
    ref = run(be, q, k, v, H, n, T, mask=words_of(seen), weights=w0)
    check(ref, q, k, v, H, n, T, seen, w0, torch.zeros_like(w0))
    q[1] = bad
    out = run(be, q, k, v, H, n, T, mask=words_of(seen), weights=w)
    assert not bool(torch.isfinite(out[1]).any()) and not bool(torch.isfinite(w[:, :n + 2]).any())
    assert torch.equal(w[:, n + 2:], w0[:, n + 2:])
    keep = [t for t in range(T) if t != 1]
    assert torch.equal(out[keep], ref[keep])


@pytest.mark.parametrize("T", [4, 70])
def test_totals_of_a_spoiled_key(be, T):
    """Drafted key 2 is NaN and token 3 alone sees it: rows that token 3 sees
    have no total, the others' are as without it.  (Both runs are within the
    derived tolerance of the definition: 2 * 72 u D, D below 30 for 64 products
    of q and k, and (40 + 70 + 140 + 64) u; twice that is below 6e-4.)"""
    H, kv, hd, n = 4, 2, 64, 40
    seen = np.eye(T, dtype=bool)
    seen[3, 2] = True
    seen[2, 2] = False
    q, k, v = inputs(H, kv, hd, n, T, n + T, 59)
    w0, w = (torch.zeros(kv, n + T, device="cuda") for _ in range(2))
    run(be, q, k, v, H, n, T, mask=words_of(seen), weights=w0)
    k[:, n + 2] = float("nan")
    run(be, q, k, v, H, n, T, mask=words_of(seen), weights=w)
    lost = [*range(n), n + 2, n + 3]
    rest = [r for r in range(n + T) if r not in lost]
    assert not bool(torch.isfinite(w[:, lost]).any())
    assert bool(((w - w0)[:, rest].abs() <= 6e-4 * w0[:, rest]).all())
