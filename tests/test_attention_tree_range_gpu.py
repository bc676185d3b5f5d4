"""Attention of drafted tokens where magnitudes differ widely, against the definition in
64 bits with the tolerance derived in test_attention_tree_gpu.py, unless a test says
otherwise."""
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
