"""Totals and eviction step by step, each against the step before it on the
device: what a call added to each row's total, within the attention's derived
bound on that row's own weight, and the rows that a selection keeps and a move
leaves, exactly."""
import numpy as np
import pytest
import torch

from test_attention_tree_gpu import check, random_parents, run, tree_bits, words_of

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("H,kv,hd", [(8, 2, 64), (12, 2, 128)])
def test_kept_rows_are_those_of_the_largest_totals(be, H, kv, hd):
    max_ctx, budget, first, last = 160, 96, 4, 16
    rng = np.random.default_rng(5)
    g = torch.Generator(device="cuda").manual_seed(5)
    k, v = (torch.randn(kv, max_ctx, hd, device="cuda", generator=g) for _ in range(2))
    w = torch.zeros(kv, max_ctx, device="cuda")
    n = 100
    for step in range(5):
        T = 11 + step
        seen = tree_bits(random_parents(T, rng))
        k[:, n:n + T], v[:, n:n + T] = (torch.randn(kv, T, hd, device="cuda", generator=g) for _ in range(2))
        w[:, n:n + T] = 0
        before = w.clone()
        q = torch.randn(T, H * hd, device="cuda", generator=g)
        out = run(be, q, k, v, H, n, T, mask=words_of(seen), weights=w)
        check(out, q, k, v, H, n, T, seen, w, before)
        n += T
        # the selection, from the totals as the device has them
        rows = torch.empty(kv, budget, dtype=torch.int32, device="cuda")
        torch.cuda.synchronize()
        be.cache_select(w.data_ptr(), kv, max_ctx, n, budget, first, last, rows.data_ptr())
        be.synchronize()
        totals = w.cpu().numpy()
        want = []
        for h in range(kv):
            mid = np.argsort(-totals[h, first:n - last], kind="stable")[:budget - first - last]
            want.append([*range(first), *(first + np.sort(mid)), *range(n - last, n)])
        want = torch.tensor(np.array(want))
        assert torch.equal(rows.cpu().long(), want)
        old = [x.clone() for x in (k, v, w)]
        be.cache_move(k.data_ptr(), v.data_ptr(), kv, hd, max_ctx, rows.data_ptr(), budget, 0, per_head=True,
                      weights=w.data_ptr())
        be.synchronize()
        for new, was in zip((k, v, w), old):
            for h in range(kv):
                assert torch.equal(new[h, :budget], was[h, want[h].cuda()])
                assert torch.equal(new[h, budget:], was[h, budget:])
        n = budget
    assert be.device_errors() == 0
