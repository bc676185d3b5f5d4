"""The draft-verification entry points where there is no GPU: they are
exported and bound, refuse a missing context or model, and the generator's log
probabilities follow the model's."""
import ctypes

import pytest

from smallm_engine_b200 import Generator, TokenLogprobs, _lib

NEW = ["smallm_attention_tree", "smallm_attention_tree_workspace", "smallm_cache_select", "smallm_cache_move",
       "smallm_logprobs", "smallm_model_logprobs"]


@pytest.mark.parametrize("name", NEW)
def test_declared_bound_and_null_safe(name):
    assert name in _lib.declared_symbols()
    f = getattr(_lib.lib(), name)
    args = [t() if t in (ctypes.c_uint32, ctypes.c_uint64, ctypes.c_int) else None
            for t in _lib.SIGNATURES[name][1]]
    assert f(*args) == _lib.ERR_INVALID
    assert b"NULL" in _lib.lib().smallm_last_error()


class CountingModel:
    """Token i follows token i - 1; log probabilities are recorded."""

    def config(self):
        return self

    n_layers = 0

    def __init__(self):
        self.last, self.asked = 0, []

    def forward(self, token, pos, want_logits=True):
        self.last = token
        return [float(i == token + 1) for i in range(50)]

    def truncate_cache(self, n):
        pass

    def logprobs(self, token, top):
        self.asked.append((self.last, token, top))
        return TokenLogprobs(token, -0.5, 0.1, [(token, -0.5)] * top)


class First:
    def sample(self, logits):
        return max(range(len(logits)), key=lambda i: logits[i])


@pytest.mark.parametrize("top", [None, 0, 3])
def test_generator_scores_each_token_before_it_is_fed(top):
    m = CountingModel()
    g = Generator(m, First(), batched_prefill=False, logprobs=top)
    assert g.generate([4, 5], 4) == [6, 7, 8, 9]
    if top is None:
        assert m.asked == [] and g.logprobs == []
    else:
        assert m.asked == [(5, 6, top), (6, 7, top), (7, 8, top), (8, 9, top)]
        assert [r.token for r in g.logprobs] == [6, 7, 8, 9] and len(g.logprobs[0].top) == top
    g.generate([4], 1)
    assert len(g.logprobs) == (0 if top is None else 1)  # of the last call alone
