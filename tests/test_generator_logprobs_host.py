"""The generator's log probabilities where a call returns nothing or fails."""
import pytest

from smallm_engine_b200 import Generator
from test_draft_host import CountingModel, First


def test_an_empty_call_has_no_log_probabilities():
    """They belong to the tokens of the last call, which returned none."""
    g = Generator(CountingModel(), First(), batched_prefill=False, logprobs=1)
    assert g.generate([4, 5], 2) == [6, 7] and len(g.logprobs) == 2
    assert g.generate([], 2) == [] and g.logprobs == []


class CacheModel(CountingModel):
    """Keeps the tokens that its cache holds."""

    def __init__(self):
        super().__init__()
        self.rows, self.fail = [], False

    def forward(self, token, pos, want_logits=True):
        assert pos == len(self.rows)
        self.rows.append(token)
        return super().forward(token, pos, want_logits)

    def truncate_cache(self, n):
        assert n <= len(self.rows)
        del self.rows[n:]

    def logprobs(self, token, top):
        if self.fail:
            raise ValueError("refused")
        return super().logprobs(token, top)


def test_a_failed_call_leaves_no_stale_prefix():
    """A refused number of alternatives ends a call half way; the next one must
    not take rows of that call's prompt for rows of an earlier one's."""
    m = CacheModel()
    g = Generator(m, First(), batched_prefill=False, logprobs=1)
    assert g.generate([1, 2, 10, 11], 2) == [12, 13]
    m.fail = True
    with pytest.raises(ValueError):
        g.generate([1, 2, 30, 31, 32], 2)
    m.fail = False
    assert g.generate([1, 2, 10, 11, 12], 2) == [13, 14]
    assert m.rows == [1, 2, 10, 11, 12, 13, 14]
    assert g.stats.reused_tokens == 2
