"""The generator's log probabilities where a call returns nothing or fails."""
import pytest

from smallm_engine_b200 import Generator
from test_draft_host import CountingModel, First


def test_an_empty_call_has_no_log_probabilities():
    """They belong to the tokens of the last call, which returned none."""
    g = Generator(CountingModel(), First(), batched_prefill=False, logprobs=1)
    assert g.generate([4, 5], 2) == [6, 7] and len(g.logprobs) == 2
    assert g.generate([], 2) == [] and g.logprobs == []
