"""What the generator's log probabilities refer to: softmax of the model's
logits, whatever the sampler makes of them.  Tolerance as for the operator on
the model's vocabulary: 700 u (u = 2^-24)."""
import numpy as np
import pytest

from smallm_engine_b200 import CudaModel, Generator, TemperatureSampler, TopKSampler, TopPSampler, synth

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


@pytest.mark.parametrize("sampler", [lambda: TemperatureSampler(0.25, 3), lambda: TemperatureSampler(4.0, 3),
                                     lambda: TopKSampler(3, 0.5, 3), lambda: TopPSampler(0.3, 2.0, 3)],
                         ids=["cold", "hot", "top-k", "top-p"])
def test_logprobs_are_of_the_logits(gguf_dir, sampler):
    m = CudaModel(synth.write_gguf(synth.tiny_spec("llama-q4_0"), 8, gguf_dir / "lp-meaning.gguf"))
    prompt = [5, 9, 200, 31]
    g = Generator(m, sampler(), batched_prefill=False, logprobs=4)
    out = g.generate(prompt, 6)
    assert [r.token for r in g.logprobs] == out
    m.reset_cache()
    for pos, t in enumerate(prompt):
        logits = m.forward(t, pos)
    for i, r in enumerate(g.logprobs):
        d = logits.astype(np.float64) - logits.max()
        ref = d - np.log(np.exp(d).sum())
        assert abs(r.logprob - ref[r.token]) <= 700 * U
        assert [t for t, _ in r.top] == np.argsort(-logits, kind="stable")[:4].tolist()
        logits = m.forward(r.token, len(prompt) + i)
    m.close()
