"""The device error word: each reader clears the bits that it answers for."""
import numpy as np
import pytest
import torch

import oracle as O
from smallm_engine_b200 import CudaModel, SmallmError, synth
from test_kernels_gpu import _residual_sum

pytestmark = pytest.mark.gpu


def raise_bit_7(be):
    """A list that is not ascending (smallm_cache_move)."""
    k, v = torch.zeros(2, 1, 64, 32, device="cuda")
    rows = torch.tensor([3, 3], dtype=torch.int32, device="cuda")
    torch.cuda.synchronize()
    be.cache_move(k.data_ptr(), v.data_ptr(), 1, 32, 64, rows.data_ptr(), 2, 0)
    be.synchronize()


def raise_bit_3(be):
    """A part whose arrival flag never comes up: its wait ends after a second."""
    rows, cols = 32, 512
    W = synth.quantize(O.Q4_0, np.zeros(rows * cols, np.float32))
    qm = be.upload(W, O.Q4_0, rows, cols)
    x, parts, w = torch.zeros(cols, device="cuda"), torch.zeros(2, cols, device="cuda"), torch.ones(cols, device="cuda")
    epoch, flags = (torch.tensor(t, dtype=torch.int32, device="cuda") for t in ([7], [8, 0]))
    out, y = torch.empty(cols, device="cuda"), torch.empty(rows, device="cuda")
    _residual_sum(be, qm, x, parts, flags, epoch, w, 1e-5, out, y)
    torch.cuda.synchronize()


def test_logprobs_of_a_model_answers_for_itself(be, gguf_dir):
    """What the word holds from others neither fails the call nor is cleared."""
    m = CudaModel(synth.write_gguf(synth.tiny_spec("llama-q4_0"), 8, gguf_dir / "errors-lp.gguf"))
    m.forward(5, 0)
    want = m.logprobs(7, 4)
    assert be.device_errors() == 0
    raise_bit_7(be)
    raise_bit_3(be)
    assert m.logprobs(7, 4) == want and m.logprobs().entropy == want.entropy
    assert be.device_errors() == 128 + 8 and be.device_errors() == 0
    m.close()


def test_a_steps_error_leaves_the_operators_bits(be, gguf_dir):
    """A step that finds a step's bit answers for that one: the bad list's stays
    for the caller of smallm_cache_move."""
    m = CudaModel(synth.write_gguf(synth.tiny_spec("llama-q4_0"), 8, gguf_dir / "errors.gguf"))
    want = m.forward(5, 0)
    assert be.device_errors() == 0
    raise_bit_7(be)
    raise_bit_3(be)
    assert be.device_errors(clear=False) == 128 + 8
    m.reset_cache()
    with pytest.raises(SmallmError, match="flags 8"):
        m.forward(5, 0)
    assert be.device_errors(clear=False) == 128
    m.reset_cache()
    np.testing.assert_array_equal(m.forward(5, 0), want)
    assert be.device_errors() == 128 and be.device_errors() == 0
    m.close()
