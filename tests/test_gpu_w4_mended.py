"""Calls of the products with 4-bit weights that once went wrong, one test each."""
import numpy as np
import pytest

from test_gpu_w4 import Q4_0, stored_rows

pytestmark = pytest.mark.gpu


def test_a_failed_allocation_is_not_the_next_calls_error(rb, c1_model):
    """A handle too large for the device is an error of its own; a product and an engine's step behind it are not concerned."""
    import torch

    raw = stored_rows(np.random.default_rng(1), Q4_0, 32, 64)
    m = rb.W4Matrix(Q4_0, raw, 32, 64)
    x = torch.ones(2, 64, device="cuda")
    want = rb.w4_matvec(m, x)
    engine = rb.Engine(str(c1_model), rb.EngineConfig(n_ctx=64, n_seq_max=1, n_batch=32, n_ubatch=32))
    lib = rb.load_library()
    too_large = lambda: lib.retro_b200_w4_new(Q4_0, raw.ctypes.data, 32 * 1048575, 262144, 1)      # 4.9 TB
    assert not too_large() and b"out of memory" in lib.retro_last_error()
    assert torch.equal(rb.w4_matvec(m, x), want)
    assert not too_large()
    engine.step([rb.StepRow(0, 0, [5, 9, 3], 0, sample=True, sampling=rb.SamplingParamsV2.greedy())], rb.StepOutput())
    engine.close()
