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


MOE = dict(arch="olmoe", layers=2, d=192, heads=4, kv_heads=4, vocab=600, experts=12, experts_used=3, dtype="q8_0", seed=34)


def test_the_memory_report_counts_the_expert_layers_units_and_workspace(rb, models):
    """Q4_0 banks are held as Q8_0 rows and, where a layer runs on the few-token kernels, as units with a workspace. A down bank whose rows are no
    multiple of 32 is stored as F16: then nothing is held for those kernels."""
    def report(ff, dtype):
        engine = rb.Engine(str(models(f"moe_{dtype}_{ff}", **MOE, ff=ff, expert_dtype=dtype)), rb.EngineConfig(n_ctx=64, n_seq_max=1, n_batch=32, n_ubatch=32))
        r = engine.memory_report()
        engine.close()
        return r["model_weight_bytes"], r["generation_compute_bytes"]

    assert report(168, "q4_0") == report(168, "q8_0")
    (w4, c4), (w8, c8) = report(160, "q4_0"), report(160, "q8_0")
    gate, up, down = (rb.W4Matrix(Q4_0, np.zeros(12 * n_out * n_in // 32 * 18, np.uint8), n_out, n_in, n_expert=12) for n_out, n_in in ((160, 192), (160, 192), (192, 160)))
    assert w4 - w8 == MOE["layers"] * (gate.nbytes + up.nbytes + down.nbytes)
    assert c4 - c8 == rb.w4_moe_workspace(gate, 16, MOE["experts_used"])


@pytest.mark.parametrize("handle", [False, True])
def test_operands_of_a_call_on_another_stream_may_be_dropped_at_once(rb, handle):
    """The call waits on its stream while its operands are dropped and tensors of their sizes are made: those get other memory."""
    import torch

    rng = np.random.default_rng(2)
    make = lambda n_out, n_in, E=1: rb.W4Matrix(Q4_0, np.concatenate([stored_rows(rng, Q4_0, n_out, n_in) for _ in range(E)]), n_out, n_in, n_expert=E)
    m, up, gates, ups, downs = make(512, 512), make(512, 512), make(64, 512, 4), make(64, 512, 4), make(512, 64, 4)
    side = torch.cuda.Stream()
    base = {"x": torch.randn(4, 512, device="cuda"), "norm": torch.randn(512, device="cuda"), "bias": torch.randn(512, device="cuda"),
            "residual": torch.randn(4, 512, device="cuda"), "router": torch.randn(4, 512, device="cuda")}
    calls = {
        "matvec": (("x", "norm", "bias", "residual"), lambda o, s: rb.w4_matvec(m, o["x"], norm=o["norm"], bias=o["bias"], residual=o["residual"], stream=s)),
        "glu": (("x", "norm"), lambda o, s: rb.w4_glu(m, up, o["x"], norm=o["norm"], stream=s)),
        "moe": (("x", "norm", "residual", "router"), lambda o, s: rb.w4_moe(o["router"], gates, ups, downs, o["x"], 2, norm=o["norm"], residual=o["residual"], stream=s)),
    }
    for names, call in calls.values():
        want = call(base, None)
        torch.cuda.synchronize()
        operands = {name: base[name].clone() for name in names}
        at = {name: t.data_ptr() for name, t in operands.items()}
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            torch.cuda._sleep(50_000_000)
        y = call(operands, side.cuda_stream if handle else side)
        shapes = [base[name].shape for name in names]
        operands.clear()
        fresh = [torch.zeros(shape, device="cuda") for shape in shapes for _ in range(3)]
        assert not {t.data_ptr() for t in fresh} & set(at.values())
        side.synchronize()
        assert torch.equal(y, want)


def test_operands_that_require_a_gradient_are_refused_where_one_is_recorded(rb):
    import torch

    rng = np.random.default_rng(3)
    make = lambda n_out, n_in, E=1: rb.W4Matrix(Q4_0, np.concatenate([stored_rows(rng, Q4_0, n_out, n_in) for _ in range(E)]), n_out, n_in, n_expert=E)
    m, up, gates, ups, downs = make(64, 64), make(64, 64), make(32, 64, 2), make(32, 64, 2), make(64, 32, 2)
    plain = {"x": torch.randn(2, 64, device="cuda"), "norm": torch.randn(64, device="cuda"), "bias": torch.randn(64, device="cuda"),
             "residual": torch.randn(2, 64, device="cuda"), "router": torch.randn(2, 64, device="cuda"), "out": torch.empty(2, 64, device="cuda")}
    calls = {
        ("x", "norm", "bias", "residual", "out"): lambda o: rb.w4_matvec(m, o["x"], norm=o["norm"], bias=o["bias"], residual=o["residual"], out=o["out"]),
        ("x", "norm", "out"): lambda o: rb.w4_glu(m, up, o["x"], norm=o["norm"], out=o["out"]),
        ("router", "x", "norm", "residual", "out"): lambda o: rb.w4_moe(o["router"], gates, ups, downs, o["x"], 1, norm=o["norm"], residual=o["residual"], out=o["out"]),
    }
    for names, call in calls.items():
        want = call(plain).clone()
        for name in names:
            operands = {**plain, name: plain[name].clone().requires_grad_()}
            with pytest.raises(rb.InvalidArgument, match=f"{name} requires a gradient"):
                call(operands)
            for quiet in (torch.no_grad, torch.inference_mode):
                with quiet():
                    assert torch.equal(call(operands), want)
            assert operands[name].grad is None
