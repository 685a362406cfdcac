"""Calls of the products with 4-bit weights that once went wrong, one test each."""
import numpy as np
import pytest

from test_gpu_w4 import MXFP4, Q4_0, decode, dtype_of, f32_bound, stored_rows

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
             "residual": torch.randn(2, 64, device="cuda"), "router": torch.randn(2, 64, device="cuda"), "out": torch.empty(2, 64, device="cuda"), "weights": torch.empty(2, 1, device="cuda")}
    calls = {
        ("x", "norm", "bias", "residual", "out"): lambda o: rb.w4_matvec(m, o["x"], norm=o["norm"], bias=o["bias"], residual=o["residual"], out=o["out"]),
        ("x", "norm", "out"): lambda o: rb.w4_glu(m, up, o["x"], norm=o["norm"], out=o["out"]),
        ("router", "x", "norm", "residual", "out", "weights"): lambda o: rb.w4_moe(o["router"], gates, ups, downs, o["x"], 1, norm=o["norm"], residual=o["residual"], out=o["out"],
                                                                                 weights=o["weights"]),
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


@pytest.mark.parametrize("kind", [Q4_0, MXFP4])
@pytest.mark.parametrize("tokens", [1, 2, 6, 16])
def test_the_largest_magnitudes(rb, kind, tokens):
    """Up to the largest f32 below 65520 2^100 a token's results are the definition's, from there on none is finite; other tokens keep theirs. Under a norm
    whose squares overflow f32 the rows are zeros up to the same limit. Bounds as in test_gpu_w4.py."""
    import torch

    rng = np.random.default_rng(tokens + kind)
    n_in = 224
    raw = stored_rows(rng, kind, 90, n_in, scale_spread=1)
    w, mag = decode(kind, raw)
    m = rb.W4Matrix(kind, raw, 90, n_in)
    limit = np.float32(65520 * 2.0 ** 100)
    plain = rng.normal(0, 1, (tokens, n_in)).clip(-0.9, 0.9).astype(np.float32)
    for top in (np.float32(2.0 ** 112), np.float32(2.0 ** 113), np.float32(1.5 * 2.0 ** 114), np.nextafter(limit, np.float32(0))):
        x = plain.copy()
        x[tokens // 2] *= top
        x[tokens // 2, 5] = top
        x64 = x.astype(np.float64)
        y = rb.w4_matvec(m, torch.tensor(x).cuda()).double().cpu().numpy()
        assert (np.abs(y - x64 @ w.T) <= f32_bound(n_in) * (np.abs(x64) @ mag.T)).all(), top
        assert (rb.w4_matvec(m, torch.tensor(x).cuda(), norm=torch.ones(n_in, device="cuda"))[tokens // 2] == 0).all(), top
    want = rb.w4_matvec(m, torch.tensor(plain).cuda())
    others = [t for t in range(tokens) if t != tokens // 2]
    for top, act in ((limit, "f32"), (np.float32(2.0 ** 120), "f32"), (np.float32(3e38), "f32"), (np.float32(2.0 ** 116), "bf16")):
        x = torch.tensor(plain).to(dtype_of(torch, act)).cuda()
        base = rb.w4_matvec(m, x) if act == "bf16" else want
        x[tokens // 2, 5] = float(top)
        y = rb.w4_matvec(m, x)
        assert not torch.isfinite(y[tokens // 2]).any() and torch.equal(y[others], base[others]), top


@pytest.mark.parametrize("n_out,n_in,tokens", [(40, 32, 1), (129, 992, 5), (64, 4096, 17)])
def test_the_row_kernel_on_stored_q4_0_rows(rb, n_out, n_in, tokens):
    """gemm_rows_kernel, which serves every stored type: sums of n_in f32 products in any order, each product and its weight rounded once."""
    rng = np.random.default_rng(n_in)
    raw = stored_rows(rng, Q4_0, n_out, n_in)
    w, _ = decode(Q4_0, raw)
    x = rng.normal(0, 1, (tokens, n_in)).astype(np.float32)
    y, _ = rb.op_gemm(Q4_0, raw, n_out, n_in, x, path=1)
    x64 = x.astype(np.float64)
    assert (np.abs(y - x64 @ w.T) <= (n_in + 2) * 2.0 ** -24 * (np.abs(x64) @ np.abs(w).T)).all()


@pytest.mark.parametrize("kind", [Q4_0, MXFP4])
def test_rows_on_the_device_are_read_where_they_are(rb, kind):
    """At any address, and behind a stream that is still writing them when the handle is made; they may be overwritten as soon as it is there."""
    import torch

    rng = np.random.default_rng(kind)
    raw = stored_rows(rng, kind, 70, 416)
    x = torch.randn(3, 416, device="cuda")
    want = rb.w4_matvec(rb.W4Matrix(kind, raw, 70, 416), x)
    source, side = torch.tensor(raw).cuda().view(-1), torch.cuda.Stream()
    for offset in (0, 1, 2, 7, 16):
        place = torch.zeros(source.numel() + offset, dtype=torch.uint8, device="cuda")[offset:]
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            torch.cuda._sleep(20_000_000)
            place.copy_(source)
        m = rb.W4Matrix(kind, place, 70, 416)
        place.zero_()
        assert torch.equal(rb.w4_matvec(m, x), want), offset


def test_a_backward_pass_notices_that_a_call_wrote_what_it_saved(rb):
    import torch

    rng = np.random.default_rng(3)
    make = lambda n_out, n_in, E=1: rb.W4Matrix(Q4_0, np.concatenate([stored_rows(rng, Q4_0, n_out, n_in) for _ in range(E)]), n_out, n_in, n_expert=E)
    m, up, gates, ups, downs = make(64, 64), make(64, 64), make(32, 64, 2), make(32, 64, 2), make(64, 32, 2)
    x, router = torch.randn(2, 64, device="cuda"), torch.randn(2, 64, device="cuda")
    moe = lambda **kw: rb.w4_moe(router, gates, ups, downs, x, 1, **kw)
    for shape, call in (((2, 64), lambda t: rb.w4_matvec(m, x, out=t)), ((2, 64), lambda t: rb.w4_glu(m, up, x, out=t)), ((2, 64), lambda t: moe(out=t)),
                        ((2, 1), lambda t: moe(weights=t))):
        saved, scale = torch.randn(shape, device="cuda"), torch.ones(shape, device="cuda", requires_grad=True)
        loss = (saved * scale).sum()
        call(saved)
        with pytest.raises(RuntimeError, match="inplace operation"):
            loss.backward()
        with torch.inference_mode():
            call(torch.randn(shape, device="cuda"))


def test_the_null_stream_by_its_handle_while_another_is_current(rb):
    import torch

    m = rb.W4Matrix(Q4_0, stored_rows(np.random.default_rng(1), Q4_0, 96, 128), 96, 128)
    x = torch.randn(3, 128, device="cuda")
    want = rb.w4_matvec(m, x)
    with torch.cuda.stream(torch.cuda.Stream()):
        y = rb.w4_matvec(m, x, stream=0)
        z = rb.w4_matvec(m, x, stream=torch.cuda.default_stream())
    torch.cuda.synchronize()
    assert torch.equal(y, want) and torch.equal(z, want)
