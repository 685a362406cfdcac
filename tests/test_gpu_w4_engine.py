"""Models with Q4_0 weights, and MXFP4 experts under RB200_MOE=few: the steps of at most sixteen tokens run the products with
4-bit weights, longer ones the kernels of the re-coded weights; both against the oracle on the stored weights."""
import numpy as np
import pytest

from helpers import ParityReport, check_step, expect_greedy

pytestmark = pytest.mark.gpu

DENSE = {
    # GQA with a fused q, k, v and a gated pair of whole row blocks
    "llama": dict(arch="llama", layers=2, d=256, heads=4, kv_heads=2, ff=704, vocab=1003, dtype="q4_0", seed=31),
    # biases, tied head, and an ff that is no multiple of 32: its down projection is stored as F16, the gated pair stays two products
    "qwen2": dict(arch="qwen2", layers=2, d=192, heads=6, kv_heads=2, ff=304, vocab=700, dtype="q4_0", bias=1, seed=32),
    # 4-bit matrices between others: the embedding and the head in Q8_0
    "mixed": dict(arch="llama", layers=3, d=320, heads=5, kv_heads=5, head_dim=64, ff=448, vocab=512, dtype="q4_0", embd_dtype="q8_0", seed=33),
}
MOE = dict(arch="olmoe", layers=2, d=192, heads=4, kv_heads=4, ff=160, vocab=600, experts=12, experts_used=3, dtype="q8_0", seed=34)


def _workload(rb, oracle, path, sizes, vocab, steps=4, n_batch=128):
    """Prompts of the given lengths in one step each, then decode steps of all of them together; every step against the oracle."""
    n = len(sizes)
    engine = rb.Engine(str(path), rb.EngineConfig(n_ctx=2048, n_seq_max=n, n_batch=n_batch, n_ubatch=n_batch))
    octx = oracle.Context(oracle.Model(str(path)), n, 512)
    out, rep, g = rb.StepOutput(), ParityReport(), rb.SamplingParamsV2.greedy()
    rng = np.random.default_rng(11)
    last = []
    for i, size in enumerate(sizes):
        rows = [rb.StepRow(i, i, rng.integers(3, vocab, size).tolist(), 0, sample=True, sampling=g)]
        expect_greedy(oracle, check_step(rb, engine, octx, oracle, rows, out, rep), rep)
        last.append(out.row(0).token)
    for step in range(steps):
        rows = [rb.StepRow.decode(i, i, last[i], sizes[i] + step, g) for i in range(n)]
        expect_greedy(oracle, check_step(rb, engine, octx, oracle, rows, out, rep), rep)
        last = [out.row(i).token for i in range(n)]
    return engine, octx, rep, last


@pytest.mark.parametrize("name", list(DENSE))
def test_q4_0_models_match_the_oracle_in_short_and_long_steps(rb, oracle, models, name):
    spec = DENSE[name]
    path = models(f"q4_0_{name}", **spec)
    for sizes in ((1, 7), (16, 17, 40, 3, 2)):
        engine, _, rep, _ = _workload(rb, oracle, path, sizes, spec["vocab"])
        print(f"q4_0 {name} {sizes}: max|dlogit|={rep.max_logit_diff:.2e}, ties {rep.tie_events}")
        engine.close()


def test_q4_0_steps_replay_as_graphs_with_the_same_results(rb, models, monkeypatch):
    """Seen twice, a step shape is captured and replayed; eager and replayed steps, and the profiled ones, agree bit for bit."""
    path = models("q4_0_llama", **DENSE["llama"])
    g = rb.SamplingParamsV2.greedy()
    streams = []
    for graphs in (True, False):
        monkeypatch.setenv("RB200_GRAPHS", "1" if graphs else "0")
        engine = rb.Engine(str(path), rb.EngineConfig(n_ctx=512, n_seq_max=3, n_batch=64, n_ubatch=64))
        out = rb.StepOutput()
        got = []
        for i in range(3):
            engine.step([rb.StepRow(i, i, [5 + i, 9, 11 * i + 3], 0, sample=True, sampling=g)], out)
            got.append(out.row(0).token)
        last = list(got)
        for step in range(6):
            engine.step([rb.StepRow.decode(i, i, last[i], 3 + step, g) for i in range(3)], out)
            last = [out.row(i).token for i in range(3)]
            got.append((tuple(last), engine.last_logits(2).tobytes()))
        assert (engine.graph_stats()[0] > 0) == graphs
        streams.append(got)
        engine.close()
    assert streams[0] == streams[1]


def test_per_row_adapters_over_q4_0_weights(rb, oracle, models, tmp_path):
    gguf = pytest.importorskip("gguf")
    spec = DENSE["llama"]
    path = models("q4_0_llama", **spec)
    d, dkv, ff = spec["d"], 128, spec["ff"]
    rng = np.random.default_rng(8)
    w = gguf.GGUFWriter(str(tmp_path / "a.gguf"), "llama")
    w.add_string("general.type", "adapter")
    w.add_string("adapter.type", "lora")
    w.add_float32("adapter.lora.alpha", 16.0)
    for layer in range(2):
        for t, (n_in, n_out) in {"attn_q": (d, d), "attn_v": (d, dkv), "ffn_gate": (d, ff), "ffn_down": (ff, d)}.items():
            w.add_tensor(f"blk.{layer}.{t}.weight.lora_a", rng.normal(0, 0.05, (8, n_in)).astype(np.float32))
            w.add_tensor(f"blk.{layer}.{t}.weight.lora_b", rng.normal(0, 0.05, (n_out, 8)).astype(np.float32))
    w.write_header_to_file()
    w.write_kv_data_to_file()
    w.write_tensors_to_file()
    w.close()
    engine = rb.Engine(str(path), rb.EngineConfig(n_ctx=512, n_seq_max=3, n_batch=64, n_ubatch=64))
    om = oracle.Model(str(path))
    octx = oracle.Context(om, 3, 256)
    ida = engine.adapter_load(str(tmp_path / "a.gguf"))
    assert ida == om.lora_load(str(tmp_path / "a.gguf"))
    out, rep, g = rb.StepOutput(), ParityReport(), rb.SamplingParamsV2.greedy()
    rows = [rb.StepRow(i, i, rng.integers(3, 1003, 4).tolist(), 0, sample=True, sampling=g, adapter=a) for i, a in enumerate((ida, rb.ADAPTER_BASE, ida))]
    expect_greedy(oracle, check_step(rb, engine, octx, oracle, rows, out, rep), rep)
    engine.close()


@pytest.mark.parametrize("expert_dtype,few", [("q4_0", False), ("mxfp4", True)])
def test_expert_layers_match_the_oracle_and_its_routing(rb, oracle, models, monkeypatch, expert_dtype, few):
    if few:
        monkeypatch.setenv("RB200_MOE", "few")
    path = models(f"moe_{expert_dtype}_w4", **MOE, expert_dtype=expert_dtype)
    for sizes in ((1,), (5, 16, 30, 2)):
        engine, octx, rep, last = _workload(rb, oracle, path, sizes, MOE["vocab"])
        # the routes of a short step, expert by expert, where the oracle's choice is not a matter of rounding
        n = len(sizes)
        out, g = rb.StepOutput(), rb.SamplingParamsV2.greedy()
        rows = [rb.StepRow.decode(i, i, last[i], sizes[i] + 4, g) for i in range(n)]
        expect_greedy(oracle, check_step(rb, engine, octx, oracle, rows, out, rep), rep)
        got = engine.last_routes().reshape(MOE["layers"], n, MOE["experts_used"])
        want = octx.last_routes().reshape(got.shape)
        # logits of this size differ by less than 1e-5 between the two sides: a gap above 4e-5 decides on both alike
        clear = octx.last_route_margins().reshape(MOE["layers"], n) > 4e-5
        assert np.array_equal(got[clear], want[clear]) and clear.mean() > 0.7
        print(f"experts {expert_dtype} {sizes}: max|dlogit|={rep.max_logit_diff:.2e}")
        engine.close()


def test_the_expert_inventory_names_the_stored_type(rb, models):
    path = models("moe_q4_0_w4", **MOE, expert_dtype="q4_0")
    engine = rb.Engine(str(path), rb.EngineConfig(n_ctx=64, n_seq_max=1, n_batch=32, n_ubatch=32))
    banks = engine.expert_banks()
    assert len(banks) == 6 and all(b["type_name"] == "Q4_0" for b in banks), banks
    assert all(b["n_bytes"] == 12 * 160 * 192 // 32 * 18 for b in banks)
    assert engine.expert_storage(0) == (8, 8, 8)        # what steps above sixteen tokens read: Q8_0 blocks of the same values
    engine.close()
