"""Products with 4-bit weights for few tokens: layouts, values and callers that the sizes in test_gpu_w4.py do not reach.

Tolerances are those derived there; "the same" is bit for bit.
"""
import numpy as np
import pytest

from test_gpu_w4 import MXFP4, Q4_0, activations, decode, dtype_of, expert_parts, f32_bound, half_step, moe64, moe_inputs, normed, route64, stored_rows

pytestmark = pytest.mark.gpu


def matrix(rb, rng, kind, n_out, n_in, spread=3):
    raw = stored_rows(rng, kind, n_out, n_in, scale_spread=spread)
    return rb.W4Matrix(kind, raw, n_out, n_in), *decode(kind, raw)


def bank(rb, raws, kinds, E, d, ff):
    gate, up = (rb.W4Matrix(kinds[0], np.stack(r), ff, d, n_expert=E) for r in raws[:2])
    return gate, up, rb.W4Matrix(kinds[1], np.stack(raws[2]), d, ff, n_expert=E)


def within(torch, y, want, mag, act, n_in):
    bound = f32_bound(n_in) * mag + half_step(torch, act) * np.abs(want)
    return (np.abs(y.double().cpu().numpy() - want) <= bound).all()


@pytest.mark.parametrize("kind", [Q4_0, MXFP4])
@pytest.mark.parametrize("n_in", [65536, 131072, 262144])
def test_long_rows(rb, kind, n_in):
    """Rows that fill the shared memory of a cluster, at every number of tokens that changes a kernel's room."""
    import torch

    rng = np.random.default_rng(n_in + kind)
    m, w, mag = matrix(rb, rng, kind, 40, n_in)
    for tokens in (1, 2, 3, 4, 5, 8, 9, 16):
        for act in ("bf16", "f32"):
            x, x64 = activations(rng, torch, tokens, n_in, act)
            assert within(torch, rb.w4_matvec(m, x), x64 @ w.T, np.abs(x64) @ mag.T, act, n_in), (tokens, act)


@pytest.mark.parametrize("kind", [Q4_0, MXFP4])
@pytest.mark.parametrize("tokens,act", [(1, "f32"), (3, "bf16"), (4, "f32"), (11, "f16"), (18, "f32")])
def test_strides_offsets_and_column_ranges(rb, kind, tokens, act):
    import torch

    rng = np.random.default_rng(tokens + kind)
    n_out, n_in = 75, 416
    m, w, mag = matrix(rb, rng, kind, n_out, n_in, spread=1)
    norm = torch.tensor(rng.normal(1, 0.2, n_in + 1), dtype=torch.float32).cuda()[1:]      # not 16-byte aligned
    plain = torch.tensor(rng.normal(0, 1, (tokens, n_in)), dtype=torch.float32).to(dtype_of(torch, act)).cuda()
    want = rb.w4_matvec(m, plain, norm=norm)
    for offset, gap in ((1, 0), (3, 5), (8, 8), (4, 1)):
        wide = torch.full((tokens, offset + n_in + gap), float("nan"), dtype=plain.dtype, device="cuda")
        x = wide[:, offset: offset + n_in]
        x.copy_(plain)
        assert torch.equal(rb.w4_matvec(m, x, norm=norm), want), (offset, gap)
    # result and residual are column ranges of one buffer, the result in place; what lies around them stays
    buffer = torch.tensor(rng.normal(0, 1, (tokens + 1, 3 * n_out + 5)), dtype=torch.float32).to(plain.dtype).cuda()
    before = buffer.clone()
    out, residual = buffer[:tokens, 2: 2 + n_out], buffer[:tokens, n_out + 3: 2 * n_out + 3]
    y = rb.w4_matvec(m, plain, norm=norm, residual=residual, out=out)
    assert y is out
    alone = rb.w4_matvec(m, plain, norm=norm, residual=residual.contiguous())
    assert torch.equal(out, alone)
    before[:tokens, 2: 2 + n_out] = alone
    assert torch.equal(buffer, before)
    # one row for every token
    one = plain[:1].expand(tokens, n_in)
    assert one.stride(0) == 0 or tokens == 1
    assert torch.equal(rb.w4_matvec(m, one), rb.w4_matvec(m, one.contiguous()))


def test_result_types(rb):
    """The result's type is the caller's choice: one rounding of the same f32 sum."""
    import torch

    rng = np.random.default_rng(4)
    m, _, _ = matrix(rb, rng, Q4_0, 70, 256, spread=1)
    for tokens in (1, 6, 12):
        for act in ("f32", "f16", "bf16"):
            x = torch.tensor(rng.normal(0, 1, (tokens, 256)), dtype=torch.float32).to(dtype_of(torch, act)).cuda()
            full = rb.w4_matvec(m, x, out=torch.empty(tokens, 70, device="cuda"))
            for t in (torch.float16, torch.bfloat16):
                assert torch.equal(rb.w4_matvec(m, x, out=torch.empty(tokens, 70, dtype=t, device="cuda")), full.to(t))


@pytest.mark.parametrize("kind", [Q4_0, MXFP4])
@pytest.mark.parametrize("tokens", [1, 2, 4, 7, 16])
def test_small_and_large_magnitudes(rb, kind, tokens):
    """Rows of zeros, rows down to the smallest f32 and up to 2^100. Below 2^-104 an activation is a multiple of 2^-142 (the scale that takes
    sums back has to be an f32 too) and off by half of that."""
    import torch

    rng = np.random.default_rng(tokens + kind)
    n_in = 224
    m, w, mag = matrix(rb, rng, kind, 90, n_in, spread=1)
    for exponent in (-140, -130, -120, -112, -108, -104, -100, -60, 60, 100):
        base = rng.normal(0, 1, (tokens, n_in)).clip(-3, 3)
        x = torch.tensor((base * 2.0 ** exponent).astype(np.float32)).cuda()
        if tokens > 1:
            x[tokens // 2] = 0
        x64 = x.double().cpu().numpy()
        y = rb.w4_matvec(m, x).double().cpu().numpy()
        # 2^-149: the result's own half step below the normal numbers, in each of the cluster's partial sums and the factor's product
        bound = f32_bound(n_in) * (np.abs(x64) @ mag.T) + 2.0 ** -143 * mag.sum(1) + 8 * 2.0 ** -149
        assert (np.abs(y - x64 @ w.T) <= bound).all(), exponent
        if tokens > 1:
            assert (y[tokens // 2] == 0).all()


@pytest.mark.parametrize("kind", [Q4_0, MXFP4])
@pytest.mark.parametrize("tokens", [2, 4, 6, 16])
def test_tokens_do_not_reach_one_another(rb, kind, tokens):
    """A token with an infinity or a NaN: its own results are not finite, the others are what they were. In the expert layer the other token's
    choice of experts moves the points where the sums are cut: both results are then within the bound of the definition."""
    import torch

    rng = np.random.default_rng(tokens)
    d, ff, E = 256, 96, 6
    m, _, _ = matrix(rb, rng, kind, d, d, spread=1)
    g, _, _ = matrix(rb, rng, kind, d, d, spread=1)
    raws, clean, router = moe_inputs(rng, torch, kind, kind, E, d, ff, tokens, "f32")
    gate, up, down = bank(rb, raws, (kind, kind), E, d, ff)
    banks = [[decode(kind, r) for r in b] for b in raws]
    router, norm = torch.tensor(router).cuda(), torch.ones(d, device="cuda")
    for bad in (float("inf"), float("-inf"), float("nan")):
        for act in (torch.float32, torch.bfloat16):
            x = clean.to(act)
            dirty = x.clone()
            dirty[1, 77] = bad
            others = [t for t in range(tokens) if t != 1]
            for call in (lambda v: rb.w4_matvec(m, v), lambda v: rb.w4_matvec(m, v, norm=norm), lambda v: rb.w4_glu(m, g, v)):
                a, b = call(x), call(dirty)
                assert torch.equal(a[others], b[others])
            ids, dirty_ids = (torch.zeros(tokens, 2, dtype=torch.int32, device="cuda") for _ in range(2))
            a = rb.w4_moe(router, gate, up, down, x, 2, ids=ids).double().cpu().numpy()
            b = rb.w4_moe(router, gate, up, down, dirty, 2, ids=dirty_ids).double().cpu().numpy()
            assert torch.equal(ids[others], dirty_ids[others]) and not np.isfinite(b[1]).any()
            x64, chosen = x.double().cpu().numpy(), ids.cpu().numpy().astype(np.int64)
            _, p, _ = route64(x64, router.double().cpu().numpy(), 2, False)
            want, bound = moe64(x64, p, chosen, *banks, False)
            bound = bound + 4e-5 * expert_parts(x64, p, chosen, *banks, False) + 2.0 ** -22 * np.abs(want)
            bound = bound + half_step(torch, "bf16" if act == torch.bfloat16 else "f32") * np.abs(want)
            for y in (a, b):
                assert (np.abs(y - want) <= bound)[others].all()
            assert not torch.isfinite(rb.w4_matvec(m, dirty)[1]).any()


def test_routing_of_ties_and_nan(rb):
    """Equal probabilities go to the lowest ids; a token whose logits are NaN gets n_used different experts and NaN weights."""
    import torch

    rng = np.random.default_rng(8)
    for E, k, tokens in ((4, 2, 1), (40, 32, 5), (256, 32, 16), (33, 1, 2)):
        d, ff = 96, 64
        raws, x, _ = moe_inputs(rng, torch, Q4_0, MXFP4, E, d, ff, tokens, "f32")
        gate, up, down = bank(rb, raws, (Q4_0, MXFP4), E, d, ff)
        ids = torch.full((tokens, k), -1, dtype=torch.int32, device="cuda")
        weights = torch.zeros(tokens, k, device="cuda")
        rb.w4_moe(torch.zeros(E, d, device="cuda"), gate, up, down, x, k, ids=ids, weights=weights)
        assert (ids.cpu() == torch.arange(k, dtype=torch.int32)).all() and (weights.cpu() - 1 / E).abs().max() <= 2 ** -22 / E
        # two equal rows of the router, one of them the last: the lower id comes first
        router = torch.tensor(rng.normal(0, 1, (E, d)), dtype=torch.float32).cuda()
        router[E - 1] = router[0]
        rb.w4_moe(router, gate, up, down, x, k, ids=ids)
        for row in ids.cpu().tolist():
            assert len(set(row)) == k and (E - 1 not in row or 0 in row and row.index(0) < row.index(E - 1))
        x[0, 5] = float("nan")
        rb.w4_moe(router, gate, up, down, x, k, ids=ids, weights=weights)
        assert sorted(set(ids[0].cpu().tolist())) == sorted(ids[0].cpu().tolist()) and ids.min() >= 0 and ids.max() < E
        assert weights[0].isnan().all() and weights[1:].isfinite().all()


@pytest.mark.parametrize("tokens", [1, 4, 8, 16])
def test_every_run_gives_the_same_bits(rb, tokens):
    import torch

    rng = np.random.default_rng(tokens)
    m, _, _ = matrix(rb, rng, Q4_0, 2000, 4096)
    raws, x, router = moe_inputs(rng, torch, MXFP4, MXFP4, 16, 512, 480, tokens, "f32")
    gate, up, down = bank(rb, raws, (MXFP4, MXFP4), 16, 512, 480)
    router = torch.tensor(router).cuda()
    v = torch.tensor(rng.normal(0, 1, (tokens, 4096)), dtype=torch.float32).cuda()
    first = rb.w4_matvec(m, v), rb.w4_moe(router, gate, up, down, x, 4)
    for _ in range(20):
        assert torch.equal(rb.w4_matvec(m, v), first[0]) and torch.equal(rb.w4_moe(router, gate, up, down, x, 4), first[1])


def layer(rb, w, x, workspace=None, stream=None):
    """A layer as a decoder runs it: a product with norm, residual and bias, a gated pair and its down product, an expert layer in place."""
    h = rb.w4_matvec(w["proj"], x, norm=w["norm"], bias=w["bias"], residual=x, stream=stream)
    g = rb.w4_glu(w["ffn_gate"], w["ffn_up"], h, norm=w["norm"], stream=stream)
    h2 = rb.w4_matvec(w["ffn_down"], g, residual=h, stream=stream)
    return rb.w4_moe(w["router"], w["gate"], w["up"], w["down"], h2, 3, norm=w["norm"], normalise=True, residual=h2, out=h2, workspace=workspace, stream=stream)


@pytest.fixture(scope="module")
def weights(rb):
    import torch

    rng = np.random.default_rng(77)
    d, ff, eff, E = 512, 1376, 288, 12
    raws, _, router = moe_inputs(rng, torch, MXFP4, Q4_0, E, d, eff, 1, "f32")
    gate, up, down = bank(rb, raws, (MXFP4, Q4_0), E, d, eff)
    w = {"gate": gate, "up": up, "down": down, "router": torch.tensor(router).cuda(), "experts": raws,
         "norm": torch.tensor(rng.normal(1, 0.1, d), dtype=torch.float32).cuda(), "bias": torch.tensor(rng.normal(0, 1, d), dtype=torch.float32).cuda()}
    for name, n_out, n_in in (("proj", d, d), ("ffn_gate", ff, d), ("ffn_up", ff, d), ("ffn_down", d, ff)):
        raw = stored_rows(rng, Q4_0, n_out, n_in, scale_spread=1)
        w[name], w[name + "64"] = rb.W4Matrix(Q4_0, raw, n_out, n_in), decode(Q4_0, raw)[0]
    return w


@pytest.mark.parametrize("tokens", [1, 3, 8, 16, 20])
def test_a_layer_against_float64(rb, weights, tokens):
    """The operators one behind the other. Each stage's relative error is below 2^-17 of its output's norm (the bounds above at these sizes),
    and the four stages with their norms and the gated pair's slopes pass it on enlarged by less than 2^4."""
    import torch

    w = weights
    rng = np.random.default_rng(tokens)
    x = torch.tensor(rng.normal(0, 1, (tokens, 512)), dtype=torch.float32).cuda()
    y = layer(rb, w, x).double().cpu().numpy()
    norm, bias = (w[k].double().cpu().numpy() for k in ("norm", "bias"))
    x64 = x.double().cpu().numpy()
    h = normed(x64, norm, 1e-5) @ w["proj64"].T + bias + x64
    n = normed(h, norm, 1e-5)
    a = n @ w["ffn_gate64"].T
    h = h + (a / (1 + np.exp(-a)) * (n @ w["ffn_up64"].T)) @ w["ffn_down64"].T
    n = normed(h, norm, 1e-5)
    order, p, gap = route64(n, w["router"].double().cpu().numpy(), 3, True)
    for t in range(tokens):
        if gap[t] < 1e-3:
            continue            # experts so close that either choice is right
        total = h[t].copy()
        for e in order[t, :3]:
            gt, ut, dn = (decode(k, w["experts"][i][e])[0] for i, k in enumerate((MXFP4, MXFP4, Q4_0)))
            a = gt @ n[t]
            total += p[t, e] / p[t, order[t, :3]].sum() * (dn @ (a / (1 + np.exp(-a)) * (ut @ n[t])))
        assert np.linalg.norm(y[t] - total) <= 2.0 ** -13 * np.linalg.norm(total)
    assert (gap >= 1e-3).any()


@pytest.mark.parametrize("tokens", [1, 16])
def test_another_stream(rb, weights, tokens):
    import torch

    x = torch.randn(tokens, 512, device="cuda")
    want = layer(rb, weights, x)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    for stream in (side, side.cuda_stream):
        ys = [layer(rb, weights, x, stream=stream) for _ in range(5)]
        side.synchronize()
        assert all(torch.equal(y, want) for y in ys)
    with torch.cuda.stream(side):
        ys = [layer(rb, weights, x) for _ in range(5)]
    side.synchronize()
    assert all(torch.equal(y, want) for y in ys)


@pytest.mark.parametrize("tokens", [1, 5, 16])
def test_two_graphs_with_workspaces_of_their_own(rb, weights, tokens):
    """Two captured layers replayed at the same time on two streams; each again with new inputs in the same places."""
    import torch

    need = rb.w4_moe_workspace(weights["gate"], tokens, 3)
    graphs = []
    for _ in range(2):
        x = torch.randn(tokens, 512, device="cuda")
        space = torch.empty(need, dtype=torch.uint8, device="cuda")
        graph, stream = torch.cuda.CUDAGraph(), torch.cuda.Stream()
        with torch.cuda.graph(graph, stream=stream):
            y = layer(rb, weights, x, workspace=space)
        graphs.append((graph, stream, x, y, space))
    for _ in range(4):
        wants = []
        for _, _, x, _, _ in graphs:
            x.normal_()
            wants.append(layer(rb, weights, x))
        torch.cuda.synchronize()
        for _ in range(3):
            for graph, stream, *_ in graphs:
                with torch.cuda.stream(stream):
                    graph.replay()
        torch.cuda.synchronize()
        for (_, _, _, y, _), want in zip(graphs, wants):
            assert torch.equal(y, want)


def test_first_call_inside_a_capture(rb):
    """Nothing has to run before a capture: a fresh process whose first product is a captured one."""
    import subprocess
    import sys

    code = """
import numpy as np, torch, retrograd_b200 as rb
raw = np.zeros((64, 64 // 32 * 18), np.uint8); raw[:, 1::18] = 0x3c; raw[:, 0::18] = 0
m = rb.W4Matrix(2, raw, 64, 64)
x = torch.ones(2, 64, device="cuda"); y = torch.zeros(2, 64, device="cuda"); torch.cuda.synchronize()
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    rb.w4_matvec(m, x, out=y)
g.replay(); torch.cuda.synchronize()
assert (y == -8 * 64).all()
"""
    run = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300)
    assert run.returncode == 0, run.stderr[-2000:]


def test_first_calls_of_several_threads(rb):
    """A fresh process whose threads make their first calls at once, each on a stream of its own, with one weight handle."""
    import subprocess
    import sys

    code = """
import threading
import numpy as np, torch, retrograd_b200 as rb
raw = np.random.default_rng(0).integers(0, 256, (4096, 4096 // 32 * 18), dtype=np.uint8); raw[:, 1::18] = 0x2c
m = rb.W4Matrix(2, raw, 4096, 4096)
xs = {n: torch.randn(n, 4096, device="cuda") for n in (1, 3, 7, 16)}
torch.cuda.synchronize()
gate = threading.Barrier(8)
got = [None] * 8
def work(i):
    stream = torch.cuda.Stream()
    gate.wait()
    got[i] = {n: [rb.w4_matvec(m, x, stream=stream) for _ in range(10)] for n, x in xs.items()}
    stream.synchronize()
threads = [threading.Thread(target=work, args=(i,)) for i in range(8)]
[t.start() for t in threads]; [t.join() for t in threads]
want = {n: rb.w4_matvec(m, x) for n, x in xs.items()}
assert all(torch.equal(y, want[n]) for g in got for n, ys in g.items() for y in ys)
"""
    run = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300)
    assert run.returncode == 0, run.stderr[-2000:]


def test_in_place_expert_layer(rb, weights):
    import torch

    w = weights
    for tokens in (1, 4, 16, 33):
        for act in (torch.float32, torch.bfloat16):
            x = torch.randn(tokens, 512, device="cuda").to(act)
            args = w["router"], w["gate"], w["up"], w["down"]
            want = rb.w4_moe(*args, x, 3, norm=w["norm"], residual=x)
            y = x.clone()
            assert rb.w4_moe(*args, y, 3, norm=w["norm"], residual=y, out=y) is y and torch.equal(y, want)
            want = rb.w4_moe(*args, x, 3)
            y = x.clone()
            rb.w4_moe(*args, y, 3, out=y)
            assert torch.equal(y, want)


@pytest.mark.parametrize("kind,d,ff,tokens", [(Q4_0, 65536, 64, 16), (MXFP4, 65536, 64, 3), (MXFP4, 262144, 32, 16), (Q4_0, 262144, 32, 1), (Q4_0, 64, 65536, 16), (MXFP4, 4096, 8192, 5)])
def test_expert_layer_of_long_rows(rb, kind, d, ff, tokens):
    """Columns that the routing takes in pieces, and passes of fewer tokens where sixteen rows do not fit. Bounds as in test_moe_against_float64."""
    import torch

    rng = np.random.default_rng(d + ff)
    E, k = 3, 2
    raws, x, router = moe_inputs(rng, torch, kind, kind, E, d, ff, tokens, "f32")
    gate, up, down = bank(rb, raws, (kind, kind), E, d, ff)
    norm = rng.normal(1, 0.2, d).astype(np.float32)
    ids = torch.zeros(tokens, k, dtype=torch.int32, device="cuda")
    y = rb.w4_moe(torch.tensor(router).cuda(), gate, up, down, x, k, norm=torch.tensor(norm).cuda(), ids=ids).double().cpu().numpy()
    xn = normed(x.double().cpu().numpy(), norm.astype(np.float64), 1e-5)
    order, p, gap = route64(xn, router.astype(np.float64), k, False)
    chosen = ids.cpu().numpy().astype(np.int64)
    clear = gap > 4e-5
    assert clear.any() and np.array_equal(chosen[clear], order[clear, :k])
    banks = [[decode(kind, r) for r in b] for b in raws]
    want, bound = moe64(xn, p, chosen, *banks, False)
    bound = bound + 4e-5 * expert_parts(xn, p, chosen, *banks, False) + 2.0 ** -22 * np.abs(want)
    assert (np.abs(y - want) <= bound).all()


def test_no_tokens(rb, weights):
    import torch

    w = weights
    x = torch.empty(0, 512, device="cuda")
    assert rb.w4_matvec(w["proj"], x).shape == (0, 512) and rb.w4_glu(w["ffn_gate"], w["ffn_up"], x).shape == (0, 1376)
    assert rb.w4_moe(w["router"], w["gate"], w["up"], w["down"], x, 3).shape == (0, 512)


def test_refusals(rb, weights):
    """Every refusal is decided on the host, with nothing enqueued."""
    import torch

    w = weights
    x, out = torch.zeros(2, 512, device="cuda"), torch.full((2, 512), 7.0, device="cuda")
    moe = lambda v=x, k=3, router=w["router"], down=w["down"], **kw: rb.w4_moe(router, w["gate"], w["up"], down, v, k, **kw)
    closed = rb.W4Matrix(Q4_0, stored_rows(np.random.default_rng(0), Q4_0, 32, 32), 32, 32)
    closed.close()
    big = torch.zeros(2, 1100, device="cuda")
    bad = [
        lambda: rb.w4_matvec(w["proj"], x.double()), lambda: rb.w4_matvec(w["proj"], x[:, :511]), lambda: rb.w4_matvec(w["proj"], x[0]),
        lambda: rb.w4_matvec(w["proj"], x.cpu()), lambda: rb.w4_matvec(w["proj"], torch.zeros(512, 2, device="cuda").t()),
        lambda: rb.w4_matvec(w["proj"], x, out=out[:1]), lambda: rb.w4_matvec(w["proj"], x, out=out[:1].expand(2, 512)),
        lambda: rb.w4_matvec(w["proj"], x, out=out.double()), lambda: rb.w4_matvec(w["proj"], x, out=x),
        lambda: rb.w4_matvec(w["proj"], big[:, :512], out=big[:, 500:1012]), lambda: rb.w4_matvec(w["proj"], x, residual=x.half()),
        lambda: rb.w4_matvec(w["proj"], x, norm=w["norm"].half()), lambda: rb.w4_matvec(w["proj"], x, norm=w["norm"][:100]),
        lambda: rb.w4_matvec(w["proj"], x, norm=w["norm"], eps=-1.0), lambda: rb.w4_matvec(w["proj"], x, norm=w["norm"], eps=float("nan")),
        lambda: rb.w4_matvec(w["proj"], x, bias=x[0].double()), lambda: rb.w4_matvec(w["gate"], x), lambda: rb.w4_matvec(closed, x[:, :32]),
        lambda: rb.w4_matvec(w["proj"], x, residual=out.view(-1)[1:513].view(1, 512).expand(2, 512), out=out),
        lambda: rb.w4_glu(w["ffn_gate"], w["proj"], x), lambda: rb.w4_glu(w["gate"], w["up"], x),
        lambda: moe(k=0), lambda: moe(k=13), lambda: moe(k=33), lambda: moe(router=w["router"][:, :511]), lambda: moe(router=None),
        lambda: moe(down=w["ffn_down"]), lambda: moe(down=w["gate"]), lambda: moe(ids=torch.zeros(2, 3, device="cuda")),
        lambda: moe(weights=torch.zeros(2, 2, device="cuda")), lambda: moe(workspace=torch.zeros(64, dtype=torch.uint8, device="cuda")),
        lambda: moe(workspace=torch.zeros(1 << 20, dtype=torch.uint8)), lambda: moe(workspace=torch.zeros(1 << 20, dtype=torch.uint8, device="cuda")[1:]),
        lambda: moe(out=x[:, :256]), lambda: moe(out=out, residual=out.half()),
        lambda: rb.W4Matrix(8, np.zeros(34, np.uint8), 1, 32), lambda: rb.W4Matrix(Q4_0, np.zeros(18, np.uint8), 1, 33),
        lambda: rb.W4Matrix(Q4_0, np.zeros(17, np.uint8), 1, 32), lambda: rb.W4Matrix(MXFP4, np.full(17, 255, np.uint8), 1, 32),
        lambda: rb.W4Matrix(Q4_0, np.zeros(18 * 300, np.uint8), 1, 32, n_expert=300), lambda: rb.W4Matrix(Q4_0, np.zeros(18, np.uint8), -1, 32),
    ]
    for i, call in enumerate(bad):
        with pytest.raises(rb.InvalidArgument):
            call()
            pytest.fail(f"call {i} was not refused")
    torch.cuda.synchronize()
    assert (out == 7.0).all() and (x == 0).all()
