"""How near the products with 4-bit weights come to their definition: integers that f32 holds exactly, and the size of the typical error.

Cases and tolerances are derived in w4_precision.py; test_w4_precision_host.py plants the mistakes that they have to see.
"""
import numpy as np
import pytest

from test_gpu_w4 import decode, dtype_of, normed, route64, silu64, stored_rows
from w4_precision import DENSE, EXACT, EXACT_TOKENS, LAYERS, allowed, layer64, layer_inputs, relative, sparse_integers, unit_rows

pytestmark = pytest.mark.gpu


def cuda(torch, x, act="f32"):
    t = torch.tensor(x, dtype=torch.float32).to(dtype_of(torch, act)).cuda()
    assert np.array_equal(t.double().cpu().numpy(), x)
    return t


@pytest.mark.parametrize("kind,n_in,act", EXACT)
def test_products_of_integers_are_exact(rb, kind, n_in, act):
    import torch

    rng = np.random.default_rng(n_in + kind)
    raw = unit_rows(rng, kind, 40, n_in)
    w = decode(kind, raw)[0]
    m = rb.W4Matrix(kind, raw, 40, n_in)
    for tokens in EXACT_TOKENS:
        for shift in (0, 1) if tokens == 16 else (tokens % 2,):
            x = sparse_integers(rng, tokens, n_in, act, shift)
            y = rb.w4_matvec(m, cuda(torch, x, act), out=torch.empty(tokens, 40, device="cuda")).double().cpu().numpy()
            assert np.array_equal(y, x @ w.T), (tokens, shift, np.argwhere(y != x @ w.T)[:5])


@pytest.mark.parametrize("kind,n_in", DENSE)
def test_typical_error(rb, kind, n_in):
    import torch

    rng = np.random.default_rng(n_in + kind)
    raws = [stored_rows(rng, kind, 600, n_in, scale_spread=1) for _ in range(2)]
    (w, _), (u, _) = (decode(kind, r) for r in raws)
    m, up = (rb.W4Matrix(kind, r, 600, n_in) for r in raws)
    scale = 1 / (w.std() * np.sqrt(n_in))           # the gated pair's values are around 1
    norm = rng.normal(1, 0.2, n_in).astype(np.float32)
    for tokens, act in ((1, "f32"), (1, "bf16"), (3, "f32"), (6, "f16"), (7, "f32"), (16, "f32"), (16, "bf16")):
        x = torch.tensor(rng.normal(0, scale, (tokens, n_in)), dtype=torch.float32).to(dtype_of(torch, act)).cuda()
        x64, new = x.double().cpu().numpy(), lambda: torch.empty(tokens, 600, device="cuda")
        got = relative(rb.w4_matvec(m, x, out=new()).double().cpu().numpy(), x64 @ w.T)
        assert got <= allowed("matvec", n_in), (tokens, act, got)
        got = relative(rb.w4_matvec(m, x, norm=torch.tensor(norm).cuda(), out=new()).double().cpu().numpy(), normed(x64, norm.astype(np.float64), 1e-5) @ w.T)
        assert got <= allowed("matvec", n_in), ("norm", tokens, act, got)
        got = relative(rb.w4_glu(m, up, x, out=new()).double().cpu().numpy(), silu64(x64 @ w.T) * (x64 @ u.T))
        assert got <= allowed("glu", n_in), ("glu", tokens, act, got)


@pytest.mark.parametrize("kind,kind_down,d,ff", [(2, 2, 512, 480), (39, 39, 2880, 704), (2, 39, 4096, 256)])
def test_typical_error_of_an_expert_layer(rb, kind, kind_down, d, ff):
    import torch

    rng = np.random.default_rng(d + ff)
    E, k = 6, 2
    raws = [[stored_rows(rng, kd, n_out, n_in, scale_spread=1) for _ in range(E)] for kd, n_out, n_in in ((kind, ff, d), (kind, ff, d), (kind_down, d, ff))]
    banks = [[decode(kd, r)[0] for r in bank] for kd, bank in zip((kind, kind, kind_down), raws)]
    gate, up = (rb.W4Matrix(kind, np.stack(r), ff, d, n_expert=E) for r in raws[:2])
    down = rb.W4Matrix(kind_down, np.stack(raws[2]), d, ff, n_expert=E)
    scale = 1 / (banks[0][0].std() * np.sqrt(d))
    router = torch.tensor(rng.normal(0, 1 / (scale * np.sqrt(d)), (E, d)), dtype=torch.float32)
    for tokens, act in ((1, "f32"), (4, "bf16"), (5, "f32"), (16, "f32"), (16, "f16")):
        x = torch.tensor(rng.normal(0, scale, (tokens, d)), dtype=torch.float32).to(dtype_of(torch, act)).cuda()
        ids = torch.zeros(tokens, k, dtype=torch.int32, device="cuda")
        y = rb.w4_moe(router.cuda(), gate, up, down, x, k, normalise=True, ids=ids, out=torch.empty(tokens, d, device="cuda")).double().cpu().numpy()
        x64 = x.double().cpu().numpy()
        order, p, gap = route64(x64, router.double().numpy(), k, True)
        chosen = ids.cpu().numpy().astype(np.int64)
        clear = gap > 4e-5
        assert np.array_equal(chosen[clear], order[clear, :k])
        want = np.zeros_like(y)
        for t in range(tokens):
            w = p[t, chosen[t]] / p[t, chosen[t]].sum()
            for j, e in enumerate(chosen[t]):
                want[t] += w[j] * (banks[2][e] @ (silu64(banks[0][e] @ x64[t]) * (banks[1][e] @ x64[t])))
        got = relative(y, want)
        assert got <= allowed("moe", d, ff), (tokens, act, got)


@pytest.mark.parametrize("kind,d,ff,tokens", LAYERS)
def test_expert_layers_of_long_rows(rb, kind, d, ff, tokens):
    import torch

    raws, experts, x = layer_inputs(kind, d, ff, tokens)
    gate, up = (rb.W4Matrix(kind, np.stack(r), ff, d, n_expert=2) for r in raws[:2])
    down = rb.W4Matrix(kind, np.stack(raws[2]), d, ff, n_expert=2)
    y = rb.w4_moe(torch.zeros(2, d, device="cuda"), gate, up, down, cuda(torch, x), 2).double().cpu().numpy()
    got = relative(y, layer64(experts, x))
    assert got <= allowed("moe", d, ff), got
