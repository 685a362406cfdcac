"""The tolerances of test_gpu_w4_precision.py see the mistakes they are there for: each is planted in the definition, in float64."""
import numpy as np
import pytest

from test_gpu_w4 import MXFP4, Q4_0, decode, stored_rows
from w4_precision import DENSE, EXACT, LAYERS, allowed, layer64, layer_inputs, relative, sparse_integers, unit_rows


def bf16(x):
    u = x.astype(np.float32).view(np.uint32)
    return ((u + 0x7FFF + ((u >> 16) & 1)) & 0xFFFF0000).astype(np.uint32).view(np.float32).astype(np.float64)


def eleven_bits(x):
    """The hi parts alone: every row's largest magnitude brought into [2^13, 2^14), as f16."""
    up = np.exp2(13 - np.floor(np.log2(np.abs(x).max(1, keepdims=True))))
    return (x * up).astype(np.float16).astype(np.float64) / up


def without_a_group(x):
    """The first group of 32 columns in which every token has something, or each token's own first one, is missing."""
    y = x.copy()
    for t in range(len(x)):
        k = np.flatnonzero(x[t])[0] // 32 * 32
        y[t, k:k + 32] = 0
    return y


@pytest.mark.parametrize("kind,n_in,act", EXACT)
def test_exact_cases_see_every_mistake(kind, n_in, act):
    rng = np.random.default_rng(n_in + kind)
    w = decode(kind, unit_rows(rng, kind, 5, n_in))[0]
    x = sparse_integers(rng, 3, n_in, act)
    want = x @ w.T
    # sums in f32, in whatever order, are the same numbers
    products = (w[:, None, :] * x[None]).astype(np.float32)
    for order in (products, products[..., ::-1]):
        assert np.array_equal(np.add.accumulate(order, axis=2)[..., -1].T, want)
    wrong = [without_a_group(x), np.roll(x, 1, 1)]
    if act == "f32":
        wrong += [bf16(x), eleven_bits(x)]
    for bad in wrong:
        assert (bad @ w.T != want).any(1).all()


@pytest.mark.parametrize("kind,n_in", DENSE)
def test_dense_cases_see_lost_parts_and_columns(kind, n_in):
    rng = np.random.default_rng(n_in + kind)
    w = decode(kind, stored_rows(rng, kind, 300, n_in, scale_spread=1))[0]
    x = rng.normal(0, 1, (3, n_in))
    want = x @ w.T
    for op in ("matvec", "glu"):
        limit = allowed(op, n_in)
        assert relative(x.astype(np.float32).astype(np.float64) @ w.T, want) < limit / 8
        for bad in (bf16(x), eleven_bits(x), without_a_group(x)):
            assert relative(bad @ w.T, want) > 8 * limit
    # products that lost ten of an f32's bits before they were added: 1.6e-6 of the result
    assert 1.6e-6 > 1.6 * allowed("matvec", n_in)


@pytest.mark.parametrize("kind,d,ff,tokens", LAYERS)
def test_layers_of_long_rows_see_lost_parts_and_columns(kind, d, ff, tokens):
    _, experts, x = layer_inputs(kind, d, ff, tokens)
    x = x[:2]
    want, limit = layer64(experts, x), allowed("moe", d, ff)
    assert np.isfinite(want).all()

    def short(h, n):
        h = h.copy()
        h[:, -n:] = 0
        return h

    wrong = [np.zeros_like(want), layer64(experts, bf16(x)), layer64(experts, eleven_bits(x)), layer64(experts, without_a_group(x)),
             layer64(experts, x, hidden=lambda h: short(h, 32)), layer64(experts, x, hidden=eleven_bits)]
    for i, y in enumerate(wrong):
        assert relative(y, want) > 8 * limit, (i, relative(y, want))
