"""Products with 4-bit weights for few tokens against their definition in float64.

Tolerance of an f32 result, derived before the first run: with A = sum_k |w'_k| |x_k| (w' = |w| + 8 |d| for Q4_0, whose offset -8 d
enters as a separate term, |w| for MXFP4) the activations' split loses 2^-22, a group's tensor-core chain adds four
terms whose alignment may drop 2^-23 each per product (32 products), and the group sums and partial sums are added one after another, at most
n_in / 32 + 64 + 8 additions of 2^-24: |error| <= (2^-22 + 36 * 2^-23 + (n_in / 32 + 72) * 2^-24) A. The RMSNorm multiplies by
factors with a relative error of 2^-21 (its sum of squares: n_in additions of positive terms in blocks of at most n_in / 256 + 64). A
result of 16 bits adds half a step of its type.
"""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

Q4_0, MXFP4 = 2, 39
E2M1 = np.array([0, 0.5, 1, 1.5, 2, 3, 4, 6], dtype=np.float64)


def stored_rows(rng, kind, rows, n_in, scale_spread=3):
    """Random stored rows (uint8 [rows, bytes]): every nibble and scales over some powers of two, of both signs for Q4_0."""
    blocks = n_in // 32
    quants = rng.integers(0, 256, (rows, blocks, 16), dtype=np.uint8)
    if kind == Q4_0:
        d = (rng.choice([-1.0, 1.0], (rows, blocks)) * np.exp2(rng.uniform(-scale_spread, scale_spread, (rows, blocks)) - 6)).astype(np.float16)
        head = d.view(np.uint8).reshape(rows, blocks, 2)
    else:
        head = rng.integers(127 - 2 * scale_spread - 6, 127 - 6, (rows, blocks, 1), dtype=np.uint8)
    return np.concatenate([head, quants], 2).reshape(rows, -1)


def decode(kind, raw):
    """(weights, magnitudes A is taken over), float64."""
    rows = raw.shape[0]
    b = raw.reshape(rows, -1, 18 if kind == Q4_0 else 17)
    if kind == Q4_0:
        d = b[:, :, :2].copy().view(np.float16).astype(np.float64)
        q = b[:, :, 2:]
        v = np.concatenate([q & 15, q >> 4], 2).astype(np.float64) - 8
        extra = 8 * np.abs(d)
    else:
        d = np.exp2(b[:, :, :1].astype(np.float64) - 127)
        q = b[:, :, 1:]
        n = np.concatenate([q & 15, q >> 4], 2)
        v = E2M1[n & 7] * np.where(n & 8, -1.0, 1.0)
        extra = 0.0
    return (v * d).reshape(rows, -1), (np.abs(v * d) + extra).reshape(rows, -1)


def dtype_of(torch, name):
    return {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}[name]


def half_step(torch, name):
    return 0.0 if name == "f32" else torch.finfo(dtype_of(torch, name)).eps / 2


def f32_bound(n_in):
    return 2.0 ** -22 + 36 * 2.0 ** -23 + (n_in / 32 + 72) * 2.0 ** -24


def normed(x, norm, eps):
    return x if norm is None else x / np.sqrt((x ** 2).mean(1, keepdims=True) + eps) * norm


def activations(rng, torch, tokens, n_in, act):
    """Tokens of different magnitude with outliers; what the kernel sees, and its values in float64."""
    x = rng.normal(0, 1, (tokens, n_in)) * np.exp2(rng.uniform(-8, 8, (tokens, 1))) * np.where(rng.random((1, n_in)) < 0.01, 30.0, 1.0)
    t = torch.tensor(x, dtype=torch.float32).to(dtype_of(torch, act)).cuda()
    return t, t.double().cpu().numpy()


SIZES = [
    # n_out, n_in: one block and one row, odd rows, a half step at the end, one step per CTA of a cluster, many row tiles
    (1, 32), (15, 32), (17, 64), (33, 96), (688, 256), (1377, 992), (64, 4096), (129, 2880), (5000, 160), (96, 14336), (4096, 4096), (70001, 64),
]


@pytest.mark.parametrize("kind", [Q4_0, MXFP4])
@pytest.mark.parametrize("n_out,n_in", SIZES)
def test_matvec_against_float64(rb, kind, n_out, n_in):
    import torch

    rng = np.random.default_rng(n_out * 1000 + n_in + kind)
    raw = stored_rows(rng, kind, n_out, n_in)
    w, mag = decode(kind, raw)
    m = rb.W4Matrix(kind, raw, n_out, n_in)
    for tokens, act in ((1, "f32"), (2, "bf16"), (3, "f32"), (4, "f32"), (5, "f16"), (7, "f32"), (8, "bf16"), (9, "f32"), (16, "f32"), (16, "f16"), (19, "f32")):
        x, x64 = activations(rng, torch, tokens, n_in, act)
        y = rb.w4_matvec(m, x)
        assert y.dtype == x.dtype and tuple(y.shape) == (tokens, n_out)
        want = x64 @ w.T
        bound = f32_bound(n_in) * (np.abs(x64) @ mag.T) + half_step(torch, act) * np.abs(want) + (2.0 ** -25 if act == "f16" else 0)
        if act == "f16":    # what f16 cannot hold is infinite
            over = np.abs(want) > 65000
            want, bound = np.where(over, 0, want), np.where(over, np.inf, bound)
        got = y.double().cpu().numpy()
        error = np.where(np.isinf(bound), 0, np.abs(np.where(np.isinf(bound), 0, got) - want) - bound)
        assert error.max() <= 0, (tokens, act, float(error.max()), np.unravel_index(error.argmax(), error.shape))
    m.close()


@pytest.mark.parametrize("kind", [Q4_0, MXFP4])
@pytest.mark.parametrize("n_out,n_in,tokens", [(48, 64, 1), (97, 992, 3), (640, 4096, 6), (31, 2880, 13)])
def test_norm_bias_and_residual(rb, kind, n_out, n_in, tokens):
    import torch

    rng = np.random.default_rng(n_out + n_in)
    raw = stored_rows(rng, kind, n_out, n_in)
    w, mag = decode(kind, raw)
    m = rb.W4Matrix(kind, raw, n_out, n_in)
    norm = rng.normal(1, 0.2, n_in).astype(np.float32)
    bias = rng.normal(0, 1, n_out).astype(np.float32)
    for act in ("f32", "bf16"):
        x, x64 = activations(rng, torch, tokens, n_in, act)
        res, res64 = activations(rng, torch, tokens, n_out, act)
        y = rb.w4_matvec(m, x, norm=torch.tensor(norm).cuda(), eps=1e-5, bias=torch.tensor(bias).cuda(), residual=res)
        xn = normed(x64, norm.astype(np.float64), 1e-5)
        want = xn @ w.T + bias + res64
        bound = (f32_bound(n_in) + 2.0 ** -21) * (np.abs(xn) @ mag.T) + 2.0 ** -22 * (np.abs(want) + np.abs(bias) + np.abs(res64)) + half_step(torch, act) * np.abs(want)
        assert (np.abs(y.double().cpu().numpy() - want) - bound).max() <= 0
        # in place
        again = rb.w4_matvec(m, x, norm=torch.tensor(norm).cuda(), eps=1e-5, bias=torch.tensor(bias).cuda(), residual=res, out=res)
        assert again.data_ptr() == res.data_ptr() and torch.equal(res, y)


def silu64(a):
    return a / (1 + np.exp(-a))


@pytest.mark.parametrize("kind", [Q4_0, MXFP4])
@pytest.mark.parametrize("n_out,n_in,tokens,act", [(1, 32, 1, "f32"), (688, 256, 2, "f32"), (1377, 992, 5, "bf16"), (130, 4096, 8, "f32"), (4096, 1024, 16, "f32"), (77, 160, 21, "f16")])
def test_glu_against_float64(rb, kind, n_out, n_in, tokens, act):
    import torch

    rng = np.random.default_rng(n_out + 7 * n_in)
    raws = [stored_rows(rng, kind, n_out, n_in, scale_spread=1) for _ in range(2)]
    (wg, mg), (wu, mu) = (decode(kind, r) for r in raws)
    gate, up = (rb.W4Matrix(kind, r, n_out, n_in) for r in raws)
    norm = rng.normal(1, 0.2, n_in).astype(np.float32)
    x, x64 = activations(rng, torch, tokens, n_in, act)
    y = rb.w4_glu(gate, up, x, norm=torch.tensor(norm).cuda()).double().cpu().numpy()
    xn = normed(x64, norm.astype(np.float64), 1e-5)
    a, b = xn @ wg.T, xn @ wu.T
    ea, eb = ((f32_bound(n_in) + 2.0 ** -21) * (np.abs(xn) @ m.T) for m in (mg, mu))
    want = silu64(a) * b
    # |silu'| <= 1.1; silu itself is within 2^-20 (expf and a division), its exponent's argument error is in ea
    bound = 1.1 * ea * np.abs(b) + np.abs(silu64(a)) * eb + 1.1 * ea * eb + 2.0 ** -20 * np.abs(want) + half_step(torch, act) * np.abs(want) + (2.0 ** -25 if act == "f16" else 1e-37)
    over = np.abs(want) > (65000 if act == "f16" else np.inf)
    assert np.where(over, 0, np.abs(np.where(over, 0, y - want)) - bound).max() <= 0


def route64(x, router, k, normalise):
    """Chosen experts (likeliest first, ties to the lowest), their weights, and the probability gap that decided the choice."""
    logits = x @ router.T
    p = np.exp(logits - logits.max(1, keepdims=True))
    p /= p.sum(1, keepdims=True)
    order = np.argsort(-p, axis=1, kind="stable")
    ranked = np.take_along_axis(p, order, 1)
    gap = np.full(len(p), np.inf)
    if p.shape[1] > 1:
        top = ranked[:, : k + 1]
        gap = ((top[:, :-1] - top[:, 1:]) / top[:, :-1]).min(1)
    return order, p, gap


def moe64(x, p, ids, gate, up, down, normalise):
    """The layer's sum over experts for given choices, with a bound on an f32 kernel's error. gate, up, down: lists of decode() pairs."""
    tokens, k = ids.shape
    d = down[0][0].shape[0]
    y, bound = np.zeros((tokens, d)), np.zeros((tokens, d))
    n_in, ff = x.shape[1], down[0][0].shape[1]
    for t in range(tokens):
        w = p[t, ids[t]]
        if normalise:
            w = w / w.sum()
        for j, e in enumerate(ids[t]):
            a, b = gate[e][0] @ x[t], up[e][0] @ x[t]
            ea, eb = ((f32_bound(n_in) + 2.0 ** -21) * (m[e][1] @ np.abs(x[t])) for m in (gate, up))
            h = silu64(a) * b
            eh = 1.1 * ea * np.abs(b) + np.abs(silu64(a)) * eb + 1.1 * ea * eb + 2.0 ** -20 * np.abs(h)
            y[t] += w[j] * (down[e][0] @ h)
            bound[t] += w[j] * (down[e][1] @ (eh + (f32_bound(ff) + 2.0 ** -20) * np.abs(h)))
    return y, bound


def moe_inputs(rng, torch, kind, kind_down, E, d, ff, tokens, act):
    raws = [[stored_rows(rng, kd, n_out, n_in, scale_spread=1) for _ in range(E)] for kd, n_out, n_in in ((kind, ff, d), (kind, ff, d), (kind_down, d, ff))]
    x = torch.tensor(rng.normal(0, 1, (tokens, d)), dtype=torch.float32).to(dtype_of(torch, act)).cuda()
    router = rng.normal(0, 2 / np.sqrt(d), (E, d)).astype(np.float32)
    return raws, x, router


MOE = [
    # kind, kind of down, experts, used, hidden, ff, tokens, act
    (MXFP4, MXFP4, 1, 1, 32, 32, 1, "f32"), (Q4_0, Q4_0, 2, 1, 64, 96, 3, "f32"), (MXFP4, MXFP4, 8, 2, 256, 160, 5, "bf16"),
    (Q4_0, MXFP4, 32, 4, 320, 288, 16, "f32"), (MXFP4, Q4_0, 33, 32, 96, 64, 9, "f32"), (Q4_0, Q4_0, 256, 8, 128, 64, 16, "f16"),
    (MXFP4, MXFP4, 4, 2, 2880, 2880, 2, "f32"), (Q4_0, Q4_0, 3, 3, 1056, 2048, 21, "f32"), (MXFP4, MXFP4, 6, 2, 64, 4096, 16, "bf16"),
    (Q4_0, Q4_0, 2, 2, 4096, 64, 16, "f32"),
]


@pytest.mark.parametrize("kind,kind_down,E,k,d,ff,tokens,act", MOE)
def test_moe_against_float64(rb, kind, kind_down, E, k, d, ff, tokens, act):
    import torch

    rng = np.random.default_rng(E * 1000 + d + ff + tokens)
    raws, x, router = moe_inputs(rng, torch, kind, kind_down, E, d, ff, tokens, act)
    gate, up = (rb.W4Matrix(kind, np.stack(r), ff, d, n_expert=E) for r in raws[:2])
    down = rb.W4Matrix(kind_down, np.stack(raws[2]), d, ff, n_expert=E)
    decoded = [[decode(kd, r) for r in bank] for kd, bank in ((kind, raws[0]), (kind, raws[1]), (kind_down, raws[2]))]
    norm = rng.normal(1, 0.2, d).astype(np.float32)
    x64 = x.double().cpu().numpy()
    for use_norm, use_residual, normalise in ((False, False, False), (True, True, True)):
        ids = torch.full((tokens, k), -1, dtype=torch.int32, device="cuda")
        weights = torch.full((tokens, k), float("nan"), device="cuda")
        residual = torch.tensor(rng.normal(0, 1, (tokens, d)), dtype=torch.float32).to(x.dtype).cuda() if use_residual else None
        y = rb.w4_moe(torch.tensor(router).cuda(), gate, up, down, x, k, normalise=normalise, norm=torch.tensor(norm).cuda() if use_norm else None,
                      residual=residual, ids=ids, weights=weights)
        xn = normed(x64, norm.astype(np.float64) if use_norm else None, 1e-5)
        order, p, gap = route64(xn, router.astype(np.float64), k, normalise)
        got_ids = ids.cpu().numpy()
        # logits differ by less than 1e-5 (|x| |r| d 2^-24 and the norm's 2^-21): probabilities closer than that may swap places
        clear = gap > 4e-5
        assert np.array_equal(got_ids[clear], order[clear, :k]) and clear.mean() > 0.8
        assert all(len(set(row)) == k for row in got_ids.tolist()) and got_ids.min() >= 0 and got_ids.max() < E
        w = np.take_along_axis(p, got_ids.astype(np.int64), 1)
        w = w / w.sum(1, keepdims=True) if normalise else w
        assert np.abs(weights.double().cpu().numpy() - w).max() <= 4e-5 * w.max()
        want, bound = moe64(xn, p, got_ids, *decoded, normalise)
        total = want + (residual.double().cpu().numpy() if use_residual else 0)
        # a weight's relative error (the logits' error twice, exponentials, sums): 4e-5, on every expert's part
        bound = bound + 4e-5 * expert_parts(xn, p, got_ids, *decoded, normalise)
        bound = bound + 2.0 ** -22 * (np.abs(total) + np.abs(want)) + half_step(torch, act) * np.abs(total)
        error = np.abs(y.double().cpu().numpy() - total)
        assert (error <= bound).all(), float((error / bound).max())


def expert_parts(x, p, ids, gate, up, down, normalise):
    """Sum of the magnitudes of the experts' parts of y: what an error of the routing weights is relative to."""
    out = np.zeros((ids.shape[0], down[0][0].shape[0]))
    for t in range(ids.shape[0]):
        w = p[t, ids[t]] / (p[t, ids[t]].sum() if normalise else 1.0)
        for j, e in enumerate(ids[t]):
            out[t] += w[j] * np.abs(down[e][0] @ (silu64(gate[e][0] @ x[t]) * (up[e][0] @ x[t])))
    return out
