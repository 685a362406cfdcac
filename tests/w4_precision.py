"""Inputs, definitions in float64 and tolerances for the precision of the products with 4-bit weights, shared by the GPU tests and by
the CPU test that plants mistakes in the definitions.

Exact cases. Activations are odd integers times a power of two, and at most one of a 32-column group and MOST of a row are not zero; block scales
are 1 or -1. All products and all their sums in any order and grouping are then integers times one power of two: w x is at most 8 * 4095 in
steps of 1 (Q4_0, whose nibbles alone reach 15 * 4095) or 12 * 4095 in steps of 1/2 (MXFP4), MOST = 256 of them stay below 2^24, so f32 holds each. f32
activations have twelve bits, one more than an f16 part holds. The result has to be equal, whatever the length of the row.

Dense cases: the norm of a token's error over the norm of its result. In units of 2^-24 of the root of the sum of the squared
products (Q4_0: |q| and |8 - q| are 1.9 and 1 on that scale): the activations' two parts lose 1.2 x 1.9 = 2; a group's chain of two to four matrix
instructions adds sums of up to 1.7 of it, each step rounding 17 addends down by half a unit, sqrt(17) / 2 x 1.7 x 2 = 7; adding n_in / 32 groups
in runs of at least 1/8 of them gives 0.6 x n_in / (32 * 8) x sqrt(8) / sqrt(2 n_in / 32): 5 at 14336 columns. In squares 9, doubled for inputs less even than
that: 2^-20 is 16. A row of 262144 columns adds 20 in the last term: 2^-19. RMSNorm's factor adds 2. The gated pair a -> silu(a) b passes errors of a and b on with
1.8 and 1 times the size they have for values of a around 1, and an expert layer's down product adds its own: 2.3 of a product's error in squares, 2^-19 (2^-18 for long rows).
"""
import numpy as np

from test_gpu_w4 import MXFP4, Q4_0, decode, silu64, stored_rows

MOST = 256
PRODUCT, PAIR = 2.0 ** -20, 2.0 ** -19
LONG = 2.0                                  # times as much for rows above 14336 columns
LARGEST = {"f32": 4095, "f16": 2047, "bf16": 255}
EXACT = [(kind, n_in, act) for kind in (Q4_0, MXFP4) for n_in in (32, 992, 14336, 262144) for act in ("f32", "f16", "bf16")]
EXACT_TOKENS = (1, 2, 3, 4, 5, 8, 9, 16)
DENSE = [(kind, n_in) for kind in (Q4_0, MXFP4) for n_in in (256, 4096, 14336)]
LAYERS = [(Q4_0, 65536, 64, 16), (MXFP4, 65536, 64, 3), (MXFP4, 262144, 32, 16), (Q4_0, 262144, 32, 1), (Q4_0, 64, 65536, 16), (MXFP4, 1024, 2048, 5)]


def unit_rows(rng, kind, rows, n_in):
    """Stored rows of random nibbles with block scales 1 and, for Q4_0, -1."""
    raw = stored_rows(rng, kind, rows, n_in).reshape(rows, n_in // 32, -1)
    if kind == Q4_0:
        raw[:, :, 0], raw[:, :, 1] = 0, rng.choice(np.array([0x3C, 0xBC], np.uint8), raw.shape[:2])
    else:
        raw[:, :, 0] = 127
    return raw.reshape(rows, -1)


def sparse_integers(rng, tokens, n_in, act, shift=0, exponent=None):
    """Activations of an exact case, float64. Sixteen tokens together have every group (of 262144 columns: with shifts 0 and 1)."""
    x = np.zeros((tokens, n_in))
    groups, top = n_in // 32, LARGEST[act]
    apart = -(-groups // MOST)
    for t in range(tokens):
        g = np.arange((t * apart // 16 + shift) % apart, groups, apart)
        k = g * 32 + (5 * t + 7 * g + 11 * shift) % 32
        x[t, k] = (2 * rng.integers(top // 4, (top + 1) // 2, k.size) + 1) * rng.choice([-1.0, 1.0], k.size)
    assert (x != 0).sum(1).max() <= MOST and np.abs(x).max() <= top
    return x * np.exp2(rng.integers(-10, 5, (tokens, 1)) if exponent is None else exponent)


def relative(y, want):
    """The largest of the tokens' error norms over their results' norms."""
    return float((np.linalg.norm(y - want, axis=1) / np.linalg.norm(want, axis=1)).max())


def allowed(op, n_in, width=0):
    return (PRODUCT if op == "matvec" else PAIR) * (LONG if max(n_in, width) > 14336 else 1)


def layer_inputs(kind, d, ff, tokens):
    """Two experts, both used, and activations of an exact case: a zero router gives each the weight 1 / 2 exactly. (stored banks, decoded experts, x)"""
    rng = np.random.default_rng(d + 3 * ff + tokens + kind)
    raws = [[unit_rows(rng, kind, n_out, n_in) for _ in range(2)] for n_out, n_in in ((ff, d), (ff, d), (d, ff))]
    few = min(MOST, d // 32)
    experts = [[decode(kind, bank[e])[0].astype(np.float32) for bank in raws] for e in range(2)]        # exact: small integers and halves
    return raws, experts, sparse_integers(rng, tokens, d, "f32", exponent=-13.0 - np.round(np.log2(few) / 2))


def layer64(experts, x, hidden=lambda h: h):
    y = 0
    for gate, up, down in experts:
        y = y + hidden(0.5 * silu64(x @ gate.T.astype(np.float64)) * (x @ up.T.astype(np.float64))) @ down.T.astype(np.float64)
    return y
