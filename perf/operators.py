"""Performance cases of the products with 4-bit weights for few tokens: `w4_matvec`, `w4_glu` and `w4_moe`.

A case is one call as a decode step of one to sixteen tokens makes it: a projection (with the RMSNorm before it or the residual
after it), the gated pair of a dense FFN, or a whole mixture-of-experts layer. Shapes are those of the benchmark's workloads (the
tiny decoder, the Llama-3-8B shape, the 20B-class mixture-of-experts shape) and generic ones; weights are random normals in
the stored block formats Q4_0 and MXFP4, activations random normals with per-token magnitudes.

Fields of a case:
  op       "matvec", "glu" or "moe"               type     "q4_0" or "mxfp4": how the weights are stored
  tokens   tokens of the call                     act      element type of x and y: "f32", "f16" or "bf16"
  n_in, n_out   columns and rows of the matrix (of gate and up for "glu"; hidden size and expert width for "moe")
  norm     RMSNorm in front                       residual, bias   what is added to the product
  experts, used, normalise   "moe": experts, experts per token, whether the chosen probabilities are divided by their sum
"""
import math

import torch

own = False

ACT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
BLOCK_BYTES = {"q4_0": 18, "mxfp4": 17}
GGML_TYPE = {"q4_0": 2, "mxfp4": 39}
EPS = 1e-5
E2M1 = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]


def _case(name, op, type, tokens, n_in, n_out, act="f32", norm=False, residual=False, bias=False, experts=0, used=0, normalise=False):
    return dict(name=name, op=op, type=type, tokens=tokens, n_in=n_in, n_out=n_out, act=act, norm=norm, residual=residual, bias=bias,
                experts=experts, used=used, normalise=normalise)


def listed():
    return [
        # the smallest call: the tiny decoder's up projection for one token, where the launch is everything
        _case("tiny_up_1", "matvec", "q4_0", 1, 256, 688),
        # one chat user of an 8B model: the stacked q, k, v projection with its norm (and the biases some models have)
        _case("qkv_1", "matvec", "q4_0", 1, 4096, 6144, norm=True, bias=True),
        # the same user's down projection, added to the residual stream
        _case("down_1", "matvec", "q4_0", 1, 14336, 4096, residual=True),
        # a lightly loaded server: the down projection of eleven users in half precision
        _case("down_11_f16", "matvec", "q4_0", 11, 14336, 4096, act="f16", residual=True),
        # the vocabulary projection of one user
        _case("vocab_1", "matvec", "q4_0", 1, 4096, 128256, norm=True),
        # the vocabulary projection of the 20B-class shape for a full small step
        _case("vocab_16_bf16", "matvec", "mxfp4", 16, 2880, 201088, act="bf16"),
        # the dense FFN's first half, one user and a full small step
        _case("ffn_1", "glu", "q4_0", 1, 4096, 14336, norm=True),
        _case("ffn_16", "glu", "q4_0", 16, 4096, 14336, norm=True),
        # a small ragged one: rows that are no multiple of a tile, five tokens
        _case("ffn_odd_5", "glu", "mxfp4", 5, 992, 1377, act="bf16"),
        # the 20B-class expert layer: one user, and a full small step that reaches most experts
        _case("moe_20b_1", "moe", "mxfp4", 1, 2880, 2880, norm=True, residual=True, experts=32, used=4),
        _case("moe_20b_16", "moe", "mxfp4", 16, 2880, 2880, residual=True, experts=32, used=4),
        # many small experts, a few users in half precision
        _case("moe_64x8_6", "moe", "q4_0", 6, 2048, 1024, act="bf16", experts=64, used=8, normalise=True),
    ]


def draw(rng):
    """One more case: any operator, type and token count; rows, columns and experts spread over their logarithms."""
    def log_int(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    def columns(lo, hi):
        return 32 * log_int(lo // 32, hi // 32)

    op = rng.choice(["matvec", "matvec", "glu", "moe", "moe"])
    common = dict(op=op, type=rng.choice(["q4_0", "mxfp4"]), tokens=log_int(1, 16), act=rng.choice(["f32", "f32", "f16", "bf16"]),
                  norm=rng.random() < 0.5, residual=False, bias=False, experts=0, used=0, normalise=False)
    if op == "moe":
        d, ff, experts = columns(64, 4096), columns(64, 4096), log_int(2, 128)
        while experts * d * ff * 3 > 800_000_000:
            experts = max(2, experts // 2)
            if experts == 2:
                break
        used = min(experts, log_int(1, 8))
        return dict(common, n_in=d, n_out=ff, residual=rng.random() < 0.7, experts=experts, used=used, normalise=rng.random() < 0.5)
    n_in = columns(64, 14336)
    n_out = log_int(1, min(150_000, (500_000_000 if op == "matvec" else 250_000_000) // n_in))
    if op == "matvec":
        common.update(residual=rng.random() < 0.5, bias=rng.random() < 0.3)
    return dict(common, n_in=n_in, n_out=n_out)


# ---- inputs


def _quantise(w, type):
    """[rows, n_in] floats -> the stored rows, uint8 [rows, n_in / 32 * block bytes]."""
    rows, n_in = w.shape
    v = w.view(rows, n_in // 32, 32)
    if type == "q4_0":
        top = v.gather(2, v.abs().argmax(2, keepdim=True))
        d = (top / -8).half()
        df = d.float()
        inverse = torch.where(df != 0, 1 / df, torch.zeros_like(df))
        q = (v * inverse + 8.5).floor_().clamp_(0, 15).to(torch.uint8)
        head = d.view(torch.uint8)
    else:
        top = v.abs().amax(2, keepdim=True)
        e = torch.ceil(torch.log2(top / 6)).clamp_(-100, 100)
        z = v * torch.exp2(-e)
        edges = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0], device=w.device)
        q = torch.bucketize(z.abs(), edges).to(torch.uint8) | (z < 0).to(torch.uint8) << 3
        head = (e + 127).to(torch.uint8)
    packed = q[..., :16] | q[..., 16:] << 4
    return torch.cat([head, packed], 2).view(rows, -1)


def _weights(gen, rows, n_in, type, std):
    out = torch.empty(rows, n_in // 32 * BLOCK_BYTES[type], dtype=torch.uint8, device="cuda")
    step = max(1, (1 << 26) // n_in)
    for r in range(0, rows, step):
        n = min(step, rows - r)
        out[r:r + n] = _quantise(torch.randn(n, n_in, device="cuda", generator=gen) * std, type)
    return out


def _data(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    T, n_in, n_out, act = case["tokens"], case["n_in"], case["n_out"], ACT[case["act"]]
    randn = lambda *shape: torch.randn(*shape, device="cuda", generator=gen)
    s = {"case": case}
    # tokens differ in magnitude, and single features stand out, as in a residual stream
    magnitude = torch.exp(randn(T, 1) * 0.5)
    outlier = torch.where(randn(1, n_in).abs() > 3, 10.0, 1.0)
    s["x"] = (randn(T, n_in) * magnitude * outlier).to(act)
    s["norm"] = 1 + 0.1 * randn(n_in) if case["norm"] else None
    std = 1 / math.sqrt(n_in)
    if case["op"] == "matvec":
        s["w"] = _weights(gen, n_out, n_in, case["type"], std)
    elif case["op"] == "glu":
        s["gate"] = _weights(gen, n_out, n_in, case["type"], std)
        s["up"] = _weights(gen, n_out, n_in, case["type"], std)
    else:
        E = case["experts"]
        s["router"] = randn(E, n_in) * std
        s["gate"] = _weights(gen, E * n_out, n_in, case["type"], std)
        s["up"] = _weights(gen, E * n_out, n_in, case["type"], std)
        s["down"] = _weights(gen, E * n_in, n_out, case["type"], 1 / math.sqrt(n_out))
    width = n_in if case["op"] == "moe" else n_out
    s["residual"] = randn(T, width).to(act) if case["residual"] else None
    s["bias"] = 0.1 * randn(n_out) if case["bias"] else None
    return s


def prepare(case, seed):
    s = _data(case, seed)
    if own:
        import retrograd_b200 as rb

        kind, n_in, n_out, E = GGML_TYPE[case["type"]], case["n_in"], case["n_out"], max(1, case["experts"])
        for key in ("w", "gate", "up"):
            if key in s:
                s[key] = rb.W4Matrix(kind, s[key], n_out, n_in, n_expert=E)
        if "down" in s:
            s["down"] = rb.W4Matrix(kind, s["down"], n_in, n_out, n_expert=E)
    return s


# ---- the operators


def _dequantise(rows, type):
    """Stored rows uint8 [..., blocks * bytes] -> float32 [..., blocks * 32]."""
    b = rows.view(*rows.shape[:-1], -1, BLOCK_BYTES[type])
    if type == "q4_0":
        scale = b[..., :2].contiguous().view(torch.float16).float()
        nibbles = b[..., 2:]
        values = torch.cat([nibbles & 15, nibbles >> 4], -1).float() - 8
    else:
        scale = torch.exp2(b[..., :1].float() - 127)
        nibbles = b[..., 1:]
        table = torch.tensor(E2M1 + [-v for v in E2M1], device=rows.device)
        values = table[torch.cat([nibbles & 15, nibbles >> 4], -1).int()]
    return (values * scale).flatten(-2)


def _plain(s):
    case = s["case"]
    T, act, type = case["tokens"], ACT[case["act"]], case["type"]
    x = s["x"].float()
    if s["norm"] is not None:
        x = x * torch.rsqrt((x * x).mean(1, keepdim=True) + EPS) * s["norm"]
    if case["op"] == "matvec":
        y = x @ _dequantise(s["w"], type).T
        if s["bias"] is not None:
            y = y + s["bias"]
    elif case["op"] == "glu":
        a = x @ _dequantise(s["gate"], type).T
        y = a / (1 + torch.exp(-a)) * (x @ _dequantise(s["up"], type).T)
    else:
        E, k, d, ff = case["experts"], case["used"], case["n_in"], case["n_out"]
        logits = x @ s["router"].T
        p = torch.exp(logits - logits.amax(1, keepdim=True))
        p = p / p.sum(1, keepdim=True)
        weight, chosen = torch.sort(p, dim=1, descending=True, stable=True)
        weight, chosen = weight[:, :k], chosen[:, :k]
        if case["normalise"]:
            weight = weight / weight.sum(1, keepdim=True)
        gate, up, down = s["gate"].view(E, ff, -1), s["up"].view(E, ff, -1), s["down"].view(E, d, -1)
        rows = []
        for t in range(T):
            a = _dequantise(gate[chosen[t]], type) @ x[t]
            h = a / (1 + torch.exp(-a)) * (_dequantise(up[chosen[t]], type) @ x[t])
            rows.append((torch.bmm(_dequantise(down[chosen[t]], type), h.unsqueeze(2)).squeeze(2) * weight[t].unsqueeze(1)).sum(0))
        y = torch.stack(rows)
    if s["residual"] is not None:
        y = y + s["residual"].float()
    return y.to(act)


def run(state):
    if not own:
        return _plain(state)
    import retrograd_b200 as rb

    case = state["case"]
    if case["op"] == "matvec":
        return rb.w4_matvec(state["w"], state["x"], norm=state["norm"], eps=EPS, bias=state["bias"], residual=state["residual"])
    if case["op"] == "glu":
        return rb.w4_glu(state["gate"], state["up"], state["x"], norm=state["norm"], eps=EPS)
    return rb.w4_moe(state["router"], state["gate"], state["up"], state["down"], state["x"], case["used"], norm=state["norm"], eps=EPS,
                     normalise=case["normalise"], residual=state["residual"])


# ---- what a pass cannot do without, and its value in 64 bits


def work(case):
    T, n_in, n_out = case["tokens"], case["n_in"], case["n_out"]
    act = 4 if case["act"] == "f32" else 2
    matrix = n_in // 32 * BLOCK_BYTES[case["type"]] * n_out
    n_bytes = T * n_in * act + (4 * n_in if case["norm"] else 0)
    if case["op"] == "matvec":
        n_bytes += matrix + T * n_out * act * (2 if case["residual"] else 1) + (4 * n_out if case["bias"] else 0)
        flops = 2 * T * n_in * n_out
    elif case["op"] == "glu":
        n_bytes += 2 * matrix + T * n_out * act
        flops = 4 * T * n_in * n_out
    else:
        E, k = case["experts"], case["used"]
        reached = E * (1 - (1 - k / E) ** T)       # experts that T tokens with independent choices reach, on average
        n_bytes += 3 * matrix * reached + 4 * E * n_in + T * n_in * act * (2 if case["residual"] else 1)
        flops = 6 * T * k * n_in * n_out + 2 * T * E * n_in
    return {"bytes": int(n_bytes), "flops": int(flops)}


def _decode64(rows, type):
    """The stored rows as float64, element by element from the formats' definitions."""
    n = rows.shape[0]
    size = BLOCK_BYTES[type]
    blocks = rows.reshape(n, rows.shape[1] // size, size)
    out = torch.empty(n, blocks.shape[1], 32, dtype=torch.float64, device=rows.device)
    if type == "q4_0":
        raw = blocks[:, :, 0].to(torch.int32) + 256 * blocks[:, :, 1].to(torch.int32)
        sign = 1.0 - 2.0 * (raw // 32768).double()
        exponent, fraction = (raw // 1024) % 32, (raw % 1024).double()
        normal = (1 + fraction / 1024) * torch.pow(2.0, (exponent - 15).double())
        scale = sign * torch.where(exponent == 0, fraction * 2.0 ** -24, normal)
        code = blocks[:, :, 2:].to(torch.int32)
        out[:, :, :16] = (code % 16 - 8).double()
        out[:, :, 16:] = (code // 16 - 8).double()
    else:
        scale = torch.pow(2.0, blocks[:, :, 0].double() - 127)
        code = blocks[:, :, 1:].to(torch.int32)
        for half, nibble in enumerate((code % 16, code // 16)):
            exponent, fraction = (nibble // 2) % 4, (nibble % 2).double()
            size_ = torch.where(exponent == 0, fraction / 2, (1 + fraction / 2) * torch.pow(2.0, (exponent - 1).double()))
            out[:, :, 16 * half:16 * half + 16] = torch.where(nibble >= 8, -size_, size_)
    return (out * scale[:, :, None]).reshape(n, -1)


def _product64(rows, type, x):
    step = max(1, (1 << 25) // x.shape[1])
    return torch.cat([x @ _decode64(rows[r:r + step], type).T for r in range(0, rows.shape[0], step)], 1)


def exact(case, seed):
    s = _data(case, seed)
    type = case["type"]
    x = s["x"].double()
    if s["norm"] is not None:
        x = x / torch.sqrt((x ** 2).sum(1, keepdim=True) / case["n_in"] + EPS) * s["norm"].double()
    if case["op"] == "matvec":
        y = _product64(s["w"], type, x)
        if s["bias"] is not None:
            y += s["bias"].double()
    elif case["op"] == "glu":
        a = _product64(s["gate"], type, x)
        y = a * torch.sigmoid(a) * _product64(s["up"], type, x)
    else:
        E, k, d, ff = case["experts"], case["used"], case["n_in"], case["n_out"]
        p = torch.softmax(x @ s["router"].double().T, 1).cpu().tolist()
        y = torch.zeros(case["tokens"], d, dtype=torch.float64, device="cuda")
        for t, row in enumerate(p):
            chosen = sorted(range(E), key=lambda e: (-row[e], e))[:k]
            total = sum(row[e] for e in chosen) if case["normalise"] else 1.0
            for e in chosen:
                a = _product64(s["gate"][e * ff:(e + 1) * ff], type, x[t:t + 1])
                h = a * torch.sigmoid(a) * _product64(s["up"][e * ff:(e + 1) * ff], type, x[t:t + 1])
                y[t] += row[e] / total * _product64(s["down"][e * d:(e + 1) * d], type, h)[0]
    if s["residual"] is not None:
        y += s["residual"].double()
    return y
