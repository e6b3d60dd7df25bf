"""The low-bit operators of the serving path as cases that can be timed and checked.

A decoder layer whose weights are held in 4 bits (e2m1 codes, one power-of-two scale per 32 values of a row) and
whose projection inputs are bf16 or 8-bit rows (e4m3 values, one power-of-two scale per 32).  Sizes are the 8B
layer shape of the repository's benchmark (hidden 4096, MLP 14336, fused q/k/v of 6144 and gate/up of 28672 rows,
32 decode rows, 1024- and 4096-token prefill steps), and generic odd ones.

Kinds of cases:
  norm    residual add + RMSNorm with an 8-bit output
  swiglu  the SwiGLU product with an 8-bit output
  linear  a projection over 4-bit weights, from bf16 ("bf16") or 8-bit ("mx8") rows
  mlp     norm -> gate/up product -> SwiGLU -> down product, as a decode step runs them

8-bit outputs come back as the values that they stand for (exact in bf16).
"""

import math

import torch

own = False

DEV = "cuda"
BF16 = torch.bfloat16
EPS = 1e-5
BLOCK = 32  # values per scale
E4M3_MAX = 448.0
E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


# ------------------------------------------------------------------------------------------ cases
def listed():
    return [
        # one sequence's decode row between two projections: the smallest call, latency
        dict(name="norm_1x4096", kind="norm", rows=1, hidden=4096, residual=True),
        # a 4096-token prefill step's rows
        dict(name="norm_4096x4096", kind="norm", rows=4096, hidden=4096, residual=True),
        # the first norm of a ragged step (no residual yet), a hidden size that fills no thread count
        dict(name="norm_333x2080", kind="norm", rows=333, hidden=2080, residual=False),
        # the MLP of a 32-sequence decode step
        dict(name="swiglu_32x14336", kind="swiglu", rows=32, width=14336),
        # the MLP of a 4096-token prefill step
        dict(name="swiglu_4096x14336", kind="swiglu", rows=4096, width=14336),
        # gate/up of one sequence's decode step: a matrix-vector product
        dict(name="linear_1_gate_up", kind="linear", tokens=1, n=28672, k=4096, x="bf16", bias=False),
        # the output projection of 32 decode rows, which reads the attention's bf16 rows
        dict(name="linear_32_o", kind="linear", tokens=32, n=4096, k=4096, x="bf16", bias=False),
        # the down projection of 32 decode rows, from the 8-bit SwiGLU output
        dict(name="linear_32_down_mx8", kind="linear", tokens=32, n=4096, k=14336, x="mx8", bias=False),
        # fused q/k/v with a bias of a ragged step of 7 rows
        dict(name="linear_7_qkv_mx8", kind="linear", tokens=7, n=6144, k=4096, x="mx8", bias=True),
        # fused q/k/v of a prompt's last, ragged piece
        dict(name="linear_1000_qkv", kind="linear", tokens=1000, n=6144, k=4096, x="bf16", bias=False),
        # gate/up of a 4096-token prefill step: the largest
        dict(name="linear_4096_gate_up_mx8", kind="linear", tokens=4096, n=28672, k=4096, x="mx8", bias=False),
        # the MLP block of an 8-sequence decode step
        dict(name="mlp_8", kind="mlp", rows=8, hidden=4096, width=14336),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["norm", "swiglu", "linear", "linear", "linear", "mlp"])
    if kind == "norm":
        hidden = BLOCK * _log_int(rng, 32, 512)
        return dict(kind=kind, rows=min(_log_int(rng, 1, 8192), 2 ** 26 // hidden), hidden=hidden, residual=rng.random() < 0.7)
    if kind == "swiglu":
        width = BLOCK * _log_int(rng, 32, 896)
        return dict(kind=kind, rows=min(_log_int(rng, 1, 8192), 2 ** 26 // width), width=width)
    if kind == "linear":
        n, k = _log_int(rng, 200, 28672), BLOCK * _log_int(rng, 16, 448)
        tokens = _log_int(rng, 1, rng.choice([64, 8192]))
        return dict(kind=kind, tokens=max(1, min(tokens, 2 ** 38 // (n * k))), n=n, k=k, x=rng.choice(["bf16", "mx8"]),
                    bias=rng.random() < 0.3)
    hidden = BLOCK * _log_int(rng, 48, 192)
    return dict(kind=kind, rows=_log_int(rng, 1, 64), hidden=hidden, width=BLOCK * rng.randint(hidden // 16, hidden // 8))


# ------------------------------------------------------------------------------------------ inputs
def _gen(seed):
    return torch.Generator(device=DEV).manual_seed((int(seed) * 1000003 + 17) % (1 << 62))


def _hidden(g, rows, width):
    """Rows as a decoder's hidden states have them: a few channels far larger than the rest."""

    gain = torch.exp(0.5 * torch.randn(width, generator=g, device=DEV))
    gain[torch.randint(width, (max(1, width // 500),), generator=g, device=DEV)] *= 20
    return (torch.randn((rows, width), generator=g, device=DEV) * gain).to(BF16)


def _exponents(amax, top):
    """Scale bytes: the smallest power of two whose multiple by `top` reaches amax (a mantissa of top's own or less
    keeps top's exponent)."""

    m, e = torch.frexp(amax)  # amax = m 2^e, m in [0.5, 1)
    tm, te = math.frexp(top)
    return torch.where(amax > 0, (e - te + (m > tm).to(e.dtype) + 127).clamp(0, 254), torch.zeros_like(e))


def _codes(g, n, k):
    """A normal weight matrix in 4 bits: codes, two of a byte (the even one low), and scale bytes."""

    w = torch.randn((n, k // BLOCK, BLOCK), generator=g, device=DEV) * (0.7 * k ** -0.5)
    w *= torch.exp(0.3 * torch.randn((n, 1, 1), generator=g, device=DEV))
    scale = _exponents(w.abs().amax(-1), E2M1[-1])
    v = torch.ldexp(w, 127 - scale[..., None])
    mids = torch.tensor([(a + b) / 2 for a, b in zip(E2M1, E2M1[1:])], device=DEV)
    code = torch.bucketize(v.abs(), mids, out_int32=True).to(torch.uint8) | (v < 0).to(torch.uint8) << 3
    code = code.view(n, k // 2, 2)
    return code[..., 0] | code[..., 1] << 4, scale.to(torch.uint8)


def _rows8(g, rows, width):
    """8-bit rows: e4m3 values and scale bytes."""

    y = _hidden(g, rows, width).float().view(rows, -1, BLOCK)
    scale = _exponents(y.abs().amax(-1), E4M3_MAX)
    q = torch.ldexp(y, 127 - scale[..., None]).to(torch.float8_e4m3fn)
    return q.view(rows, width), scale.to(torch.uint8)


def prepare(case, seed):
    g = _gen(seed)
    s = dict(case)
    kind = case["kind"]
    if kind == "norm":
        s["in"] = _hidden(g, case["rows"], case["hidden"])
        s["residual"] = _hidden(g, case["rows"], case["hidden"]) if case["residual"] else None
        s["weight"] = (1 + 0.2 * torch.randn(case["hidden"], generator=g, device=DEV)).to(BF16)
    elif kind == "swiglu":
        both = 1.5 * torch.randn((case["rows"], 2 * case["width"]), generator=g, device=DEV)
        both = both.to(BF16)  # one product's row: gate beside up
        s["gate"], s["up"] = both[:, :case["width"]], both[:, case["width"]:]
    elif kind == "linear":
        s["codes"], s["scales"] = _codes(g, case["n"], case["k"])
        if case["x"] == "mx8":
            s["in"] = _rows8(g, case["tokens"], case["k"])
        else:
            s["in"] = _hidden(g, case["tokens"], case["k"])
        s["b"] = torch.randn(case["n"], generator=g, device=DEV).to(BF16) if case["bias"] else None
    else:
        s["in"] = _hidden(g, case["rows"], case["hidden"])
        s["residual"] = _hidden(g, case["rows"], case["hidden"])
        s["weight"] = (1 + 0.2 * torch.randn(case["hidden"], generator=g, device=DEV)).to(BF16)
        s["codes"], s["scales"] = _codes(g, 2 * case["width"], case["hidden"])
        s["codes2"], s["scales2"] = _codes(g, case["hidden"], case["width"])
    if own:  # the handles that a program makes once, as it loads its weights
        from lastkv_amd import ops

        if "codes" in s:
            s["w"] = ops.mx4_pack(s["codes"], s["scales"])
        if "codes2" in s:
            s["w2"] = ops.mx4_pack(s["codes2"], s["scales2"])
        if kind == "linear" and case["x"] == "mx8":
            s["in"] = ops.MX8Rows(*s["in"])
    return s


# ------------------------------------------------------------------------------------------ the plain forms
def _quantized(y):
    """The values that an 8-bit output of y stands for, from y in 64 bits (next to a border 32 would choose otherwise)."""

    b = y.view(y.shape[0], -1, BLOCK)
    scale = (_exponents(b.abs().amax(-1), E4M3_MAX) - 127)[..., None]
    v = torch.ldexp(b, -scale)
    _, e = torch.frexp(v)  # |v| in [2^(e-1), 2^e): 3 mantissa bits, the smallest normal exponent is -6
    step = (e - 1).clamp(min=-6) - 3
    q = torch.ldexp(torch.round(torch.ldexp(v, -step)), step)
    return torch.ldexp(q, scale).view(y.shape)


def _weights(codes, scales):
    """The fp32 matrix of codes and scale bytes."""

    table = torch.tensor(E2M1 + tuple(-v for v in E2M1), device=DEV)
    low, high = table[(codes & 15).int()], table[(codes >> 4).int()]
    w = torch.stack((low, high), dim=-1).view(codes.shape[0], -1, BLOCK)
    return torch.ldexp(w, scales.int()[..., None] - 127).view(codes.shape[0], -1)


def _norm(s):
    h = s["in"].float()
    if s["residual"] is not None:
        s["residual"].copy_(s["residual"].float() + h)
        h = s["residual"].float()
    h = h.double()
    return s["weight"].double() * (h * torch.rsqrt((h * h).mean(-1, keepdim=True) + EPS))


def _swiglu(gate, up):
    g = gate.double()
    return g / (1 + torch.exp(-g)) * up.double()


def _plain(s):
    kind = s["kind"]
    if kind == "norm":
        y = _quantized(_norm(s)).to(BF16)
        return (y, s["residual"]) if s["residual"] is not None else y
    if kind == "swiglu":
        return _quantized(_swiglu(s["gate"], s["up"])).to(BF16)
    if kind == "linear":
        if s["x"] == "mx8":
            q, e = s["in"]
            x = torch.ldexp(q.float().view(q.shape[0], -1, BLOCK), e.int()[..., None] - 127).view(q.shape)
        else:
            x = s["in"].float()
        y = x @ _weights(s["codes"], s["scales"]).t()
        return (y if s["b"] is None else y + s["b"].float()).to(BF16)
    x = _quantized(_norm(s)).float()
    both = (x @ _weights(s["codes"], s["scales"]).t()).to(BF16)
    m = _quantized(_swiglu(*both.chunk(2, dim=-1))).float()
    return (m @ _weights(s["codes2"], s["scales2"]).t()).to(BF16), s["residual"]


def run(s):
    if not own:
        return _plain(s)
    from lastkv_amd import ops

    kind = s["kind"]
    if kind == "norm":
        y = ops.mx8_unpack(ops.rmsnorm_mx8(s["in"], s["weight"], EPS, residual=s["residual"]))
        return (y, s["residual"]) if s["residual"] is not None else y
    if kind == "swiglu":
        return ops.mx8_unpack(ops.silu_mul_mx8(s["gate"], s["up"]))
    if kind == "linear":
        return ops.mx4_linear(s["in"], s["w"], bias=s["b"])
    x = ops.rmsnorm_mx8(s["in"], s["weight"], EPS, residual=s["residual"])
    both = ops.mx4_linear(x, s["w"])
    m = ops.silu_mul_mx8(both[:, :s["width"]], both[:, s["width"]:])
    return ops.mx4_linear(m, s["w2"]), s["residual"]


def work(case):
    kind = case["kind"]
    if kind == "norm":
        v = case["rows"] * case["hidden"]
        res = 4 * v if case["residual"] else 0
        return {"bytes": 2 * v + res + v + v / BLOCK + 2 * case["hidden"], "flops": 8 * v}
    if kind == "swiglu":
        v = case["rows"] * case["width"]
        return {"bytes": 4 * v + v + v / BLOCK, "flops": 8 * v}
    if kind == "linear":
        m, n, k = case["tokens"], case["n"], case["k"]
        x = m * k * (1 + 1 / BLOCK if case["x"] == "mx8" else 2)
        return {"bytes": n * k * (0.5 + 1 / BLOCK) + x + 2 * m * n, "flops": 2 * m * n * k}
    m, h, w = case["rows"], case["hidden"], case["width"]
    return {"bytes": 3 * h * w * (0.5 + 1 / BLOCK) + 8 * m * h, "flops": 6 * m * h * w}


# ------------------------------------------------------------------------------------------ in 64 bits
def _to_e4m3_blocks(y):
    """64-bit rows as e4m3 blocks: the scale by trying exponents, the values by searching the format's own."""

    grid = sorted(m * 2.0 ** e for e in range(-9, 9) for m in ([1, 1.125, 1.25, 1.375, 1.5, 1.625, 1.75, 1.875] if e >= -6 else
                  [1, 1.25, 1.5, 1.75] if e == -7 else [1, 1.5] if e == -8 else [1]) if m * 2.0 ** e <= E4M3_MAX)
    grid = torch.tensor([0.0] + grid, dtype=torch.float64, device=y.device)
    mids = (grid[1:] + grid[:-1]) / 2
    b = y.reshape(-1, BLOCK)
    amax = b.abs().max(dim=1, keepdim=True).values
    e = torch.floor(torch.log2(amax.clamp(min=1e-300))) - 10
    for _ in range(3):
        e = torch.where(E4M3_MAX * 2.0 ** e >= amax, e, e + 1)
    scale = 2.0 ** e.clamp(-127, 127)
    v = (b / scale).abs()
    down, up = torch.bucketize(v, mids), torch.bucketize(v, mids, right=True)  # they differ on a midpoint: the even index
    q = grid[torch.where(down % 2 == 0, down, up)]
    return (torch.sign(b) * q * scale).reshape(y.shape)


def _exact_weights(codes, scales):
    c = torch.stack((codes % 16, codes // 16), dim=2).reshape(codes.shape[0], -1).to(torch.int64)
    magnitude, exponent, mantissa = c % 8, c % 8 // 2, c % 2
    v = torch.where(magnitude < 2, 0.5 * magnitude.double(), (1 + 0.5 * mantissa.double()) * 2.0 ** (exponent - 1).double())
    return torch.where(c >= 8, -v, v) * (2.0 ** (scales.double() - 127)).repeat_interleave(BLOCK, dim=1)


def _exact_norm(s):
    h = s["in"].double()
    if s["residual"] is not None:
        h = (s["residual"].double() + h).to(BF16).double()
    return h / torch.sqrt((h ** 2).sum(1, keepdim=True) / h.shape[1] + EPS) * s["weight"].double(), h


def exact(case, seed):
    global own
    keep, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = keep
    kind = case["kind"]
    if kind == "norm":
        y, h = _exact_norm(s)
        y = _to_e4m3_blocks(y)
        return (y, h) if case["residual"] else y
    if kind == "swiglu":
        g = s["gate"].double()
        return _to_e4m3_blocks(g * torch.sigmoid(g) * s["up"].double())
    if kind == "linear":
        if case["x"] == "mx8":
            q, e = s["in"]
            x = q.double() * (2.0 ** (e.double() - 127)).repeat_interleave(BLOCK, dim=1)
        else:
            x = s["in"].double()
        y = torch.matmul(x, _exact_weights(s["codes"], s["scales"]).T)
        return y + s["b"].double() if case["bias"] else y
    y, h = _exact_norm(s)
    both = torch.matmul(_to_e4m3_blocks(y), _exact_weights(s["codes"], s["scales"]).T).to(BF16).double()
    g, u = both[:, :case["width"]], both[:, case["width"]:]
    m = _to_e4m3_blocks(g * torch.sigmoid(g) * u)
    return torch.matmul(m, _exact_weights(s["codes2"], s["scales2"]).T), h
