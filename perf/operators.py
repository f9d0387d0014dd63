"""Products of 4-bit weights over 8-bit rows, and the kernels that make such rows: the calls that are timed, and what they compute.

Blocks of 32 neighbouring columns share a power of two: rows are kept as e4m3 numbers, weights as e2m1 numbers, and the scale of a
block is the smallest power of two by which its largest number comes into the type's range.  A case names its ``kind`` and its sizes:

``rows``    rows of an attention's output or of the stream become 8-bit rows;
``norm``    the residual stream takes a sublayer's result (``y``) and its root-mean-square norm is written as 8-bit rows;
``linear``  8-bit rows times a 4-bit weight, with bias, activation and residual where the case has them;
``gated``   the first half of a gated feed-forward: act(gate h) * (up h), written as 8-bit rows for the product behind it.

Widths are those of this repository's shapes (768, 1024, 1280, 1600, 2048, 4096 and their inner widths)."""

from __future__ import annotations

import math

import torch

own = False

EPS = 1e-6
BLOCK = 32
DTYPES = {"bfloat16": torch.bfloat16, "float32": torch.float32}
E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


# ------------------------------------------------------------------- cases --

def listed():
    return [
        # the attention's output of a decode step of the XL shape at 8 requests, before the output projection
        {"name": "rows-8x1600", "kind": "rows", "rows": 8, "width": 1600, "dtype": "bfloat16", "strided": False},
        # columns of a wider float32 matrix (a joined projection's) while two prompts are read
        {"name": "rows-2048x2048-slice", "kind": "rows", "rows": 2048, "width": 2048, "dtype": "float32", "strided": True},
        # one user of the small model: the least work there is, where latency is all
        {"name": "norm-1x768", "kind": "norm", "rows": 1, "width": 768, "y": "float32"},
        # 64 requests decode: the stream takes the attention's result and opens the feed-forward
        {"name": "norm-64x1600", "kind": "norm", "rows": 64, "width": 1600, "y": "bfloat16"},
        # a ragged portion, the norm alone (the first layer's)
        {"name": "norm-377x1280-alone", "kind": "norm", "rows": 377, "width": 1280, "y": "none"},
        # a full batch of prompt rows of the widest shape
        {"name": "norm-8192x4096", "kind": "norm", "rows": 8192, "width": 4096, "y": "bfloat16"},
        # one user: query, key and value projection of the XL shape, a matrix-vector product
        {"name": "linear-1x1600-4800", "kind": "linear", "rows": 1, "width": 1600, "out": 4800, "bias": True, "act": "none", "residual": False},
        # 8 requests: the projection back from a wide feed-forward onto the float32 stream
        {"name": "linear-8x16384-4096", "kind": "linear", "rows": 8, "width": 16384, "out": 4096, "bias": False, "act": "none", "residual": True},
        # an odd number of requests through the XL shape's first feed-forward product
        {"name": "linear-61x1600-6400", "kind": "linear", "rows": 61, "width": 1600, "out": 6400, "bias": True, "act": "gelu_tanh", "residual": False},
        # two long prompts through the widest shape's first feed-forward product
        {"name": "linear-4096x4096-16384", "kind": "linear", "rows": 4096, "width": 4096, "out": 16384, "bias": False, "act": "none", "residual": False},
        # 8 requests through a gated feed-forward's first half
        {"name": "gated-8x4096-8192", "kind": "gated", "rows": 8, "width": 4096, "out": 8192, "act": "silu"},
        # two prompts of unequal length through it
        {"name": "gated-1801x2048-8192", "kind": "gated", "rows": 1801, "width": 2048, "out": 8192, "act": "gelu_tanh"},
    ]


def _spread(rng, low, high):
    """A whole number between low and high, even over its logarithm."""
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    kind = rng.choice(["rows", "norm", "linear", "linear", "gated"])
    width = BLOCK * _spread(rng, 4, 16384 // BLOCK)
    if kind in ("rows", "norm"):
        rows = _spread(rng, 1, min(16384, (8192 * 4096) // width))
        if kind == "rows":
            return {"kind": kind, "rows": rows, "width": width, "dtype": rng.choice(list(DTYPES)), "strided": rng.random() < 0.5}
        return {"kind": kind, "rows": rows, "width": width, "y": rng.choice(["none", "bfloat16", "float32"])}
    most = 4096 * 4096 * 16384
    if kind == "gated":
        out = BLOCK * _spread(rng, 1, 512)
        rows = _spread(rng, 1, max(1, min(8192, most // (2 * width * out))))
        return {"kind": kind, "rows": rows, "width": width, "out": out, "act": rng.choice(["silu", "gelu_tanh", "relu2"])}
    out = _spread(rng, 16, 16384)
    rows = _spread(rng, 1, max(1, min(8192, most // (width * out))))
    return {"kind": kind, "rows": rows, "width": width, "out": out, "bias": rng.random() < 0.5,
            "act": rng.choice(["none", "gelu_tanh", "silu"]), "residual": rng.random() < 0.3}


def work(case):
    T, K = case["rows"], case["width"]
    row8 = 1 + 1 / BLOCK                                   # bytes of a number with its share of the scale
    if case["kind"] == "rows":
        return {"bytes": T * K * ((2 if case["dtype"] == "bfloat16" else 4) + row8), "flops": 3 * T * K}
    if case["kind"] == "norm":
        y = {"none": 0, "bfloat16": 2 + 4, "float32": 4 + 4}[case["y"]]                  # y read, the stream written
        return {"bytes": T * K * (4 + y + row8) + 4 * K, "flops": 7 * T * K}
    N = case["out"]
    weight = N * K * (0.5 + 1 / BLOCK)
    if case["kind"] == "gated":
        return {"bytes": 2 * weight + T * K * row8 + T * N * row8, "flops": 4 * T * N * K}
    out = 8 if case["residual"] else 2
    return {"bytes": weight + T * K * row8 + T * N * out + (4 * N if case["bias"] else 0), "flops": 2 * T * N * K}


# ------------------------------------------------------------------ inputs --

def _blocks_of(x, most, smallest=-127):
    """x [T, K] float32 -> (x over its block's scale, the scales' exponents [T, K / 32])."""
    v = x.view(x.shape[0], -1, BLOCK)
    m, e = torch.frexp(v.abs().amax(-1))
    top, at = math.frexp(most)
    e = torch.where(m > 0, e - at + (m > top), smallest).clamp(-127, 127)
    return (v.double() * torch.exp2(-e.double()).unsqueeze(-1)).view(x.shape), e


def _scales(e):
    return (e + 127).to(torch.uint8).view(torch.float8_e8m0fnu)


def _weight(N, K, std, gen):
    """A random weight in 4 bits: codes [N, K / 2] (two to a byte, the even column in the low half) and scales [N, K / 32]."""
    w = torch.randn((N, K), generator=gen, device="cuda") * std
    w *= torch.exp(0.3 * torch.randn((N, 1), generator=gen, device="cuda"))
    q, e = _blocks_of(w, 6.0)
    borders = torch.tensor([(a + b) / 2 for a, b in zip(E2M1, E2M1[1:])], device="cuda", dtype=torch.float32)
    code = (torch.bucketize(q.abs().float(), borders) + 8 * (q < 0)).to(torch.uint8)
    return code[:, 0::2] | (code[:, 1::2] << 4), _scales(e)


def _rows8(T, K, gen):
    """Normed activations in 8 bits: a few channels are large, and a padded row is empty."""
    x = torch.randn((T, K), generator=gen, device="cuda")
    x *= torch.exp(0.5 * torch.randn((1, K), generator=gen, device="cuda"))
    if T > 2:
        x[T // 2] = 0
    q, e = _blocks_of(x, 448.0)
    return q.float().to(torch.float8_e4m3fn), _scales(e)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    T, K, kind = case["rows"], case["width"], case["kind"]
    state = {"case": case}
    if kind == "rows":
        wide = torch.randn((T, 2 * K if case["strided"] else K), generator=gen, device="cuda")
        wide *= torch.exp(torch.randn((1, wide.shape[1]), generator=gen, device="cuda"))
        state["x"] = wide.to(DTYPES[case["dtype"]])[:, -K:]
        return state
    if kind == "norm":
        state["x"] = torch.randn((T, K), generator=gen, device="cuda") * torch.exp(0.5 * torch.randn((1, K), generator=gen, device="cuda"))
        state["weight"] = 1 + 0.1 * torch.randn((K,), generator=gen, device="cuda")
        state["y"] = None
        if case["y"] != "none":
            state["y"] = (0.3 * torch.randn((T, K), generator=gen, device="cuda")).to(DTYPES[case["y"]])
        return state
    N = case["out"]
    state["codes"], state["scales"] = _rows8(T, K, gen)
    state["weights"] = [_weight(N, K, 1 / math.sqrt(K), gen) for _ in range(2 if kind == "gated" else 1)]
    if kind == "linear":
        state["bias"] = torch.randn((N,), generator=gen, device="cuda") if case["bias"] else None
        state["residual"] = 2 * torch.randn((T, N), generator=gen, device="cuda") if case["residual"] else None
    if own:
        # what a program keeps: rows as the operators hand them on, weights laid out once when they are loaded
        from ayaka_py_b200 import ops
        state["rows"] = ops.Rows8(state.pop("codes"), state.pop("scales"))
        state["weights"] = [ops.Matrix4.from_codes(codes, scales) for codes, scales in state["weights"]]
    return state


# ------------------------------------------------------------- plain forms --

def _quantise(h):
    """float32 rows -> (e4m3 numbers, scales): the scale is the smallest power of two that brings the block's largest number to 448 at most."""
    v = h.view(h.shape[0], -1, BLOCK)
    m, e = torch.frexp(v.abs().amax(-1))
    scales = _scales(torch.where(m > 0, e - 9 + (m > 0.875), -127).clamp(-127, 127))
    return (v / scales.float().unsqueeze(-1)).to(torch.float8_e4m3fn).view(h.shape), scales


def _rows(codes, scales):
    return (codes.float().view(codes.shape[0], -1, BLOCK) * scales.float().unsqueeze(-1)).view(codes.shape)


def _matrix(codes, scales):
    table = torch.tensor(E2M1 + tuple(-v for v in E2M1), dtype=torch.float32, device=codes.device)
    numbers = torch.stack((table[(codes & 15).int()], table[(codes >> 4).int()]), dim=-1)
    return (numbers.view(codes.shape[0], -1, BLOCK) * scales.float().unsqueeze(-1)).view(codes.shape[0], -1)


def _activation(z, act):
    if act == "silu":
        return z / (1 + torch.exp(-z))
    if act == "gelu_tanh":
        return 0.5 * z * (1 + torch.tanh(math.sqrt(2 / math.pi) * (z + 0.044715 * z * z * z)))
    if act == "relu2":
        return z.clamp(min=0) ** 2
    return z


def _plain(state):
    case = state["case"]
    if case["kind"] == "rows":
        return _quantise(state["x"].float().contiguous())
    if case["kind"] == "norm":
        x = state["x"]
        if state["y"] is not None:
            x += state["y"].float()
        codes, scales = _quantise(x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * state["weight"])
        return (codes, scales) if state["y"] is None else (codes, scales, x)
    a = _rows(state["codes"], state["scales"])
    if case["kind"] == "gated":
        g, u = (a @ _matrix(*w).T for w in state["weights"])
        return _quantise(_activation(g, case["act"]) * u)
    z = a @ _matrix(*state["weights"][0]).T
    if state["bias"] is not None:
        z = z + state["bias"]
    z = _activation(z, case["act"])
    return z + state["residual"] if state["residual"] is not None else z.to(torch.bfloat16)


def run(state):
    if not own:
        return _plain(state)
    from ayaka_py_b200 import ops
    case = state["case"]
    if case["kind"] == "rows":
        rows = ops.rows8(state["x"])
    elif case["kind"] == "norm":
        rows = ops.rmsnorm_rows8(state["x"], state["weight"], EPS, state["y"])
        if state["y"] is not None:
            return rows.codes, rows.scales, state["x"]
    elif case["kind"] == "gated":
        rows = ops.gated_linear4(state["rows"], *state["weights"], case["act"])
    else:
        return ops.linear4(state["rows"], state["weights"][0], state["bias"], case["act"], state["residual"],
                           torch.bfloat16 if state["residual"] is None else torch.float32)
    return rows.codes, rows.scales


# ---------------------------------------------------- the definition, 64 bits --

def _exact_codes(h):
    """The numbers that the codes stand for before they are rounded.  The scales have no value of their own here: each is a power of
    two that these numbers show, since they are taken over it."""
    T, K = h.shape
    v = h.reshape(T, K // BLOCK, BLOCK)
    largest = v.abs().max(-1).values
    e = torch.ceil(torch.log2(largest / 448.0))
    e = torch.where(largest > 448.0 * torch.exp2(e), e + 1, e)             # the logarithm's own rounding, either way
    e = torch.where(largest <= 448.0 * torch.exp2(e - 1), e - 1, e)
    e = torch.where(largest > 0, e, torch.full_like(e, -127.0)).clamp(-127, 127)
    return (v * torch.exp2(-e)[:, :, None]).reshape(T, K)


def _exact_weight(codes, scales):
    at = torch.stack([codes & 15, codes >> 4], -1).reshape(codes.shape[0], -1).long()
    magnitude = at % 8
    exponent, half = magnitude // 2, magnitude % 2
    value = torch.where(exponent == 0, 0.5 * half, (1 + 0.5 * half) * torch.exp2((exponent - 1).double()))
    value = torch.where(at >= 8, -value, value)
    return value * scales.view(torch.uint8).double().sub(127).exp2().repeat_interleave(BLOCK, dim=1)


def _exact_activation(z, act):
    if act == "silu":
        return z * torch.sigmoid(z)
    if act == "gelu_tanh":
        return z * torch.sigmoid(2 * math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3))
    if act == "relu2":
        return torch.where(z > 0, z * z, torch.zeros_like(z))
    return z


def exact(case, seed):
    global own
    before, own = own, False
    try:
        state = prepare(case, seed)
    finally:
        own = before
    if case["kind"] == "rows":
        return _exact_codes(state["x"].double()), None
    if case["kind"] == "norm":
        x = state["x"].double() if state["y"] is None else state["x"].double() + state["y"].double()
        codes = _exact_codes(x / torch.sqrt((x * x).sum(-1, keepdim=True) / case["width"] + EPS) * state["weight"].double())
        return (codes, None) if state["y"] is None else (codes, None, x)
    a = state["codes"].double() * state["scales"].view(torch.uint8).double().sub(127).exp2().repeat_interleave(BLOCK, dim=1)
    z = [torch.matmul(a, _exact_weight(*w).t()) for w in state["weights"]]
    if case["kind"] == "gated":
        return _exact_codes(_exact_activation(z[0], case["act"]) * z[1]), None
    out = _exact_activation(z[0] if state["bias"] is None else z[0] + state["bias"].double(), case["act"])
    return out if state["residual"] is None else out + state["residual"].double()
