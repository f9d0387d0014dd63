"""Rows in 8 bits and products with 4-bit weights on the GPU, against plain arithmetic in 64 bits.

Tolerances.  A code of e4m3 is half a step off at most: 2^-4 of the value, 2^-10 of the block's scale near zero.  The products of
codes and scales are exact in 32-bit; a sum over K in any order of float32 additions, rounded or cut off, is within
(K / 32 + 40) 2^-23 of the sum of the magnitudes (32 products come in at a time, joined in at most 40 further additions, each off
by at most 2^-23 of what has been summed).  Activations are off by 2^-18 of their value and carry an input's error on with a
slope of at most 1.13 (2 |z| for the square).  A bfloat16 result is half a step off at most: 2^-8 of the value."""

import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

import math

from ayaka_py_b200 import ops
from ayaka_py_b200.microscale import Matrix4, Rows8, matrix4

ACTS = {"none": lambda z: z, "gelu_erf": lambda z: z * 0.5 * (1 + torch.erf(z / math.sqrt(2))),
        "gelu_tanh": lambda z: 0.5 * z * (1 + torch.tanh(math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3))),
        "quick_gelu": lambda z: z * torch.sigmoid(1.702 * z), "relu2": lambda z: z.clamp(min=0) ** 2, "silu": lambda z: z * torch.sigmoid(z)}


def generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def random_rows(T, K, seed):
    gen = generator(seed)
    x = torch.randn(T, K, generator=gen, device="cuda") * torch.exp(torch.randn(1, K, generator=gen, device="cuda"))
    if T > 2:
        x[T // 2] = 0
    codes = torch.randn(T, K, generator=gen, device="cuda").mul(40).clamp(-448, 448).to(torch.float8_e4m3fn)
    if T > 2:
        codes[T // 2] = 0
    scales = torch.randint(118, 126, (T, K // 32), generator=gen, device="cuda", dtype=torch.uint8).view(torch.float8_e8m0fnu)
    return Rows8(codes, scales)


def random_matrix(N, K, seed):
    gen = generator(seed)
    codes = torch.randint(0, 256, (N, K // 2), generator=gen, device="cuda", dtype=torch.uint8)
    scales = torch.randint(119, 123, (N, K // 32), generator=gen, device="cuda", dtype=torch.uint8)
    return Matrix4.from_codes(codes, scales)


def product64(a, w):
    """(a w^T, the sum's bound) in 64 bits."""
    x, m = a.decoded().double(), w.decoded().double()
    return x @ m.T, (x.shape[1] / 32 + 40) * 2.0 ** -23 * (x.abs() @ m.abs().T)


def activated64(z, bound, act):
    y = ACTS[act](z)
    slope = 1.0 if act == "none" else 2 * (z.abs() + bound) if act == "relu2" else 1.13
    return y, bound * slope + (0 if act == "none" else 2.0 ** -18 * y.abs())


def check_rows(rows, want, bound):
    """Codes and scales against 64-bit numbers that the kernel knows to within ``bound``."""
    T, K = want.shape
    s = rows.scales.view(torch.uint8).double().sub(127).exp2().unsqueeze(-1)
    v, b = want.view(T, K // 32, 32), bound.view(T, K // 32, 32)
    largest, slack = v.abs().amax(-1, keepdim=True), b.amax(-1, keepdim=True)
    assert bool((largest - slack <= 448 * s).all()) and bool(((largest + slack > 224 * s) | (s == 2.0 ** -127)).all())
    off = (rows.codes.double().view(T, K // 32, 32) * s - v).abs()
    allowed = b + torch.maximum(2.0 ** -4 * (v.abs() + b), 2.0 ** -10 * s)
    assert bool((off <= allowed).all()), float((off / allowed).max())


def check_quantised(rows, x):
    """Numbers that are known exactly give the same codes, bit for bit."""
    T, K = x.shape
    v = x.double().view(T, K // 32, 32)
    m, e = torch.frexp(v.abs().amax(-1).float())
    e = torch.where(m > 0, e - 9 + (m > 0.875), -127).clamp(-127, 127)
    assert torch.equal(rows.scales.view(torch.uint8).int(), (e + 127).int())
    codes = (v * torch.exp2(-e.double()).unsqueeze(-1)).float().view(T, K).to(torch.float8_e4m3fn)
    assert torch.equal(rows.codes.view(torch.uint8), codes.view(torch.uint8))


# ---------------------------------------------------------------- rows8 --

@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("T,K", [(0, 32), (1, 32), (1, 768), (3, 96), (7, 1600), (130, 2080), (2, 16384), (5, 20000 // 32 * 32), (1000, 64)])
def test_rows8(dtype, T, K):
    gen = generator(K)
    x = (torch.randn(T, K, generator=gen, device="cuda") * torch.exp(3 * torch.randn(T, K, generator=gen, device="cuda"))).to(dtype)
    if T:
        x[0, :32] = 0
        x[-1, -1] = 3e38 if dtype == torch.float32 else 2.0 ** 127
        x[-1, 0] = 1e-41                                     # below the smallest normal number
    rows = ops.rows8(x)
    assert rows.shape == (T, K)
    check_quantised(rows, x)
    again = Rows8(rows.codes, rows.scales)                    # laid out as the products read them
    assert again.codes is rows.codes and again.scales is rows.scales


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("offset", [0, 1, 3, 8])
def test_rows8_of_columns_of_a_wider_matrix(dtype, offset):
    wide = torch.randn(37, 461, generator=generator(offset), device="cuda").to(dtype)
    check_quantised(ops.rows8(wide[:, offset:offset + 416]), wide[:, offset:offset + 416])
    one = wide[5:6, offset:offset + 416]
    check_quantised(ops.rows8(one), one)
    same = wide[:1, :416].expand(4, 416)                      # one row, read four times
    check_quantised(ops.rows8(same), same)


def test_rows8_borders_and_ties():
    """Largest numbers at and beside 448 2^e, codes half-way between two."""
    below, above = torch.tensor(448.0).nextafter(torch.tensor(0.0)), torch.tensor(448.0).nextafter(torch.tensor(1e9))
    x = torch.zeros(6, 32, device="cuda")
    x[:, 0] = torch.tensor([448.0, float(below), float(above), 448.0 * 2 ** 20, float(above) * 2.0 ** -30, -448.0])
    x[:, 1:9] = torch.tensor([17.0, 19.0, 21.0, 2 ** -10, 3 * 2 ** -10, 2 ** -9, -2 ** -10, -25.0])
    check_quantised(ops.rows8(x), x)
    assert ops.rows8(x).scales.float()[:, 0].tolist() == [1.0, 1.0, 2.0, 2.0 ** 20, 2.0 ** -4, 1.0]      # the fifth row's largest is 25: 14 < 25 <= 28


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")])
def test_a_block_with_no_number_is_nan_and_the_others_are_not(bad):
    x = torch.randn(4, 128, generator=generator(1), device="cuda")
    x[2, 40] = bad
    rows = ops.rows8(x)
    s = rows.scales.float()
    assert bool(torch.isnan(s[2, 1])) and int(torch.isnan(s).sum()) == 1
    y = ops.linear4(rows, random_matrix(64, 128, 2), out_dtype=torch.float32)
    assert bool(torch.isnan(y[2]).all()) and not bool(torch.isnan(y[[0, 1, 3]]).any())
    g = ops.gated_linear4(rows, random_matrix(64, 128, 2), random_matrix(64, 128, 3))
    assert bool(torch.isnan(g.decoded()[2]).all()) and not bool(torch.isnan(g.decoded()[[0, 1, 3]]).any())


# -------------------------------------------------------------- rmsnorm --

@pytest.mark.parametrize("y_dtype", [None, torch.float32, torch.bfloat16])
@pytest.mark.parametrize("T,K", [(0, 64), (1, 32), (1, 768), (5, 1600), (64, 4096), (333, 1280), (3, 16384), (2, 32 * 700), (700, 96)])
def test_rmsnorm_rows8(y_dtype, T, K):
    gen = generator(T + K)
    x = torch.randn(T, K, generator=gen, device="cuda") * torch.exp(torch.randn(1, K, generator=gen, device="cuda"))
    w = 1 + 0.2 * torch.randn(K, generator=gen, device="cuda")
    y = None if y_dtype is None else torch.randn(T, K, generator=gen, device="cuda").to(y_dtype)
    if T > 2:
        x[1] = 0
        if y is not None:
            y[1] = 0
    want_x = x.clone() if y is None else x + y.float()
    rows = ops.rmsnorm_rows8(x, w, 1e-6, y)
    assert torch.equal(x, want_x)                             # one float32 addition
    v = want_x.double()
    want = v / torch.sqrt(v.square().mean(-1, keepdim=True) + 1e-6) * w.double()
    # the sum of K squares in 32-bit by 32 or more partial sums: (K / 32 + 16) 2^-24 of it, halved by the root; four more roundings
    check_rows(rows, want, want.abs() * ((K / 32 + 16) * 2.0 ** -25 + 4 * 2.0 ** -24))


def test_rmsnorm_rows8_of_columns_of_wider_matrices():
    gen = generator(3)
    for off_x, off_y in ((0, 0), (1, 0), (0, 1), (4, 8), (3, 5)):
        wide, ywide = torch.randn(9, 700, generator=gen, device="cuda"), torch.randn(9, 810, generator=gen, device="cuda").to(torch.bfloat16)
        kept, w = wide.clone(), torch.randn(640, generator=gen, device="cuda")
        x, y = wide[:, off_x:off_x + 640], ywide[:, off_y:off_y + 640]
        rows = ops.rmsnorm_rows8(x, w, 1e-5, y)
        kept[:, off_x:off_x + 640] += y.float()
        assert torch.equal(wide, kept)                        # and nothing beside the columns was touched
        v = kept[:, off_x:off_x + 640].double()
        want = v / torch.sqrt(v.square().mean(-1, keepdim=True) + 1e-5) * w.double()
        check_rows(rows, want, want.abs() * (40 * 2.0 ** -24))


# -------------------------------------------------------------- products --

SHAPES = [(1, 32, 32), (1, 1, 64), (1, 4800, 1600), (2, 129, 96), (8, 4096, 4096), (15, 300, 1056), (16, 512, 2048), (17, 33, 160),
          (31, 1000, 544), (33, 128, 4096), (64, 257, 8192), (65, 1600, 768), (100, 640, 1280), (128, 128, 128), (129, 384, 288), (255, 131, 512),
          (300, 2049, 1088), (513, 1000, 2048), (1801, 520, 352)]


@pytest.mark.parametrize("T,N,K", SHAPES)
def test_linear4(T, N, K):
    a, w = random_rows(T, K, T + K), random_matrix(N, K, N)
    z, bound = product64(a, w)
    got = ops.linear4(a, w)
    assert got.shape == (T, N) and got.dtype == torch.bfloat16
    assert bool(((got.double() - z).abs() <= bound + 2.0 ** -8 * (z.abs() + bound)).all())
    exact = ops.linear4(a, w, out_dtype=torch.float32)
    assert bool(((exact.double() - z).abs() <= bound).all())
    assert torch.equal(exact.to(torch.bfloat16), got)                          # the same sums, rounded once
    assert torch.equal(ops.linear4(a, w, out_dtype=torch.float32), exact)      # and the same again
    assert ops.tc_error() == 0


@pytest.mark.parametrize("act", list(ACTS))
@pytest.mark.parametrize("T,N,K", [(1, 200, 64), (40, 130, 256), (200, 300, 160)])
def test_linear4_epilogue(act, T, N, K):
    gen = generator(T)
    a, w = random_rows(T, K, T), random_matrix(N, K, N)
    z, bound = product64(a, w)
    bias = torch.randn(N, generator=gen, device="cuda") * float(z.std())
    residual = torch.randn(T, N, generator=gen, device="cuda") * float(z.std())
    y, bound = activated64(z + bias.double(), bound + 2.0 ** -23 * (z.abs() + bias.double().abs()), act)
    got = ops.linear4(a, w, bias, act)
    assert bool(((got.double() - y).abs() <= bound + 2.0 ** -8 * (y.abs() + bound)).all())
    y, bound = y + residual.double(), bound + 2.0 ** -23 * (y.abs() + residual.double().abs())
    got = ops.linear4(a, w, bias, act, residual)
    assert bool(((got.double() - y).abs() <= bound + 2.0 ** -8 * (y.abs() + bound)).all())
    out = torch.empty(T, N, device="cuda")
    assert ops.linear4(a, w, bias, act, residual, torch.float32, out) is out
    assert bool(((out.double() - y).abs() <= bound).all())
    in_place = residual.clone()
    ops.linear4(a, w, bias, act, in_place, torch.float32, in_place)            # the stream takes the product
    assert torch.equal(in_place, out)


@pytest.mark.parametrize("act", list(ACTS))
@pytest.mark.parametrize("T,N,K", [(1, 32, 32), (1, 8192, 1024), (8, 160, 4096), (16, 1024, 96), (33, 96, 544), (64, 128, 2048), (65, 416, 160),
                                   (200, 256, 1056), (530, 1056, 512)])
def test_gated_linear4(act, T, N, K):
    a, gate, up = random_rows(T, K, T), random_matrix(N, K, N), random_matrix(N, K, N + 1)
    (zg, bg), (zu, bu) = product64(a, gate), product64(a, up)
    yg, bg = activated64(zg, bg, act)
    want = yg * zu
    rows = ops.gated_linear4(a, gate, up, act)
    assert rows.shape == (T, N)
    check_rows(rows, want, bg * zu.abs() + (yg.abs() + bg) * bu + 2.0 ** -23 * want.abs())
    again = ops.gated_linear4(a, gate, up, act)
    assert torch.equal(rows.codes.view(torch.uint8), again.codes.view(torch.uint8))
    assert torch.equal(rows.scales.view(torch.uint8), again.scales.view(torch.uint8))
    assert ops.tc_error() == 0


def test_no_rows():
    a, w = random_rows(0, 64, 1), random_matrix(96, 64, 1)
    assert ops.linear4(a, w).shape == (0, 96) and ops.gated_linear4(a, w, w).shape == (0, 96)


@pytest.mark.parametrize("T", [1, 20, 300])
def test_rows_of_any_layout(T):
    """Codes and scales that lie in wider rows, from a boundary on that the products take, or copied to one."""
    K, N = 416, 200
    w = random_matrix(N, K, 5)
    a = random_rows(T, K, T)
    want = ops.linear4(a, w, out_dtype=torch.float32)
    wide = torch.full((T, K + 48), 0x7f, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn)      # NaN beside the rows
    scales = torch.full((T, 24), 0xff, dtype=torch.uint8, device="cuda").view(torch.float8_e8m0fnu)
    for c0, s0 in ((16, 4), (32, 0), (3, 1)):
        wide.view(torch.uint8).fill_(0x7f)
        scales.view(torch.uint8).fill_(0xff)
        wide[:, c0:c0 + K].copy_(a.codes)
        scales[:, s0:s0 + K // 32].copy_(a.scales)
        rows = Rows8(wide[:, c0:c0 + K], scales[:, s0:s0 + K // 32])
        assert torch.equal(ops.linear4(rows, w, out_dtype=torch.float32), want)


@pytest.mark.parametrize("T,N,K", [(5, 200, 160), (130, 77, 160), (300, 301, 288), (270, 130, 96), (257, 1008, 544)])
@pytest.mark.parametrize("at,residual_at", [(0, 0), (1, 0), (2, 2), (3, 1), (4, 8), (8, 3)])
def test_results_and_residuals_that_start_anywhere(T, N, K, at, residual_at):
    """Rows of the result and of the residual from any number on, next to others that stay as they are."""
    gen = generator(N)
    a, w = random_rows(T, K, 1), random_matrix(N, K, 2)
    bias = torch.randn(N, generator=gen, device="cuda")
    z, bound = product64(a, w)
    residual = torch.randn(residual_at + T * N, generator=gen, device="cuda")[residual_at:].view(T, N)
    y, slack = z + bias.double(), bound + 2.0 ** -23 * (z.abs() + bias.double().abs())
    for dtype in (torch.float32, torch.bfloat16):
        for r in (None, residual):
            store = torch.full((at + T * N + 9,), 7.0, dtype=dtype, device="cuda")
            out = store[at:at + T * N].view(T, N)
            ops.linear4(a, w, bias, residual=r, out_dtype=dtype, out=out)
            want = y if r is None else y + r.double()
            allowed = slack + 2.0 ** -23 * want.abs() + (0 if r is None else 2.0 ** -23 * r.double().abs())
            if dtype == torch.bfloat16:
                allowed = allowed + 2.0 ** -8 * (want.abs() + allowed)
            assert bool(((out.double() - want).abs() <= allowed).all())
            assert bool((store[:at] == 7.0).all()) and bool((store[at + T * N:] == 7.0).all())
    stream = torch.cat((torch.full((at,), 7.0, device="cuda"), residual.reshape(-1)))
    inside = stream[at:].view(T, N)
    ops.linear4(a, w, bias, "none", inside, torch.float32, inside)
    assert torch.equal(inside, ops.linear4(a, w, bias, "none", residual, torch.float32)) and bool((stream[:at] == 7.0).all())


@pytest.mark.parametrize("T,N,K", [(3, 200, 160), (130, 200, 160)])
def test_what_lies_behind_the_rows_is_left_alone(T, N, K):
    a, w = random_rows(T, K, 1), random_matrix(N, K, 2)
    store = torch.full((T + 3, N), 7.0, device="cuda")
    ops.linear4(a, w, out_dtype=torch.float32, out=store[:T])
    assert bool((store[T:] == 7.0).all())
    assert torch.equal(store[:T], ops.linear4(a, w, out_dtype=torch.float32))


@pytest.mark.parametrize("T", [2, 40, 200])
def test_scales_at_the_ends_of_their_range(T):
    """Powers of two from 2^-127 to 2^127 on both sides, whose products are ordinary numbers again; and products that are too small."""
    K, N = 256, 96
    gen = generator(T)
    codes = torch.randn(T, K, generator=gen, device="cuda").to(torch.float8_e4m3fn)
    nibbles = torch.randint(0, 256, (N, K // 2), generator=gen, device="cuda", dtype=torch.uint8)
    for row, weight in ((0, 250), (1, 254), (254, 0), (253, 2), (127, 127), (0, 0), (0, 127), (10, 100)):
        a = Rows8(codes, torch.full((T, K // 32), row, dtype=torch.uint8, device="cuda").view(torch.float8_e8m0fnu))
        w = Matrix4.from_codes(nibbles, torch.full((N, K // 32), weight, dtype=torch.uint8, device="cuda"))
        x = codes.double() * 2.0 ** (row - 127)
        m = Matrix4.from_codes(nibbles, torch.full((N, K // 32), 127, dtype=torch.uint8, device="cuda")).decoded().double() * 2.0 ** (weight - 127)
        z, bound = x @ m.T, (K / 32 + 40) * 2.0 ** -23 * (x.abs() @ m.abs().T)
        got = ops.linear4(a, w, out_dtype=torch.float32).double()
        assert bool(((got - z).abs() <= bound + 2.0 ** -126).all()), (row, weight)        # below 2^-126: no worse than zero


def test_offsets_beyond_32_bits():
    """More than 2^31 numbers of a result, and of rows."""
    T, N, K = 70001, 32000, 32
    a, w = random_rows(T, K, 1), random_matrix(N, K, 2)
    got = ops.linear4(a, w)
    for lo in (0, 67000, T - 40):
        z, bound = product64(Rows8(a.codes[lo:lo + 40], a.scales[lo:lo + 40]), w)
        assert bool(((got[lo:lo + 40].double() - z).abs() <= bound + 2.0 ** -8 * (z.abs() + bound)).all())
    rows = ops.rows8(got)
    for lo in (0, 67000, T - 40):
        check_quantised(Rows8(rows.codes[lo:lo + 40], rows.scales[lo:lo + 40]), got[lo:lo + 40])
    del got
    z = ops.linear4(Rows8(rows.codes[-9:], rows.scales[-9:]), random_matrix(64, N, 3), out_dtype=torch.float32)
    want, bound = product64(Rows8(rows.codes[-9:].clone(), rows.scales[-9:].clone()), random_matrix(64, N, 3))
    assert bool(((z.double() - want).abs() <= bound).all())
    u = ops.linear4(rows, random_matrix(32, N, 4))
    want, bound = product64(Rows8(rows.codes[-300:], rows.scales[-300:]), random_matrix(32, N, 4))
    assert bool(((u[-300:].double() - want).abs() <= bound + 2.0 ** -8 * (want.abs() + bound)).all())


@pytest.mark.parametrize("T", [1, 9, 70, 400])
def test_a_feed_forward_as_a_block_runs_it(T):
    """norm of the stream -> gate, up -> down onto the stream, each step against 64 bits on the rows that the one before made."""
    d, inner = 768, 2048
    gen = generator(T)
    x, y = torch.randn(T, d, generator=gen, device="cuda"), torch.randn(T, d, generator=gen, device="cuda").to(torch.bfloat16)
    norm = 1 + 0.1 * torch.randn(d, generator=gen, device="cuda")
    gate, up, down = (matrix4(torch.randn(s, generator=gen, device="cuda") / math.sqrt(s[1])) for s in ((inner, d), (inner, d), (d, inner)))
    start = x.double() + y.double()
    h = ops.rmsnorm_rows8(x, norm, 1e-6, y)
    want = start / torch.sqrt(start.square().mean(-1, keepdim=True) + 1e-6) * norm.double()
    check_rows(h, want, want.abs() * (40 * 2.0 ** -24))
    u = ops.gated_linear4(h, gate, up, "silu")
    (zg, bg), (zu, bu) = product64(h, gate), product64(h, up)
    yg, bg = activated64(zg, bg, "silu")
    check_rows(u, yg * zu, bg * zu.abs() + (yg.abs() + bg) * bu + 2.0 ** -23 * (yg * zu).abs())
    before = x.clone()
    ops.linear4(u, down, None, "none", x, torch.float32, x)
    z, bound = product64(u, down)
    assert bool(((x.double() - before.double() - z).abs() <= bound + 2.0 ** -23 * (before.double().abs() + z.abs())).all())
    # near the same feed-forward in 64 bits without codes: their rounding alone is 2^-4 a number (weights 2^-2), at random
    assert float((x.double() - start).norm()) > 0 and bool(torch.isfinite(x).all())


@pytest.mark.parametrize("T", [1, 17, 200])
@pytest.mark.parametrize("kind", ["mlp", "gated_mlp"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_feed_forward_parts_with_4_bit_weights(dtype, kind, T):
    """The parts against the same steps in 64 bits over the rounded weights.  Rows are 8-bit: 2^-4 a number at random signs, twice
    in a row, over the activation between (slope at most 1.13); the outputs' norm takes well under 2^-3 of itself from that."""
    from ayaka_py_b200.parts import PartSpec, make_part
    d, inner = 256, 672
    gen = generator(T)
    part = make_part(PartSpec(kind, {"width": d, "inner": inner, "activation": "gelu_tanh", "weight_bits": 4}), dtype, "cuda")
    tensors = {}
    for name, decl in part.tensors().items():
        scale = 1 / math.sqrt(decl.shape[1]) if decl.kind == "matrix" else 0.1
        tensors[name] = (torch.randn(decl.shape, generator=gen, device="cuda") * scale).to(dtype if decl.kind == "matrix" else torch.float32)
    kept = {name: (matrix4(t).decoded() if t.dim() == 2 else t).double() for name, t in tensors.items()}
    part.bind(tensors)
    assert part.join_input(torch.zeros(8, d, device="cuda"), None) is None
    h = torch.randn(T, d, generator=gen, device="cuda").to(dtype)
    stream = torch.randn(T, d, generator=gen, device="cuda")
    before = stream.double()
    out = part.forward(h, stream, None)
    assert out is stream
    act = ACTS["gelu_tanh"]
    if kind == "mlp":
        want = act(h.double() @ kept["up_weight"].T + kept["up_bias"]) @ kept["down_weight"].T + kept["down_bias"]
    else:
        want = (act(h.double() @ kept["gate_weight"].T) * (h.double() @ kept["up_weight"].T)) @ kept["down_weight"].T
    got = out.double() - before
    assert float((got - want).norm() / want.norm()) < 2.0 ** -3
    if kind == "gated_mlp":
        alone = part.forward(h, None, None)
        assert alone.dtype == torch.float32 and float((alone.double() - want).norm() / want.norm()) < 2.0 ** -3


@pytest.mark.parametrize("T", [1, 12, 150])
def test_captured_and_replayed_beside_another_stream(T):
    d, inner = 512, 640
    gen = generator(T)
    gate, up, down = random_matrix(inner, d, 1), random_matrix(inner, d, 2), random_matrix(d, inner, 3)
    norm = torch.ones(d, device="cuda")

    def run(x, y):
        h = ops.rmsnorm_rows8(x, norm, 1e-6, y)
        return ops.linear4(ops.gated_linear4(h, gate, up), down, residual=x, out_dtype=torch.float32)

    inputs = [(torch.randn(T, d, generator=gen, device="cuda"), torch.randn(T, d, generator=gen, device="cuda")) for _ in range(3)]
    want = [run(x.clone(), y) for x, y in inputs]
    graphs = []
    for _ in range(2):                                        # two graphs, replayed at the same time on two streams
        x, y = torch.empty(T, d, device="cuda"), torch.empty(T, d, device="cuda")
        stream = torch.cuda.Stream()
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            run(x.zero_(), y.zero_())
        stream.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            out = run(x, y)
        graphs.append((graph, x, y, out, stream))
    for i in range(3):
        for j, (graph, x, y, out, stream) in enumerate(graphs):
            source = inputs[(i + j) % 3]
            stream.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(stream):
                x.copy_(source[0])
                y.copy_(source[1])
                graph.replay()
        third = run(inputs[i][0].clone(), inputs[i][1])       # beside them, on the current stream
        torch.cuda.synchronize()
        assert torch.equal(third, want[i])
        for j, (_, _, _, out, _) in enumerate(graphs):
            assert torch.equal(out, want[(i + j) % 3])
    assert ops.tc_error() == 0


def test_other_devices_are_refused():
    a, w = random_rows(2, 64, 1), random_matrix(32, 64, 1)
    with pytest.raises(ops.KernelError, match="current device"):
        ops.linear4(Rows8(a.codes.cpu(), a.scales.cpu()), w)
    with pytest.raises(ops.KernelError, match="current device"):
        ops.linear4(a, w, bias=torch.zeros(32))
    with pytest.raises(ops.KernelError, match="current device"):
        ops.rmsnorm_rows8(torch.zeros(2, 64, device="cuda"), torch.ones(64), 1e-6)
