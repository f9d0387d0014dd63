"""Products with 4-bit weights in tiles of every width, where a CTA takes several tiles and where tiles start anywhere in the weight's groups
of 128 features; feed-forward parts step by step.  Against plain arithmetic in 64 bits, with the tolerances of ``test_gpu_low_bits``."""

import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

import math

from test_gpu_low_bits import activated64, check_quantised, check_rows, generator, product64, random_matrix, random_rows

from ayaka_py_b200 import ops
from ayaka_py_b200.microscale import Rows8, matrix4


def sizes(width, gated, several, whole):
    """(T, N, K) that the rule gives tiles of this width to: ``several`` times as many as there are multiprocessors, and one more; else two tiles
    along the features at least.  ``whole``: N a multiple of 32, else odd.  K is four column blocks and a quarter at least."""
    sms = torch.cuda.get_device_properties(0).multi_processor_count
    features = {(0, False): (1001, 2901, 4101, 6001, 385, 333, 131, 65), (0, True): (992, 2912, 4128, 6016, 2080, 3040, 384, 288, 160),
                (1, False): (31, 33, 65, 97, 129, 257, 385), (1, True): (32, 64, 96, 128, 160, 192, 320, 416)}[bool(several), whole]
    for K in (544, 672, 1184):
        for T in (19001, 38401, 60001) if several else (129, 300, 513, 1000, 1301, 2500):
            for N in features:
                tiles, along = -(-T // 128) * -(-N // width), -(-N // width)
                if (tiles > several * sms if several else along > 1) and ops.linear4_plan(T, N, K, gated, sms) == (128, width):
                    return T, N, K
    raise AssertionError(f"no product among these has tiles of {width}")


@pytest.mark.parametrize("whole", [False, True])
@pytest.mark.parametrize("several", [0, 2])
@pytest.mark.parametrize("width", [32, 64, 96, 128, 192, 224])
def test_linear4_in_tiles_of_every_width(width, several, whole):
    T, N, K = sizes(width, False, several, whole)
    a, w = random_rows(T, K, T), random_matrix(N, K, N)
    bad = sorted({0, T // 3, T - 1})
    a.scales.view(torch.uint8)[bad, -1] = 255                   # rows that are no numbers: they and no others give none
    good = torch.ones(T, dtype=torch.bool, device="cuda")
    good[bad] = False
    gen = generator(T)
    bias, residual = torch.randn(N, generator=gen, device="cuda"), torch.randn(T, N, generator=gen, device="cuda")
    z, bound = product64(a, w)
    got = ops.linear4(a, w, out_dtype=torch.float32)
    assert bool(torch.isnan(got[~good]).all())
    assert bool(((got[good].double() - z[good]).abs() <= bound[good]).all())
    assert torch.equal(ops.linear4(a, w)[good], got[good].to(torch.bfloat16))
    y, slack = activated64(z + bias.double(), bound + 2.0 ** -23 * (z.abs() + bias.double().abs()), "gelu_tanh")
    y, slack = y + residual.double(), slack + 2.0 ** -23 * (y.abs() + residual.double().abs())
    ops.linear4(a, w, bias, "gelu_tanh", residual, torch.float32, residual)
    assert bool(((residual[good].double() - y[good]).abs() <= slack[good]).all())
    assert ops.tc_error() == 0


@pytest.mark.parametrize("several", [0, 2])
@pytest.mark.parametrize("width", [32, 64, 96])
def test_gated_linear4_in_tiles_of_every_width(width, several):
    T, N, K = sizes(width, True, several, True)
    a, gate, up = random_rows(T, K, T), random_matrix(N, K, N), random_matrix(N, K, N + 1)
    bad = sorted({0, T // 3, T - 1})
    a.scales.view(torch.uint8)[bad, 0] = 255
    good = torch.ones(T, dtype=torch.bool, device="cuda")
    good[bad] = False
    rows = ops.gated_linear4(a, gate, up, "silu")
    assert bool(torch.isnan(rows.decoded()[~good]).all())
    (zg, bg), (zu, bu) = product64(a, gate), product64(a, up)
    yg, bg = activated64(zg, bg, "silu")
    want, slack = yg * zu, bg * zu.abs() + (yg.abs() + bg) * bu + 2.0 ** -23 * (yg * zu).abs()
    check_rows(Rows8(rows.codes[good], rows.scales[good]), want[good], slack[good])
    assert ops.tc_error() == 0


@pytest.mark.parametrize("T", [1, 17, 200])
@pytest.mark.parametrize("kind", ["mlp", "gated_mlp"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_feed_forward_parts_step_by_step(dtype, kind, T):
    """A part gives what its calls give one after the other, bit for bit, and each of them is right on the rows that the one before made."""
    from ayaka_py_b200.parts import PartSpec, make_part
    d, inner = 256, 672
    gen = generator(T)
    part = make_part(PartSpec(kind, {"width": d, "inner": inner, "activation": "gelu_tanh", "weight_bits": 4}), dtype, "cuda")
    tensors = {}
    for name, decl in part.tensors().items():
        scale = 1 / math.sqrt(decl.shape[1]) if decl.kind == "matrix" else 0.1
        tensors[name] = (torch.randn(decl.shape, generator=gen, device="cuda") * scale).to(dtype if decl.kind == "matrix" else torch.float32)
    part.bind(tensors)
    m = {name: matrix4(t) for name, t in tensors.items() if t.dim() == 2}
    h, stream = torch.randn(T, d, generator=gen, device="cuda").to(dtype), torch.randn(T, d, generator=gen, device="cuda")
    before, got = stream.double(), part.forward(h, stream.clone(), None)
    a = ops.rows8(h)
    check_quantised(a, h)
    if kind == "mlp":
        z, bound = product64(a, m["up_weight"])
        bias = tensors["up_bias"].double()
        y, bound = activated64(z + bias, bound + 2.0 ** -23 * (z.abs() + bias.abs()), "gelu_tanh")
        u = ops.linear4(a, m["up_weight"], tensors["up_bias"], "gelu_tanh", out_dtype=dtype)
        assert bool(((u.double() - y).abs() <= bound + (2.0 ** -8 * (y.abs() + bound) if dtype == torch.bfloat16 else 0)).all())
        rows = ops.rows8(u)
        check_quantised(rows, u)
        down_bias = tensors["down_bias"]
    else:
        (zg, bg), (zu, bu) = product64(a, m["gate_weight"]), product64(a, m["up_weight"])
        yg, bg = activated64(zg, bg, "gelu_tanh")
        rows = ops.gated_linear4(a, m["gate_weight"], m["up_weight"], "gelu_tanh")
        check_rows(rows, yg * zu, bg * zu.abs() + (yg.abs() + bg) * bu + 2.0 ** -23 * (yg * zu).abs())
        down_bias = None
    assert torch.equal(got, ops.linear4(rows, m["down_weight"], down_bias, "none", stream, torch.float32))
    z, bound = product64(rows, m["down_weight"])
    y = z if down_bias is None else z + down_bias.double()
    bound = bound + 2.0 ** -22 * (z.abs() + (0 if down_bias is None else down_bias.double().abs()) + before.abs())      # two additions
    assert bool(((got.double() - (y + before)).abs() <= bound).all())
