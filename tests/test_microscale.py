"""Rows in 8 bits and weights in 4 bits: formats, layouts and refusals, without a GPU."""

import pytest

torch = pytest.importorskip("torch")

from ayaka_py_b200 import ops
from ayaka_py_b200.microscale import E2M1, FormatError, Matrix4, Rows8, matrix4, scale_columns


def scales_of(exponents):
    return (torch.as_tensor(exponents) + 127).to(torch.uint8).view(torch.float8_e8m0fnu)


def random_codes(N, K, seed):
    gen = torch.Generator().manual_seed(seed)
    codes = torch.randint(0, 256, (N, K // 2), generator=gen, dtype=torch.uint8)
    scales = torch.randint(100, 140, (N, K // 32), generator=gen, dtype=torch.uint8)
    return codes, scales


@pytest.mark.parametrize("N,K", [(1, 32), (5, 96), (128, 128), (129, 160), (300, 1056), (257, 64)])
def test_layout_of_a_matrix(N, K):
    codes, scales = random_codes(N, K, N + K)
    m = Matrix4.from_codes(codes, scales)
    assert m.shape == (N, K) and m.codes.shape == (-(-K // 128), -(-N // 128) * 128, 64) and m.scales.shape == (-(-K // 128), -(-N // 128), 512)
    back, back_scales = m.row_major()
    assert torch.equal(back, codes) and torch.equal(back_scales, scales)
    # the places that the kernels compute: column block, row, byte; scales at 16 (r % 32) + 4 (r // 32) + block
    for n, k in {(0, 0), (N - 1, K - 1), (N // 2, K // 3), (N - 1, 0), (0, K - 1)}:
        byte = m.codes[k // 128, n, (k % 128) // 2]
        assert int(byte) == int(codes[n, k // 2])
        assert int(m.scales[k // 128, n // 128, (n % 32) * 16 + (n % 128 // 32) * 4 + (k % 128) // 32]) == int(scales[n, k // 32])
        code = int(codes[n, k // 2]) >> 4 * (k % 2) & 15
        value = (-1) ** (code >> 3) * E2M1[code & 7] * 2.0 ** (int(scales[n, k // 32]) - 127)
        assert float(m.decoded()[n, k]) == value
    # what the last blocks have too much is zeros
    assert int(m.codes.view(torch.uint8).long().sum()) == int(codes.long().sum())
    assert int(m.scales.long().sum()) == int(scales.long().sum())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("N,K", [(3, 64), (130, 288)])
def test_a_weight_is_rounded_to_the_nearest_codes(dtype, N, K):
    gen = torch.Generator().manual_seed(K)
    w = (torch.randn(N, K, generator=gen) * torch.exp(2 * torch.randn(N, 1, generator=gen))).to(dtype)
    w[0, :32] = 0
    m = matrix4(w, rows_at_once=64)
    codes, scales = m.row_major()
    v = w.double().view(N, -1, 32)
    s = scales.view(torch.float8_e8m0fnu).double().unsqueeze(-1)
    largest = v.abs().amax(-1, keepdim=True)
    assert bool((largest <= 6 * s).all())                                    # nothing is cut off
    assert bool(((largest > 3 * s) | (largest == 0)).all())                  # and half the scale would be too small
    assert bool((scales.view(N, -1)[0, 0] == 0)) and bool((m.decoded()[0, :32] == 0).all())
    grid = torch.tensor(sorted({a for a in E2M1} | {-a for a in E2M1}), dtype=torch.float64)
    nearest = (v / s).unsqueeze(-1).sub(grid).abs().amin(-1)
    assert torch.equal((m.decoded().double().view(N, -1, 32) / s - v / s).abs(), nearest)


def test_ties_of_a_weight_go_to_the_even_code():
    """In a block whose scale is 1 (its largest is 6): 0.25 -> 0, 0.75 -> 1, 1.25 -> 1, 1.75 -> 2, 2.5 -> 2, 3.5 -> 4, 5 -> 4."""
    row = torch.zeros(1, 32)
    row[0, :8] = torch.tensor([6.0, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0])
    row[0, 8:16] = -row[0, :8]
    want = torch.tensor([6.0, 0.0, 1.0, 1.0, 2.0, 2.0, 4.0, 4.0])
    got = matrix4(row).decoded()[0]
    assert torch.equal(got[:8], want) and torch.equal(got[8:16], -want)


def test_a_weight_of_any_strides_and_extremes():
    w = torch.randn(64, 256, generator=torch.Generator().manual_seed(1))
    assert torch.equal(matrix4(w.t().contiguous().t()).decoded(), matrix4(w).decoded())
    assert torch.equal(matrix4(w[:, 64:128]).decoded(), matrix4(w[:, 64:128].contiguous()).decoded())
    large = torch.full((1, 32), torch.finfo(torch.float32).max)
    codes, scales = matrix4(large).row_major()
    assert int(scales) == 126 + 127 and bool((codes == 0x66).all())               # 4 * 2^126: nearly 2^128, rounded up to it
    small = torch.full((1, 32), 2.0 ** -130)
    assert torch.equal(matrix4(small).decoded(), torch.zeros(1, 32))               # 2^-130 / 2^-127 = 0.125 -> 0


@pytest.mark.parametrize("bad", [
    lambda: matrix4(torch.zeros(4, 40)), lambda: matrix4(torch.zeros(0, 32)), lambda: matrix4(torch.zeros(2, 32, dtype=torch.float64)),
    lambda: matrix4(torch.zeros(32)), lambda: matrix4(torch.tensor([[float("nan")] + [0.0] * 31])),
    lambda: matrix4(torch.tensor([[float("-inf")] + [0.0] * 31])),
    lambda: Matrix4.from_codes(torch.zeros(4, 16, dtype=torch.int8), torch.zeros(4, 1, dtype=torch.uint8)),
    lambda: Matrix4.from_codes(torch.zeros(4, 24, dtype=torch.uint8), torch.zeros(4, 1, dtype=torch.uint8)),
    lambda: Matrix4.from_codes(torch.zeros(4, 16, dtype=torch.uint8), torch.zeros(4, 2, dtype=torch.uint8)),
    lambda: Matrix4.from_codes(torch.zeros(4, 16, dtype=torch.uint8), torch.full((4, 1), 255, dtype=torch.uint8)),
    lambda: Matrix4.from_codes(torch.zeros(0, 16, dtype=torch.uint8), torch.zeros(0, 1, dtype=torch.uint8)),
    lambda: Matrix4(torch.zeros(1, 128, 64, dtype=torch.uint8), torch.zeros(1, 1, 512, dtype=torch.uint8), (129, 128)),
    lambda: Rows8(torch.zeros(2, 32), scales_of([[0], [0]])),
    lambda: Rows8(torch.zeros(2, 48).to(torch.float8_e4m3fn), scales_of([[0], [0]])),
    lambda: Rows8(torch.zeros(2, 64).to(torch.float8_e4m3fn), scales_of([[0], [0]])),
    lambda: Rows8(torch.zeros(2, 32).to(torch.float8_e4m3fn), torch.zeros(2, 1, dtype=torch.uint8)),
    lambda: Rows8(torch.zeros(32).to(torch.float8_e4m3fn), scales_of([[0]])),
])
def test_refused_formats(bad):
    with pytest.raises(FormatError):
        bad()


@pytest.mark.parametrize("T,K", [(0, 32), (1, 32), (3, 96), (5, 512), (2, 544)])
def test_rows_are_laid_out_as_the_kernels_read_them(T, K):
    gen = torch.Generator().manual_seed(K)
    codes = torch.randn(T, K, generator=gen).to(torch.float8_e4m3fn)
    scales = scales_of(torch.randint(-5, 5, (T, K // 32), generator=gen))
    wide = torch.zeros(T, K + 5, dtype=torch.uint8).view(torch.float8_e4m3fn)
    wide[:, 5:].copy_(codes)
    for c in (codes, wide[:, 5:]):
        for s in (scales, scales.t().contiguous().t()):
            rows = Rows8(c, s)
            assert rows.shape == (T, K) and torch.equal(rows.codes.float(), codes.float()) and torch.equal(rows.scales.float(), scales.float())
            assert rows.codes.data_ptr() % 16 == 0 and rows.scales.data_ptr() % 16 == 0
            if T > 1:
                assert rows.codes.stride(0) % 16 == 0 and rows.scales.stride(0) % 16 == 0
            want = codes.float() * scales.float().repeat_interleave(32, dim=1)
            assert torch.equal(rows.decoded(), want)
    made = Rows8.empty(T, K, "cpu")
    assert made.shape == (T, K) and made.scales.shape == (T, K // 32) and made.scales.stride(0) == scale_columns(K)


@pytest.mark.parametrize("kind,params", [("mlp", {"width": 48, "inner": 64, "activation": "gelu_tanh"}),
                                         ("gated_mlp", {"width": 64, "inner": 72, "activation": "silu"}),
                                         ("gated_mlp", {"width": 64, "inner": 64, "activation": "limited_glu"}),
                                         ("mlp", {"width": 64, "inner": 64, "activation": "gelu_tanh", "weight_bits": 8})])
def test_feed_forwards_that_cannot_have_4_bit_weights(kind, params):
    from ayaka_py_b200.parts import PartSpec, make_part
    with pytest.raises(ValueError):
        make_part(PartSpec(kind, {"weight_bits": 4, **params}), torch.bfloat16, "cpu")


@pytest.mark.parametrize("weight_bits", [16, 4])
def test_the_joined_matrix_of_a_gated_feed_forward(weight_bits):
    from ayaka_py_b200.parts import PartSpec, make_part
    part = make_part(PartSpec("gated_mlp", {"width": 64, "inner": 96, "activation": "silu", "weight_bits": weight_bits}), torch.float32, "cpu")
    w = {name: torch.randn(decl.shape, generator=torch.Generator().manual_seed(4)) for name, decl in part.tensors().items()}
    part.bind(w)
    if weight_bits == 4:
        assert part.in_weight is None
    else:
        assert torch.equal(part.in_weight, torch.cat((w["gate_weight"], w["up_weight"])))


def test_feed_forwards_take_their_arguments_in_the_order_that_they_had():
    from ayaka_py_b200.parts.mlp import MLP, GatedMLP
    plain = MLP(64, 96, "gelu_tanh", False, torch.bfloat16, "cpu")
    gated = GatedMLP(64, 96, "silu", None, 1.702, 1.0, torch.bfloat16, "cpu")
    assert plain.dtype == gated.dtype == torch.bfloat16 and plain.weight_bits == gated.weight_bits == 16


def test_a_part_binds_its_4_bit_weights():
    from ayaka_py_b200.parts import PartSpec, make_part
    from ayaka_py_b200.parts.base import NotLowered
    part = make_part(PartSpec("mlp", {"width": 64, "inner": 96, "activation": "gelu_tanh", "bias": False, "weight_bits": 4}), torch.float32, "cpu")
    w = {name: torch.randn(decl.shape, generator=torch.Generator().manual_seed(1)) for name, decl in part.tensors().items()}
    part.bind(w)
    assert torch.equal(part.up4.decoded(), matrix4(w["up_weight"]).decoded()) and part.down4.shape == (64, 96) and part.up_weight is None
    assert sum(t.numel() for t in part.laid_out()) == 2 * (128 * 64 + 512)                # one tile each
    gated = make_part(PartSpec("gated_mlp", {"width": 64, "inner": 96, "activation": "silu", "weight_bits": 4}), torch.float32, "cpu")
    assert gated.laid_out() == []
    gated.bind({name: torch.randn(decl.shape, generator=torch.Generator().manual_seed(2)) for name, decl in gated.tensors().items()})
    assert sum(t.numel() for t in gated.laid_out()) == 3 * (128 * 64 + 512) and gated.join_input(torch.zeros(8, 64), None) is None
    import copy
    import pickle
    for again in (copy.deepcopy(gated), pickle.loads(pickle.dumps(gated))):
        assert torch.equal(again.matrices[1].decoded(), gated.matrices[1].decoded()) and again.matrices[1].shape == (96, 64)
    with pytest.raises(NotLowered):
        part.lower(None, 0, 0)


@pytest.mark.parametrize("again", ["copy", "deepcopy", "pickle"])
def test_copies_of_a_matrix_pass_through_its_constructor(again, monkeypatch):
    """Which waits until the matrix is complete in memory: the kernels read it ahead of earlier work in their stream."""
    import copy
    import pickle
    made, init = [], Matrix4.__init__

    def counted(self, codes, scales, shape):
        made.append(shape)
        init(self, codes, scales, shape)

    monkeypatch.setattr(Matrix4, "__init__", counted)
    m = matrix4(torch.randn(130, 96, generator=torch.Generator().manual_seed(3)))
    del made[:]
    other = {"copy": copy.copy, "deepcopy": copy.deepcopy, "pickle": lambda x: pickle.loads(pickle.dumps(x))}[again](m)
    assert made == [(130, 96)] and other.shape == m.shape and torch.equal(other.codes, m.codes) and torch.equal(other.scales, m.scales)


# --------------------------------------------------------- the kernels' choices --

def test_choice_of_a_products_kernel():
    """Measured on both sides: few rows stay with the kernel that streams the weight, which splits K where tiles alone leave
    multiprocessors idle; many rows go to the persistent one, unless few features and a long K leave that one's tiles too few."""
    for T in (1, 16, 17, 32, 33, 64):
        for N, K in ((32, 32), (768, 768), (4096, 16384), (16384, 4096)):
            for gated in (False, True):
                rows, parts = ops.linear4_plan(T, N, K, gated)
                assert rows == (16 if T <= 16 else 32 if T <= 32 else 64) and 1 <= parts <= min(8, -(-K // 128))
    # clusters that do not run at once are a second wave: 34 tiles in fours 11.3 us, in threes 6.8; 16 in eights 11.8, in sixes 7.3
    assert ops.linear4_plan(50, 4226, 2976) == (64, 3) and ops.linear4_plan(49, 2048, 7424)[1] in (5, 6)
    assert ops.linear4_plan(64, 1600, 6400) == (64, 8) and ops.linear4_plan(8, 4096, 4096)[1] >= 4
    assert ops.linear4_plan(1, 768, 256) == (16, 1)                                        # 2.3 us; in two 2.7
    assert ops.linear4_plan(8, 4096, 16384) == (16, 8) and ops.linear4_plan(61, 6400, 1600)[1] in (1, 2)
    assert ops.linear4_plan(128, 1600, 6400)[0] == 64 and ops.linear4_plan(1024, 1600, 6400)[0] == 128          # 7.4 / 16.6, 29.7 / 18.4 us
    assert ops.linear4_plan(128, 16384, 4096)[0] == 128 and ops.linear4_plan(128, 4096, 16384)[0] == 64          # 21.9 / 13.6, 19.6 / 38.5
    assert ops.linear4_plan(4096, 16384, 4096) == (128, 224) and ops.linear4_plan(4096, 16384, 4096, True) == (128, 96)
    for bad in ((0, 32, 32), (1, 0, 32), (1, 32, 40), (1, 32, 32, False, 0)):
        with pytest.raises(ops.KernelError):
            ops.linear4_plan(*bad)
    for sms in (1, 7, 20, 132):                                                            # parts of a GPU, other GPUs
        assert ops.linear4_plan(3, 4096, 4096, False, sms)[0] == 16 and ops.linear4_plan(3000, 4096, 4096, True, sms)[0] in (64, 128)
    widths = {ops.linear4_plan(T, N, K)[1] for T in (100, 300, 1000, 3000) for N in (64, 500, 1600, 4096, 9000) for K in (256, 2048)
              if ops.linear4_plan(T, N, K)[0] == 128}
    assert widths == {32, 64, 96, 128, 192, 224}                                                                # every width has its products


@pytest.mark.parametrize("bad", [(2 ** 32 + 5, 64, 64), (5, 2 ** 32 + 64, 64), (5, 64, 2 ** 32 + 64), (2 ** 31 - 200, 64, 64), (5, 64, 64, False, 2 ** 32 + 1),
                                 (5, 40, 64, True), (-1, 64, 64), (5, 64, 2 ** 31 - 32)])
def test_no_plan_for_what_is_no_product(bad):
    """Numbers beyond 32 bits among them, and gated products whose rows are not whole blocks: those the calls refuse as well."""
    with pytest.raises(ops.KernelError):
        ops.linear4_plan(*bad)


@pytest.mark.parametrize("N,K,gated", [(128, 9216, True), (128, 16384, True), (128, 9216, False), (32, 32, False)])
def test_more_rows_than_a_grid_has_tiles_of_64(N, K, gated):
    """65,535 tiles of rows at most: more rows go to the kernel whose grid does not grow with them, whichever takes less time."""
    for T in (65535 * 64 + 1, 65536 * 64, 2 ** 31 - 257):
        assert ops.linear4_plan(T, N, K, gated)[0] == 128


# ------------------------------------------------------- refusals of the calls --

class NoLaunch:
    def __getattr__(self, name):
        raise AssertionError(f"{name} was reached")


def rows_of(T, K):
    return Rows8(torch.zeros(T, K).to(torch.float8_e4m3fn), scales_of(torch.zeros(T, K // 32)))


@pytest.mark.parametrize("call,words", [
    (lambda: ops.rows8(torch.zeros(2, 40)), "whole blocks"),
    (lambda: ops.rows8(torch.zeros(2, 0)), "whole blocks"),
    (lambda: ops.rows8(torch.zeros(64)), "whole blocks"),
    (lambda: ops.rows8(torch.zeros(64, 32).t().contiguous().t()), "unit column stride"),
    (lambda: ops.rows8(torch.zeros(2, 32, dtype=torch.float16)), "not supported"),
    (lambda: ops.rows8(torch.zeros(2, 32)), "current device"),
    (lambda: ops.rmsnorm_rows8(torch.zeros(2, 32, dtype=torch.bfloat16), torch.ones(32), 1e-6), "float32"),
    (lambda: ops.rmsnorm_rows8(torch.zeros(2, 48), torch.ones(48), 1e-6), "whole blocks"),
    (lambda: ops.rmsnorm_rows8(torch.zeros(2, 32), torch.ones(64), 1e-6), "row width"),
    (lambda: ops.rmsnorm_rows8(torch.zeros(2, 32), torch.ones(32, dtype=torch.bfloat16), 1e-6), "float32"),
    (lambda: ops.rmsnorm_rows8(torch.zeros(2, 32), torch.ones(32), 1e-6, torch.zeros(1, 32)), "stream's shape"),
    (lambda: ops.rmsnorm_rows8(torch.zeros(2, 32), torch.ones(32), 1e-6, torch.zeros(2, 32, dtype=torch.float16)), "not supported"),
    (lambda: ops.rmsnorm_rows8(torch.zeros(1, 32).expand(2, 32), torch.ones(32), 1e-6, torch.zeros(2, 32)), "overlap"),
    (lambda: ops.rmsnorm_rows8(torch.zeros(2, 32), torch.ones(32), 1e-6), "current device"),
    (lambda: ops.linear4(rows_of(2, 64), matrix4(torch.zeros(8, 32))), "do not fit"),
    (lambda: ops.linear4(rows_of(2, 32), matrix4(torch.zeros(8, 32)), activation="tanh"), "unknown activation"),
    (lambda: ops.linear4(rows_of(2, 32), matrix4(torch.zeros(8, 32)), torch.zeros(7)), "one bias"),
    (lambda: ops.linear4(rows_of(2, 32), matrix4(torch.zeros(8, 32)), torch.zeros(8, dtype=torch.bfloat16)), "float32"),
    (lambda: ops.linear4(rows_of(2, 32), matrix4(torch.zeros(8, 32)), residual=torch.zeros(2, 7)), "output's shape"),
    (lambda: ops.linear4(rows_of(2, 32), matrix4(torch.zeros(8, 32)), out_dtype=torch.float16), "not supported"),
    (lambda: ops.linear4(rows_of(2, 32), matrix4(torch.zeros(8, 32)), out=torch.zeros(2, 8)), "output dtype"),
    (lambda: ops.linear4(rows_of(2, 32), matrix4(torch.zeros(8, 32)), out=torch.zeros(8, 2, dtype=torch.bfloat16).t()), "contiguous"),
    (lambda: ops.linear4(rows_of(2, 32), matrix4(torch.zeros(8, 32))), "current device"),
    (lambda: ops.gated_linear4(rows_of(2, 32), matrix4(torch.zeros(32, 32)), matrix4(torch.zeros(64, 32))), "do not fit"),
    (lambda: ops.gated_linear4(rows_of(2, 64), matrix4(torch.zeros(32, 32)), matrix4(torch.zeros(32, 32))), "do not fit"),
    (lambda: ops.gated_linear4(rows_of(2, 32), matrix4(torch.zeros(40, 32)), matrix4(torch.zeros(40, 32))), "whole blocks"),
    (lambda: ops.gated_linear4(rows_of(2, 32), matrix4(torch.zeros(32, 32)), matrix4(torch.zeros(32, 32)), "sigmoid"), "unknown activation"),
    (lambda: ops.gated_linear4(rows_of(2, 32), matrix4(torch.zeros(32, 32)), matrix4(torch.zeros(32, 32))), "current device"),
])
def test_refused_calls(call, words, monkeypatch):
    """Refused before anything is launched; the last of each operator is a tensor that is not on the current device."""
    monkeypatch.setattr(ops, "_ready", lambda: NoLaunch())
    monkeypatch.setattr(ops, "_current_device", lambda: 0)
    with pytest.raises(ops.KernelError, match=words):
        call()


@pytest.mark.parametrize("dtype,out_at,residual_at,refused", [
    (torch.float32, 0, 0, False), (torch.float32, 0, 4 * 32, False), (torch.float32, 4 * 32, 0, False), (torch.float32, 0, 32, True), (torch.float32, 32, 0, True),
    (torch.float32, 1, 0, True), (torch.float32, 0, 4 * 32 - 1, True), (torch.bfloat16, 0, 0, True), (torch.bfloat16, 0, 32, True), (torch.bfloat16, 0, 64, False),
    (torch.bfloat16, 2 * 4 * 32, 0, False), (torch.bfloat16, 2 * 4 * 32 - 2, 0, True)])
def test_a_residual_that_overlaps_the_result(dtype, out_at, residual_at, refused, monkeypatch):
    """Four rows of 32, from any number of one store on: the same place or apart (then the call goes on to where the tensors are)."""
    monkeypatch.setattr(ops, "_ready", lambda: NoLaunch())
    monkeypatch.setattr(ops, "_current_device", lambda: 0)
    store = torch.zeros(512)
    out = store.view(dtype)[out_at:out_at + 128].view(4, 32)
    residual = store[residual_at:residual_at + 128].view(4, 32)
    with pytest.raises(ops.KernelError, match="overlap" if refused else "current device"):
        ops.linear4(rows_of(4, 64), matrix4(torch.ones(32, 64)), residual=residual, out_dtype=dtype, out=out)
