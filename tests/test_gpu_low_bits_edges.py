"""Products with 4-bit weights at the edges of what may be asked of them."""

import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from test_gpu_low_bits import ACTS, generator, random_matrix

from ayaka_py_b200 import ops


@pytest.mark.parametrize("act", list(ACTS))
@pytest.mark.parametrize("T,N,K", [(4, 64, 128), (1, 1601, 1088), (33, 200, 96), (64, 4096, 256), (300, 4101, 544), (1301, 2912, 544)])
def test_rows_that_are_no_numbers_stay_so_under_every_activation(act, T, N, K):
    x = torch.randn(T, K, generator=generator(T), device="cuda")
    bad = sorted({0, T // 2, T - 1})
    for i, value in zip(bad, (float("nan"), float("inf"), float("-inf"))):
        x[i, (7 * i + 5) % K] = value
    good = torch.ones(T, dtype=torch.bool, device="cuda")
    good[bad] = False
    a, w = ops.rows8(x), random_matrix(N, K, 2)
    residual = torch.randn(T, N, generator=generator(N), device="cuda")
    for dtype in (torch.float32, torch.bfloat16):
        y = ops.linear4(a, w, activation=act, residual=residual, out_dtype=dtype)
        assert bool(torch.isnan(y[~good]).all()) and bool(torch.isfinite(y[good]).all())
    N = N // 32 * 32
    u = ops.gated_linear4(a, random_matrix(N, K, 3), random_matrix(N, K, 4), act).decoded()
    assert bool(torch.isnan(u[~good]).all()) and bool(torch.isfinite(u[good]).all())
