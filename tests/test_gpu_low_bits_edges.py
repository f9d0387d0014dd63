"""Products with 4-bit weights at the edges of what may be asked of them."""

import ctypes
import subprocess
import sys
from pathlib import Path

import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from test_gpu_low_bits import ACTS, generator, random_matrix, random_rows

from ayaka_py_b200 import ops
from ayaka_py_b200.csrc import build


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


@pytest.fixture(scope="module")
def impatient(tmp_path_factory):
    """The products' source built so that every hand-over between a CTA's warps gets one poll."""
    out = tmp_path_factory.mktemp("impatient") / "impatient.so"
    try:
        nvcc = build.find_nvcc()
    except RuntimeError as problem:
        pytest.skip(str(problem))
    flags = [f for f in build.NVCC_FLAGS if f not in ("-Xptxas", "-v")]
    subprocess.run([nvcc, *flags, "-DAYK_IMPATIENT", "-shared", "-I", str(build.HERE), str(build.HERE / "linear4.cu"), str(build.HERE / "elementwise.cu"),
                    "-o", str(out)], check=True, capture_output=True)
    lib = ctypes.CDLL(str(out))
    lib.ayk_last_error.restype = ctypes.c_char_p
    lib.ayk_set_pdl(ctypes.c_int(1))
    for name in ("ayk_linear4", "ayk_gated_linear4"):
        getattr(lib, name).argtypes = (ctypes.c_char_p,)
    return lib


@pytest.mark.parametrize("T,N,K", [(1, 128, 32), (8, 4096, 4096), (20, 700, 1600), (61, 6400, 1600), (64, 4096, 8192), (300, 4101, 544), (300, 4128, 544),
                                   (38401, 64, 544), (2500, 2912, 2208)])
@pytest.mark.parametrize("kind", ["linear", "gated"])
def test_kernels_whose_waits_run_out_leave_nothing_behind(impatient, monkeypatch, kind, T, N, K):
    """Warps of a CTA give up with copies on their way: the call returns, a code says so, and the launches behind it, in whose shared and
    tensor memory a late copy or product would land, give what they gave before."""
    N = N // 32 * 32 if kind == "gated" else N
    a, w, up = random_rows(T, K, T), random_matrix(N, K, N), random_matrix(N, K, N + 1)

    def run():
        if kind == "linear":
            return ops.linear4(a, w, out_dtype=torch.float32)
        return ops.gated_linear4(a, w, up).codes.view(torch.uint8)

    want, later = run(), []
    for _ in range(8):
        with monkeypatch.context() as patch:
            patch.setattr(ops, "_lib", impatient)
            run()
        later.append(run())
    torch.cuda.synchronize()
    code = impatient.ayk_linear4_error()
    impatient.ayk_linear4_clear_error()
    assert code in (101, 103, 104, 105, 111, 113, 114, 115, 116, 117, 118, 119)
    assert ops.tc_error() == 0 and all(torch.equal(got, want) for got in later)


def test_copies_of_a_matrix_are_complete_when_they_are_handed_out(monkeypatch):
    import copy
    import pickle
    m, waits = random_matrix(300, 256, 1), []
    here = torch.cuda.current_stream

    class Waited:
        def __init__(self, device):
            self.stream = here(device)

        def synchronize(self):
            waits.append(self.stream)
            self.stream.synchronize()

    monkeypatch.setattr(torch.cuda, "current_stream", Waited)
    for again in (copy.deepcopy, lambda x: pickle.loads(pickle.dumps(x))):
        del waits[:]
        other = again(m)
        assert len(waits) == 1 and other.codes.data_ptr() != m.codes.data_ptr() and torch.equal(other.decoded(), m.decoded())


FIRST_CALL = """
import sys
import torch
from ayaka_py_b200 import ops
from ayaka_py_b200.microscale import Rows8, matrix4
kind, T = sys.argv[1], int(sys.argv[2])
x, w = torch.randn(T, 256, device="cuda"), matrix4(torch.randn(128, 256, device="cuda"))
a = Rows8(torch.randn(T, 256, device="cuda").to(torch.float8_e4m3fn), torch.full((T, 8), 127, dtype=torch.uint8, device="cuda").view(torch.float8_e8m0fnu))
norm = torch.ones(256, device="cuda")
def run():
    if kind == "linear":
        return ops.linear4(a, w)
    rows = ops.rows8(x) if kind == "rows" else ops.rmsnorm_rows8(x, norm, 1e-6) if kind == "norm" else ops.gated_linear4(a, w, w)
    return rows.decoded()
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    y = run()
graph.replay()
torch.cuda.synchronize()
assert torch.equal(y, run()) and bool(torch.isfinite(y).all())
"""


@pytest.mark.parametrize("kind", ["rows", "norm", "linear", "gated"])
@pytest.mark.parametrize("T", [3, 300])
def test_a_process_whose_first_call_is_captured(kind, T):
    done = subprocess.run([sys.executable, "-c", FIRST_CALL, kind, str(T)], cwd=str(Path(__file__).resolve().parent.parent), capture_output=True, text=True, timeout=300)
    assert done.returncode == 0, done.stderr[-2000:]
