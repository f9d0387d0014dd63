"""Rows in 8 bits and weights in 4 bits, in blocks of 32 neighbouring columns that share a power of two.

A block's scale is the smallest power of two by which its largest magnitude comes into the type's range (448 for the rows' e4m3,
6 for the weights' e2m1), kept as its biased exponent (e8m0); the numbers over it are rounded to the nearest, ties to even, so
nothing is cut off.  The scale of a block of zeros is the smallest there is.  A block of rows that holds an infinity or a NaN has
the scale NaN, so that the products of its row are NaN too; a weight that holds one is refused.

``Rows8`` is what the kernels hand on (``ops.rows8``, ``ops.rmsnorm_rows8``, ``ops.gated_linear4``), ``Matrix4`` what they
multiply by (``ops.linear4``, ``ops.gated_linear4``).  Nothing here needs a GPU."""

from __future__ import annotations

import torch

BLOCK = 32                                       # columns that share a scale
E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)  # magnitudes of the codes 0 ... 7; 8 ... 15 are their negatives
TILE = 128                                       # columns of a block of a laid-out matrix; its rows are whole tiles of as many


class FormatError(ValueError):
    """Tensors that cannot be rows in 8 bits or a weight in 4."""


def scale_columns(width: int) -> int:
    """Bytes from one row's scales to the next row's: the kernels read them in whole 16-byte pieces."""
    return (width // BLOCK + 15) & ~15


class Rows8:
    """``codes`` [T, K] float8_e4m3fn and ``scales`` [T, K / 32] float8_e8m0fnu: row t is codes[t, k] * scales[t, k // 32].
    Tensors that do not lie as the kernels read them (rows of codes and of scales from 16-byte boundaries, columns side by side) are
    copied into such.  ``apart``: bytes from a row of codes, and of scales, to the next."""

    __slots__ = ("codes", "scales", "apart")

    def __init__(self, codes: torch.Tensor, scales: torch.Tensor):
        if codes.dim() != 2 or codes.dtype != torch.float8_e4m3fn:
            raise FormatError(f"codes must be [rows, width] of float8_e4m3fn, got {tuple(codes.shape)} of {codes.dtype}")
        T, K = codes.shape
        if K < BLOCK or K % BLOCK:
            raise FormatError(f"a row of {K} is not whole blocks of {BLOCK}")
        if scales.dtype != torch.float8_e8m0fnu or tuple(scales.shape) != (T, K // BLOCK) or scales.device != codes.device:
            raise FormatError(f"scales must be {(T, K // BLOCK)} of float8_e8m0fnu beside the codes, got {tuple(scales.shape)} of {scales.dtype}")
        if codes.stride(1) != 1 or (T > 1 and (codes.stride(0) % 16 or codes.stride(0) < K)) or codes.data_ptr() % 16:
            codes = torch.empty((T, K), dtype=codes.dtype, device=codes.device).copy_(codes)
        if (K > BLOCK and scales.stride(1) != 1) or (T > 1 and (scales.stride(0) % 16 or scales.stride(0) < K // BLOCK)) or scales.data_ptr() % 16:
            scales = torch.empty((T, scale_columns(K)), dtype=scales.dtype, device=scales.device)[:, :K // BLOCK].copy_(scales)
        self.codes, self.scales = codes, scales
        self.apart = (codes.stride(0), scales.stride(0)) if T > 1 else (K, scale_columns(K))      # a single row's stride says nothing

    @classmethod
    def empty(cls, rows: int, width: int, device) -> "Rows8":
        """Rows to be written, laid out as the kernels read them."""
        made = cls.__new__(cls)
        made.apart = apart = (width, (width // BLOCK + 15) & ~15)
        made.codes = torch.empty_strided((rows, width), (width, 1), dtype=torch.float8_e4m3fn, device=device)      # the quickest of torch's allocations
        made.scales = torch.empty_strided((rows, width // BLOCK), (apart[1], 1), dtype=torch.float8_e8m0fnu, device=device)
        return made

    @property
    def shape(self) -> tuple[int, int]:
        return tuple(self.codes.shape)

    def decoded(self) -> torch.Tensor:
        """The rows as float32 numbers (exact)."""
        T, K = self.codes.shape
        return (self.codes.float().view(T, K // BLOCK, BLOCK) * self.scales.float().unsqueeze(-1)).view(T, K)


class Matrix4:
    """A weight [N, K] of e2m1 codes with a scale for every 32 columns, laid out once for the kernels: column blocks of 128 one
    behind the other, in each the rows (rounded up to whole 128) as 64 bytes (two codes to a byte, the even column in the low
    half); and for every column block and 128 rows the 128 x 4 scales as the tensor cores take them (row r, block b at byte
    16 (r % 32) + 4 (r // 32) + b).  What the last blocks have too much is zeros.  Made by ``Matrix4.from_codes`` or ``matrix4``
    and complete in memory by then (the stream is waited for, so not while one is captured): the kernels may read it ahead of
    earlier work in their stream, so it is not written to again."""

    __slots__ = ("codes", "scales", "shape")

    def __init__(self, codes: torch.Tensor, scales: torch.Tensor, shape: tuple[int, int]):
        N, K = shape
        nt, kt = -(-N // TILE), -(-K // TILE)
        if (tuple(codes.shape) != (kt, nt * TILE, TILE // 2) or codes.dtype != torch.uint8 or not codes.is_contiguous()
                or tuple(scales.shape) != (kt, nt, TILE * TILE // BLOCK) or scales.dtype != torch.uint8 or not scales.is_contiguous()
                or N < 1 or K < BLOCK or K % BLOCK or codes.device != scales.device or codes.data_ptr() % 32 or scales.data_ptr() % 16):
            raise FormatError(f"not the blocks of a weight {tuple(shape)}: codes {tuple(codes.shape)}, scales {tuple(scales.shape)}")
        if codes.is_cuda:
            torch.cuda.current_stream(codes.device).synchronize()
        self.codes, self.scales, self.shape = codes, scales, (int(N), int(K))

    def __reduce__(self):
        return Matrix4, (self.codes, self.scales, self.shape)      # copies and what is read back are waited for as well

    @classmethod
    def from_codes(cls, codes: torch.Tensor, scales: torch.Tensor) -> "Matrix4":
        """From row-major codes, uint8 [N, K / 2] (two to a byte, the even column in the low half), and their scales
        [N, K / 32], float8_e8m0fnu or its bytes as uint8."""
        if codes.dim() != 2 or codes.dtype != torch.uint8 or scales.dim() != 2 or scales.dtype not in (torch.uint8, torch.float8_e8m0fnu):
            raise FormatError(f"codes must be [N, K / 2] of uint8 and scales [N, K / {BLOCK}] of float8_e8m0fnu or uint8, got "
                              f"{tuple(codes.shape)} of {codes.dtype} and {tuple(scales.shape)} of {scales.dtype}")
        N, K = codes.shape[0], 2 * codes.shape[1]
        if N < 1 or K < BLOCK or K % BLOCK or tuple(scales.shape) != (N, K // BLOCK) or scales.device != codes.device:
            raise FormatError(f"codes {tuple(codes.shape)} (two to a byte) and scales {tuple(scales.shape)} are not a weight in blocks of {BLOCK}")
        scales = scales.view(torch.uint8)
        if bool((scales == 255).any()):
            raise FormatError("a scale of the weight is NaN")
        nt, kt = -(-N // TILE), -(-K // TILE)

        def whole(t: torch.Tensor, columns: int) -> torch.Tensor:
            if t.shape == (nt * TILE, columns):
                return t.contiguous()
            out = torch.zeros((nt * TILE, columns), dtype=torch.uint8, device=t.device)
            out[:N, :t.shape[1]] = t
            return out

        c = whole(codes, kt * TILE // 2).view(nt * TILE, kt, TILE // 2).transpose(0, 1)
        s = whole(scales, kt * TILE // BLOCK).view(nt, 4, 32, kt, 4).permute(3, 0, 2, 1, 4)
        return cls(c.clone(memory_format=torch.contiguous_format), s.clone(memory_format=torch.contiguous_format).view(kt, nt, TILE * TILE // BLOCK), (N, K))

    def row_major(self) -> tuple[torch.Tensor, torch.Tensor]:
        """(codes, scales as uint8), as ``from_codes`` takes them."""
        (N, K), (kt, nt) = self.shape, self.scales.shape[:2]
        codes = self.codes.transpose(0, 1).reshape(nt * TILE, kt * TILE // 2)[:N, :K // 2]
        scales = self.scales.view(kt, nt, 32, 4, 4).permute(1, 3, 2, 0, 4).reshape(nt * TILE, kt * TILE // BLOCK)[:N, :K // BLOCK]
        return codes.contiguous(), scales.contiguous()

    def decoded(self) -> torch.Tensor:
        """The weight as float32 numbers (exact)."""
        (N, K), (codes, scales) = self.shape, self.row_major()
        table = torch.tensor(E2M1 + tuple(-v for v in E2M1), dtype=torch.float32, device=codes.device)
        numbers = torch.stack((table[(codes & 15).int()], table[(codes >> 4).int()]), dim=-1).view(N, K // BLOCK, BLOCK)
        return (numbers * scales.view(torch.float8_e8m0fnu).float().unsqueeze(-1)).view(N, K)


def matrix4(weight: torch.Tensor, rows_at_once: int = 4096) -> Matrix4:
    """A float32, bfloat16 or float16 weight [N, K] rounded to 4 bits, on its own device."""
    if weight.dim() != 2 or weight.dtype not in (torch.float32, torch.bfloat16, torch.float16):
        raise FormatError(f"a weight is [N, K] of float32, bfloat16 or float16, got {tuple(weight.shape)} of {weight.dtype}")
    N, K = weight.shape
    if N < 1 or K < BLOCK or K % BLOCK:
        raise FormatError(f"a weight's rows are whole blocks of {BLOCK}, got {tuple(weight.shape)}")
    codes = torch.empty((N, K // 2), dtype=torch.uint8, device=weight.device)
    scales = torch.empty((N, K // BLOCK), dtype=torch.uint8, device=weight.device)
    magnitudes = torch.tensor(E2M1, dtype=torch.float32, device=weight.device)
    for a in range(0, N, rows_at_once):                     # 32-bit copies of some rows at a time
        v = weight[a:a + rows_at_once].float().reshape(-1, K // BLOCK, BLOCK)
        largest = v.abs().amax(-1)
        if not bool(torch.isfinite(largest).all()):
            raise FormatError("the weight holds an infinity or a NaN")
        m, e = torch.frexp(largest)
        e = torch.where(largest > 0, e - 3 + (m > 0.75), -127).clamp(-127, 127)       # 6 = 0.75 * 2^3
        q = (v.double() * torch.exp2(-e.double()).unsqueeze(-1)).abs().float().contiguous()
        # ties go to the even code: from below a border to an even code the border itself goes up, to an odd one it stays
        low = torch.bucketize(q, (magnitudes[1:] + magnitudes[:-1]) / 2, right=False)
        high = torch.bucketize(q, (magnitudes[1:] + magnitudes[:-1]) / 2, right=True)
        code = torch.where(low % 2 == 0, low, high).to(torch.uint8)
        code = (code | (torch.signbit(v).to(torch.uint8) << 3)).view(-1, K)
        codes[a:a + rows_at_once] = code[:, 0::2] | (code[:, 1::2] << 4)
        scales[a:a + rows_at_once] = (e + 127).to(torch.uint8).view(-1, K // BLOCK)
    return Matrix4.from_codes(codes, scales)
