"""Results of the 8-bit product whose rows start on 16 bytes but do not end on them: a view of columns of a wider matrix, say.  Nothing behind the last column is written, in the rest
of its 16 bytes either, nor behind the last row's end."""
import ctypes as C
import re
from pathlib import Path

import pytest
import torch

from mini_nccl_b200.ops import gemm_fp8

KERNEL = Path(__file__).resolve().parent.parent / "csrc" / "kernels" / "gemm_fp8.cu"
E4M3 = torch.float8_e4m3fn
SHAPES = [(3953, 5, 83), (2000, 1003, 512), (2000, 1001, 300), (2000, 1006, 128), (600, 1031, 300), (4096, 1537, 128), (8192, 769, 128), (8192, 1059, 64), (1001, 5003, 640), (32768, 61, 128),
          (8192, 4129, 64), (777, 1003, 1544), (300, 2010, 200), (64, 1003, 512), (16, 1003, 4096), (5, 1003, 512), (2, 1003, 512), (1, 77, 9001)]


def _plan(M, N, K, b_rows):
    import mini_nccl_b200 as mn

    tile, slices = C.c_int(0), C.c_int(0)
    return mn.lib().mncclGemmFp8Plan(M, N, K, b_rows, 1, 148, C.byref(tile), C.byref(slices)), tile.value


def test_the_shapes_reach_every_width_and_the_source_keeps_the_rule():
    assert {_plan(*shape, b_rows) for shape in SHAPES for b_rows in (1, 128)} >= {(0, 64), (0, 128), (0, 192), (0, 256), (1, 16), (2, 8)}
    text = re.sub(r"//[^\n]*", "", KERNEL.read_text())
    assert "const bool ragged = g.N % kChunk != 0;" in text
    assert re.findall(r"if \(([^\n]*)\) tma_store_2d\(", text) == ["!ragged || col + (p + 1) * kPer <= g.N"]


@pytest.mark.gpu
@pytest.mark.parametrize("M,N,K", SHAPES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("b_rows", [128, 1])
def test_nothing_is_written_behind_a_row(M, N, K, dtype, b_rows):
    """Whole numbers of up to 4: sums of up to 16 * 9001 < 2^18, exact in fp32, rounded once."""
    g = torch.Generator(device="cuda").manual_seed(M + N + K)
    a, b = (torch.empty(rows, -(-K // 16) * 16, device="cuda").to(E4M3)[:, :K].copy_(torch.randint(-4, 5, (rows, K), generator=g, device="cuda").float()) for rows in (M, N))
    sa, sb = torch.ones(M, -(-K // 128), device="cuda"), torch.ones(-(-N // b_rows), -(-K // 128), device="cuda")
    bias = torch.randint(-8, 9, (N,), generator=g, device="cuda").to(dtype)
    want = ((a.double() @ b.double().t()) + bias.double()).float().to(dtype)
    for ld in (-(-N // 8) * 8, -(-N // 8) * 8 + 8, -(-N // 8) * 8 + 16):
        memory = torch.full((M * ld + 64,), 7.0, dtype=dtype, device="cuda")
        out = memory[:(M - 1) * ld + N].as_strided((M, N), (ld, 1))   # ends with its last element
        for _ in range(2):
            gemm_fp8(a, sa, b, sb, out=out, bias=bias)
            assert torch.equal(out, want)
            assert bool((memory[M * ld:] == 7).all()) and bool((memory[:M * ld].view(M, ld)[:, N:] == 7).all()), "wrote outside the result"
    memory = torch.full((M, N + 24), 7.0, dtype=dtype, device="cuda")   # columns of a wider matrix, dense or not
    for first in (0, 8, 16, 3):
        memory.fill_(7.0)
        gemm_fp8(a, sa, b, sb, out=memory[:, first:first + N], bias=bias)
        assert torch.equal(memory[:, first:first + N], want)
        assert bool((memory[:, :first] == 7).all()) and bool((memory[:, first + N:] == 7).all()), "wrote outside the result"
