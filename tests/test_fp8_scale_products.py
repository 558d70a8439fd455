"""Every kernel of the 8-bit product multiplies the two scales of a block first, in fp32, and the block's sum by that: a result does not hang on which kernel the
sizes of a call choose, for ordinary scales and for those whose product leaves fp32's range."""
import ctypes as C

import pytest
import torch

from mini_nccl_b200.ops import gemm_fp8

SHAPES = [(1, 256, 128), (1, 300, 100), (2, 300, 1100), (3, 1024, 128), (4, 1000, 2048), (16, 2048, 128), (16, 4096, 4096), (24, 8192, 8192), (64, 4096, 4096), (40, 4096, 640), (16, 14336, 256),
          (200, 3000, 128), (100, 16384, 128), (64, 20000, 384), (256, 1000, 128), (1000, 640, 100), (2048, 640, 128), (4096, 1536, 128), (2000, 2000, 512)]


def _plan(M, N, K, b_rows):
    import mini_nccl_b200 as mn

    tile, slices = C.c_int(0), C.c_int(0)
    return mn.lib().mncclGemmFp8Plan(M, N, K, b_rows, N % 4 == 0, 148, C.byref(tile), C.byref(slices)), tile.value, slices.value


def test_the_shapes_reach_every_kernel():
    plans = [_plan(*shape, b_rows) for shape in SHAPES for b_rows in (1, 128)]
    assert {p[:2] for p in plans} >= {(2, 8), (1, 16), (1, 32), (1, 64), (0, 64), (0, 128), (0, 192), (0, 256)} and any(p[2] > 1 for p in plans)


def _operands(M, N, K, block, a_rows, b_rows):
    """Whole numbers of up to 4, other than 0 in one block of K only, where the sums are then exact; scales from a list of pairs."""
    g = torch.Generator(device="cuda").manual_seed(M + N + K)
    blocks = -(-K // 128)
    ops = []
    for rows in (M, N):
        t = torch.zeros(rows, -(-K // 16) * 16, device="cuda")[:, :K]
        t[:, block * 128:(block + 1) * 128] = torch.randint(-4, 5, t[:, block * 128:(block + 1) * 128].shape, generator=g, device="cuda").float()
        ops.append(torch.empty(rows, -(-K // 16) * 16, device="cuda").to(torch.float8_e4m3fn)[:, :K].copy_(t))
    ops[0][M // 2] = 0.0   # sums of 0
    sums = (ops[0].double() @ ops[1].double().t()).float()
    return ops, sums, torch.ones(-(-M // a_rows), blocks, device="cuda"), torch.ones(-(-N // b_rows), blocks, device="cuda"), g


def _rows(s, per, n):
    return s.repeat_interleave(per, 0)[:n]


@pytest.mark.gpu
@pytest.mark.parametrize("M,N,K", SHAPES)
@pytest.mark.parametrize("a_rows,b_rows", [(1, 128), (1, 1), (128, 128)])
def test_the_scales_are_multiplied_first(M, N, K, a_rows, b_rows):
    """Bit for bit: (sa * sb) and its product with an exact sum are each rounded once; the other blocks add zeros."""
    block = (M + N) % -(-K // 128)
    (a, b), sums, sa, sb, g = _operands(M, N, K, block, a_rows, b_rows)
    for s in (sa, sb):
        s.copy_(torch.rand(s.shape, generator=g, device="cuda") + 0.1)
    want = sums * (_rows(sa, a_rows, M)[:, block, None] * _rows(sb, b_rows, N)[:, block])
    assert torch.equal(gemm_fp8(a, sa, b, sb, out_dtype=torch.float32), want)


@pytest.mark.gpu
@pytest.mark.parametrize("M,N,K", SHAPES)
@pytest.mark.parametrize("b_rows", [128, 1])
def test_scales_at_the_ends_of_their_range(M, N, K, b_rows):
    """Products within fp32's range are exact however far out the scales are; beyond it they are infinite or 0 in every kernel."""
    block = (M + N) % -(-K // 128)
    (a, b), sums, sa, sb, _ = _operands(M, N, K, block, 1, b_rows)
    for p, q in ((120, -100), (-100, 120), (-140, 30), (127, -149), (-149, 127), (-126, -10), (100, 40), (-100, -60)):
        sa[:, block], sb[:, block] = 2.0 ** p, 2.0 ** q
        got = gemm_fp8(a, sa, b, sb, out_dtype=torch.float32)
        both = torch.tensor(2.0 ** p, device="cuda") * torch.tensor(2.0 ** q, device="cuda")
        assert torch.equal(torch.nan_to_num(got, 12345.0), torch.nan_to_num(sums * both, 12345.0)), (p, q)
        if p + q <= 127 and p + q > -149:
            assert torch.equal(got.double(), sums.double() * 2.0 ** (p + q))
