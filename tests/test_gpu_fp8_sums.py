"""The sums of the 8-bit product hold 24 bits, in the tensor cores and between blocks: numbers for which fp32 is exact in any order, and just so."""
import ctypes as C

import pytest
import torch

from mini_nccl_b200.ops import gemm_fp8

E4M3 = torch.float8_e4m3fn
SHAPES = [(1, 1024, 4096), (2, 300, 1100), (4, 1000, 2048), (16, 4096, 4096), (24, 8192, 2048), (64, 4096, 4096), (16, 14336, 384), (64, 8192, 4096), (256, 4096, 4096), (1000, 640, 640), (2048, 640, 512),
          (4096, 1536, 128), (2000, 2000, 1536), (300, 300, 4096)]


def _plan(M, N, K, b_rows):
    import mini_nccl_b200 as mn

    tile, slices = C.c_int(0), C.c_int(0)
    return mn.lib().mncclGemmFp8Plan(M, N, K, b_rows, N % 4 == 0, 148, C.byref(tile), C.byref(slices)), tile.value


def test_the_shapes_reach_every_kernel():
    assert {_plan(*shape, b_rows) for shape in SHAPES for b_rows in (1, 128)} >= {(2, 8), (1, 16), (1, 64), (0, 64), (0, 128), (0, 192), (0, 256)}


@pytest.mark.gpu
@pytest.mark.parametrize("M,N,K", SHAPES)
@pytest.mark.parametrize("b_rows", [128, 1])
def test_sums_hold_24_bits(M, N, K, b_rows):
    """In each block of K one product of 448 * 448 = 200704, its sign alternating from block to block, the others whole multiples of 2^-6 of at most 225 * 2^-6.  Sums
    over any run of blocks, and over any part of a block, are multiples of 2^-6 below 200704 + 32 * 127 * 225 / 64 < 2^18: 24 bits, exact in fp32 in whatever
    order they are added.  A sum that keeps one bit less is off."""
    g = torch.Generator(device="cuda").manual_seed(M + N + K)
    blocks = -(-K // 128)
    ops = []
    at = torch.randint(0, 128, (blocks,), generator=g, device="cuda")
    at = (torch.arange(blocks, device="cuda") * 128 + at).clamp_max(K - 1)
    for rows, sign in ((M, 1.0), (N, -1.0)):
        t = torch.randint(-15, 16, (rows, K), generator=g, device="cuda").float() / 8
        t[:, at] = 448.0 * torch.where(torch.arange(blocks, device="cuda") % 2 == 0, 1.0, sign)
        ops.append(torch.empty(rows, -(-K // 16) * 16, device="cuda").to(E4M3)[:, :K].copy_(t))
        assert torch.equal(ops[-1].float(), t)
    a, b = ops
    want = a.double() @ b.double().t()
    assert torch.equal(want.float().double(), want) and bool(((want * 64) % 2 == 1).any())
    got = gemm_fp8(a, torch.full((M, blocks), 0.125, device="cuda"), b, torch.full((-(-N // b_rows), blocks), 8.0, device="cuda"), out_dtype=torch.float32)
    assert torch.equal(got.double(), want)


@pytest.mark.gpu
@pytest.mark.parametrize("M,N,K", [(1, 4096, 4096), (16, 14336, 4096), (64, 4096, 4096), (256, 4096, 4096), (777, 1003, 1544), (4096, 1536, 128)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_a_product_repeats_itself_bit_for_bit(M, N, K, dtype):
    """Sums are added in an order that the sizes alone decide, whatever runs before and beside the call."""
    g = torch.Generator(device="cuda").manual_seed(M)
    a, b = (torch.empty(rows, -(-K // 16) * 16, device="cuda").to(E4M3)[:, :K].copy_(torch.randn(rows, K, generator=g, device="cuda") * 50) for rows in (M, N))
    sa, sb = torch.rand(M, -(-K // 128), generator=g, device="cuda") + 0.1, torch.rand(-(-N // 128), -(-K // 128), generator=g, device="cuda") + 0.1
    bias = torch.randn(N, generator=g, device="cuda").to(dtype)
    want = gemm_fp8(a, sa, b, sb, out_dtype=dtype, bias=bias)
    beside, noise = torch.cuda.Stream(), torch.randn(2048, 2048, device="cuda")
    beside.wait_stream(torch.cuda.current_stream())
    differ = torch.zeros((), device="cuda")
    for i in range(60):
        if i % 3 == 0:
            with torch.cuda.stream(beside):
                noise @ noise
        if i % 4 == 0:
            gemm_fp8(b[:128], sb.new_ones(128, sb.shape[1]), a, sa)
        differ += (gemm_fp8(a, sa, b, sb, out_dtype=dtype, bias=bias) != want).sum()
    assert not bool(differ)
