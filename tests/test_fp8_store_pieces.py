"""Results of the 8-bit product on CTA pairs leave a warp in pieces through two places in shared memory that alternate.  A place may be laid out anew
once the store that read it last has done so, whichever tile that store belonged to."""
import ctypes as C
import re
from pathlib import Path

import pytest
import torch

from mini_nccl_b200.ops import gemm_fp8

KERNEL = Path(__file__).resolve().parent.parent / "csrc" / "kernels" / "gemm_fp8.cu"
# Few blocks of K, so that little time lies between a tile's last store and the next tile's first; more tiles than the GPU has pairs of SMs; an odd number
# of pieces: tiles of 192 and of 64 columns, and the ragged right edge of tiles of 256.
SHAPES = [(8192, 1056, 64), (16384, 544, 128), (4096, 1536, 128), (8192, 768, 128), (32768, 64, 128), (40000, 64, 100), (8192, 4128, 64), (8192, 1288, 64), (8192, 5000, 128)]


def _plan(M, N, K, b_rows):
    import mini_nccl_b200 as mn

    tile, slices = C.c_int(0), C.c_int(0)
    return mn.lib().mncclGemmFp8Plan(M, N, K, b_rows, 1, 148, C.byref(tile), C.byref(slices)), tile.value


def _pieces(N, tile):
    """Pieces of 32 columns of a 16-bit type that a promotion warp stores, for each half of each column of tiles."""
    half = tile // 2
    return {-(-min(half, N - col) // 32) for col in range(0, -(-N // tile) * tile, half) if col < N}


@pytest.mark.parametrize("b_rows", [128, 1])
def test_the_shapes_have_odd_numbers_of_pieces_and_several_tiles_a_pair(b_rows):
    widths = set()
    for M, N, K in SHAPES:
        kind, tile = _plan(M, N, K, b_rows)
        assert kind == 0 and -(-M // 256) * -(-N // tile) > 74 and any(n % 2 for n in _pieces(N, tile)), (M, N, K)
        widths.add(tile)
    assert widths == {64, 192, 256}


def _reused_too_early(per_tile, over_tiles):
    """Which stores may still be reading the place that the next piece is laid out in, with a wait that leaves the latest store alone: the warp's
    sequence of (wait, lay out, store), tile by tile."""
    early, last, n, total = [], {}, 0, 0
    for tile, pieces in enumerate(per_tile):
        for p in range(pieces):
            place = (total if over_tiles else p) % 2
            if place in last and last[place] == total - 1:   # the latest store, which the wait does not cover
                early.append((tile, p))
            last[place] = total
            total += 1
    return early


def test_places_alternate_over_all_tiles_of_a_warp():
    for per_tile in ([3, 3, 3], [1, 1, 1], [4, 4, 1, 4], [4, 2, 4], [3, 4, 1, 1, 2]):
        assert _reused_too_early(per_tile, True) == []
    assert _reused_too_early([3, 3], False) == [(1, 0)] and _reused_too_early([1, 1, 1], False) == [(1, 0), (2, 0)]   # counted within a tile
    text = re.sub(r"//[^\n]*", "", KERNEL.read_text())
    store = text[text.index("store_rows("):text.index("gemm_fp8_pair_kernel(")]
    assert "uint32_t& pieces" in store and re.findall(r"scratch \+ ([^;]*);", store) == ["(pieces++ & 1u) * kPieceBytes"]
    assert re.findall(r"bulk_wait_read<(\d)>", text) == ["1"] and "kScratchBytes = 2 * kPieceBytes" in text
    promoters = text[text.index("setmaxnreg.inc"):]
    assert promoters.index("uint32_t pieces = 0;") < promoters.index("for (int t = pair;") and promoters.count("pieces = ") == 1


def _whole(rows, cols, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    out = torch.zeros(rows, -(-cols // 16) * 16, device="cuda").to(torch.float8_e4m3fn)[:, :cols]
    return out.copy_(torch.randint(-4, 5, (rows, cols), generator=g, device="cuda").float().to(torch.float8_e4m3fn))


@pytest.mark.gpu
@pytest.mark.parametrize("M,N,K", SHAPES)
@pytest.mark.parametrize("b_rows", [128, 1])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_results_of_many_tiles_are_exact(M, N, K, b_rows, dtype):
    """Values of up to 4, scales of powers of two from 1/4 to 4: a sum is a multiple of 1/16 and at most 128 * 16 * 16 = 2^15, so exact in fp32;
    only the one rounding is left.  Over and over, into rows that are dense and rows that are apart."""
    a, b = _whole(M, K, M + K), _whole(N, K, N + K)
    g = torch.Generator(device="cuda").manual_seed(M)
    sa = torch.exp2(torch.randint(-2, 3, (M, 1), generator=g, device="cuda").float())
    sb = torch.exp2(torch.randint(-2, 3, (-(-N // b_rows), 1), generator=g, device="cuda").float())
    bias = torch.randint(-8, 9, (N,), generator=g, device="cuda").to(dtype)
    sums = (a.double() @ b.double().t()) * sa.double() * sb.double().repeat_interleave(b_rows, 0)[:N].t()
    wide = torch.full((M + 1, N + 16), 7.0, dtype=dtype, device="cuda")
    for bias in (None, bias):
        want = (sums if bias is None else sums + bias.double()).float().to(dtype)
        for out in (torch.empty(M, N, dtype=dtype, device="cuda"), wide[:M, :N]):
            for _ in range(6):
                out.zero_()
                gemm_fp8(a, sa, b, sb, out=out, bias=bias)
                gemm_fp8(a, sa, b, sb, out=out, bias=bias)   # at once behind the other
                assert torch.equal(out, want)
    assert bool((wide[M] == 7).all()) and bool((wide[:, N:] == 7).all()), "wrote outside the result"
