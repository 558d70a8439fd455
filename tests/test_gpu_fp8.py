"""8-bit quantisation, products and the linear layer against their definitions in 64 bits."""
import ctypes as C
import os
import subprocess
import sys

import pytest
import torch
import torch.utils.checkpoint

from mini_nccl_b200.ops import gemm_fp8, linear_fp8, quantize_fp8

E4M3 = torch.float8_e4m3fn
TYPES = [torch.bfloat16, torch.float16, torch.float32]
INF, NAN = float("inf"), float("nan")


def _blocks(n):
    return -(-n // 128)


def _define(x, rows):
    """(x / scale rounded to e4m3, scale) by arithmetic in 64 bits; NaN throughout a block that is not finite."""
    x = x.double().cpu()
    m, k = x.shape
    q, scale = torch.empty_like(x), torch.empty(-(-m // rows), _blocks(k), dtype=torch.float64)
    for i in range(scale.shape[0]):
        for j in range(scale.shape[1]):
            at = (slice(i * rows, (i + 1) * rows), slice(j * 128, (j + 1) * 128))
            v, top = x[at], float(x[at].abs().max())
            if not bool(torch.isfinite(v).all()):
                q[at], scale[i, j] = NAN, NAN
                continue
            e = -126
            while 448.0 * 2.0 ** e < top:
                e += 1
            v = v / 2.0 ** e
            step = torch.full_like(v, 2.0 ** -9)     # e4m3: multiples of 2^-9 up to 2^-6, then eight steps to a power of two
            for p in range(-6, 9):
                step[v.abs() >= 2.0 ** p] = 2.0 ** (p - 3)
            q[at], scale[i, j] = torch.round(v / step) * step, 2.0 ** e
    return q, scale


def _same(got, want):
    assert torch.equal(torch.nan_to_num(got.double().cpu(), 12345.0), torch.nan_to_num(want, 12345.0))


def _spread(scale, rows, shape):
    return scale.double().cpu().repeat_interleave(rows, 0)[:shape[0]].repeat_interleave(128, 1)[:, :shape[1]]


def _input(m, k, dtype, seed=0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(m, k, generator=g) * torch.exp(torch.randn(m, 1, generator=g))
    if m > 2:
        x[m // 2] = 0.0
    return x.to(dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("m,k", [(1, 1), (1, 128), (1, 4096), (2, 16), (3, 129), (15, 130), (17, 1000), (128, 128), (129, 127), (300, 648), (257, 1031)])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows", [1, 128])
def test_quantize(m, k, dtype, rows):
    x = _input(m, k, dtype, seed=m * 31 + k)
    q, scale = quantize_fp8(x.cuda(), block_rows=rows)
    assert q.dtype == E4M3 and scale.dtype == torch.float32 and q.shape == (m, k) and scale.shape == (-(-m // rows), _blocks(k))
    want = _define(x, rows)
    _same(q, want[0])
    _same(scale, want[1])
    both = quantize_fp8(x.cuda(), block_rows=rows, transposed=True)
    _same(both[0], want[0])
    _same(both[1], want[1])
    assert both[2].shape == (k, m)
    want = _define(x.t(), rows)
    _same(both[2], want[0])
    _same(both[3], want[1])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_quantize_the_edges_of_a_type(dtype):
    """Largest and smallest numbers, magnitudes on and next to 448 times a power of two, ties, infinities and NaN."""
    f = torch.finfo(dtype)
    rows = [[f.max, 1.0], [f.tiny, -f.tiny / 2], [f.smallest_normal * 448, 0.0], [448.0, 1.0625, 1.1875, 0.03125], [450.0, 1.0], [-896.0, 3.0], [0.0, -0.0],
            [INF, 1.0], [1.0, -INF], [NAN, 2.0], [448.0, 2.0 ** -10, 3 * 2.0 ** -10, 2.0 ** -9], [1.75, 1e-3], [1.7578125, 1e-3]]
    x = torch.zeros(len(rows), 200, dtype=dtype)
    for i, r in enumerate(rows):
        x[i, :len(r)] = torch.tensor(r, dtype=torch.float64).to(dtype)
        x[i, 190] = 1.0   # another block of the row
    for block_rows in (1, 128):
        q, scale, qt, scale_t = quantize_fp8(x.cuda(), block_rows=block_rows, transposed=True)
        for got, want in zip((q, scale, qt, scale_t), (*_define(x, block_rows), *_define(x.t(), block_rows))):
            _same(got, want)


@pytest.mark.gpu
def test_quantize_layouts_streams_and_nothing():
    base = _input(70, 500, torch.bfloat16).cuda()
    for x in (base[3:, 5:301], base[::2, 8:], base[:1, 3:], base[10:11], base[:, :1], base.t().contiguous().t()[:, :1]):
        for got, want in zip(quantize_fp8(x, transposed=True), (*_define(x, 1), *_define(x.t(), 1))):
            _same(got, want)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    q, scale = quantize_fp8(base, stream=side)
    torch.cuda.current_stream().wait_stream(side)
    _same(q, _define(base, 1)[0])
    for shape in ((0, 300), (5, 0)):
        q, scale, qt, scale_t = quantize_fp8(torch.empty(shape, device="cuda"), transposed=True)
        assert q.shape == shape and scale.shape == (shape[0], _blocks(shape[1])) and qt.shape == shape[::-1] and scale_t.shape == (shape[1], _blocks(shape[0]))


# ---- products


def _rows16(t):
    """The same values in rows that start on 16 bytes."""
    n = t.shape[1]
    out = torch.full((t.shape[0], (n + 15) // 16 * 16 + 16), 3.0, device=t.device).to(E4M3)[:, :n]
    return out.copy_(t)


def _whole(rows, cols, seed, most=4):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return _rows16(torch.randint(-most, most + 1, (rows, cols), generator=g, device="cuda").float().to(E4M3))


def _powers(rows, cols, seed, layout):
    g = torch.Generator(device="cuda").manual_seed(seed)
    s = torch.exp2(torch.randint(-2, 3, (rows, cols), generator=g, device="cuda").float())
    return s if layout == 0 else s.t().contiguous().t() if layout == 1 else torch.stack((s, s), 2).transpose(0, 1).contiguous().transpose(0, 1)[..., 1]


def _product(a, sa, b, sb):
    def values(q, s):
        return q.double() * s.double().repeat_interleave(1 if s.shape[0] == q.shape[0] else 128, 0)[:q.shape[0]].repeat_interleave(128, 1)[:, :q.shape[1]]

    return values(a, sa) @ values(b, sb).t()


SHAPES = [(1, 1, 1), (1, 128, 128), (1, 129, 4096), (2, 64, 72), (15, 300, 136), (16, 14336, 256), (17, 1003, 1544), (33, 257, 3000), (64, 512, 8192), (65, 127, 640),
          (127, 1024, 1024), (129, 640, 320), (256, 256, 256), (255, 4096, 129), (300, 300, 14336), (777, 1003, 1544), (1024, 2048, 512), (2000, 130, 700),
          (4096, 3584, 384), (5, 50257, 128), (8192, 136, 200),
          (1, 4096, 4096), (1, 77, 9001), (2, 1001, 1031), (3, 600, 129), (4, 1024, 2048), (4, 4096, 4096), (1, 14336, 4096),
          (20, 2048, 2048), (64, 2048, 2048), (24, 8192, 8192), (32, 4096, 4096), (64, 4096, 4096), (512, 1024, 4096), (600, 1024, 300), (1001, 5000, 1288), (5000, 1288, 1001)]


def _plan(M, N, K, b_rows=128):
    import mini_nccl_b200 as mn

    tile, slices = C.c_int(0), C.c_int(0)
    small = mn.lib().mncclGemmFp8Plan(M, N, K, b_rows, N % 8 == 0, 148, C.byref(tile), C.byref(slices))
    return small, tile.value, slices.value


def test_the_shapes_reach_every_kernel():
    plans = {_plan(*shape, b_rows) for shape in SHAPES for b_rows in (1, 128)}
    assert {t for kind, t, _ in plans if kind == 1} == {16, 32, 64} and {s for kind, _, s in plans if kind == 1} == {1, 2, 4, 8}
    assert {t for kind, t, _ in plans if kind == 0} == {64, 128, 192, 256}
    assert {M for M, N, K in SHAPES if _plan(M, N, K)[0] == 2} == {1, 2, 3, 4}
    assert _plan(0, 8, 8)[0] == -1 and _plan(8, 8, 8, 64)[0] == -1
    assert _plan(1, 4096, 4096)[0] == 2 and _plan(1, 14336, 4096)[:2] == (1, 16) and _plan(16, 14336, 4096)[:2] == (1, 16)
    assert _plan(4096, 14336, 4096)[0] == 0


@pytest.mark.gpu
@pytest.mark.parametrize("M,N,K", SHAPES)
@pytest.mark.parametrize("a_rows,b_rows", [(1, 128), (1, 1), (128, 128), (128, 1)])
def test_products_of_whole_numbers_are_exact(M, N, K, a_rows, b_rows):
    """Values of up to 4 and scales from 1/4 to 4: partial sums are multiples of 1/16, and with signs at random below 2^20 (a product's
    root mean square is 28, and 14336 of them with both scales stay under 28 * 120 * 16 but for chance), so exact in fp32 in any order: only the
    last rounding is left.  Nothing is written outside the result."""
    dtype = TYPES[(M + N + K) % 3]
    a, b = _whole(M, K, M * 7 + K), _whole(N, K, N * 3 + K)
    sa, sb = _powers(-(-M // a_rows), _blocks(K), 1, (M + N) % 3), _powers(-(-N // b_rows), _blocks(K), 2, (M + K) % 3)
    g = torch.Generator(device="cuda").manual_seed(5)
    bias = torch.randint(-8, 9, (N,), generator=g, device="cuda").to(dtype) if (M + N) % 2 else None
    guard = torch.full((M + 1, N + 3), 7.0, dtype=dtype, device="cuda")
    out = guard[:M, :N]
    assert gemm_fp8(a, sa, b, sb, out=out, bias=bias) is out
    want = _product(a, sa, b, sb) + (bias.double() if bias is not None else 0.0)
    assert torch.equal(out, want.float().to(dtype))
    assert torch.all(guard[M] == 7) and torch.all(guard[:, N:] == 7), "wrote outside the result"
    assert torch.equal(gemm_fp8(a, sa, b, sb, out_dtype=dtype, bias=bias), out)


@pytest.mark.gpu
@pytest.mark.parametrize("M,N,K", [(1, 4096, 4096), (16, 1000, 4096), (100, 260, 1000), (777, 1003, 1544), (1024, 1024, 4096)])
@pytest.mark.parametrize("b_rows", [128, 1])
def test_products_with_any_scales(M, N, K, b_rows):
    """Off the exact product by the fp32 additions at most: K + 3 K / 128 of them, each off by one step of the partial sum (2^-23; sums inside a
    block may be cut off rather than rounded), which the sum of magnitudes bounds; and the last rounding."""
    g = torch.Generator(device="cuda").manual_seed(M + N + K)
    a, b = (_rows16((torch.randn(n, K, generator=g, device="cuda") * 100).clamp(-448, 448).to(E4M3)) for n in (M, N))
    sa = torch.rand(M, _blocks(K), generator=g, device="cuda") + 0.1
    sb = torch.rand(-(-N // b_rows), _blocks(K), generator=g, device="cuda") + 0.1
    want = _product(a, sa, b, sb)
    off = (K + 3 * _blocks(K)) * 2.0 ** -23 * _product(a.float().abs(), sa, b.float().abs(), sb)
    for dtype in TYPES:
        got = gemm_fp8(a, sa, b, sb, out_dtype=dtype).double()
        if dtype == torch.float16:
            want16 = want.clamp(-65504, 65504)
            fits = want.abs() <= 65000
            assert bool(((got - want16).abs() <= off + (want.abs() + off) * torch.finfo(dtype).eps / 2)[fits].all())
            continue
        assert bool(((got - want).abs() <= off + (want.abs() + off) * torch.finfo(dtype).eps / 2).all())


@pytest.mark.gpu
def test_a_block_that_is_not_finite_reaches_its_rows_alone():
    x, w = _input(40, 300, torch.bfloat16).cuda(), _input(200, 300, torch.bfloat16, 1).cuda()
    x[7, 140], x[9, 3], w[130, 299] = NAN, INF, -INF
    y = gemm_fp8(*quantize_fp8(x), *quantize_fp8(w, block_rows=128), out_dtype=torch.float32)
    bad = torch.zeros_like(y, dtype=torch.bool)
    bad[7], bad[9], bad[:, 128:] = True, True, True
    assert torch.equal(torch.isnan(y), bad)
    scale = torch.ones(200, 3, device="cuda")
    scale[5, 1], scale[6, 2] = INF, 0.0
    y = gemm_fp8(*quantize_fp8(x[:4]), _whole(200, 300, 3), scale)
    assert not bool(torch.isfinite(y[0, 5])) and bool(torch.isfinite(y[:, 6:]).all())


@pytest.mark.gpu
def test_products_of_nothing_on_other_streams_and_in_graphs():
    a, b = _whole(50, 300, 1), _whole(70, 300, 2)
    sa, sb = _powers(50, 3, 1, 0), _powers(1, 3, 2, 0)
    want = _product(a, sa, b, sb).float()
    assert gemm_fp8(a[:0], sa[:0], b, sb).shape == (0, 70) and gemm_fp8(a, sa, b[:0], sb[:0]).shape == (50, 0)
    bias = torch.arange(70, device="cuda").float()
    empty = torch.empty(50, 0, device="cuda").to(E4M3), torch.empty(50, 0, device="cuda"), torch.empty(70, 0, device="cuda").to(E4M3), torch.empty(1, 0, device="cuda")
    assert torch.equal(gemm_fp8(*empty, out_dtype=torch.float32, bias=bias), bias.expand(50, 70)) and not gemm_fp8(*empty).any()
    streams = [torch.cuda.Stream() for _ in range(3)]
    outs = []
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
        outs.append(gemm_fp8(a, sa, b, sb, out_dtype=torch.float32, stream=s))
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in outs)
    x = torch.zeros(50, 300, device="cuda")
    graphs, results = [], []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            q, scale = quantize_fp8(x)
            results.append(gemm_fp8(q, scale, b, sb, out_dtype=torch.float32))
        graphs.append(graph)
    x.copy_(a.float() * sa.repeat_interleave(128, 1)[:, :300])
    for s, graph in zip(streams, graphs):
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            graph.replay()
    torch.cuda.synchronize()
    eager = gemm_fp8(*quantize_fp8(x), b, sb, out_dtype=torch.float32)
    assert all(torch.equal(r, eager) for r in results)


@pytest.mark.gpu
@pytest.mark.parametrize("M", [3, 40, 600])
def test_offsets_behind_32_bits(M):
    """Rows so far apart that the last element's offset passes 2^31 elements (and, for what is not 8 bits, 2^32 bytes)."""
    step = -(-(2**31 + 4096) // (M - 1) // 16) * 16 + 16

    def apart(t):
        far = torch.empty((M - 1) * step + t.shape[1], dtype=t.dtype, device="cuda").as_strided(t.shape, (step, 1))
        return far.copy_(t) if t.dtype != E4M3 else far.view(torch.uint8).copy_(t.view(torch.uint8)).view(E4M3)

    x, b = torch.randn(M, 520, device="cuda", dtype=torch.bfloat16), torch.randn(1100, 520, device="cuda")
    q, s, qt, st = quantize_fp8(x, transposed=True)
    for got, want in zip(quantize_fp8(apart(x), transposed=True), (q, s, qt, st)):
        assert torch.equal(got.float(), want.float())
    w, ws = quantize_fp8(b, block_rows=128)
    want = gemm_fp8(q, s, w, ws)
    assert torch.equal(gemm_fp8(apart(q), s, w, ws), want)
    out = apart(torch.zeros_like(want))
    assert torch.equal(gemm_fp8(q, s, w, ws, out=out), want) and out.stride(0) == step
    assert torch.equal(gemm_fp8(w, ws, apart(q), s), gemm_fp8(w, ws, q, s))


@pytest.mark.gpu
@pytest.mark.parametrize("m,n,k", [(1, 1024, 1024), (4, 2048, 2048), (16, 4096, 4096), (64, 4096, 4096), (300, 2000, 3000), (777, 1003, 1544), (2000, 3000, 1000)])
def test_calls_that_follow_one_another_see_what_the_others_wrote(m, n, k):
    """Kernels start before the one ahead of them has ended: chains of calls, whose memory is used again at once, against the same with a
    synchronisation after every call."""
    torch.manual_seed(m)
    weights = [torch.randn(n, k, device="cuda", dtype=torch.bfloat16) * 0.05 for _ in range(2)]

    def chain(x, then):
        seen = []
        for w in weights:
            q = quantize_fp8(x)
            then()
            y = gemm_fp8(*q, *quantize_fp8(w, block_rows=128))
            then()
            q = quantize_fp8(y, transposed=True)[:2]
            then()
            x = gemm_fp8(*q, *quantize_fp8(w, block_rows=128, transposed=True)[2:])
            then()
            seen += [y, x]
        return seen

    for _ in range(10):
        x = torch.randn(m, k, device="cuda", dtype=torch.bfloat16)
        got = chain(x, lambda: None)
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(got, chain(x, torch.cuda.synchronize)))


@pytest.mark.gpu
def test_first_product_of_a_process_may_be_captured():
    """What a product needs once for each process (the word for waits that ran out) is made without breaking a capture that is under way."""
    code = """
import torch
import torch.utils.checkpoint
from mini_nccl_b200.ops import gemm_fp8
a, s = torch.ones(16, 256, device="cuda").to(torch.float8_e4m3fn), torch.ones(16, 2, device="cuda")
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    out = gemm_fp8(a, s, a, s)
graph.replay()
assert bool((out == 256).all())
"""
    r = subprocess.run([sys.executable, "-c", code], cwd=os.path.dirname(os.path.dirname(os.path.abspath(__file__))), capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stderr


# ---- the linear layer


def _quantised(t, rows):
    q, scale = _define(t, rows)
    return q * _spread(scale, rows, t.shape)


def _defined_linear(x, w, bias, grad):
    x, w, grad = (t.detach().cpu() for t in (x, w, grad))
    xq, wq, g = _quantised(x, 1), _quantised(w, 128), _quantised(grad, 1)
    y = xq @ wq.t() + (bias.detach().double().cpu() if bias is not None else 0.0)
    return y, g @ wq, _quantised(grad.t(), 1) @ _quantised(x.t(), 1).t(), grad.double().sum(0)


def _near(got, want, terms):
    """The last rounding, and fp32 sums of `terms` products against the size of the whole result: sums of random signs come out near
    sqrt(terms) of a term, an addition is off by 2^-23 of the sum, so terms * 2^-23 of the largest result covers them."""
    got = got.detach().double().cpu()
    eps = torch.finfo(torch.float32).eps
    return bool(((got - want).abs() <= want.abs() * torch.finfo(_near.dtype).eps / 2 + terms * eps * want.abs().max()).all())


@pytest.mark.gpu
@pytest.mark.parametrize("lead,n,k", [((1,), 8, 16), ((3, 5), 130, 129), ((64,), 128, 256), ((2, 100), 264, 300), ((257,), 100, 640)])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("bias", [False, True])
def test_linear_and_its_gradients(lead, n, k, dtype, bias):
    _near.dtype = dtype
    x, w = _input(torch.Size(lead).numel(), k, dtype, 1).view(*lead, k).cuda().requires_grad_(), _input(n, k, dtype, 2).cuda().requires_grad_()
    b = _input(1, n, dtype, 3)[0].cuda().requires_grad_() if bias else None
    grad = _input(torch.Size(lead).numel(), n, dtype, 4).view(*lead, n).cuda()
    y = linear_fp8(x, w, b)
    assert y.shape == (*lead, n) and y.dtype == dtype
    leaves = [t for t in (x, w, b) if t is not None]
    got = torch.autograd.grad(y, leaves, grad, retain_graph=True)
    want = _defined_linear(x.reshape(-1, k), w, b, grad.reshape(-1, n))
    tokens = x.numel() // k
    assert _near(y.reshape(-1, n), want[0], k + 8)
    assert got[0].shape == x.shape and _near(got[0].reshape(-1, k), want[1], n + 8) and _near(got[1], want[2], tokens + 8)
    if bias:
        assert _near(got[2], want[3], tokens + 8)
    again = torch.autograd.grad(y, leaves, grad)
    assert all(torch.equal(p, q) for p, q in zip(got, again))
    # one leaf alone, the others frozen
    for i, leaf in enumerate(leaves):
        ins = [t if t is leaf or t is None else t.detach() for t in (x, w, b)]
        assert torch.equal(torch.autograd.grad(linear_fp8(*ins), [leaf], grad)[0], got[i])


@pytest.mark.gpu
def test_linear_gradient_is_that_of_differences():
    """Whole numbers up to 8, which e4m3 holds, on both ends of every step: the layer is then the plain bilinear map, the loss moves by
    exactly the gradient times the step, and the gradient (of whole numbers too) has no rounding."""
    g = torch.Generator().manual_seed(3)
    x, w, grad = (torch.randint(-3, 4, shape, generator=g).float().cuda() for shape in ((40, 200), (70, 200), (40, 70)))
    x.requires_grad_(), w.requires_grad_()
    loss = lambda a, b: float((linear_fp8(a, b).detach().double() * grad.double()).sum())  # noqa: E731
    dx, dw = torch.autograd.grad(linear_fp8(x, w), [x, w], grad)
    for leaf, d, f in ((x, dx, lambda t: loss(t, w)), (w, dw, lambda t: loss(x, t))):
        step = torch.randint(-1, 2, leaf.shape, generator=g).float().cuda()
        moved = (f((leaf + step).detach()) - f((leaf - step).detach())) / 2
        assert moved == float((d.double() * step.double()).sum())


@pytest.mark.gpu
def test_linear_strides_hooks_autocast_and_nothing():
    x, w = _input(60, 256, torch.bfloat16, 1).cuda(), _input(96, 256, torch.bfloat16, 2).cuda()
    grad = _input(60, 96, torch.bfloat16, 4).cuda()

    def both(x, w, grad=grad):
        x, w = x.requires_grad_(), w.requires_grad_()
        y = linear_fp8(x, w)
        return (y, *torch.autograd.grad(y, [x, w], grad))

    want = both(x.clone(), w.clone())
    got = both(x.t().contiguous().t(), w.t().contiguous().t(), grad.t().contiguous().t())
    assert all(torch.equal(p, q) for p, q in zip(want, got))
    with torch.autograd.graph.saved_tensors_hooks(lambda s: s.cpu(), lambda s: s.cuda()):
        got = both(x.clone(), w.clone())
    assert all(torch.equal(p, q) for p, q in zip(want, got))
    y, = (linear_fp8(t, w) for t in [x.view(3, 4, 5, 256).expand(2, 3, 4, 5, 256)])
    assert torch.equal(y[1].reshape(60, 96), want[0])
    one = torch.ones(1, 1, device="cuda", dtype=torch.bfloat16).expand(60, 96)   # the gradient of a sum
    p, q = both(x.clone(), w.clone(), one), both(x.clone(), w.clone(), one.contiguous())
    assert all(torch.equal(a, b) for a, b in zip(p, q))
    with torch.autocast("cuda", dtype=torch.bfloat16):
        assert torch.equal(linear_fp8(x.float(), w.float()), want[0])
    xe, we = torch.empty(0, 256, device="cuda", requires_grad=True), w.float().detach().requires_grad_()
    y = linear_fp8(xe, we, torch.zeros(96, device="cuda"))
    dx, dw = torch.autograd.grad(y, [xe, we], torch.empty(0, 96, device="cuda"))
    assert y.shape == (0, 96) and dx.shape == (0, 256) and dw.shape == (96, 256) and not dw.any()
    x.requires_grad_()
    d, = torch.autograd.grad(linear_fp8(x, w).sum(), [x], create_graph=True)
    with pytest.raises(RuntimeError):
        d.float().sum().backward()
    none = w[:0].detach().requires_grad_()   # a layer without output features
    y = linear_fp8(x, none, w[:0, 0])
    dx, dw = torch.autograd.grad(y, [x, none], torch.empty(60, 0, device="cuda", dtype=x.dtype))
    assert y.shape == (60, 0) and dx.shape == x.shape and not dx.any() and dw.shape == (0, 256)
    with torch.no_grad():
        y = linear_fp8(x, w)
    assert torch.equal(y, want[0]) and not y.requires_grad and y.grad_fn is None
    with pytest.raises(RuntimeError, match="no rule"):
        torch.func.vmap(lambda t: linear_fp8(t, w))(x)
    with torch.autograd.forward_ad.dual_level():
        with pytest.raises(RuntimeError, match="no rule"):
            linear_fp8(torch.autograd.forward_ad.make_dual(x.detach(), grad[:, :1].expand(60, 256)), w)
    y = linear_fp8(x, w)
    y.sum().backward()
    with pytest.raises(RuntimeError, match="second time"):
        y.sum().backward()
    x.grad = None
    torch.utils.checkpoint.checkpoint(linear_fp8, x, w, use_reentrant=False).backward(grad)
    assert torch.equal(x.grad, want[1])


# ---- the binding


@pytest.mark.gpu
@pytest.mark.parametrize("tokens,n,k", [(2, 256, 384), (40, 300, 264), (1100, 1288, 520)])
def test_linear_step_captured_and_replayed_on_two_streams(tokens, n, k):
    torch.manual_seed(tokens)
    steps = []
    for _ in range(2):
        x, w, b = (torch.randn(*shape, device="cuda", dtype=torch.bfloat16).requires_grad_() for shape in ((tokens, k), (n, k), (n,)))
        grad = torch.randn(tokens, n, device="cuda", dtype=torch.bfloat16)

        def step(x=x, w=w, b=b, grad=grad):
            y = linear_fp8(x, w, b)
            return [y.detach(), *torch.autograd.grad(y, [x, w, b], grad)]

        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step()
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            results = step()
        with torch.no_grad():
            for t in (x, w, b, grad):
                t.normal_()
        steps.append((graph, results, step, side))
    torch.cuda.synchronize()
    for _ in range(10):   # both at once, over and over
        for graph, _, _, side in steps:
            with torch.cuda.stream(side):
                graph.replay()
    torch.cuda.synchronize()
    for _, results, step, _ in steps:
        assert all(torch.equal(got, want) for got, want in zip(results, step()))


@pytest.mark.gpu
def test_calls_through_ctypes_do_the_same():
    """What stands in for the extension where that cannot be built."""
    import mini_nccl_b200 as mn
    from mini_nccl_b200 import _lib
    from mini_nccl_b200._ctypes_calls import Calls

    ext, plain = _lib.ext(), Calls(mn.lib())
    x, w = _input(70, 300, torch.bfloat16).cuda(), _input(140, 300, torch.float32, 1).cuda()
    bias = torch.randn(140, device="cuda").half()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    for rows, both, stream in ((1, True, None), (128, True, None), (1, False, side)):
        got, want = ([c.quantize_fp8(x, rows, both, stream) for c in (plain, ext)])
        torch.cuda.synchronize()
        for p, q in zip(got, want):
            assert (p is None) == (q is None) and (p is None or (p.shape == q.shape and torch.equal(p[:, :64].float(), q[:, :64].float())))
    args = (*quantize_fp8(x), *quantize_fp8(w, block_rows=128))
    assert torch.equal(plain.gemm_fp8(*args, None, torch.float16, bias, None), ext.gemm_fp8(*args, None, torch.float16, bias, None))
    for lead in ((), (5,), (2, 3)):
        for wide in (1000, 1008):
            logits = torch.randn(*lead, wide, device="cuda")[..., :1000]
            n = logits.numel() // 1000
            ids, top = torch.randint(-1, 1000, (n, 7), device="cuda"), torch.randn(n, 7, device="cuda")
            ids[0, 0] = 3
            for reduction in (0, 1, 2):
                results = []
                for c in (plain, ext):
                    loss, p, stats, counts, tokens = c.distill_forward(logits, ids, top, 2.0, reduction)
                    results.append((loss, p, tokens, c.distill_backward(logits, ids, p, stats, counts, tokens if reduction == 2 else None, 2.0, torch.ones_like(loss))))
                assert all(torch.equal(a, b) and a.shape == b.shape and a.stride() == b.stride() for a, b in zip(*results))
                assert results[0][0].shape == (lead if reduction == 0 else ()) and results[0][3].shape == logits.shape
    for dtype in TYPES:
        x, w, b = _input(30, 200, dtype, 3).view(3, 10, 200).cuda(), _input(130, 200, dtype, 4).cuda(), _input(1, 130, dtype, 5)[0].cuda()
        grad = _input(30, 130, dtype, 6).view(3, 10, 130).cuda()
        for want_x, want_w, bias in ((True, True, b), (True, False, None), (False, True, b), (False, False, b)):
            results = []
            for c in (plain, ext):
                leaves = [t if t is None else t.detach().requires_grad_(want) for t, want in ((x, want_x), (w, want_w), (bias, True))]
                y = c.linear_fp8(*leaves)
                y.backward(grad)
                results.append((y.detach(), *(None if t is None else t.grad for t in leaves)))
            assert all((a is None) == (q is None) and (a is None or torch.equal(a, q)) for a, q in zip(*results))
            assert [r is not None for r in results[0][1:]] == [want_x, want_w, bias is not None]
    from mini_nccl_b200.ops.distill import _gradient_again

    z, ids, top = torch.randn(4, 90, device="cuda"), torch.randint(0, 90, (4, 5), device="cuda"), torch.randn(4, 5, device="cuda")
    for reduction in (0, 1, 2):
        results = []
        for c in (plain, ext):
            leaf = z.detach().requires_grad_()
            loss = c.distillation(leaf, ids, top, 2.0, reduction, _gradient_again)
            first, = torch.autograd.grad(loss.sum(), [leaf], retain_graph=True)
            dz, = torch.autograd.grad(loss.sum(), [leaf], create_graph=True)
            results.append((loss.detach(), first, dz.detach(), *torch.autograd.grad(dz.square().sum(), [leaf])))
        assert all(torch.equal(a, q) for a, q in zip(*results))
        assert torch.allclose(results[0][1], results[0][2], rtol=1e-4, atol=1e-6)
    x = _input(70, 300, torch.bfloat16).cuda()
    for bad, error in ((lambda c: c.quantize_fp8(x.double(), 1, False, None), TypeError), (lambda c: c.quantize_fp8([1], 1, False, None), TypeError),
                       (lambda c: c.quantize_fp8(x, 2, False, None), ValueError), (lambda c: c.gemm_fp8(*args, None, torch.int8, None, None), TypeError),
                       (lambda c: c.gemm_fp8(*args, None, None, bias[:3], None), ValueError), (lambda c: c.gemm_fp8(args[0], args[0], *args[2:], None, None, None, None), TypeError)):
        for c in (plain, ext):
            with pytest.raises(error):
                bad(c)


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [1, 128])
@pytest.mark.parametrize("M,K", [(100, 24), (5, 130), (128, 128), (250, 300)])
def test_quantize_writes_nothing_behind_its_rows(M, K, rows):
    """Buffers of the C interface with longer rows than they need: bytes behind the padding, and the rows after the last, stay as they were."""
    import mini_nccl_b200 as mn

    x = torch.randn(M, K, device="cuda")
    q, qt = torch.full((M + 1, 512), 7, dtype=torch.uint8, device="cuda"), torch.full((K + 1, 512), 7, dtype=torch.uint8, device="cuda")
    scale, scale_t = torch.empty(_blocks(K) * M, device="cuda"), torch.empty(_blocks(M) * K, device="cuda")
    rc = mn.lib().mncclQuantizeFp8(x.data_ptr(), 7, K, M, K, rows, q.data_ptr(), 512, scale.data_ptr(), qt.data_ptr(), 512, scale_t.data_ptr(), None,
                                   torch.cuda.current_stream().cuda_stream)
    assert rc == 0
    for buffer, (m, k) in ((q, (M, K)), (qt, (K, M))):
        assert bool((buffer[m:] == 7).all()) and bool((buffer[:, -(-k // 16) * 16:] == 7).all())
    want = quantize_fp8(x, block_rows=rows, transposed=True)
    assert torch.equal(q[:M, :K], want[0].view(torch.uint8)) and torch.equal(qt[:K, :M], want[2].view(torch.uint8))


# ---- refusals


def test_entry_points_refuse_bad_arguments():
    import mini_nccl_b200 as mn

    L = mn.lib()
    p = C.c_void_p(4096)   # never looked at: every call below is refused before anything is launched
    q = [p, 9, 128, 4, 128, 1, p, 128, p, None, 0, None, None, None]
    for at, value, code in ((0, None, -1), (6, None, -1), (8, None, -1), (3, 0, -1), (4, -1, -1), (1, 3, -2), (2, 64, -2), (5, 2, -2), (6, C.c_void_p(4097), -2), (7, 120, -2),
                            (7, 112, -2), (4, 65536 * 128, -2), (12, p, -2)):
        bad = list(q)
        bad[at] = value
        assert L.mncclQuantizeFp8(*bad) == code, (at, value)
    assert L.mncclQuantizeFp8(*q[:9], p, 16, None, None, None) == -1 and L.mncclQuantizeFp8(*q[:9], p, 8, p, None, None) == -2
    assert L.mncclSumBlocks(None, 1, 8, p, 9, None) == -1 and L.mncclSumBlocks(p, 0, 8, p, 9, None) == -1 and L.mncclSumBlocks(p, 1, 8, p, 8, None) == -2
    g = [p, 128, p, 1, 4, 1, p, 128, p, 1, 1, 128, p, 64, 9, None, 4, 64, 128, None]
    for at, value, code in ((0, None, -1), (2, None, -1), (6, None, -1), (8, None, -1), (12, None, -1), (16, 0, -1), (17, 0, -1), (18, -5, -1), (0, C.c_void_p(4100), -2), (1, 120, -2),
                            (7, 112, -2), (5, 64, -2), (11, 0, -2), (13, 63, -2), (14, 8, -2)):
        bad = list(g)
        bad[at] = value
        assert L.mncclGemmFp8(*bad) == code, (at, value)


def test_cpu_tensors_are_refused():
    x = torch.zeros(4, 128)
    with pytest.raises(TypeError, match="CUDA"):
        quantize_fp8(x)
    with pytest.raises(TypeError, match="CUDA"):
        gemm_fp8(x.to(E4M3), torch.ones(4, 1), x.to(E4M3), torch.ones(4, 1))
    with pytest.raises(TypeError, match="CUDA"):
        linear_fp8(x, x)


@pytest.mark.gpu
def test_sizes_behind_32_bit_indices_are_refused():
    one = torch.zeros(1, device="cuda")   # matrices that are one element over and over
    w = torch.zeros(8, 16, device="cuda")
    for bad in (lambda: quantize_fp8(torch.zeros(1, 65535 * 128 + 1, device="cuda")),
                lambda: linear_fp8(one.expand(2**31, 16), w), lambda: linear_fp8(one.expand(2**16, 2**15, 16), w),
                lambda: linear_fp8(w, one.expand(65535 * 128 + 1, 16))):
        with pytest.raises(ValueError, match="at most"):
            bad()


@pytest.mark.gpu
def test_refusals():
    x = torch.zeros(40, 256, device="cuda")
    for bad, error in ((lambda: quantize_fp8(x.double()), TypeError), (lambda: quantize_fp8(x.t()), ValueError), (lambda: quantize_fp8(x[0]), ValueError),
                       (lambda: quantize_fp8(x, block_rows=64), ValueError), (lambda: quantize_fp8(x[:1].expand(40, 256)), ValueError),
                       (lambda: quantize_fp8(x.to(E4M3)), TypeError)):
        with pytest.raises(error):
            bad()
    a, sa, b, sb = _whole(40, 256, 1), torch.ones(40, 2, device="cuda"), _whole(200, 256, 2), torch.ones(2, 2, device="cuda")
    out = torch.empty(40, 200, device="cuda")
    for bad, error in ((lambda: gemm_fp8(a.float(), sa, b, sb), TypeError), (lambda: gemm_fp8(a, sa, b[:, :128], sb), ValueError),
                       (lambda: gemm_fp8(a, sa[:39], b, sb), ValueError), (lambda: gemm_fp8(a, sa[:, :1], b, sb), ValueError), (lambda: gemm_fp8(a, sa.double(), b, sb), TypeError),
                       (lambda: gemm_fp8(a, sa.cpu(), b, sb), TypeError), (lambda: gemm_fp8(a, sa, b, sb, out=out[:, :100]), ValueError),
                       (lambda: gemm_fp8(a, sa, b, sb, out=out.t().contiguous().t()), ValueError), (lambda: gemm_fp8(a, sa, b, sb, out=out.double()), TypeError),
                       (lambda: gemm_fp8(a, sa, b, sb, out_dtype=torch.int32), TypeError), (lambda: gemm_fp8(a, sa, b, sb, out=out, out_dtype=torch.bfloat16), ValueError),
                       (lambda: gemm_fp8(a, sa, b, sb, out=out, bias=torch.zeros(200, device="cuda").half()), ValueError),
                       (lambda: gemm_fp8(a, sa, b, sb, out=out, bias=torch.zeros(400, device="cuda")[::2]), ValueError),
                       (lambda: gemm_fp8(a[:, 1:], sa, b[:, 1:], sb), ValueError), (lambda: gemm_fp8(a.view(torch.uint8).view(torch.float8_e5m2), sa, b, sb), TypeError)):
        with pytest.raises(error):
            bad()
    w = torch.zeros(8, 256, device="cuda")
    for bad, error in ((lambda: linear_fp8(x, w.half()), TypeError), (lambda: linear_fp8(x, w[:, :128]), ValueError), (lambda: linear_fp8(x, w, w[:, 0].cpu()), TypeError),
                       (lambda: linear_fp8(x, w, x[0, :9]), ValueError), (lambda: linear_fp8(x[:, :0], w[:, :0]), ValueError), (lambda: linear_fp8(x.double(), w.double()), TypeError)):
        with pytest.raises(error):
            bad()
