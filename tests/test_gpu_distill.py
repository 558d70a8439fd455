"""Distillation from a teacher's top logits against its definition in 64 bits, token by token.

Tolerances.  A row's statistics: exponents are differences of fp32 numbers times a constant (three roundings, 3 * 2^-24 of an exponent of
at most 90 before the result underflows: 1.6e-5 of terms that small, 3e-6 of those above e^-16), 2^-22 for the exponential and fp32 sums: 1e-5 of the
sum of magnitudes covers the loss.  A gradient is that far off before its rounding, half a step of its type."""
import math

import pytest
import torch
import torch.nn.functional as F

from mini_nccl_b200.ops import distillation_loss, lm_head_distillation
from mini_nccl_b200.ops.distill import _LmHeadDistillation, _native, _reference

TYPES = [torch.bfloat16, torch.float16, torch.float32]
INF, NAN = float("inf"), float("nan")


def _define(logits, ids, top, tau, reduction="mean", grad=1.0):
    """(loss, gradient) by the formula, in Python for each token."""
    V, K = logits.shape[-1], ids.shape[-1]
    z, i, t = logits.detach().double().cpu().reshape(-1, V), ids.cpu().reshape(-1, K), top.double().cpu().reshape(-1, K)
    grad = torch.as_tensor(grad, dtype=torch.float64).cpu().reshape(-1).expand(z.shape[0]) if not isinstance(grad, float) else torch.full((z.shape[0],), grad, dtype=torch.float64)
    losses, d, counts = torch.zeros(z.shape[0], dtype=torch.float64), torch.zeros_like(z), torch.zeros(z.shape[0], dtype=torch.bool)
    size = torch.zeros(z.shape[0], dtype=torch.float64)
    for r in range(z.shape[0]):
        there = (i[r] >= 0) & (t[r] != -INF)
        if not bool(there.any()):
            continue
        counts[r] = True
        at, log_p, log_q = i[r][there], torch.log_softmax(t[r][there] / tau, 0), torch.log_softmax(z[r] / tau, 0)
        if bool((at >= V).any()):
            losses[r], d[r] = NAN, NAN
            continue
        p = log_p.exp()
        terms = torch.where(p > 0, p * (log_p - log_q[at]), 0.0) * tau * tau
        losses[r], size[r] = terms.sum(), (p * (log_p.abs() + log_q[at].abs()).nan_to_num(0, 0, 0)).sum() * tau * tau
        d[r] = log_q.exp()
        for k in range(len(at)):
            d[r, at[k]] -= p[k]
        d[r] *= tau * grad[r]
    n = counts.sum()
    if reduction == "mean":
        return losses.sum() / n, torch.where(counts.unsqueeze(1), d / n, 0.0).view(logits.shape), size.sum() / n
    return (losses.sum(), d.view(logits.shape), size.sum()) if reduction == "sum" else (losses.view(logits.shape[:-1]), d.view(logits.shape), size.view(logits.shape[:-1]))


def _case(lead, V, K, dtype=torch.float32, seed=0, repeats=False, empty=0.3, device="cuda", spread=3.0):
    g = torch.Generator().manual_seed(seed)
    logits = (torch.randn(*lead, V, generator=g) * spread).to(dtype)
    ids = torch.randint(0, V, (*lead, K), generator=g)
    if repeats and K > 2:
        ids[..., K // 2] = ids[..., 0]
        ids[..., K - 1] = ids[..., 0]
    top = torch.randn(*lead, K, generator=g) * 2 + 5
    ids[torch.rand(ids.shape, generator=g) < 0.2] = -1
    top[torch.rand(ids.shape, generator=g) < 0.1] = -INF
    ids[torch.rand(lead, generator=g) < empty] = -100
    first = ids.view(-1, K)[0], top.view(-1, K)[0]
    first[0][0], first[1][0] = 3 % V, 5.0
    return logits.to(device).requires_grad_(), ids.to(device), top.to(device)


def _check(loss, d, want, dtype, tau=1.0, grad=1.0):
    loss, d = loss.detach().double().cpu(), d.double().cpu()
    # However small the loss: each of the two sums is of exponentials off by 2^-22 of themselves and is rounded to 2^-24, so their logarithms, which
    # the loss takes the difference of, are off by 2 * (2^-22 + 2^-24) < 2^-20, times tau squared.
    assert bool(((loss - want[0]).abs() <= 1e-5 * (want[2] + want[0].abs()) + tau * tau * 2.0 ** -20).all()), (loss, want[0])
    # the softmax and the entries are each 1e-5 off at most; their difference is rounded once; below the type's normal numbers steps are fixed
    g = torch.as_tensor(grad, dtype=torch.float64).abs().max() * tau
    f = torch.finfo(dtype)
    assert bool(((d - want[1]).abs() <= want[1].abs() * f.eps / 2 + 1e-5 * (want[1].abs() + g * _softmax_bound(want[1], g)) + f.smallest_normal * f.eps).all())


def _softmax_bound(d, g):
    """Where entries cancel against the softmax both are below 1; elsewhere the gradient is the softmax itself."""
    return torch.where(d <= 0, 1.0, (d / g).clamp_max(1.0)) if float(g) else 0.0


SHAPES = [((1,), 1, 1), ((1,), 7, 3), ((2, 3), 8, 2), ((5,), 129, 16), ((3,), 1000, 8), ((4, 16), 2049, 5), ((33,), 4099, 40), ((3,), 50257, 64),
          ((2,), 131072, 300), ((1,), 30011, 1024), ((300,), 515, 7)]


@pytest.mark.gpu
@pytest.mark.parametrize("lead,V,K", SHAPES)
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("tau,reduction", [(1.0, "mean"), (2.0, "sum"), (0.5, "none")])
def test_loss_and_gradient(lead, V, K, dtype, tau, reduction):
    logits, ids, top = _case(lead, V, K, dtype, seed=V + K, repeats=True)
    assert _native(logits, ids, top)
    loss = distillation_loss(logits, ids, top, temperature=tau, reduction=reduction)
    assert loss.dtype == torch.float32 and loss.shape == (lead if reduction == "none" else ())
    grad = torch.rand(loss.shape, generator=torch.Generator().manual_seed(1)) + 0.5
    d, = torch.autograd.grad(loss, [logits], grad.cuda(), retain_graph=True)
    assert d.dtype == dtype and d.shape == logits.shape
    _check(loss, d, _define(logits, ids, top, tau, reduction, grad), dtype, tau, grad)
    again, = torch.autograd.grad(loss, [logits], grad.cuda())
    assert torch.equal(d, again)


@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
@pytest.mark.parametrize("V,K", [(1, 1), (129, 16), (1000, 40)])
def test_plain_operators_on_the_cpu(V, K, reduction):
    for dtype in (torch.float64, torch.float32, torch.bfloat16):
        logits, ids, top = _case((2, 5), V, K, dtype, seed=V, repeats=True, device="cpu")
        assert not _native(logits, ids, top)
        loss = distillation_loss(logits, ids, top, temperature=1.5, reduction=reduction)
        d, = torch.autograd.grad(loss, [logits], torch.ones_like(loss))
        _check(loss, d, _define(logits, ids, top, 1.5, reduction), dtype, 1.5)


def test_gradient_is_that_of_differences():
    logits, ids, top = _case((7,), 50, 5, torch.float64, seed=2, repeats=True, device="cpu")
    assert torch.autograd.gradcheck(lambda z: distillation_loss(z, ids, top, 1.3), [logits])


@pytest.mark.gpu
def test_gradient_of_the_kernels_is_that_of_differences():
    """(f(z + h) - f(z - h)) / 2h in fp32: f is off by 1e-5 of the size of its terms, third derivatives are below tau^-1 of the row's loss scale."""
    logits, ids, top = _case((6,), 300, 5, seed=8)
    tau, h = 1.0, 0.05
    d, = torch.autograd.grad(distillation_loss(logits, ids, top, tau, "sum"), [logits])
    g = torch.Generator().manual_seed(4)
    for _ in range(4):
        u = torch.randn(logits.shape, generator=g).cuda()
        u /= u.abs().max(dim=1, keepdim=True).values
        up, down = (distillation_loss((logits + s * h * u).detach(), ids, top, tau, "none").double() for s in (1, -1))
        moved, want = (up - down).sum() / (2 * h), (d.double() * u.double()).sum()
        size = 2 * 1e-5 * float(_define(logits, ids, top, tau, "sum")[2]) / (2 * h)
        # |third derivative of log sum exp along u| <= 2 * max|u|^3 = 2 a token, h^2 / 6 of it
        assert abs(float(moved - want)) <= size + 6 * 2 * h * h / 6 + 1e-5


def _same_nans(got, ref):
    got, ref = got.detach().float().cpu(), ref.detach().float().cpu()
    assert torch.equal(torch.isnan(got), torch.isnan(ref)) and torch.equal(torch.isinf(got), torch.isinf(ref))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_values_that_are_not_finite(dtype):
    """The kernels and the plain operators agree; tokens that count for nothing may hold anything."""
    V, K = 700, 6
    logits, ids, top = (t.detach().clone() for t in _case((24,), V, K, dtype, seed=3, empty=0.0))
    ids[:, :] = torch.arange(K, device="cuda") * 100
    top[:, :] = torch.arange(K, device="cuda").float()
    low = torch.finfo(dtype).min
    logits[0, 650], logits[1, 650], logits[2, 650] = NAN, INF, -INF
    logits[3], logits[4], logits[5, 200], logits[6] = -INF, low, -INF, INF
    top[7, 2], top[8, 2], top[9, 2] = NAN, INF, -INF
    top[10], ids[11], ids[12, 3] = -INF, -1, V
    ids[13, 3] = 2**40
    logits[10], logits[11, ::2] = NAN, INF
    top[14, :] = torch.finfo(torch.float32).min
    logits[15] = torch.finfo(dtype).max
    logits[16, :600], logits[17, 200] = -INF, low
    top[18, 1:] = -2e30
    logits[18, 100:600] = -INF       # entries of weight 0 on classes that the student cannot reach
    ids[19, 2], top[19, 2] = V + 5, -INF
    zs = logits.clone().requires_grad_(), logits.clone().requires_grad_()
    losses = distillation_loss(zs[0], ids, top, 1.0, "none"), _reference(zs[1], ids, top, 1.0, "none")
    _same_nans(*losses)
    assert torch.equal(torch.isnan(losses[0]).nonzero().flatten().cpu(), torch.tensor([0, 1, 3, 6, 7, 8, 12, 13]))
    ds = [torch.autograd.grad(loss.sum(), [z])[0] for loss, z in zip(losses, zs)]
    fine = [2, 4, 5, 9, 10, 11, 14, 15, 16, 17, 18, 19, 20, 21, 22, 23]
    assert torch.isfinite(ds[0][fine]).all() and not ds[0][[10, 11]].any()
    assert torch.isnan(ds[0][[0, 1, 3, 6, 12, 13]]).all(1).all()
    entries = torch.zeros(V, dtype=torch.bool, device="cuda")
    entries[ids[7]] = True           # a teacher that is not finite: its weights are NaN, the softmax is not
    assert torch.equal(torch.isnan(ds[0][[7, 8]]), entries.expand(2, V))
    if dtype == torch.float32:
        want = _define(logits[[2, 4, 9, 14, 15, 17, 18, 19]], ids[[2, 4, 9, 14, 15, 17, 18, 19]], top[[2, 4, 9, 14, 15, 17, 18, 19]], 1.0, "none")
        _check(losses[0][[2, 4, 9, 14, 15, 18, 19]], ds[0][[2, 4, 9, 14, 15, 18, 19]], [w[[0, 1, 2, 3, 4, 6, 7]] for w in want], dtype)
    for reduction in ("mean", "sum"):
        assert torch.isnan(distillation_loss(logits, ids, top, 1.0, reduction))
    nothing = torch.full_like(ids, -1)
    z = logits.clone().requires_grad_()
    loss = distillation_loss(z, nothing, top)
    assert torch.isnan(loss) and not torch.autograd.grad(loss, [z])[0].any()
    assert float(distillation_loss(z.detach(), nothing, top, reduction="sum")) == 0.0


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_layouts_give_one_result(dtype):
    V, K = 1003, 12
    logits, ids, top = _case((3, 20), V, K, dtype, seed=9)

    def both(z, ids=ids, top=top):
        z = z.detach().requires_grad_()
        loss = distillation_loss(z, ids, top, 1.5)
        return loss.detach(), torch.autograd.grad(loss, [z])[0]

    want = both(logits)
    for extra, first in ((5, 0), (1008 - V, 0), (20, 3), (21, 8)):
        wide = torch.full((3, 20, V + extra), NAN, dtype=dtype, device="cuda")
        wide[..., first:first + V] = logits.detach()
        got = both(wide[..., first:first + V])
        assert torch.allclose(got[0], want[0], rtol=1e-6, atol=0) and torch.allclose(got[1].float(), want[1].float(), rtol=2 * torch.finfo(dtype).eps + 1e-5, atol=1e-7)
    for z in (logits.transpose(0, 2).contiguous().transpose(0, 2), logits[:, :1].expand(3, 20, V)):
        one = ids if z.stride(1) else ids[:, :1].expand(3, 20, K), top if z.stride(1) else top[:, :1].expand(3, 20, K)
        got, dense = both(z, *one), both(z.contiguous(), *(t.contiguous() for t in one))
        assert torch.equal(got[0], dense[0]) and torch.equal(got[1], dense[1])
    got = both(logits, ids.int(), top.double())
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = both(logits)
    torch.cuda.synchronize()
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    with torch.autograd.graph.saved_tensors_hooks(lambda s: s.cpu(), lambda s: s.cuda()):
        got = both(logits)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


@pytest.mark.gpu
def test_offsets_behind_32_bits():
    """Logits of more than 2^31 elements, and rows so far apart that offsets pass it: the last rows' losses and gradients are those of these rows alone."""
    T, V, K = 43000, 50257, 5
    few, ids, top = (t.detach() for t in _case((6,), V, K, torch.bfloat16, seed=11))
    logits = torch.zeros(T, V, dtype=torch.bfloat16, device="cuda")
    logits[-6:] = few
    all_ids, all_top = torch.full((T, K), -1, device="cuda"), torch.zeros(T, K, device="cuda")
    all_ids[-6:], all_top[-6:] = ids, top
    few = few.requires_grad_()
    want = distillation_loss(few, ids, top, 2.0, "none")
    dwant, = torch.autograd.grad(want.sum(), [few])
    far = torch.empty(5 * 2**29 + V, dtype=torch.bfloat16, device="cuda").as_strided((6, V), (2**29, 1))
    far.copy_(few.detach())
    for z, i, t in ((logits, all_ids, all_top), (far, ids, top)):
        z = z.requires_grad_()
        got = distillation_loss(z, i, t, 2.0, "none")
        d, = torch.autograd.grad(got.sum(), [z])
        assert torch.allclose(got[-6:], want, rtol=1e-5) and not got[:-6].any()
        assert torch.allclose(d[-6:].float(), dwant.float(), rtol=2 * torch.finfo(torch.bfloat16).eps, atol=1e-7)
        assert len(d) == 6 or not d[:1000].any() and not d[-1006:-6].any()


@pytest.mark.gpu
def test_captured_and_replayed():
    logits, ids, top = (t.detach() for t in _case((40,), 4001, 9, torch.bfloat16, seed=4))
    z, i, t = torch.zeros_like(logits).requires_grad_(), torch.zeros_like(ids), torch.zeros_like(top)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        torch.autograd.grad(distillation_loss(z, i, t, 2.0), [z])
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        loss = distillation_loss(z, i, t, 2.0)
        d, = torch.autograd.grad(loss, [z])
    with torch.no_grad():
        z.copy_(logits), i.copy_(ids), t.copy_(top)
    for _ in range(2):
        graph.replay()
    torch.cuda.synchronize()
    _check(loss, d, _define(logits, ids, top, 2.0), torch.bfloat16, 2.0)


@pytest.mark.gpu
def test_what_autograd_may_do():
    logits, ids, top = _case((9,), 300, 6, seed=6)

    def second(f):
        d, = torch.autograd.grad(f(logits), [logits], create_graph=True)
        return torch.autograd.grad((d ** 2).sum() * 100, [logits])[0]

    got, ref = second(lambda z: distillation_loss(z, ids, top, 1.5)), second(lambda z: _reference(z, ids, top, 1.5, "mean"))
    assert float((got - ref).norm() / ref.norm()) <= 1e-5
    seen = []
    torch.func.vmap(lambda z: (seen.append(_native(z, ids, top)), distillation_loss(z, ids[0], top[0]))[1])(logits.detach())
    assert seen == [False]
    with torch.no_grad():
        assert not distillation_loss(logits, ids, top).requires_grad
    loss = distillation_loss(logits, ids, top)
    with torch.no_grad():
        logits.mul_(2)
    with pytest.raises(RuntimeError, match="modified"):
        loss.backward()


@pytest.mark.gpu
@pytest.mark.parametrize("lead,V,d,K", [((3, 5), 65, 16, 4), ((4, 64), 2049, 128, 10), ((130,), 512, 72, 3), ((2, 333), 50257, 128, 20)])
def test_head(lead, V, d, K):
    """Operands whose logits bf16 holds exactly, as for the cross-entropy; the oracle rounds the logits' gradient where the node does."""
    g = torch.Generator().manual_seed(V)
    x = (torch.randint(-2, 3, (*lead, d), generator=g).to(torch.bfloat16) * 0.5).cuda().requires_grad_()
    w = (torch.randint(-1, 2, (V, d), generator=g).to(torch.bfloat16) * 0.25).cuda().requires_grad_()
    _, ids, top = _case(lead, V, K, seed=V + 1, repeats=True)
    loss = _LmHeadDistillation.apply(x, w, ids.view(-1, K), top.view(-1, K), 2.0)
    dx, dw = torch.autograd.grad(loss * 3.0, [x, w])
    logits = x.detach().double().cpu() @ w.detach().double().cpu().t()
    want = _define(logits, ids, top, 2.0, grad=3.0)
    assert abs(float(loss) - float(want[0])) <= 1e-5 * (float(want[2]) + abs(float(want[0])))
    dz = want[1].to(torch.bfloat16).double().view(-1, V)
    rel = lambda got, ref: float((got.double().cpu() - ref).norm() / ref.norm())  # noqa: E731
    bound = 2.0 ** -8   # one rounding to bf16; the library's product over an odd number of classes rounds its slices as well
    assert rel(dx.view(-1, d), dz @ w.detach().double().cpu()) <= bound * (1 if V % 8 == 0 else 3)
    assert rel(dw, dz.t() @ x.detach().double().cpu().view(-1, d)) <= bound
    only, = torch.autograd.grad(_LmHeadDistillation.apply(x.detach(), w, ids.view(-1, K), top.view(-1, K), 2.0) * 3.0, [w])
    assert torch.equal(only, dw)
    plain = lm_head_distillation(x.float(), w.float(), ids, top, 2.0)
    assert abs(float(plain) * 3 - float(loss) * 3) <= 1e-4 * abs(float(want[2])) * 3


def test_head_on_the_cpu_is_the_loss_of_the_projection():
    g = torch.Generator().manual_seed(0)
    x, w = torch.randn(3, 4, 16, generator=g), torch.randn(33, 16, generator=g)
    _, ids, top = _case((3, 4), 33, 5, device="cpu")
    assert torch.equal(lm_head_distillation(x, w, ids, top, 2.0), distillation_loss(F.linear(x, w), ids, top, 2.0))


def test_refusals():
    import ctypes as C

    import mini_nccl_b200 as mn

    z, ids, top = torch.zeros(3, 9), torch.zeros(3, 2, dtype=torch.int64), torch.zeros(3, 2)
    for bad, error in ((lambda: distillation_loss(z, ids[:2], top), ValueError), (lambda: distillation_loss(z, ids, top[:, :1]), ValueError), (lambda: distillation_loss(z, ids[:, :0], top[:, :0]), ValueError),
                       (lambda: distillation_loss(z, ids.float(), top), TypeError), (lambda: distillation_loss(z, ids, top.long()), TypeError), (lambda: distillation_loss(z, ids, top, 0.0), ValueError),
                       (lambda: distillation_loss(z, ids, top, NAN), ValueError), (lambda: distillation_loss(z, ids, top, reduction="batch"), ValueError), (lambda: distillation_loss(z.long(), ids, top), TypeError),
                       (lambda: distillation_loss(z[:, :0], ids, top), ValueError), (lambda: distillation_loss(z, [0], top), TypeError), (lambda: lm_head_distillation(z, z.t(), ids, top), ValueError)):
        with pytest.raises(error):
            bad()
    L = mn.lib()
    p = C.c_void_p(4096)   # never looked at
    f = [p, 9, 64, 4, 64, p, p, 8, 1.0, p, p, p, p, p, p, p, None]
    for at, value, code in ((0, None, -1), (5, None, -1), (6, None, -1), (9, None, -1), (10, None, -1), (11, None, -1), (12, None, -1), (15, None, -1), (3, 0, -1), (4, 0, -1), (7, 0, -1),
                            (7, 1025, -2), (8, 0.0, -2), (8, NAN, -2), (1, 8, -2), (2, 63, -2), (0, C.c_void_p(4097), -2), (10, C.c_void_p(4100), -2)):
        bad = list(f)
        bad[at] = value
        assert L.mncclDistillForward(*bad) == code, (at, value)
    b = [p, 9, 64, 4, 64, p, p, 8, 1.0, p, p, p, 0, None, p, 64, None]
    for at, value, code in ((0, None, -1), (5, None, -1), (6, None, -1), (9, None, -1), (10, None, -1), (11, None, -1), (14, None, -1), (7, 2000, -2), (8, INF, -2), (1, 0, -2), (15, 63, -2),
                            (14, C.c_void_p(4097), -2)):
        bad = list(b)
        bad[at] = value
        assert L.mncclDistillBackward(*bad) == code, (at, value)
    assert math.isfinite(float(distillation_loss(z, ids, top)))
