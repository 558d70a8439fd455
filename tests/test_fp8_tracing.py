"""The 8-bit operators while something records, replaces or watches the single operators: what would record the allocation of a result without the kernel
that fills it is refused, what looks on gets the numbers as ever."""
import pytest
import torch
import torch.utils.checkpoint
from torch.fx.experimental.proxy_tensor import make_fx
from torch._subclasses import FakeTensorMode
from torch.utils.flop_counter import FlopCounterMode

from mini_nccl_b200.models import GPT2Config, GPT2Model
from mini_nccl_b200.ops import gemm_fp8, linear_fp8, quantize_fp8

E4M3 = torch.float8_e4m3fn


class Tagged(torch.Tensor):
    """A subclass whose results are of its kind."""


class Wrapper(torch.Tensor):
    """A subclass that has every operator's calls for itself, and no memory."""

    __torch_function__ = torch._C._disabled_torch_function_impl

    @staticmethod
    def __new__(cls, t):
        return torch.Tensor._make_wrapper_subclass(cls, t.shape, dtype=t.dtype, device=t.device)

    @classmethod
    def __torch_dispatch__(cls, func, types, args=(), kwargs=None):
        raise AssertionError("nothing is to reach an operator")


class Quiet(torch.nn.Parameter):
    """A parameter class of a user's own: no rules beyond a parameter's."""


def _calls(device):
    x, w = (torch.linspace(-1, 1, rows * 256, device=device).view(rows, 256) for rows in (8, 130))
    q, s, v = x.to(E4M3), torch.ones(8, 2, device=device), torch.ones(130, 2, device=device)
    return {"quantize_fp8": (lambda t: quantize_fp8(t)[0], x), "gemm_fp8": (lambda t: gemm_fp8(q, t, w.to(E4M3), v), s), "linear_fp8": (lambda t: linear_fp8(t, w), x)}


def _refusals(device):
    for name, (f, t) in _calls(device).items():
        with pytest.raises(RuntimeError, match=name + " has no rule"):
            torch.jit.trace(f, t)
        with pytest.raises(RuntimeError, match=name + " has no rule"):
            make_fx(f)(t)
        with pytest.raises(RuntimeError, match=name + " has no rule"):
            torch.func.vmap(f)(t.unsqueeze(0))
        with FakeTensorMode(allow_non_fake_inputs=True) as mode:
            for fake in (t, mode.from_tensor(t)):
                with pytest.raises(RuntimeError, match=name + " has no rule"):
                    f(fake)
        fake = mode.from_tensor(t)
        for other in (t.as_subclass(Tagged), Wrapper(t), fake):
            with pytest.raises(TypeError, match=name + " has no rule"):
                f(other)
    with pytest.raises(RuntimeError, match="has no rule"):
        torch.jit.trace(GPT2Model(GPT2Config(n_layer=1, d_model=64, n_head=1, vocab_size=8, seq_len=4, linear="fp8")).to(device), torch.zeros(1, 4, dtype=torch.int64, device=device))


def test_recorded_calls_are_refused_before_anything_else():
    _refusals("cpu")


@pytest.mark.gpu
def test_recorded_calls_are_refused():
    _refusals("cuda")


@pytest.mark.gpu
def test_calls_that_are_watched_give_the_same_numbers():
    g = torch.Generator(device="cuda").manual_seed(1)
    x, w = (torch.randn(*shape, generator=g, device="cuda").requires_grad_() for shape in ((40, 300), (136, 300)))
    grad = torch.randn(40, 136, generator=g, device="cuda")

    def step(f=linear_fp8, w=w):
        y = f(x, w)
        return [y.detach(), *torch.autograd.grad(y, [x, w], grad)]

    want = step()
    with FlopCounterMode(display=False):
        got = step()
    assert all(torch.equal(p, q) for p, q in zip(got, want))
    with torch.device("cuda"):
        got = step()
    assert all(torch.equal(p, q) for p, q in zip(got, want))

    def keep(ctx, op, *args, **kwargs):
        return torch.utils.checkpoint.CheckpointPolicy.PREFER_RECOMPUTE

    def checkpointed(x, w):
        contexts = lambda: torch.utils.checkpoint.create_selective_checkpoint_contexts(keep)  # noqa: E731
        return torch.utils.checkpoint.checkpoint(linear_fp8, x, w, use_reentrant=False, context_fn=contexts)

    got = step(checkpointed)
    assert all(torch.equal(p, q) for p, q in zip(got, want))
    got = step(w=Quiet(w.detach()))
    assert all(torch.equal(p, q) for p, q in zip(got, want))


@pytest.mark.gpu
@pytest.mark.parametrize("backend", ["eager", "aot_eager"])
def test_compiled_calls_run_as_they_are(backend):
    """The compiler leaves the call outside of its graphs."""
    g = torch.Generator(device="cuda").manual_seed(2)
    x, w = (torch.randn(*shape, generator=g, device="cuda").requires_grad_() for shape in ((24, 256), (130, 256)))
    f = lambda x, w: torch.relu(linear_fp8(x * 2, w) + 1)  # noqa: E731
    got, want = torch.compile(f, backend=backend)(x, w), f(x, w)
    assert torch.equal(got, want) and all(torch.equal(p, q) for p, q in zip(torch.autograd.grad(got.sum(), [x, w]), torch.autograd.grad(want.sum(), [x, w])))
