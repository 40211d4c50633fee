"""When wave_attn_q8 may pass by the dispatcher: only where the dispatcher would do nothing but call the kernel."""
from __future__ import annotations

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode
from torch.autograd import forward_ad as fad
from torch.overrides import TorchFunctionMode
from torch.utils._python_dispatch import TorchDispatchMode

import __graft_entry__

__graft_entry__.load_package()
from wavefront_decoding_b200 import attention as wa  # noqa: E402
from wavefront_decoding_b200 import ops  # noqa: E402
from wavefront_decoding_b200 import runtime as rt  # noqa: E402


class Sub(torch.Tensor):
    pass


class Dispatch(TorchDispatchMode):
    def __torch_dispatch__(self, func, types, args=(), kwargs=None):
        return func(*args, **(kwargs or {}))


class Function(TorchFunctionMode):
    def __torch_function__(self, func, types, args=(), kwargs=None):
        return func(*args, **(kwargs or {}))


def cpu_args():
    q, kv = torch.zeros((1, 2, 64)), torch.zeros((1, 2, 64))
    K = torch.zeros((1, 1, 8, 2, 64), dtype=torch.uint8).view(torch.float8_e4m3fn)
    e = torch.zeros((1, 1, 2, 8), dtype=torch.int8)
    return [q, kv, kv.clone(), K, K.clone(), e, e.clone(), torch.tensor([[0, 0, 0, 1, 0]], dtype=torch.int32), 1]


@pytest.fixture
def direct(monkeypatch):
    """wave_attn_q8 on CPU tensors: what reaches the kernel's host code without the dispatcher."""
    seen = []
    monkeypatch.setattr(ops, "_wave_attn_q8_out_cuda", lambda *a: seen.append(a))
    monkeypatch.setattr(rt, "require_cuda", lambda *t: torch.device("cpu"))
    return seen


def bypassed(direct, call):
    """Whether `call` reached the kernel's host code directly (the op has no CPU kernel: the dispatcher refuses)."""
    del direct[:]
    try:
        call()
    except (NotImplementedError, RuntimeError):
        assert not direct
    return bool(direct)


def test_a_plain_call_goes_directly(direct):
    a = cpu_args()
    assert bypassed(direct, lambda: wa.wave_attn_q8(*a))
    with torch.no_grad():
        assert bypassed(direct, lambda: wa.wave_attn_q8(*a))
    with torch.inference_mode():
        b = cpu_args()
        assert bypassed(direct, lambda: wa.wave_attn_q8(*b))
        assert bypassed(direct, lambda: wa.wave_attn_q8(*a, lens=torch.zeros((1, 1), dtype=torch.int32)))


def test_modes_see_the_call(direct):
    a = cpu_args()
    for mode in (Dispatch(), Function(), FakeTensorMode(allow_non_fake_inputs=True)):
        with mode:
            assert not ops.plain_eager(a[:3], a[3:8])
            assert not bypassed(direct, lambda: wa.wave_attn_q8(*a))
    for prof in (torch.profiler.profile(), torch.autograd.profiler.profile()):
        with prof:
            assert not bypassed(direct, lambda: wa.wave_attn_q8(*a))
    assert bypassed(direct, lambda: wa.wave_attn_q8(*a))


@pytest.mark.parametrize("make,at", [(m, i) for m in ("subclass", "requires_grad", "functional", "negated", "dual")
                                     for i in (0, 1, 2)] + [("subclass", 4), ("subclass", 7)])
def test_a_tensor_that_is_not_plain_sends_the_call_to_the_dispatcher(direct, make, at):
    a = cpu_args()
    if make == "subclass":
        a[at] = a[at].as_subclass(Sub)
    elif make == "requires_grad":
        a[at].requires_grad_()
    elif make == "functional":
        a[at] = torch._to_functional_tensor(a[at])
    elif make == "negated":
        a[at] = torch.view_as_complex(torch.zeros((1, 2, 64, 2))).conj().imag
        assert a[at].is_neg()
    else:
        with fad.dual_level():
            a[at] = fad.make_dual(a[at], torch.ones_like(a[at]))
            assert not bypassed(direct, lambda: wa.wave_attn_q8(*a))
        return
    assert not ops.plain_eager(a[:3], a[3:8])
    assert not bypassed(direct, lambda: wa.wave_attn_q8(*a))


def test_transforms_see_the_call(direct):
    a = cpu_args()
    taken = []

    def f(x):
        taken.append(ops.plain_eager(a[:3], a[3:8]) or ops.plain_eager((x,), ()))
        return x.sum()

    torch.vmap(f)(torch.zeros((3, 2)))
    torch.func.grad(f)(torch.zeros(3))
    torch.func.jvp(f, (torch.zeros(3),), (torch.ones(3),))
    torch.jit.trace(f, (torch.zeros(3),), check_trace=False)
    assert len(taken) >= 4 and not any(taken)
