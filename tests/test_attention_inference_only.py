"""Packed and prefix attention refuse operands of which something is to be recorded (CPU): it would be lost."""

import functools

import pytest
import torch
from torch.autograd import forward_ad

BF16 = torch.bfloat16


def _calls():
    """Each operand's place in a call of each, as a function of that operand."""
    import ltxk

    q, k = torch.zeros(4, 128, dtype=BF16), torch.zeros(4, 64, dtype=BF16)
    offsets = torch.tensor([0, 4], dtype=torch.int32)
    packed, prefix = (q, k, k), (q[None], k[None], k[None], k, k)

    def with_(operands, i, x):
        return [*operands[:i], x, *operands[i + 1:]]

    for i in range(3):
        yield packed[i], functools.partial(lambda i, x: ltxk.packed_attention(*with_(packed, i, x), 2, offsets, 1), i)
    for i in range(5):
        yield prefix[i], functools.partial(lambda i, x: ltxk.prefix_attention(*with_(prefix, i, x), 2, 1), i)


@pytest.mark.parametrize("i", range(8))
def test_derivatives_are_refused(i):
    """A gradient to record, of a parameter and of a result, and a tangent; without one the call goes on (to the device
    check: this is the CPU)."""
    x, call = list(_calls())[i]
    for y in (x.clone().requires_grad_(), torch.nn.Parameter(x.clone()), x.clone().requires_grad_() * 2):
        with pytest.raises(RuntimeError, match="for inference.*gradient"):
            call(y)
        with torch.no_grad(), pytest.raises(RuntimeError, match="ROCm device"):
            call(y)
        with torch.inference_mode(), pytest.raises(RuntimeError, match="ROCm device"):
            call(y)
    with pytest.raises(RuntimeError, match="ROCm device"):
        call(x)
    with forward_ad.dual_level():
        with pytest.raises(RuntimeError, match="for inference.*derivative"):
            call(forward_ad.make_dual(x, x))
        with pytest.raises(RuntimeError, match="ROCm device"):
            call(x)


@pytest.mark.parametrize("i", range(8))
def test_transforms_and_tracers_are_refused(i):
    from torch.fx.experimental.proxy_tensor import make_fx

    x, call = list(_calls())[i]
    with pytest.raises(RuntimeError, match="for inference"):
        torch.func.jvp(call, (x,), (x,))
    with pytest.raises(RuntimeError, match="for inference"):
        torch.func.grad(lambda t: call(t).float().sum())(x)
    with pytest.raises(RuntimeError, match="for inference"):
        torch.func.vmap(call)(x[None])
    with pytest.raises(RuntimeError, match="for inference"):
        make_fx(lambda t: call(t))(x)
    with pytest.raises(RuntimeError, match="for inference"):
        torch.jit.trace(lambda t: call(t), x, check_trace=False)
