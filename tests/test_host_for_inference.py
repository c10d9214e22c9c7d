"""The public rotation kernels refuse what torch is asked to follow through them, before they ask for a GPU."""

import pytest
import torch
from torch.autograd import forward_ad

from minillm.model import kernels

BF16 = torch.bfloat16


def rotary(x, **kw):
    a = dict(q=x, k=torch.zeros(2, 2, 3, 64, dtype=BF16), positions=torch.zeros(2, 3, dtype=torch.int64), inv_freq=torch.zeros(32)) | kw
    return kernels.rotary(**a)


def qk_norm_rope(x, **kw):
    table, weight = torch.zeros(2, 3, 64, dtype=BF16), torch.ones(64, dtype=BF16)
    a = dict(q=x, k=torch.zeros(2, 2, 3, 64, dtype=BF16), cos=table, sin=table, q_weight=weight, k_weight=weight, eps=1e-5) | kw
    return kernels.qk_norm_rope(**a)


CALLS = pytest.mark.parametrize("call,others", [(rotary, ("k", "inv_freq")), (qk_norm_rope, ("k", "cos", "sin", "q_weight", "k_weight"))])
SHAPES = dict(k=(2, 2, 3, 64), cos=(2, 3, 64), sin=(2, 3, 64), q_weight=(64,), k_weight=(64,), inv_freq=(32,))


def operand(name):
    return torch.zeros(SHAPES[name], dtype=torch.float32 if name == "inv_freq" else BF16)


@CALLS
def test_tangents(call, others):
    q = torch.zeros(2, 4, 3, 64, dtype=BF16)
    with forward_ad.dual_level():
        with pytest.raises(RuntimeError, match="forward-mode"):
            call(forward_ad.make_dual(q, torch.ones_like(q)))
        for name in others:
            x = operand(name)
            with pytest.raises(RuntimeError, match="forward-mode"):
                call(q, **{name: forward_ad.make_dual(x, torch.ones_like(x))})
        with torch.no_grad(), pytest.raises(RuntimeError, match="forward-mode"):  # no_grad does not drop a tangent
            call(forward_ad.make_dual(q, torch.ones_like(q)))
        with pytest.raises(ValueError, match="on a GPU"):  # none of the operands has one
            call(q)


@CALLS
def test_gradients(call, others):
    q = torch.zeros(2, 4, 3, 64, dtype=BF16)
    with pytest.raises(RuntimeError, match="no gradient"):
        call(q.clone().requires_grad_())
    for name in others:
        with pytest.raises(RuntimeError, match="no gradient"):
            call(q, **{name: operand(name).requires_grad_()})
    with torch.no_grad(), pytest.raises(ValueError, match="on a GPU"):
        call(q.clone().requires_grad_())


@pytest.mark.filterwarnings("ignore::torch.jit.TracerWarning")
@CALLS
def test_traces_and_transforms(call, others):
    q = torch.zeros(2, 4, 3, 64, dtype=BF16)
    with pytest.raises(RuntimeError, match="traced or transformed"):
        torch.jit.trace(lambda x: call(x), (q,), check_trace=False)
    with pytest.raises(RuntimeError, match="traced or transformed|forward-mode"):
        torch.func.jvp(lambda x: call(x), (q,), (torch.ones_like(q),))
    with pytest.raises(RuntimeError, match="traced or transformed"):
        torch.func.vmap(lambda x: call(x))(q[None])
    with pytest.raises(RuntimeError, match="traced or transformed|no gradient"):
        torch.func.grad(lambda x: call(x)[0].sum())(q)
