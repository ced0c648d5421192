"""Calls of scarches_amd.ops from inside torch's transformations, which see no more than an allocation of a kernel that is
launched through addresses: refused instead of answered wrongly (no GPU needed)."""
import pytest
import torch
from torch.autograd import forward_ad

from scarches_amd import ops


def t(*shape, dtype=torch.float32):
    return torch.ones(*shape, dtype=dtype)


W8, W4 = torch.ones(5, 4, dtype=torch.int8), torch.ones(4, 4, dtype=torch.int8)
# the operator as a function of one fp32 tensor [3, 4] that it differentiates, or should
CALLS = {
    "layer_norm": lambda x: ops.layer_norm(x, t(4), t(4)),
    "layer_norm weight": lambda x: ops.layer_norm(t(3, 4), x[0], t(4)),
    "layer_norm bias": lambda x: ops.layer_norm(t(3, 4), t(4), x[0]),
    "layer_norm beside a weight that learns": lambda x: ops.layer_norm(x, t(4).requires_grad_(), t(4)),
    "layer_norm_fwd": lambda x: ops.layer_norm_fwd(x, t(4), t(4)),
    "layer_norm_bwd": lambda x: ops.layer_norm_bwd(x, t(3, 4), t(4), t(2, 3)),
    "layer_norm_bwd stats": lambda x: ops.layer_norm_bwd(t(3, 4), t(3, 4), t(4), x[:2, :3].contiguous()),
    "quantize_int8": lambda x: ops.quantize_int8(x),
    "int8_matmul": lambda x: ops.int8_matmul(t(3, 4, dtype=torch.int8), x[:, 0].contiguous(), W8, t(5)),
    "int8_linear": lambda x: ops.int8_linear(x, W8, t(5)),
    "int8_linear bias": lambda x: ops.int8_linear(t(3, 4), W4, t(4), x[0]),
}


@pytest.mark.parametrize("name", CALLS)
def test_forward_mode_is_refused(name):
    with forward_ad.dual_level():
        x = forward_ad.make_dual(t(3, 4), 2 * t(3, 4))
        with pytest.raises(RuntimeError, match="forward-mode|jvp"):
            CALLS[name](x)


def test_a_level_without_tangents_is_none():
    """Inside a dual level, tensors that carry no tangent reach the check of their device as ever."""
    with forward_ad.dual_level():
        with pytest.raises(RuntimeError, match="HIP device"):
            ops.layer_norm(t(3, 4), t(4), t(4))
        with pytest.raises(RuntimeError, match="HIP device"):
            ops.int8_linear(t(3, 4), W8, t(5))


RECORDED = {k: f for k, f in CALLS.items() if "learns" not in k}


@pytest.mark.parametrize("name", RECORDED)
def test_traces_are_refused(name):
    """What torch.jit.trace and make_fx record of a call is an allocation: its replays would return what lies there."""
    def f(x):
        out = RECORDED[name](x * 1)
        return out[0] if isinstance(out, tuple) else out
    with pytest.raises(RuntimeError, match="trace does not record"):
        torch.jit.trace(f, (t(3, 4),))
    from torch.fx.experimental.proxy_tensor import make_fx
    for mode in ("real", "fake", "symbolic"):
        with pytest.raises(RuntimeError, match="trace does not record"):
            make_fx(f, tracing_mode=mode)(t(3, 4))


def test_fake_tensors_are_refused():
    """Their addresses are 0: nothing may be launched on them, the optimizer's table of addresses included."""
    from torch._subclasses.fake_tensor import FakeTensorMode
    with FakeTensorMode():
        with pytest.raises(RuntimeError, match="trace does not record"):
            ops.layer_norm(t(3, 4), t(4), t(4))
        p = t(3)
        p.grad = t(3)
        with pytest.raises(RuntimeError, match="trace does not record"):
            ops.AdamW([p]).step()


def test_other_modes_pass():
    """A mode that only looks on (the counter of flops) is none of these."""
    from torch.utils.flop_counter import FlopCounterMode
    with FlopCounterMode(display=False):
        with pytest.raises(RuntimeError, match="HIP device"):
            ops.layer_norm(t(3, 4), t(4), t(4))


def test_quantizing_what_learns_is_refused():
    """As the product does: the scale depends on x, and its gradient would be lost."""
    w = t(3, 4).requires_grad_()
    with pytest.raises(RuntimeError, match="have no gradient"):
        ops.quantize_int8(w)
    for call in (lambda: ops.quantize_int8(w.detach()), lambda: torch.no_grad()(ops.quantize_int8)(w)):
        with pytest.raises(RuntimeError, match="HIP device"):
            call()
