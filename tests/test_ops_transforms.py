"""Calls of scarches_amd.ops from inside torch's transformations, which see no more than an allocation of a kernel that is
launched through addresses: refused instead of answered wrongly (no GPU needed)."""
import pytest
import torch
from torch.autograd import forward_ad

from scarches_amd import ops


def t(*shape, dtype=torch.float32):
    return torch.ones(*shape, dtype=dtype)


W8 = torch.ones(5, 4, dtype=torch.int8)
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
    "int8_linear bias": lambda x: ops.int8_linear(t(3, 4), W8[:4], t(4), x[0]),
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
