"""Operators around the dense layers of a network, on tensors of a HIP device: layer norm with weight and bias (forward,
backward, autograd), AdamW over a network's whole parameter list (32-bit or 8-bit states), and the product in 8-bit integers
with a scale per row and per output channel for serving.

    y = ops.layer_norm(x, weight, bias)                          # differentiable
    opt = ops.AdamW(net.parameters(), lr=1e-3, state_bits=8)     # torch.optim.Optimizer
    wq, ws = ops.quantize_int8(weight.detach())                  # once
    y = ops.int8_linear(x, wq, ws, bias)                         # per request

All arithmetic runs in the HIP kernels behind include/scarches_hip.h (sca_layernorm_*, sca_adamw_step, sca_quant_rows_i8,
sca_gemm_i8) on the current stream of the tensors' device; there is no CPU fallback.  Wrong shapes and types raise ValueError
/ TypeError before anything is launched; torch.jit.trace, make_fx, fake tensors and forward-mode tangents RuntimeError.
"""
from __future__ import annotations

import ctypes
from typing import Optional

import numpy as np
import torch
from torch.autograd import forward_ad as _forward_ad
from torch.optim import optimizer as _optimizer

from . import _lib

_DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
_MAX_WIDTH = 0x7ffff000
_F8_M, _F8_V = torch.float8_e4m3fn, torch.float8_e5m2

# What a small call costs is its host side (a launch takes 4 us, each allocation 1.5): entry points are looked up once, the
# device and the stream are asked for as numbers (current_stream() builds an object: 2 us).
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (lambda i: torch.cuda.current_stream(i).cuda_stream)
_current_device = getattr(torch._C, "_cuda_getDevice", None) or torch.cuda.current_device   # (tensors are there: initialised)
_fns = {}


def _fn(name):
    fn = _fns.get(name)
    if fn is None:
        fn = _fns[name] = getattr(_lib.load(), name)
    return fn


def _dtype_code(t: torch.Tensor, what: str) -> int:
    code = _DTYPES.get(t.dtype)
    if code is None:
        raise TypeError(f"{what} must be float32, bfloat16 or float16, not {t.dtype}")
    return code


def _recording() -> bool:
    """True inside torch.jit.trace, make_fx and on fake tensors: what they record of an operator is the allocation of its
    results, and what they replay computes nothing.  (Under torch.compile an operator is a graph break and runs as ever.)"""
    if torch._C._is_tracing():
        return True
    key = torch._C._TorchDispatchModeKey
    return torch._C._len_torch_dispatch_stack() > 0 and (torch._C._get_dispatch_mode(key.PROXY) is not None
                                                         or torch._C._get_dispatch_mode(key.FAKE) is not None)


def _no_tangents(tensors):
    """A dual tensor does not require grad: its tangent would be lost without a word (and read as zero)."""
    if any(t is not None and _forward_ad.unpack_dual(t).tangent is not None for t in tensors):
        raise RuntimeError("scarches_amd.ops has no forward-mode derivatives (a tensor of the call carries a tangent)")


def _same_device(*tensors) -> int:
    """The number of the one HIP device that all tensors (or None) are on.  Every operator asks before it launches anything."""
    if _forward_ad._current_level >= 0:
        _no_tangents(tensors)
    if _recording():
        raise RuntimeError("the kernels of scarches_amd.ops are launched through addresses, which a trace does not record")
    index = tensors[0].get_device()
    for t in tensors:
        if t is not None and t.get_device() != index:
            raise ValueError(f"the operator's tensors are on {tensors[0].device} and {t.device}")
    if index < 0:
        raise _lib.HipLibraryError("scarches_amd runs on a HIP device only (no CPU fallback)")
    return index


def _call(index, name, *args):
    """One entry point of the library on device `index`, behind what its current stream holds."""
    if _current_device() == index:
        rc = _fn(name)(*args, _raw_stream(index))
    else:
        with torch.cuda.device(index):
            rc = _fn(name)(*args, _raw_stream(index))
    if rc:
        _lib.check(rc, name)


def _rows(t: torch.Tensor):
    """(tensor whose rows are contiguous, rows, pitch) of a [..., n] tensor; a copy only where no such view exists."""
    if t.dim() != 2:
        t = t.reshape(-1, t.shape[-1])
    rows, n = t.shape
    if n > 1 and t.stride(1) != 1:
        t = t.contiguous()
    return t, rows, t.stride(0) if rows > 1 else n


def _check_width(n):
    if n > _MAX_WIDTH:
        raise ValueError(f"rows of {n} values: the kernels count columns in 32 bits, up to {_MAX_WIDTH}")


def _like(x):
    """A new contiguous tensor of x's shape and type."""
    return torch.empty_like(x) if x.is_contiguous() else x.new_empty(x.shape)


# ---------------------------------------------------------------------------------------------- layer norm
def _ln_check(x, weight, bias):
    if x.dim() < 1 or x.shape[-1] == 0:
        raise ValueError(f"layer norm needs a last dimension of at least one value, got shape {tuple(x.shape)}")
    _check_width(x.shape[-1])
    code = _dtype_code(x, "x")
    if weight is None:
        if bias is not None:
            raise ValueError("layer norm takes a bias only together with a weight")
        return code, code
    wcode = _dtype_code(weight, "weight")
    if wcode != 0 and wcode != code:
        raise TypeError(f"weight must be float32 or of x's type {x.dtype}, not {weight.dtype}")
    n = x.shape[-1]
    for name, t in (("weight", weight), ("bias", bias)):
        if t is None:
            continue
        if t.dim() != 1 or t.shape[0] != n:
            raise ValueError(f"{name} has shape {tuple(t.shape)}, x's rows need ({n},)")
        if t.dtype != weight.dtype:
            raise TypeError(f"weight is {weight.dtype}, bias {t.dtype}")
        if not t.is_contiguous():
            raise ValueError(f"{name} must be contiguous")
    return code, wcode


def layer_norm_fwd(x, weight=None, bias=None, eps=1e-5):
    """(y, stats): layer norm of the rows of x [..., n] (float32, bfloat16 or float16, rows of any pitch) and stats [2, rows]
    = (mean, 1 / sqrt(variance + eps)) in float32 for `layer_norm_bwd`.  weight / bias: [n], float32 or x's type."""
    code, wcode = _ln_check(x, weight, bias)
    if not eps >= 0:
        raise ValueError(f"eps must not be negative, got {eps}")
    index = _same_device(x, weight, bias)
    x2, rows, ldx = _rows(x)
    n = x.shape[-1]
    y = _like(x)
    stats = x.new_empty((2, rows), dtype=torch.float32)
    if rows:
        _call(index, "sca_layernorm_fwd", x2.data_ptr(), ldx, code, rows, n, _lib.ptr(weight), _lib.ptr(bias), wcode, eps,
              y.data_ptr(), n, stats.data_ptr())
    return y, stats


def layer_norm_bwd(dy, x, weight, stats, need=(True, True, True)):
    """(dx, dweight, dbias) of layer norm for the gradient dy of its result: x and weight as they were given to
    `layer_norm_fwd`, stats as it returned them.  `need`: which of the three are wanted (the others are None, and so are
    dweight and dbias without a weight).  dweight and dbias are sums over all rows, taken in float32 in a fixed order."""
    code, wcode = _ln_check(x, weight, None)
    if dy.shape != x.shape or dy.dtype != x.dtype:
        raise ValueError(f"dy is {dy.dtype} {tuple(dy.shape)}, x {x.dtype} {tuple(x.shape)}")
    index = _same_device(x, dy, weight, stats)
    x2, rows, ldx = _rows(x)
    dy2, _, lddy = _rows(dy)
    n = x.shape[-1]
    if stats.dtype != torch.float32 or tuple(stats.shape) != (2, rows) or not stats.is_contiguous():
        raise ValueError(f"stats must be the float32 tensor [2, {rows}] that the forward pass returned")
    need_w, need_b = need[1] and weight is not None, need[2] and weight is not None
    dx = _like(x) if need[0] else None
    dw = torch.empty_like(weight) if need_w else None
    db = torch.empty_like(weight) if need_b else None
    ws = None
    if need_w or need_b or n > 16384:
        ws = x.new_empty((_fn("sca_layernorm_bwd_workspace_floats")(rows, n),), dtype=torch.float32)
    _call(index, "sca_layernorm_bwd", dy2.data_ptr(), lddy, x2.data_ptr(), ldx, code, rows, n, _lib.ptr(weight), wcode,
          stats.data_ptr(), _lib.ptr(dx), n, _lib.ptr(dw), _lib.ptr(db), _lib.ptr(ws))
    return dx, dw, db


class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps):
        y, stats = layer_norm_fwd(x, weight, bias, eps)
        ctx.save_for_backward(x, weight, stats)
        return y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        x, weight, stats = ctx.saved_tensors
        return (*layer_norm_bwd(dy, x, weight, stats, ctx.needs_input_grad[:3]), None)


def layer_norm(x, weight=None, bias=None, eps=1e-5):
    """Layer norm over the last dimension of x with optional weight and bias [n]; gradients of x, weight and bias (reverse mode,
    once; a tensor with a forward-mode tangent is refused here and by every operator of this module).

    Statistics and sums are held in float32 whatever x's type, and each result is rounded once.  A row with NaN or an
    infinity gives NaN in that row (and in the weight's gradient) only."""
    if torch.is_grad_enabled() and (x.requires_grad or (weight is not None and weight.requires_grad)
                                    or (bias is not None and bias.requires_grad)):
        if _forward_ad._current_level >= 0:         # (what apply() calls does not see tangents)
            _no_tangents((x, weight, bias))
        return _LayerNorm.apply(x, weight, bias, eps)
    return layer_norm_fwd(x, weight, bias, eps)[0]


# ---------------------------------------------------------------------------------------------- 8-bit integer product
_PAD_K = 128        # pitch of quantized rows: a multiple of the product's k step, the bytes behind a row's end are zero


def quantize_int8(x):
    """(q, scale) of the rows of x [..., k]: int8 q [..., k] and float32 scale [...] with x ~ q * scale[..., None], scale =
    max |x| / 127 of the row.  q is a view of rows padded with zeros to a multiple of 128 bytes, as `int8_matmul` reads them
    fastest.  A row of zeros has scale 0; a row with NaN or an infinity has scale NaN, and so have results computed from it.
    No gradient: a parameter is quantized under torch.no_grad() or detached."""
    if x.dim() < 1 or x.shape[-1] == 0:
        raise ValueError(f"quantize_int8 needs rows of at least one value, got shape {tuple(x.shape)}")
    _check_width(x.shape[-1])
    code = _dtype_code(x, "x")
    _no_grad(x)
    index = _same_device(x)
    x2, rows, ldx = _rows(x)
    k = x.shape[-1]
    pitch = -(-k // _PAD_K) * _PAD_K
    q = x.new_empty((*x.shape[:-1], pitch), dtype=torch.int8)
    scale = x.new_empty(x.shape[:-1], dtype=torch.float32)
    if rows:
        _call(index, "sca_quant_rows_i8", x2.data_ptr(), ldx, code, rows, k, q.data_ptr(), pitch, scale.data_ptr())
    return q[..., :k], scale


def _i8_check(k, wq, w_scale, bias, out_dtype):
    """The codes of the bias' and of the result's type."""
    code = _DTYPES.get(out_dtype)
    if code is None:
        raise TypeError(f"results can be float32, bfloat16 or float16, not {out_dtype}")
    if wq.dtype != torch.int8 or wq.dim() != 2:
        raise TypeError(f"wq must be an int8 matrix [out, in], not {wq.dtype} {tuple(wq.shape)}")
    n, wk = wq.shape
    _check_width(n)
    if wk != k or k == 0:
        raise ValueError(f"x has rows of {k} values, wq is {tuple(wq.shape)}")
    if w_scale.dtype != torch.float32 or w_scale.dim() != 1 or w_scale.shape[0] != n or not w_scale.is_contiguous():
        raise ValueError(f"w_scale must be a contiguous float32 vector [{n}], one value per output channel")
    if bias is not None and (bias.dim() != 1 or bias.shape[0] != n or bias.dtype not in (torch.float32, out_dtype)
                             or not bias.is_contiguous()):
        raise ValueError(f"bias must be a contiguous vector [{n}] of float32 or {out_dtype}")
    if k > _fn("sca_gemm_i8_max_k")():
        raise ValueError(f"rows of {k} values: the sum of more than {_fn('sca_gemm_i8_max_k')()} products can pass int32")
    return 0 if bias is None else _DTYPES[bias.dtype], code


def _no_grad(*tensors):
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors):
        raise RuntimeError("the 8-bit integer operators are for serving and have no gradient: call them under torch.no_grad()")


def _weight_rows(wq):
    """(wq with contiguous rows, their pitch)."""
    n, k = wq.shape
    if k > 1 and wq.stride(1) != 1:
        wq = wq.contiguous()
    return wq, wq.stride(0) if n > 1 else k


def int8_matmul(xq, x_scale, wq, w_scale, bias: Optional[torch.Tensor] = None, out_dtype=torch.float32):
    """y [..., n] = (xq wq^T) * x_scale[..., None] * w_scale + bias for int8 xq [..., k] with one scale per row (as
    `quantize_int8` gives them) and an int8 weight wq [n, k] with one scale per output channel.  The integer sum is exact
    (k < 2^17); scales and bias are applied in float32 and the result is rounded once to out_dtype."""
    if xq.dtype != torch.int8 or xq.dim() < 1:
        raise TypeError(f"xq must be int8 rows [..., k], not {xq.dtype} {tuple(xq.shape)}")
    k = xq.shape[-1]
    bcode, code = _i8_check(k, wq, w_scale, bias, out_dtype)
    if x_scale.dtype != torch.float32 or x_scale.shape != xq.shape[:-1] or not x_scale.is_contiguous():
        raise ValueError(f"x_scale must be contiguous float32 {tuple(xq.shape[:-1])}, one value per row of xq")
    _no_grad(x_scale, w_scale, bias)
    index = _same_device(wq, xq, x_scale, w_scale, bias)
    x2, rows, ldx = _rows(xq)
    wq, ldw = _weight_rows(wq)
    n = wq.shape[0]
    y = wq.new_empty((*xq.shape[:-1], n), dtype=out_dtype)
    if rows and n:
        _call(index, "sca_gemm_i8", x2.data_ptr(), ldx, x_scale.data_ptr(), wq.data_ptr(), ldw, w_scale.data_ptr(),
              _lib.ptr(bias), bcode, rows, n, k, y.data_ptr(), code, n)
    return y


def int8_linear(x, wq, w_scale, bias: Optional[torch.Tensor] = None, out_dtype=None):
    """y = x W^T + bias in 8-bit integers: x [..., k] (float32, bfloat16 or float16) is quantized row by row as by
    `quantize_int8`, then multiplied as by `int8_matmul`.  out_dtype: x's type by default.  Serving only: no gradient."""
    if x.dim() < 1:
        raise ValueError("int8_linear needs rows [..., k]")
    xcode = _dtype_code(x, "x")
    k = x.shape[-1]
    out_dtype = x.dtype if out_dtype is None else out_dtype
    bcode, code = _i8_check(k, wq, w_scale, bias, out_dtype)
    _no_grad(x, w_scale, bias)
    index = _same_device(x, wq, w_scale, bias)
    x2, rows, ldx = _rows(x)
    wq, ldw = _weight_rows(wq)
    n = wq.shape[0]
    y = x.new_empty((*x.shape[:-1], n), dtype=out_dtype)
    if rows and n:
        size = _fn("sca_linear_i8_workspace_bytes")(rows, n, k)
        ws = x.new_empty((size,), dtype=torch.int8) if size else None
        _call(index, "sca_linear_i8", x2.data_ptr(), ldx, xcode, wq.data_ptr(), ldw, w_scale.data_ptr(), _lib.ptr(bias),
              bcode, rows, n, k, y.data_ptr(), code, n, _lib.ptr(ws))
    return y


# ---------------------------------------------------------------------------------------------- AdamW
def _layout(t):
    """What two tensors have in common whose elements lie in the same order: () if contiguous, else the strides."""
    return () if t.is_contiguous() else tuple(t.stride())


def _dense(t):
    """True when t's elements fill one range of memory, each once (any order of the dimensions)."""
    if t.is_contiguous():
        return True
    size = 1
    for stride, n in sorted((t.stride(d), t.shape[d]) for d in range(t.dim()) if t.shape[d] != 1):
        if stride != size:
            return False
        size *= n
    return True


class AdamW(torch.optim.Optimizer):
    """torch.optim.AdamW (decoupled weight decay) over all parameters of a group at once.

    params, lr, betas, eps, weight_decay: as torch.optim.AdamW.  Parameters are float32, bfloat16 or float16; a step is
    computed in float32 and rounded once.
    state_bits=32: `exp_avg`, `exp_avg_sq` in float32 whatever the parameter's type.
    state_bits=8: `exp_avg` float8_e4m3fn and `exp_avg_sq` float8_e5m2, each with one float32 power of two per 256 elements
    (`exp_avg_scale`, `exp_avg_sq_scale`): 2.03 bytes per value instead of 8.  Rounding to 8 bits is stochastic, from a
    generator of (seed, parameter, element, step): the same seed gives the same run, and a state dict holds it.  A gradient
    that is not finite makes the moments of its 256 elements NaN.

    The step number of each parameter lies on the device, so `step()` may be captured into a HIP graph after one ordinary
    call (lr and the other scalars are taken as they are at capture; a graph captured before `load_state_dict` goes on with the
    states it was captured with; a second graph over gradients in other storage needs an ordinary call in between;
    the optimizer has to outlive its graphs).  Gradients have their parameter's type and memory order;
    sparse gradients are refused.  One stream at a time may run an optimizer: work that uses it on another stream has to be
    ordered behind the first, as for any tensor."""

    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=1e-2, *, state_bits=32, seed=0):
        if isinstance(lr, torch.Tensor):
            raise TypeError("lr must be a number")
        if not lr >= 0:
            raise ValueError(f"Invalid learning rate: {lr}")
        if not eps >= 0:
            raise ValueError(f"Invalid epsilon value: {eps}")
        for i in (0, 1):
            if not 0 <= betas[i] < 1:
                raise ValueError(f"Invalid beta parameter at index {i}: {betas[i]}")
        if not weight_decay >= 0:
            raise ValueError(f"Invalid weight_decay value: {weight_decay}")
        if state_bits not in (8, 32):
            raise ValueError(f"state_bits must be 8 or 32, not {state_bits}")
        self.state_bits, self.seed = state_bits, int(seed) & 0xFFFFFFFFFFFFFFFF
        self._steps = {}            # group number -> int64 [parameters] on the device: their steps
        # group number -> (the step of the parameters that take part, which ones: a bit each, or None for all that come);
        # (None, None) where only the device knows
        self._host_steps = {}
        self._plans = {}            # group number -> the table of the last step()
        self._captured = []         # tables (and what they point to) that captured graphs read
        super().__init__(params, dict(lr=lr, betas=tuple(betas), eps=eps, weight_decay=weight_decay))

    # Copies and pickles hold the settings, the states and the steps; tables of addresses are made anew.
    def __getstate__(self):
        return dict(super().__getstate__(), state_bits=self.state_bits, seed=self.seed, _steps=self._steps,
                    _host_steps=dict(self._host_steps), _plans={}, _captured=[])

    # ------------------------------------------------------------------------------------------ state
    def _check_param(self, p):
        _dtype_code(p, "a parameter")
        if not _dense(p):
            raise ValueError("AdamW needs parameters whose elements fill one range of memory")
        _same_device(p)

    def add_param_group(self, param_group):
        super().add_param_group(param_group)
        group = self.param_groups[-1]
        for p in group["params"]:
            if p.dtype not in _DTYPES:
                self.param_groups.pop()
                raise TypeError(f"a parameter must be float32, bfloat16 or float16, not {p.dtype}")

    def _init_state(self, p):
        self._check_param(p)
        if torch.cuda.is_current_stream_capturing():        # zeros that only a replay would write
            raise RuntimeError("AdamW.step(): a parameter without states; call step() once before the capture")
        st = self.state[p]
        if self.state_bits == 32:
            for k in ("exp_avg", "exp_avg_sq"):
                st[k] = torch.zeros_like(p, dtype=torch.float32, memory_format=torch.preserve_format)
            return
        blocks = -(-p.numel() // _lib.load().sca_adamw_block_elements())
        for k, f8 in (("exp_avg", _F8_M), ("exp_avg_sq", _F8_V)):
            st[k] = torch.zeros_like(p, dtype=torch.uint8, memory_format=torch.preserve_format).view(f8)
            st[k + "_scale"] = torch.zeros(blocks, dtype=torch.float32, device=p.device)

    def _group_steps(self, gi):
        ctr = self._steps.get(gi)
        params = self.param_groups[gi]["params"]
        if ctr is None:
            ctr = self._steps[gi] = torch.zeros(len(params), dtype=torch.int64, device=params[0].device)
        return ctr

    def set_step(self, step: int):
        """Set the number of steps that every parameter has behind it (a run taken up from states of another program)."""
        if int(step) < 0:
            raise ValueError(f"a parameter cannot have {step} steps behind it")
        for gi, group in enumerate(self.param_groups):
            if not group["params"]:
                continue
            self._group_steps(gi).fill_(int(step))
            if self._host_steps.get(gi, (0,))[0] is not None:
                self._host_steps[gi] = (int(step), None)

    def state_dict(self):
        """torch's layout; every parameter's state has `step` as a whole number (read from the device), and with 8-bit states
        every group the `seed` of the rounding."""
        sd = super().state_dict()
        if self.state_bits == 8:
            sd["param_groups"] = [dict(group, seed=self.seed) for group in sd["param_groups"]]
        sd["state"] = {pid: st for pid, st in sd["state"].items() if st}        # (looking one up leaves an empty one)
        for gi, packed in enumerate(sd["param_groups"]):
            if gi not in self._steps:
                continue
            steps = self._steps[gi].tolist()
            for i, pid in enumerate(packed["params"]):
                if pid in sd["state"]:
                    sd["state"][pid] = dict(sd["state"][pid], step=steps[i])
        return sd

    def load_state_dict(self, state_dict):
        """Take up the states of a `state_dict()` of this class with the same state_bits, or (32 bits) of torch.optim.AdamW.
        8-bit states bring the seed of their rounding along, so that the run goes on as it would have.
        ValueError for a run whose rule is another one (amsgrad, maximize, torch.optim.Adam's coupled decay) or whose states
        are not these: nothing is changed then."""
        for group in state_dict["param_groups"]:
            if not {"lr", "betas", "eps", "weight_decay"} <= set(group):
                raise ValueError("the state dict is of another optimizer: its groups lack lr, betas, eps or weight_decay")
            for key in ("amsgrad", "maximize"):
                if group.get(key):
                    raise ValueError(f"the state dict is of a run with {key}=True, which this optimizer does not have")
            if not group.get("decoupled_weight_decay", True):
                raise ValueError("the state dict is of torch.optim.Adam, whose weight decay is part of the gradient")
            if any(isinstance(x, torch.Tensor) for x in (group["lr"], *group["betas"])):
                raise ValueError("the state dict's lr and betas must be numbers")
        keys = {"exp_avg", "exp_avg_sq"} | ({"exp_avg_scale", "exp_avg_sq_scale"} if self.state_bits == 8 else set())
        for st in state_dict["state"].values():
            if set(st) - {"step"} not in (keys, set()):
                raise ValueError(f"the state dict holds {sorted(st)}, this optimizer keeps {self.state_bits}-bit states")
        seeds = {int(group["seed"]) for group in state_dict["param_groups"] if "seed" in group}
        if len(seeds) > 1:
            raise ValueError(f"the state dict's groups hold different seeds: {sorted(seeds)}")
        super().load_state_dict(state_dict)
        for group in self.param_groups:
            group.pop("seed", None)
        if seeds:
            self.seed = seeds.pop()
        self._plans = {}
        for gi, (group, packed) in enumerate(zip(self.param_groups, state_dict["param_groups"])):
            steps = []
            if not group["params"]:
                continue
            for p, pid in zip(group["params"], packed["params"]):
                st = state_dict["state"].get(pid, {})
                steps.append(int(st.get("step", 0)))
                if "exp_avg" in st:     # the types of the states are theirs, not the parameter's
                    self.state[p] = {k: st[k].to(p.device, torch.float32 if self.state_bits == 32 else st[k].dtype,
                                                 copy=True) for k in keys}
                else:
                    self.state.pop(p, None)
            self._group_steps(gi).copy_(torch.tensor(steps))
            if self._host_steps.get(gi, (0,))[0] is not None:
                taken, mask = set(steps) - {0}, 0
                for t in steps:
                    mask = mask << 1 | (t > 0)
                self._host_steps[gi] = (0, None) if not taken else (taken.pop(), mask) if len(taken) == 1 else (None, None)

    # ------------------------------------------------------------------------------------------ step
    def _table(self, gi, group, key, grads):
        """The device table of a group: entries, chunks, and the tensors that hold them."""
        if torch.cuda.is_current_stream_capturing():
            raise RuntimeError("AdamW.step(): the parameters, gradients or states differ from the last call; call it once "
                               "with them before the capture")
        lib = _lib.load()
        chunk = lib.sca_adamw_chunk_elements()
        block = lib.sca_adamw_block_elements()
        steps = self._group_steps(gi)
        if steps.numel() != len(group["params"]):
            raise RuntimeError(f"AdamW.step(): parameter group {gi} had {steps.numel()} parameters when it was first used and has "
                               f"{len(group['params'])} now; others join by add_param_group()")
        first = sum(len(g["params"]) for g in self.param_groups[:gi])
        dev, rows = steps.device, []
        for i, p in enumerate(group["params"]):
            g = p.grad
            if g is None:
                continue
            st = self.state[p]
            self._check_param(p)
            if g.is_sparse or g.layout != torch.strided:
                raise RuntimeError("AdamW does not support sparse gradients")
            if g.dtype != p.dtype or g.shape != p.shape or _layout(g) != _layout(p):
                raise ValueError(f"the gradient of parameter {i} is {g.dtype} {tuple(g.shape)} strides {tuple(g.stride())}, "
                                 f"the parameter {p.dtype} {tuple(p.shape)} strides {tuple(p.stride())}")
            _same_device(steps, p, g, *st.values())
            for k, want in (("exp_avg", _F8_M), ("exp_avg_sq", _F8_V)):
                t = st[k]
                want = torch.float32 if self.state_bits == 32 else want
                if t.dtype != want or t.shape != p.shape or _layout(t) != _layout(p):
                    raise ValueError(f"{k} of parameter {i} must be {want} in the parameter's shape and memory order")
                if self.state_bits == 8:
                    s = st[k + "_scale"]
                    if s.dtype != torch.float32 or s.numel() != -(-p.numel() // block) or not s.is_contiguous():
                        raise ValueError(f"{k}_scale of parameter {i} must hold one float32 per {block} elements")
            m, v = st["exp_avg"], st["exp_avg_sq"]
            size, state_align = p.element_size(), 16 if self.state_bits == 32 else 4
            vec = not ((p.data_ptr() | g.data_ptr()) % (4 * size) or (m.data_ptr() | v.data_ptr()) % state_align)
            ms, vs = st.get("exp_avg_scale"), st.get("exp_avg_sq_scale")
            rows.append(_lib.AdamWTensor(p.data_ptr(), g.data_ptr(), m.data_ptr(), v.data_ptr(), _lib.ptr(ms), _lib.ptr(vs),
                                         p.numel(), steps.data_ptr() + 8 * i, float(group["weight_decay"]),
                                         _DTYPES[p.dtype], int(vec), first + i))
        counts = np.array([-(-r.n // chunk) for r in rows], dtype=np.int64)
        chunks = np.empty((int(counts.sum()), 2), dtype=np.int32)
        chunks[:, 0] = np.repeat(np.arange(len(rows)), counts)
        chunks[:, 1] = np.arange(len(chunks)) - np.repeat(np.cumsum(counts) - counts, counts)
        entries = bytes((_lib.AdamWTensor * len(rows))(*rows))
        # one pinned block, one copy on the current stream (the caching host allocator keeps the block until it has run);
        # the kernels' scratch comes first, where the block's alignment is
        size = lib.sca_adamw_scratch_bytes(len(rows))
        host = torch.from_numpy(np.frombuffer(bytes(size) + entries + chunks.tobytes(), dtype=np.uint8).copy()).pin_memory()
        table = host.to(dev, non_blocking=True)
        at = table.data_ptr() + size
        return dict(key=key, grads=grads, captured=False, table=table, streams={_raw_stream(dev.index)}, entries=at,
                    n=len(rows), chunks=at + len(entries), n_chunks=len(chunks), steps=steps, scratch=table.data_ptr(),
                    index=dev.index)

    def _step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        scales = self.state_bits == 8
        for gi, group in enumerate(self.param_groups):
            # what the table was made of: addresses, sizes, types and layouts
            key, grads, taken, mask = [group["weight_decay"]], [], [], 0
            for p in group["params"]:
                g = p.grad
                mask <<= 1
                if g is None:
                    continue
                mask |= 1
                st = self.state[p]
                if not st:
                    self._init_state(p)
                grads.append(g.data_ptr())
                taken.append(p)
                flat = p.is_contiguous() and g.is_contiguous() or (p.stride(), g.stride())
                key += (p.data_ptr(), p.numel(), p.dtype, g.nbytes, flat, st["exp_avg"].data_ptr(), st["exp_avg_sq"].data_ptr())
                if scales:
                    key += (st["exp_avg_scale"].data_ptr(), st["exp_avg_sq_scale"].data_ptr())
            if not grads:           # (nobody takes a step: nothing to count)
                continue
            plan = self._plans.get(gi)
            known = plan is not None and plan["key"] == key
            moved = known and plan["grads"] != grads
            if not known or moved and (plan["captured"] or any(at % 16 for at in grads)
                                       or any(p.grad.dtype != p.dtype for p in taken)):
                plan = self._plans[gi] = self._table(gi, group, key, grads)
                moved = False
            stream = _raw_stream(plan["index"])
            if stream not in plan["streams"]:
                plan["streams"].add(stream)
                if not torch.cuda.is_current_stream_capturing():
                    plan["table"].record_stream(torch.cuda.current_stream(plan["table"].device))
            if moved:       # gradients in new storage (a graph's table is its own, and stays)
                _call(plan["index"], "sca_adamw_set_grads", plan["entries"], plan["n"], (ctypes.c_void_p * len(grads))(*grads))
                plan["grads"] = grads
            # As long as the same parameters take every step and no graph takes steps that nobody here sees, the step number
            # is given; else the device counts.
            t, of = self._host_steps.get(gi, (0, None))
            if of is not None and of != mask:
                t = None
            if torch.cuda.is_current_stream_capturing():    # replays read the table and what it points to
                self._captured.append((plan, [(p, p.grad, dict(self.state[p])) for p in taken]))
                plan["captured"] = True
                if moved:   # the table changes when the graph runs, not now
                    del self._plans[gi]
                t = None
            if t is None:
                self._host_steps[gi] = (None, None)
            else:
                t += 1
            b1, b2 = group["betas"]
            _call(plan["index"], "sca_adamw_step", plan["entries"], plan["n"], plan["chunks"], plan["n_chunks"],
                  self.state_bits, None, t or 0, group["lr"], b1, b2, group["eps"], self.seed, plan["scratch"])
            if t is not None:       # (a call that raised has counted nothing)
                self._host_steps[gi] = (t, mask)
            # the kernel writes through addresses: autograd has to hear that what it may have saved is not there any more
            torch._C._increment_version(taken)              # (torch.autograd.graph.increment_version)
        return loss

    # torch wraps step() to run its hooks and to be seen by the profiler, which takes 6 us: here only where one is wanted
    _hooked_step = torch.optim.Optimizer.profile_hook_step(_step)

    def step(self, closure=None):
        """One step of every parameter that has a gradient; `closure` (optional) is called first and its value returned."""
        if (self._optimizer_step_pre_hooks or self._optimizer_step_post_hooks or _optimizer._global_optimizer_pre_hooks
                or _optimizer._global_optimizer_post_hooks or torch.autograd.profiler._is_profiler_enabled):
            return self._hooked_step(closure)
        return self._step(closure)

    step.hooked = True
