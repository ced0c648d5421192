"""What scarches_amd.ops refuses before anything is launched (no GPU needed)."""
import pytest
import torch

from scarches_amd import _lib, ops


def t(*shape, dtype=torch.float32):
    return torch.zeros(*shape, dtype=dtype)


@pytest.mark.parametrize("args,error", [
    ((t(3, 0),), ValueError), ((t(()),), ValueError), ((t(3, 4, dtype=torch.float64),), TypeError),
    ((t(3, 4, dtype=torch.int32),), TypeError), ((t(3, 4), t(5)), ValueError), ((t(3, 4), t(1, 4)), ValueError),
    ((t(3, 4), t(4), t(3)), ValueError), ((t(3, 4), None, t(4)), ValueError), ((t(3, 4), t(4, dtype=torch.bfloat16)), TypeError),
    ((t(3, 4), t(4), t(4, dtype=torch.float16)), TypeError), ((t(3, 4), t(8)[::2]), ValueError), ((t(3, 4), t(4), t(4), -1.0), ValueError),
    ((t(3, 4), t(4), t(4), float("nan")), ValueError), ((t(3, 4), t(4), t(4)), _lib.HipLibraryError)])
def test_layer_norm(args, error):
    with pytest.raises(error):
        ops.layer_norm_fwd(*args)
    with pytest.raises(error):
        ops.layer_norm(*args)


@pytest.mark.parametrize("args,error", [
    ((t(3, 5), t(3, 4), t(4), t(2, 3)), ValueError), ((t(3, 4, dtype=torch.float16), t(3, 4), t(4), t(2, 3)), ValueError),
    ((t(3, 4), t(3, 4), t(5), t(2, 3)), ValueError), ((t(3, 4), t(3, 4), t(4), t(2, 3)), _lib.HipLibraryError)])
def test_layer_norm_bwd(args, error):
    with pytest.raises(error):
        ops.layer_norm_bwd(*args)


I8 = torch.int8


@pytest.mark.parametrize("args,error", [
    ((t(3, 4), t(3), t(5, 4, dtype=I8), t(5)), TypeError), ((t(3, 4, dtype=I8), t(3), t(5, 4), t(5)), TypeError),
    ((t(3, 4, dtype=I8), t(3), t(5, 6, dtype=I8), t(5)), ValueError), ((t(3, 4, dtype=I8), t(4), t(5, 4, dtype=I8), t(5)), ValueError),
    ((t(3, 4, dtype=I8), t(3), t(5, 4, dtype=I8), t(4)), ValueError),
    ((t(3, 4, dtype=I8), t(3, dtype=torch.float16), t(5, 4, dtype=I8), t(5)), ValueError),
    ((t(3, 4, dtype=I8), t(3), t(5, 4, dtype=I8), t(10)[::2]), ValueError),
    ((t(3, 4, dtype=I8), t(3), t(5, 4, dtype=I8), t(5), t(4)), ValueError),
    ((t(3, 4, dtype=I8), t(3), t(5, 4, dtype=I8), t(5), t(5, dtype=torch.float16)), ValueError),
    ((t(3, 4, dtype=I8), t(3), t(5, 4, dtype=I8), t(5), None, torch.float64), TypeError),
    ((t(3, 0, dtype=I8), t(3), t(5, 0, dtype=I8), t(5)), ValueError),
    ((t(1, 1 << 17, dtype=I8), t(1), t(1, 1 << 17, dtype=I8), t(1)), ValueError),
    ((t(3, 4, dtype=I8), t(3).requires_grad_(), t(5, 4, dtype=I8), t(5)), RuntimeError),
    ((t(3, 4, dtype=I8), t(3), t(5, 4, dtype=I8), t(5)), _lib.HipLibraryError)])
def test_int8_matmul(args, error):
    with pytest.raises(error):
        ops.int8_matmul(*args)


@pytest.mark.parametrize("call,error", [
    (lambda: ops.int8_linear(t(3, 4).requires_grad_(), t(5, 4, dtype=I8), t(5)), RuntimeError),
    (lambda: ops.int8_linear(t(3, 4, dtype=torch.float64), t(5, 4, dtype=I8), t(5)), TypeError),
    (lambda: ops.int8_linear(t(3, 4), t(5, 3, dtype=I8), t(5)), ValueError),
    (lambda: ops.int8_linear(t(3, 4), t(5, 4, dtype=I8), t(5)), _lib.HipLibraryError),
    (lambda: ops.quantize_int8(t(3, 0)), ValueError), (lambda: ops.quantize_int8(t(3, 4, dtype=I8)), TypeError),
    (lambda: ops.quantize_int8(t(3, 4)), _lib.HipLibraryError)])
def test_int8_linear(call, error):
    with pytest.raises(error):
        call()


@pytest.mark.parametrize("kw,error", [
    (dict(lr=-1.0), ValueError), (dict(lr=torch.tensor(1.0)), TypeError), (dict(eps=-1e-8), ValueError), (dict(betas=(1.0, 0.9)), ValueError),
    (dict(betas=(0.9, -0.1)), ValueError), (dict(weight_decay=-0.1), ValueError), (dict(state_bits=16), ValueError)])
def test_adamw_arguments(kw, error):
    with pytest.raises(error):
        ops.AdamW([t(3)], **kw)


def test_adamw_parameters():
    with pytest.raises(TypeError):
        ops.AdamW([t(3, dtype=torch.float64)])
    with pytest.raises(ValueError):                 # the same tensor twice in a group, or in two
        p = t(3)
        ops.AdamW([dict(params=[p]), dict(params=[p])])
    p = t(3)
    opt = ops.AdamW([p])
    opt.step()                                      # nothing has a gradient: nothing to do
    p.grad = t(3)
    with pytest.raises(_lib.HipLibraryError):
        opt.step()
    q = t(3, 4).expand(2, 3, 4)
    q.grad = t(2, 3, 4)
    with pytest.raises(ValueError, match="one range of memory"):
        ops.AdamW([q]).step()


def test_entry_points_check_their_arguments():
    """-1 from the C entry points, before a kernel is launched (the addresses are never read)."""
    lib = _lib.load()
    a = 4096
    ok = (a, 8, 0, 4, 8, a, a, 0, 1e-5, a, 8, a, None)
    for i, bad in ((0, None), (1, -1), (2, 3), (3, -1), (4, 0), (7, 1), (8, -1.0), (9, None), (10, 7)):
        assert lib.sca_layernorm_fwd(*ok[:i], bad, *ok[i + 1:]) == -1, i
    ok = (a, 8, a, 8, 0, 4, 8, a, 0, a, a, 8, a, a, a, None)
    for i, bad in ((0, None), (1, -1), (2, None), (3, -1), (4, 7), (5, -1), (6, 0), (8, 2), (9, None), (11, 7), (14, None)):
        assert lib.sca_layernorm_bwd(*ok[:i], bad, *ok[i + 1:]) == -1, i
    assert lib.sca_layernorm_bwd_workspace_floats(-1, 3) == -1 and lib.sca_layernorm_bwd_workspace_floats(5, 0) == -1
    ok = (a, 8, 0, 4, 8, a, 8, a, None)
    for i, bad in ((0, None), (1, -1), (2, 5), (3, -1), (4, 0), (5, None), (6, 7), (7, None)):
        assert lib.sca_quant_rows_i8(*ok[:i], bad, *ok[i + 1:]) == -1, i
    ok = (a, 8, a, a, 8, a, a, 0, 4, 5, 8, a, 0, 5, None)
    for i, bad in ((0, None), (1, -1), (2, None), (3, None), (4, 7), (5, None), (7, 1), (8, -1), (9, -1), (10, 0),
                   (10, lib.sca_gemm_i8_max_k() + 1), (11, None), (12, 3), (13, 4)):
        assert lib.sca_gemm_i8(*ok[:i], bad, *ok[i + 1:]) == -1, i
    ok = (a, 8, 0, a, 8, a, a, 0, 40, 5, 8, a, 0, 5, a, None)
    for i, bad in ((0, None), (1, -1), (2, 3), (3, None), (4, 7), (5, None), (7, 1), (8, -1), (9, -1), (10, 0), (11, None), (12, -1),
                   (13, 4), (14, None), (14, a + 8)):
        assert lib.sca_linear_i8(*ok[:i], bad, *ok[i + 1:]) == -1, i
    assert lib.sca_linear_i8_workspace_bytes(40, 5, 8) >= 40 * (8 + 4) and lib.sca_linear_i8_workspace_bytes(1, 5, 8) == 0
    assert lib.sca_linear_i8_workspace_bytes(-1, 5, 8) == lib.sca_linear_i8_workspace_bytes(1, -1, 8) == -1
    assert lib.sca_linear_i8_workspace_bytes(1, 5, 1 << 17) == -1
    ok = (a, 1, a, 1, 32, None, 0, 1e-3, 0.9, 0.999, 1e-8, 0, a, None)
    for i, bad in ((0, None), (1, -1), (2, None), (3, -1), (4, 16), (6, -1), (8, 1.0), (9, -0.1), (10, -1.0), (12, None), (12, a + 8)):
        assert lib.sca_adamw_step(*ok[:i], bad, *ok[i + 1:]) == -1, i
    assert lib.sca_adamw_step(a, 1, a, 1, 8, a, 0, 1e-3, 0.9, 0.999, 1e-8, 0, a, None) == -1       # hyper: 32 bits only
    assert lib.sca_adamw_step(a, 1, a, 1, 32, a, 3, 1e-3, 0.9, 0.999, 1e-8, 0, a, None) == -1      # and no step number


def test_too_wide():
    """Columns are counted in 32 bits; a width that would wrap is refused (nothing of that size is allocated here)."""
    wide = t(1).expand(2 ** 32 + 5)
    for call in (lambda: ops.layer_norm(wide), lambda: ops.quantize_int8(wide),
                 lambda: ops.int8_linear(t(4), torch.zeros(1, 1, dtype=I8).expand(2 ** 32 + 5, 4), t(1).expand(2 ** 32 + 5))):
        with pytest.raises(ValueError):
            call()
    lib, a, n = _lib.load(), 1 << 20, 0x7fffffff
    assert lib.sca_layernorm_fwd(a, n, 0, 1, n, None, None, 0, 1e-5, a, n, a, None) == -1
    assert lib.sca_layernorm_bwd_workspace_floats(1, n) == -1
    assert lib.sca_quant_rows_i8(a, n, 0, 1, n, a, n, a, None) == -1
    assert lib.sca_gemm_i8(a, 4, a, a, 4, a, None, 0, 1, n, 4, a, 0, n, None) == -1
    # rows beyond the registers need the workspace for dx as well
    assert lib.sca_layernorm_bwd(a, 30000, a, 30000, 0, 1, 30000, None, 0, a, a, 30000, None, None, None, None) == -1
    assert lib.sca_adamw_set_grads(None, 1, a, None) == -1 and lib.sca_adamw_set_grads(a, -1, a, None) == -1
    assert lib.sca_adamw_set_grads(None, 0, None, None) == 0
    with pytest.raises(ValueError):
        ops.AdamW([t(3)]).set_step(-1)


def test_csr_rows_entry_point():
    lib, a = _lib.load(), 1 << 20
    ok = (a, a, a, None, 4, 100, 1, a, 112, a, None)
    for i, bad in ((0, None), (1, None), (2, None), (4, -1), (5, 0), (7, None), (7, a + 4), (8, 96), (8, 100), (9, None)):
        assert lib.sca_csr_quant_rows_i8(*ok[:i], bad, *ok[i + 1:]) == -1, i
    assert lib.sca_csr_quant_rows_i8(a, a, a, None, 4, 65537, 1, a, 65552, a, None) == -2       # wider than the LDS
    assert lib.sca_csr_quant_rows_i8(a, a, a, None, 0, 100, 1, a, 112, a, None) == 0


def torch_states(cls, steps=2, **kw):
    p = t(4, 3).requires_grad_()
    opt = cls([p], lr=1e-2, weight_decay=0.1, **kw)
    for _ in range(steps):
        p.grad = t(4, 3) + 0.5
        opt.step()
    return opt.state_dict()


@pytest.mark.parametrize("cls,kw,error", [
    (torch.optim.AdamW, dict(amsgrad=True), "amsgrad"), (torch.optim.AdamW, dict(maximize=True), "maximize"),
    (torch.optim.AdamW, dict(amsgrad=True, steps=0), "amsgrad"), (torch.optim.Adam, dict(), "torch.optim.Adam,"),
    (torch.optim.SGD, dict(momentum=0.9), "another optimizer")])
def test_adamw_takes_up_no_other_rule(cls, kw, error):
    """A state dict whose next step would not be this class's: refused, with the optimizer as it was."""
    opt = ops.AdamW([t(4, 3)], lr=0.3)
    sd = torch_states(cls, **kw)
    with pytest.raises(ValueError, match=error):
        opt.load_state_dict(sd)
    assert opt.param_groups[0]["lr"] == 0.3 and not opt.state


def test_adamw_takes_up_torch_states():
    sd = torch_states(torch.optim.AdamW)
    p = t(4, 3)
    opt = ops.AdamW([p], lr=0.3)
    opt.load_state_dict(sd)
    assert opt.param_groups[0]["lr"] == 1e-2 and opt.state_dict()["state"][0]["step"] == 2
    assert torch.equal(opt.state[p]["exp_avg_sq"], sd["state"][0]["exp_avg_sq"])
    for change in (lambda s: s["state"][0].pop("exp_avg"), lambda s: s["state"][0].update(max_exp_avg_sq=t(4, 3)),
                   lambda s: s["param_groups"][0].update(lr=torch.tensor(0.1)),
                   lambda s: s["param_groups"][0].update(betas=(torch.tensor(0.9), 0.999))):
        other = torch_states(torch.optim.AdamW)
        change(other)
        with pytest.raises(ValueError):
            opt.load_state_dict(other)
    with pytest.raises(ValueError, match="8-bit states"):
        ops.AdamW([p], state_bits=8).load_state_dict(sd)
    assert opt.state_dict()["state"][0]["step"] == 2


def test_one_launch_for_one_row_has_its_limit():
    """A workspace (two launches) where the direct kernel would start 2^32 threads or more."""
    lib = _lib.load()
    most = (1 << 27) - 16
    for m in (1, 2):
        assert lib.sca_linear_i8_workspace_bytes(m, most, 8) == 0 and lib.sca_linear_i8_workspace_bytes(m, most + 1, 8) >= m * 12


def test_int8_latents_of_too_many_genes():
    """Refused where the weight is quantized, before any cell is gathered."""
    import types

    from scarches_amd.engine import CVAEEngine
    lib, layer = types.SimpleNamespace(_lib=_lib.load()), lambda n: [types.SimpleNamespace(n_in=n, w="w")]
    most = _lib.load().sca_gemm_i8_max_k()
    for n, error in ((most + 1, ValueError), (most, _lib.HipLibraryError)):
        eng = types.SimpleNamespace(lib=lib, enc=layer(n), p=dict(w=t(2, n)))
        with pytest.raises(error):
            CVAEEngine.quantize_first_layer(eng)
