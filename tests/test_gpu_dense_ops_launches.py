"""GPU tests of scarches_amd.ops at sizes that one launch does not hold (2^32 threads and more): widths, outputs and rows that
the documentation allows.  References and bounds as in test_gpu_dense_ops."""
import numpy as np
import pytest
import torch

from tests.test_gpu_dense_ops import TYPES, gen, grid_ref, ln_check_bwd, philox_words

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops():
    from scarches_amd import ops as m
    return m


@pytest.mark.parametrize("n,dtype", [((1 << 24) + 5, t) for t in TYPES] + [((1 << 26) + 3, torch.float32)], ids=str)
def test_layer_norm_gradients_of_wide_rows(ops, n, dtype):
    x, dy = (torch.randn(2, n, device="cuda", generator=gen(s)).to(dtype) for s in (1, 2))
    w = (1 + 0.2 * torch.randn(n, device="cuda", generator=gen(3))).to(dtype)
    _, stats = ops.layer_norm_fwd(x, w, w)
    ln_check_bwd(ops, dy, x, w, stats)
    _, _, db = ops.layer_norm_bwd(dy, x, w, stats, (False, False, True))
    assert torch.equal(db, (dy[0].float() + dy[1].float()).to(dtype))          # one rounding in fp32, one to the type
    assert db[-1] != 0 and db[-1].isfinite()


@pytest.mark.parametrize("m", [1, 2, 3])
def test_int8_linear_of_very_many_outputs(ops, m):
    """Small integers: quantized without a remainder (the largest is 127), and sums that every type holds."""
    n, k = (1 << 27) + 5, 4
    x = torch.randint(-3, 4, (m, k), device="cuda", generator=gen(m)).float()
    x[:, 0] = 127
    wq = torch.randint(-3, 4, (n, k), device="cuda", generator=gen(4), dtype=torch.int8)
    ws = torch.ones(n, device="cuda")
    got = ops.int8_linear(x, wq, ws)
    for r in range(m):
        want = sum(x[r, c] * wq[:, c].float() for c in range(k))
        assert torch.equal(got[r], want), r


def test_int8_matmul_of_very_many_rows(ops):
    """Rows behind the first slice of a launch's worth, with an odd pitch."""
    m, n, k = (1 << 31) + 70, 1, 1
    xq = torch.empty(m, k, dtype=torch.int8, device="cuda").random_(-3, 4, generator=gen(1))
    sx = torch.ones(m, device="cuda")
    sx[-5:] = 2.0
    wq = torch.full((n, k), 3, dtype=torch.int8, device="cuda")
    got = ops.int8_matmul(xq, sx, wq, torch.ones(n, device="cuda"), None, torch.bfloat16)
    xq.mul_(3)                                              # (within int8)
    xq[-5:].mul_(2)
    step = 1 << 28
    for lo in range(0, m, step):
        assert torch.equal(got[lo:lo + step], xq[lo:lo + step].bfloat16()), lo


@pytest.mark.parametrize("chosen", [False, True])
def test_csr_rows_of_very_many_cells(ops, chosen):
    """Cells behind the first launch's, of all rows and of rows that are chosen (here: backwards)."""
    from scarches_amd import _lib
    lib, b = _lib.load(), (1 << 26) + 3
    data = torch.empty(b, device="cuda").random_(0, 50, generator=gen(1))              # one count per cell, in column cell % 3
    indptr = torch.arange(b + 1, device="cuda")
    indices = (torch.arange(b, device="cuda") % 3).int()
    rows = torch.arange(b - 1, -1, -1, device="cuda") if chosen else None
    q = torch.full((b + 1, 16), 99, dtype=torch.int8, device="cuda")
    scale = torch.full((b + 1,), -1.0, device="cuda")
    _lib.check(lib.sca_csr_quant_rows_i8(indptr.data_ptr(), indices.data_ptr(), data.data_ptr(), _lib.ptr(rows), b, 3, 0, q.data_ptr(),
                                         16, scale.data_ptr(), torch.cuda.current_stream().cuda_stream), "csr_quant")
    if chosen:
        data, indices = data.flip(0), indices.flip(0)
    assert torch.equal(scale[:b], data / torch.full_like(data, 127)) and scale[b] == -1
    want = (indices[:, None] == torch.arange(16, device="cuda", dtype=torch.int32)[None]) & (data > 0)[:, None]
    assert torch.equal(q[:b], want.to(torch.int8) * 127) and (q[b] == 99).all()


def words_at(first, n, tensor, t, seed, monkeypatch):
    """Random words of elements [first, first + n) of a tensor, first a multiple of 4: the counter starts there."""
    arange = np.arange
    monkeypatch.setattr(np, "arange", lambda k, dtype: arange(first // 4, first // 4 + k, dtype=dtype))
    words = philox_words(n, tensor, t, seed)
    monkeypatch.undo()
    return words


def test_adamw_8_bits_behind_32_bit_offsets(ops, monkeypatch):
    """The codes of the last block of a tensor of more than 2^31 values, value by value."""
    n, few = (1 << 31) + 1111, 1111 % 256
    first = n - few
    assert first % 256 == 0
    x = torch.full((n,), 0.5, device="cuda", dtype=torch.bfloat16)
    x.grad = torch.full((n,), 0.25, device="cuda", dtype=torch.bfloat16)
    x.grad[first:] = torch.linspace(-2, 2, few, device="cuda").bfloat16()
    opt = ops.AdamW([x], lr=0.1, state_bits=8, seed=3)
    opt.step()
    st, g = opt.state[x], x.grad[first:].double().cpu()
    words = words_at(first, few, 0, 1, 3, monkeypatch)
    for key, value, rnd, kind in (("exp_avg", (1 - 0.9) * g, words & 0xffff, torch.float8_e4m3fn),
                                  ("exp_avg_sq", (1 - 0.999) * g * g, words >> 16, torch.float8_e5m2)):
        code, scale = grid_ref(value.float().numpy(), rnd, kind)
        np.testing.assert_array_equal(st[key][first:].view(torch.uint8).cpu().numpy(), code[:few])
        assert st[key + "_scale"][-1].item() == scale[0] and len(set(code[:few])) > 20, key
