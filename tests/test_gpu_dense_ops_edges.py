"""GPU tests of scarches_amd.ops at the edges of what its documentation allows: rows beyond the registers in both directions,
gradients that autograd hands over as one repeated row or value, copies and pickles of the optimizer, gradients in new storage
at every step, calls side by side on two streams.  Bounds as in test_gpu_dense_ops."""
import copy
import io

import numpy as np
import pytest
import torch

from tests.test_gpu_dense_ops import TYPES, U, gen, ln_check_bwd, ln_check_fwd, matrix, quant_ref, within

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops():
    from scarches_amd import ops as m
    return m


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("layout", ["plain", "odd", "expanded"])
@pytest.mark.parametrize("rows,n", [(1, 16385), (7, 33538), (600, 20001), (9, 131072), (300, 20480), (520, 20477), (700, 24573), (40, 40960)])
def test_layer_norm_long_rows(ops, rows, n, layout, dtype):
    x, dy = matrix(rows, n, dtype, n, layout), matrix(rows, n, dtype, n + 1, layout)
    w = (1 + 0.2 * torch.randn(n, device="cuda", generator=gen(1))).to(dtype)
    _, stats = ln_check_fwd(ops, x, w, w)
    ln_check_bwd(ops, dy, x, w, stats)
    dx, dw, db = ops.layer_norm_bwd(dy, x, w, stats)
    for need in ((True, False, False), (False, True, True), (False, False, True), (False, False, False)):
        for one, some in zip((dx, dw, db), ops.layer_norm_bwd(dy, x, w, stats, need)):
            assert some is None or torch.equal(one, some)
        assert [g is not None for g in ops.layer_norm_bwd(dy, x, w, stats, need)] == list(need)


@pytest.mark.parametrize("n", [3, 128, 1001, 20000])
def test_layer_norm_repeated_gradients(ops, n):
    """sum(0) hands one row of gradients to every row, sum() one value."""
    x = matrix(37, n, torch.float32, 5).clone().requires_grad_()
    w = (1 + 0.1 * torch.randn(n, device="cuda", generator=gen(6))).requires_grad_()
    b = torch.zeros(n, device="cuda", requires_grad=True)
    row = torch.randn(n, device="cuda", generator=gen(7))
    for loss, dy in ((lambda y: (y.sum(0) * row).sum(), row.expand(37, n)),
                     (lambda y: 0.5 * y.sum(), torch.full((1, 1), 0.5, device="cuda").expand(37, n))):
        got = torch.autograd.grad(loss(ops.layer_norm(x, w, b)), (x, w, b))
        _, stats = ops.layer_norm_fwd(x.detach(), w.detach(), b.detach())
        ln_check_bwd(ops, dy, x.detach(), w.detach(), stats)
        for a, c in zip(got, ops.layer_norm_bwd(dy, x.detach(), w.detach(), stats)):
            assert torch.equal(a, c)


def params(seed, dtype=torch.float32):
    return [torch.randn(s, device="cuda", generator=gen(seed + i)).to(dtype).requires_grad_()
            for i, s in enumerate([(33, 20), (33,), (1, 5000), (257,)])]


def set_grads(ps, seed, fresh=True):
    for i, p in enumerate(ps):
        g = torch.randn(p.shape, device="cuda", generator=gen(1000 * seed + i)).to(p.dtype)
        if fresh or p.grad is None:
            p.grad = g
        else:
            p.grad.copy_(g)


@pytest.mark.parametrize("bits", [32, 8])
def test_adamw_copies(ops, bits):
    """A deep copy and a pickle take the next steps as the original does."""
    ps = params(1)
    opt = ops.AdamW(ps, lr=1e-2, state_bits=bits, seed=9)
    for s in range(3):
        set_grads(ps, s)
        opt.step()
    both = copy.deepcopy((ps, opt))
    buf = io.BytesIO()
    torch.save((ps, opt), buf)              # (torch's pickler: tensors on the device)
    buf.seek(0)
    again = torch.load(buf, weights_only=False)
    for s in range(3, 6):
        for group, o in ((ps, opt), both, again):
            set_grads(group, s)
            o.step()
    for group, o in (both, again):
        assert o.state_dict()["state"][0]["step"] == 6
        for a, b in zip(ps, group):
            assert a is not b and torch.equal(a, b)


@pytest.mark.parametrize("bits", [32, 8])
def test_adamw_new_gradients_every_step(ops, bits):
    """Gradients that are dropped and made anew, and gradients in one place, give the same bits."""
    a, b = params(2), params(2)
    oa, ob = ops.AdamW(a, state_bits=bits), ops.AdamW(b, state_bits=bits)
    held = []
    for s in range(8):
        oa.zero_grad(set_to_none=True)
        set_grads(a, s)
        held += [p.grad for p in a][: s % 3]                # keeps the allocator from giving back the same storage
        set_grads(b, s, fresh=False)
        oa.step()
        ob.step()
    for p, q in zip(a, b):
        assert torch.equal(p, q)


@pytest.mark.parametrize("bits", [32, 8])
def test_adamw_steps_known_and_counted(ops, bits):
    """The step number given by the host and the one that the device counts, before and after a parameter misses a step."""
    a, b = params(3), params(3)
    oa, ob = ops.AdamW(a, state_bits=bits), ops.AdamW(b, state_bits=bits)
    ob._host_steps[0] = (None, None)
    for s in range(6):
        set_grads(a, s)
        set_grads(b, s)
        if s == 3:
            a[1].grad = b[1].grad = None
        oa.step()
        ob.step()
    steps = [oa.state_dict()["state"][i]["step"] for i in range(4)]
    assert steps == [ob.state_dict()["state"][i]["step"] for i in range(4)] == [6, 5, 6, 6]
    for p, q in zip(a, b):
        # the coefficients' logarithms are the host's in one, the device's in the other: their roundings may differ
        within(p.detach(), q.detach().double(), 64 * U * (q.detach().double().abs() + 6e-3), "p")
    oa.set_step(10)
    set_grads(a, 9)
    oa.step()
    assert [oa.state_dict()["state"][i]["step"] for i in range(4)] == [11] * 4


@pytest.mark.parametrize("bits", [32, 8])
def test_adamw_frozen_parameters(ops, bits):
    """Parameters without gradients take no step and count none; one that joins later starts at its own first step, also after
    the states went through a state dict."""
    a, b, c = params(6), params(6), params(6)
    oa, ob = ops.AdamW(a, state_bits=bits), ops.AdamW(b, state_bits=bits)
    ob._host_steps[0] = (None, None)                       # counted on the device throughout
    for s in range(4):
        for ps in (a, b):
            set_grads(ps, s)
            ps[2].grad = None
        oa.step()
        ob.step()
    assert oa._host_steps[0] == (4, 0b1101) and torch.equal(a[2], c[2])
    oc = ops.AdamW(c, state_bits=bits)
    oc.load_state_dict(oa.state_dict())
    for p, q in zip(c, a):
        p.data.copy_(q.data)
    assert oc._host_steps[0] == (4, 0b1101)
    for s in range(4, 8):
        for ps, o in ((a, oa), (b, ob), (c, oc)):
            set_grads(ps, s)
            if s < 6:
                ps[2].grad = None
            o.step()
    for o in (oa, ob, oc):
        assert [o.state_dict()["state"][i]["step"] for i in range(4)] == [8, 8, 2, 8]
    for p, q, r in zip(a, b, c):
        assert torch.equal(p, r)
        within(p.detach(), q.detach().double(), 64 * U * (q.detach().double().abs() + 1e-2), "p")


def test_adamw_first_step_is_not_captured(ops):
    """States that a capture would create are zeroed by its replays only: refused, and nothing is left behind."""
    ps = params(4)
    set_grads(ps, 0)
    opt = ops.AdamW(ps)
    with pytest.raises(RuntimeError, match="before the capture"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            ps[0].grad.zero_()                  # (never replayed; the graph is not left without a node)
            opt.step()
    assert all(not opt.state[p] for p in ps)
    opt.step()
    torch.cuda.synchronize()


@pytest.mark.parametrize("bits", [32, 8])
def test_adamw_captured_with_its_gradients(ops, bits):
    """Gradients that are made inside the capture, and eager steps with others before, between and after the replays."""
    a, b = params(5), params(5)
    scale = torch.ones((), device="cuda")
    oa, ob = ops.AdamW(a, state_bits=bits, seed=1), ops.AdamW(b, state_bits=bits, seed=1)
    def gradients(ps):
        for p in ps:
            p.grad = p.detach() * scale + 0.1
    for o, ps in ((oa, a), (ob, b)):
        set_grads(ps, 1)
        o.step()
        set_grads(ps, 2)
        o.step()
    graph = torch.cuda.CUDAGraph()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.graph(graph, stream=s):
        gradients(b)
        ob.step()
    with pytest.raises(RuntimeError, match="before the capture"):      # the table of the first one is the graph's
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            gradients(b)
            ob.step()
    for i in range(8):
        if i % 3 == 2:
            set_grads(a, 20 + i)
            set_grads(b, 20 + i)
            oa.step()
            ob.step()
        else:
            scale.fill_(1.0 + i)
            gradients(a)
            oa.step()
            graph.replay()
        if i % 2:
            torch.cuda.synchronize()
        for p, q in zip(a, b):
            assert torch.equal(p, q), i
    assert ob.state_dict()["state"][0]["step"] == 10


def test_adamw_many_tensors(ops):
    """More tensors than one launch of addresses holds."""
    ps = [torch.randn(3, device="cuda", generator=gen(i)).requires_grad_() for i in range(1000)]
    qs = [p.detach().clone().requires_grad_() for p in ps]
    a, b, held = ops.AdamW(ps), ops.AdamW(qs), []
    for s in range(3):
        set_grads(ps, s)
        held.append([p.grad for p in ps])               # new storage at every step
        set_grads(qs, s, fresh=False)
        a.step()
        b.step()
    assert all(torch.equal(p, q) for p, q in zip(ps, qs))


def test_two_streams(ops):
    """Every operator at once on two streams, each call with tensors and workspaces of its own."""
    def work(seed):
        x = matrix(2000, 1001, torch.bfloat16, seed)
        w = torch.ones(1001, device="cuda", dtype=torch.bfloat16)
        y, stats = ops.layer_norm_fwd(x, w, w)
        grads = ops.layer_norm_bwd(y, x, w, stats)
        wq, ws = ops.quantize_int8(matrix(300, 1001, torch.float32, seed + 1))
        out = ops.int8_linear(x, wq, ws), ops.int8_linear(x[:1], wq, ws)
        ps = params(seed)
        opt = ops.AdamW(ps, state_bits=8, seed=seed)
        for s in range(3):
            set_grads(ps, s)
            opt.step()
        return [y, *grads, *out, *[p.detach() for p in ps]]
    alone = [work(1), work(2)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(3):
        together = []
        for seed, st in zip((1, 2), streams):
            st.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(st):
                together.append(work(seed))
        torch.cuda.synchronize()
        for one, two in zip(alone, together):
            for a, b in zip(one, two):
                assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("rows,k", [(5, 16388), (3, 20480), (4, 20481), (3, 32768), (2, 32771), (3, 40960), (2, 40961), (2, 65536), (2, 65537)])
def test_quantize_long_rows(ops, rows, k, dtype):
    x = matrix(rows, k, dtype, rows + k, "odd", scale=3.0)
    q, s = ops.quantize_int8(x)
    rq, rs = quant_ref(x.float().cpu().numpy())
    assert torch.equal(s.cpu(), torch.from_numpy(rs)) and torch.equal(q.cpu(), torch.from_numpy(rq))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=str)
@pytest.mark.parametrize("power", [0, -9, 7])
def test_quantize_every_short_value(ops, dtype, power):
    """Rows that hold every value of the type in the nine binades below their largest, for every fraction of the largest (bf16;
    every ninth of fp16): the quotients lie next to the middles between two integers all the time."""
    bits = 7 if dtype == torch.bfloat16 else 10
    frac = torch.arange(2 ** bits, 2 ** (bits + 1), dtype=torch.float64) / 2 ** bits          # [1, 2)
    values = torch.cat([frac * 2.0 ** -e for e in range(9)])
    values = torch.cat([values, -values])
    top = frac if bits == 7 else frac[::9]
    x = torch.where(values.abs()[None] <= top[:, None], values[None], torch.zeros(()).double())
    x = torch.cat([x, top[:, None]], 1) * 2.0 ** power
    x = x.to(dtype)                     # (exact but for what fp16 holds as denormal numbers, below 2^-14)
    q, s = ops.quantize_int8(x.cuda())
    rq, rs = quant_ref(x.float().numpy())
    assert torch.equal(s.cpu(), torch.from_numpy(rs)) and torch.equal(q.cpu(), torch.from_numpy(rq))


def test_quantize_next_to_every_middle(ops):
    """fp32 rows of random scales with the values next to all 127 middles, up to three steps of the type to either side."""
    g = np.random.default_rng(3)
    top = (g.random(400) + 0.5).astype(np.float32) * np.exp2(g.integers(-60, 60, 400)).astype(np.float32)
    top[:3] = 127.0, 254.0, 1.0
    s = top / np.float32(127)
    mid = np.float32((np.arange(127) + 0.5) * s.astype(np.float64)[:, None])
    rows = [top[:, None]]
    for direction in (np.float32(0), np.float32(np.inf)):
        v = mid
        for _ in range(4):
            rows += [v, -v]
            v = np.nextafter(v, direction)
    x = np.minimum(np.maximum(np.concatenate(rows, 1), -top[:, None]), top[:, None]).astype(np.float32)
    q, sc = ops.quantize_int8(torch.from_numpy(x).cuda())
    rq, rs = quant_ref(x)
    np.testing.assert_array_equal(sc.cpu().numpy(), rs)
    np.testing.assert_array_equal(q.cpu().numpy(), rq)


@pytest.mark.parametrize("m,n,ks", [(33, 40, range(1, 300)), (2000, 512, range(391, 660, 11)), (4096, 800, range(123, 400, 13)),
                                    (8192, 1536, range(60, 330, 27))])
def test_int8_every_tail(ops, m, n, ks):
    """Rows of every length: small integers, whose products' sums fp32 holds exactly, with padded and with packed rows."""
    g = gen(m)
    for k in ks:
        pitch = -(-k // 128) * 128
        xq, wq = (torch.full((s, pitch), 100, dtype=torch.int8, device="cuda")[:, :k] for s in (m, n))
        xq.random_(-3, 4, generator=g)
        wq.random_(-3, 4, generator=g)
        want = (xq.float() @ wq.float().t().contiguous())
        one_m, one_n = torch.ones(m, device="cuda"), torch.ones(n, device="cuda")
        for x, w in ((xq, wq), (xq.contiguous(), wq.contiguous())):
            assert torch.equal(ops.int8_matmul(x, one_m, w, one_n), want), (k, x.stride())


@pytest.mark.parametrize("k", [16, 112, 127, 128, 129, 1008, 2000, 2048, 8064, 8070])
@pytest.mark.parametrize("m,n", [(1, 50), (2, 33), (3, 50), (100, 130), (700, 600)])
def test_int8_linear_is_its_two_parts(ops, m, n, k):
    """Quantized in the launch, in a workspace of whichever pitch, or by the caller: the same bits."""
    x = matrix(m, k, torch.float32, m + k, "pitch")
    wq, ws = ops.quantize_int8(torch.randn(n, k, device="cuda", generator=gen(3)))
    bias = torch.randn(n, device="cuda", generator=gen(4))
    q, s = ops.quantize_int8(x)
    want = ops.int8_matmul(q, s, wq, ws, bias)
    assert torch.equal(ops.int8_linear(x, wq, ws, bias), want)
    # the workspace is as large as it says: guarded by a block of known bytes behind it
    from scarches_amd import _lib
    lib = _lib.load()
    size = lib.sca_linear_i8_workspace_bytes(m, n, k)
    buf = torch.full((size + 4096,), 85, dtype=torch.int8, device="cuda")
    y = torch.empty(m, n, device="cuda")
    _lib.check(lib.sca_linear_i8(x.data_ptr(), x.stride(0), 0, wq.data_ptr(), wq.stride(0), ws.data_ptr(), bias.data_ptr(), 0, m,
                                 n, k, y.data_ptr(), 0, n, buf.data_ptr(), torch.cuda.current_stream().cuda_stream), "linear_i8")
    assert torch.equal(y, want) and (buf[size:] == 85).all()


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("m,n,k", [(512, 700, 512), (513, 1025, 1001), (2000, 300, 2049), (600, 2100, 777), (900, 333, 20001)])
def test_int8_linear_aligns_the_weight(ops, m, n, k, dtype):
    """Weights that lie packed, with an odd pitch or from an odd address give the bits of the padded one."""
    x = matrix(m, k, dtype, m + k, "odd")
    wq, ws = ops.quantize_int8(torch.randn(n, k, device="cuda", generator=gen(3)))
    q, s = ops.quantize_int8(x)
    want = ops.int8_matmul(q, s, wq, ws, None, dtype)
    buf = torch.full((n * (k + 7) + 1,), -128, dtype=torch.int8, device="cuda")
    for w in (wq, wq.contiguous(), torch.as_strided(buf, (n, k), (k + 7, 1), 1).copy_(wq),
              wq.t().contiguous().t()):
        assert torch.equal(ops.int8_linear(x, w, ws), want), w.stride()
