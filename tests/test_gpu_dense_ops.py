"""GPU tests of scarches_amd.ops: layer norm, AdamW with 32- and 8-bit states, the 8-bit integer product, each against a plain
64-bit implementation, at the sizes, pitches and values where they can go wrong.

Tolerances: U = 2^-24 is the largest relative error of one fp32 rounding, HALF[t] that of the rounding to the result's type.
A sum of n terms of which a lane takes n / 64 one after another, followed by a tree over 64 lanes, is off by at most
(n / 64 + 6) U times the sum of the terms' absolute values; each test multiplies the magnitudes that enter its formula by the
number of roundings on the way."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
TYPES = [torch.float32, torch.bfloat16, torch.float16]
HALF = {t: torch.finfo(t).eps / 2 for t in TYPES}
TINY = {t: torch.finfo(t).smallest_normal * torch.finfo(t).eps for t in TYPES}       # spacing of the denormal numbers


@pytest.fixture(scope="module")
def ops():
    from scarches_amd import ops as m
    return m


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def within(got, want, bound, what):
    """|got - want| <= bound everywhere (64-bit tensors); names the worst place."""
    assert got.shape == want.shape, (what, got.shape, want.shape)
    off = (got.double() - want).abs() - bound
    if off.numel():
        assert torch.isfinite(got.double()).all(), what
        i = int(off.argmax())
        assert off.reshape(-1)[i] <= 0, (what, i, got.reshape(-1)[i].item(), want.reshape(-1)[i].item(),
                                         bound.expand_as(off).reshape(-1)[i].item())


# ---------------------------------------------------------------------------------------------- layer norm
def matrix(rows, n, dtype, seed, layout="plain", scale=1.0):
    """[rows, n] values with an offset per row: contiguous, with a pitch, from an odd address, or one row repeated."""
    g = gen(seed)
    if layout == "expanded":
        return torch.randn(1, n, device="cuda", generator=g).to(dtype).expand(rows, n)
    pad = {"plain": 0, "pitch": 5, "odd": 3}[layout]
    v = torch.randn(rows, n + pad, device="cuda", generator=g) * scale + torch.randn(rows, 1, device="cuda", generator=g)
    if layout == "odd":
        return v.to(dtype)[:, 1:1 + n]
    return v.to(dtype)[:, :n]


def ln_ref(x, w, b, eps):
    x = x.double()
    mean = x.mean(1, keepdim=True)
    rstd = 1 / ((x - mean).square().mean(1, keepdim=True) + eps).sqrt()
    h = (x - mean) * rstd
    y = h * (1 if w is None else w.double()) + (0 if b is None else b.double())
    return y, mean, rstd, h


def ln_check_fwd(ops, x, w, b, eps=1e-5):
    y, stats = ops.layer_norm_fwd(x, w, b, eps)
    n = x.shape[-1]
    ref, mean, rstd, h = ln_ref(x.reshape(-1, n), w, b, eps)
    c = (n / 64 + 16) * U
    aw = 1.0 if w is None else w.double().abs()
    mag = x.reshape(-1, n).double().abs().mean(1, keepdim=True)
    # the mean's error shifts the row; rstd, the product and the sum with b are off by a few roundings each
    bound = c * (mag * rstd + h.abs()) * aw + 2 * U * (0 if b is None else b.double().abs()) + HALF[x.dtype] * ref.abs() \
        + TINY[x.dtype]
    within(y.reshape(-1, n), ref, bound, "y")
    within(stats[0], mean[:, 0], c * mag[:, 0] + 1e-37, "mean")
    within(stats[1], rstd[:, 0], c * rstd[:, 0] * (1 + (mag * rstd)[:, 0]), "rstd")
    return y, stats


def ln_check_bwd(ops, dy, x, w, stats):
    n = x.shape[-1]
    dx, dw, db = ops.layer_norm_bwd(dy, x, w, stats)
    xd, dyd = x.reshape(-1, n).double(), dy.reshape(-1, n).double()
    rows = xd.shape[0]
    mean, rstd = stats[0].double()[:, None], stats[1].double()[:, None]
    h = (xd - mean) * rstd
    a = dyd * (1 if w is None else w.double())
    m1, m2 = a.mean(1, keepdim=True), (a * h).mean(1, keepdim=True)
    ref = rstd * (a - m1 - h * m2)
    # h itself carries the cancellation of x - mean: U (|x| + |mean|) rstd
    eh = 3 * U * (xd.abs() + mean.abs()) * rstd
    bound = (n / 64 + 16) * U * rstd * (a.abs() + a.abs().mean(1, keepdim=True) + h.abs() * (a * h).abs().mean(1, keepdim=True)) \
        + rstd * (eh * m2.abs() + h.abs() * (a.abs() * eh).mean(1, keepdim=True)) + HALF[x.dtype] * ref.abs() + TINY[x.dtype]
    within(dx.reshape(-1, n), ref, bound, "dx")
    if w is None:
        assert dw is None and db is None
        return
    c = (min(rows, 256) + rows / 256 + 8) * U           # up to 256 partial sums, each over its share of the rows
    for got, terms, err, name in ((dw, dyd * h, dyd.abs() * eh, "dw"), (db, dyd, 0 * dyd, "db")):
        ref = terms.sum(0)
        within(got, ref, c * terms.abs().sum(0) + err.sum(0) + HALF[w.dtype] * ref.abs() + TINY[w.dtype], name)


LN_SIZES = [(1, 1), (1, 7), (3, 64), (5, 10), (128, 128), (67, 200), (33, 257), (1021, 1001), (64, 2000), (9, 4100), (2, 8192),
            (3, 16385), (2, 40000), (300, 3), (20000, 16), (4097, 96)]


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("rows,n", LN_SIZES)
def test_layer_norm_sizes(ops, rows, n, dtype):
    x = matrix(rows, n, dtype, rows + 7 * n)
    w = (1 + 0.2 * torch.randn(n, device="cuda", generator=gen(1))).to(dtype)
    b = (0.3 * torch.randn(n, device="cuda", generator=gen(2))).to(dtype)
    dy = matrix(rows, n, dtype, rows + 7 * n + 1)
    _, stats = ln_check_fwd(ops, x, w, b)
    ln_check_bwd(ops, dy, x, w, stats)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("layout", ["pitch", "odd", "expanded"])
@pytest.mark.parametrize("rows,n", [(65, 128), (37, 1001), (11, 4096), (260, 33)])
def test_layer_norm_layouts(ops, rows, n, layout, dtype):
    """Rows with a pitch, from addresses that are aligned to their element only, and one row repeated (pitch 0); without
    weight, with a float32 weight on 16-bit rows, and through more than two dimensions."""
    x, dy = matrix(rows, n, dtype, 3, layout), matrix(rows, n, dtype, 4, layout)
    for w, b in ((None, None), (1 + 0.1 * torch.randn(n, device="cuda", generator=gen(5)), None)):
        _, stats = ln_check_fwd(ops, x, w, b)
        ln_check_bwd(ops, dy, x, w, stats)
    x4 = torch.randn(2, 3, 4, n, device="cuda", generator=gen(6)).to(dtype).transpose(0, 2)
    y, stats = ln_check_fwd(ops, x4, w, w)
    assert y.shape == x4.shape
    odd = torch.empty(n + 1, device="cuda").normal_(generator=gen(8)).to(dtype)[1:]
    ln_check_fwd(ops, x, odd, odd)


@pytest.mark.parametrize("n", [1, 5, 100, 3000, 20000])
def test_layer_norm_values(ops, n):
    """Constant rows (variance 0), large offsets, values near the type's ends, NaN and infinities in one row only."""
    x = torch.randn(8, n, device="cuda", generator=gen(n))
    x[0] = 3.0
    x[1] += 1e4
    x[2] *= 1e-18
    x[3] *= 1e15
    w = 1 + 0.1 * torch.randn(n, device="cuda", generator=gen(9))
    _, stats = ln_check_fwd(ops, x, w, w)
    ln_check_bwd(ops, torch.randn_like(x), x, w, stats)
    bad = x.clone()
    bad[4, n // 2] = float("nan")
    bad[6, 0] = float("inf")
    y, st = ops.layer_norm_fwd(bad, w, w)
    good, _ = ops.layer_norm_fwd(x, w, w)
    for r in range(8):
        assert torch.isnan(y[r]).all() if r in (4, 6) else torch.equal(y[r], good[r]), r
    dx, dw, _ = ops.layer_norm_bwd(torch.ones_like(x), bad, w, st)
    keep, _, _ = ops.layer_norm_bwd(torch.ones_like(x), x, w, stats)
    assert torch.isnan(dx[4]).all() and torch.isnan(dx[6]).all() and torch.isnan(dw).all()
    assert torch.equal(dx[[0, 1, 2, 3, 5, 7]], keep[[0, 1, 2, 3, 5, 7]])


@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_layer_norm_no_rows_and_parts(ops, dtype):
    x = torch.empty(0, 40, device="cuda", dtype=dtype)
    w = torch.ones(40, device="cuda", dtype=dtype)
    y, stats = ops.layer_norm_fwd(x, w, w)
    assert y.shape == (0, 40) and stats.shape == (2, 0)
    dx, dw, db = ops.layer_norm_bwd(x, x, w, stats)
    assert dx.shape == (0, 40) and not dw.any() and not db.any()
    x = torch.randn(30, 40, device="cuda", generator=gen(1)).to(dtype)
    _, stats = ops.layer_norm_fwd(x, w, w)
    full = ops.layer_norm_bwd(x, x, w, stats)
    for need in ((True, False, False), (False, True, False), (False, False, True), (False, True, True), (True, False, True)):
        for got, want, asked in zip(ops.layer_norm_bwd(x, x, w, stats, need), full, need):
            assert torch.equal(got, want) if asked else got is None


def test_layer_norm_repeats_bit_for_bit_and_writes_only_its_rows(ops):
    from scarches_amd import _lib
    lib = _lib.load()
    x, dy = matrix(3001, 777, torch.float32, 1), matrix(3001, 777, torch.float32, 2)
    w = torch.ones(777, device="cuda")
    _, stats = ops.layer_norm_fwd(x, w, w)
    a, b = ops.layer_norm_bwd(dy, x, w, stats), ops.layer_norm_bwd(dy, x, w, stats)
    assert all(torch.equal(p, q) for p, q in zip(a, b))
    # into the middle of a larger matrix: nothing beside, before or behind it changes
    for rows, n in ((5, 12), (130, 33), (4, 5000)):
        out = torch.full((rows + 2, n + 6), 7.0, device="cuda")
        xs = matrix(rows, n, torch.float32, 3)
        ws = torch.ones(n, device="cuda")
        st = torch.cuda.current_stream().cuda_stream
        _lib.check(lib.sca_layernorm_fwd(xs.data_ptr(), xs.stride(0), 0, rows, n, ws.data_ptr(), None, 0, 1e-5,
                                         out[1, 3:].data_ptr(), n + 6, None, st), "ln")
        y, stats = ops.layer_norm_fwd(xs, ws)
        assert torch.equal(out[1:-1, 3:-3], y)
        out[1:-1, 3:-3] = 7.0
        assert (out == 7.0).all()
        _lib.check(lib.sca_layernorm_bwd(xs.data_ptr(), xs.stride(0), xs.data_ptr(), xs.stride(0), 0, rows, n, ws.data_ptr(), 0,
                                         stats.data_ptr(), out[1, 3:].data_ptr(), n + 6, None, None, None, st), "ln bwd")
        assert torch.equal(out[1:-1, 3:-3], ops.layer_norm_bwd(xs, xs, ws, stats)[0])
        out[1:-1, 3:-3] = 7.0
        assert (out == 7.0).all()


def test_layer_norm_autograd(ops):
    """Gradients against torch's own layer norm in 64 bits and against differences; an input that is broadcast and a weight
    that two calls share; no graph where none is wanted."""
    g = gen(11)
    x0, w0, b0 = (torch.randn(*s, device="cuda", generator=g) for s in ((6, 50), (50,), (50,)))
    probe = torch.randn(4, 6, 50, device="cuda", generator=g)

    def run(f, dt):
        x, w, b = (t.to(dt).clone().requires_grad_() for t in (x0, w0, b0))
        y = f(f(x.expand(4, 6, 50), w, b), w, b)
        (y * probe.to(dt)).sum().backward()
        return y.detach(), x.grad, w.grad, b.grad

    got = run(lambda x, w, b: ops.layer_norm(x, w, b, 1e-3), torch.float32)
    want = run(lambda x, w, b: torch.nn.functional.layer_norm(x, (50,), w, b, 1e-3), torch.float64)
    for a, b, name in zip(got, want, ("y", "dx", "dw", "db")):
        # two layers of at most (n / 64 + 16) + (rows + 24) roundings each, on values of a few units
        assert (a.double() - b).abs().max() <= 100 * U * b.abs().max().clamp_min(1) * 8, name

    x = x0.clone()
    d = torch.randn_like(x0)
    y = lambda e: ops.layer_norm_fwd(x + e * d, w0, b0)[0].double()
    _, stats = ops.layer_norm_fwd(x, w0, b0)
    dy = probe[0]
    dx, _, _ = ops.layer_norm_bwd(dy, x, w0, stats)
    h = 1e-2        # central difference: O(h^2) of the third derivative (values of ~1: 1e-4 of the sum), rounding U / h
    slope = ((y(h) - y(-h)) * dy.double()).sum() / (2 * h)
    assert abs(slope - (dx.double() * d.double()).sum()) <= 2e-3 * (dx.double() * d.double()).abs().sum()
    with torch.no_grad():
        assert not ops.layer_norm(x0.clone().requires_grad_(), w0, b0).requires_grad
    with pytest.raises(RuntimeError):       # once differentiable
        xr = x0.clone().requires_grad_()
        gx, = torch.autograd.grad(ops.layer_norm(xr, w0, b0).sum(), xr, create_graph=True)
        gx.sum().backward()


def test_layer_norm_offsets_past_32_bits(ops):
    rows, n = (1 << 31) // 1000 + 9, 1000
    x = torch.zeros(rows, n, dtype=torch.bfloat16, device="cuda")
    tail = torch.randn(6, n, device="cuda", generator=gen(1)).bfloat16()
    x[-6:] = tail
    w = torch.ones(n, device="cuda", dtype=torch.bfloat16)
    y, stats = ops.layer_norm_fwd(x, w, w)
    ty, ts = ops.layer_norm_fwd(tail, w, w)
    assert torch.equal(y[-6:], ty) and torch.equal(stats[:, -6:], ts) and (y[:6] == 1).all()
    del y
    dx, dw, db = ops.layer_norm_bwd(x, x, w, stats)
    tx, tw, tb = ops.layer_norm_bwd(tail, tail, w, ts)
    assert torch.equal(dx[-6:], tx)
    # six rows with values among zeros: sums of the same six terms, whatever the order
    assert (dw.float() - tw.float()).abs().max() <= 2 * HALF[torch.bfloat16] * tw.float().abs().max() + 1e-30
    assert (db.float() - tb.float()).abs().max() <= 2 * HALF[torch.bfloat16] * tb.float().abs().max() + 1e-30


# ---------------------------------------------------------------------------------------------- 8-bit integer product
def quant_ref(x):
    """(q, scale) of numpy rows: the quotient in 64 bits, ties to even, the scale in 32."""
    amax = np.abs(x).max(1)
    with np.errstate(invalid="ignore", divide="ignore"):
        s = (amax.astype(np.float32) / np.float32(127)).astype(np.float32)
        s = np.where(np.isfinite(amax), s, np.float32("nan"))
        q = np.rint(x.astype(np.float64) / s.astype(np.float64)[:, None])
    return np.where(np.isfinite(q) & (s > 0)[:, None], np.clip(q, -127, 127), 0).astype(np.int8), s


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("layout", ["plain", "pitch", "odd"])
@pytest.mark.parametrize("rows,k", [(1, 1), (1, 4000), (3, 127), (129, 128), (65, 1972), (300, 64), (7, 9001), (2, 40000), (9000, 3)])
def test_quantize_rows(ops, rows, k, layout, dtype):
    x = matrix(rows, k, dtype, rows + k, layout, scale=3.0)
    q, s = ops.quantize_int8(x)
    rq, rs = quant_ref(x.float().cpu().numpy())
    assert torch.equal(s.cpu(), torch.from_numpy(rs)) and torch.equal(q.cpu(), torch.from_numpy(rq))
    assert q.shape == x.shape and q.stride(0) % 128 == 0
    base = torch.as_strided(q, (rows, q.stride(0)), (q.stride(0), 1))
    assert not base[:, k:].any()


def test_quantize_rows_values(ops):
    """Middles between two integers (ties to even), rows of zeros, of denormal and of huge values, NaN and infinities."""
    k = 254
    rows = [np.arange(-127, 127) / 2 + 0.5, np.zeros(k), np.full(k, 1e-44), np.arange(k) * 1e-43, np.arange(k) * 1e36,
            np.where(np.arange(k) == 3, np.nan, 1.0), np.where(np.arange(k) == 200, -np.inf, 1.0), np.linspace(-1e-36, 1e-36, k),
            np.linspace(-9e-36, 9e-36, k), -np.ones(k)]
    rows[0][0] = 127.0
    # quotients next to a middle, from either side
    s = np.float32(0.1234567)
    near = np.float32((np.arange(k) % 120 + 0.5) * np.float64(s))
    near = np.where(np.arange(k) % 3 == 0, np.nextafter(near, np.float32(0)), np.where(np.arange(k) % 3 == 1, near, np.nextafter(near, np.float32(9e9))))
    near[0] = s * np.float32(127)
    x = np.stack(rows + [near]).astype(np.float32)
    q, sc = ops.quantize_int8(torch.from_numpy(x).cuda())
    rq, rs = quant_ref(x)
    np.testing.assert_array_equal(sc.cpu().numpy(), rs)
    np.testing.assert_array_equal(q.cpu().numpy(), rq)


def i8_check(y, xq, sx, wq, sw, bias):
    acc = torch.zeros(xq.shape[0], wq.shape[0], dtype=torch.float64, device="cuda")
    # products of whole numbers below 2^53: exact in any order
    acc += xq.double().contiguous() @ wq.double().t().contiguous()
    main = acc * sx.double()[:, None] * sw.double()
    ref = main if bias is None else main + bias.double()
    # the sum's conversion, two products and the addition of the bias: one rounding each
    within(y, ref, 4 * U * main.abs() + U * ref.abs() + HALF[y.dtype] * ref.abs() + TINY[y.dtype], "y")


I8_SIZES = [(1, 1, 1), (1, 4096, 4000), (2, 17, 63), (16, 16, 64), (17, 130, 200), (5, 3, 1000), (33, 282, 1972), (64, 64, 128),
            (128, 128, 2000), (130, 257, 129), (255, 31, 4097), (512, 512, 512), (700, 128, 2000), (1025, 1000, 96),
            (300, 1, 777), (4100, 5, 40), (2050, 2100, 320)]


def ints(shape, seed, pad=0, lo=-127):
    return torch.randint(lo, 128, (shape[0], shape[1] + pad), device="cuda", generator=gen(seed), dtype=torch.int8)[:, :shape[1]]


@pytest.mark.parametrize("out", TYPES, ids=str)
@pytest.mark.parametrize("m,n,k", I8_SIZES)
def test_int8_matmul_sizes(ops, m, n, k, out):
    g = gen(m + n + k)
    xq, wq = ints((m, k), 1, -(-k // 128) * 128 - k), ints((n, k), 2)
    sx, sw = (torch.rand(s, device="cuda", generator=g) * 0.01 for s in (m, n))
    bias = torch.randn(n, device="cuda", generator=g)
    for b in (None, bias, bias.to(out)):
        i8_check(ops.int8_matmul(xq, sx, wq, sw, b, out), xq, sx, wq, sw, b)


@pytest.mark.parametrize("m,n,k", [(1, 40, 200), (20, 70, 1001), (200, 130, 260), (515, 300, 1972), (1000, 520, 512)])
@pytest.mark.parametrize("px,pw,ox,ow", [(0, 0, 0, 0), (1, 0, 0, 0), (0, 3, 0, 0), (16, 16, 0, 0), (12, 4, 4, 8), (7, 5, 1, 3)])
def test_int8_matmul_pitches(ops, m, n, k, px, pw, ox, ow):
    """Operands whose rows start anywhere; the bytes around them hold -128, which must not enter a sum."""
    def put(src, pad, off):
        buf = torch.full((src.shape[0] * (src.shape[1] + pad) + 64,), -128, dtype=torch.int8, device="cuda")
        v = torch.as_strided(buf, src.shape, (src.shape[1] + pad, 1), 16 + off)
        v.copy_(src)
        return v
    xq, wq = put(ints((m, k), 5, lo=-128), px, ox), put(ints((n, k), 6, lo=-128), pw, ow)
    sx, sw = (torch.rand(s, device="cuda", generator=gen(7)) * 0.01 for s in (m, n))
    i8_check(ops.int8_matmul(xq, sx, wq, sw), xq, sx, wq, sw, None)


@pytest.mark.parametrize("m,n", [(1, 8), (40, 50), (300, 300)])
def test_int8_matmul_extremes(ops, m, n):
    """The longest rows with the largest products: the int32 sum comes to 2^31 - 16384."""
    from scarches_amd import _lib
    k = _lib.load().sca_gemm_i8_max_k()
    xq, wq = (torch.full((r, k), -128, dtype=torch.int8, device="cuda") for r in (m, n))
    one = lambda r: torch.ones(r, device="cuda")
    y = ops.int8_matmul(xq, one(m), wq, one(n))
    assert (y == float(np.float32(k * 16384.0))).all()
    y = ops.int8_matmul(xq, one(m), -1 - wq, one(n))
    assert (y == float(np.float32(-k * 128.0 * 127.0))).all()


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("m,n,k", [(1, 300, 500), (77, 128, 1972), (513, 64, 2000), (6, 5, 4)])
def test_int8_linear(ops, m, n, k, dtype):
    x = torch.relu(matrix(m, k, dtype, 3, "pitch"))
    x[0] = 0
    wq, sw = ops.quantize_int8(torch.randn(n, k, device="cuda", generator=gen(4)))
    bias = torch.randn(n, device="cuda", generator=gen(5)).to(dtype)
    y = ops.int8_linear(x, wq, sw, bias)
    q, s = ops.quantize_int8(x)
    assert y.dtype == dtype and torch.equal(y, ops.int8_matmul(q, s, wq, sw, bias, dtype))
    assert torch.equal(y[0], bias)
    i8_check(y, q, s, wq, sw, bias)
    y3 = ops.int8_linear(x.expand(2, m, k), wq, sw, None, torch.float32)
    assert y3.shape == (2, m, n) and torch.equal(y3[0], y3[1])
    bad = x.clone()
    bad[-1, 1] = float("nan")
    yb = ops.int8_linear(bad, wq, sw, bias)
    assert torch.isnan(yb[-1]).all() and torch.equal(yb[:-1], y[:-1])
    assert ops.int8_linear(x[:0], wq, sw, bias).shape == (0, n)
    assert ops.int8_linear(x, wq[:0], sw[:0]).shape == (m, 0)


def test_int8_results_stay_inside_their_rows(ops):
    from scarches_amd import _lib
    lib = _lib.load()
    for m, n, k in ((3, 21, 100), (70, 130, 256), (600, 300, 400)):
        xq, wq = ints((m, k), 1), ints((n, k), 2)
        sx, sw = torch.ones(m, device="cuda"), torch.ones(n, device="cuda")
        out = torch.full((m + 2, n + 8), 7.0, device="cuda")
        _lib.check(lib.sca_gemm_i8(xq.data_ptr(), k, sx.data_ptr(), wq.data_ptr(), k, sw.data_ptr(), None, 0, m, n, k,
                                   out[1, 3:].data_ptr(), 0, n + 8, torch.cuda.current_stream().cuda_stream), "i8")
        assert torch.equal(out[1:-1, 3:3 + n], ops.int8_matmul(xq, sx, wq, sw))
        out[1:-1, 3:3 + n] = 7.0
        assert (out == 7.0).all()


def test_int8_offsets_past_32_bits(ops):
    k = 4096
    m = (1 << 31) // k + 70
    xq = torch.zeros(m, k, dtype=torch.int8, device="cuda")
    tail = ints((100, k), 1)
    xq[-100:] = tail
    wq, sw, sx = ints((24, k), 2), torch.ones(24, device="cuda"), torch.ones(m, device="cuda")
    y = ops.int8_matmul(xq, sx, wq, sw)
    assert torch.equal(y[-100:], ops.int8_matmul(tail, sx[:100], wq, sw)) and not y[:-100].any()
    del xq
    x = torch.zeros((1 << 31) // 1024 + 5, 1024, dtype=torch.bfloat16, device="cuda")
    x[-1] = torch.randn(1024, device="cuda", generator=gen(3))
    q, s = ops.quantize_int8(x)
    tq, ts = ops.quantize_int8(x[-1:])
    assert torch.equal(q[-1:], tq) and torch.equal(s[-1:], ts) and not s[:-1].any()


def test_more_rows_than_a_grid_holds(ops):
    """70 million short rows: 2^32 threads are not enough to give each its own."""
    rows = 70_000_000
    x = torch.arange(rows, device="cuda", dtype=torch.float32)[:, None] * torch.tensor([1.0, -0.5, 0.25], device="cuda")
    q, s = ops.quantize_int8(x)
    # (-0.5 and 0.25 of the largest value are -63.5 and 31.75 scales up to the scale's rounding: which integer -63.5 goes to
    # depends on it, so the reference is the quotient in 64 bits)
    same = bool((s == x[:, 0] / torch.full_like(s, 127)).all())
    ref = torch.round(x[1:].double() / s[1:, None].double())
    same = same and bool((q[1:] == ref).all()) and not bool(q[0].any())
    assert same
    del q, s, ref
    y, stats = ops.layer_norm_fwd(x)
    at = torch.tensor([0, 1, 5, 67_108_863, 67_108_864, rows - 1], device="cuda")
    want, _ = ops.layer_norm_fwd(x[at])
    assert torch.equal(y[at], want) and torch.equal(stats[0, at], ops.layer_norm_fwd(x[at])[1][0])
    assert (y[2:, 0] > 1).all()
    dx, _, _ = ops.layer_norm_bwd(y, x, None, stats)
    assert torch.equal(dx[at], ops.layer_norm_bwd(want, x[at], None, stats[:, at].contiguous())[0])


# ---------------------------------------------------------------------------------------------- AdamW
LR, B1, B2, EPS, WD = 3e-3, 0.9, 0.999, 1e-8, 0.05


def tensors(sizes, dtype, seed):
    g = gen(seed)
    p = [torch.randn(s, device="cuda", generator=g).to(dtype) for s in sizes]
    for t in p:
        t.grad = (torch.randn(t.shape, device="cuda", generator=g) * 0.01).to(dtype)
    return p


def check_update(p, p0, m0, g, m, v, t, lr=LR, wd=WD, eps=EPS):
    """The parameter after a step whose new moments (64 bits, unrounded) are m, v."""
    denom = (v / (1 - B2 ** t)).sqrt() + eps
    upd = lr / (1 - B1 ** t) * m / denom
    ref = p0 * (1 - lr * wd) - upd
    # m: b1 m0 and (1 - b1) g may cancel, three roundings each; then root, quotient, sums: a dozen
    dm = 3 * U * (B1 * m0.abs() + (1 - B1) * g.abs())
    bound = 3 * U * p0.abs() + 12 * U * upd.abs() + lr / (1 - B1 ** t) * dm / denom + HALF[p.dtype] * ref.abs() + TINY[p.dtype]
    within(p, ref, bound, "p")


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("sizes", [[(1,)], [(5,), (2048,), (0,), (2049,), (3, 1)], [(64, 33), (4095,), (128, 2000), (7, 7, 7)],
                                   [(10,)] * 300], ids=["one", "edges", "network", "many"])
def test_adamw_32_bits(ops, sizes, dtype):
    p = tensors(sizes, dtype, 1)
    opt = ops.AdamW(p, lr=LR, betas=(B1, B2), eps=EPS, weight_decay=WD)
    for t in range(1, 4):
        before = [(x.double(), {k: s.double() for k, s in opt.state[x].items()} if opt.state[x] else None) for x in p]
        for x in p:
            x.grad.mul_(-1.5)
        opt.step()
        for x, (p0, st) in zip(p, before):
            g = x.grad.double()
            m0, v0 = (st["exp_avg"], st["exp_avg_sq"]) if st else (0 * g, 0 * g)
            m, v = B1 * m0 + (1 - B1) * g, B2 * v0 + (1 - B2) * g * g
            within(opt.state[x]["exp_avg"], m, 3 * U * (B1 * m0.abs() + (1 - B1) * g.abs()), "m")
            within(opt.state[x]["exp_avg_sq"], v, 5 * U * v + 1e-44, "v")
            check_update(x, p0, m0, g, m, v, t)


def test_adamw_matches_torch_over_steps(ops):
    """Twenty steps beside torch.optim.AdamW in 64 bits: two groups, a parameter without a gradient now and then (its step
    number stands still), a changed learning rate and decay."""
    a = tensors([(40, 50), (77,), (300,)], torch.float32, 2)
    b = [x.double() for x in a]
    opts = [c([dict(params=q[:2]), dict(params=q[2:], lr=0.01, weight_decay=0.3)], lr=1e-3)
            for c, q in ((ops.AdamW, a), (torch.optim.AdamW, b))]
    for i in range(20):
        for x, y in zip(a, b):
            x.grad = torch.randn(x.shape, device="cuda", generator=gen(100 + i))
            y.grad = x.grad.double()
        if i % 3 == 1:
            a[1].grad = b[1].grad = None
        if i == 10:
            for o in opts:
                o.param_groups[0]["lr"], o.param_groups[1]["weight_decay"] = 5e-4, 0.1
        for o in opts:
            o.step()
    for x, y in zip(a, b):
        # 20 steps of at most 0.01, each off by at most 20 roundings of the value and the step
        within(x, y, 20 * 20 * U * (y.abs() + 0.01), "p")
    sd = opts[0].state_dict()
    assert [sd["state"][i]["step"] for i in range(3)] == [20, 13, 20]


def philox_words(n, tensor, t, seed):
    u = np.uint64
    m32 = u(0xFFFFFFFF)
    i = np.arange(-(-n // 4), dtype=u)
    c = [i & m32, i >> u(32), np.full_like(i, tensor), np.full_like(i, t)]
    k = [u(seed & 0xFFFFFFFF), u(seed >> 32)]
    for _ in range(10):
        a, b = c[0] * u(0xD2511F53), c[2] * u(0xCD9E8D57)
        c = [(b >> u(32)) ^ c[1] ^ k[0], b & m32, (a >> u(32)) ^ c[3] ^ k[1], a & m32]
        k = [(k[0] + u(0x9E3779B9)) & m32, (k[1] + u(0xBB67AE85)) & m32]
    return np.stack(c, 1).reshape(-1)[:n].astype(np.int64)


def grid_ref(x, rnd, kind):
    """What 8 bits hold of x: (bytes, scales), by a search in the type's values."""
    every = torch.arange(128, dtype=torch.uint8).view(kind).double().numpy()
    every = every[np.isfinite(every)]
    blocks = lambda a: np.pad(a, (0, -len(a) % 256)).reshape(-1, 256)
    x, rnd = blocks(x.astype(np.float64)), blocks(rnd)
    amax = np.abs(x).max(1) if len(x) else np.zeros(0)
    fine = np.isfinite(amax)
    with np.errstate(divide="ignore", invalid="ignore"):
        scale = np.where(amax > 0, 2.0 ** np.maximum(np.ceil(np.log2(amax / every[-1])), -126), 0)
        t = np.where((fine & (amax > 0))[:, None], np.abs(x) / scale[:, None], 0)
    low = np.searchsorted(every, t, "right") - 1
    up = np.minimum(low + 1, len(every) - 1)
    code = np.where((t - every[low]) / np.where(up > low, every[up] - every[low], 1) >= 1 - rnd / 65536, up, low)
    if kind == torch.float8_e5m2:
        code = np.where((x > 0) & (code == 0) & fine[:, None], 1, code)
    code = np.where((x < 0) & (code > 0), code + 128, code)
    return code.reshape(-1).astype(np.uint8), np.where(fine, scale, np.nan).astype(np.float32)


def check_8_bit_step(ops, opt, params, t, seed):
    before = [(x.double().cpu(), {k: s.clone() for k, s in opt.state[x].items()}) for x in params]
    opt.step()
    for j, (x, (p0, st)) in enumerate(zip(params, before)):
        n = x.numel()
        each = lambda k: st[k].float().reshape(-1).double().cpu() * st[k + "_scale"].double().cpu().repeat_interleave(256)[:n]
        g = x.grad.double().reshape(-1).cpu()
        m0, v0 = each("exp_avg"), each("exp_avg_sq")
        m, v = B1 * m0 + (1 - B1) * g, B2 * v0 + (1 - B2) * g * g
        word = philox_words(n, j, t, seed)
        now = opt.state[x]
        for k, val, rnd, kind in (("exp_avg", m, word & 0xFFFF, torch.float8_e4m3fn), ("exp_avg_sq", v, word >> 16, torch.float8_e5m2)):
            code, scale = grid_ref(val.float().numpy(), rnd, kind)
            assert now[k].dtype == kind and now[k].shape == x.shape
            np.testing.assert_array_equal(now[k + "_scale"].cpu().numpy(), scale)
            np.testing.assert_array_equal(now[k].view(torch.uint8).reshape(-1).cpu().numpy(), code[:n])
        ok = torch.isfinite(m) & torch.isfinite(v)
        sel = lambda a: a.reshape(-1).cpu()[ok]
        check_update(sel(x), sel(p0), m0[ok], g[ok], m[ok], v[ok], t)
        assert not torch.isfinite(x.reshape(-1).cpu()[~ok]).any()


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("sizes", [[(1,)], [(5,), (256,), (0,), (257,), (2048,), (2305,), (3, 1)], [(64, 33), (128, 300), (7, 7, 7)]],
                         ids=["one", "edges", "network"])
def test_adamw_8_bits(ops, sizes, dtype):
    """Every byte and every scale against an independent search in the types' values, over several steps."""
    p = tensors(sizes, dtype, 3)
    seed = 0x123456789ABCD
    opt = ops.AdamW(p, lr=LR, betas=(B1, B2), eps=EPS, weight_decay=WD, state_bits=8, seed=seed)
    for x in p:
        opt._init_state(x)
    for t in range(1, 5):
        for i, x in enumerate(p):
            x.grad = (torch.randn(x.shape, device="cuda", generator=gen(50 * t + i))
                      * torch.exp(3 * torch.randn(x.shape, device="cuda", generator=gen(50 * t + i + 25)) - 4)).to(dtype)
        check_8_bit_step(ops, opt, p, t, seed)


def test_adamw_8_bits_values(ops):
    """Blocks of zeros, of denormal, tiny and huge gradients, and with values that are not finite (their block only)."""
    x = torch.randn(8 * 256 + 100, device="cuda", generator=gen(1))
    x.grad = torch.randn(x.shape, device="cuda", generator=gen(2))
    x.grad[:256] = 0
    x.grad[256:512] *= 1e-42
    x.grad[512:768] *= 1e-30
    x.grad[768:1024] *= 1e17
    x.grad[1030] = float("nan")
    x.grad[1300] = -float("inf")
    x.grad[1600:1700] = 0
    x.grad[-1] = float("inf")
    opt = ops.AdamW([x], lr=LR, betas=(B1, B2), eps=EPS, weight_decay=WD, state_bits=8, seed=5)
    opt._init_state(x)
    for t in (1, 2, 3):
        check_8_bit_step(ops, opt, [x], t, 5)
    bad = torch.isnan(opt.state[x]["exp_avg_scale"]).cpu().tolist()
    assert bad == [False, False, False, False, True, True, False, False, True]
    keep = torch.isfinite(x).reshape(-1)
    assert keep[:1024].all() and keep[1536:2048].all() and not keep[2048:].any()


def test_adamw_8_bits_keeps_the_mean(ops):
    """Stochastic rounding is unbiased: 65536 equal moments between two grid values average to the exact one."""
    n = 1 << 16
    x = torch.zeros(n, device="cuda")
    x.grad = torch.full((n,), 0.3, device="cuda")
    x.grad[::256] = 1.0         # the largest of each block sets the scale
    opt = ops.AdamW([x], lr=0.0, betas=(B1, B2), weight_decay=0.0, state_bits=8, seed=1)
    opt.step()
    st = opt.state[x]
    some = torch.arange(n, device="cuda") % 256 != 0
    for k, want, step in (("exp_avg", 0.1 * 0.3, 1 / 8), ("exp_avg_sq", 0.001 * 0.09, 1 / 4)):
        val = st[k].float() * st[k + "_scale"].repeat_interleave(256)
        # a value lies within one grid step (a share `step` of it at most); standard error of the mean step / 2 / 255, taken 6 times
        assert abs(val[some].double().mean().item() / want - 1) <= 6 * step / 2 / 255
        assert len(val[some].unique()) == 2


@pytest.mark.parametrize("bits", [32, 8])
def test_adamw_layouts_and_alignment(ops, bits):
    """Views that start at odd elements and transposed parameters take the same step as their contiguous copies."""
    base = torch.randn(5000, device="cuda", generator=gen(1))
    for dtype in TYPES:
        odd = base.to(dtype)[1:3001]
        odd.grad = (base.flip(0) * 0.1).to(dtype)[3:3003]
        turned = base.to(dtype)[:2000].clone().view(40, 50).t()
        turned.grad = (base * 0.2).to(dtype)[:2000].clone().view(40, 50).t()
        plain = [odd.detach().clone(), turned.t().detach().clone()]
        plain[0].grad, plain[1].grad = odd.grad.clone(), turned.grad.t().clone()
        mixed, ref = (ops.AdamW(q, lr=LR, state_bits=bits, seed=3) for q in ([odd, turned], plain))
        for _ in range(3):
            mixed.step()
            ref.step()
        assert torch.equal(odd, plain[0]) and torch.equal(turned.t(), plain[1])
        for x, y in zip((odd, turned), plain):
            for k in ref.state[y]:
                s, r = mixed.state[x][k].float().cpu(), ref.state[y][k].float().cpu()
                assert torch.equal(s.t() if x is turned and s.dim() == 2 else s, r), k


@pytest.mark.parametrize("bits", [32, 8])
def test_adamw_state_dict(ops, bits):
    """Save, load into a new optimizer and go on: the same bits as without the break (float8 and scales keep their types)."""
    import io
    p = tensors([(300, 7), (1000,)], torch.bfloat16, 6)
    q = [x.detach().clone() for x in p]
    a = ops.AdamW(p, lr=LR, state_bits=bits, seed=9)
    for _ in range(3):
        a.step()
    for x, y in zip(p, q):
        y.copy_(x)
        y.grad = x.grad.clone()
    buf = io.BytesIO()
    torch.save(a.state_dict(), buf)
    buf.seek(0)
    sd = torch.load(buf, weights_only=True)
    assert sd["state"][0]["step"] == 3
    b = ops.AdamW(q, lr=1.0, state_bits=bits, seed=9)
    b.load_state_dict(sd)
    assert b.param_groups[0]["lr"] == LR
    for _ in range(2):
        a.step()
        b.step()
    for x, y in zip(p, q):
        assert torch.equal(x, y)
        for k, v in a.state[x].items():
            assert v.dtype == b.state[y][k].dtype and torch.equal(v.float(), b.state[y][k].float()), k
    with pytest.raises(ValueError, match="-bit states"):
        ops.AdamW(q, state_bits=40 - bits).load_state_dict(sd)


@pytest.mark.parametrize("bits", [32, 8])
def test_adamw_under_graph_capture(ops, bits):
    """A captured step counts on when it is replayed; eager work and synchronizations between the replays."""
    p = tensors([(500, 9), (33,), (4000,)], torch.float32, 8)
    q = [x.detach().clone() for x in p]
    grads = [torch.zeros_like(x) for x in q]
    for x, y, g in zip(p, q, grads):
        x.grad = torch.zeros_like(x)
        y.grad = g
    a, b = ops.AdamW(p, lr=LR, state_bits=bits, seed=2), ops.AdamW(q, lr=LR, state_bits=bits, seed=2)
    a.step()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        b.step()
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        b.step()
    for i in range(6):
        for x, g in zip(p, grads):
            x.grad = torch.randn(x.shape, device="cuda", generator=gen(i))
            g.copy_(x.grad)
        a.step()
        graph.replay()
        if i % 2:
            torch.cuda.synchronize()
        for x, y in zip(p, q):
            assert torch.equal(x, y), i
    assert b.state_dict()["state"][0]["step"] == 7
    new = torch.zeros_like(grads[0])
    q[0].grad = new
    other = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="before the capture"):
        with torch.cuda.graph(other):
            grads[0].zero_()                    # (never replayed; no graph here is left without a node)
            b.step()


def test_adamw_is_a_torch_optimizer(ops):
    """Step hooks run once per step, schedulers change the rate, a closure is called and its value returned, parameters may
    join later."""
    p = tensors([(20,), (30,)], torch.float32, 4)
    q = [x.clone() for x in p]
    opt = ops.AdamW(p[:1], lr=0.1, weight_decay=0.0)
    calls = []
    opt.step()
    opt.register_step_pre_hook(lambda o, a, k: calls.append("pre"))
    handle = opt.register_step_post_hook(lambda o, a, k: calls.append("post"))
    assert opt.step(lambda: 3.5) == 3.5 and calls == ["pre", "post"]
    handle.remove()
    sched = torch.optim.lr_scheduler.StepLR(opt, 1, 0.5)
    opt.add_param_group(dict(params=p[1:], lr=0.2))
    opt.step()
    sched.step()
    assert opt.param_groups[0]["lr"] == 0.05
    opt.step()
    ref = torch.optim.AdamW([x.double() for x in q[:1]], lr=0.1, weight_decay=0.0)
    y = ref.param_groups[0]["params"][0]
    y.grad = p[0].grad.double()
    for lr in (0.1, 0.1, 0.1, 0.05):
        ref.param_groups[0]["lr"] = lr
        ref.step()
    within(p[0], y, 4 * 20 * U * (y.abs() + 0.1), "p")
    assert [v["step"] for v in opt.state_dict()["state"].values()] == [4, 2]
    with torch.profiler.profile(activities=[torch.profiler.ProfilerActivity.CPU]) as prof:
        opt.step()
    assert any("AdamW.step" in e.key for e in prof.key_averages())


def test_adamw_offsets_past_32_bits(ops):
    n = (1 << 31) + 1111
    x = torch.full((n,), 0.5, device="cuda", dtype=torch.bfloat16)
    x.grad = torch.full((n,), 0.25, device="cuda", dtype=torch.bfloat16)
    y = torch.full((1111,), 0.5, device="cuda", dtype=torch.bfloat16)
    y.grad = torch.full((1111,), 0.25, device="cuda", dtype=torch.bfloat16)
    for bits in (32, 8):
        a, b = ops.AdamW([x], lr=0.1, state_bits=bits), ops.AdamW([y], lr=0.1, state_bits=bits)
        a.step()
        b.step()
        assert torch.equal(x[-1111:], y) and torch.equal(x[:1111], y)
        if bits == 8:
            assert torch.equal(a.state[x]["exp_avg_scale"][-5:], b.state[y]["exp_avg_scale"])
            w = philox_words(4, 0, 1, 0)
            assert a.state[x]["exp_avg"][-1].float() > 0 and len(w) == 4
        else:
            assert torch.equal(a.state[x]["exp_avg_sq"][-1111:], b.state[y]["exp_avg_sq"])
        del a, b


# ---------------------------------------------------------------------------------------------- together
def test_streams_and_graphs(ops):
    """The three kinds on a stream of their own, two streams at once, and captured into one graph that is replayed."""
    x, w = matrix(400, 300, torch.float32, 1), torch.ones(300, device="cuda")
    wq, ws = ops.quantize_int8(torch.randn(64, 300, device="cuda", generator=gen(2)))

    def work(inp):
        y, stats = ops.layer_norm_fwd(inp, w, w)
        return (y, *ops.layer_norm_bwd(inp, inp, w, stats), ops.int8_linear(y, wq, ws))

    want = work(x)
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    for _ in range(5):
        for s in streams:
            with torch.cuda.stream(s):
                got.append(work(x))
    torch.cuda.synchronize()
    for res in got:
        assert all(torch.equal(a, b) for a, b in zip(res, want))
    static = x.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = work(static)
    for i in range(4):
        static.copy_(x * (i + 1) + i)
        graph.replay()
        if i == 2:
            torch.cuda.synchronize()
        now = work(static)
        assert all(torch.equal(a, b) for a, b in zip(held, now)), i


@pytest.mark.parametrize("bits", [32, 8])
def test_train_a_normalised_block_and_serve_it(ops, bits):
    """Linear -> layer norm -> ReLU -> Linear: gradients through ops.layer_norm, steps of ops.AdamW beside the same network in
    64 bits with torch's AdamW, then the trained weights served in 8-bit integers."""
    g = gen(21)
    shapes = [(96, 200), (96,), (96,), (96,), (17, 96), (17,)]
    init = [torch.randn(s, device="cuda", generator=g) * (0.08 if len(s) == 2 else 0.1) for s in shapes]
    init[2] += 1
    x = torch.log1p(torch.poisson(torch.rand(64, 200, device="cuda", generator=g) * 2, generator=g))
    t = torch.randn(64, 17, device="cuda", generator=g)

    def net(p, x, norm):
        h = torch.relu(norm(torch.nn.functional.linear(x, p[0], p[1]), p[2], p[3]))
        return torch.nn.functional.linear(h, p[4], p[5])

    def train(dt, norm, opt_of):
        p = [i.to(dt).clone().requires_grad_() for i in init]
        opt, grads = opt_of(p), None
        for k in range(5):
            opt.zero_grad()
            (net(p, x.to(dt), norm) - t.to(dt)).square().mean().backward()
            grads = grads or [q.grad.clone() for q in p]
            opt.step()
        return p, grads, opt

    p, grads, opt = train(torch.float32, ops.layer_norm, lambda q: ops.AdamW(q, lr=1e-3, state_bits=bits))
    r, ref, _ = train(torch.float64, lambda v, w, b: torch.nn.functional.layer_norm(v, (96,), w, b),
                      lambda q: torch.optim.AdamW(q, lr=1e-3))
    for a, b in zip(grads, ref):        # sums of at most 64 * 17 + 200 terms of the gradient's size
        assert (a.double() - b).abs().max() <= 1300 * U * b.abs().max() * 8
    for a, b, i in zip(p, r, init):
        # no step moves a value by more than lr (1 + a little): m^2 <= v at t = 1, and |m| / sqrt(v) <= sqrt(10) later
        assert (a.double() - i.double()).abs().max() <= 5 * 1e-3 * 3.2
        if bits == 32:                  # elements whose gradient is of rounding size may go either way
            assert (a.double() - b).abs().median() <= 1e-5
    with torch.no_grad():
        wq0, ws0 = ops.quantize_int8(p[0])
        wq1, ws1 = ops.quantize_int8(p[4])
        a = ops.int8_linear(x, wq0, ws0, p[1])
        h = torch.relu(ops.layer_norm(a, p[2], p[3]))
        y = ops.int8_linear(h, wq1, ws1, p[5])
    for got, v, w, b, wq, ws in ((a, x, p[0], p[1], wq0, ws0), (y, h, p[4], p[5], wq1, ws1)):
        v, w, b, ws = v.double(), w.detach().double(), b.detach().double(), ws.double()
        sv = v.abs().amax(1, keepdim=True) / 127
        # x w - x^ w^ = x (w - w^) + (x - x^) w^: half a step of either factor's scale; then the product's roundings
        off = 0.5001 * (v.abs().sum(1, keepdim=True) * ws + sv * (wq.double().abs().sum(1) * ws))
        size = v.abs() @ w.abs().t().contiguous()
        within(got, v @ w.t().contiguous() + b, off + 8 * U * (size + off + b.abs()), "served")
