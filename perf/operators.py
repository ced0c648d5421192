"""Workloads of the operators that stand around the conditional networks' dense layers: layer norm with weight and bias
(forward, backward), AdamW over a network's whole parameter list (32-bit and 8-bit states) and the product in 8-bit
integers with a scale per cell and per output channel.

`run` computes them in plain torch operations, or (`own = True`) through scarches_amd.ops."""
import math

import numpy as np
import torch

own = False

DEV = "cuda"
TYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}
LR, BETA1, BETA2, EPS, DECAY = 1e-3, 0.9, 0.999, 1e-8, 0.01
BLOCK = 256             # elements of a tensor that share one scale of the 8-bit states
M32 = 0xFFFFFFFF


def listed():
    return [
        # one default minibatch (128 cells) through a 128-wide hidden layer: latency
        dict(name="ln_fwd_minibatch", op="ln_fwd", rows=128, n=128, dtype="float32", affine=True, pad=0),
        # a 16384-cell block over 4000 genes in 16 bits: bandwidth
        dict(name="ln_fwd_genes_bf16", op="ln_fwd", rows=16384, n=4000, dtype="bfloat16", affine=True, pad=0),
        # backward over the 2000 genes of a large minibatch
        dict(name="ln_bwd_genes", op="ln_bwd", rows=8192, n=2000, dtype="float32", affine=True, pad=0),
        # odd sizes, rows with a pitch: a slice of a wider fp16 matrix
        dict(name="ln_bwd_odd_fp16", op="ln_bwd", rows=1021, n=1001, dtype="float16", affine=True, pad=7),
        # the parameters of the default-size network: 2000 genes, hidden [128, 128], 5 conditions (12 tensors, 6e5 values)
        dict(name="adamw32_network", op="adamw", bits=32, genes=2000, h1=128, h2=128, latent=10, conds=5, dtype="float32"),
        # a full-transcriptome network with wide layers
        dict(name="adamw32_wide", op="adamw", bits=32, genes=20000, h1=4096, h2=1024, latent=64, conds=20, dtype="float32"),
        # the same two with 8-bit states, the wide one with 16-bit parameters
        dict(name="adamw8_network", op="adamw", bits=8, genes=2000, h1=128, h2=128, latent=10, conds=5, dtype="float32"),
        dict(name="adamw8_wide_bf16", op="adamw", bits=8, genes=20000, h1=2048, h2=1024, latent=64, conds=20,
             dtype="bfloat16"),
        # one cell through a wide layer (a request that is answered by itself): the weight's bytes
        dict(name="int8_one_cell", op="int8", rows=1, n=4096, k=4000, dtype="float32", bias=True),
        # first encoder layer of the mapping of query cells: 8192 cells, 2000 genes -> 128
        dict(name="int8_map_cells", op="int8", rows=8192, n=128, k=2000, dtype="float32", bias=True),
        # odd sizes: 1972 genes, a part of a block of cells, 282 gene programs
        dict(name="int8_odd", op="int8", rows=509, n=282, k=1972, dtype="bfloat16", bias=False),
        # wide hidden layer: matrix-core rate
        dict(name="int8_wide_bf16", op="int8", rows=8192, n=4096, k=4096, dtype="bfloat16", bias=True),
    ]


def _spread(rng, lo, hi):
    """A whole number in [lo, hi], even over its logarithm."""
    return int(min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["ln_fwd", "ln_bwd", "adamw", "adamw", "int8", "int8"])
    dtype = rng.choice(list(TYPES))
    if op in ("ln_fwd", "ln_bwd"):
        n = _spread(rng, 1, 16384)
        rows = _spread(rng, 1, min(65536, 32_000_000 // n))
        return dict(op=op, rows=rows, n=n, dtype=dtype, affine=rng.random() < 0.8, pad=rng.choice([0, 0, 3, 8]))
    if op == "adamw":
        return dict(op=op, bits=rng.choice([32, 8]), genes=_spread(rng, 100, 20000), h1=_spread(rng, 16, 2048),
                    h2=_spread(rng, 16, 1024), latent=_spread(rng, 2, 64), conds=_spread(rng, 1, 20), dtype=dtype)
    k = _spread(rng, 16, 8192)
    n = _spread(rng, 1, 8192)
    rows = _spread(rng, 1, max(1, min(65536, 8192 * 4096 * 4096 // (k * n), 60_000_000 // max(k, n))))
    return dict(op=op, rows=rows, n=n, k=k, dtype=dtype, bias=rng.random() < 0.5)


def shapes_of(case):
    """The parameter tensors of a conditional network: dispersions, two encoder layers, the two heads in one matrix, two
    decoder layers, the output layer."""
    g, h1, h2, z, c = (case[k] for k in ("genes", "h1", "h2", "latent", "conds"))
    return [(g, c), (h1, g), (h1,), (h1, c), (h2, h1), (h2,), (2 * z, h2), (2 * z,), (h2, z), (h1, h2), (g, h1), (g,)]


def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(int(seed))
    dt = TYPES[case["dtype"]]

    def normal(*shape):
        return torch.randn(*shape, device=DEV, generator=gen)

    if case["op"] in ("ln_fwd", "ln_bwd"):
        rows, n = case["rows"], case["n"]
        pitch = n + case["pad"]
        # pre-activations: every row has an offset and a spread of its own
        x = (normal(rows, pitch) * (0.5 + torch.rand(rows, 1, device=DEV, generator=gen)) + normal(rows, 1)).to(dt)[:, :n]
        s = dict(case=case, x=x, w=None, b=None, eps=1e-5)
        if case["affine"]:
            s["w"], s["b"] = (1 + 0.1 * normal(n)).to(dt), (0.1 * normal(n)).to(dt)
        if case["op"] == "ln_bwd":
            s["dy"] = normal(rows, pitch).to(dt)[:, :n]
            xf = x.float()
            mu = xf.mean(1)
            s["stats"] = torch.stack([mu, ((xf - mu[:, None]).square().mean(1) + 1e-5).rsqrt()])
        return s
    if case["op"] == "adamw":
        p, g, states = [], [], []
        for shape in shapes_of(case):
            fan = shape[-1] if len(shape) > 1 else 16
            p.append((normal(*shape) / math.sqrt(fan)).to(dt))
            # gradients of very different sizes, as rare and common genes give them
            size = torch.exp(2 * normal(*shape[:-1], 1) - 6) if len(shape) > 1 else torch.exp(normal(1) - 6)
            g.append((normal(*shape) * size).to(dt))
            gf = g[-1].float()
            m, v = gf * (0.3 + 0.3 * normal(*shape)), gf.square() * (0.5 + torch.rand(*shape, device=DEV, generator=gen))
            if case["bits"] == 32:
                states.append(dict(exp_avg=m, exp_avg_sq=v))
                continue
            nb = -(-m.numel() // BLOCK)

            def held(t, to, top):
                t = torch.nn.functional.pad(t.reshape(-1), (0, nb * BLOCK - t.numel())).view(nb, BLOCK)
                scale = torch.exp2(torch.ceil(torch.log2(t.abs().amax(1).clamp_min(1e-30) / top)))
                return (t / scale[:, None]).to(to).view(-1)[:m.numel()].view(shape), scale

            mq, ms = held(m, torch.float8_e4m3fn, 448.0)
            vq, vs = held(v, torch.float8_e5m2, 57344.0)
            states.append(dict(exp_avg=mq, exp_avg_scale=ms, exp_avg_sq=vq, exp_avg_sq_scale=vs))
        # of every block of 256: its number in its tensor, and the tensor's
        count = torch.tensor([-(-x.numel() // BLOCK) for x in p], device=DEV)
        tensor = torch.repeat_interleave(torch.arange(len(p), device=DEV), count)
        block = torch.arange(len(tensor), device=DEV) - (count.cumsum(0) - count)[tensor]
        return dict(case=case, p=p, g=g, states=states, step=100, seed=int(seed) & 0xFFFF, blocks=(block, tensor))
    rows, n, k = case["rows"], case["n"], case["k"]
    # log1p of counts whose rates differ from gene to gene and from cell to cell
    rate = torch.exp(1.5 * normal(1, k) - 1.5) * torch.exp(0.3 * normal(rows, 1))
    x = torch.log1p(torch.poisson(rate, generator=gen)).to(dt)
    w = normal(n, k) / math.sqrt(k)
    ws = w.abs().amax(1) / 127
    wq = torch.round(w / ws[:, None]).clamp_(-127, 127).to(torch.int8)
    return dict(case=case, x=x, wq=wq, ws=ws, bias=(0.1 * normal(n)).to(dt) if case["bias"] else None)


# ------------------------------------------------------------------------------------------------ plain forms
def _ln_fwd(s):
    x = s["x"].float()
    mu = x.mean(1)
    d = x - mu[:, None]
    r = torch.rsqrt(d.square().mean(1) + s["eps"])
    y = d * r[:, None]
    if s["w"] is not None:
        y = y * s["w"].float() + s["b"].float()
    return dict(y=y.to(s["x"].dtype), stats=torch.stack([mu, r]))


def _ln_bwd(s):
    dt = s["x"].dtype
    dy, r = s["dy"].float(), s["stats"][1][:, None]
    h = (s["x"].float() - s["stats"][0][:, None]) * r
    a = dy * s["w"].float() if s["w"] is not None else dy
    dx = r * (a - a.mean(1, keepdim=True) - h * (a * h).mean(1, keepdim=True))
    out = dict(dx=dx.to(dt))
    if s["w"] is not None:
        out |= dict(dw=(dy * h).sum(0).to(dt), db=dy.sum(0).to(dt))
    return out


def _update(p, m, v, t):
    denom = v.sqrt() / math.sqrt(1 - BETA2 ** t) + EPS
    return p * (1 - LR * DECAY) - (LR / (1 - BETA1 ** t)) * (m / denom)


def _philox(block, tensor, t, seed):
    """[nb, BLOCK] random 32-bit words (as int64) of the blocks number `block` of the tensors number `tensor`:
    Philox4x32-10 at counter (i >> 2, tensor, t), word i & 3 for element i of a tensor."""
    i = block[:, None] * (BLOCK // 4) + torch.arange(BLOCK // 4, device=block.device)
    c0, c1, c2, c3 = i & M32, i >> 32, tensor[:, None].expand_as(i), torch.full_like(i, t & M32)
    k0, k1 = seed & M32, (seed >> 32) & M32
    for _ in range(10):
        a, b = c0 * 0xD2511F53, c2 * 0xCD9E8D57
        c0, c1, c2, c3 = ((b >> 32) & M32) ^ c1 ^ k0, b & M32, ((a >> 32) & M32) ^ c3 ^ k1, a & M32
        k0, k1 = (k0 + 0x9E3779B9) & M32, (k1 + 0xBB67AE85) & M32
    return torch.stack([c0, c1, c2, c3], 2).view(-1, BLOCK)


def _held8(x32, random16, mant, bias, least):
    """x32 [nb, BLOCK] on the grid of an 8-bit float with `mant` fraction bits and exponent bias `bias`, behind a power of
    two per block; rounded up where the discarded part exceeds the random number.  (codes, scales)"""
    top = 8 if mant == 3 else 15                            # exponent of the largest value, 1.75 * 2^top
    amax = x32.abs().amax(1)
    abits = amax.view(torch.int32)
    e = ((abits >> 23) - 127 - top + ((abits & 0x7FFFFF) > 0x600000)).clamp_min(-126)
    bad, none = ~torch.isfinite(amax), amax == 0
    e = torch.where(bad | none, 0, e)
    scale = ((e + 127) << 23).view(torch.float32)           # 2^e, and 2^-e below
    t = x32.abs() * ((127 - e) << 23).view(torch.float32)[:, None]
    small = (t * 2.0 ** (bias - 1 + mant + 16)).clamp_max(2.0 ** 30).to(torch.int32) + random16 >> 16
    drop = 23 - mant
    code = torch.where(t < 2.0 ** (1 - bias), small,
                       (t.view(torch.int32) + (random16 << (drop - 16)) >> drop) - ((127 - bias) << mant))
    if least:
        code = torch.where((x32 > 0) & (code == 0), 1, code)
    code = code | ((x32 < 0) & (code > 0)).int() * 128
    code = torch.where((bad | none)[:, None], 0, code)
    return code.to(torch.uint8), torch.where(bad, math.nan, torch.where(none, 0.0, scale))


def _blocks(tensors, to):
    """All tensors behind one another, each filled up with zeros to whole blocks: [nb, BLOCK]."""
    return torch.cat([torch.nn.functional.pad(x.reshape(-1).to(to), (0, -x.numel() % BLOCK)) for x in tensors]).view(-1, BLOCK)


def _adamw(s):
    t = s["step"] + 1
    s["step"] = t
    p, g, states = s["p"], s["g"], s["states"]
    if s["case"]["bits"] == 32:
        for x, y, st in zip(p, g, states):
            gf, m, v = y.float(), st["exp_avg"], st["exp_avg_sq"]
            m.mul_(BETA1).add_(gf, alpha=1 - BETA1)
            v.mul_(BETA2).add_(gf.square(), alpha=1 - BETA2)
            x.copy_(_update(x.float(), m, v, t))
        return _adamw_out(s)
    gd = _blocks(g, torch.float64)                         # 64 bits: a moment decides between two codes
    m, v = (_blocks([st[k].float() for st in states], torch.float64)
            * torch.cat([st[k + "_scale"] for st in states]).double()[:, None] for k in ("exp_avg", "exp_avg_sq"))
    m = (BETA1 * m + (1 - BETA1) * gd).float()
    v = (BETA2 * v + (1 - BETA2) * gd * gd).float()
    word = _philox(*s["blocks"], t, s["seed"])
    new = dict(p=_update(_blocks(p, torch.float32), m, v, t))
    new["exp_avg"], new["exp_avg_scale"] = _held8(m, (word & 0xFFFF).int(), 3, 7, False)
    new["exp_avg_sq"], new["exp_avg_sq_scale"] = _held8(v, (word >> 16).int(), 2, 15, True)
    out = _adamw_out(s)
    for k, flat in new.items():
        count = [-(-x.numel() // BLOCK) * (flat.numel() // len(m)) for x in p]
        for x, y in zip(out[k], flat.view(-1).split(count)):
            (x.view(torch.uint8) if "float8" in str(x.dtype) else x).copy_(y[:x.numel()].view(x.shape))
    return out


def _adamw_out(s):
    return dict(p=s["p"], **{k: [st[k] for st in s["states"]] for k in s["states"][0]})


def _int8(s):
    x = s["x"].float()
    amax = x.abs().amax(1)
    sx = amax / torch.full_like(amax, 127)                 # (by a number it would be a product with 1 / 127)
    # 64 bits for the quotient: a value next to the middle of two integers goes to the nearer one
    q = torch.round(x.double() / sx.double()[:, None].clamp_min(1e-300)).clamp_(-127, 127).float()
    y = (q @ s["wq"].float().t()) * sx[:, None] * s["ws"]
    if s["bias"] is not None:
        y = y + s["bias"].float()
    return y.to(s["x"].dtype)


# ------------------------------------------------------------------------------------------------ one pass
def run(state):
    op = state["case"]["op"]
    if own:
        from scarches_amd import ops
        if op == "ln_fwd":
            y, stats = ops.layer_norm_fwd(state["x"], state["w"], state["b"], state["eps"])
            return dict(y=y, stats=stats)
        if op == "ln_bwd":
            dx, dw, db = ops.layer_norm_bwd(state["dy"], state["x"], state["w"], state["stats"])
            return dict(dx=dx) if dw is None else dict(dx=dx, dw=dw, db=db)
        if op == "adamw":
            opt = state.get("opt")
            if opt is None:                 # the optimizer that a program keeps, taken up at its 100th step
                opt = ops.AdamW(state["p"], lr=LR, betas=(BETA1, BETA2), eps=EPS, weight_decay=DECAY,
                                state_bits=state["case"]["bits"], seed=state["seed"])
                for p, g, st in zip(state["p"], state["g"], state["states"]):
                    p.grad = g
                    opt.state[p] = st
                opt.set_step(state["step"])
                state["opt"] = opt
            opt.step()
            return _adamw_out(state)
        return ops.int8_linear(state["x"], state["wq"], state["ws"], state["bias"])
    return {"ln_fwd": _ln_fwd, "ln_bwd": _ln_bwd, "adamw": _adamw, "int8": _int8}[op](state)


def work(case):
    size = 4 if case["dtype"] == "float32" else 2
    if case["op"] == "ln_fwd":
        rows, n = case["rows"], case["n"]
        return dict(bytes=2 * size * rows * n + 8 * rows + (2 * size * n if case["affine"] else 0), flops=8 * rows * n)
    if case["op"] == "ln_bwd":
        rows, n = case["rows"], case["n"]
        return dict(bytes=3 * size * rows * n + 8 * rows + (3 * size * n if case["affine"] else 0), flops=14 * rows * n)
    if case["op"] == "adamw":
        n = sum(math.prod(s) for s in shapes_of(case))
        nb = sum(-(-math.prod(s) // BLOCK) for s in shapes_of(case))
        states = 16 * n if case["bits"] == 32 else 4 * n + 16 * nb
        return dict(bytes=3 * size * n + states, flops=15 * n)
    rows, n, k = case["rows"], case["n"], case["k"]
    return dict(bytes=size * rows * k + n * k + 4 * n + size * rows * n + (size * n if case["bias"] else 0),
                flops=2 * rows * n * k)


# ------------------------------------------------------------------------------------------------ 64 bits
def _words(n, tensor, t, seed):
    """Random words of Philox4x32-10, on the host."""
    u = np.uint64
    c = np.zeros((4, -(-n // 4)), u)
    c[0], c[2], c[3] = np.arange(c.shape[1]), tensor, t
    key = np.array([seed & M32, seed >> 32], u)
    for _ in range(10):
        hi, lo = np.divmod(c[[0, 2]] * np.array([[0xD2511F53], [0xCD9E8D57]], u), u(2 ** 32))
        c = np.stack([hi[1] ^ c[1] ^ key[0], lo[1], hi[0] ^ c[3] ^ key[1], lo[0]])
        key = (key + np.array([0x9E3779B9, 0xBB67AE85], u)) % u(2 ** 32)
    return c.T.reshape(-1)[:n].astype(np.int64)


def _on_grid(x, random16, kind):
    """(values, scales) of what an 8-bit type holds of x behind its blocks' scales: of the two neighbours on the type's
    grid the upper one where the way from the lower one is at least 1 - random16 / 65536 of the step."""
    every = torch.arange(128, dtype=torch.uint8).view(kind).double().numpy()
    every = every[np.isfinite(every)]
    pad = np.pad(x.astype(np.float64), (0, -len(x) % BLOCK)).reshape(-1, BLOCK)
    amax = np.abs(pad).max(1)
    scale = np.where(amax > 0, 2.0 ** np.maximum(np.ceil(np.log2(np.maximum(amax, 1e-300) / every[-1])), -126), 0)
    t = np.abs(pad) / np.where(scale > 0, scale, 1)[:, None]
    low = np.searchsorted(every, t, "right") - 1
    up = np.minimum(low + 1, len(every) - 1)
    way = (t - every[low]) / np.where(up > low, every[up] - every[low], 1)
    took = np.where(way >= 1 - np.pad(random16, (0, -len(x) % BLOCK)).reshape(-1, BLOCK) / 65536, up, low)
    if kind == torch.float8_e5m2:
        took = np.where((pad > 0) & (took == 0), 1, took)
    return (np.sign(pad) * every[took]).reshape(-1)[:len(x)], scale


def exact(case, seed):
    s = prepare(case, seed)
    f = torch.float64
    if case["op"] == "ln_fwd":
        x = s["x"].to(f)
        var, mu = torch.var_mean(x, dim=1, correction=0)
        y = (x - mu[:, None]) / (var + s["eps"]).sqrt()[:, None]
        if case["affine"]:
            y = torch.addcmul(s["b"].to(f), y, s["w"].to(f))
        return dict(y=y, stats=torch.stack([mu, 1 / (var + s["eps"]).sqrt()]))
    if case["op"] == "ln_bwd":
        n = case["n"]
        mu, r = s["stats"].to(f)[0, :, None], s["stats"].to(f)[1, :, None]
        hat, dy = (s["x"].to(f) - mu) * r, s["dy"].to(f)
        a = dy * s["w"].to(f) if case["affine"] else dy
        dx = (r / n) * (n * a - a.sum(1, True) - hat * torch.linalg.vecdot(a, hat, dim=1)[:, None])
        out = dict(dx=dx)
        if case["affine"]:
            out |= dict(dw=torch.linalg.vecdot(dy, hat, dim=0), db=dy.sum(0))
        return out
    if case["op"] == "adamw":
        t = s["step"] + 1
        c1, c2 = 1 - BETA1 ** t, 1 - BETA2 ** t
        held = ["exp_avg", "exp_avg_sq"] if case["bits"] == 32 else list(s["states"][0])
        out = dict(p=[], **{k: [] for k in held})
        for j, (p, g, st) in enumerate(zip(s["p"], s["g"], s["states"])):
            m, v = st["exp_avg"].to(f), st["exp_avg_sq"].to(f)
            if case["bits"] == 8:
                per = [st[k].to(f).repeat_interleave(BLOCK)[:p.numel()].view(p.shape)
                       for k in ("exp_avg_scale", "exp_avg_sq_scale")]
                m, v = m * per[0], v * per[1]
            m, v = torch.lerp(g.to(f), m, BETA1), torch.lerp(g.to(f) ** 2, v, BETA2)
            new = p.to(f) - LR * (DECAY * p.to(f) + (m / c1) / ((v / c2) ** 0.5 + EPS))
            out["p"].append(new)
            if case["bits"] == 32:
                got = dict(exp_avg=m, exp_avg_sq=v)
            elif p.numel() > 1 << 20:
                got = dict.fromkeys(held)                   # one by one on the host: the small tensors only
            else:
                word = _words(p.numel(), j, t, s["seed"])
                got = {}
                for k, x, r, kind in (("exp_avg", m, word & 0xFFFF, torch.float8_e4m3fn),
                                      ("exp_avg_sq", v, word >> 16, torch.float8_e5m2)):
                    got[k], got[k + "_scale"] = _on_grid(x.float().cpu().numpy().reshape(-1), r, kind)
                    got[k] = got[k].reshape(p.shape)
            for k in held:
                out[k].append(got[k])
        return out
    x = s["x"].to(f)
    sx = (x.abs().amax(1) / 127).float().to(f)              # the scale is held in 32 bits
    q = torch.round(x / torch.where(sx > 0, sx, torch.ones_like(sx))[:, None]).clamp(-127, 127)
    y = torch.mm(q, s["wq"].to(f).t().contiguous()) * (sx[:, None] * s["ws"].to(f)[None, :])
    return y if s["bias"] is None else y + s["bias"].to(f)
