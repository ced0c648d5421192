"""The models' own paths on the dense operators: AdamW in the engine's training step (eager, recorded and captured) and in the
trainers, the first encoder layer's product in 8-bit integers in get_latent."""
import contextlib
import io

import numpy as np
import pytest
import torch

from tests.test_gpu_api import synth
from tests.test_gpu_dense_ops import HALF, U, within
from tests.test_gpu_step import make_engine

pytestmark = pytest.mark.gpu


def adamw_ref(p, m, v, g, t, lr, eps, wd):
    """(p, m, v) in 64 bits after a step, and how far fp32 may be off p."""
    m1, v1 = 0.9 * m + 0.1 * g, 0.999 * v + 0.001 * g * g
    denom = (v1 / (1 - 0.999 ** t)).sqrt() + eps
    upd = lr / (1 - 0.9 ** t) * m1 / denom
    # decay and step: three roundings of p; moments, root, quotient and the fp32 bias corrections: some sixteen of the step
    bound = 3 * U * p.abs() + 16 * U * upd.abs() + 3 * U * lr / (1 - 0.9 ** t) * (0.9 * m.abs() + 0.1 * g.abs()) / denom
    return p * (1 - lr * wd) - upd, m1, v1, bound


@pytest.mark.parametrize("mode", [False, "plan", True], ids=["eager", "plan", "graph"])
def test_engine_steps_with_adamw(mode):
    eng, z, cfg, W, _, _ = make_engine("trvae_nb_ln_small")
    B, lr, eps, wd = cfg["B"], 3e-3, 0.01, 0.5
    over = {k: 0.0 for k in eng.names if "theta" in k}
    frozen = [k for k in eng.names if "FC.L1" in k] or eng.names[-1:]
    eng.set_trainable([k for k in eng.names if k not in frozen])
    eng.set_optimizer("adamw")
    rows = torch.arange(B, device="cuda")
    cond = torch.tensor(z["batch"]).to(torch.int32).cuda()
    moved = 0.0
    for t in range(1, 5):
        before = [{k: d[k].double().clone() for k in eng.names} for d in
                  (eng.p, {k: eng.flat_m[eng.offsets[k]:eng.offsets[k] + eng.p[k].numel()].view_as(eng.p[k]) for k in eng.names},
                   {k: eng.flat_v[eng.offsets[k]:eng.offsets[k] + eng.p[k].numel()].view_as(eng.p[k]) for k in eng.names})]
        eng.train_step(rows, cond, B, alpha_kl=0.5, lr=lr, eps=eps, weight_decay=wd, use_graph=mode, wd_overrides=over)
        torch.cuda.synchronize()
        for k in eng.names:
            p0 = before[0][k]
            if k in frozen:
                assert torch.equal(eng.p[k].double(), p0), k
                continue
            ref, m, v, bound = adamw_ref(p0, before[1][k], before[2][k], eng.g[k].double(), t, lr, eps, over.get(k, wd))
            within(eng.p[k], ref, bound, (t, k))
            moved = max(moved, (eng.p[k].double() - p0).abs().max().item())
    assert moved > 1e-4
    # the same engine goes back to the coupled form: its step is Adam's again
    eng.set_optimizer("adam")
    p0 = {k: eng.p[k].double().clone() for k in eng.names}
    m0, v0 = eng.flat_m.double().clone(), eng.flat_v.double().clone()
    eng.train_step(rows, cond, B, alpha_kl=0.5, lr=lr, eps=eps, weight_decay=wd, use_graph=mode, wd_overrides=over)
    torch.cuda.synchronize()
    for k in eng.names:
        if k in frozen:
            continue
        o, n = eng.offsets[k], eng.p[k].numel()
        g = eng.g[k].double() + over.get(k, wd) * p0[k]
        m, v = (0.9 * m0[o:o + n].view_as(g) + 0.1 * g), (0.999 * v0[o:o + n].view_as(g) + 0.001 * g * g)
        upd = lr / (1 - 0.9 ** 5) * m / ((v / (1 - 0.999 ** 5)).sqrt() + eps)
        # (that kernel takes 1 - b2 in fp32: 1.3e-5 of what a step adds to v)
        within(eng.p[k], p0[k] - upd, 4 * U * p0[k].abs() + 3e-5 * lr + 2e-5 * upd.abs(), k)
    with pytest.raises(ValueError, match="optimizer"):
        eng.set_optimizer("sgd")


@pytest.mark.parametrize("model", ["trvae", "scpoli"])
def test_trainers_take_the_optimizer(model):
    from scarches_amd.anndata_lite import CellData
    from scarches_amd.models import TRVAE, scPoli
    X, obs = synth(400, 64, 3, 3, seed=5)
    ad = CellData(X, obs)
    kw = dict(n_epochs=2, lr=1e-3, batch_size=64, monitor=False)
    with contextlib.redirect_stdout(io.StringIO()):
        torch.manual_seed(0)
        if model == "trvae":
            m = TRVAE(ad, condition_key="study", hidden_layer_sizes=[32], latent_dim=5)
        else:
            m = scPoli(ad, condition_keys="study", cell_type_keys="cell_type", hidden_layer_sizes=[32], latent_dim=5,
                       embedding_dims=3)
            kw["pretraining_epochs"] = 2
        start = {k: v.clone() for k, v in m.model.state_dict().items()}
        m.train(optimizer="adamw", weight_decay=10.0, **kw)
        eng = m.model.engine()
        assert eng.optimizer == "adamw"
        # decoupled: no step moves a value by more than 1e-3 (10 |p| + some), however large the decay
        name = next(k for k in start if k.endswith("expr_L.weight"))
        steps = eng.adam_t
        now, was = m.model.state_dict()[name].cpu(), start[name].cpu()
        assert steps > 0 and (now - was).abs().max() <= steps * 1e-3 * (10 * was.abs().max() + 4)
        assert torch.isfinite(now).all() and not torch.equal(now, was)
        m.train(**kw)
        assert eng.optimizer == "adam"
        with pytest.raises(ValueError, match="optimizer"):
            m.train(optimizer="lion", **kw)


@pytest.mark.parametrize("hidden,use_bn", [([64, 32], False), ([48], False), ([40, 24], True)])
def test_latent_in_8_bit_integers(hidden, use_bn):
    """get_latent(int8=True): the first layer's product is the operator's on what the loader gathered, the layers behind it
    are the ordinary ones (64-bit reference from that product)."""
    from scarches_amd import ops
    from scarches_amd.anndata_lite import CellData
    from scarches_amd.models import TRVAE
    X, obs = synth(500, 197, 3, 3, seed=6)
    ad = CellData(X, obs)
    with contextlib.redirect_stdout(io.StringIO()):
        torch.manual_seed(1)
        m = TRVAE(ad, condition_key="study", hidden_layer_sizes=hidden, latent_dim=6, use_bn=use_bn)
    m.model.eval()
    eng = m.model.engine()
    mu = torch.from_numpy(m.get_latent(mean=True, int8=True)).cuda()
    eng.noise_off = True
    assert m.get_latent(int8=True).shape == (500, 6) and len(m.get_latent(mean_var=True, int8=True)) == 2
    m.get_latent(mean=True)                 # leaves the gathered cells in the workspace
    x = eng.ws["x"][:500 * 197].view(-1)[:500 * 197].view(500, 197) if eng.ws["x"].dim() == 1 else eng.ws["x"][:500]
    ly = eng.enc[0]
    wq, ws = eng.quantize_first_layer()
    prod = ops.int8_linear(x.contiguous(), wq, ws)
    q, s = ops.quantize_int8(x.contiguous())
    off = 0.5001 * (x.double().abs().sum(1, keepdim=True) * ws.double() + s.double()[:, None] * (wq.double().abs().sum(1) * ws.double()))
    full = x.double() @ eng.p[ly.w].double().t().contiguous()
    within(prod, full, off + 8 * U * (x.double().abs() @ eng.p[ly.w].double().abs().t().contiguous() + off), "product")
    labels = torch.from_numpy(m._encode_labels(ad.obs["study"])).long().cuda()
    a = prod.double()
    for i, ly in enumerate(eng.enc):
        if i:
            a = a @ eng.p[ly.w].double().t().contiguous()
        a = a + eng.p[ly.b].double()
        if ly.wc:
            a = a + eng.p[ly.wc].double().t()[labels]
        if use_bn:
            mean, var = (eng.buffers[ly.bn + k].double() for k in (".running_mean", ".running_var"))
            a = (a - mean) / (var + 1e-5).sqrt() * eng.p[ly.bn + ".weight"].double() + eng.p[ly.bn + ".bias"].double()
        else:
            a = torch.nn.functional.layer_norm(a, (ly.n_out,))
        a = torch.relu(a)
    ref = a @ eng.heads_w[:6].double().t().contiguous() + eng.heads_b[:6].double()
    # two or three short products and normalisations in fp32: rel 1e-5 of the largest, as for the fp32 encoder
    assert (mu.double() - ref).abs().max() <= 1e-5 * max(1.0, ref.abs().max().item())
    exact = torch.from_numpy(m.get_latent(mean=True)).cuda()
    assert not torch.equal(exact, mu)


@pytest.mark.parametrize("G,nnz,log1p", [(197, 40, 1), (2000, 284, 1), (2000, 1999, 0), (15, 3, 1), (20011, 900, 1), (65536, 70, 0)])
def test_csr_rows_in_8_bit_integers(G, nnz, log1p):
    """Rows of a CSR matrix, quantized on the way: bit for bit the gather followed by the row quantization - empty rows, stored
    zeros, unsorted columns, repeated and permuted rows, values that are not finite, a scale below what fp32 inverts."""
    from scarches_amd import _lib, ops
    lib = _lib.load()
    g = np.random.default_rng(G + nnz)
    counts = g.integers(0, nnz + 1, 37)
    counts[[0, 5]] = 0
    counts[1] = nnz
    indptr = np.concatenate([[0], np.cumsum(counts)]).astype(np.int64)
    indices = np.concatenate([g.permutation(G)[:c] for c in counts]).astype(np.int32)
    data = (g.integers(0, 60, indptr[-1]) if log1p else g.standard_normal(indptr[-1])).astype(np.float32)
    if log1p == 0:
        data[indptr[2]:indptr[3]] *= np.float32(1e-38)
        data[indptr[3]:indptr[3] + 1] = np.nan
        data[indptr[4]:indptr[4] + 1] = np.inf
    ip, ix, dv = (torch.from_numpy(t).cuda() for t in (indptr, indices, data))
    for rows in (None, torch.from_numpy(g.integers(0, 37, 300)).cuda()):
        B = 37 if rows is None else 300
        x = torch.empty(B, G, device="cuda")
        st = torch.cuda.current_stream().cuda_stream
        _lib.check(lib.sca_csr_gather_rows(ip.data_ptr(), ix.data_ptr(), dv.data_ptr(), _lib.ptr(rows), B, G, log1p, x.data_ptr(),
                                           G, torch.empty(B, device="cuda").data_ptr(), st), "gather")
        want, scale = ops.quantize_int8(x)
        pitch = -(-G // 128) * 128
        q = torch.full((B + 1, pitch), 77, dtype=torch.int8, device="cuda")
        s = torch.empty(B, device="cuda")
        _lib.check(lib.sca_csr_quant_rows_i8(ip.data_ptr(), ix.data_ptr(), dv.data_ptr(), _lib.ptr(rows), B, G, log1p,
                                             q.data_ptr(), pitch, s.data_ptr(), st), "csr_quant_rows_i8")
        assert torch.equal(q[:B, :G], want) and torch.equal(s.view(torch.int32), scale.view(torch.int32))
        assert not q[:B, G:].any() and (q[B] == 77).all()               # padded with zeros; the row behind is left alone


def small_model(model):
    from scarches_amd.anndata_lite import CellData
    from scarches_amd.models import EXPIMAP, TRVAE, scPoli
    X, obs = synth(400, 64, 3, 3, seed=5)
    ad = CellData(X, obs)
    torch.manual_seed(0)
    if model == "trvae":
        return TRVAE(ad, condition_key="study", hidden_layer_sizes=[32], latent_dim=5)
    if model == "expimap":
        mask = np.random.default_rng(2).random((8, 64)) < 0.4             # [programs, genes]
        return EXPIMAP(ad, condition_key="study", hidden_layer_sizes=[32, 32], mask=mask.astype(np.float32), recon_loss="nb")
    return scPoli(ad, condition_keys="study", cell_type_keys="cell_type", hidden_layer_sizes=[32], latent_dim=5, embedding_dims=3)


def test_expimap_trains_with_adamw():
    with contextlib.redirect_stdout(io.StringIO()):
        m = small_model("expimap")
        start = {k: v.clone() for k, v in m.model.state_dict().items()}
        m.train(n_epochs=2, lr=1e-3, batch_size=64, monitor=False, optimizer="adamw", weight_decay=10.0, alpha=1e-4)
    eng = m.model.engine()
    assert eng.optimizer == "adamw"
    name = next(k for k in start if k.startswith("encoder") and k.endswith("expr_L.weight"))
    now, was = m.model.state_dict()[name].cpu(), start[name].cpu()
    assert eng.adam_t > 0 and (now - was).abs().max() <= eng.adam_t * 1e-3 * (10 * was.abs().max() + 4)
    assert torch.isfinite(now).all() and not torch.equal(now, was)


@pytest.mark.parametrize("model", ["trvae", "expimap", "scpoli"])
def test_latent_from_csr_and_from_dense_rows(model, monkeypatch):
    """get_latent(int8=True) gives the same bits whether the cells go to 8-bit integers from CSR or from gathered rows."""
    with contextlib.redirect_stdout(io.StringIO()):
        m = small_model(model)
        args = (m.adata.X, m.adata.obs["study"]) if model != "scpoli" else (m.adata,)
        one = m.get_latent(*args, mean=True, int8=True)
        monkeypatch.setattr(type(m.model.engine()), "_quantized_cells", lambda *a: None)
        two = m.get_latent(*args, mean=True, int8=True)
        exact = m.get_latent(*args, mean=True)
    assert np.array_equal(one, two) and np.isfinite(one).all() and not np.array_equal(one, exact)


@pytest.mark.parametrize("decay", [0.0, 10.0])
@pytest.mark.parametrize("model", ["trvae", "expimap", "scpoli"])
def test_every_step_of_a_trainer_is_adamw(model, decay):
    """Each step that a trainer takes, as it launches it by default, against the formula on the gradient that the step left."""
    kw = dict(n_epochs=2, lr=1e-3, eps=0.02, batch_size=64, monitor=False, optimizer="adamw", weight_decay=decay)
    with contextlib.redirect_stdout(io.StringIO()):
        m = small_model(model)
        if model == "expimap":
            kw["alpha"] = 1e-4
        if model == "scpoli":
            kw["pretraining_epochs"] = 2
        eng = m.model.engine()
        name = "adam_step" if model == "scpoli" else "train_step"
        step, taken = getattr(eng, name), []

        def parts():
            return [[flat[eng.offsets[k]:eng.offsets[k] + eng.p[k].numel()].view_as(eng.p[k]).double().clone() for k in eng.names]
                    for flat in (eng.flat_p, eng.flat_m, eng.flat_v)]

        def checked(*args, **kwargs):
            before = parts()
            out = step(*args, **kwargs)
            over = kwargs.get("wd_overrides") or {}
            for k, p, mo, v in zip(eng.names, *before):
                if eng.trainable[k]:
                    ref, _, _, bound = adamw_ref(p, mo, v, eng.g[k].double(), eng.adam_t, 1e-3, 0.02, over.get(k, decay))
                    within(eng.p[k], ref, bound, (eng.adam_t, k))
                else:
                    assert torch.equal(eng.p[k].double(), p), k
            taken.append(eng.adam_t)
            return out
        setattr(eng, name, checked)
        m.train(**kw)
    assert len(taken) >= 10 and taken == list(range(1, len(taken) + 1))
