"""GPU tests of what ops.AdamW and the operators owe to torch around them: version counters, state dicts that stand by themselves,
refusals inside torch's transformations."""
import pytest
import torch
from torch.autograd import forward_ad

from tests.test_gpu_dense_ops import gen
from tests.test_gpu_dense_ops_edges import params, set_grads

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops():
    from scarches_amd import ops as m
    return m


@pytest.mark.parametrize("bits", [32, 8])
def test_a_step_between_two_backward_passes(ops, bits):
    """The second pass needs the parameter that the first one used: an error, as with torch's optimizers."""
    p, q = (torch.randn(300, device="cuda", generator=gen(s)).requires_grad_() for s in (1, 2))
    opt = ops.AdamW([p, q], state_bits=bits)
    loss = (p * q).sum()
    loss.backward(retain_graph=True)
    was = p._version
    opt.step()
    assert p._version > was
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()


def test_resumed_with_another_seed(ops):
    """8-bit states saved and loaded into an optimizer that was made with the default seed: the same bits as without the break."""
    p, q = params(3), params(3)
    a, b = ops.AdamW(p, state_bits=8, seed=77), ops.AdamW(q, state_bits=8)
    for s in range(2):
        set_grads(p, s)
        a.step()
    with torch.no_grad():
        for x, y in zip(p, q):
            y.copy_(x)
    b.load_state_dict(a.state_dict())
    for s in range(2, 5):
        set_grads(p, s)
        set_grads(q, s)
        a.step()
        b.step()
    for x, y in zip(p, q):
        assert torch.equal(x, y)
        for k in a.state[x]:
            assert torch.equal(a.state[x][k].view(torch.uint8), b.state[y][k].view(torch.uint8)), k


def test_a_gradient_that_became_shorter(ops):
    """Refused where its length shows; the optimizer goes on with the right one."""
    ps = params(5)
    opt = ops.AdamW(ps)
    set_grads(ps, 0)
    opt.step()
    before = [p.detach().clone() for p in ps]
    good = ps[2].grad
    ps[2].grad.data = torch.ones(16, device="cuda")
    with pytest.raises(ValueError, match="gradient of parameter 2"):
        opt.step()
    assert all(torch.equal(a, b) for a, b in zip(ps, before))
    set_grads(ps, 1)
    opt.step()
    assert opt.state_dict()["state"][2]["step"] == 2
    del good


def test_transformations_are_refused(ops):
    x, w = torch.randn(8, 40, device="cuda", generator=gen(1)), torch.ones(40, device="cuda")
    wq, ws = ops.quantize_int8(torch.randn(5, 40, device="cuda", generator=gen(2)))
    calls = (lambda v: ops.layer_norm(v, w, w), lambda v: ops.int8_linear(v, wq, ws), lambda v: ops.quantize_int8(v)[1])
    for call in calls:
        want = call(x)
        with forward_ad.dual_level():
            with pytest.raises(RuntimeError, match="forward-mode"):
                call(forward_ad.make_dual(x, x))
            assert torch.equal(call(x), want)                       # (no tangent: as ever)
        with pytest.raises(RuntimeError, match="trace does not record"):
            torch.jit.trace(call, (x,))
        assert torch.equal(call(x), want)
    with forward_ad.dual_level():
        with pytest.raises(RuntimeError, match="forward-mode"):
            ops.layer_norm(forward_ad.make_dual(x, x), w.clone().requires_grad_(), w)


def test_under_torch_compile(ops):
    """A graph break: the operators run as ever, forward and backward."""
    x, w = torch.randn(8, 40, device="cuda", generator=gen(1)), torch.ones(40, device="cuda", requires_grad=True)
    wq, ws = ops.quantize_int8(torch.randn(5, 40, device="cuda", generator=gen(2)))

    def f(v):
        return ops.layer_norm(v * 2, w, w) + 1

    def g(v):
        return ops.int8_linear(v * 2, wq, ws) + 1
    for backend in ("eager", "aot_eager"):
        for call in (f, g):
            torch._dynamo.reset()
            assert torch.equal(torch.compile(call, backend=backend)(x), call(x)), (backend, call)
        torch._dynamo.reset()
        got, = torch.autograd.grad(torch.compile(f, backend=backend)(x).square().sum(), w)
        want, = torch.autograd.grad(f(x).square().sum(), w)
        assert torch.equal(got, want), backend


@pytest.mark.parametrize("bits", [32, 8])
def test_a_training_step_in_one_graph(ops, bits):
    """Forward, backward through autograd and the optimizer's step captured together, replayed between eager work, against the
    same steps taken eagerly."""
    def leaves():
        return [t.requires_grad_() for t in (torch.randn(64, 96, device="cuda", generator=gen(1)), torch.ones(96, device="cuda"),
                                             torch.zeros(96, device="cuda"))]

    def step(ps, opt, dy):
        opt.zero_grad(set_to_none=True)
        ops.layer_norm(*ps).backward(dy)
        opt.step()
    a, b = leaves(), leaves()
    oa, ob = (ops.AdamW(ps, lr=1e-2, state_bits=bits, seed=5) for ps in (a, b))
    oa._host_steps[0] = (None, None)                        # (the device counts in both: the same bits)
    static = torch.randn(64, 96, device="cuda", generator=gen(2))
    for _ in range(3):
        step(a, oa, static)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(3):
            step(b, ob, static)
    torch.cuda.current_stream().wait_stream(side)
    ob.zero_grad(set_to_none=True)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(b, ob, static)
    for i in range(6):
        static.copy_(torch.randn(64, 96, device="cuda", generator=gen(10 + i)))
        graph.replay()
        step(a, oa, static)
        if i % 2:
            torch.cuda.synchronize()
        for p, q in zip(a, b):
            assert torch.equal(p, q), i
    assert ob.state_dict()["state"][2]["step"] == 9
