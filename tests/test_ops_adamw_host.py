"""The host side of ops.AdamW on stubs (no GPU needed): the table of addresses and the launches are recorded, not made."""
import pytest
import torch

from scarches_amd import ops


@pytest.fixture
def calls(monkeypatch):
    made = []

    def table(self, gi, group, key, grads):
        steps = self._group_steps(gi)
        return dict(key=key, grads=grads, captured=False, table=steps, streams={0}, entries=0, n=len(grads), chunks=0, n_chunks=0,
                    steps=steps, scratch=0, index=0)
    monkeypatch.setattr(ops, "_same_device", lambda *tensors: 0)
    monkeypatch.setattr(ops, "_raw_stream", lambda index: 0)
    monkeypatch.setattr(ops, "_call", lambda index, name, *args: made.append((name, args)))
    monkeypatch.setattr(ops.AdamW, "_table", table)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    return made


def param(*shape):
    return torch.ones(*shape, requires_grad=True)


def step_number(call):
    assert call[0] == "sca_adamw_step"
    return call[1][6]


def test_parameters_change_their_version(calls):
    """backward, step, backward: what the first backward saved has changed, and autograd has to know it."""
    p, q, frozen = param(3), param(3), param(3)
    opt = ops.AdamW([p, frozen, q])
    loss = (p * q).sum()
    loss.backward(retain_graph=True)
    before = [x._version for x in (p, q, frozen)]
    opt.step()
    assert [x._version for x in (p, q, frozen)] == [before[0] + 1, before[1] + 1, before[2]]
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()


def test_a_failed_call_counts_no_step(calls, monkeypatch):
    """The step that is taken after an error is the one that the error kept from being taken."""
    p = param(3)
    opt = ops.AdamW([p])
    p.grad = torch.ones(3)
    opt.step()
    assert step_number(calls[-1]) == 1
    with monkeypatch.context() as m:
        def fail(index, name, *args):
            raise ops._lib.HipLibraryError("launch")
        m.setattr(ops, "_call", fail)
        with pytest.raises(ops._lib.HipLibraryError):
            opt.step()
        opt.param_groups[0]["eps"] = "a"                    # what ctypes refuses never gets as far as the launch either
    with monkeypatch.context() as m:
        m.setattr(ops, "_call", lambda index, name, *args: ops._lib.load().sca_adamw_step(*args, None))
        with pytest.raises(Exception, match="argument 11"):
            opt.step()
    opt.param_groups[0]["eps"] = 1e-8
    opt.step()
    assert step_number(calls[-1]) == 2 and opt._host_steps[0] == (2, 1)


def test_a_failed_call_that_the_device_counts(calls, monkeypatch):
    """Where the device counts, nobody here can tell how far it came: it goes on counting."""
    p, q = param(3), param(3)
    opt = ops.AdamW([p, q])
    p.grad = torch.ones(3)
    opt.step()
    q.grad = torch.ones(3)
    with monkeypatch.context() as m:
        def fail(index, name, *args):
            raise ops._lib.HipLibraryError("launch")
        m.setattr(ops, "_call", fail)
        with pytest.raises(ops._lib.HipLibraryError):
            opt.step()
    q.grad = None
    opt.step()
    assert step_number(calls[-1]) == 0
