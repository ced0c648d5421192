"""The host side of ops.AdamW on stubs (no GPU needed): the table of addresses and the launches are recorded, not made."""
import pytest
import torch

from scarches_amd import ops


TABLE = ops.AdamW._table


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


def test_the_state_dict_holds_the_seed(calls):
    """A run that is taken up by an optimizer of another seed goes on with its own: the rounding of its states hangs on it."""
    p, q = param(300), param(300)
    opt, other = ops.AdamW([p], state_bits=8, seed=2 ** 63 + 9), ops.AdamW([q], state_bits=8)
    p.grad = q.grad = torch.ones(300)
    opt.step()
    sd = opt.state_dict()
    other.load_state_dict(sd)
    other.step()
    assert other.seed == 2 ** 63 + 9 and calls[-1][1][11] == 2 ** 63 + 9
    assert "seed" not in other.param_groups[0] and other.state_dict()["param_groups"] == sd["param_groups"]
    for group in sd["param_groups"]:
        del group["seed"]                                   # saved before there was one: the constructor's
    third = ops.AdamW([param(300)], state_bits=8, seed=4)
    third.load_state_dict(sd)
    assert third.seed == 4
    two = ops.AdamW([dict(params=[param(3)]), dict(params=[param(3)])], state_bits=8)
    sd = two.state_dict()
    sd["param_groups"][1]["seed"] = 1
    with pytest.raises(ValueError, match="different seeds"):
        two.load_state_dict(sd)
    assert "seed" not in ops.AdamW([param(3)]).state_dict()["param_groups"][0]


def test_a_group_without_parameters(calls):
    """torch allows one (all of its parameters frozen away, say): it takes no part in anything."""
    p = param(3)
    p.grad = torch.ones(3)
    opt = ops.AdamW([dict(params=[]), dict(params=[p], lr=0.5)])
    opt.set_step(7)
    opt.step()
    assert len(calls) == 1 and step_number(calls[0]) == 8
    other = ops.AdamW([dict(params=[]), dict(params=[param(3)])])
    other.load_state_dict(opt.state_dict())
    assert other.param_groups[1]["lr"] == 0.5 and other._host_steps == {1: (7, 1)}


def test_tensors_that_change_in_place(calls):
    """Behind .data a tensor may become another one at the same address, or a gradient a shorter one: the table is made anew
    then, where the layouts are checked, instead of being given other addresses."""
    made = []
    table = ops.AdamW._table

    def counted(self, *args):
        made.append(0)
        return table(self, *args)
    p = param(6, 6)
    opt = ops.AdamW([p])
    opt._table = counted.__get__(opt)
    p.grad = torch.ones(6, 6)
    opt.step()
    p.grad = torch.ones(6, 6)                               # other storage alone is not that
    held = torch.ones(64)                                   # (so that no address comes back)
    opt.step()
    assert len(made) == 1
    p.grad.data = torch.ones(4)
    opt.step()
    assert len(made) == 2
    p.grad.data = torch.ones(6, 6)
    opt.step()
    assert len(made) == 3
    p.data = p.data.t()
    opt.step()
    assert len(made) == 4
    del held


def test_parameters_without_states(calls, monkeypatch):
    """A parameter that never took a step has no entry in the state dict, also behind a capture or an error; dicts that hold an
    empty one load."""
    p, frozen = param(3), param(3)
    opt = ops.AdamW([p, frozen])
    p.grad = torch.ones(3)
    opt.step()
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    opt.step()
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    assert set(opt.state_dict()["state"]) == {0}
    opt.state[frozen]
    sd = opt.state_dict()
    assert set(sd["state"]) == {0}
    sd["state"][1] = dict(step=0)
    other = ops.AdamW([param(3), param(3)])
    other.load_state_dict(sd)
    assert set(other.state_dict()["state"]) == {0} and other._steps[0][1] == 0
    joins = other.param_groups[0]["params"][1]
    joins.grad = torch.ones(3)
    other.step()
    assert set(other.state[joins]) == {"exp_avg", "exp_avg_sq"}


def test_a_group_that_was_changed_by_hand(calls, monkeypatch):
    """Each parameter's step number has its place in an array as long as the group was: no table over another length."""
    monkeypatch.setattr(ops.AdamW, "_table", TABLE)
    opt = ops.AdamW([param(3)])
    opt.set_step(4)
    for change in (lambda ps: ps.append(param(3)), lambda ps: ps.append(param(3)), lambda ps: ps.__delitem__(slice(None, None))):
        change(opt.param_groups[0]["params"])
        for p in opt.param_groups[0]["params"]:
            p.grad = torch.ones(3)
        if opt.param_groups[0]["params"]:
            with pytest.raises(RuntimeError, match="add_param_group"):
                opt.step()
    assert not calls
