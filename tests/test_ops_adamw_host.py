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
