"""Recorded and captured steps over what ordinary training does between them: ragged minibatches, an encoder pass, another matrix.
Every step starts from the parameters and moments of the same step of an eager run (the noise of the float atomics would grow over
many), and has to give its losses; bounds as in test_gpu_look_ahead."""
import gc

import pytest
import torch

from tests.test_gpu_look_ahead import assert_same, batches, data, make_engine, run        # noqa: F401 (data: a fixture)

pytestmark = pytest.mark.gpu


def captured(eng):
    return {k[0] for k in eng._plans if k[1]}


def same_steps(data, bs, mode, hook=lambda eng, i, *batch: batch, ahead=True):      # noqa: F811
    """Runs the steps eagerly, then as `mode` launches them; the engine of the second run."""
    states = []

    def keeps(eng, i, *batch):
        states.append([t.clone() for t in (eng.flat_p, eng.flat_m, eng.flat_v)])
        return hook(eng, i, *batch)

    def takes(eng, i, *batch):
        for t, was in zip((eng.flat_p, eng.flat_m, eng.flat_v), states[i]):
            t.copy_(was)
        return hook(eng, i, *batch)
    ref = run(data, bs, False, ahead=False, hook=keeps)
    got = run(data, bs, mode, ahead=ahead, hook=takes)
    assert_same(got, ref)
    return got[2]


def test_ragged_minibatches_between_captured_ones(data):            # noqa: F811
    full, ragged = batches(data, 1024, 6, seed=11), batches(data, 300, 2, seed=12)
    eng = same_steps(data, full[:3] + ragged[:1] + full[3:] + ragged[1:], "auto")
    assert captured(eng) == {1024} and {k[0] for k in eng._plans} == {1024, 300}


def test_steps_behind_an_encoder_pass_are_planned(data):            # noqa: F811
    """No captured step is replayed behind the pass, none is captured.  (A pass moves the counter of the random numbers, so the
    eager run has the same ones.)"""
    probe = batches(data, 512, 1, seed=6)[0]
    seen = []

    def hook(eng, i, rows, cond, nxt):
        if i in (0, 1):                                             # the one in front of the first step changes nothing
            before = captured(eng)
            eng.encode(probe[0], probe[1], 512)
            if before:
                seen.append(before)
                for g in eng._plans.values():                       # (a replay would fail here, and not run)
                    g["fwd"] = None
        return rows, cond, nxt
    eng = same_steps(data, batches(data, 1024, 4, seed=11), "auto", hook)
    assert seen == [{1024}] and any(not k[1] for k in eng._plans)


def test_engines_that_go_while_their_step_runs(data):               # noqa: F811
    """Dropped right behind an asynchronous step, and found by the collector: the device is idle afterwards, the next engine's
    steps are its own."""
    bs = batches(data, 1024, 3, seed=11)
    for cycle in (False, True):
        eng = make_engine(data)
        for rows, cond in bs:
            eng.train_step(rows, cond, 1024, 0.5, 1e-3)
        if cycle:
            eng.me = eng
        del eng
        gc.collect()
        assert torch.cuda.current_stream().query()
        same_steps(data, bs, "auto")


@pytest.mark.parametrize("mode", ["plan", True, "auto"])
def test_another_matrix_between_the_steps(data, mode):              # noqa: F811
    """A recorded step holds the addresses of the matrix that it gathers from: cells of another one (a second data set, the
    upload of a second trainer) are not to be read there, nor what was gathered ahead from it."""
    indptr, indices, vals = data["csr"]
    other = (indptr, indices, (vals * 3 + 1).contiguous())

    def hook(eng, i, rows, cond, nxt):
        if i in (2, 4):
            eng.bind_csr(*(other if i == 2 else data["csr"]))
        return rows, cond, nxt
    same_steps(data, batches(data, 1024, 6, seed=11), mode, hook)


@pytest.mark.parametrize("mode", ["plan", "auto"])
def test_noise_switched_off_between_the_steps(data, mode):          # noqa: F811
    def hook(eng, i, rows, cond, nxt):
        eng.noise_off = i >= 2
        return rows, cond, nxt
    # (the second size outgrows the zeros of the first)
    same_steps(data, batches(data, 1024, 4, seed=11) + batches(data, 1500, 2, seed=12), mode, hook)
