"""AdamW's step counters: every parameter counts its own steps, as torch.optim.AdamW's do."""

from __future__ import annotations

import copy
import io

import pytest
import torch

import fused_hoad

pytestmark = pytest.mark.gpu
# float32 states follow the same formula: sixteen roundings a step at most
UNIT = 16 * 2.0**-24


def pair(bits=32, **kwargs):
    g = torch.Generator(device="cuda").manual_seed(0)
    mine = [torch.randn(300, generator=g, device="cuda").requires_grad_() for _ in range(4)]
    theirs = [p.detach().clone().requires_grad_() for p in mine]
    return (mine, fused_hoad.AdamW(mine, lr=1e-2, state_bits=bits, **kwargs),
            theirs, torch.optim.AdamW(theirs, lr=1e-2, weight_decay=1e-2, **kwargs))


def set_grads(t, mine, theirs, active):
    g = torch.Generator(device="cuda").manual_seed(100 + t)
    for k, (p, q) in enumerate(zip(mine, theirs)):
        value = torch.randn(300, generator=g, device="cuda")
        p.grad = value if k in active else None
        q.grad = value.clone() if k in active else None


def compare(mine, theirs, steps):
    for k, (p, q) in enumerate(zip(mine, theirs)):
        assert torch.allclose(p, q, rtol=0, atol=UNIT * steps * 4.0), k


def test_first_gradients_at_different_steps():
    """A parameter that joins late, one that skips steps and one that never has a gradient."""
    mine, a, theirs, b = pair()
    for t in range(40):
        active = {0} | ({1} if t >= 30 else set()) | ({2} if t % 3 == 0 else set())
        set_grads(t, mine, theirs, active)
        a.step()
        b.step()
        compare(mine, theirs, t + 1)
    assert [int(a.state[p]["step"]) for p in mine[:3]] == [40, 10, 14] and mine[3] not in a.state


def test_parameters_in_step_share_a_counter():
    mine, a, theirs, b = pair()
    for t in range(3):
        set_grads(t, mine, theirs, {0, 1, 2, 3})
        a.step()
        b.step()
    assert len({a.state[p]["step"].data_ptr() for p in mine}) == 1
    set_grads(3, mine, theirs, {0, 1})
    a.step()
    b.step()
    assert [int(a.state[p]["step"]) for p in mine] == [4, 4, 3, 3]
    for t in range(4, 8):
        set_grads(t, mine, theirs, {0, 1, 2, 3})
        a.step()
        b.step()
    compare(mine, theirs, 8)


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("through_file", [False, True])
def test_counters_through_a_checkpoint(bits, through_file):
    mine, a, theirs, b = pair(bits)
    for t in range(6):
        set_grads(t, mine, theirs, {0, 1} if t < 2 else {0, 1, 2})
        a.step()
    state = a.state_dict()
    if through_file:
        file = io.BytesIO()
        torch.save(state, file)
        file.seek(0)
        state = torch.load(file)
    copies = [p.detach().clone().requires_grad_() for p in mine]
    again = fused_hoad.AdamW(copies, lr=1.0, state_bits=bits)
    again.load_state_dict(state)
    assert len({again.state[p]["step"].data_ptr() for p in copies[:3]}) == 2
    for t in range(6, 9):
        set_grads(t, mine, copies, {0, 1, 2, 3})
        a.step()
        again.step()
    assert [int(again.state[p]["step"]) for p in copies] == [9, 9, 7, 3]
    for p, q in zip(mine, copies):
        assert torch.equal(p, q)


def test_checkpoint_with_one_counter_a_group():
    """The older layout: a group's counter instead of the parameters'."""
    mine, a, theirs, b = pair()
    for t in range(5):
        set_grads(t, mine, theirs, {0, 1, 2, 3})
        a.step()
        b.step()
    state = copy.deepcopy(a.state_dict())
    for s in state["state"].values():
        step = s.pop("step")
    state["param_groups"][0]["step"] = step
    again = fused_hoad.AdamW(mine)
    again.load_state_dict(state)
    for t in range(5, 8):
        set_grads(t, mine, theirs, {0, 1, 2, 3})
        again.step()
        b.step()
    compare(mine, theirs, 8)


def test_checkpoint_of_the_library_optimizer():
    """torch.optim.AdamW's moments and step counts (float32, on the host) are taken over."""
    mine, a, theirs, b = pair()
    for t in range(5):
        set_grads(t, mine, theirs, {0, 1, 2, 3} if t else {0, 1})
        b.step()
    with torch.no_grad():
        for p, q in zip(mine, theirs):
            p.copy_(q)
    a.load_state_dict(b.state_dict())
    for t in range(5, 8):
        set_grads(t, mine, theirs, {0, 1, 2, 3})
        a.step()
        b.step()
        compare(mine, theirs, 3)


def test_late_parameter_in_a_graph():
    """A replay advances the counters on the device, each its own."""
    mine, a, theirs, b = pair()
    set_grads(0, mine, theirs, {0, 1})
    a.step()
    b.step()
    set_grads(1, mine, theirs, {0, 1, 2, 3})
    a.step()
    b.step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        a.step()
    for _ in range(5):
        graph.replay()
        b.step()
    compare(mine, theirs, 7)
    assert [int(a.state[p]["step"]) for p in mine] == [7, 7, 6, 6]


def test_states_made_in_a_capture_are_refused():
    """A replay would make them anew: a first step, and one that would part a counter."""
    mine, a, theirs, b = pair()
    set_grads(0, mine, theirs, {0, 1})
    for active in ({0, 1}, {0}):
        set_grads(0, mine, theirs, active)
        before = [p.detach().clone() for p in mine]
        with pytest.raises(RuntimeError, match="before the captured one"):
            with torch.cuda.graph(torch.cuda.CUDAGraph()):
                a.step()
        assert all(torch.equal(p, q) for p, q in zip(mine, before))
        set_grads(0, mine, theirs, {0, 1})
        a.step()
        b.step()
    compare(mine, theirs, 2)


def test_states_that_are_not_taken_over():
    mine, a, theirs, b = pair()
    for option in ("amsgrad", "maximize"):
        other = torch.optim.AdamW(theirs, **{option: True})
        with pytest.raises(ValueError, match="not supported"):
            a.load_state_dict(other.state_dict())
