"""What the beam search calls tell autograd: nothing is recorded, and tensors that they write count as modified."""
import numpy as np
import pytest

from test_gpu_beam import on

pytestmark = pytest.mark.gpu

PARENTS = np.array([[1, 1, 0, 3]], np.int32)


@pytest.mark.parametrize("into", [False, True])
def test_a_backward_pass_over_a_moved_state_raises(device, into):
    """The product's gradient needs the values that were there before they moved."""
    import torch
    import radx_amd
    leaf = torch.arange(12.0, device=device).reshape(4, 3).requires_grad_()
    other = torch.ones(4, 3, device=device)
    state = leaf * 2.0
    loss = (state * state).sum()
    (grad,) = torch.autograd.grad(loss, leaf, retain_graph=True)
    assert torch.equal(grad, 8.0 * leaf)
    if into:
        radx_amd.beam_reorder(other, on(PARENTS, device), into=state)
    else:
        radx_amd.beam_reorder(state, on(PARENTS, device))
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()


def test_tensors_that_are_written_and_no_others(device):
    import torch
    import radx_amd
    parents = on(PARENTS, device)
    states, into = [[torch.zeros(4, 3, device=device) for _ in range(2)] for _ in range(2)]
    whole = torch.zeros(4, 8, device=device)
    radx_amd.beam_reorder(states, parents, into=into)
    radx_amd.beam_reorder(whole[:, 2:5], parents)
    assert [t._version for t in states + into + [whole, parents]] == [0, 0, 1, 1, 1, 0]
    sel = radx_amd.BeamSelector(1, 4, 50, 4)
    logits, cum = torch.randn(4, 50, device=device, requires_grad=True), torch.zeros(1, 4, device=device)
    out = [o.clone() for o in sel.select(logits, cum, 4)]
    before = [t._version for t in out]
    got = sel.select(logits, cum, 4, out=out)
    assert [t._version for t in out] == [v + 1 for v in before]
    assert logits._version == cum._version == 0 and not got[0].requires_grad
    record = torch.zeros(1, 4, 6, dtype=torch.int32, device=device)
    steps = torch.zeros(6, 1, 4, dtype=torch.int32, device=device)
    radx_amd.beam_backtrace(steps, steps, out=record)
    assert record._version == 1 and steps._version == 0
    sel.close()


def test_inference_mode(device):
    """Tensors made in inference mode have no versions, in it and outside."""
    import torch
    import radx_amd
    with torch.inference_mode():
        state = torch.arange(4.0, device=device).reshape(4, 1)
        parents = on(PARENTS, device)
        radx_amd.beam_reorder(state, parents)
    radx_amd.beam_reorder([state, torch.zeros(4, 1, device=device)], parents)
    assert state.flatten().tolist() == [1.0, 1.0, 1.0, 3.0]
