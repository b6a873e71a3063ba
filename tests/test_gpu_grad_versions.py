"""Clipping writes gradients outside autograd's sight: it moves their version counters as torch's own in-place operations do, so that a
backward pass that saved them says so instead of using clipped values."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def _set(cuda):
    flat = torch.ones(100, device=cuda)
    own = torch.ones(7, device=cuda)
    with torch.inference_mode():
        untracked = torch.ones(5, device=cuda)
    return [flat[:40], flat[40:], own, untracked], flat, own


@pytest.mark.parametrize("kind", ["full_model", "norm", "value"])
def test_clipping_moves_the_versions_and_measuring_does_not(cuda, kind):
    from yolo_amd.solver import GradientClipper
    grads, flat, own = _set(cuda)
    c = GradientClipper(grads, kind, 0.5)
    before = flat._version, own._version
    c.measure()
    assert (flat._version, own._version) == before
    c.clip_()
    assert flat._version > before[0] and own._version > before[1] and grads[0]._version == flat._version
    assert max(float(g.max()) for g in grads) < 1


@pytest.mark.parametrize("kind", ["norm", "value"])
def test_a_saved_gradient_is_not_used_after_clipping(cuda, kind):
    from yolo_amd.solver import clip_grad_norm_, clip_grad_value_
    p = torch.nn.Parameter(torch.ones(4, device=cuda))
    (p ** 3).sum().backward(create_graph=True)
    penalty = (p.grad * p.grad).sum()          # saves p.grad
    if kind == "norm":
        clip_grad_norm_([p], 0.1)
    else:
        clip_grad_value_([p], 0.1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        penalty.backward()
