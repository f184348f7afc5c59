"""What clip refuses of tensors that require a gradient; all of it on the host, before the device is asked for."""
import pytest
import torch

from autolabel_amd import clip


@pytest.mark.parametrize('call', [
    lambda t, p: clip.clip_grad_norm_([p], 1.0),
    lambda t, p: clip.clip_grad_norm_(torch.nn.Linear(3, 3).parameters(), 1.0),
    lambda t, p: clip.clip_grad_norm_([t, p], 1.0),
    lambda t, p: clip.clip_grad_norm_([t], 1.0, out=[p]),
    lambda t, p: clip.clip_grad_norm_([p], 1.0, out=[t]),
    lambda t, p: clip.clip_grad_norm_([p * 2], 1.0),
    lambda t, p: clip.grad_norm([p]),
    lambda t, p: clip.grad_norm([t, p * 2]),
])
def test_refused_where_gradients_are_tracked(call):
    with pytest.raises(ValueError, match='requires a gradient'):
        call(torch.zeros(3), torch.zeros(3, requires_grad=True))


def test_without_gradients_a_leaf_is_refused_in_place_only():
    t, p = torch.zeros(3), torch.zeros(3, requires_grad=True)
    with torch.no_grad():
        with pytest.raises(ValueError, match='requires a gradient'):
            clip.clip_grad_norm_([p], 1.0)
        with pytest.raises(ValueError, match='requires a gradient'):
            clip.clip_grad_norm_([t, p], 1.0, out=[torch.zeros(3), p])
        for allowed in (lambda: clip.clip_grad_norm_([t], 1.0, out=[p]), lambda: clip.clip_grad_norm_([p], 1.0, out=[t]), lambda: clip.grad_norm([p])):
            with pytest.raises(ValueError, match='no CPU path'):      # (it gets as far as the device)
                allowed()
    with torch.enable_grad():
        q = p * 2
    with torch.no_grad(), pytest.raises(ValueError, match='no CPU path'):
        clip.clip_grad_norm_([q], 1.0)


def test_a_norm_that_requires_a_gradient():
    with pytest.raises(ValueError, match='norm requires a gradient'):
        clip.grad_norm([torch.zeros(3)], norm=torch.zeros((), requires_grad=True))
