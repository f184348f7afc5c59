"""What clip_grad_norm_ writes is known to autograd, and what it may not write is refused (the counterpart of the checks of fp8.linear(out=))."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope='module')
def clip():
    from autolabel_amd import clip, hip
    hip.require_gpu()
    hip.lib()
    return clip


@pytest.mark.parametrize('how', ['in place', 'out', 'in place, slow checks', 'not clipped'])
def test_a_saved_tensor_that_is_clipped_fails_its_backward_pass(clip, how):
    t, o = torch.ones(100, device='cuda'), torch.ones(100, device='cuda')
    leaf = torch.ones(100, device='cuda', requires_grad=True)
    loss = (leaf * (o if how == 'out' else t)).sum()
    other = torch.ones(7, device='cuda').half()
    if how == 'out':
        clip.clip_grad_norm_([t], 0.5, out=[o])
    elif how == 'in place, slow checks':
        clip.clip_grad_norm_([t, other], 0.5, found_inf=torch.zeros(1, dtype=torch.int32, device='cuda'))
    else:
        clip.clip_grad_norm_(t, 1e9 if how == 'not clipped' else 0.5)
    with pytest.raises(RuntimeError, match='modified by an inplace operation'):
        loss.backward()


def test_what_is_only_read_may_be_saved(clip):
    t = torch.ones(100, device='cuda')
    leaf = torch.ones(100, device='cuda', requires_grad=True)
    loss = (leaf * t).sum()
    clip.grad_norm([t])
    clip.clip_grad_norm_([t], 0.5, out=[torch.empty_like(t)])
    loss.backward()
    assert torch.equal(leaf.grad, t)


def test_parameters_are_not_gradients(clip):
    net = torch.nn.Linear(30, 20).cuda()
    net(torch.ones(4, 30, device='cuda')).sum().backward()
    weights = [p.detach().clone() for p in net.parameters()]
    for mode in (torch.enable_grad, torch.no_grad):
        with mode(), pytest.raises(ValueError, match='requires a gradient'):
            clip.clip_grad_norm_(net.parameters(), 1e-3)
    assert all(torch.equal(p, w) for p, w in zip(net.parameters(), weights))
    norm = clip.clip_grad_norm_([p.grad for p in net.parameters()], 1e-3)
    assert float(norm) > 1e-3
    assert sum(float((p.grad.double() ** 2).sum()) for p in net.parameters()) ** 0.5 <= 1e-3 * (1 + 1e-5)


def test_gradients_with_a_graph_of_their_own(clip):
    """create_graph=True: refused while gradients are tracked (the result would carry none), clipped with a version under no_grad."""
    w = torch.ones(50, device='cuda', requires_grad=True)
    g, = torch.autograd.grad((w ** 3).sum(), w, create_graph=True)
    with pytest.raises(ValueError, match='no_grad'):
        clip.clip_grad_norm_([g], 1.0)
    with pytest.raises(ValueError, match='no_grad'):
        clip.grad_norm([g])
    penalty = (g * g).sum()
    with torch.no_grad():
        clip.clip_grad_norm_([g], 1.0)
        assert abs(float(clip.grad_norm([g])) - 1.0) < 1e-5
    with pytest.raises(RuntimeError, match='modified by an inplace operation'):
        penalty.backward()


def test_inference_tensors(clip):
    with torch.inference_mode():
        t = torch.ones(100, device='cuda')
        clip.clip_grad_norm_([t], 1.0)
    o = torch.empty(100, device='cuda')
    clip.clip_grad_norm_([t], 0.5, out=[o])
    clip.clip_grad_norm_([t], 0.5)
    assert abs(float(clip.grad_norm([t])) - 0.5) < 1e-5 and abs(float(clip.grad_norm([o])) - 0.5) < 1e-5


def test_the_norm_and_the_flag_are_written_too(clip):
    t = torch.ones(100, device='cuda')
    leaf = torch.ones((), device='cuda', requires_grad=True)
    for apply in (False, True):
        norm, flag = torch.ones((), device='cuda'), torch.zeros(1, dtype=torch.int32, device='cuda')
        loss, version = leaf * norm, flag._version
        clip.clip_grad_norm_([t], 1.0, norm=norm, found_inf=flag) if apply else clip.grad_norm([t], norm=norm, found_inf=flag)
        assert flag._version > version
        with pytest.raises(RuntimeError, match='modified by an inplace operation'):
            loss.backward()
    with pytest.raises(ValueError, match='norm requires a gradient'):
        clip.grad_norm([t], norm=torch.zeros((), device='cuda', requires_grad=True))
