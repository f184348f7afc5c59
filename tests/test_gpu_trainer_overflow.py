"""The generic loop with max_grad_norm: a step whose gradients have no finite norm is skipped, with and without a loss scaler."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

from test_gpu_api import _host_batches, _trainer, make_model


def _setup(fp16, value):
    ds, batches = _host_batches(3)
    bound = float(((ds.max_bounds - ds.min_bounds) - (ds.min_bounds + ds.max_bounds) * 0.5).max())
    torch.manual_seed(0)
    model = make_model(D=64, C_=7, bound=bound, grid_scale=1.0)
    tr = _trainer(model, False, fp16=fp16)
    assert not tr.fused and tr.scaler.is_enabled() == fp16
    tr.max_grad_norm = 1.0
    state = {'bad': True}
    p = model.sigma_net.params
    p.register_hook(lambda g: torch.full_like(g, value) if state['bad'] else g)
    return model, tr, batches, state


def _flat(model):
    return torch.cat([p.detach().reshape(-1).clone() for _, p in model._param_blocks()])


@pytest.mark.parametrize('value', [3e38, math.inf, math.nan])
@pytest.mark.parametrize('fp16', [False, True])
def test_a_norm_that_is_not_finite_skips_the_step(fp16, value):
    """3e38: every gradient is finite (3e38 / 65536 with the scaler, whose own check passes; the norm of some 1e4 of them is then finite as well), the
    norm without the scaler is 3e40."""
    model, tr, batches, state = _setup(fp16, value)
    before = _flat(model)
    tr.train_iterations(iter(batches[:1]), 1)
    finite = fp16 and value == 3e38
    assert torch.equal(_flat(model), before) != finite
    assert torch.isfinite(_flat(model)).all()
    state['bad'] = False
    tr.train_iterations(iter(batches[1:]), 2)
    assert not torch.equal(_flat(model), before) and torch.isfinite(_flat(model)).all()


def test_a_norm_over_fp32_behind_a_scaler_skips_the_step():
    """Gradients that are finite once unscaled but whose norm is not: the scaler's own check lets them pass."""
    model, tr, batches, state = _setup(True, 3e38)
    tr.scaler = torch.amp.GradScaler('cuda', init_scale=1.0, growth_interval=1000)
    before = _flat(model)
    tr.train_iterations(iter(batches[:1]), 1)
    assert torch.equal(_flat(model), before)
    assert float(tr.scaler.get_scale()) == 1.0     # (no overflow of the scaled gradients)
    state['bad'] = False
    tr.train_iterations(iter(batches[1:]), 2)
    assert not torch.equal(_flat(model), before)


@pytest.mark.parametrize('fp16', [False, True])
def test_one_step_at_a_time(fp16):
    """InteractiveTrainer.take_step."""
    from autolabel_amd.trainer import InteractiveTrainer
    model, tr, batches, state = _setup(fp16, math.inf)
    it = InteractiveTrainer('ngp', tr.opt, model, device='cuda:0', workspace=None, optimizer=lambda m: torch.optim.Adam(m.parameters(), lr=1e-3), fp16=fp16,
                            lr_scheduler=lambda o: torch.optim.lr_scheduler.StepLR(o, gamma=0.5, step_size=1), fused=False, mute=True, max_grad_norm=1.0)
    it.iterator, it.step = iter(batches), 0
    model.train()
    before = _flat(model)
    it.take_step()
    assert torch.equal(_flat(model), before)
    state['bad'] = False
    it.take_step()
    assert not torch.equal(_flat(model), before) and torch.isfinite(_flat(model)).all()
