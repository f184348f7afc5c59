"""The framework's own paths through the 8-bit products and the gradient clipping: the training engine and the trainers with max_grad_norm, the
wide feature head with set_semantic_fp8, the compression autoencoder with fp8=True, and a training step that runs them together."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

from test_gpu_api import _host_batches, _trainer
from test_gpu_fp8 import blocks64, check, product_bound


def _engine(layout, scene_seed=0, **kw):
    from autolabel_amd.engine import TrainEngine
    from autolabel_amd.pipeline import HipPipeline, Params
    P = Params(layout, torch.device('cuda'))
    P.init_(seed=scene_seed)
    return TrainEngine(HipPipeline(layout, P), num_steps=32, upsample_steps=32, **kw)


@pytest.fixture(scope='module')
def cube():
    from autolabel_amd import synthetic
    from autolabel_amd.dataset import DeviceFrames
    from autolabel_amd.pipeline import ModelLayout
    scene = synthetic.make_cube_scene(n_frames=8, size=32, seed=0)
    return DeviceFrames.from_scene(scene, 'cuda'), ModelLayout('hg+freq', 15, 128, 128, 64, scene['n_classes'], bound=3.0)


def _run(eng, frames, steps, start=0):
    batch = frames.alloc_batch(1024)
    for i in range(start, start + steps):
        frames.next_train(batch, seed=5, step=i)
        eng.step(batch, seed=7, step=i)
    torch.cuda.synchronize()


def _state(eng):
    return eng.P.flat.clone(), eng.m.clone(), eng.v.clone(), eng.P.table16.clone(), eng.state_i[:9].clone(), eng.state_f.clone()


def test_engine_with_a_bound_that_is_never_met_steps_as_without(cube):
    frames, layout = cube
    a, b = _engine(layout, fuse_grid_adam=False), _engine(layout, max_grad_norm=math.inf)
    assert not b.fuse_grid_adam and a.grad_norm is None
    _run(a, frames, 5)
    _run(b, frames, 5)
    assert all(torch.equal(x, y) for x, y in zip(_state(a), _state(b))) and float(b.grad_norm) > 0


def test_engine_clips_to_the_bound(cube):
    """Three steps, each against the same step taken by hand from the same state: the gradients, their norm in 64 bits, the factor, the optimizer.

    The factor may differ by its rounding (2^-24, the norm's own sum is taken in another order).  That moves m = b1 m + c1 g by 2^-22 |c1 g| at
    most, v by 2^-21 c2 g^2, and a parameter, whose step is lr m / sqrt(v) with sqrt(v) >= sqrt(c2) |g| = 0.1 |g|, by lr 2^-20 < 1e-8.  (Not so over
    several steps: the next forward pass rounds the parameters to fp16, and Adam divides small gradients by their own size.)"""
    frames, layout = cube
    a, b = _engine(layout, max_grad_norm=1e-3), _engine(layout, fuse_grid_adam=False)
    batch = frames.alloc_batch(1024)
    for i in range(3):
        for x, y in ((b.P.flat, a.P.flat), (b.m, a.m), (b.v, a.v), (b.state_i, a.state_i), (b.state_f, a.state_f)):
            x.copy_(y)
        b.P.refresh_shadows()
        p0, m0, v0 = a.P.flat.clone(), a.m.clone(), a.v.clone()
        frames.next_train(batch, seed=5, step=i)
        scale = float(b.state_f[0])
        a.step(batch, seed=7, step=i)
        b.forward_backward(batch, 7, i)
        g = b.P.grad[:layout.n_total]
        norm = math.sqrt(float((g.double() ** 2).sum())) / scale
        assert norm > 1e-3                     # (or the test tests nothing)
        assert abs(float(a.grad_norm) - norm) <= 2.0 ** -22 * norm
        g.mul_(torch.tensor(min(1.0, 1e-3 / (norm + 1e-6)), dtype=torch.float32, device='cuda'))
        clipped = g.clone()
        b.optimizer_step()
        torch.cuda.synchronize()
        assert torch.equal(a.state_i, b.state_i) and torch.equal(a.state_f, b.state_f)
        # (every sum rounds relative to its operands: the old moments and the weight decay 1e-6 p among them, which may cancel)
        gi = clipped.abs() / scale + 1e-6 * p0.abs()
        assert ((a.m - b.m).abs() <= 2.0 ** -22 * (gi + m0.abs()) + 1e-38).all()
        assert ((a.v - b.v).abs() <= 2.0 ** -20 * (gi * gi + v0.abs()) + 1e-38).all()
        assert ((a.P.flat - b.P.flat).abs() <= 1e-7 + 2.0 ** -23 * b.P.flat.abs()).all()


def test_engine_overflow_skips_the_step(cube):
    frames, layout = cube
    eng = _engine(layout, max_grad_norm=1.0, scaler={'init_scale': 2.0 ** 40})
    before = eng.P.flat.clone()
    _run(eng, frames, 1)
    assert torch.equal(eng.P.flat, before) and float(eng.state_f[0]) == 2.0 ** 39 and int(eng.state_i[0]) == 0
    assert (eng.P.grad[:layout.n_total] == 0).all() and int(eng.state_i[2]) == 0
    _run(eng, frames, 30, start=1)
    assert int(eng.state_i[0]) > 0 and torch.isfinite(eng.P.flat).all()


def test_engine_captured_step_clips_as_the_eager_one(cube):
    frames, layout = cube
    a, b = _engine(layout, max_grad_norm=1e-3), _engine(layout, max_grad_norm=1e-3)
    _run(a, frames, 8)
    batch = frames.alloc_batch(1024)
    g = b.graphed(frames, batch, data_seed=5, seed=7, first_step=0, warmup=2)
    while g.steps < 8:
        g()
        torch.cuda.synchronize()
        assert float(b.grad_norm) > 0
    assert all(torch.equal(x, y) for x, y in zip(_state(a), _state(b)))
    assert torch.equal(a.grad_norm, b.grad_norm)


@pytest.mark.parametrize('fused', [False, True])
def test_trainers_take_max_grad_norm(fused):
    from test_gpu_api import make_model
    ds, batches = _host_batches(3)
    bound = float(((ds.max_bounds - ds.min_bounds) - (ds.min_bounds + ds.max_bounds) * 0.5).max())
    torch.manual_seed(0)
    model = make_model(D=64, C_=7, bound=bound, grid_scale=1.0)
    assert max(int(b['semantic'].max()) for b in batches) < 7      # (the room scene has seven classes)
    tr = _trainer(model, fused)
    tr.max_grad_norm = 1e-3
    norms = []
    if not fused:
        step = tr.optimizer.step
        def spy(*a, **k):
            norms.append(math.sqrt(sum(float((p.grad.double() ** 2).sum()) for p in model.parameters() if p.grad is not None)))
            return step(*a, **k)
        tr.optimizer.step = spy
    loader = iter(batches)
    tr.train_iterations(loader, 3)
    if fused:
        assert float(tr.engine.grad_norm) > 0 and tr.engine.max_grad_norm == 1e-3
    else:
        assert norms and all(n <= 1e-3 * (1 + 1e-5) for n in norms)


def test_wide_head_in_8_bits(cube):
    """set_semantic_fp8: the same chain of calls by hand, bit for bit, and near the fp16 head; off again, the fp16 head's bits."""
    from autolabel_amd import fp8
    from autolabel_amd.models import ALNetwork
    torch.manual_seed(0)
    model = ALNetwork(encoding='hg+freq', num_layers=2, hidden_dim=128, geo_feat_dim=15, num_layers_color=2, hidden_dim_color=128,
                      hidden_dim_semantic=512, semantic_classes=4, bound=2.0).cuda()
    geo = torch.randn(1003, 15, device='cuda')
    logits, feat = model.semantic(geo)
    model.set_semantic_fp8()
    logits8, feat8 = model.semantic(geo)
    assert torch.isfinite(feat8).all() and torch.isfinite(logits8).all()
    # the hidden activation of the fp16 head, from the kernels that the head runs, then the last layer by hand
    pipe, W = model._pipe, model._pipe.P.wide_w['semf']
    so = torch.zeros(1003, 16, device='cuda', dtype=torch.float16)
    so[:, 1:] = geo.half()
    h2 = torch.empty(1003, 512, device='cuda', dtype=torch.float16)
    pipe._nt_gen(1003, h2, so)
    assert torch.equal(feat8, fp8.linear(h2, fp8.quantize(W[2])))
    want, tol = product_bound(blocks64(h2.cpu(), 'e4m3')[0], blocks64(W[2].cpu(), 'e4m3')[0], 512, torch.float16)
    check(feat8, want, tol)
    # one layer, every value of its operands off by at most 2^-4 of itself: within 2^-3 in the norm, and far less for sums of 512
    assert ((feat8 - feat).float().norm() / feat.float().norm()) < 2.0 ** -3
    assert not torch.equal(feat8, feat)
    o = torch.zeros(64, 3, device='cuda')
    d = torch.nn.functional.normalize(torch.randn(64, 3, device='cuda'), dim=-1)
    n = torch.ones(64, 1, device='cuda')
    with torch.inference_mode():
        r8 = model.eval().render(o, d, n, staged=True, perturb=False, num_steps=64, upsample_steps=0)
    model.set_semantic_fp8(False)
    with torch.inference_mode():
        r16 = model.render(o, d, n, staged=True, perturb=False, num_steps=64, upsample_steps=0)
    assert torch.equal(r8['image'], r16['image']) and torch.equal(r8['depth'], r16['depth'])
    assert not torch.equal(r8['semantic_features'], r16['semantic_features'])
    model.set_semantic_fp8()
    tracked = model.render(o, d, n, staged=True, perturb=False, num_steps=64, upsample_steps=0)     # with gradients: fp16
    assert torch.equal(tracked['semantic_features'], r16['semantic_features'])
    tracked['semantic_features'].sum().backward()
    model.set_semantic_fp8(False)
    again = model.semantic(geo)
    assert torch.equal(again[0], logits) and torch.equal(again[1], feat)
    narrow = ALNetwork(encoding='hg+freq', num_layers=2, hidden_dim=128, num_layers_color=2, hidden_dim_color=128)
    with pytest.raises(ValueError, match='not wide'):
        narrow.set_semantic_fp8()
    narrow.set_semantic_fp8(False)


class _Linear64(torch.autograd.Function):
    """The 8-bit layer by its definition in 64 bits, on the CPU."""

    @staticmethod
    def forward(ctx, x, w):
        ctx.save_for_backward(x, w)
        return blocks64(x.float(), 'e4m3')[0] @ blocks64(w.float(), 'e4m3')[0].t()

    @staticmethod
    def backward(ctx, g):
        x, w = ctx.saved_tensors
        q = lambda t: blocks64(t.float().contiguous(), 'e4m3')[0]
        return q(g) @ q(w.t()).t(), q(g.t()) @ q(x.t()).t()


def test_autoencoder_step_in_8_bits():
    """Forward, loss, backward, clipping and Adam of the compression autoencoder: its gradients against the definition in 64 bits.

    Between the layers the product's fp32 rounding differs from the 64-bit one by some 2^-20 of a value; where that crosses a border between two
    8-bit values (less than one in 2^15 of them) the value moves by a step, 2^-3 of itself at most: sqrt(2^-15) 2^-3 < 2^-10 of a tensor."""
    from autolabel_amd import clip
    from autolabel_amd.models import Autoencoder
    torch.manual_seed(0)
    net = Autoencoder(512, 64, fp8=True).cuda()
    plain = Autoencoder(512, 64)
    assert list(plain.state_dict()) == list(net.state_dict())
    plain.load_state_dict(net.state_dict())
    x = torch.rand(700, 512)
    code = net.encoder(x.cuda())
    loss = torch.nn.functional.mse_loss(net.decoder(code), x.cuda())
    loss.backward()
    w = [p.detach().double().requires_grad_() for p in plain.parameters()]
    h = x.double()
    for i, p in enumerate(w):
        h = _Linear64.apply(h, p)
        if i < 3:
            h = torch.relu(h)
    want = torch.nn.functional.mse_loss(h, x.double())
    want.backward()
    assert abs(float(loss) - float(want)) <= 2.0 ** -10 * float(want)
    for p, q in zip(net.parameters(), w):
        assert ((p.grad.cpu().double() - q.grad).norm() / q.grad.norm()) < 2.0 ** -10
    grads = [p.grad for p in net.parameters()]
    norm = math.sqrt(sum(float((g.double() ** 2).sum()) for g in grads))
    got = clip.clip_grad_norm_(grads, norm / 3)
    assert abs(float(got) - norm) <= 2.0 ** -22 * norm
    clipped = math.sqrt(sum(float((g.double() ** 2).sum()) for g in grads))
    assert abs(clipped - norm / 3) <= 1e-5 * norm
    opt = torch.optim.Adam(net.parameters(), lr=1e-3)
    for _ in range(3):
        opt.zero_grad()
        code = net(x.cuda())[0]
        torch.nn.functional.mse_loss(code, x.cuda()).backward()
        clip.clip_grad_norm_([p.grad for p in net.parameters()], 1.0)
        opt.step()
    assert all(torch.isfinite(p).all() for p in net.parameters())


def test_gradients_against_differences():
    """On values that the 8-bit grid holds exactly the layer is the plain product, and its gradients are differences of it."""
    from autolabel_amd import fp8
    g = torch.Generator().manual_seed(0)
    small = lambda *s: torch.randint(-3, 4, s, generator=g).float()
    x, w, gy = small(6, 20).cuda().requires_grad_(), small(5, 20).cuda(), small(6, 5).cuda()
    layer = fp8.Linear(20, 5, device='cuda')
    with torch.no_grad():
        layer.weight.copy_(w)
    f = lambda: float((layer(x) * gy).sum())
    (layer(x) * gy).sum().backward()
    for t in (x, layer.weight):
        for at in [(0, 0), (3, 7), (4, 19)]:
            with torch.no_grad():
                t[at] += 1
                up = f()
                t[at] -= 2
                down = f()
                t[at] += 1
            assert (up - down) / 2 == float(t.grad[at])


def test_8_bit_training_step_in_a_graph():
    """Forward, backward and clipping captured together, replayed on new inputs with eager steps of the same leaves between."""
    from autolabel_amd import clip, fp8
    torch.manual_seed(0)
    layer = fp8.Linear(200, 72, device='cuda')
    x, gy = torch.randn(900, 200, device='cuda'), torch.randn(900, 72, device='cuda')

    def body():
        with torch.enable_grad():
            y = layer(x)
            dw, = torch.autograd.grad(y, layer.weight, gy)
        norm = clip.clip_grad_norm_(dw, 0.5)
        return y.detach(), dw, norm
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        body()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = body()
    for i in range(4):
        x.copy_(torch.randn(900, 200))
        with torch.no_grad():
            layer.weight.add_(0.01)
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in out]
        want = body()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want)), i
