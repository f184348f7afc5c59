"""TrainEngine.grad_norm is the norm of the last clipped step, however that step ran: eager, replayed from either of the two graphs that a marching
engine captures, or eager steps between replays."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope='module')
def scene():
    from autolabel_amd import synthetic
    from autolabel_amd.dataset import DeviceFrames
    s = synthetic.make_cube_scene(n_frames=8, size=32, seed=0)
    return s, DeviceFrames.from_scene(s, 'cuda')


def marching_engine(s):
    """lr = 0: the parameters stay, so the norm of step i depends on the step number alone, whichever way the steps before it ran."""
    from autolabel_amd.engine import TrainEngine
    from autolabel_amd.models import ALNetwork
    torch.manual_seed(0)
    model = ALNetwork(encoding='hg+freq', num_layers=2, hidden_dim=128, geo_feat_dim=15, num_layers_color=2, hidden_dim_color=128, hidden_dim_semantic=64,
                      semantic_classes=s['n_classes'], bound=3.0, cuda_ray=True, density_scale=1, grid_size=32, max_steps=128, march_samples=32).cuda()
    pipe = model._ensure_device()
    pipe.occ.update_interval = 4
    eng = TrainEngine(pipe, lr=0.0, max_grad_norm=1e-3)
    eng.model = model              # (holds the parameters)
    return eng


def eager_norms(s, frames, steps):
    eng = marching_engine(s)
    batch = frames.alloc_batch(1024)
    norms = []
    for i in range(steps):
        frames.next_train(batch, seed=5, step=i)
        eng.step(batch, seed=7, step=i)
        norms.append(float(eng.grad_norm))
    return norms


def near(a, b):
    """The same sums in another order (compaction and atomics): 2^17 additions of 2^-24 each at the very most are 2^-7; 1e-3 is met with ease."""
    return all(math.isclose(x, y, rel_tol=1e-3) for x, y in zip(a, b))


def test_both_graphs_of_a_marching_engine_report_their_norm(scene):
    s, frames = scene
    want = eager_norms(s, frames, 12)
    assert all(math.isfinite(n) and n > 1e-3 for n in want) and len(set(want)) == len(want)
    eng = marching_engine(s)
    batch = frames.alloc_batch(1024)
    g = eng.graphed(frames, batch, data_seed=5, seed=7, first_step=0, warmup=2)
    assert g.alt_graph is not None and g.steps == 2
    got = []
    while g.steps < 12:
        g()
        got.append(float(eng.grad_norm))
    assert near(got, want[2:]), (got, want[2:])


def test_eager_steps_between_replays(scene):
    s, frames = scene
    want = eager_norms(s, frames, 9)
    eng = marching_engine(s)
    batch = frames.alloc_batch(1024)
    g = eng.graphed(frames, batch, data_seed=5, seed=7, first_step=0, warmup=2)
    g()                                            # step 2
    held = eng.grad_norm
    frames.next_train(batch, seed=5, step=1)
    eng.step(batch, seed=7, step=1, grid_update=False)
    assert near([float(eng.grad_norm)], [want[1]])
    eng.state_i[0:1].copy_(torch.tensor([3], dtype=torch.int32))
    g()                                            # step 3, the plain graph
    assert near([float(eng.grad_norm)], [want[3]])
    g()                                            # step 4, with the grid's refresh
    assert near([float(eng.grad_norm)], [want[4]]) and eng.grad_norm is held


def test_no_clipping_no_norm(scene):
    from autolabel_amd.engine import TrainEngine
    s, _ = scene
    eng = marching_engine(s)
    assert float(eng.grad_norm) == 0.0             # (before the first step)
    assert TrainEngine(eng.pipe).grad_norm is None


def test_clip_writes_the_norm_where_it_is_told():
    from autolabel_amd import clip
    t = [torch.randn(1000, device='cuda'), torch.randn(70, device='cuda').half()]
    want = clip.grad_norm(t)
    buf = torch.full((), 7.0, device='cuda')
    assert clip.grad_norm(t, norm=buf) is buf and torch.equal(buf, want)
    buf.fill_(7.0)
    assert clip.clip_grad_norm_(t, 0.5 * float(want), norm=buf) is buf and torch.equal(buf, want)
    for bad in (torch.zeros((), device='cuda', dtype=torch.float64), torch.zeros(()), 1.0):
        with pytest.raises(ValueError, match='norm must be'):
            clip.grad_norm(t, norm=bad)
