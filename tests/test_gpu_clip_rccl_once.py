"""The clipped data-parallel step over a process group of one rank (RCCL), run ONCE: whatever goes wrong from the first training launch on fails the test.
Only the set-up of the group -- init_process_group and one small collective -- is tried again, and only after a Python exception: a worker that ended by a
signal, or past that mark, is not started a second time."""
import os
import socket

import pytest
import torch
import torch.distributed as dist
import torch.multiprocessing as mp

pytestmark = pytest.mark.gpu


def set_up(port, ret):
    os.environ.update(MASTER_ADDR='127.0.0.1', MASTER_PORT=str(port), RANK='0', WORLD_SIZE='1', LOCAL_RANK='0')
    os.environ.setdefault('HSA_ENABLE_IPC_MODE_LEGACY', '0')
    torch.cuda.set_device(0)
    dev = torch.device('cuda', 0)
    dist.init_process_group('nccl', device_id=dev)
    one = torch.ones(4, device=dev)
    dist.all_reduce(one)
    torch.cuda.synchronize()
    assert float(one.sum()) == 4.0
    ret['ready'] = True
    return dev


def worker(rank, port, ret):
    dev = set_up(port, ret)
    from autolabel_amd import synthetic
    from autolabel_amd.dataset import DeviceFrames
    from autolabel_amd.engine import TrainEngine
    from autolabel_amd.pipeline import HipPipeline, ModelLayout, Params
    scene = synthetic.make_cube_scene(n_frames=8, size=32, seed=0, device=dev)
    frames = DeviceFrames.from_scene(scene, dev)
    layout = ModelLayout('hg+freq', 15, 128, 128, 64, scene['n_classes'], bound=3.0)
    out = {}
    for name, pg, payload, overlap in (('single', None, 'f32', False), ('simple', dist.group.WORLD, 'f32', False), ('overlap', dist.group.WORLD, 'f32', True)):
        P = Params(layout, dev)
        P.init_(seed=0)
        eng = TrainEngine(HipPipeline(layout, P), process_group=pg, num_steps=32, upsample_steps=32, overlap_comm=overlap, grad_payload=payload,
                          exchange_at_world_1=pg is not None, max_grad_norm=1e-3)
        batch = frames.alloc_batch(1024)
        norms = []
        for i in range(3):
            frames.next_train(batch, seed=5, step=i)
            eng.step(batch, seed=7, step=i)
            norms.append(float(eng.grad_norm))
        torch.cuda.synchronize()
        out[name] = dict(flat=P.flat.cpu(), norms=norms, dp=eng.dp)
    dist.barrier()
    torch.cuda.synchronize()
    ret['out'] = out
    dist.destroy_process_group()


def failing_set_up(rank, port, ret):
    ret['starts'] = ret.get('starts', 0) + 1
    raise RuntimeError('no group')


def failing_step(rank, port, ret):
    ret['starts'] = ret.get('starts', 0) + 1
    ret['ready'] = True
    raise RuntimeError('a step failed')


def killed(rank, port, ret):
    ret['starts'] = ret.get('starts', 0) + 1
    os.abort()


def run(target, tries=2):
    with mp.Manager() as mgr:
        ret = mgr.dict()
        for left in reversed(range(tries)):
            s = socket.socket()
            s.bind(('127.0.0.1', 0))
            port = s.getsockname()[1]
            s.close()
            try:
                mp.spawn(target, args=(port, ret), nprocs=1, join=True)
                return dict(ret)
            except mp.ProcessRaisedException as e:
                if ret.get('ready') or not left:
                    e.starts = ret.get('starts')
                    raise
            except mp.ProcessExitedException as e:
                e.starts = ret.get('starts')
                raise


def test_the_clipped_step_over_a_group_of_one():
    got = run(worker)['out']
    assert not got['single']['dp'] and got['simple']['dp'] and got['single']['norms'][0] > 1e-3
    for other in ('simple', 'overlap'):
        assert torch.equal(got['single']['flat'], got[other]['flat']) and got['single']['norms'] == got[other]['norms']
