"""Which failures of the data-parallel test's worker are tried again (tests/test_gpu_clip_rccl_once.py): a set-up that raised, nothing else."""
import pytest
import torch.multiprocessing as mp

from test_gpu_clip_rccl_once import failing_set_up, failing_step, killed, run


@pytest.mark.parametrize('target, error, starts', [(failing_set_up, mp.ProcessRaisedException, 2), (failing_step, mp.ProcessRaisedException, 1),
                                                   (killed, mp.ProcessExitedException, 1)])
def test_what_is_tried_again(target, error, starts):
    with pytest.raises(error) as e:
        run(target)
    assert e.value.starts == starts
