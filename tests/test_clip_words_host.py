"""aln_grad_clip refuses a loss scale, a norm or an overflow flag that lies in a tensor that it scales: one block would write what others still read."""
import ctypes as C

import pytest

from autolabel_amd import hip

A = 1 << 20        # aligned to everything; never followed: every call fails on the host


def call(apply, loss_scale, norm, found_inf, grads=(A, A + 4096), numel=(10, 10), out=None):
    arr = lambda t, v: (t * len(v))(*v) if v is not None else None
    hip.call('aln_grad_clip', len(grads), arr(C.c_void_p, grads), arr(C.c_void_p, out), arr(C.c_int64, numel), arr(C.c_int32, (2,) * len(grads)), 1.0, apply, loss_scale, norm,
             found_inf, A + (1 << 16), 1 << 14, None)


@pytest.mark.parametrize('at', [A, A + 36, A + 4096, A + 4096 + 36])
@pytest.mark.parametrize('which', range(3))
def test_a_word_inside_a_tensor(which, at):
    words = [None, None, None]
    words[which] = at
    with pytest.raises(RuntimeError, match='share memory'):
        call(1, *words)


def test_a_word_inside_an_output_or_another_word():
    with pytest.raises(RuntimeError, match='share memory'):
        call(1, None, A + 8192 + 4, None, out=(A + 8192, A + 12288))
    with pytest.raises(RuntimeError, match='share memory'):
        call(1, A + 16384, A + 16384, None)
