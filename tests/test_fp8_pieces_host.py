"""The addresses that the 8-bit weight gradient reads, enumerated on the CPU (tests/native/fp8_pieces.cpp) from the arithmetic that the kernel itself uses.

On the GPU an over-read of up to seven values behind the tensors could go unseen: an allocation is larger than its tensor, and what the values belong to are
columns behind the last, which are never stored."""
import os
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CPP = os.path.join(ROOT, 'tests', 'native', 'fp8_pieces.cpp')


def build_and_run(tmp_path, source):
    exe = tmp_path / 'fp8_pieces'
    subprocess.run(['g++', '-O2', '-fsanitize=undefined', '-fno-sanitize-recover=all', '-std=c++17', str(source), '-o', str(exe)], check=True, capture_output=True, text=True)
    return subprocess.run([str(exe)], capture_output=True, text=True, timeout=300)


@pytest.mark.skipif(shutil.which('g++') is None, reason='needs g++')
def test_every_piece_is_inside_its_tensor(tmp_path):
    r = build_and_run(tmp_path, CPP)
    assert r.returncode == 0, r.stdout[-2000:] + r.stderr[-2000:]
    assert 'inside their tensors' in r.stdout


@pytest.mark.skipif(shutil.which('g++') is None, reason='needs g++')
@pytest.mark.parametrize('guard, without', [('&& (col + 32 <= C || left * ld >= 7)', ''), ('left * ld >= 7', 'left * ld >= 6'), ('- 8};', '- 7};'),
                                            ('(C - 1 - col) & ~7', 'C & ~7'), ('at > e.end ? at - e.end : 0', '0')])
def test_the_enumeration_sees_a_missing_guard(tmp_path, guard, without):
    """The same run over arithmetic with one bound taken out or moved, on the CPU."""
    head = open(os.path.join(ROOT, 'autolabel_amd', 'csrc', 'fp8_pieces.h')).read()
    assert head.count(guard) == 1
    (tmp_path / 'fp8_pieces.h').write_text(head.replace(guard, without))
    cpp = open(CPP).read().replace('../../autolabel_amd/csrc/fp8_pieces.h', str(tmp_path / 'fp8_pieces.h'))
    (tmp_path / 'planted.cpp').write_text(cpp)
    r = build_and_run(tmp_path, tmp_path / 'planted.cpp')
    assert r.returncode == 1 and ('out of the tensor' in r.stdout or 'another value' in r.stdout), r.stdout[-500:] + r.stderr[-500:]
