"""CPU test of the rows that the join of an attention's parts reads (tests/native/join_rows_check.cpp, built with g++ from the kernel's own header): a
sequence without rows behind the last one must read nothing, since the workspace ends where its first row would begin."""
import shutil
import subprocess
from pathlib import Path

import pytest

HERE = Path(__file__).resolve().parent


@pytest.mark.skipif(shutil.which('g++') is None, reason='needs g++')
def test_joined_rows_lie_in_the_workspace(tmp_path):
    exe = tmp_path / 'join_rows_check'
    subprocess.run(['g++', '-O2', '-I', str(HERE.parent / 'yanlongvla_amd' / 'csrc'), '-o', str(exe), str(HERE / 'native' / 'join_rows_check.cpp')], check=True)
    out = subprocess.run([str(exe)], capture_output=True, text=True, timeout=120)
    assert out.returncode == 0 and out.stdout == 'ok\n', out.stdout + out.stderr
