"""CPU test: an entry that launches its kernel more than once reports an error of any of the launches. The launches go to a stand-in for the
runtime's functions, which fails the one that it is told to; no kernel runs."""
import shutil
import subprocess
import sys
from pathlib import Path

import pytest

LIB = Path(__file__).resolve().parents[1] / 'yanlongvla_amd' / 'libtcq.so'
pytestmark = pytest.mark.skipif(not LIB.exists() or not shutil.which('gcc'), reason='libtcq.so not built, or no C compiler')

STAND_IN = r'''
static int count, fail, last;
void stand_in(int which) { count = last = 0; fail = which; }
int stand_in_launches(void) { return count; }
int hipLaunchKernel(const void* f, ...) { (void)f; return last = ++count == fail ? 719 : 0; }
int hipGetLastError(void) { int e = last; last = 0; return e; }
int __hipPushCallConfiguration(void) { return 0; }             // (the launch's size, which nothing here reads)
int __hipPopCallConfiguration(void) { return 0; }
int hipFuncSetAttribute(const void* f, int a, int v) { (void)f; (void)a; (void)v; return 0; }
'''
CALLER = r'''
import ctypes, sys
sys.path.insert(0, sys.argv[3])
fake = ctypes.CDLL(sys.argv[1], mode=ctypes.RTLD_GLOBAL)
lib = ctypes.CDLL(sys.argv[2])
P, I, L, F = ctypes.c_void_p, ctypes.c_int, ctypes.c_int64, ctypes.c_float
lib.tcq_kv8_attend.argtypes = [P, L, L, I, P, P, I, I, I, I, I, I, I, P, P, P, I, F, I, P, P, P]
at = 1 << 12                                                   # an aligned address that nothing reads
def attend(rows, keys, fail):
    fake.stand_in(fail)
    rc = lib.tcq_kv8_attend(at, 1024, 64, 1, None, at, rows, rows, 1, 16, 1, 64, 100, at, at, at, 1, 0.1, keys, at, at, None)
    print(rc, fake.stand_in_launches())
for fail in (0, 1, 2):
    attend(65600, 64, fail)                                    # 32800 tiles of 32 rows
for fail in (0, 1, 2, 3):
    attend(200000, 64, fail)                                   # 100000 tiles: two launches
for fail in (0, 1, 2):
    attend(1, 6400, fail)                                      # parts and their join
'''


def test_attend_reports_every_launch(tmp_path):
    (tmp_path / 'f.c').write_text(STAND_IN)
    (tmp_path / 'c.py').write_text(CALLER)
    subprocess.run(['gcc', '-shared', '-fPIC', '-o', tmp_path / 'f.so', tmp_path / 'f.c'], check=True)
    out = subprocess.run([sys.executable, tmp_path / 'c.py', tmp_path / 'f.so', LIB, LIB.parents[1]], capture_output=True, text=True, timeout=300)
    assert out.returncode == 0, out.stderr
    got = [tuple(map(int, x.split())) for x in out.stdout.split('\n') if x]
    assert got == [(0, 1), (719, 1), (0, 1),
                   (0, 2), (719, 1), (719, 2), (0, 2),
                   (0, 2), (719, 1), (719, 2)]
