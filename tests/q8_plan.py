"""The launch rules of the 8-bit products (csrc/q8_plan.h), compiled for the host."""
import ctypes
import functools
import os
import subprocess
import tempfile
from collections import namedtuple

FITS, WIDE, MANY = range(3)
FEW, SHORT, LONG = range(3)
Plan = namedtuple('Plan', 'refusal kernel grid_x grid_y tiles cuts across split wc rt')


@functools.lru_cache(None)
def library():
    here = os.path.dirname(os.path.abspath(__file__))
    with tempfile.TemporaryDirectory() as d:
        so = os.path.join(d, 'plan.so')
        subprocess.check_call(['g++', '-std=c++17', '-O1', '-Wall', '-Wextra', '-Werror', '-shared', '-fPIC', '-o', so, os.path.join(here, 'q8_plan_shim.cpp')])
        return ctypes.CDLL(so)


def plan(M, n_cols, K, out_bytes=4, n_seg=1, ragged=False, n_cu=256):
    to = (ctypes.c_int64 * len(Plan._fields))()
    library().plan(M, n_seg, int(ragged), n_cols, K, out_bytes, n_cu, to)
    return Plan(*to)
