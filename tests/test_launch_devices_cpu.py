"""What launchers of kernels with more than the plain shared memory or cluster size do on a second device of the process: the library's own code against a stand-in for the runtime's launches
(tests/cpp/fake_launch_runtime.c), in a process of its own."""
import os
import subprocess
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
LIB = os.path.join(ROOT, "simplellminference_b200", "lib", "libsllm_b200.so")

CHILD = """
import ctypes as C, sys
fake = C.CDLL(sys.argv[1], mode=C.RTLD_GLOBAL)          # in front of the runtime's own symbols
sys.path.insert(0, sys.argv[2])
from simplellminference_b200 import _lib
lib, at = _lib.load(), 0x7F0000000000
b = _lib.SeqBatch()
b.nseg, b.n_qtiles, b.max_pages, b.page_len = 2, 2, 8, 64
for name in ("tok_slot", "tok_pos", "seg_start", "seg_len", "seg_slot", "seg_pos0", "block_table", "qt_seg", "qt_off", "seg_tile0"):
    setattr(b, name, at)
def attend(T, dim):
    b.T = T
    return lib.sllm_seq_attention8(C.byref(b), at, 8 * dim, 8, 2, dim, dim, 0.1, at, at, at, at, 10, at, 1 << 40, None, at, 8 * dim, None, None)
def draw(n):
    return lib.sllm_sample_rows(at, n, 2, n, None, None, None, None, at, at, None, None)
call = {"draw": lambda: draw(128256), "decode": lambda: attend(2, 128), "decode_64": lambda: attend(2, 64), "portions": lambda: attend(40, 128), "portions_64": lambda: attend(40, 64)}[sys.argv[3]]
for device in (0, 1, 1, 0, 3):
    fake.cudaSetDevice(device)
    rc = call()
    print(rc, fake.fake_sets(), fake.fake_launches(), lib.sllm_last_error())
"""


@pytest.mark.parametrize("call,sets,launches", [("draw", 2, 1), ("decode", 1, 1), ("decode_64", 1, 1), ("portions", 2, 3), ("portions_64", 2, 3)])
def test_attributes_are_set_on_every_device_once(tmp_path, call, sets, launches):
    if not os.path.exists(LIB):
        pytest.skip("library not built")
    fake = str(tmp_path / "libfake.so")
    subprocess.run(["gcc", "-shared", "-fPIC", "-Wall", "-Werror", "-I/usr/local/cuda/include", "-o", fake, os.path.join(ROOT, "tests", "cpp", "fake_launch_runtime.c")], check=True)
    out = subprocess.run([sys.executable, "-c", CHILD, fake, ROOT, call], capture_output=True, text=True)
    assert out.returncode == 0, out.stderr
    got = [tuple(int(x) for x in line.split()[:3]) for line in out.stdout.splitlines()]
    assert got == [(0, k * sets, (i + 1) * launches) for i, k in enumerate((1, 2, 2, 2, 3))], out.stdout
