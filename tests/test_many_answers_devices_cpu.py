"""Launchers of the operators for many answers to one prompt on a second device of the process: the library's own code against a stand-in for the runtime's launches
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
b.T, b.nseg, b.n_qtiles, b.max_pages, b.page_len = 40, 2, 2, 8, 64
for name in ("tok_slot", "tok_pos", "seg_start", "seg_len", "seg_slot", "seg_pos0", "block_table", "qt_seg", "qt_off", "seg_tile0"):
    setattr(b, name, at)
def attend(dim, dtype):
    return lib.sllm_seq_attention_shared(C.byref(b), 1, at, at, at, 8 * dim, 8, 2, dim, dim, 0.1, at, at, dtype, 10, at, 1 << 40, None, at, 8 * dim, None, None)
def product(T, n):
    return lib.sllm_seq_linear8(at, 4096, at, at, 4096, at, None, at, n, T, n, 4096, 0, None)
call = {"tokens": lambda: lib.sllm_token_logprobs(at, 128256, 2, 128256, at, at, at, at, 20, at, at, None), "quantise": lambda: lib.sllm_seq_quantise_rows(at, 1, 4096, at, 4096, at, 64, 4096, None),
        "few": lambda: product(2, 4096), "tiles": lambda: product(40, 4096), "pairs": lambda: product(2000, 14336), "shared": lambda: attend(128, 1), "shared_64": lambda: attend(64, 1),
        "shared_f32": lambda: attend(256, 0)}[sys.argv[3]]
for device in (0, 1, 1, 0, 3):
    fake.cudaSetDevice(device)
    rc = call()
    print(rc, fake.fake_sets(), fake.fake_launches(), lib.sllm_last_error())
"""


@pytest.mark.parametrize("call,sets,launches", [("tokens", 0, 1), ("quantise", 0, 1), ("few", 0, 1), ("tiles", 2, 1), ("pairs", 2, 1), ("shared", 1, 2), ("shared_64", 1, 2), ("shared_f32", 1, 2)])
def test_attributes_are_set_on_every_device_once(tmp_path, call, sets, launches):
    if not os.path.exists(LIB):
        pytest.skip("library not built")
    fake = str(tmp_path / "libfake.so")
    subprocess.run(["gcc", "-shared", "-fPIC", "-Wall", "-Werror", "-I/usr/local/cuda/include", "-o", fake, os.path.join(ROOT, "tests", "cpp", "fake_launch_runtime.c")], check=True)
    out = subprocess.run([sys.executable, "-c", CHILD, fake, ROOT, call], capture_output=True, text=True)
    assert out.returncode == 0, out.stderr
    got = [tuple(int(x) for x in line.split()[:3]) for line in out.stdout.splitlines()]
    assert got == [(0, k * sets, (i + 1) * launches) for i, k in enumerate((1, 2, 2, 2, 3))], out.stdout
