"""A library built against the stand-in headers, met by a runtime with frames of another layout."""
import os
import re
import subprocess
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
LIB = os.path.join(ROOT, "xla_b200", "lib")

PROGRAM = """
import ctypes as C, sys
lib = C.CDLL(sys.argv[1])
for name in sys.argv[2:]:
    handler = getattr(lib, name)
    handler.restype, handler.argtypes = C.c_void_p, [C.c_void_p]
    for size in range(8, 512, 8):
        frame = (C.c_uint64 * 64)(size, *[0xdeadbeefdeadbeef] * 63)      # pointers that lead nowhere
        before = bytes(frame)
        assert handler(C.addressof(frame)) is None and bytes(frame) == before, (name, size)
"""


def test_handlers_leave_frames_of_another_layout_alone():
    with open(os.path.join(LIB, "ffi_root")) as f:
        if f.read().strip() != "ffi_standin":
            pytest.skip("built against XLA's own headers")
    header = open(os.path.join(ROOT, "include", "b200_scaled_dot.h")).read()
    names = sorted(set(re.findall(r"\bvoid\* (b200sd_ffi_[a-z0-9_]+)\(void\* call_frame\)", header)))
    assert len(names) == 18
    done = subprocess.run([sys.executable, "-c", PROGRAM, os.path.join(LIB, "libb200_scaled_dot.so"), *names], capture_output=True, text=True)
    assert done.returncode == 0, (done.returncode, done.stderr[-2000:])
    assert "XLA_ROOT" in done.stderr
