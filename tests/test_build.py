"""What a build makes again, with compilers that only note what they were asked for."""
import os
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(ROOT, "xla_b200", "csrc")
OF_THE_FFI_LAYER = {"ffi_handlers.o", "libb200_mock_ffi.so", "libb200_scaled_dot.so"}


@pytest.fixture
def make(tmp_path):
    """Runs the Makefile into a folder of its own and returns the names of the files that it made."""
    compiler, log = tmp_path / "cc", tmp_path / "log"
    compiler.write_text(f'''#!/bin/sh
while [ $# -gt 0 ]; do
  if [ "$1" = -o ]; then touch "$2"; basename "$2" >> {log}; fi
  shift
done
''')
    compiler.chmod(0o755)

    def run(*args, status=0):
        log.write_text("")
        done = subprocess.run(["make", "-C", CSRC, "-j4", f"OUT={tmp_path}/lib", f"NVCC={compiler}", f"CXX={compiler}", "all", *args],
                              env={k: v for k, v in os.environ.items() if k != "XLA_ROOT"}, capture_output=True, text=True)
        assert done.returncode == status, done.stdout + done.stderr
        return set(log.read_text().split())

    return run


def test_other_ffi_headers_rebuild_what_includes_them(make, tmp_path):
    xla = tmp_path / "xla_checkout"
    shutil.copytree(os.path.join(CSRC, "ffi_standin", "xla"), xla / "xla")
    assert OF_THE_FFI_LAYER < make()
    assert make() == set()
    assert make(f"XLA_ROOT={xla}") == OF_THE_FFI_LAYER
    assert make(f"XLA_ROOT={xla}") == set()
    header = xla / "xla" / "ffi" / "api" / "ffi.h"
    os.utime(header, (os.path.getmtime(tmp_path / "lib" / "libb200_mock_ffi.so") + 5,) * 2)
    assert make(f"XLA_ROOT={xla}") == OF_THE_FFI_LAYER
    os.utime(header, (0, 0))
    make(f"XLA_ROOT={tmp_path}/none", status=2)
    assert make(f"XLA_ROOT={xla}") == set()
    assert make() == OF_THE_FFI_LAYER
    assert make() == set()
