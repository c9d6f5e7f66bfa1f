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


@pytest.mark.parametrize("compiler,ready,named,last,want", [
    (True, True, None, "ffi_standin", []),                 # the stand-in headers
    (True, False, None, None, []),
    (True, True, "xla", "ffi_standin", ["xla"]),
    (True, True, None, "xla", ["xla"]),                    # built for an XLA that is still there ...
    (True, True, None, "gone", None),                      # ... or not any more: the libraries stay as they are
    (True, False, None, "gone", []),
    (False, True, None, "ffi_standin", None),              # no compiler: ready libraries serve
    (False, True, "xla", None, None),
    (False, False, None, None, RuntimeError),
])
def test_what_build_makes(monkeypatch, tmp_path, compiler, ready, named, last, want):
    import __graft_entry__ as entry

    lib = tmp_path / "lib"
    lib.mkdir()
    header = tmp_path / "xla" / "xla" / "ffi" / "api" / "ffi.h"
    header.parent.mkdir(parents=True)
    header.write_text("")
    for name in entry.LIBRARIES if ready else ():
        (lib / name).write_text("")
    if last is not None:
        (lib / "ffi_root").write_text((last if last == "ffi_standin" else str(tmp_path / last)) + "\n")
    made = []
    monkeypatch.setattr(entry, "LIB", str(lib))
    monkeypatch.setattr(entry, "XLA_ROOT", str(tmp_path / (named or "none")))
    monkeypatch.setattr(entry.shutil, "which", lambda name: "/bin/nvcc" if compiler else None)
    monkeypatch.setattr(entry.subprocess, "check_call", lambda command: made.append([a[len("XLA_ROOT="):] for a in command if a.startswith("XLA_ROOT=")]))
    if want is RuntimeError:
        with pytest.raises(RuntimeError):
            entry._make_libraries()
    else:
        entry._make_libraries()
    assert made == ([] if want in (None, RuntimeError) else [[str(tmp_path / w) for w in want]])
