"""Builds of the library that run at the same time, with a compiler that only writes down what it was told."""
import os
import subprocess
import sys
import time

from falkon_b200 import _lib

NVCC = """#!/bin/sh
out=; inputs=; compile=; flags=
while [ $# -gt 0 ]; do
  case "$1" in
    -o) out=$2; shift ;;
    -c) compile=1 ;;
    -DKIND=*) flags="$flags $1" ;;
    *.o) inputs="$inputs $1" ;;
  esac
  shift
done
if [ -n "$compile" ]; then
  echo "$flags" > "$out"
else
  if [ -n "$HOLD" ]; then
    touch "$HOLD.waits"
    n=0
    while [ ! -e "$HOLD" ] && [ $n -lt 600 ]; do sleep 0.1; n=$((n + 1)); done
  fi
  cat $inputs > "$out"
fi
"""


def test_builds_of_two_libraries_share_no_objects(tmp_path):
    """A build of one library with its own flags, from begin to end between another one's compilation and its link."""
    nvcc = tmp_path / "nvcc"
    nvcc.write_text(NVCC)
    nvcc.chmod(0o755)
    root = os.path.dirname(os.path.dirname(os.path.abspath(_lib.__file__)))

    def start(name, **env):
        env = dict(os.environ, NVCC=str(nvcc), FALKON_B200_LIB=str(tmp_path / f"{name}.so"), FALKON_B200_NVCC_EXTRA=f"-DKIND={name}", **env)
        return subprocess.Popen([sys.executable, "-c", "from falkon_b200 import _lib; _lib.build()"], cwd=root, env=env)

    first = start("first", HOLD=str(tmp_path / "go"))
    for _ in range(1200):
        if (tmp_path / "go.waits").exists() or first.poll() is not None:
            break
        time.sleep(0.1)
    assert start("second").wait(timeout=120) == 0
    (tmp_path / "go").touch()
    assert first.wait(timeout=120) == 0
    units = sum(s.endswith(".cu") for s in _lib.sources())
    for name in ("first", "second"):
        assert (tmp_path / f"{name}.so").read_text().split() == [f"-DKIND={name}"] * units
