"""The library, the command-line tools and the self-test build without Python's headers; the Python extension, which needs
them, is built where they are and left out, with a word, where they are not."""
import os
import subprocess
import sys

PKG = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "mbr-cuda-tile_b200")


def _plan(python):
    """What `make all` would run from scratch."""
    r = subprocess.run(["make", "-n", "-B", "-C", PKG, "all", f"PYTHON={python}"], capture_output=True, text=True)
    assert r.returncode == 0, r.stderr
    return r.stdout


def test_make_all_with_and_without_python_headers(tmp_path):
    with_python = _plan(sys.executable)
    assert "binding/stream_calls.c" in with_python
    bare = tmp_path / "python"
    bare.write_text(f"#!/bin/sh\necho {tmp_path}/nowhere\n")
    bare.chmod(0o755)
    for python in (str(bare), str(tmp_path / "missing")):
        plan = _plan(python)
        assert "binding/stream_calls.c" not in plan and "_stream_calls.so" in plan  # the word about it
        for what in ("-o libmbr_b200.so", "tensor_selftest.cpp", "-o cudasep_infer", "-o tensor_bench"):
            assert what in plan and what in with_python
