"""A library of another build is refused on import, by name."""
import os
import subprocess
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.mark.parametrize("version,message", [(6, "ABI version 6"), (7, "lacks")])
def test_a_library_of_another_build_is_refused(tmp_path, version, message):
    src, lib = tmp_path / "old.c", tmp_path / "libold.so"
    src.write_text(f"int didi_version(void) {{ return {version}; }}\n")
    subprocess.run(["gcc", "-shared", "-fPIC", "-o", str(lib), str(src)], check=True)
    r = subprocess.run([sys.executable, "-c", "import didi_amd._lib"], cwd=ROOT, env={**os.environ, "DIDI_HIP_LIB": str(lib)}, capture_output=True, text=True)
    assert r.returncode != 0 and "ImportError" in r.stderr and message in r.stderr, r.stderr
