"""The keys of an attention tile (csrc/g4_key_span.h), on the CPU: for any window, and for rows at negative
positions, a span inside the cache that holds every key a row sees."""
import os
import shutil
import subprocess

import pytest

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(os.path.dirname(HERE), "gemma4-webgpu-engine_amd", "csrc")


@pytest.mark.skipif(shutil.which("g++") is None, reason="needs g++")
def test_spans_stay_in_the_cache(tmp_path):
    exe = tmp_path / "span_check"
    subprocess.run(["g++", "-std=c++17", "-O1", "-ftrapv", "-Wall", "-Werror", "-I", CSRC,
                    os.path.join(HERE, "key_span_check.cc"), "-o", str(exe)], check=True)
    out = subprocess.run([str(exe)], capture_output=True, text=True)
    assert out.returncode == 0 and out.stdout.strip() == "ok", out.stdout + out.stderr
