"""What the tensor kernel of a chunk's attention does when a wait runs out, which no test
lets happen on a GPU: its own functions, compiled for the host (chunk_host.cpp)."""

import os
import subprocess

import pytest

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(os.path.dirname(HERE), "ffai_b200", "csrc")


def part(name, begin, end):
    text = open(os.path.join(CSRC, name)).read()
    return text[text.index(begin):text.index(end)]


def test_a_call_that_is_left_early_leaves_nothing_behind(tmp_path):
    cuda = os.environ.get("CUDA_HOME", "/usr/local/cuda")
    if not os.path.exists(os.path.join(cuda, "include", "cuda_runtime.h")):
        pytest.skip("no CUDA headers")
    parts = [part("chunk.cuh", "constexpr int kChKeys", "// One row's result"),
             part("chunk_tc.cu", "constexpr int kCtStages", "// ---------------------------------------------------------------- MMA issuers")]
    (tmp_path / "parts.inc").write_text("\n".join(parts))
    exe = tmp_path / "chunk_host"
    subprocess.run(["g++", "-std=c++20", "-O1", "-w", "-pthread", "-I", str(tmp_path), "-I", CSRC,
                    "-I", os.path.join(cuda, "include"), "-o", str(exe), os.path.join(HERE, "chunk_host.cpp")],
                   check=True)
    assert subprocess.run([str(exe)], check=True, capture_output=True, text=True, timeout=300).stdout == ""
