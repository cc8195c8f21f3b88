"""Workspaces of the stream handle that means another stream in every thread
(hipStreamPerThread), on the CPU: tests/native/pool_threads.cpp under
ThreadSanitizer and AddressSanitizer."""
import os
import shutil
import subprocess

import pytest

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(os.path.dirname(HERE), "rusty_whisper_amd", "csrc")


@pytest.mark.skipif(shutil.which("g++") is None, reason="needs g++")
@pytest.mark.parametrize("sanitizer", ["thread", "address"])
def test_a_buffer_per_thread(tmp_path, sanitizer):
    exe = str(tmp_path / f"pool_threads_{sanitizer}")
    subprocess.run(["g++", "-std=c++17", "-O1", "-g", f"-fsanitize={sanitizer}", f"-I{CSRC}",
                    os.path.join(HERE, "native", "pool_threads.cpp"), "-o", exe, "-pthread"], check=True)
    r = subprocess.run([exe], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0 and "bad=0 live=0" in r.stdout, r.stdout + r.stderr
    assert "WARNING: ThreadSanitizer" not in r.stderr


def test_the_library_keys_that_handle_by_thread():
    """In the one function that all entries without a caller workspace use."""
    src = open(os.path.join(CSRC, "rw_rocm.hip")).read()
    body = src[src.index("static int stream_workspace("):]
    body = body[: body.index("\n}\n")]
    assert "hipStreamPerThread" in body and "ThreadNumber::mine()" in body
    assert src.count("ws_pool().acquire(") == 1
