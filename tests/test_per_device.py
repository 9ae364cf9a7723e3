"""csrc/per_device.h, the numbers that the host asks the driver for once per device
(SMs, resident CTAs and clusters), compiled by itself and asked by a fake."""
import os
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(ROOT, "i.sam3.opencl_b200", "csrc")


def build(tmp_path, name, *flags):
    exe = str(tmp_path / name)
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Wextra", "-Werror", *flags, "-I" + CSRC,
                    os.path.join(ROOT, "tests", "c", name + ".cc"), "-o", exe], check=True, capture_output=True, text=True)
    return exe


def test_a_failed_question_is_asked_again(tmp_path):
    r = subprocess.run([build(tmp_path, "per_device")], capture_output=True, text=True, timeout=60)
    assert r.returncode == 0, r.stdout


def test_threads_ask_at_the_same_time(tmp_path):
    """Under ThreadSanitizer where the compiler has it."""
    (tmp_path / "empty.cc").write_text("int main() { return 0; }\n")
    empty = str(tmp_path / "empty")
    has = subprocess.run(["g++", "-fsanitize=thread", empty + ".cc", "-o", empty], capture_output=True).returncode == 0
    if not has or subprocess.run([empty], capture_output=True, timeout=60).returncode != 0:
        pytest.skip("no ThreadSanitizer here")
    r = subprocess.run([build(tmp_path, "per_device_threads", "-fsanitize=thread", "-g", "-pthread")], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0, r.stdout + r.stderr[-3000:]
