"""csrc/per_device.h, the numbers that the host asks the driver for once per device
(SMs, resident CTAs and clusters), compiled by itself and asked by a fake."""
import os
import subprocess

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
