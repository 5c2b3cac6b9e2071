"""Which rows of a step belong to a sequence, and which buffers overlap, on the host: the functions themselves in a small driver
(tests/native/attn_parts.cpp)."""
import os
import subprocess

HERE = os.path.dirname(os.path.abspath(__file__))


def test_parts(tmp_path):
    exe = str(tmp_path / "attn_parts")
    subprocess.run(["g++", "-O1", "-std=c++17", "-Wall", "-Wextra", "-fsanitize=undefined", "-fno-sanitize-recover=undefined",
                    os.path.join(HERE, "native", "attn_parts.cpp"), "-o", exe], check=True)
    p = subprocess.run([exe], capture_output=True, text=True, timeout=60)
    assert p.returncode == 0 and p.stdout.strip() == "ok", p.stdout + p.stderr
