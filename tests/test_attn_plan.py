"""How attention is divided over the device: the grid, the splits and the workspace for some thousand batches, on the host (the
functions that the entry point calls, in tests/native/attn_plan.cpp)."""
import os
import subprocess

HERE = os.path.dirname(os.path.abspath(__file__))


def test_grids_and_workspaces(tmp_path):
    exe = str(tmp_path / "attn_plan")
    subprocess.run(["g++", "-O2", "-std=c++17", "-Wall", "-Wextra", "-fsanitize=undefined", "-fno-sanitize-recover=undefined",
                    os.path.join(HERE, "native", "attn_plan.cpp"), "-o", exe], check=True)
    p = subprocess.run([exe], capture_output=True, text=True, timeout=120)
    assert p.returncode == 0 and p.stdout.strip() == "ok", p.stdout + p.stderr
