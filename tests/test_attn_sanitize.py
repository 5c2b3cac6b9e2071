"""The attention side's entry points under AddressSanitizer and UndefinedBehaviorSanitizer (host code): tests/native/attn_sanitize,
built by brimkern_amd/build.py. A sanitizer report aborts the driver."""
import os
import subprocess

import pytest

DRIVER = os.path.join(os.path.dirname(os.path.abspath(__file__)), "native", "attn_sanitize")


def run(*args, timeout):
    assert os.path.exists(DRIVER), f"{DRIVER} is missing: run `python -m brimkern_amd.build`"
    p = subprocess.run([DRIVER, *args], capture_output=True, text=True, timeout=timeout)
    out = p.stdout + p.stderr
    print(out[-4000:], flush=True)
    assert p.returncode == 0 and "ERROR: AddressSanitizer" not in out and "runtime error" not in out, out[-4000:]
    return out


def test_without_a_device():
    assert "host checks only (no device): 0 failure(s)" in run("nodev", timeout=120)


@pytest.mark.gpu
def test_on_the_gpu():
    print("attn_sanitize: device run", flush=True)
    assert "device checks done: 0 failure(s)" in run(timeout=110)
