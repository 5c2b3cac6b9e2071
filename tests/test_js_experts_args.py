"""Integers of the Node facade's experts and 8-bit products: what 32 bits do not hold, and fractions, are refused, not cut off."""
import json
import os
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
NODE = shutil.which("node")


@pytest.mark.gpu
@pytest.mark.skipif(NODE is None, reason="node not installed")
def test_integers():
    r = subprocess.run([NODE, os.path.join(ROOT, "tests", "js", "experts_integers.js")], cwd=ROOT, capture_output=True, text=True, timeout=100)
    assert r.returncode == 0, r.stdout + r.stderr
    assert json.loads(r.stdout.strip().splitlines()[-1]) == []
