"""Windows up to the largest integer, which callers take for "no window": the same as none, for rows before the first token, rows
inside a prefix and rows behind it, by every way the keys are divided."""
import numpy as np
import pytest

import kvref as R
from test_gpu_attention import Case, close

pytestmark = pytest.mark.gpu


@pytest.fixture()
def dev(ctx):
    d = R.Dev(ctx)
    yield d
    d.free()


@pytest.mark.parametrize("window", [(1 << 31) - 1, (1 << 31) - 8, 1 << 30])
@pytest.mark.parametrize("seqs", [2, 14])
@pytest.mark.parametrize("prefix", [0, 100])
def test_same_as_none(dev, window, seqs, prefix):
    """A long sequence and others that end just behind, or before, their first own token; 14 of them are shared out."""
    lens = [prefix + n for n in ([1700, 3] + [3 + b for b in range(12)])[:seqs]]
    a = Case(dev, "q8", 16, 16, 64, 32, [8] * seqs, lens, prefix=prefix, window=window, seed=prefix)
    got = a.check()
    a.args.window = 0
    assert np.array_equal(got, a.run())


@pytest.mark.parametrize("fmt", ["q8", "q4"])
def test_many_rows(dev, fmt):
    a = Case(dev, fmt, 4, 2, 64, 16, [150, 300], [100, 380], prefix=70, window=(1 << 31) - 1, seed=2)
    close(a.run(), a.want())
