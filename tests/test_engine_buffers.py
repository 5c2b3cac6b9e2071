"""What the engine's methods allocate goes back when they raise, whatever they raise; over a stand-in for the library."""
import pytest

from brimkern_amd.capi import BrikError, BRIK_EINVAL, Context, DeviceBuffer
from brimkern_amd.engine import Engine, QWeight


class Stub(Context):
    """A context whose calls all fail with `error`, or do nothing; it counts the buffers that are out."""

    def __init__(self, error=None):
        self.error, self.out, self.handle = error, [], 1
        self.lib = self

    def __getattr__(self, name):
        if not name.startswith("brik_"):
            raise AttributeError(name)
        def call(*args):
            if self.error:
                raise self.error
            return 0
        return call

    def alloc(self, n):
        self.out.append(DeviceBuffer(self, 4096 * (len(self.out) + 1), n))
        return self.out[-1]

    def upload(self, a):
        return self.alloc(a.nbytes)

    def free(self, b):
        self.out.remove(b)

    def close(self):
        pass


X = {"i8": 16, "isc": 32}
W8 = QWeight(codes=16, sc=32)
CALLS = {
    "moe_route": lambda e, **how: e.moe_route(16, 4, 8, 2, **how),
    "quantize_i8": lambda e, **how: e.quantize_i8(16, 4, 64, **how),
    "mm_i8": lambda e, **how: e.mm_i8(X, how.get("w", X), 4, 64, 8),
    "quantize": lambda e, **how: e.quantize("q8", how.get("src", 16), 512),
    "conv2d": lambda e, **how: e.conv2d(16, W8, how.get("bias"), 1, 4, 4, 1, 3, 3, 1, 1),
}
WRONG = {"moe_route": dict(renormalize=True), "quantize_i8": dict(act="gelu"), "mm_i8": dict(w={"codes": 16}), "quantize": dict(src="no address"),
         "conv2d": dict(bias="no bias")}


@pytest.mark.parametrize("name", CALLS)
def test_buffers_go_back(name):
    for error in (BrikError(BRIK_EINVAL, "refused"), TypeError("no such argument"), KeyboardInterrupt()):
        eng = Engine.__new__(Engine)
        eng.ctx = Stub(error)
        with pytest.raises(type(error)):
            CALLS[name](eng)
        assert eng.ctx.out == []
    eng.ctx = Stub()
    with pytest.raises((TypeError, KeyError, ValueError)):
        CALLS[name](eng, **WRONG[name])
    assert eng.ctx.out == []
    CALLS[name](eng)
    assert len(eng.ctx.out) == 1
