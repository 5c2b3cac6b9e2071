"""Engine.kv_cache over a stand-in for the device context."""
import pytest

from brimkern_amd.capi import BrikError, BRIK_ENOMEM
from brimkern_amd.engine import Engine


class Stub:
    def __init__(self, left):
        self.left, self.freed = left, []

    def alloc(self, n):
        if self.left == 0:
            raise BrikError(BRIK_ENOMEM, "out of memory")
        self.left -= 1
        return n

    def free(self, b):
        self.freed.append(b)


def test_second_allocation_fails():
    """The first buffer goes back, and the error is the allocation's."""
    eng = Engine.__new__(Engine)
    eng.ctx = Stub(1)
    with pytest.raises(BrikError) as e:
        eng.kv_cache("q4", 2, 64, 16, 4)
    assert e.value.code == BRIK_ENOMEM and len(eng.ctx.freed) == 1
