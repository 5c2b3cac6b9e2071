"""Sizes that 32 bits do not hold are refused by Context's methods of experts and 8-bit products, not cut off; without a device."""
import pytest

from brimkern_amd.capi import BrikError, BRIK_EINVAL, Context


class Stub(Context):
    """A context whose library calls only count."""

    def __init__(self):
        self.handle, self.calls, self.lib = 1, 0, self

    def __getattr__(self, name):
        if not name.startswith("brik_"):
            raise AttributeError(name)
        def call(*args):
            self.calls += 1
            return 0
        return call

    def close(self):
        pass


CALLS = [
    (lambda c, *s: c.moe_route_args(16, *s, 16, 16), (4, 8, 2)),
    (lambda c, *s: c.moe_sort(16, *s, 16, 16, 16), (4, 2, 8)),
    (lambda c, *s: c.moe_dispatch(16, 16, None, 16, *s), (4, 2, 8)),
    (lambda c, *s: c.moe_combine(16, 16, None, None, 16, *s), (4, 2, 8)),
    (lambda c, *s: c.moe_combine_grad(16, 16, 16, None, 16, 16, *s), (4, 2, 8)),
    (lambda c, *s: c.quantize_i8(16, 16, 16, *s), (4, 64)),
    (lambda c, *s: c.matmul_t_i8(16, 16, 16, 16, 16, *s), (4, 64, 8)),
    (lambda c, *s: c.moe_matmul_t_i8(16, 16, 16, 16, 16, 16, *s[:4], src=16, k=s[4], x_rows=s[5]), (2, 8, 64, 8, 2, 4)),
]


@pytest.mark.parametrize("call,good", CALLS)
def test_refused(call, good):
    c = Stub()
    call(c, *good)
    done = c.calls
    for i in range(len(good)):
        for v in ((1 << 32) + good[i], 1 << 31, -(1 << 31) - 1, (1 << 64) + good[i]):
            with pytest.raises(BrikError) as e:
                call(c, *good[:i], v, *good[i + 1:])
            assert e.value.code == BRIK_EINVAL and c.calls == done
