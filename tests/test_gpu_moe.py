"""Routing, sorting, tokens to their experts and back, gradients (brik_moe_*), against plain forms in 64 bits."""
import numpy as np
import pytest

import moeref as R
from brimkern_amd.capi import BrikError, BRIK_EALIGN, BRIK_EINVAL

pytestmark = pytest.mark.gpu


class Dev:
    """Buffers of a test, freed at its end."""

    def __init__(self, ctx):
        self.ctx, self.bufs = ctx, []

    def up(self, a):
        b = self.ctx.upload(np.ascontiguousarray(a)) if np.size(a) else self.ctx.alloc(16)
        self.bufs.append(b)
        return b

    def full(self, shape, value=0, dtype=np.float32):
        return self.up(np.full(shape, value, dtype))

    def get(self, b, shape, dtype=np.float32):
        return self.ctx.download(b, dtype, int(np.prod(shape))).reshape(shape)

    def free(self):
        for b in self.bufs:
            self.ctx.free(b)


@pytest.fixture
def dev(ctx):
    d = Dev(ctx)
    yield d
    d.free()


def run_route(dev, logits, k, bias=None, sort=True, stride=0, E=None, **how):
    T, E = logits.shape[0], E or logits.shape[1]
    n = T * k
    ids, w = dev.full((T, k), 77, np.int32), dev.full((T, k), 9.0)
    made = {}
    if sort:
        made = {"row_off": dev.full(E + 1, 55, np.int32), "src": dev.full(n, 55, np.int32), "slot": dev.full(n, 55, np.int32)}
    args = dev.ctx.moe_route_args(dev.up(logits), T, E, k, ids, w, bias=None if bias is None else dev.up(bias), logit_stride=stride, **made, **how)
    dev.ctx.moe_route(args)
    got = [dev.get(ids, (T, k), np.int32), dev.get(w, (T, k))]
    if sort:
        got += [dev.get(made["row_off"], E + 1, np.int32), dev.get(made["src"], n, np.int32), dev.get(made["slot"], (T, k), np.int32)]
    return got


def check_route(got, logits, k, bias=None, sigmoid=False, renorm=False, scale=1.0):
    E = logits.shape[1]
    ids, w = R.route(logits, k, sigmoid, renorm, scale, bias)
    assert (got[0] == ids).all()
    # exp of a rounded difference, two roundings of exp and of each of the sums, the quotients: an lane's sum has E / 64 terms,
    # the lanes' six more additions; the sums are of one sign
    l = np.where(np.isfinite(logits), logits, 0)
    tol = (float(np.abs(l).max() if l.size else 0) * 2 + E / 64 + 24) * R.HALF
    assert (np.abs(got[1] - w) <= tol * np.abs(w) + 2.0 ** -125 * abs(scale)).all()
    if len(got) > 2:
        for a, b in zip(got[2:], R.sort(ids, E)):
            assert (a == b).all()


HOW = [dict(), dict(renorm=True), dict(sigmoid=True, scale=2.5), dict(sigmoid=True, renorm=True, scale=0.5)]


@pytest.mark.parametrize("how", range(4))
@pytest.mark.parametrize("T,E,k", [(1, 1, 1), (1, 64, 8), (3, 5, 2), (64, 64, 8), (65, 40, 6), (70, 128, 8), (300, 65, 4), (33, 256, 8),
                                   (9, 1000, 64), (5, 1024, 3), (2000, 16, 2)])
def test_route(dev, T, E, k, how):
    logits = (np.random.default_rng(T * E + k).standard_normal((T, E)) * 2).astype(np.float32)
    check_route(run_route(dev, logits, k, **HOW[how]), logits, k, **HOW[how])


@pytest.mark.parametrize("how", range(4))
@pytest.mark.parametrize("T,E,k", [(7, 8, 2), (200, 64, 6), (40, 257, 8), (3, 1024, 9)])
def test_route_with_bias(dev, T, E, k, how):
    rng = np.random.default_rng(T + E)
    logits, bias = (rng.standard_normal((T, E)) * 2).astype(np.float32), (rng.standard_normal(E) * 0.1).astype(np.float32)
    bias[0] = -np.inf                                    # never chosen
    check_route(run_route(dev, logits, k, bias=bias, **HOW[how]), logits, k, bias=bias, **HOW[how])


@pytest.mark.parametrize("E", [1, 20, 300])
@pytest.mark.parametrize("how", range(4))
def test_route_with_bias_at_its_ends(dev, E, how):
    """Biases of NaN and -infinity are never chosen, +infinity always; large ones swallow the scores (as in 64 bits), so ties by lower id;
    a token of which nothing is left, and an infinite logit (a softmax of NaN: nothing to choose)."""
    rng = np.random.default_rng(E)
    logits = rng.standard_normal((40, E)).astype(np.float32)
    logits[5] = -np.inf
    logits[6, ::2] = np.nan
    ends = [np.nan] if E == 1 else [np.nan, np.inf, -np.inf, np.inf, 1e30, 1e30, -1e30, 3e38, -3e38, 2.0 ** 40, 2.0 ** 40, 0.0, -0.0]
    bias = np.resize(np.array(ends, np.float32), E)
    for b in (bias, np.zeros(E, np.float32)):
        check_route(run_route(dev, logits, min(E, 12), bias=b, **HOW[how]), logits, min(E, 12), bias=b, **HOW[how])
    if E > 1 and not HOW[how].get("sigmoid"):
        logits[:, 3] = np.inf
        ids, w = run_route(dev, logits, 4, bias=np.zeros(E, np.float32), **HOW[how])[:2]
        assert (ids == -1).all() and (w == 0).all()


@pytest.mark.parametrize("sort", [True, False])
def test_route_ties_masks_and_strides(dev, sort):
    """Equal logits by lower id; masked experts, NaN, rows with fewer experts than k and with none; rows of a wider buffer."""
    rng = np.random.default_rng(5)
    wide = rng.integers(-2, 3, (90, 75)).astype(np.float32)
    logits = wide[:, :70]
    logits[3] = -np.inf
    logits[4, 5:] = -np.inf
    logits[5, ::2] = np.nan
    logits[6] = np.nan
    logits[7] = -0.0
    logits[7, 10:20] = 0.0
    logits[8] = np.float32(-3.4e38)
    logits[9] = 1.0
    logits[9, 10:20] = np.float32(1.0 + 2.0 ** -23)
    for how in HOW:
        check_route(run_route(dev, wide, 8, sort=sort, stride=75, E=70, **how), logits, 8, **how)


def test_route_extreme_logits(dev):
    """Sigmoids that underflow keep their ratio; an infinite logit is the whole softmax (NaN) and one of the sigmoids."""
    logits = np.full((4, 64), -1000.0, np.float32)
    logits[0, 10], logits[0, 11] = -900, -901
    logits[1] = -120
    logits[2, 3], logits[2, 4] = 500, 499
    logits[3, 7] = np.inf
    got = run_route(dev, logits[:3], 2, sigmoid=True, renorm=True)
    check_route(got, logits[:3], 2, sigmoid=True, renorm=True)
    assert abs(got[1][0, 0] - 1 / (1 + np.exp(-1))) < 1e-6
    ids, w = run_route(dev, logits[3:], 1, sigmoid=True)[:2]
    assert ids[0, 0] == 7 and w[0, 0] == 1
    ids, w = run_route(dev, logits[3:], 1)[:2]
    assert ids[0, 0] == 7 and np.isnan(w[0, 0])


@pytest.mark.parametrize("T,k,E", [(0, 4, 8), (1, 1, 1), (5, 3, 4), (100, 8, 64), (1000, 8, 64), (5000, 2, 1024), (4097, 1, 3), (70000, 1, 16), (20000, 8, 200)])
def test_sort(dev, T, k, E):
    """Assignments from elsewhere: experts of other devices, none, the same one twice, all on one expert."""
    rng = np.random.default_rng(T + E)
    ids = rng.integers(-1, E + 2, (T, k)).astype(np.int32)
    ids[: T // 3] = E - 1
    if T:
        ids[0, 0] = 2 ** 31 - 1
        ids[-1, -1] = -(2 ** 31)
    row_off, src, slot = dev.full(E + 1, 9, np.int32), dev.full(T * k, 9, np.int32), dev.full((T, k), 9, np.int32)
    dev.ctx.moe_sort(dev.up(ids), T, k, E, row_off, src, slot)
    want = R.sort(ids, E) if T else (np.zeros(E + 1, np.int32), np.zeros(0, np.int32), np.zeros((0, k), np.int32))
    assert (dev.get(row_off, E + 1, np.int32) == want[0]).all()
    if T:
        assert (dev.get(src, T * k, np.int32) == want[1]).all() and (dev.get(slot, (T, k), np.int32) == want[2]).all()


def assignments(rng, T, k, E, none=0.2):
    ids = np.stack([rng.permutation(E)[:k] for _ in range(T)]).astype(np.int32) if T else np.zeros((0, k), np.int32)
    ids[rng.random((T, k)) < none] = -1
    return ids


@pytest.mark.parametrize("T,k,width", [(1, 1, 4), (1, 8, 2048), (3, 2, 1028), (64, 8, 768), (257, 4, 260), (40, 6, 8192), (5, 20, 100), (2, 64, 12)])
@pytest.mark.parametrize("weighted", [True, False])
def test_there_and_back(dev, T, k, width, weighted):
    """Rows without an assignment stay as they are; what lies in them (NaN) reaches nothing; out may be res."""
    rng = np.random.default_rng(T * k)
    ids = assignments(rng, T, k, max(k, 16))
    row_off, src, slot = R.sort(ids, max(k, 16))
    n, kept = T * k, int(row_off[-1])
    x, y = rng.standard_normal((T, width)).astype(np.float32), rng.standard_normal((n, width)).astype(np.float32)
    y[kept:] = np.nan
    res, w = rng.standard_normal((T, width)).astype(np.float32), rng.standard_normal((T, k)).astype(np.float32)
    w[slot < 0] = np.nan
    wd, sd, xs, out = dev.up(w) if weighted else None, dev.up(slot), dev.full((n, width), 7.0), dev.up(res)
    dev.ctx.moe_dispatch(dev.up(x), sd, wd, xs, T, k, width)
    dev.ctx.moe_combine(dev.up(y), sd, wd, out, out, T, k, width)
    got = dev.get(xs, (n, width))
    assert (got[kept:] == 7.0).all()
    for r in range(kept):
        t, j = divmod(int(src[r]), k)
        assert (got[r] == (x[t] * w[t, j] if weighted else x[t])).all()
    got, alone = dev.get(out, (T, width)), dev.full((T, width), 3.0)
    dev.ctx.moe_combine(dev.up(y), sd, wd, None, alone, T, k, width)
    alone = dev.get(alone, (T, width))
    for t in range(T):
        rows = [(1.0 if not weighted else float(w[t, j]), y[slot[t, j]].astype(np.float64)) for j in range(k) if slot[t, j] >= 0]
        want, size = sum((a * b for a, b in rows), np.zeros(width)), sum((np.abs(a * b) for a, b in rows), np.zeros(width))
        assert (np.abs(alone[t] - want) <= (k + 1) * R.HALF * size).all()
        assert (np.abs(got[t] - (want + res[t])) <= (k + 2) * R.HALF * (size + np.abs(res[t]))).all()


@pytest.mark.parametrize("T,k,width", [(1, 1, 4), (3, 2, 1028), (64, 8, 768), (5, 20, 100), (2, 9, 8192), (4, 3, 0)])
def test_gradient_of_combine(dev, T, k, width):
    rng = np.random.default_rng(k)
    ids = assignments(rng, T, k, max(k, 16))
    row_off, src, slot = R.sort(ids, max(k, 16))
    n, kept = T * k, int(row_off[-1])
    dout, y = rng.standard_normal((T, width)).astype(np.float32), rng.standard_normal((n, width)).astype(np.float32)
    y[kept:] = np.nan
    w = rng.standard_normal((T, k)).astype(np.float32)
    dy, dw, both = dev.full((n, width), 7.0), dev.full((T, k), 7.0), dev.up(y)
    args = (dev.up(dout), dev.up(slot), dev.up(w))
    dev.ctx.moe_combine_grad(args[0], both, args[1], args[2], dy, dw, T, k, width)
    dev.ctx.moe_combine_grad(args[0], both, args[1], args[2], both, None, T, k, width)     # in place, no weights' gradient
    got, gw = dev.get(dy, (n, width)), dev.get(dw, (T, k))
    assert (got[kept:] == 7.0).all() and (dev.get(both, (n, width))[:kept] == got[:kept]).all()
    for t in range(T):
        for j in range(k):
            r = slot[t, j]
            if r < 0:
                assert gw[t, j] == 0
                continue
            assert (got[r] == dout[t] * w[t, j]).all()
            terms = dout[t].astype(np.float64) * y[r]
            # a thread adds quads one after the other, 4 products each, then 8 levels of the block
            assert abs(gw[t, j] - terms.sum()) <= (4 * (width / 1024 + 1) + 9) * R.HALF * np.abs(terms).sum()


@pytest.mark.parametrize("how", range(4))
@pytest.mark.parametrize("T,E,k", [(1, 1, 1), (9, 40, 4), (30, 64, 8), (5, 130, 3), (4, 1024, 12)])
def test_gradient_of_route(dev, T, E, k, how):
    """Against the chain rule; a place without an expert (and a token without any) has none; against differences of the weights."""
    rng = np.random.default_rng(E)
    h = HOW[how]
    logits = (rng.standard_normal((T, E)) * 1.5).astype(np.float32)
    ids, _ = R.route(logits, k, **h)
    ids[-1, -1] = -1
    dw = rng.standard_normal((T, k)).astype(np.float32)
    dw[-1, -1] = np.nan
    dl = dev.full((T, E), 7.0)
    args = dev.ctx.moe_route_args(dev.up(logits), T, E, k, dev.up(ids), None, **h)
    dev.ctx.moe_route_grad(args, dev.up(dw), dl)
    got = dev.get(dl, (T, E))
    want, size = R.route_grad(logits, ids, np.where(ids >= 0, dw, 0), h.get("sigmoid", False), h.get("renorm", False), h.get("scale", 1.0))
    # both factors of a product have the error of a weight (as in check_route), a sum of k terms and five roundings between; the
    # reference's own 64-bit terms of the experts that were not chosen cancel to some 2^-53 of them, where the formula is 0
    tol = (2 * (2 * float(np.abs(logits).max()) + E / 64 + 24) + k + 5) * R.HALF
    assert (np.abs(got - want) <= tol * size + 2.0 ** -48 * size.max(-1, keepdims=True) + 2.0 ** -120).all()
    if k > 1 or E > 1:
        step, t, e = 1e-6, 0, int(ids[0, 0])
        def loss(d):
            l = logits.astype(np.float64).copy()
            l[t, e] += d
            s = R.scores(l, h.get("sigmoid", False))[t][ids[t]]
            s = np.where(ids[t] >= 0, s, 0)
            return h.get("scale", 1.0) * (np.where(ids[t] >= 0, dw[t], 0) * (s / s.sum() if h.get("renorm") else s)).sum()
        slope = (loss(step) - loss(-step)) / (2 * step)
        assert abs(got[t, e] - slope) <= tol * size[t, e] + 1e-8 * (1 + np.abs(np.where(ids[t] >= 0, dw[t], 0)).sum())


def test_recorded_routing_follows_its_inputs(dev):
    """A captured step: routed, sorted and spread anew at every replay, with eager calls of other sizes between."""
    ctx, rng, T, E, k, H = dev.ctx, np.random.default_rng(1), 200, 64, 8, 256
    n = T * k
    ld, xd = dev.full((T, E)), dev.full((T, H))
    ids, w, off, src, slot = dev.full((T, k), 0, np.int32), dev.full((T, k)), dev.full(E + 1, 0, np.int32), dev.full(n, 0, np.int32), dev.full((T, k), 0, np.int32)
    xs, out = dev.full((n, H)), dev.full((T, H))
    args = ctx.moe_route_args(ld, T, E, k, ids, w, row_off=off, src=src, slot=slot, renorm=True)
    def step():
        ctx.moe_route(args)
        ctx.moe_dispatch(xd, slot, None, xs, T, k, H)
        ctx.moe_combine(xs, slot, w, None, out, T, k, H)
    step()
    ctx.graph_begin()
    step()
    graph = ctx.graph_end()
    for i in range(4):
        logits, x = rng.standard_normal((T, E)).astype(np.float32), rng.standard_normal((T, H)).astype(np.float32)
        logits[i * 7:] = -np.inf if i % 2 else logits[i * 7:]
        ctx.h2d(ld, logits)
        ctx.h2d(xd, x)
        graph.launch()
        check_route([dev.get(ids, (T, k), np.int32), dev.get(w, (T, k)), dev.get(off, E + 1, np.int32), dev.get(src, n, np.int32),
                     dev.get(slot, (T, k), np.int32)], logits, k, renorm=True)
        live = (R.route(logits, k)[0] >= 0).any(1)[:, None]
        assert (np.abs(dev.get(out, (T, H)) - np.where(live, x, 0)) <= (k + 20 + 8) * R.HALF * np.abs(x)).all()
        other = rng.standard_normal((1500, 100)).astype(np.float32)
        check_route(run_route(dev, other, 5), other, 5)
    graph.destroy()


def test_past_32_bits(dev):
    """Sorted rows of more than 2^32 bytes, there and back, and the gradient of that: the last rows."""
    ctx, rng, T, k, H = dev.ctx, np.random.default_rng(5), 33001, 8, 4096
    n, last = T * k, 3
    slot = np.arange(n, dtype=np.int32).reshape(T, k)
    slot[-last:] = slot[-last:, ::-1]
    x, w = rng.standard_normal((last, H)).astype(np.float32), rng.standard_normal((last, k)).astype(np.float32)
    xd, wd, rows, sd = ctx.alloc(4 * T * H), ctx.alloc(4 * n), ctx.alloc(4 * n * H), dev.up(slot)
    out, dw = ctx.alloc(4 * T * H), ctx.alloc(4 * n)                                # (what lies before the last rows does not matter)
    dev.bufs += [xd, wd, rows, out, dw]
    ctx.h2d(xd, x, 4 * (T - last) * H)
    ctx.h2d(wd, w, 4 * (T - last) * k)
    ctx.moe_dispatch(xd, sd, wd, rows, T, k, H)
    got = ctx.download(rows, np.float32, last * k * H, 4 * (n - last * k) * H).reshape(last, k, H)
    want = (w[:, :, None] * x[:, None])[:, ::-1]
    assert (got == want).all()
    ctx.moe_combine(rows, sd, None, None, out, T, k, H)
    back = ctx.download(out, np.float32, last * H, 4 * (T - last) * H).reshape(last, H)
    assert (np.abs(back - want.astype(np.float64).sum(1)) <= k * R.HALF * np.abs(want).sum(1)).all()
    ctx.moe_combine_grad(xd, rows, sd, wd, rows, dw, T, k, H)
    g = ctx.download(dw, np.float32, last * k, 4 * (T - last) * k).reshape(last, k)
    terms = x[:, None].astype(np.float64) * want[:, ::-1]
    # the products and sums of a thread's 16 values, 6 steps over the lanes and 2 over the waves
    assert (np.abs(g - terms.sum(-1)) <= (16 + 6 + 2 + 2) * R.HALF * np.abs(terms).sum(-1)).all()
    assert (ctx.download(rows, np.float32, last * k * H, 4 * (n - last * k) * H).reshape(last, k, H) == want).all()


def test_two_contexts_at_once(dev):
    from brimkern_amd.capi import Context
    rng, T, E, k = np.random.default_rng(2), 3000, 64, 6
    with Context(0) as second:
        d2 = Dev(second)
        logits = [rng.standard_normal((T, E)).astype(np.float32) for _ in range(2)]
        runs = []
        for d, l in zip((dev, d2), logits):
            made = [d.full((T, k), 0, np.int32), d.full((T, k)), d.full(E + 1, 0, np.int32), d.full(T * k, 0, np.int32), d.full((T, k), 0, np.int32)]
            runs.append((d, made, d.ctx.moe_route_args(d.up(l), T, E, k, made[0], made[1], row_off=made[2], src=made[3], slot=made[4])))
        for _ in range(5):
            for d, made, args in runs:
                d.ctx.moe_route(args)
        for (d, made, _), l in zip(runs, logits):
            shapes = [((T, k), np.int32), ((T, k), np.float32), (E + 1, np.int32), (T * k, np.int32), ((T, k), np.int32)]
            check_route([d.get(b, s, t) for b, (s, t) in zip(made, shapes)], l, k)
        d2.free()


def test_refusals(dev):
    ctx = dev.ctx
    b = dev.full(4096)
    good = dict(logits=b, tokens=4, experts=8, k=2, ids=b, weights=b)
    def refused(code, call):
        with pytest.raises(BrikError) as e:
            call()
        assert e.value.code == code
    for bad in (dict(k=9), dict(k=65, experts=100), dict(experts=1025), dict(tokens=-1), dict(k=-1), dict(tokens=1 << 24), dict(logits=None),
                dict(ids=None), dict(weights=None), dict(logit_stride=7), dict(scale=float("nan")), dict(row_off=b), dict(slot=b, src=b)):
        refused(BRIK_EINVAL, lambda: ctx.moe_route(ctx.moe_route_args(**{**good, **bad})))
    for name in ("logits", "ids", "weights", "bias"):
        refused(BRIK_EALIGN, lambda: ctx.moe_route(ctx.moe_route_args(**{**good, name: b.ptr + 2})))
    flags = ctx.moe_route_args(**good)
    flags.flags = 4
    refused(BRIK_EINVAL, lambda: ctx.moe_route(flags))
    args = ctx.moe_route_args(**good)
    refused(BRIK_EINVAL, lambda: ctx.moe_route_grad(args, None, b))
    refused(BRIK_EINVAL, lambda: ctx.moe_route_grad(args, b, None))
    refused(BRIK_EALIGN, lambda: ctx.moe_route_grad(args, b, b.ptr + 1))
    refused(BRIK_EINVAL, lambda: ctx.moe_sort(None, 4, 2, 8, b, b, b))
    refused(BRIK_EINVAL, lambda: ctx.moe_sort(b, 4, 2, 8, None, b, b))
    refused(BRIK_EINVAL, lambda: ctx.moe_sort(b, 4, 2, 8, b, b, None))
    refused(BRIK_EINVAL, lambda: ctx.moe_sort(b, 4, 2, 2000, b, b, b))
    refused(BRIK_EALIGN, lambda: ctx.moe_sort(b, 4, 2, 8, b, b.ptr + 2, b))
    for width in (-4, 6):
        refused(BRIK_EINVAL, lambda: ctx.moe_dispatch(b, b, None, b, 2, 2, width))
    refused(BRIK_EINVAL, lambda: ctx.moe_dispatch(None, b, None, b, 2, 2, 8))
    refused(BRIK_EINVAL, lambda: ctx.moe_combine(b, None, None, None, b, 2, 2, 8))
    refused(BRIK_EINVAL, lambda: ctx.moe_combine(b, b, None, None, None, 2, 2, 8))
    refused(BRIK_EALIGN, lambda: ctx.moe_combine(b, b, None, b.ptr + 4, b, 2, 2, 8))
    refused(BRIK_EINVAL, lambda: ctx.moe_combine_grad(None, b, b, None, b, b, 2, 2, 8))
    refused(BRIK_EINVAL, lambda: ctx.moe_combine_grad(b, None, b, None, b, b, 2, 2, 8))
    refused(BRIK_EALIGN, lambda: ctx.moe_combine_grad(b, b, b, None, b.ptr + 8, b, 2, 2, 8))
    for nothing in (lambda: ctx.moe_route(ctx.moe_route_args(None, 0, 8, 2, None, None)), lambda: ctx.moe_dispatch(None, None, None, None, 0, 2, 8),
                    lambda: ctx.moe_combine(None, b, None, None, None, 2, 2, 0),
                    lambda: ctx.moe_combine_grad(b, b, b, None, None, None, 2, 2, 8)):
        nothing()
