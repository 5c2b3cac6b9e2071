"""Rows quantized to 8 bits and products of 8-bit integers (brik_quantize_i8, brik_matmul_t_i8, brik_moe_matmul_t_i8), against
plain forms in 64 bits, and a whole mixture-of-experts layer of them."""
import numpy as np
import pytest

import moeref as R
from brimkern_amd.capi import BrikError, BRIK_EALIGN, BRIK_EINVAL, BRIK_I8_K, BRIK_OPT_I8_KERNEL, BRIK_OPT_I8_SPLITS
from test_gpu_moe import Dev, dev, run_route        # noqa: F401

pytestmark = pytest.mark.gpu
KERNELS = 12


def run_quantize(dev, x, gate=None, gelu=False, x_stride=0, gate_stride=0, K=None):
    M, K = x.shape[0], K or x.shape[1]
    codes, scales = dev.full((M, K), 99, np.int8), dev.full(M, 99.0)
    dev.ctx.quantize_i8(dev.up(x), codes, scales, M, K, x_stride=x_stride, gate=None if gate is None else dev.up(gate), gate_stride=gate_stride, gelu=gelu)
    return dev.get(codes, (M, K), np.int8), dev.get(scales, M)


@pytest.mark.parametrize("M,K", [(1, 32), (5, 1024), (3, 1056), (2, 4096), (7, 4128), (1, 9728), (2, 16384), (3, 16416), (1, 40000 // 32 * 32), (333, 96)])
def test_quantize(dev, M, K):
    """Codes and scales are those of the formula, ties upward: rows of small integers and halves meet many."""
    rng = np.random.default_rng(K)
    x = (rng.standard_normal((M, K)) * np.exp(3 * rng.standard_normal((M, 1)))).astype(np.float32)
    x[M // 2] = rng.integers(-254, 255, K) / 2.0
    x[M // 2, 0] = -127
    codes, scales = R.quantize(x)
    got = run_quantize(dev, x)
    assert (got[1] == scales).all() and (got[0] == codes).all()


def test_quantize_borders_of_f32(dev):
    """Values next to a border between two codes, a step of f32 to either side of it, for many scales."""
    rng = np.random.default_rng(0)
    rows = []
    for _ in range(400):
        top = np.float32(np.exp(20 * rng.standard_normal()))
        s = np.float32(np.float64(top) / 127)
        at = (s * (rng.integers(-126, 126, 84) + 0.5)).astype(np.float32)
        rows.append(np.concatenate([[top], at, np.nextafter(at, np.float32(np.inf)), np.nextafter(at, np.float32(-np.inf)), [0, -0.0, -top]]))
    x = np.stack(rows).astype(np.float32)
    x = x[:, : x.shape[1] // 32 * 32]
    codes, scales = R.quantize(x)
    got = run_quantize(dev, x)
    assert (got[1] == scales).all() and (got[0] == codes).all()


def test_quantize_special_rows(dev):
    """Zeros, subnormals, rows whose scale leaves the normal range, NaN and infinities."""
    x = np.random.default_rng(1).standard_normal((9, 64)).astype(np.float32)
    x[0] = 0
    x[1] *= np.float32(1e-40)
    x[2] = 0
    x[2, 3] = 127 * 2.0 ** -126
    x[3] = 0
    x[3, 3] = np.float32(126.9 * 2.0 ** -126)
    x[4, 60] = np.nan
    x[5, 0] = np.inf
    x[6, 1] = -np.inf
    x[7] = np.float32(3.4028235e38)
    codes, scales = R.quantize(x)
    got = run_quantize(dev, x)
    assert np.array_equal(got[1], scales, equal_nan=True) and (got[0] == codes).all()
    assert np.isnan(got[1][4:7]).all() and got[1][3] == 0 and got[1][2] == np.float32(2.0 ** -126) and got[0][2, 3] == 127


@pytest.mark.parametrize("gelu", [False, True])
@pytest.mark.parametrize("M,K", [(3, 768), (5, 1536), (2, 9728), (1, 20000 // 32 * 32)])
def test_quantize_with_gate(dev, M, K, gelu):
    """act(gate) * x in 64 bits; gate and up side by side in one buffer."""
    rng = np.random.default_rng(K)
    both = rng.standard_normal((M, 2 * K + 8)).astype(np.float32) * 3
    both[0, :4] = [-1000, 1000, 0, -87]
    h = R.act(both[:, :K], gelu) * both[:, K:2 * K]
    buf = dev.up(both)
    codes, scales = dev.full((M, K), 99, np.int8), dev.full(M, 99.0)
    dev.ctx.quantize_i8(buf.ptr + 4 * K, codes, scales, M, K, x_stride=2 * K + 8, gate=buf, gate_stride=2 * K + 8, gelu=gelu)
    want = R.quantize(h)
    assert (dev.get(scales, M) == want[1]).all() and (dev.get(codes, (M, K), np.int8) == want[0]).all()


def operands(rng, M, K, N):
    x, w = rng.integers(-128, 128, (M, K)).astype(np.int8), rng.integers(-128, 128, (N, K)).astype(np.int8)
    return x, rng.uniform(0.5, 2, M).astype(np.float32), w, (rng.uniform(0.5, 2, N) * 2.0 ** -10).astype(np.float32)


def run_product(dev, x, xs, w, ws, res=None, in_place=False):
    (M, K), N = x.shape, w.shape[0]
    y = dev.up(res) if in_place else dev.full((M, N), 7.0)
    r = None if res is None else y if in_place else dev.up(res)
    dev.ctx.matmul_t_i8(dev.up(x), dev.up(xs), dev.up(w), dev.up(ws), y, M, K, N, res=r)
    return dev.get(y, (M, N))


def close(got, want, bound):
    assert (np.abs(got.astype(np.float64) - want) <= bound).all()


SHAPES = [(1, 32, 1), (1, 2560, 300), (2, 96, 17), (16, 64, 16), (17, 992, 33), (31, 4128, 70), (64, 1024, 130), (65, 288, 129), (100, 2560, 257),
          (300, 160, 513), (257, 64, 300), (520, 1056, 260)]


@pytest.mark.parametrize("M,K,N", SHAPES)
def test_product(dev, M, K, N):
    rng = np.random.default_rng(M + K + N)
    ops = operands(rng, M, K, N)
    res = rng.standard_normal((M, N)).astype(np.float32)
    close(run_product(dev, *ops), *R.product(*ops))
    close(run_product(dev, *ops, res=res), *R.product(*ops, res=res))
    close(run_product(dev, *ops, res=res, in_place=True), *R.product(*ops, res=res))


@pytest.mark.parametrize("kernel", range(1, KERNELS + 1))
@pytest.mark.parametrize("splits", [0, 3])
def test_every_kernel(dev, kernel, splits):
    """Every kernel at sizes that it would not be picked for, with K split over blocks: the same bits."""
    ctx = dev.ctx
    try:
        for M, K, N in ((1, 32, 1), (70, 1120, 45), (300, 96, 290), (33, 4128, 17), (130, 2592, 300)):
            ops = operands(np.random.default_rng(K), M, K, N)
            ctx.set_option(BRIK_OPT_I8_KERNEL, 0)
            ctx.set_option(BRIK_OPT_I8_SPLITS, 0)
            auto = run_product(dev, *ops)
            ctx.set_option(BRIK_OPT_I8_KERNEL, kernel)
            ctx.set_option(BRIK_OPT_I8_SPLITS, splits)
            got = run_product(dev, *ops)
            close(got, *R.product(*ops))
            assert (got == auto).all()
    finally:
        ctx.set_option(BRIK_OPT_I8_KERNEL, 0)
        ctx.set_option(BRIK_OPT_I8_SPLITS, 0)


def test_recorded_products_follow_their_inputs(dev):
    """A captured step with K split over blocks (sums in the context's workspace), replayed with other inputs and smaller calls between;
    after a call that needed a larger workspace the recording is refused."""
    ctx, M, K, N = dev.ctx, 40, 4096, 100
    ops = operands(np.random.default_rng(0), M, K, N)
    x, xs, w, ws, res, y, h = *[dev.up(o) for o in ops], dev.full((M, N)), dev.full((M, N)), dev.full((M, K))
    try:
        ctx.set_option(BRIK_OPT_I8_KERNEL, 9)
        ctx.set_option(BRIK_OPT_I8_SPLITS, 4)
        def step():
            ctx.quantize_i8(h, x, xs, M, K)
            ctx.matmul_t_i8(x, xs, w, ws, y, M, K, N, res=res)
            ctx.matmul_t_i8(x, xs, w, ws, y, M, K, N, res=y)
        step()
        ctx.graph_begin()
        step()
        graph = ctx.graph_end()
        for i in range(4):
            rng = np.random.default_rng(i)
            hv, r = rng.standard_normal((M, K)).astype(np.float32), rng.standard_normal((M, N)).astype(np.float32)
            ctx.h2d(h, hv)
            ctx.h2d(res, r)
            graph.launch()
            codes, scales = R.quantize(hv)
            p, bound = R.product(codes, scales, *ops[2:], res=r)
            want, more = R.product(codes, scales, *ops[2:], res=p)
            close(dev.get(y, (M, N)), want, bound + more + R.HALF * bound)
            small = operands(rng, 3, 512, 60)
            close(run_product(dev, *small), *R.product(*small))
        ctx.set_option(BRIK_OPT_I8_SPLITS, 16)
        large = operands(np.random.default_rng(9), 130, 4096, 1100)
        close(run_product(dev, *large), *R.product(*large))
        with pytest.raises(BrikError) as e:
            graph.launch()
        assert e.value.code == BRIK_EINVAL
        graph.destroy()
    finally:
        ctx.set_option(BRIK_OPT_I8_KERNEL, 0)
        ctx.set_option(BRIK_OPT_I8_SPLITS, 0)


def test_two_contexts_at_once(dev):
    from brimkern_amd.capi import Context
    from test_gpu_moe import Dev
    M, K, N = 200, 4096, 300
    with Context(0) as second:
        d2, runs = Dev(second), []
        for i, d in enumerate((dev, d2)):
            ops = operands(np.random.default_rng(i), M, K, N)
            d.ctx.set_option(BRIK_OPT_I8_SPLITS, 5)
            runs.append((d, ops, [d.up(o) for o in ops], d.full((M, N))))
        try:
            for _ in range(5):
                for d, _, b, y in runs:
                    d.ctx.matmul_t_i8(*b, y, M, K, N)
            for d, ops, _, y in runs:
                close(d.get(y, (M, N)), *R.product(*ops))
        finally:
            dev.ctx.set_option(BRIK_OPT_I8_SPLITS, 0)
            d2.free()


@pytest.mark.parametrize("large", ["x", "y", "y by experts"])
def test_past_32_bits(dev, large):
    """The last rows of operands of more than 2^32 bytes."""
    ctx, rng, last = dev.ctx, np.random.default_rng(3), 20
    M, K, N = (33001, 131040, 9) if large == "x" else (60001, 32, 20000)
    x, xs, w, ws = operands(rng, last, K, N)
    xd, sd, yd = ctx.alloc(M * K), ctx.alloc(4 * M), ctx.alloc(4 * M * N)      # (what lies before the last rows does not matter)
    dev.bufs += [xd, sd, yd]
    ctx.h2d(xd, x, (M - last) * K)
    ctx.h2d(sd, xs, 4 * (M - last))
    if large == "y by experts":
        ctx.moe_matmul_t_i8(xd, sd, dev.up(np.array([0, M - 7, M], np.int32)), dev.up(np.concatenate([w, w[::-1]])), dev.up(np.concatenate([ws, ws[::-1]])),
                            yd, 2, M, K, N)
    else:
        ctx.matmul_t_i8(xd, sd, dev.up(w), dev.up(ws), yd, M, K, N)
    got = ctx.download(yd, np.float32, last * N, 4 * (M - last) * N).reshape(last, N)
    want, bound = R.product(x, xs, w, ws)
    if large == "y by experts":
        want[-7:], bound[-7:] = want[-7:, ::-1].copy(), bound[-7:, ::-1].copy()
    close(got, want, bound)


@pytest.mark.parametrize("M", [1, 100])
def test_largest_sums(dev, M):
    """K at its limit with all codes -128: the largest sum that 31 bits hold."""
    x, w = np.full((M, BRIK_I8_K), -128, np.int8), np.full((3, BRIK_I8_K), -128, np.int8)
    w[1] = 127
    xs, ws = np.full(M, 0.5, np.float32), np.array([1, 2, 0.25], np.float32)
    got = run_product(dev, x, xs, w, ws)
    sums = np.array([16384 * BRIK_I8_K, -16256 * BRIK_I8_K, 16384 * BRIK_I8_K])
    assert (got == (sums.astype(np.float32) * ws * np.float32(0.5))[None]).all()


def test_no_sum_and_special_scales(dev):
    """K = 0 gives res or 0; zero, NaN and infinite scales act on their rows and channels alone."""
    ctx = dev.ctx
    res, y = np.arange(12, dtype=np.float32).reshape(3, 4), dev.full((3, 4), 7.0)
    one = dev.full(8, 1.0)
    ctx.matmul_t_i8(None, one, None, one, y, 3, 0, 4, res=dev.up(res))
    assert (dev.get(y, (3, 4)) == res).all()
    ctx.matmul_t_i8(None, one, None, one, y, 3, 0, 4)
    assert (dev.get(y, (3, 4)) == 0).all()
    for M in (3, 80):
        x, xs, w, ws = operands(np.random.default_rng(3), M, 64, 20)
        xs[0], xs[1], ws[5] = np.nan, 0, np.nan
        got = run_product(dev, x, xs, w, ws)
        assert np.isnan(got[0]).all() and np.isnan(got[:, 5]).all()
        keep = [n for n in range(20) if n != 5]
        assert (got[1, keep] == 0).all()
        close(got[2:, keep], *R.product(x[2:], xs[2:], w[keep], ws[keep]))


def expert_rows(rng, E, rows, empty=0.3):
    """row_off of `rows` rows: some experts without any, one with many."""
    p = rng.random(E) ** 3 * (rng.random(E) > empty)
    p[rng.integers(E)] += 1
    return np.concatenate([[0], np.cumsum(rng.multinomial(rows, p / p.sum()))]).astype(np.int32)


@pytest.mark.parametrize("E,rows,K,N", [(1, 5, 64, 20), (4, 1, 96, 33), (8, 64, 2048, 130), (64, 300, 160, 70), (5, 700, 96, 257), (3, 1000, 1056, 140),
                                        (130, 40, 64, 16), (200, 3000, 64, 48)])
@pytest.mark.parametrize("gather", [True, False])
def test_by_experts(dev, E, rows, K, N, gather):
    """Rows behind the last expert's, and rows whose assignment names no row of x, are left as they are."""
    rng = np.random.default_rng(E + rows)
    behind, k = 3, 4
    off = expert_rows(rng, E, rows)
    n = rows + behind
    x_rows = -(-n // k) if gather else n
    x, xs = rng.integers(-128, 128, (x_rows, K)).astype(np.int8), rng.uniform(0.5, 2, x_rows).astype(np.float32)
    w, ws = rng.integers(-128, 128, (E, N, K)).astype(np.int8), rng.uniform(0.5, 2, (E, N)).astype(np.float32)
    src = rng.permutation(x_rows * k)[:n].astype(np.int32)
    src[rows // 2] = -1
    src[-behind - 1] = x_rows * k + 5
    y = dev.full((n, N), 7.0)
    dev.ctx.moe_matmul_t_i8(dev.up(x), dev.up(xs), dev.up(off), dev.up(w), dev.up(ws), y, E, n, K, N, src=dev.up(src) if gather else None,
                            k=k, x_rows=x_rows)
    got = dev.get(y, (n, N))
    assert (got[rows:] == 7.0).all()
    for e in range(E):
        for r in range(off[e], off[e + 1]):
            t = int(src[r]) // k if gather else r
            if gather and not 0 <= src[r] < x_rows * k:
                assert (got[r] == 7.0).all()
                continue
            close(got[r:r + 1], *R.product(x[t:t + 1], xs[t:t + 1], w[e], ws[e]))


@pytest.mark.parametrize("kernel", range(1, KERNELS + 1))
def test_every_kernel_by_experts(dev, kernel):
    rng, E, rows, K, N = np.random.default_rng(kernel), 6, 500, 1120, 150
    off = expert_rows(rng, E, rows)
    x, xs = rng.integers(-128, 128, (rows, K)).astype(np.int8), rng.uniform(0.5, 2, rows).astype(np.float32)
    w, ws = rng.integers(-128, 128, (E, N, K)).astype(np.int8), rng.uniform(0.5, 2, (E, N)).astype(np.float32)
    y = dev.full((rows, N), 7.0)
    try:
        dev.ctx.set_option(BRIK_OPT_I8_KERNEL, kernel)
        dev.ctx.moe_matmul_t_i8(dev.up(x), dev.up(xs), dev.up(off), dev.up(w), dev.up(ws), y, E, rows, K, N)
    finally:
        dev.ctx.set_option(BRIK_OPT_I8_KERNEL, 0)
    got = dev.get(y, (rows, N))
    for e in range(E):
        a, b = off[e], off[e + 1]
        close(got[a:b], *R.product(x[a:b], xs[a:b], w[e], ws[e]))


def test_malformed_offsets_stay_inside(dev):
    """Offsets that decrease, are negative or pass the rows: their rows are cut off, nothing else is written."""
    rng, E, rows, K, N = np.random.default_rng(4), 4, 40, 64, 32
    x, xs, w, ws = (rng.integers(-128, 128, (rows, K)).astype(np.int8), np.ones(rows, np.float32), rng.integers(-128, 128, (E, N, K)).astype(np.int8),
                    np.ones((E, N), np.float32))
    for kernel in (1, 10, 12):
        y = dev.full((rows + 8, N), 7.0)
        dev.ctx.set_option(BRIK_OPT_I8_KERNEL, kernel)
        try:
            dev.ctx.moe_matmul_t_i8(dev.up(x), dev.up(xs), dev.up(np.array([-5, 10, 3, 20, 1000], np.int32)), dev.up(w), dev.up(ws), y, E, rows, K, N)
        finally:
            dev.ctx.set_option(BRIK_OPT_I8_KERNEL, 0)
        got = dev.get(y, (rows + 8, N))
        assert (got[rows:] == 7.0).all()
        close(got[20:rows], *R.product(x[20:], xs[20:], w[3], ws[3]))


@pytest.mark.parametrize("T", [1, 40, 700])
def test_a_layer(dev, T):
    """Routing, gate and up projections of tokens quantized once, SwiGLU into 8 bits, down projections, back onto the residual: each
    step against the formula on what the step before it gave, eager and recorded."""
    ctx, rng, E, k, H, F = dev.ctx, np.random.default_rng(T), 16, 4, 256, 96
    n = T * k
    wgu, wd = (rng.standard_normal(s).astype(np.float32) for s in ((E, 2 * F, H), (E, H, F)))
    weights = []
    for v in (wgu, wd):
        codes, scales = dev.full(v.shape, 0, np.int8), dev.full(v.shape[:2])
        ctx.quantize_i8(dev.up(v), codes, scales, v.shape[0] * v.shape[1], v.shape[2])
        weights.append((codes, scales, dev.get(codes, v.shape, np.int8), dev.get(scales, v.shape[:2])))
        want = R.quantize(v.reshape(-1, v.shape[2]))
        assert (weights[-1][2].reshape(want[0].shape) == want[0]).all() and (weights[-1][3].ravel() == want[1]).all()
    ld, xd = dev.full((T, E)), dev.full((T, H))
    ids, rw, off, src, slot = dev.full((T, k), 0, np.int32), dev.full((T, k)), dev.full(E + 1, 0, np.int32), dev.full(n, 0, np.int32), dev.full((T, k), 0, np.int32)
    xc, xsc, gu, hc, hs, ys, out = (dev.full((T, H), 0, np.int8), dev.full(T), dev.full((n, 2 * F)), dev.full((n, F), 0, np.int8), dev.full(n),
                                    dev.full((n, H)), dev.full((T, H)))
    args = ctx.moe_route_args(ld, T, E, k, ids, rw, row_off=off, src=src, slot=slot, renorm=True)

    def step():
        ctx.moe_route(args)
        ctx.quantize_i8(xd, xc, xsc, T, H)
        ctx.moe_matmul_t_i8(xc, xsc, off, weights[0][0], weights[0][1], gu, E, n, H, 2 * F, src=src, k=k)
        ctx.quantize_i8(gu.ptr + 4 * F, hc, hs, n, F, x_stride=2 * F, gate=gu, gate_stride=2 * F)
        ctx.moe_matmul_t_i8(hc, hs, off, weights[1][0], weights[1][1], ys, E, n, F, H)
        ctx.moe_combine(ys, slot, rw, xd, out, T, k, H)

    step()
    ctx.graph_begin()
    step()
    graph = ctx.graph_end()
    for i in range(3):
        logits, x = rng.standard_normal((T, E)).astype(np.float32), rng.standard_normal((T, H)).astype(np.float32)
        if i == 2:
            logits[T // 2:] = -np.inf                    # padding
        ctx.h2d(ld, logits)
        ctx.h2d(xd, x)
        step() if i == 0 else graph.launch()
        want_ids, want_w = R.route(logits, k, renorm=True)
        ro, so, sl = R.sort(want_ids, E)
        assert (dev.get(ids, (T, k), np.int32) == want_ids).all() and (dev.get(off, E + 1, np.int32) == ro).all()
        assert (dev.get(src, n, np.int32) == so).all() and (dev.get(slot, (T, k), np.int32) == sl).all()
        c, s = R.quantize(x)
        assert (dev.get(xc, (T, H), np.int8) == c).all() and (dev.get(xsc, T) == s).all()
        kept = int(ro[-1])
        g, hq, hsc, y = dev.get(gu, (n, 2 * F)), dev.get(hc, (n, F), np.int8), dev.get(hs, n), dev.get(ys, (n, H))
        want = R.quantize(R.act(g[:kept, :F]) * g[:kept, F:])
        assert (hq[:kept] == want[0]).all() and (hsc[:kept] == want[1]).all()
        for e in range(E):
            a, b = ro[e], ro[e + 1]
            if a < b:
                t = so[a:b] // k
                close(g[a:b], *R.product(c[t], s[t], weights[0][2][e], weights[0][3][e]))
                close(y[a:b], *R.product(hq[a:b], hsc[a:b], weights[1][2][e], weights[1][3][e]))
        wr, o = dev.get(rw, (T, k)).astype(np.float64), dev.get(out, (T, H))
        terms = np.where(sl[..., None] >= 0, wr[..., None] * y[np.maximum(sl, 0)].astype(np.float64), 0)
        close(o, x + terms.sum(1), (k + 2) * R.HALF * (np.abs(x) + np.abs(terms).sum(1)))
    graph.destroy()


def test_experts_of_q4(dev):
    """The 4-bit experts' product on rows that brik_moe_route sorted and brik_moe_dispatch laid out, some tokens without experts."""
    import oracle as O
    from helpers import PLANES, componentwise_ok, moe_oracle_abs, normwise_rel
    ctx, rng, T, E, k, K, N = dev.ctx, np.random.default_rng(8), 50, 8, 2, 256, 96
    t = dict(zip(PLANES["q4"], O.quantize_q4(rng.standard_normal(E * N * K).astype(np.float32))))
    planes = [dev.up(t[p]) for p in PLANES["q4"]]
    logits, x = rng.standard_normal((T, E)).astype(np.float32), rng.standard_normal((T, K)).astype(np.float32)
    logits[7:9] = -np.inf
    ids, w, off, src, slot = run_route(dev, logits, k, renorm=True)
    rows, kept = T * k, int(off[-1])
    xs, ys, out = dev.full((rows, K)), dev.full((rows, N), np.nan), dev.full((T, N))
    sd = dev.up(slot)
    ctx.moe_dispatch(dev.up(x), sd, None, xs, T, k, K)
    ctx.moe_matmul_t_q4(xs, dev.up(off), *planes, ys, E, rows, K, N)
    ctx.moe_combine(ys, sd, dev.up(w), None, out, T, k, N)
    y, den = moe_oracle_abs(x[src[:kept] // k], off, t, E, K, N)
    got = dev.get(ys, (rows, N))
    assert normwise_rel(got[:kept], y) <= 1e-3 and componentwise_ok(got[:kept], y, den)
    o = dev.get(out, (T, N))
    assert (o[7:9] == 0).all()
    for a in range(T):
        if 7 <= a < 9:
            continue
        want = sum(float(w[a, j]) * got[slot[a, j]].astype(np.float64) for j in range(k))
        assert (np.abs(o[a] - want) <= 4 * R.HALF * sum(np.abs(w[a, j] * got[slot[a, j]]) for j in range(k))).all()


def test_fewer_rows_than_assignments_of_q4(dev):
    """Few rows of 4-bit experts, some assignments without one: the rows of the others are those of a call without them, bit for bit
    (the sizes that choose the kernel are the same)."""
    import oracle as O
    from helpers import PLANES
    ctx, rng, T, E, k, K, N = dev.ctx, np.random.default_rng(4), 12, 4, 2, 2048, 160
    t = dict(zip(PLANES["q4"], O.quantize_q4(rng.standard_normal(E * N * K).astype(np.float32))))
    planes = [dev.up(t[p]) for p in PLANES["q4"]]
    x = rng.standard_normal((T * k, K)).astype(np.float32)
    off = np.array([0, 5, 5, 9, 14], np.int32)
    full = off.copy()
    full[-1] = T * k
    out = []
    for o, rest in ((off, np.nan), (full, 0.5)):
        x[off[-1]:] = rest
        y = dev.full((T * k, N))
        ctx.moe_matmul_t_q4(dev.up(x), dev.up(o), *planes, y, E, T * k, K, N)
        out.append(dev.get(y, (T * k, N))[: off[-1]])
    assert np.isfinite(out[0]).all() and (out[0] == out[1]).all()


def test_refusals(dev):
    ctx, b = dev.ctx, dev.full(4096)
    def refused(code, call):
        with pytest.raises(BrikError) as e:
            call()
        assert e.value.code == code
    for bad in ((2, 33), (2, -32), (-1, 32), (1 << 22, 32)):
        refused(BRIK_EINVAL, lambda: ctx.quantize_i8(b, b, b, *bad))
    for bad in (dict(x_stride=48), dict(x_stride=66), dict(gate=b, gate_stride=32)):
        refused(BRIK_EINVAL, lambda: ctx.quantize_i8(b, b, b, 2, 64, **bad))
    refused(BRIK_EINVAL, lambda: ctx.quantize_i8(None, b, b, 2, 64))
    refused(BRIK_EINVAL, lambda: ctx.quantize_i8(b, b, None, 2, 64))
    refused(BRIK_EALIGN, lambda: ctx.quantize_i8(b.ptr + 4, b, b, 2, 64))
    refused(BRIK_EALIGN, lambda: ctx.quantize_i8(b, b.ptr + 8, b, 2, 64))
    for M, K, N in ((-1, 64, 4), (2, 33, 4), (2, BRIK_I8_K + 32, 4), (2, 64, -1), (1, 65536, 65536)):
        refused(BRIK_EINVAL, lambda: ctx.matmul_t_i8(b, b, b, b, b, M, K, N))
    for i in range(5):
        args = [b] * 5
        args[i] = None
        refused(BRIK_EINVAL, lambda: ctx.matmul_t_i8(*args, 2, 64, 4))
    refused(BRIK_EALIGN, lambda: ctx.matmul_t_i8(b.ptr + 4, b, b, b, b, 2, 64, 4))
    refused(BRIK_EALIGN, lambda: ctx.matmul_t_i8(b, b, b, b, b.ptr + 2, 2, 64, 4))
    refused(BRIK_EINVAL, lambda: ctx.moe_matmul_t_i8(b, b, None, b, b, b, 2, 4, 64, 4))
    refused(BRIK_EINVAL, lambda: ctx.moe_matmul_t_i8(b, b, b, b, b, b, -2, 4, 64, 4))
    refused(BRIK_EINVAL, lambda: ctx.moe_matmul_t_i8(b, b, b, b, b, b, 2, 4, 64, 4, src=b, k=0, x_rows=2))
    refused(BRIK_EINVAL, lambda: ctx.moe_matmul_t_i8(b, b, b, b, b, b, 2, 4, 64, 4, x_rows=3))
    ctx.matmul_t_i8(None, None, None, None, None, 0, 64, 4)
    ctx.moe_matmul_t_i8(None, None, None, None, None, None, 2, 0, 64, 4)
    ctx.moe_matmul_t_i8(None, None, b, b, b, b, 2, 4, 64, 4, src=b, k=2, x_rows=0)
    ctx.quantize_i8(None, None, None, 0, 64)
