"""The feed-forward operators on the GPU (csrc/ffn_*.cu) against float64, element by element, within the bounds that
tests/ffn_util.py derives. Sizes are the ones where blocks of 64, tiles of 128 x 256 and sums of 256 begin and end."""
import numpy as np
import pytest

from oracle import ffn_ops as ops
from soliton_b200._C import counter, lib
from tests.ffn_util import T, ByteBuf, Out, close, product_bound, ptr
from tests.gpu_util import CUDA, DevBuf, check_ok

pytestmark = [pytest.mark.gpu, pytest.mark.usefixtures("cuda")]

# (m, n, k); three run their forward product, input gradient and weight gradient in pairs of blocks; then rows that several warps hold, and that do not fit registers
SIZES = [(1, 1, 1), (2, 3, 5), (1, 300, 40), (64, 128, 32), (65, 63, 64), (128, 256, 64), (129, 257, 65), (333, 515, 257), (70, 130, 1100), (260, 190, 515), (1700, 1300, 200), (1700, 40, 1300), (40, 1700, 1300), (70, 90, 2500), (20, 30, 6000), (9, 20, 9000)]


def normal(rng, *shape, std=1.0):
    return (rng.standard_normal(shape) * std).astype(np.float32)


def act_bound(kind, pre, d):
    """Of act(pre) when pre is off by d: |act'| <= 1.13, and the function's own fp32 evaluation. GELU: erff and its
    argument's rounding move Phi by 4t at most, the products round three times; SiLU: expf, a sum and a quotient."""
    return 1.13 * d + 12 * T * np.abs(pre) if kind != "none" else d


def check_saved8(buf, pre, d, m, n):
    """A checkpoint of values within d of pre: the step is the least that fits, to within d, and values are within half a
    step and d."""
    q, eb = ops.ck8_unpack(buf, m, n)
    groups = eb.shape[1]
    pad = np.zeros((m, groups * 32))
    pad[:, :n] = np.abs(pre)
    padd = np.zeros((m, groups * 32))
    padd[:, :n] = d
    top, slack = pad.reshape(m, groups, 32).max(-1), padd.reshape(m, groups, 32).max(-1)
    step = np.exp2(eb.astype(np.float64) - 127)
    assert (127 * step >= top - slack).all() and ((63.5 * step <= top + slack) | (eb == 1)).all()
    close(ops.ck8_values(q, eb), pre, np.repeat(step / 2, 32, axis=1)[:, :n] + d, "pre8")


@pytest.mark.parametrize("kind", ["none", "gelu", "silu"])
@pytest.mark.parametrize("m,n,k", SIZES)
def test_linear(m, n, k, kind):
    rng = np.random.default_rng(m * 7 + n * 3 + k)
    x, w = normal(rng, m, k), normal(rng, n, k, std=k ** -0.5)
    bias, res = normal(rng, n), normal(rng, m, n)
    for skew, with_bias, with_res, save, save8 in ((0, 1, 1, 1, 1), (1, 1, 0, 0, 1), (3, 0, 1, 1, 0), (0, 0, 0, 0, 0)):
        want, pre = ops.linear(x, w, bias if with_bias else None, res if with_res else None, kind)
        s = np.abs(x).astype(np.float64) @ np.abs(w.T).astype(np.float64)
        d = product_bound(k, s) + T * np.abs(pre)
        y, p, p8 = Out(m * n, skew), Out(m * n, skew) if save else None, ByteBuf(n=ops.ck8_bytes(m, n), skew=skew) if save8 else None
        bx, bw = DevBuf(x, skew=skew), DevBuf(w, skew=skew)
        bb, br = DevBuf(bias, skew=skew) if with_bias else None, DevBuf(res, skew=skew) if with_res else None
        assert lib.slb_linear(CUDA, bx.ptr, bw.ptr, ptr(bb), ptr(br), y.ptr, ptr(p), ptr(p8), m, n, k, ops.ACTS[kind]) == 0
        check_ok()
        close(y.get(m, n), want, act_bound(kind, pre, d) + (T * np.abs(want) if with_res else 0), "y")
        if save:
            close(p.get(m, n), pre, d, "pre")
        if save8:
            check_saved8(p8.get(), pre, d, m, n)


@pytest.mark.parametrize("held8", [False, True])
@pytest.mark.parametrize("kind", ["none", "gelu", "silu"])
@pytest.mark.parametrize("m,n,k", SIZES)
def test_linear_bwd(m, n, k, kind, held8):
    rng = np.random.default_rng(m + n * 5 + k * 11)
    x, w, dy, pre = normal(rng, m, k), normal(rng, n, k, std=k ** -0.5), normal(rng, m, n, std=1e-3), normal(rng, m, n, std=1.5)
    dy[m - m // 4:] = 0  # padded rows
    bx = bp = bx8 = bp8 = None
    skew = 2 if held8 else 0
    if held8:
        qx, qp = ops.ck8_save(x), ops.ck8_save(pre)
        x, pre = ops.ck8_values(*qx), ops.ck8_values(*qp)
        bx8, bp8 = ByteBuf(ops.ck8_pack(*qx), skew=skew), ByteBuf(ops.ck8_pack(*qp), skew=skew)
    else:
        bx, bp = DevBuf(x, skew=1), DevBuf(pre, skew=1)
    bdy, bw = DevBuf(dy, skew=skew), DevBuf(w, skew=skew)
    dx, dw, db, d = ops.linear_bwd(dy, x, w, pre, kind)
    own = 0 if kind == "none" else 14 * T * np.abs(dy) * (1 + np.abs(pre))  # the derivative's own fp32 evaluation
    a, b, c = Out(m * k, skew), Out(n * k, skew), Out(n, skew)
    assert lib.slb_linear_bwd(CUDA, bdy.ptr, ptr(bx), ptr(bx8), bw.ptr, ptr(bp) if kind != "none" else None, ptr(bp8) if kind != "none" else None,
                              a.ptr, b.ptr, c.ptr, m, n, k, ops.ACTS[kind]) == 0
    check_ok()
    ad, ax, aw = np.abs(d), np.abs(x).astype(np.float64), np.abs(w).astype(np.float64)
    own = np.broadcast_to(own, ad.shape)
    close(a.get(m, k), dx, product_bound(n, ad @ aw) + own @ aw + 1e-45, "dx")
    close(b.get(n, k), dw, product_bound(m, ad.T @ ax) + own.T @ ax + 1e-45, "dw")
    close(c.get(n), db, own.sum(0) + T * (m + 8) * ad.sum(0) + 1e-45, "db")
    first = a.get(m, k).copy(), b.get(n, k).copy(), c.get(n).copy()
    for skip in range(3):  # any two alone, the same bits
        outs = [Out(m * k), Out(n * k), Out(n)]
        outs[skip] = None
        assert lib.slb_linear_bwd(CUDA, bdy.ptr, ptr(bx), ptr(bx8), bw.ptr, ptr(bp) if kind != "none" else None, ptr(bp8) if kind != "none" else None,
                                  *[ptr(o) for o in outs], m, n, k, ops.ACTS[kind]) == 0
        for o, f in zip(outs, first):
            if o is not None:
                np.testing.assert_array_equal(o.get(*f.shape), f)


@pytest.mark.parametrize("kind", ["gelu", "silu", "none"])
@pytest.mark.parametrize("m,n,k", SIZES)
def test_gated(m, n, k, kind):
    rng = np.random.default_rng(m * 3 + n + k)
    x, wg, wu = normal(rng, m, k), normal(rng, n, k, std=k ** -0.5), normal(rng, n, k, std=k ** -0.5)
    bg, bu = normal(rng, n), normal(rng, n)
    bufs = [DevBuf(t, skew=1) for t in (x, wg, wu, bg, bu)]
    for biased in (True, False):
        want, g, u = ops.gated(x, wg, wu, bg if biased else None, bu if biased else None, kind)
        ax = np.abs(x).astype(np.float64)
        dg = product_bound(k, ax @ np.abs(wg.T)) + T * np.abs(g)
        du = product_bound(k, ax @ np.abs(wu.T)) + T * np.abs(u)
        h, og, ou, g8, u8 = Out(m * n), Out(m * n, 1), Out(m * n), ByteBuf(n=ops.ck8_bytes(m, n), skew=3), ByteBuf(n=ops.ck8_bytes(m, n))
        ptrs = [b.ptr for b in bufs]
        if not biased:
            ptrs[3] = ptrs[4] = None
        assert lib.slb_gated(CUDA, *ptrs, h.ptr, og.ptr, ou.ptr, g8.ptr, u8.ptr, m, n, k, ops.ACTS[kind]) == 0
        check_ok()
        ag = act_bound(kind, g, dg)
        close(h.get(m, n), want, ag * (np.abs(u) + du) + np.abs(ops.act(g, kind)) * du + T * np.abs(want), "h")
        close(og.get(m, n), g, dg, "g")
        close(ou.get(m, n), u, du, "u")
        check_saved8(g8.get(), g, dg, m, n)
        check_saved8(u8.get(), u, du, m, n)


@pytest.mark.parametrize("held8", [False, True])
@pytest.mark.parametrize("kind", ["gelu", "silu"])
@pytest.mark.parametrize("m,n,k", SIZES)
def test_gated_bwd(m, n, k, kind, held8):
    rng = np.random.default_rng(m * 13 + n + k * 2)
    x, wg, wu = normal(rng, m, k), normal(rng, n, k, std=k ** -0.5), normal(rng, n, k, std=k ** -0.5)
    g, u, dh = normal(rng, m, n), normal(rng, m, n), normal(rng, m, n, std=1e-3)
    held = [x, g, u]
    if held8:
        qs = [ops.ck8_save(t) for t in held]
        held = [ops.ck8_values(*q) for q in qs]
        full, small = [None] * 3, [ByteBuf(ops.ck8_pack(*q)) for q in qs]
    else:
        full, small = [DevBuf(t) for t in held], [None] * 3
    x, g, u = held
    bdh, bwg, bwu = DevBuf(dh, skew=1), DevBuf(wg), DevBuf(wu)
    dx, dwg, dwu, dbg, dbu, dg, du = ops.gated_bwd(dh, x, wg, wu, g, u, kind)
    outs = [Out(m * k), Out(n * k), Out(n * k, 1), Out(n), Out(n, 1)]

    def call(o):
        assert lib.slb_gated_bwd(CUDA, bdh.ptr, ptr(full[0]), ptr(small[0]), bwg.ptr, bwu.ptr, ptr(full[1]), ptr(full[2]), ptr(small[1]), ptr(small[2]),
                                 *[ptr(t) for t in o], m, n, k, ops.ACTS[kind]) == 0
        check_ok()

    call(outs)
    ax, awg, awu = np.abs(x).astype(np.float64), np.abs(wg).astype(np.float64), np.abs(wu).astype(np.float64)
    eg = 16 * T * np.abs(dh) * np.abs(u) * (1 + np.abs(g))
    eu = 14 * T * np.abs(dh) * np.abs(g)
    # both halves share one scale, and its bound may exceed the true maximum by the tensors' own: below 2^-17 of it the
    # error is absolute, 2^-40 of the bound
    floor = 2.0 ** -38 * np.abs(dh).max() * max(np.abs(u).max(), np.abs(g).max())
    ag, au = np.abs(dg), np.abs(du)
    wants = [(dx, product_bound(2 * n, ag @ awg + au @ awu) + (eg + floor) @ awg + (eu + floor) @ awu),
             (dwg, product_bound(m, ag.T @ ax) + (eg + floor).T @ ax), (dwu, product_bound(m, au.T @ ax) + (eu + floor).T @ ax),
             (dbg, eg.sum(0) + T * (m + 8) * ag.sum(0)), (dbu, eu.sum(0) + T * (m + 8) * au.sum(0))]
    for o, (want, bound), name in zip(outs, wants, ("dx", "dwg", "dwu", "dbg", "dbu")):
        close(o.get(*want.shape), want, bound, name)
    shapes = [(m, k), (n, k), (n, k), (n,), (n,)]
    first = [o.get(*s).copy() for o, s in zip(outs, shapes)]
    for keep in ((1,), (2,), (0, 3), (4,), (1, 2)):
        some = [Out(int(np.prod(s))) if i in keep else None for i, s in enumerate(shapes)]
        call(some)
        for i, (o, f) in enumerate(zip(some, first)):
            if o is None:
                continue
            if i in (1, 2) and not {1, 2} <= set(keep):  # one weight's gradient alone is cut into other slices
                close(o.get(*f.shape), *wants[i])
            else:
                np.testing.assert_array_equal(o.get(*f.shape), f)


@pytest.mark.parametrize("outlier", [None, 3e4, 1e30])
def test_sampled_maxima(outlier):
    """Gradients of tensors large enough to be sampled for their scale, also where the largest value is one that the sample
    (4 KiB in every 64) does not see."""
    m, n, k = 6000, 4500, 72
    rng = np.random.default_rng(17)
    x, w, dy = normal(rng, m, k), normal(rng, n, k, std=0.1), normal(rng, m, n, std=1e-3)
    if outlier is not None:
        dy.reshape(-1)[16384 * 40 + 8000] = outlier
    bx, bw, bdy = DevBuf(x), DevBuf(w), DevBuf(dy)
    a, b, c = Out(m * k), Out(n * k), Out(n)
    before = counter("launches")
    assert lib.slb_linear_bwd(CUDA, bdy.ptr, bx.ptr, None, bw.ptr, None, None, a.ptr, b.ptr, c.ptr, m, n, k, 0) == 0
    check_ok()
    assert counter("launches") - before == 5  # maxima, planes, planes again, column sums, both products
    dx, dw, db, d = ops.linear_bwd(dy, x, w)
    ad, ax, aw = np.abs(d), np.abs(x).astype(np.float64), np.abs(w).astype(np.float64)
    # with one scale for the whole tensor, values below 2^-11 of the largest have an absolute error of 2^-34 of it
    floor = np.full(ad.shape, 2.0 ** -34 * ad.max())
    close(a.get(m, k), dx, product_bound(n, ad @ aw) + floor @ aw, "dx")
    close(b.get(n, k), dw, product_bound(m, ad.T @ ax) + floor.T @ ax, "dw")
    close(c.get(n), db, T * (m + 8) * ad.sum(0), "db")


def test_gated_gradients_with_sampled_maxima():
    m, n, k = 3600, 2500, 136
    rng = np.random.default_rng(18)
    x, wg, wu = normal(rng, m, k), normal(rng, n, k, std=0.1), normal(rng, n, k, std=0.1)
    g, u, dh = normal(rng, m, n), normal(rng, m, n), normal(rng, m, n, std=1e-3)
    u.reshape(-1)[16384 * 30 + 9001] = 5e5
    bufs = [DevBuf(t) for t in (dh, x, wg, wu, g, u)]
    outs = [Out(m * k), Out(n * k), Out(n * k), Out(n), Out(n)]
    bdh, bx, bwg, bwu, bg, bu = (b.ptr for b in bufs)
    assert lib.slb_gated_bwd(CUDA, bdh, bx, None, bwg, bwu, bg, bu, None, None, *[o.ptr for o in outs], m, n, k, ops.ACTS["silu"]) == 0
    check_ok()
    dx, dwg, dwu, dbg, dbu, dg, du = ops.gated_bwd(dh, x, wg, wu, g, u, "silu")
    ax, awg, awu = (np.abs(t).astype(np.float64) for t in (x, wg, wu))
    top = max(np.abs(dg).max(), np.abs(du).max())
    eg = 16 * T * np.abs(dh) * np.abs(u) * (1 + np.abs(g)) + 2.0 ** -34 * top
    eu = 14 * T * np.abs(dh) * np.abs(g) + 2.0 ** -34 * top
    ag, au = np.abs(dg), np.abs(du)
    close(outs[0].get(m, k), dx, product_bound(2 * n, ag @ awg + au @ awu) + eg @ awg + eu @ awu, "dx")
    close(outs[1].get(n, k), dwg, product_bound(m, ag.T @ ax) + eg.T @ ax, "dwg")
    close(outs[2].get(n, k), dwu, product_bound(m, au.T @ ax) + eu.T @ ax, "dwu")
