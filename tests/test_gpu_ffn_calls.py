"""The feed-forward and checkpoint entry points as they may be called: no rows, non-finite and extreme values, results
written over the residual, offsets beyond 32 bits, scratch from the caller, copies on other streams, two calls in a row."""
import ctypes as C

import numpy as np
import pytest

from oracle import ffn_ops as ops
from soliton_b200._C import counter, lib, set_option
from tests.ffn_util import T, ByteBuf, Out, close, product_bound
from tests.gpu_util import CUDA, DevBuf, check_ok

pytestmark = [pytest.mark.gpu, pytest.mark.usefixtures("cuda")]


def normal(rng, *shape, std=1.0):
    return (rng.standard_normal(shape) * std).astype(np.float32)


def linear(x, w, bias=None, act=0):
    m, k = x.shape
    n = w.shape[0]
    bx, bw, bb = DevBuf(x), DevBuf(w), None if bias is None else DevBuf(bias)
    out = Out(m * n)
    assert lib.slb_linear(CUDA, bx.ptr, bw.ptr, None if bb is None else bb.ptr, None, out.ptr, None, None, m, n, k, act) == 0
    check_ok()
    return out.get(m, n)


def test_no_rows():
    n, k = 70, 33
    dw, db = Out(n * k), Out(n)
    before = counter("launches")
    assert lib.slb_linear(CUDA, None, None, None, None, None, None, None, 0, n, k, 1) == 0
    assert lib.slb_gated(CUDA, None, None, None, None, None, None, None, None, None, None, 0, n, k, 1) == 0
    assert lib.slb_ck8_save(CUDA, None, None, 0, n) == 0 and lib.slb_ck8_load(CUDA, None, None, 0, n) == 0
    assert counter("launches") == before
    assert lib.slb_linear_bwd(CUDA, None, None, None, None, None, None, None, dw.ptr, db.ptr, 0, n, k, 1) == 0
    check_ok()
    assert not dw.get(n, k).any() and not db.get(n).any()
    outs = [Out(n * k), Out(n * k), Out(n), Out(n)]
    assert lib.slb_gated_bwd(CUDA, None, None, None, None, None, None, None, None, None, None, *[o.ptr for o in outs], 0, n, k, 2) == 0
    check_ok()
    assert not any(o.get(o.n).any() for o in outs)


def test_zero_operands_give_exact_results():
    rng = np.random.default_rng(0)
    m, n, k = 130, 200, 90
    w, bias = normal(rng, n, k), normal(rng, n)
    np.testing.assert_array_equal(linear(np.zeros((m, k), np.float32), w, bias), np.broadcast_to(bias, (m, n)))
    np.testing.assert_array_equal(linear(normal(rng, m, k), np.zeros((n, k), np.float32)), np.zeros((m, n), np.float32))
    dy, x = np.zeros((m, n), np.float32), normal(rng, m, k)
    bufs, outs = [DevBuf(t) for t in (dy, x, w)], [Out(m * k), Out(n * k), Out(n)]
    assert lib.slb_linear_bwd(CUDA, bufs[0].ptr, bufs[1].ptr, None, bufs[2].ptr, None, None, *[o.ptr for o in outs], m, n, k, 0) == 0
    check_ok()
    assert not any(o.get(o.n).any() for o in outs)


@pytest.mark.parametrize("value", [np.inf, -np.inf, np.nan])
def test_non_finite_values_stay_where_they_are(value):
    rng = np.random.default_rng(1)
    m, n, k = 200, 150, 130
    x, w = normal(rng, m, k), normal(rng, n, k, std=0.1)
    clean = linear(x, w)
    x2, w2 = x.copy(), w.copy()
    x2[77, 100], w2[33, 5] = value, value
    got = linear(x2, w2)
    bad = np.zeros((m, n), bool)
    bad[77], bad[:, 33] = True, True
    assert not np.isfinite(got[bad]).any()
    np.testing.assert_array_equal(got[~bad], clean[~bad])  # nor does it change anyone's scale
    dy = normal(rng, m, n, std=1e-3)
    dy2 = dy.copy()
    dy2[40, 9] = value
    res = []
    for t in (dy, dy2):
        bufs, outs = [DevBuf(a) for a in (t, x, w)], [Out(m * k), Out(n * k), Out(n)]
        assert lib.slb_linear_bwd(CUDA, bufs[0].ptr, bufs[1].ptr, None, bufs[2].ptr, None, None, *[o.ptr for o in outs], m, n, k, 0) == 0
        check_ok()
        res.append([o.get(*s) for o, s in zip(outs, ((m, k), (n, k), (n,)))])
    for axis_bad, clean_t, got_t in ((40, res[0][0], res[1][0]), (9, res[0][1], res[1][1])):
        assert not np.isfinite(got_t[axis_bad]).any()
        np.testing.assert_array_equal(np.delete(got_t, axis_bad, 0), np.delete(clean_t, axis_bad, 0))
    assert not np.isfinite(res[1][2][9]) and np.isfinite(np.delete(res[1][2], 9)).all()


@pytest.mark.parametrize("ex,ew", [(-100, 100), (100, -100), (60, 60), (-60, -60), (-125, 20), (110, -30)])
def test_extreme_magnitudes(ex, ew):
    """Powers of two on both operands: the result is the same but for the exponent, as long as it and its terms are normal."""
    rng = np.random.default_rng(2)
    x, w = normal(rng, 70, 100), normal(rng, 60, 100)
    base = linear(x, w)
    got = linear(np.ldexp(x, ex), np.ldexp(w, ew))
    if ex > -120:
        np.testing.assert_array_equal(got, np.ldexp(base, ex + ew))
    else:  # the smallest of these factors are denormal: two digits less than 2^-125 has
        s = np.abs(x).astype(np.float64) @ np.abs(w.T)
        close(got, np.ldexp(base.astype(np.float64), ex + ew), np.ldexp(product_bound(100, s) + 2.0 ** -22 * s, ex + ew))


def test_rows_of_very_different_magnitude():
    """Forward every row has its own scale: a row of tiny values keeps its relative precision next to one of huge ones."""
    rng = np.random.default_rng(3)
    x, w = normal(rng, 64, 200), normal(rng, 50, 200)
    scale = np.exp2(rng.integers(-60, 60, 64)).astype(np.float32)[:, None]
    np.testing.assert_array_equal(linear(x * scale, w), linear(x, w) * scale)


def test_the_residual_may_be_overwritten():
    rng = np.random.default_rng(4)
    for m, n, k in ((300, 260, 100), (77, 131, 40)):
        x, w, r = normal(rng, m, k), normal(rng, n, k), normal(rng, m, n)
        bx, bw, y, inplace = DevBuf(x), DevBuf(w), Out(m * n), DevBuf(r)
        apart = DevBuf(r)
        assert lib.slb_linear(CUDA, bx.ptr, bw.ptr, None, apart.ptr, y.ptr, None, None, m, n, k, 1) == 0
        assert lib.slb_linear(CUDA, bx.ptr, bw.ptr, None, inplace.ptr, inplace.ptr, None, None, m, n, k, 1) == 0
        check_ok()
        np.testing.assert_array_equal(inplace.get().reshape(m, n), y.get(m, n))


def test_offsets_beyond_32_bits():
    """Outputs, pre-activations and a checkpoint of more than 2^31 elements; the rows behind the border are checked."""
    m, n, k = 280001, 8200, 8
    rng = np.random.default_rng(6)
    x, w = normal(rng, m, k), normal(rng, n, k)
    bx, bw, y = DevBuf(x), DevBuf(w), DevBuf(n=m * n)
    nbytes = lib.slb_ck8_bytes(m, n)
    assert nbytes == ops.ck8_bytes(m, n)
    p = lib.sl_alloc(CUDA, nbytes)
    assert p
    assert lib.slb_linear(CUDA, bx.ptr, bw.ptr, None, None, y.ptr, None, p, m, n, k, 0) == 0
    check_ok()

    def rows_of(base, first, count):
        out = np.empty((count, n), np.float32)
        lib.sl_to_host(CUDA, out.ctypes.data, base + 4 * first * n, out.nbytes)
        return out

    spots = [0, 131000, (1 << 31) // n - 1, (1 << 31) // n + 1, m - 2]
    for first in spots:
        want = x[first:first + 2].astype(np.float64) @ w.T.astype(np.float64)
        s = np.abs(x[first:first + 2]).astype(np.float64) @ np.abs(w.T)
        close(rows_of(y.ptr, first, 2), want, product_bound(k, s))
    back = DevBuf(n=m * n)
    assert lib.slb_ck8_load(CUDA, p, back.ptr, m, n) == 0
    check_ok()
    for first in spots:  # the checkpoint that the product kept is the one that its result gives
        np.testing.assert_array_equal(rows_of(back.ptr, first, 2), ops.ck8_values(*ops.ck8_save(rows_of(y.ptr, first, 2))).astype(np.float32))
    ref = lib.sl_alloc(CUDA, nbytes)
    assert ref and lib.slb_ck8_save(CUDA, y.ptr, ref, m, n) == 0
    check_ok()
    tail_a, tail_b = np.empty(1 << 20, np.uint8), np.empty(1 << 20, np.uint8)
    for off in (0, (1 << 31) - (1 << 19), m * n - (1 << 20), nbytes - (1 << 20)):
        lib.sl_to_host(CUDA, tail_a.ctypes.data, p + off, tail_a.nbytes)
        lib.sl_to_host(CUDA, tail_b.ctypes.data, ref + off, tail_b.nbytes)
        if off <= m * n - (1 << 20) or (m * n) % 16 == 0:
            np.testing.assert_array_equal(tail_a, tail_b)
    lib.sl_free(CUDA, p, nbytes)
    lib.sl_free(CUDA, ref, nbytes)
    y.free(), back.free()
    lib.sl_empty_cache(CUDA)


@pytest.mark.parametrize("m,n,k", [(100, 90, 70), (768, 768, 4100), (600, 3000, 64)])
def test_scratch_from_the_caller(m, n, k):
    """The backend-level calls: the same bits, nothing outside the scratch, nothing from the pool -- and scratch that holds
    garbage, or the leavings of another call, does not matter."""
    rng = np.random.default_rng(7)
    x, w, dy, pre = normal(rng, m, k), normal(rng, n, k), normal(rng, m, n), normal(rng, m, n)
    bx, bw, bdy, bpre = (DevBuf(t) for t in (x, w, dy, pre))
    need = max(lib.slb_linear_scratch_bytes(m, n, k, b) for b in (0, 1))
    pad = 4096
    scratch = ByteBuf(np.random.default_rng(8).integers(0, 256, need + pad, dtype=np.uint8))
    tail = scratch.get()[need:].copy()
    ref = [Out(m * n), Out(m * k), Out(n * k), Out(n)]
    assert lib.slb_linear(CUDA, bx.ptr, bw.ptr, None, None, ref[0].ptr, None, None, m, n, k, 2) == 0
    assert lib.slb_linear_bwd(CUDA, bdy.ptr, bx.ptr, None, bw.ptr, bpre.ptr, None, *[o.ptr for o in ref[1:]], m, n, k, 2) == 0
    check_ok()
    for _ in range(2):
        got = [Out(o.n) for o in ref]
        before = (C.c_int64 * 7)()
        lib.sl_stats(CUDA, before)
        assert lib.slb_cuda_linear(bx.ptr, bw.ptr, None, None, got[0].ptr, None, None, m, n, k, 2, scratch.ptr, need) == 0
        assert lib.slb_cuda_linear_bwd(bdy.ptr, bx.ptr, None, bw.ptr, bpre.ptr, None, *[o.ptr for o in got[1:]], m, n, k, 2, scratch.ptr, need) == 0
        check_ok()
        after = (C.c_int64 * 7)()
        lib.sl_stats(CUDA, after)
        assert after[4] == before[4]  # no allocation
        for a, b in zip(got, ref):
            np.testing.assert_array_equal(a.get(a.n), b.get(b.n))
        np.testing.assert_array_equal(scratch.get()[need:], tail)


def test_gated_scratch_from_the_caller():
    m, n, k = 300, 333, 200
    rng = np.random.default_rng(9)
    x, wg, wu, g, u, dh = normal(rng, m, k), normal(rng, n, k), normal(rng, n, k), normal(rng, m, n), normal(rng, m, n), normal(rng, m, n)
    bx, bwg, bwu, bg, bu, bdh = (DevBuf(t) for t in (x, wg, wu, g, u, dh))
    need = max(lib.slb_gated_scratch_bytes(m, n, k, b) for b in (0, 1))
    scratch = ByteBuf(np.full(need, 255, np.uint8))
    ref, got = ([Out(m * n), Out(m * k), Out(n * k), Out(n * k), Out(n), Out(n)] for _ in range(2))
    assert lib.slb_gated(CUDA, bx.ptr, bwg.ptr, bwu.ptr, None, None, ref[0].ptr, None, None, None, None, m, n, k, 1) == 0
    assert lib.slb_gated_bwd(CUDA, bdh.ptr, bx.ptr, None, bwg.ptr, bwu.ptr, bg.ptr, bu.ptr, None, None, *[o.ptr for o in ref[1:]], m, n, k, 1) == 0
    assert lib.slb_cuda_gated(bx.ptr, bwg.ptr, bwu.ptr, None, None, got[0].ptr, None, None, None, None, m, n, k, 1, scratch.ptr, need) == 0
    assert lib.slb_cuda_gated_bwd(bdh.ptr, bx.ptr, None, bwg.ptr, bwu.ptr, bg.ptr, bu.ptr, None, None, *[o.ptr for o in got[1:]], m, n, k, 1, scratch.ptr, need) == 0
    check_ok()
    for a, b in zip(got, ref):
        np.testing.assert_array_equal(a.get(a.n), b.get(b.n))


def test_same_bits_every_run():
    rng = np.random.default_rng(10)
    m, n, k = 1100, 700, 2000
    x, w, dy = normal(rng, m, k), normal(rng, n, k), normal(rng, m, n)
    bx, bw, bdy = DevBuf(x), DevBuf(w), DevBuf(dy)
    runs = []
    for _ in range(3):
        outs = [Out(m * n), Out(m * k), Out(n * k), Out(n)]
        assert lib.slb_linear(CUDA, bx.ptr, bw.ptr, None, None, outs[0].ptr, None, None, m, n, k, 1) == 0
        assert lib.slb_linear_bwd(CUDA, bdy.ptr, bx.ptr, None, bw.ptr, None, None, *[o.ptr for o in outs[1:]], m, n, k, 0) == 0
        runs.append(outs)  # all in flight together
    check_ok()
    for outs in runs[1:]:
        for a, b in zip(outs, runs[0]):
            np.testing.assert_array_equal(a.get(a.n), b.get(b.n))


def test_a_pending_update_goes_first():
    """An AdamW call that the library has recorded but not launched writes the weight that the product reads."""
    rng = np.random.default_rng(11)
    m, n, k = 90, 80, 70
    x, w, g = normal(rng, m, k), normal(rng, n, k), normal(rng, n, k)
    bx, bw, bg, bm, bv = DevBuf(x), DevBuf(w), DevBuf(g), DevBuf(np.zeros(n * k)), DevBuf(np.zeros(n * k))
    y = Out(m * n)
    lib.sl_adamw(CUDA, bw.ptr, bg.ptr, bm.ptr, bv.ptr, n * k, 0.1, 0.9, 0.999, 1e-8, 0.0, 1)
    assert lib.slb_linear(CUDA, bx.ptr, bw.ptr, None, None, y.ptr, None, None, m, n, k, 0) == 0
    check_ok()
    new = bw.get().reshape(n, k)
    assert np.abs(new - w).max() > 0.05
    want = x.astype(np.float64) @ new.T.astype(np.float64)
    close(y.get(m, n), want, product_bound(k, np.abs(x).astype(np.float64) @ np.abs(new.T)))


@pytest.mark.parametrize("overlap", [0, 1])
def test_copies_beside_the_path(overlap):
    """An upload that is still in flight on its stream when a product reads its destination, and a download of the result:
    ordered by address, over several rounds through the same buffers."""
    rng = np.random.default_rng(12)
    m, n, k = 1500, 900, 800
    w = normal(rng, n, k)
    bx, bw, by = DevBuf(n=m * k), DevBuf(w), DevBuf(n=m * n)
    hx, hy = lib.slb_pinned_alloc(4 * m * k), [lib.slb_pinned_alloc(4 * m * n) for _ in range(3)]
    src = np.ctypeslib.as_array(C.cast(hx, C.POINTER(C.c_float)), (m, k))
    set_option("overlap", overlap)
    try:
        xs = []
        for r in range(3):
            xs.append(normal(rng, m, k))
            src[:] = xs[-1]
            assert lib.slb_from_host_async(1, (C.c_void_p * 1)(bx.ptr), (C.c_void_p * 1)(hx), (C.c_size_t * 1)(4 * m * k)) == 0
            assert lib.slb_linear(CUDA, bx.ptr, bw.ptr, None, None, by.ptr, None, None, m, n, k, 0) == 0
            assert lib.slb_to_host_async(1, (C.c_void_p * 1)(hy[r]), (C.c_void_p * 1)(by.ptr), (C.c_size_t * 1)(4 * m * n)) == 0
            assert lib.slb_wait_copies() == 0  # the source is written again
        check_ok()
        for r in range(3):
            y = np.ctypeslib.as_array(C.cast(hy[r], C.POINTER(C.c_float)), (m, n))
            want = xs[r].astype(np.float64) @ w.T.astype(np.float64)
            close(y, want, product_bound(k, np.abs(xs[r]).astype(np.float64) @ np.abs(w.T)))
    finally:
        set_option("overlap", 0)
        for p in [hx] + hy:
            lib.slb_pinned_free(p)


def test_out_of_memory_is_reported():
    lib.sl_empty_cache(CUDA)
    stats = (C.c_int64 * 7)()
    lib.sl_stats(CUDA, stats)
    m, n, k = 4096, 4096, 1024
    bx, bw, y = DevBuf(n=m * k), DevBuf(n=n * k), DevBuf(n=m * n)
    lib.sl_stats(CUDA, stats)
    lib.sl_set_limit(CUDA, stats[1])
    try:
        assert lib.slb_linear(CUDA, bx.ptr, bw.ptr, None, None, y.ptr, None, None, m, n, k, 0) == -2
    finally:
        lib.sl_set_limit(CUDA, 0)
    check_ok()


def test_checkpoint_of_more_than_2_30_rows():
    rows = (1 << 30) + 5
    x, ck = lib.sl_alloc(CUDA, 4 * rows), lib.sl_alloc(CUDA, lib.slb_ck8_bytes(rows, 1))
    assert x and ck
    lib.sl_fill(CUDA, x, rows, 3.0)
    tail = np.array([-1.0, 2.0 ** -20, 127.0, 128.0, 0.0], np.float32)
    lib.sl_from_host(CUDA, x + 4 * (rows - 5), tail.ctypes.data, tail.nbytes)
    assert lib.slb_ck8_save(CUDA, x, ck, rows, 1) == 0
    q, eb = ops.ck8_save(np.concatenate([np.full(3, 3.0, np.float32), tail])[:, None])
    got = np.empty(8, np.uint8)
    for first in (0, (1 << 29) + 1, rows - 8):
        lib.sl_to_host(CUDA, got.ctypes.data, ck + first, 8)
        np.testing.assert_array_equal(got.view(np.int8)[:3], q[:3, 0])
        if first == rows - 8:
            np.testing.assert_array_equal(got.view(np.int8), q[:, 0])
        lib.sl_to_host(CUDA, got.ctypes.data, ck + ops.ck8_exp_offset(rows, 1) + first, 8)
        np.testing.assert_array_equal(got[:3], eb[:3, 0])
        if first == rows - 8:
            np.testing.assert_array_equal(got, eb[:, 0])
    assert lib.slb_ck8_load(CUDA, ck, x, rows, 1) == 0
    check_ok()
    back = np.empty(5, np.float32)
    lib.sl_to_host(CUDA, back.ctypes.data, x + 4 * (rows - 5), back.nbytes)
    np.testing.assert_array_equal(back, ops.ck8_values(q, eb)[3:, 0].astype(np.float32))
    lib.sl_free(CUDA, x, 4 * rows)
    lib.sl_free(CUDA, ck, lib.slb_ck8_bytes(rows, 1))
    lib.sl_empty_cache(CUDA)
