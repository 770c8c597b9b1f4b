"""soliton_b200.ffn on tensors: shapes and refusals on meta (no GPU), and on the GPU whole training steps of a small
feed-forward stack, through checkpoints and this package's AdamW."""
import numpy as np
import pytest

from oracle import ffn_ops as ops


@pytest.fixture
def F(built):
    from soliton_b200 import ffn
    return ffn


@pytest.fixture
def T(built):
    from soliton_b200 import tensor
    return tensor


def test_shapes_on_meta(F, T):
    x, w, b, r = (T.empty(s, "meta") for s in ((2, 3, 8), (5, 8), (5,), (2, 3, 5)))
    y, pre = F.linear(x, w, b, r, "gelu", keep="ck8")
    assert y.shape == (2, 3, 5) and isinstance(pre, F.Checkpoint) and (pre.rows, pre.cols) == (6, 5)
    ck = F.Checkpoint.save(x)
    assert ck.load().shape == x.shape and F.gelu_bwd(pre, y).shape == y.shape
    assert [t.shape for t in F.linear_bwd(y, ck, w, pre, "gelu")] == [(2, 3, 8), (5, 8), (5,)]
    assert F.linear_bwd(y, x, w, need=("w",))[0] is None
    h, g, u = F.gated(x, w, w, b, keep="fp32")
    assert h.shape == g.shape == u.shape == (2, 3, 5)
    assert [t.shape for t in F.gated_bwd(h, ck, w, w, g, u)] == [(2, 3, 8), (5, 8), (5, 8), (5,), (5,)]
    assert F.gated_bwd(h, ck, w, w, g, u, bias=False)[3:] == (None, None)
    assert F.linear(T.empty((0, 8), "meta"), w).shape == (0, 5)


def test_refusals(F, T):
    x, w = T.empty((4, 8), "meta"), T.empty((5, 8), "meta")
    y = T.empty((4, 5), "meta")
    bad = [lambda: F.linear(x, T.empty((5, 7), "meta")), lambda: F.linear(x, w, T.empty((4,), "meta")), lambda: F.linear(x, w, act="relu6"),
           lambda: F.linear(x, w, residual=x), lambda: F.linear(x, w, keep="fp16"), lambda: F.linear(x, T.empty((5, 8), "cpu")),
           lambda: F.linear_bwd(y, T.empty((3, 8), "meta"), w), lambda: F.linear_bwd(y, x, w, act="gelu"), lambda: F.linear_bwd(y, x, w, need=()),
           lambda: F.linear_bwd(y, x, w, need=("z",)), lambda: F.linear_bwd(y, x, w, x, "gelu"), lambda: F.gated(x, w, T.empty((6, 8), "meta")),
           lambda: F.gated_bwd(y, x, w, w, x, y), lambda: F.gelu_bwd(x, x), lambda: F.gelu_bwd(F.Checkpoint.save(x), y),
           lambda: F.Checkpoint((3, 0), "meta"), lambda: F.linear(T.empty((4, 0), "meta"), w)]
    for f in bad:
        with pytest.raises(ValueError):
            f()
    cpu = [T.empty(s, "cpu") for s in ((4, 8), (5, 8))]
    with pytest.raises(RuntimeError):  # no host kernels
        F.linear(*cpu)
    from soliton_b200._C import lib
    lib.slb_clear_error()


def steps(F, T, dev, ck, count=3):
    """A residual gated block, then a GELU layer, mean squared error against a target: `count` steps, the gradients of each
    returned as computed on the device (or nothing on meta), with the parameters before it."""
    from soliton_b200.optim import AdamW
    rng = np.random.default_rng(5)
    m, c, f = 200, 96, 160
    shapes = dict(wg=(f, c), wu=(f, c), wd=(c, f), bd=(c,), w1=(64, c), b1=(64,))
    host = {n: (rng.standard_normal(s) * 0.1).astype(np.float32) for n, s in shapes.items()}
    x0, target = rng.standard_normal((m, c)).astype(np.float32), rng.standard_normal((m, 64)).astype(np.float32)
    p = {n: T.tensor(v, dev) for n, v in host.items()}
    x = T.tensor(x0, dev)
    opt = AdamW(list(p.values()), lr=1e-3, weight_decay=0.0)
    seen = []
    keep = "ck8" if ck else "fp32"
    for _ in range(count):
        h, g, u = F.gated(x, p["wg"], p["wu"], keep=keep)
        z = F.linear(h, p["wd"], p["bd"], residual=x)
        y, pre = F.linear(z, p["w1"], p["b1"], act="gelu", keep=keep)
        if ck:  # what the backward pass needs of the activations is put away as well
            hx, zx, xx = F.Checkpoint.save(h), F.Checkpoint.save(z), F.Checkpoint.save(x)
        else:
            hx, zx, xx = h, z, x
        dy = T.empty(y.shape, dev)
        if dev == "cuda":
            before = {n: t.numpy() for n, t in p.items()}
            dy = T.tensor((y.numpy() - target) * np.float32(2.0 / m), dev)
        dz, dw1, db1 = F.linear_bwd(dy, zx, p["w1"], pre, "gelu")
        dh, dwd, dbd = F.linear_bwd(dz, hx, p["wd"])
        _, dwg, dwu, _, _ = F.gated_bwd(dh, xx, p["wg"], p["wu"], g, u, bias=False)
        grads = dict(wg=dwg, wu=dwu, wd=dwd, bd=dbd, w1=dw1, b1=db1)
        for n, t in p.items():
            t.grad = grads[n]
        if dev == "cuda":
            seen.append((before, {n: t.numpy() for n, t in grads.items()}, dy.numpy()))
        opt.step()
        opt.zero_grad()
    return x0, seen


def expected(x, p, dy, ck):
    """The same step's gradients in 64 bits, from the same parameters and output gradient."""
    put = (lambda t: ops.ck8_values(*ops.ck8_save(t.astype(np.float32)))) if ck else (lambda t: t)
    h, g, u = ops.gated(x, p["wg"], p["wu"])
    z, _ = ops.linear(h, p["wd"], p["bd"], x)
    _, pre = ops.linear(z, p["w1"], p["b1"], kind="gelu")
    dz, dw1, db1, _ = ops.linear_bwd(dy, put(z), p["w1"], put(pre), "gelu")
    dh, dwd, dbd, _ = ops.linear_bwd(dz, put(h), p["wd"])
    _, dwg, dwu, _, _, _, _ = ops.gated_bwd(dh, put(x), p["wg"], p["wu"], put(g), put(u))
    return dict(wg=dwg, wu=dwu, wd=dwd, bd=dbd, w1=dw1, b1=db1)


@pytest.mark.gpu
@pytest.mark.parametrize("ck", [False, True])
def test_training_steps(F, T, cuda, ck):
    x, seen = steps(F, T, "cuda", ck)
    for before, got, dy in seen:
        want = expected(x, before, dy, ck)
        for n in got:
            # norm-wise: each of five products in a row is within 1e-6 of its norm on random data (a few times the rounding
            # of fp32), and their conditioning here is of order one: ten times that. With checkpoints a value that falls on
            # the other side of a rounding border moves by a step, 1/63 of its group's largest at most; about one in 2^14
            # does (values are off by 2^-22 or so, steps are 2^-7 of them), so by sqrt(2^-14) / 63 * 4 of the norm, 5e-4.
            err = np.linalg.norm(got[n] - want[n]) / np.linalg.norm(want[n])
            assert err <= (5e-4 if ck else 1e-5), (n, err)


@pytest.mark.gpu
@pytest.mark.parametrize("ck", [False, True])
def test_a_dry_run_plans_them_exactly(F, T, cuda, ck):
    def peak(dev):
        T.empty_cache(dev)
        T.reset_peak_stats(dev)
        base = T.memory_stats(dev)
        steps(F, T, dev, ck)
        after = T.memory_stats(dev)
        return after["peak_allocated"] - base["allocated"]
    got = peak("cuda")
    # the run on the GPU holds one more tensor at a time, the output gradient that comes from the host
    assert 0 <= got - peak("meta") <= 200 * 64 * 4 + 512


@pytest.mark.gpu
def test_same_bits_every_run(F, T, cuda):
    a, b = steps(F, T, "cuda", True)[1], steps(F, T, "cuda", True)[1]
    for (_, x, _), (_, y, _) in zip(a, b):
        for n in x:
            np.testing.assert_array_equal(x[n], y[n])


@pytest.mark.gpu
def test_an_arena_planned_on_meta_holds_a_step(F, T, cuda):
    """Recorded on meta, packed, installed, and replayed on the GPU: operators' scratch, checkpoints and gradients all lie
    in the one planned allocation, and the values are those of the plain pool."""
    from soliton_b200 import arena
    rng = np.random.default_rng(3)
    host = [rng.standard_normal(s).astype(np.float32) for s in ((300, 128), (256, 128), (256, 128), (128, 256))]

    def step(dev):
        x, wg, wu, wd = (T.tensor(h, dev) for h in host)
        h, g, u = F.gated(x, wg, wu, keep="ck8")
        h8 = F.Checkpoint.save(h)
        y = F.linear(h, wd, residual=x)
        del h
        dh, dwd, _ = F.linear_bwd(y, h8, wd, need=("x", "w"))
        grads = F.gated_bwd(dh, F.Checkpoint.save(x), wg, wu, g, u, bias=False)[:3] + (dwd,)
        return [t.numpy() for t in grads] if dev == "cuda" else None

    T.empty_cache("cuda")
    want = step("cuda")
    plan = arena.plan(step)
    T.empty_cache("cuda")
    before = T.memory_stats("cuda")["reserved"]
    arena.install(plan, "cuda")
    try:
        got = step("cuda")
        arena.check("cuda")
        assert T.memory_stats("cuda")["reserved"] - before == plan.bytes
    finally:
        arena.off("cuda")
    for a, b in zip(got, want):
        np.testing.assert_array_equal(a, b)
