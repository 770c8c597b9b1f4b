"""The float64 restatements of the feed-forward operators (oracle/ffn_ops.py) pinned against PyTorch's float64 autograd and
against differences, and the checkpoint format against its definition. No GPU: the GPU tests hold the kernels against these."""
import numpy as np
import pytest
import torch
import torch.nn.functional as F

from oracle import ffn_ops as ops

TORCH_ACT = {"none": lambda v: v, "gelu": F.gelu, "silu": F.silu}
# float64 against float64: sums of at most a few hundred terms of order one
TIGHT = dict(rtol=1e-12, atol=1e-12)


def leaves(rng, *shapes):
    return [torch.tensor(rng.standard_normal(s), dtype=torch.float64, requires_grad=True) for s in shapes]


@pytest.mark.parametrize("kind", ["none", "gelu", "silu"])
def test_linear_against_autograd(kind):
    x, w, b, r = leaves(np.random.default_rng(1), (9, 7), (5, 7), (5,), (9, 5))
    pre = F.linear(x, w, b)
    y = TORCH_ACT[kind](pre) + r
    dy = torch.randn(9, 5, dtype=torch.float64, generator=torch.Generator().manual_seed(0))
    grads = torch.autograd.grad(y, (x, w, b), dy)
    n = [t.detach().numpy() for t in (x, w, b, r)]
    got_y, got_pre = ops.linear(*n, kind)
    np.testing.assert_allclose(got_y, y.detach().numpy(), **TIGHT)
    for got, want in zip(ops.linear_bwd(dy.numpy(), n[0], n[1], got_pre, kind), grads):
        np.testing.assert_allclose(got, want.numpy(), **TIGHT)


@pytest.mark.parametrize("kind", ["none", "gelu", "silu"])
def test_gated_against_autograd(kind):
    x, wg, wu, bg, bu = leaves(np.random.default_rng(2), (9, 7), (5, 7), (5, 7), (5,), (5,))
    h = TORCH_ACT[kind](F.linear(x, wg, bg)) * F.linear(x, wu, bu)
    dh = torch.randn(9, 5, dtype=torch.float64, generator=torch.Generator().manual_seed(0))
    grads = torch.autograd.grad(h, (x, wg, wu, bg, bu), dh)
    n = [t.detach().numpy() for t in (x, wg, wu, bg, bu)]
    got_h, g, u = ops.gated(*n, kind)
    np.testing.assert_allclose(got_h, h.detach().numpy(), **TIGHT)
    for got, want in zip(ops.gated_bwd(dh.numpy(), n[0], n[1], n[2], g, u, kind), grads):
        np.testing.assert_allclose(got, want.numpy(), **TIGHT)


@pytest.mark.parametrize("kind", ["gelu", "silu"])
def test_derivatives_against_differences(kind):
    v = np.linspace(-9, 9, 721)
    h = 1e-5  # central differences: h^2 / 6 of a third derivative below 2, and rounding 2^-53 * 9 / h
    np.testing.assert_allclose(ops.act_grad(v, kind), (ops.act(v + h, kind) - ops.act(v - h, kind)) / (2 * h), rtol=0, atol=4e-10)


@pytest.mark.parametrize("shape", [(1, 1), (3, 31), (4, 32), (5, 65)])
def test_checkpoint_format(shape):
    rng = np.random.default_rng(3)
    x = (rng.standard_normal(shape) * np.exp2(rng.integers(-40, 40, shape))).astype(np.float32)
    q, eb = ops.ck8_save(x)
    step = np.repeat(np.exp2(eb.astype(np.float64) - 127), 32, axis=1)[:, :shape[1]]
    assert (np.abs(ops.ck8_values(q, eb) - x) <= step / 2).all()
    for r in range(shape[0]):
        for g in range(eb.shape[1]):
            top, s = float(np.abs(x[r, 32 * g:32 * g + 32]).max()), 2.0 ** (int(eb[r, g]) - 127)
            assert 127 * s >= top > 127 * s / 2
    buf = ops.ck8_pack(q, eb)
    q2, eb2 = ops.ck8_unpack(buf, *shape)
    assert np.array_equal(q, q2) and np.array_equal(eb, eb2)


def test_checkpoint_of_zeros_and_non_finite_values():
    x = np.zeros((3, 40), np.float32)
    x[1, 3], x[2, 35] = np.inf, np.nan
    q, eb = ops.ck8_save(x)
    assert eb.tolist() == [[1, 1], [255, 1], [1, 255]] and not q.any()
    v = ops.ck8_values(q, eb)
    assert np.isnan(v[1, :32]).all() and np.isnan(v[2, 32:]).all() and not v[0].any() and not v[1, 32:].any()
