"""Activation checkpoints in 8 bits on the GPU (csrc/ck8_kernels.cu): the bytes of the format's restatement, exactly."""
import numpy as np
import pytest

from oracle import ffn_ops as ops
from soliton_b200._C import lib
from tests.ffn_util import T, ByteBuf, Out, close
from tests.gpu_util import CUDA, DevBuf, check_ok

pytestmark = [pytest.mark.gpu, pytest.mark.usefixtures("cuda")]
SHAPES = [(1, 1), (1, 31), (3, 32), (7, 33), (5, 64), (1, 4096), (64, 127), (129, 2305), (300, 512), (40, 65), (61, 34)]


def special(rows, cols):
    """Magnitudes over the whole range, groups of zeros, the border values of the step, and non-finite values."""
    rng = np.random.default_rng(rows * 100 + cols)
    with np.errstate(over="ignore"):
        x = (rng.standard_normal((rows, cols)) * np.exp2(rng.integers(-150, 127, (rows, cols)))).astype(np.float32)
    x[~np.isfinite(x)] = 1.0
    flat = x.reshape(-1)
    border = np.float32(127 / 64)
    picks = [border, np.nextafter(border, np.float32(2)), np.float32(0), np.float32(-0.0), np.finfo(np.float32).max, np.float32(1e-45), np.float32(2.0 ** -126)]
    for i, v in enumerate(picks):
        at = (i * 37) % flat.size
        flat[at] = v
    if rows > 2:
        x[1] = 0
        x[2, : min(cols, 20)] = np.linspace(-2, 2, 20, dtype=np.float32)[: min(cols, 20)]
    if rows > 4:
        x[3, cols // 2], x[4, 0] = np.inf, np.nan
    return x


@pytest.mark.parametrize("skew", [0, 1])
@pytest.mark.parametrize("rows,cols", SHAPES)
def test_save_and_load(rows, cols, skew):
    for x in (special(rows, cols), np.random.default_rng(cols).standard_normal((rows, cols)).astype(np.float32)):
        q, eb = ops.ck8_save(x)
        bx, ck, back = DevBuf(x, skew=skew), ByteBuf(n=ops.ck8_bytes(rows, cols), skew=skew), Out(rows * cols, skew)
        assert lib.slb_ck8_bytes(rows, cols) == ops.ck8_bytes(rows, cols)
        assert lib.slb_ck8_save(CUDA, bx.ptr, ck.ptr, rows, cols) == 0
        assert lib.slb_ck8_load(CUDA, ck.ptr, back.ptr, rows, cols) == 0
        check_ok()
        gq, geb = ops.ck8_unpack(ck.get(), rows, cols)
        np.testing.assert_array_equal(geb, eb)
        np.testing.assert_array_equal(gq, q)
        np.testing.assert_array_equal(back.get(rows, cols), ops.ck8_values(q, eb).astype(np.float32))


@pytest.mark.parametrize("rows,cols", SHAPES)
def test_gelu_bwd(rows, cols):
    rng = np.random.default_rng(rows + cols)
    x, dy = (rng.standard_normal((rows, cols)) * 2).astype(np.float32), rng.standard_normal((rows, cols)).astype(np.float32)
    q, eb = ops.ck8_save(x)
    v = ops.ck8_values(q, eb)
    for skew in (0, 3):
        ck, bdy, dx = ByteBuf(ops.ck8_pack(q, eb), skew=skew), DevBuf(dy, skew=skew), Out(rows * cols, skew)
        assert lib.slb_ck8_gelu_bwd(CUDA, ck.ptr, bdy.ptr, dx.ptr, rows, cols) == 0
        check_ok()
        # Phi through erff (its rounding, the argument's and two more: 4t), x phi(x) through expf, one product
        close(dx.get(rows, cols), dy * ops.act_grad(v, "gelu"), 14 * T * np.abs(dy) * (1 + np.abs(v)), "dx")


def test_every_byte_pair_loads_exactly(cuda):
    """All 256 exponent bytes times all 256 values."""
    rows, cols = 256, 256
    q = np.tile(np.arange(-128, 128, dtype=np.int16).astype(np.int8), (rows, 1))
    eb = np.repeat(np.arange(256, dtype=np.uint8)[:, None], cols // 32, axis=1)
    ck, back = ByteBuf(ops.ck8_pack(q, eb)), Out(rows * cols)
    assert lib.slb_ck8_load(CUDA, ck.ptr, back.ptr, rows, cols) == 0
    check_ok()
    with np.errstate(over="ignore"):
        np.testing.assert_array_equal(back.get(rows, cols), ops.ck8_values(q, eb).astype(np.float32))
