"""What the tests of the feed-forward operators share: byte buffers and error bounds.

Bound of a product over `k` terms, as the kernels compute it, relative to S = sum |a_i b_i| (t = 2^-24 the rounding of
fp32, `eps / 2`):
  operands  each carries 22 bits (error 2^-22 of the value: hi rounds to 2^-11, lo to 2^-11 of that) and lo*lo is
            dropped (2^-22): 3 * 2^-22
  tensor    an accumulation rounds towards zero, off by one ulp at most, 2t of a partial sum that S bounds; 16 terms are
            added at once, their alignment costs at most as much again: 4t per accumulation, and 0.28t are given back for
            each on the average; 3 accumulations (products of pieces) per 16 terms, at most 384 terms in a row
  segments  one fp32 addition (t) per 256 terms
  scaling   exact (powers of two)
"""
import ctypes as C

import numpy as np

from soliton_b200._C import lib
from tests.gpu_util import CUDA, DevBuf

T = np.finfo(np.float32).eps / 2


def product_bound(k, s):
    steps = 3 * ((min(k, 384) + 15) // 16)
    return (3 * 2.0 ** -22 + 4.28 * T * steps + T * ((k + 255) // 256)) * s


class ByteBuf:
    """A device buffer of bytes, `skew` bytes into its allocation."""

    def __init__(self, data=None, n=None, skew=0):
        if data is not None:
            data = np.ascontiguousarray(data).view(np.uint8).reshape(-1)
            n = data.size
        self.n, self.nbytes = int(n), int(n) + skew
        self.base = lib.sl_alloc(CUDA, self.nbytes)
        assert self.base
        self.ptr = self.base + skew
        if data is not None:
            lib.sl_from_host(CUDA, self.ptr, data.ctypes.data, data.nbytes)

    def get(self):
        out = np.empty(self.n, np.uint8)
        lib.sl_to_host(CUDA, out.ctypes.data, self.ptr, out.nbytes)
        return out

    def __del__(self):
        try:
            lib.sl_free(CUDA, self.base, self.nbytes)
        except Exception:
            pass


MARK = np.float32(-7.25e11)


class Out:
    """An output of `n` floats between marked margins that nothing may touch."""
    MARGIN = 64

    def __init__(self, n, skew=0):
        self.n, self.skew = n, skew
        self.buf = DevBuf(np.full(n + 2 * self.MARGIN + skew, MARK, np.float32))
        self.ptr = self.buf.ptr + 4 * (self.MARGIN + skew)

    def get(self, *shape):
        a = self.buf.get()
        lo = self.MARGIN + self.skew
        assert (a[:lo] == MARK).all() and (a[lo + self.n:] == MARK).all(), "written outside the output"
        return a[lo:lo + self.n].reshape(shape)


def ptr(b):
    return None if b is None else b.ptr


def close(got, want, bound, what=""):
    got = np.asarray(got, np.float64)
    bad = ~(np.abs(got - want) <= bound)
    if bad.any():
        i = np.unravel_index(int(np.argmax(np.where(np.isnan(got), np.inf, np.abs(got - want) / bound))), got.shape)
        raise AssertionError(f"{what}: {int(bad.sum())} of {bad.size} outside; worst at {i}: {got[i]!r} against {want[i]!r}, bound {np.broadcast_to(bound, got.shape)[i]:.3g}")
