"""Feed-forward operators of a training step on this package's tensors: a product with bias, activation and residual
(`linear`), the gated block (`gated`), their backward passes, and activation checkpoints in 8 bits (`Checkpoint`), which
the backward passes take in the place of the tensors they were made from.

No counterpart in Soliton; conventions follow its `nn.Linear` (weights are (features out, features in), python/soliton/
nn.py:34). There is no autograd here: a forward function returns what its backward function wants to have back. On meta
everything allocates what it would on cuda and computes nothing, so plans made there hold.
"""
from . import tensor as T
from ._C import lib

ACTS = {"none": 0, "gelu": 1, "silu": 2}
KEEP = (None, "fp32", "ck8")


def _rows(t):
    """Rows and columns of a tensor (..., features), or of a checkpoint."""
    if isinstance(t, Checkpoint):
        return t.rows, t.cols
    if t.ndim < 1 or t.shape[-1] < 1:
        raise ValueError(f"soliton: a tensor of rows of features is wanted, not shape {t.shape}")
    return T._count(t.shape[:-1]), t.shape[-1]


def _expect(ok, what):
    if not ok:
        raise ValueError(f"soliton: {what}")


def _act(name):
    _expect(name in ACTS, f"activation {name!r} is none of {', '.join(ACTS)}")
    return ACTS[name]


def _same_device(first, *others):
    _expect(all(o is None or o.dev == first.dev for o in others), "tensors are on different devices")
    return first.dev


def _done(rc, dev):
    """The library's return code as an exception (0 ok, -2 out of memory, else the sticky error says what)."""
    if rc == -2:
        raise MemoryError(f"soliton: out of memory on {T.DEVICES[dev]} for an operator's scratch")
    if rc != 0:
        T._check(dev)
        raise RuntimeError(f"soliton: {T.DEVICES[dev]} operator refused")


def _ptr(t):
    return None if t is None else t.ptr


def _either(t):
    """(fp32 pointer, checkpoint pointer) of an operand that may be either."""
    return (None, t.ptr) if isinstance(t, Checkpoint) else (_ptr(t), None)


class Checkpoint:
    """The values of a (..., features) tensor in 8 bits: a signed byte each and, for every 32 columns of a row, a power of
    two (1.03 bytes a value). Values are off by half a step at most, a step being at most 1/63 of the largest magnitude
    among the 32 (include/soliton_b200.h has the layout)."""
    __slots__ = ("storage", "shape", "rows", "cols")

    def __init__(self, shape, dev):
        self.shape = tuple(int(n) for n in shape)
        _expect(len(self.shape) >= 1 and self.shape[-1] >= 1, f"no checkpoint of shape {self.shape}")
        self.rows, self.cols = T._count(self.shape[:-1]), self.shape[-1]
        self.storage = T.Storage(T._dev(dev), lib.slb_ck8_bytes(self.rows, self.cols))

    @property
    def dev(self):
        return self.storage.dev

    @property
    def ptr(self):
        return self.storage.ptr

    @classmethod
    def save(cls, t):
        ck = cls(t.shape, t.dev)
        _done(lib.slb_ck8_save(t.dev, t.ptr, ck.ptr, ck.rows, ck.cols), t.dev)
        return ck

    def load(self):
        out = T.empty(self.shape, self.dev)
        _done(lib.slb_ck8_load(self.dev, self.ptr, out.ptr, self.rows, self.cols), self.dev)
        return out


def gelu_bwd(x, dy):
    """dx = dy * GELU'(x) for a checkpoint x."""
    _expect(isinstance(x, Checkpoint), "gelu_bwd takes a checkpoint")
    _expect(_rows(dy) == (x.rows, x.cols), f"dy {dy.shape} does not fit a checkpoint of {x.shape}")
    dev = _same_device(x, dy)
    dx = T.empty(dy.shape, dev)
    _done(lib.slb_ck8_gelu_bwd(dev, x.ptr, dy.ptr, dx.ptr, x.rows, x.cols), dev)
    return dx


def _kept(keep, shape, dev):
    """What a forward pass keeps pre-activations in: (the object to return, fp32 pointer, checkpoint pointer)."""
    _expect(keep in KEEP, f"keep {keep!r} is none of {KEEP}")
    t = None if keep is None else T.empty(shape, dev) if keep == "fp32" else Checkpoint(shape, dev)
    return (t,) + _either(t)


def _weight(w, k, what="weight"):
    _expect(w.ndim == 2 and w.shape[1] == k and w.shape[0] >= 1, f"{what} {w.shape} does not fit {k} features")
    return w.shape[0]


def _bias(b, n):
    _expect(b is None or b.shape == (n,), f"bias {getattr(b, 'shape', None)} does not fit {n} features")


def linear(x, w, bias=None, residual=None, act="none", keep=None):
    """act(x w^T + bias) + residual. With `keep` ("fp32" or "ck8") also the pre-activations, for linear_bwd: (y, pre)."""
    kind, (m, k) = _act(act), _rows(x)
    n = _weight(w, k)
    _bias(bias, n)
    shape = x.shape[:-1] + (n,)
    _expect(residual is None or residual.shape == shape, f"residual {getattr(residual, 'shape', None)} is not {shape}")
    dev = _same_device(x, w, bias, residual)
    y = T.empty(shape, dev)
    pre, full, ck = _kept(keep, shape, dev)
    _done(lib.slb_linear(dev, x.ptr, w.ptr, _ptr(bias), _ptr(residual), y.ptr, full, ck, m, n, k, kind), dev)
    return y if keep is None else (y, pre)


def linear_bwd(dy, x, w, pre=None, act="none", need=("x", "w", "b")):
    """(dx, dw, db), None for those not in `need`. x and pre (wanted when there is an activation) are tensors or
    checkpoints. A residual's gradient is dy itself."""
    kind, (m, n), (mx, k) = _act(act), _rows(dy), _rows(x)
    _expect(mx == m and _weight(w, k) == n, f"dy {dy.shape}, x {x.shape} and weight {w.shape} do not fit")
    _expect(need and set(need) <= {"x", "w", "b"}, f"need {need!r} names none or others than x, w, b")
    _expect(act == "none" or (pre is not None and _rows(pre) == (m, n)), "pre-activations do not fit dy")
    dev = _same_device(dy, x, w, pre)
    dx = T.empty(x.shape, dev) if "x" in need else None
    dw = T.empty(w.shape, dev) if "w" in need else None
    db = T.empty((n,), dev) if "b" in need else None
    _done(lib.slb_linear_bwd(dev, dy.ptr, *_either(x), w.ptr, *_either(pre if kind else None), _ptr(dx), _ptr(dw), _ptr(db), m, n, k, kind), dev)
    return dx, dw, db


def gated(x, wg, wu, bg=None, bu=None, act="silu", keep=None):
    """act(x wg^T + bg) * (x wu^T + bu). With `keep` also both pre-activations, for gated_bwd: (h, g, u)."""
    kind, (m, k) = _act(act), _rows(x)
    f = _weight(wg, k)
    _expect(wu.shape == wg.shape, f"weights {wg.shape} and {wu.shape} differ")
    _bias(bg, f), _bias(bu, f)
    dev = _same_device(x, wg, wu, bg, bu)
    shape = x.shape[:-1] + (f,)
    h = T.empty(shape, dev)
    (g, g32, g8), (u, u32, u8) = _kept(keep, shape, dev), _kept(keep, shape, dev)
    _done(lib.slb_gated(dev, x.ptr, wg.ptr, wu.ptr, _ptr(bg), _ptr(bu), h.ptr, g32, u32, g8, u8, m, f, k, kind), dev)
    return h if keep is None else (h, g, u)


def gated_bwd(dh, x, wg, wu, g, u, act="silu", bias=True):
    """(dx, dwg, dwu, dbg, dbu); the last two None without `bias`. x, g and u are tensors or checkpoints."""
    kind, (m, f), (mx, k) = _act(act), _rows(dh), _rows(x)
    _expect(mx == m and _weight(wg, k) == f and wu.shape == wg.shape, f"dh {dh.shape}, x {x.shape} and weights {wg.shape}, {wu.shape} do not fit")
    _expect(_rows(g) == (m, f) and _rows(u) == (m, f), "pre-activations do not fit dh")
    dev = _same_device(dh, x, wg, wu, g, u)
    dx, dwg, dwu = T.empty(x.shape, dev), T.empty(wg.shape, dev), T.empty(wu.shape, dev)
    dbg, dbu = (T.empty((f,), dev), T.empty((f,), dev)) if bias else (None, None)
    (x32, x8), (g32, g8), (u32, u8) = _either(x), _either(g), _either(u)
    _done(lib.slb_gated_bwd(dev, dh.ptr, x32, x8, wg.ptr, wu.ptr, g32, u32, g8, u8, dx.ptr, dwg.ptr, dwu.ptr, _ptr(dbg), _ptr(dbu), m, f, k, kind), dev)
    return dx, dwg, dwu, dbg, dbu
