"""The feed-forward operators of a training step, as measured: matrix product with bias, activation and residual
(slb_linear), the gated feed-forward block (slb_gated), both with their backward passes, and activation checkpoints in
8 bits (slb_ck8_*), which the backward passes read in place of the fp32 tensors.

Tensors are dense row-major fp32, as everywhere in this library. A weight is (features out, features in), a bias one
value per feature out. A checkpoint of a rows x cols tensor is one buffer: rows * cols signed bytes q, padding to a
multiple of 16 bytes, then one exponent byte e for every 32 columns of a row (the last group of a row may be shorter);
it stands for q * 2^(e - 127).
"""
import functools
import math

import torch

own = False
CUDA = 2
ACT = {"none": 0, "gelu": 1, "silu": 2}
GROUP = 32


# ---------------------------------------------------------------------------------------------- the cases

def _linear(name, m, n, k, act="none", bias=True, residual=False, save="none"):
    return dict(name=name, op="linear", m=m, n=n, k=k, act=act, bias=bias, residual=residual, save=save)


def _linear_bwd(name, m, n, k, act="none", held="fp32", padded=False):
    return dict(name=name, op="linear_bwd", m=m, n=n, k=k, act=act, held=held, padded=padded)


def _gated(name, m, f, k, act="silu", save="none"):
    return dict(name=name, op="gated", m=m, n=f, k=k, act=act, save=save)


def _gated_bwd(name, m, f, k, act="silu", held="fp32", padded=False):
    return dict(name=name, op="gated_bwd", m=m, n=f, k=k, act=act, held=held, padded=padded)


def listed():
    return [
        # the tiny model's first feed-forward product, one sequence of 64 tokens: launch latency and little else
        _linear("linear tiny", 64, 128, 32, "gelu", save="fp32"),
        # attention's output projection of the 124M model at 8 x 1024 tokens, added to the residual stream
        _linear("linear proj residual", 8192, 768, 768, residual=True),
        # the medium model's first feed-forward product at 4 x 1024 tokens; backward needs the pre-activation
        _linear("linear fc gelu", 4096, 4096, 1024, "gelu", save="fp32"),
        # the vocabulary product at one sequence of 1024 tokens: an odd width, rows at every alignment
        _linear("linear head odd", 1024, 50257, 768, bias=False),
        # gradients of a small layer with nothing divisible by anything
        _linear_bwd("linear_bwd ragged", 333, 515, 257, "gelu"),
        # gradients of the projection in the 124M model: a long sum over tokens into a small weight
        _linear_bwd("linear_bwd proj", 8192, 768, 768),
        # gradients of the medium model's first product, input and pre-activation held in 8 bits
        _linear_bwd("linear_bwd fc ck8", 4096, 4096, 1024, "gelu", held="8bit"),
        # a small gated block, odd rows, its two pre-activations saved in 8 bits by the forward pass
        _gated("gated small ck8", 127, 160, 96, save="8bit"),
        # a gated block over the 124M model's width, 2048 being 8/3 of 768
        _gated("gated", 8192, 2048, 768, save="fp32"),
        # its gradients, the last tokens of the batch padding (their gradient is zero)
        _gated_bwd("gated_bwd padded", 8192, 2048, 768, padded=True),
        # a layer's activations put away in 8 bits and fetched again
        dict(name="ck8 save load", op="ck8_save_load", rows=8192, cols=4096),
        # GELU's backward pass from a checkpoint, odd columns
        dict(name="ck8 gelu_bwd odd", op="ck8_gelu_bwd", rows=4096, cols=2305),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


MOST_FLOPS = 8 * 8192 * 2048 * 768.0


def draw(rng):
    op = rng.choice(["linear", "linear_bwd", "gated", "gated_bwd", "ck8_save_load", "ck8_gelu_bwd"])
    if op.startswith("ck8"):
        while True:
            rows, cols = _log_int(rng, 1, 16384), _log_int(rng, 1, 16384)
            if rows * cols <= 8192 * 4096:
                return dict(op=op, rows=rows, cols=cols)
    while True:
        m, n, k = _log_int(rng, 1, 16384), _log_int(rng, 8, 8192), _log_int(rng, 8, 4096)
        if rng.random() < 0.5:  # the usual multiples; otherwise whatever came
            n, k = (n + 31) // 32 * 32, (k + 31) // 32 * 32
        if 2.0 * m * n * k * {"linear": 1, "linear_bwd": 2, "gated": 2, "gated_bwd": 4}[op] <= MOST_FLOPS and m * n <= 1 << 26:
            break
    act = rng.choice(["none", "gelu", "silu"]) if op.startswith("linear") else rng.choice(["gelu", "silu"])
    if op == "linear":
        save = rng.choice(["none", "fp32", "8bit"]) if act != "none" else "none"
        return dict(op=op, m=m, n=n, k=k, act=act, bias=rng.random() < 0.7, residual=rng.random() < 0.5, save=save)
    if op == "gated":
        return dict(op=op, m=m, n=n, k=k, act=act, save=rng.choice(["none", "fp32", "8bit"]))
    return dict(op=op, m=m, n=n, k=k, act=act, held=rng.choice(["fp32", "8bit"]), padded=rng.random() < 0.5)


# ---------------------------------------------------------------------------------------------- what a program has in hand

def _ck8_bytes(rows, cols):
    return (rows * cols + 15) // 16 * 16 + rows * ((cols + GROUP - 1) // GROUP)


def _groups(x):
    rows, cols = x.shape
    return torch.nn.functional.pad(x, (0, -cols % GROUP)).view(rows, -1, GROUP)


def _quantise(x):
    """(q, exponent byte): the smallest power of two 2^e with 127 * 2^e >= the group's largest magnitude, values
    rounded to the nearest multiple, ties to even."""
    v = _groups(x)
    mant, p = torch.frexp(v.abs().amax(-1))
    e = torch.clamp(p - 7 + (mant > 127 / 128).int(), min=-126)
    q = torch.round(torch.ldexp(v.double(), -e.unsqueeze(-1))).to(torch.int8)
    return q, (e + 127).to(torch.uint8)


def _stand_for(q, eb, cols):
    """The values of a checkpoint: exact in 16 bits, and in 32."""
    v = q.float() * torch.exp2(eb.float() - 127).unsqueeze(-1)
    return v.view(q.shape[0], -1)[:, :cols].contiguous()


def _checkpoint(x):
    rows, cols = x.shape
    q, eb = _quantise(x)
    buf = torch.zeros(_ck8_bytes(rows, cols), dtype=torch.uint8, device="cuda")
    buf[: rows * cols] = q.view(rows, -1)[:, :cols].reshape(-1).view(torch.uint8)
    buf[buf.numel() - eb.numel():] = eb.reshape(-1)
    return buf


def _open_checkpoint(buf, rows, cols):
    n_exp = rows * ((cols + GROUP - 1) // GROUP)
    q = _groups(buf[: rows * cols].view(torch.int8).view(rows, cols))
    return _stand_for(q, buf[buf.numel() - n_exp:].view(rows, -1), cols)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape, std=1.0, mean=0.0):
        return torch.randn(*shape, generator=gen, device="cuda") * std + mean

    s = dict(case=case)
    op = case["op"]
    if op == "ck8_save_load":
        s["x"] = normal(case["rows"], case["cols"]) * torch.exp(normal(case["rows"], 1))
        return s
    if op == "ck8_gelu_bwd":
        s["ck"] = _checkpoint(normal(case["rows"], case["cols"]))
        s["dy"] = normal(case["rows"], case["cols"], std=1e-3)
        return s
    m, n, k = case["m"], case["n"], case["k"]
    x = normal(m, k)  # what layer normalisation hands on
    std_w = 0.02 if k >= 256 else k ** -0.5
    if op.startswith("linear"):
        s["w"], s["bias"] = normal(n, k, std=std_w), normal(n, std=0.02)
        if op == "linear":
            s["x"] = x
            s["bias"] = s["bias"] if case["bias"] else None
            s["residual"] = normal(m, n) if case["residual"] else None
            return s
        pre = [("pre", x @ s["w"].T + s.pop("bias"))] if case["act"] != "none" else []
        dy = "dy"
    else:
        s["wg"], s["wu"] = normal(n, k, std=std_w), normal(n, k, std=std_w)
        s["bg"], s["bu"] = normal(n, std=0.02), normal(n, std=0.02)
        if op == "gated":
            s["x"] = x
            return s
        pre = [("g", x @ s["wg"].T + s.pop("bg")), ("u", x @ s["wu"].T + s.pop("bu"))]
        dy = "dh"
    s.pop("bias", None)
    s[dy] = normal(m, n, std=1e-3)
    if case["padded"]:
        s[dy][m - m // 8:] = 0.0
    for name, t in pre + [("x", x)]:
        if case["held"] == "8bit":
            s[name + "8"] = _checkpoint(t)
        else:
            s[name] = t
    return s


# ---------------------------------------------------------------------------------------------- the plain forms

def _act(v, act):
    if act == "gelu":
        return 0.5 * v * (1.0 + torch.erf(v * 0.5 ** 0.5))
    return v / (1.0 + torch.exp(-v)) if act == "silu" else v


def _act_grad(v, act):
    if act == "gelu":
        return 0.5 * (1.0 + torch.erf(v * 0.5 ** 0.5)) + v * torch.exp(-0.5 * v * v) * (1.0 / math.sqrt(2.0 * math.pi))
    if act == "silu":
        sig = 1.0 / (1.0 + torch.exp(-v))
        return sig * (1.0 + v * (1.0 - sig))
    return torch.ones_like(v)


def _held(s, name, rows, cols):
    return s[name] if name in s else _open_checkpoint(s[name + "8"], rows, cols)


def _saved(v, save):
    """What a forward pass keeps of a pre-activation, as a list of outputs. The values of a checkpoint have 7 bits."""
    if save == "fp32":
        return [v]
    return [_stand_for(*_quantise(v), v.shape[1]).bfloat16()] if save == "8bit" else []


def _plain_linear(s, c):
    pre = s["x"] @ s["w"].T
    if s["bias"] is not None:
        pre = pre + s["bias"]
    y = _act(pre, c["act"])
    if s["residual"] is not None:
        y = y + s["residual"]
    return [y] + _saved(pre, c["save"])


def _plain_linear_bwd(s, c):
    m, n, k = c["m"], c["n"], c["k"]
    dpre = s["dy"] if c["act"] == "none" else s["dy"] * _act_grad(_held(s, "pre", m, n), c["act"])
    return [dpre @ s["w"], dpre.T @ _held(s, "x", m, k), dpre.sum(0)]


def _plain_gated(s, c):
    g, u = s["x"] @ s["wg"].T + s["bg"], s["x"] @ s["wu"].T + s["bu"]
    return [_act(g, c["act"]) * u] + _saved(g, c["save"]) + _saved(u, c["save"])


def _plain_gated_bwd(s, c):
    m, n, k = c["m"], c["n"], c["k"]
    g, u, x = _held(s, "g", m, n), _held(s, "u", m, n), _held(s, "x", m, k)
    dg, du = s["dh"] * u * _act_grad(g, c["act"]), s["dh"] * _act(g, c["act"])
    return [dg @ s["wg"] + du @ s["wu"], dg.T @ x, du.T @ x, dg.sum(0), du.sum(0)]


def _plain_ck8_save_load(s, c):
    return [_stand_for(*_quantise(s["x"]), c["cols"])]


def _plain_ck8_gelu_bwd(s, c):
    return [s["dy"] * _act_grad(_open_checkpoint(s["ck"], c["rows"], c["cols"]), "gelu")]


# ---------------------------------------------------------------------------------------------- the framework's calls

@functools.lru_cache(maxsize=1)
def _library():
    from soliton_b200 import tensor
    from soliton_b200._C import lib
    tensor._dev(tensor.CUDA)
    return lib


def _ptr(t):
    return None if t is None else t.data_ptr()


def _ok(rc):
    if rc != 0:
        raise RuntimeError("soliton_b200: the call returned %d" % rc)


def _new(*shape):
    return torch.empty(shape, device="cuda")


def _to_save(m, n, save):
    """(fp32 buffer, checkpoint buffer) for a pre-activation that a forward pass keeps."""
    return (_new(m, n) if save == "fp32" else None,
            torch.empty(_ck8_bytes(m, n), dtype=torch.uint8, device="cuda") if save == "8bit" else None)


def _kept(lib, full, ck, m, n):
    if ck is None:
        return [] if full is None else [full]
    v = _new(m, n)
    _ok(lib.slb_ck8_load(CUDA, _ptr(ck), _ptr(v), m, n))
    return [v.bfloat16()]


def _own_linear(s, c):
    lib, m, n, k = _library(), c["m"], c["n"], c["k"]
    y, (pre, pre8) = _new(m, n), _to_save(m, n, c["save"])
    _ok(lib.slb_linear(CUDA, _ptr(s["x"]), _ptr(s["w"]), _ptr(s["bias"]), _ptr(s["residual"]), _ptr(y), _ptr(pre), _ptr(pre8),
                       m, n, k, ACT[c["act"]]))
    return [y] + _kept(lib, pre, pre8, m, n)


def _own_linear_bwd(s, c):
    lib, m, n, k = _library(), c["m"], c["n"], c["k"]
    dx, dw, db = _new(m, k), _new(n, k), _new(n)
    _ok(lib.slb_linear_bwd(CUDA, _ptr(s["dy"]), _ptr(s.get("x")), _ptr(s.get("x8")), _ptr(s["w"]), _ptr(s.get("pre")),
                           _ptr(s.get("pre8")), _ptr(dx), _ptr(dw), _ptr(db), m, n, k, ACT[c["act"]]))
    return [dx, dw, db]


def _own_gated(s, c):
    lib, m, n, k = _library(), c["m"], c["n"], c["k"]
    h, (g, g8), (u, u8) = _new(m, n), _to_save(m, n, c["save"]), _to_save(m, n, c["save"])
    _ok(lib.slb_gated(CUDA, _ptr(s["x"]), _ptr(s["wg"]), _ptr(s["wu"]), _ptr(s["bg"]), _ptr(s["bu"]), _ptr(h), _ptr(g),
                      _ptr(u), _ptr(g8), _ptr(u8), m, n, k, ACT[c["act"]]))
    return [h] + _kept(lib, g, g8, m, n) + _kept(lib, u, u8, m, n)


def _own_gated_bwd(s, c):
    lib, m, n, k = _library(), c["m"], c["n"], c["k"]
    dx, dwg, dwu, dbg, dbu = _new(m, k), _new(n, k), _new(n, k), _new(n), _new(n)
    _ok(lib.slb_gated_bwd(CUDA, _ptr(s["dh"]), _ptr(s.get("x")), _ptr(s.get("x8")), _ptr(s["wg"]), _ptr(s["wu"]),
                          _ptr(s.get("g")), _ptr(s.get("u")), _ptr(s.get("g8")), _ptr(s.get("u8")), _ptr(dx), _ptr(dwg),
                          _ptr(dwu), _ptr(dbg), _ptr(dbu), m, n, k, ACT[c["act"]]))
    return [dx, dwg, dwu, dbg, dbu]


def _own_ck8_save_load(s, c):
    lib, rows, cols = _library(), c["rows"], c["cols"]
    ck, back = torch.empty(_ck8_bytes(rows, cols), dtype=torch.uint8, device="cuda"), _new(rows, cols)
    _ok(lib.slb_ck8_save(CUDA, _ptr(s["x"]), _ptr(ck), rows, cols))
    _ok(lib.slb_ck8_load(CUDA, _ptr(ck), _ptr(back), rows, cols))
    return [back]


def _own_ck8_gelu_bwd(s, c):
    lib, rows, cols = _library(), c["rows"], c["cols"]
    dx = _new(rows, cols)
    _ok(lib.slb_ck8_gelu_bwd(CUDA, _ptr(s["ck"]), _ptr(s["dy"]), _ptr(dx), rows, cols))
    return [dx]


_PLAIN = dict(linear=_plain_linear, linear_bwd=_plain_linear_bwd, gated=_plain_gated, gated_bwd=_plain_gated_bwd,
              ck8_save_load=_plain_ck8_save_load, ck8_gelu_bwd=_plain_ck8_gelu_bwd)
_OWN = dict(linear=_own_linear, linear_bwd=_own_linear_bwd, gated=_own_gated, gated_bwd=_own_gated_bwd,
            ck8_save_load=_own_ck8_save_load, ck8_gelu_bwd=_own_ck8_gelu_bwd)


def run(state):
    c = state["case"]
    return (_OWN if own else _PLAIN)[c["op"]](state, c)


# ---------------------------------------------------------------------------------------------- work and definition

def work(case):
    """Inputs read once, outputs written once, and the products' multiply-adds."""
    op = case["op"]
    if op.startswith("ck8"):
        n, ck = case["rows"] * case["cols"], _ck8_bytes(case["rows"], case["cols"])
        return {"bytes": 8 * n + (2 * ck if op == "ck8_save_load" else ck), "flops": 0}
    m, n, k = case["m"], case["n"], case["k"]
    x, w, y = m * k, n * k, m * n
    kept = {"none": 0, "fp32": 4 * y, "8bit": _ck8_bytes(m, n)}
    if op == "linear":
        return {"bytes": 4 * (x + w + y * (2 if case["residual"] else 1) + n * case["bias"]) + kept[case["save"]], "flops": 2.0 * m * n * k}
    if op == "gated":
        return {"bytes": 4 * (x + 2 * w + y + 2 * n) + 2 * kept[case["save"]], "flops": 4.0 * m * n * k}
    held_x = 4 * x if case["held"] == "fp32" else _ck8_bytes(m, k)
    if op == "linear_bwd":
        pre = 0 if case["act"] == "none" else kept[case["held"]]
        return {"bytes": 4 * (y + w + x + w + n) + held_x + pre, "flops": 4.0 * m * n * k}
    return {"bytes": 4 * (y + 2 * w + x + 2 * w + 2 * n) + held_x + 2 * kept[case["held"]], "flops": 8.0 * m * n * k}


def _decoded64(buf, rows, cols):
    """A checkpoint's values from its definition, column by column: q * 2^(e - 127)."""
    groups = (cols + GROUP - 1) // GROUP
    q = buf[: rows * cols].to(torch.int16)
    q = torch.where(q > 127, q - 256, q).view(rows, cols).double()
    e = buf[(rows * cols + 15) // 16 * 16:][: rows * groups].view(rows, groups).double() - 127.0
    return q * torch.pow(torch.tensor(2.0, dtype=torch.float64, device="cuda"), e)[:, torch.arange(cols, device="cuda") // GROUP]


def _rounded64(x):
    """The values that a checkpoint of x holds, from the definition, with the step found by search over exponents."""
    rows, cols = x.shape
    out = torch.empty_like(x)
    for at in range(0, cols, GROUP):
        v = x[:, at:at + GROUP]
        top = v.abs().max(dim=1, keepdim=True).values
        e = torch.ceil(torch.log2(torch.clamp(top, min=2.0 ** -140) / 127.0)) - 1.0  # one below, then up until it fits
        for _ in range(2):
            e = torch.where(127.0 * torch.exp2(e) < top, e + 1.0, e)
        step = torch.exp2(torch.clamp(e, min=-126.0))
        out[:, at:at + GROUP] = torch.round(v / step) * step
    return out


def _act64(v, act):
    F = torch.nn.functional
    return F.gelu(v) if act == "gelu" else F.silu(v) if act == "silu" else v


def exact(case, seed):
    """The operators' definitions in 64 bits; gradients by differentiating the definition."""
    s, op = prepare(case, seed), case["op"]
    d = {name: t.double() for name, t in s.items() if isinstance(t, torch.Tensor) and t.dtype == torch.float32}
    if op == "ck8_save_load":
        return [_rounded64(d["x"])]
    if op == "ck8_gelu_bwd":
        x = _decoded64(s["ck"], case["rows"], case["cols"]).requires_grad_()
        return list(torch.autograd.grad(_act64(x, "gelu"), x, d["dy"]))
    m, n, k, act = case["m"], case["n"], case["k"], case["act"]
    for name, cols in (("x", k), ("pre", n), ("g", n), ("u", n)):
        if name + "8" in s:
            d[name] = _decoded64(s[name + "8"], m, cols)
    if op == "linear":
        pre = torch.nn.functional.linear(d["x"], d["w"], d.get("bias"))
        y = _act64(pre, act)
        y = y + d["residual"] if "residual" in d else y
        return [y] + {"none": [], "fp32": [pre], "8bit": [_rounded64(pre) if case["save"] == "8bit" else None]}[case["save"]]
    if op == "gated":
        g, u = (torch.nn.functional.linear(d["x"], d["w" + c], d["b" + c]) for c in "gu")
        keep = {"none": [], "fp32": [g, u], "8bit": [None, None]}[case["save"]]
        return [_act64(g, act) * u] + ([_rounded64(g), _rounded64(u)] if case["save"] == "8bit" else keep)
    if op == "linear_bwd":
        dpre = d["dy"]
        if act != "none":
            pre = d["pre"].requires_grad_()
            dpre, = torch.autograd.grad(_act64(pre, act), pre, d["dy"])
        return [torch.einsum("mn,nk->mk", dpre, d["w"]), torch.einsum("mn,mk->nk", dpre, d["x"]), torch.einsum("mn->n", dpre)]
    g, u = d["g"].requires_grad_(), d["u"].requires_grad_()
    dg, du = torch.autograd.grad(_act64(g, act) * u, (g, u), d["dh"])
    both, w = torch.cat([dg, du], 1), torch.cat([d["wg"], d["wu"]], 0)
    dw = torch.einsum("mn,mk->nk", both, d["x"])
    return [torch.einsum("mn,nk->mk", both, w), dw[:n].contiguous(), dw[n:].contiguous(), dg.sum(0), du.sum(0)]
