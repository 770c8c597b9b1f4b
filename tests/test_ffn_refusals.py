"""What the feed-forward and checkpoint entry points refuse, and what they do on meta. No GPU: nothing here launches."""
import pytest

from oracle import ffn_ops as ops

CPU, META, CUDA = 0, 1, 2
A, B, ODD = 4096, 1 << 20, 4098  # addresses that are never followed


@pytest.fixture(autouse=True)
def clean(lib):
    lib.slb_clear_error()
    yield
    lib.slb_clear_error()


def calls(dev, m=4, n=8, k=16, act=1):
    """Every pool-level call with acceptable arguments: name -> list of arguments."""
    return {
        "slb_linear": [dev, A, A, A, A, B, B, B, m, n, k, act],
        "slb_linear_bwd": [dev, A, A, None, A, A, None, B, B, B, m, n, k, act],
        "slb_gated": [dev, A, A, A, A, A, B, B, B, B, B, m, n, k, act],
        "slb_gated_bwd": [dev, A, A, None, A, A, A, A, None, None, B, B, B, B, B, m, n, k, act],
        "slb_ck8_save": [dev, A, B, m, n],
        "slb_ck8_load": [dev, A, B, m, n],
        "slb_ck8_gelu_bwd": [dev, A, A, B, m, n],
    }


@pytest.mark.parametrize("name", list(calls(0)))
def test_devices(lib, name):
    fn = getattr(lib, name)
    assert fn(*calls(CPU)[name]) == -1 and lib.sl_check(CPU) == 13
    lib.slb_clear_error()
    assert fn(*calls(META)[name]) == 0 and lib.sl_check(META) == 0
    for dev in (-1, 3):
        assert fn(*calls(dev)[name]) == -1
    lib.slb_clear_error()
    if lib.sl_cuda_count() == 0:
        assert fn(*calls(CUDA)[name]) == -1 and lib.sl_check(CUDA) == 14


@pytest.mark.parametrize("name", [n for n in calls(0) if "ck8" not in n])
@pytest.mark.parametrize("bad", [dict(m=-1), dict(n=0), dict(n=-3), dict(k=0), dict(m=(1 << 30) + 1), dict(n=1 << 40), dict(m=1 << 30, n=1 << 30),
                                 dict(act=-1), dict(act=3)])
def test_sizes_and_activations(lib, name, bad):
    assert getattr(lib, name)(*calls(META, **bad)[name]) == -1 and lib.sl_check(CUDA) == 12
    if "act" not in bad:
        size = {**dict(m=4, n=8, k=16), **bad}
        assert lib.slb_linear_scratch_bytes(size["m"], size["n"], size["k"], 1) == 0


@pytest.mark.parametrize("name", [n for n in calls(0) if "ck8" in n])
@pytest.mark.parametrize("bad", [dict(m=-1), dict(n=0), dict(m=1 << 35, n=1 << 20)])
def test_checkpoint_sizes(lib, name, bad):
    assert getattr(lib, name)(*calls(META, **bad)[name]) == -1 and lib.sl_check(CUDA) == 12
    size = {**dict(m=4, n=8), **bad}
    assert lib.slb_ck8_bytes(size["m"], size["n"]) == 0


# argument position -> value that must be refused (the device argument is position 0)
POINTERS = {
    "slb_linear": [{1: None}, {2: None}, {5: None}, {1: ODD}, {2: ODD}, {3: ODD}, {4: ODD}, {5: ODD}, {6: ODD}],
    "slb_linear_bwd": [{1: None}, {1: ODD}, {2: None}, {3: A}, {4: None}, {5: None}, {6: A}, {7: None, 8: None, 9: None}, {7: ODD}, {8: ODD}, {9: ODD}, {2: ODD},
                       {4: ODD}, {5: ODD}],
    "slb_gated": [{1: None}, {2: None}, {3: None}, {6: None}, {1: ODD}, {4: ODD}, {6: ODD}, {7: ODD}],
    "slb_gated_bwd": [{1: None}, {2: None}, {3: A}, {4: None}, {5: None}, {6: None}, {7: None}, {8: A}, {9: A}, {10: None, 11: None, 12: None, 13: None, 14: None},
                      {1: ODD}, {10: ODD}, {14: ODD}],
    "slb_ck8_save": [{1: None}, {2: None}, {1: ODD}],
    "slb_ck8_load": [{1: None}, {2: None}, {2: ODD}],
    "slb_ck8_gelu_bwd": [{1: None}, {2: None}, {3: None}, {2: ODD}, {3: ODD}],
}


@pytest.mark.parametrize("name,change", [(n, c) for n, cs in POINTERS.items() for c in cs])
def test_pointers(lib, name, change):
    args = calls(CUDA)[name]
    for at, v in change.items():
        args[at] = v
    assert getattr(lib, name)(*args) == -1 and lib.sl_check(CUDA) == 12  # before any device is asked for


@pytest.mark.parametrize("backward", [0, 1])
@pytest.mark.parametrize("which", ["linear", "gated"])
def test_backend_level_scratch(lib, which, backward):
    need = getattr(lib, f"slb_{which}_scratch_bytes")(4, 8, 16, backward)
    assert need > 0 and getattr(lib, f"slb_{which}_scratch_bytes")(0, 8, 16, backward) == 0
    name = f"slb_cuda_{which}" + ("_bwd" if backward else "")
    args = calls(CUDA)[name.replace("cuda_", "")][1:]
    for scratch, size in ((None, need), (1 << 24, need - 1), ((1 << 24) + 64, need)):
        assert getattr(lib, name)(*args, scratch, size) == -1 and lib.sl_check(CUDA) == 12
        lib.slb_clear_error()
    if lib.sl_cuda_count() == 0:
        assert getattr(lib, name)(*args, 1 << 24, need) == -1 and lib.sl_check(CUDA) == 14


def test_backward_without_what_it_does_not_need(lib):
    """No activation: no pre-activations; no dw: no x; no dx: no w. Passes the checks (and then finds no device)."""
    if lib.sl_cuda_count() > 0:
        return
    for args in ([CUDA, A, None, None, None, None, None, None, None, B, 4, 8, 16, 0], [CUDA, A, None, None, A, None, None, B, None, None, 4, 8, 16, 0],
                 [CUDA, A, None, A, None, None, A, None, B, None, 4, 8, 16, 2]):
        lib.slb_clear_error()
        assert lib.slb_linear_bwd(*args) == -1 and lib.sl_check(CUDA) == 14


def test_meta_takes_the_scratch_from_the_pool(lib):
    import ctypes
    from soliton_b200 import tensor as Tn
    Tn._dev(META)
    for name, scratch in (("slb_linear", lib.slb_linear_scratch_bytes(4, 8, 16, 0)), ("slb_linear_bwd", lib.slb_linear_scratch_bytes(4, 8, 16, 1)),
                          ("slb_gated", lib.slb_gated_scratch_bytes(4, 8, 16, 0)), ("slb_gated_bwd", lib.slb_gated_scratch_bytes(4, 8, 16, 1))):
        before, after = (ctypes.c_int64 * 7)(), (ctypes.c_int64 * 7)()
        lib.sl_reset_stats(META)
        lib.sl_stats(META, before)
        assert getattr(lib, name)(*calls(META)[name]) == 0
        lib.sl_stats(META, after)
        assert after[0] == before[0] and after[2] - before[0] == (scratch + 511) // 512 * 512 and after[4] == before[4] + 1
        assert getattr(lib, name)(*calls(META, m=0)[name]) == 0


def test_scratch_covers_the_planes(lib):
    """Four bytes a value of the operands, whole blocks of 64; the column sums; and no more than what the sums of cut tiles
    need: 3 x 74 accumulators of 256 x 256 at the most."""
    def blocks(n):
        return (n + 63) // 64

    for m, n, k in ((1, 1, 1), (64, 64, 64), (65, 129, 193), (8192, 768, 768), (768, 8192, 100)):
        fwd = 16384 * (blocks(m) * blocks(k) + blocks(n) * blocks(k))
        bwd = fwd + 16384 * blocks(m) * blocks(n) + 4 * blocks(m) * n
        cut = 3 * 74 * 256 * 256 * 4 + 16 * 1024
        assert fwd <= lib.slb_linear_scratch_bytes(m, n, k, 0) <= fwd + 256 * (blocks(m) + blocks(n)) + cut
        assert bwd <= lib.slb_linear_scratch_bytes(m, n, k, 1) <= bwd + cut
        assert lib.slb_gated_scratch_bytes(m, n, k, 1) >= bwd


def test_checkpoint_bytes(lib):
    for rows, cols in ((0, 5), (1, 1), (3, 31), (7, 33), (100000, 50257)):
        assert lib.slb_ck8_bytes(rows, cols) == ops.ck8_bytes(rows, cols)
