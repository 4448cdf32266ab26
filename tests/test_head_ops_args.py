"""What the C-ABI of the head's operators refuses, on a host without a GPU: every refusal comes before
anything is launched or read (the addresses here are never used)."""

import ctypes
import os

import pytest

REPO = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
LIB = os.path.join(REPO, "qwen0.6b_amd", "libqwen_megakernel.so")

vp, i32, i64 = ctypes.c_void_p, ctypes.c_int, ctypes.c_longlong
ERR_ARG = 1
F16, BF16, F32 = 0, 1, 2
A = 0x10000  # an aligned address


@pytest.fixture(scope="module")
def lib():
    if not os.path.exists(LIB):
        pytest.skip("library not built")
    lib = ctypes.CDLL(LIB)
    lib.qwen_cross_entropy.argtypes = [vp, i64, vp, i64, vp, i32, i32, i32, i32, i32, i64, vp, vp, vp, vp, i64, vp]
    lib.qwen_cross_entropy_workspace.argtypes = [i32, i32, i32]
    lib.qwen_cross_entropy_workspace.restype = i64
    lib.qwen_cross_entropy_backward.argtypes = [vp, i64, vp, vp, i64, vp, i64, vp, i32, i32, i32, i32, i32, i64, vp, vp, vp,
                                                vp, vp, i64, vp]
    lib.qwen_cross_entropy_backward_workspace.argtypes = [i32, i32, i32, i32, i32]
    lib.qwen_cross_entropy_backward_workspace.restype = i64
    lib.qwen_quantize_rows.argtypes = [vp, i64, i32, i32, i32, vp, vp, vp]
    lib.qwen_matmul_i8.argtypes = [vp, vp, vp, vp, vp, i32, i32, i32, i32, vp]
    return lib


FORWARD = dict(hidden=A, hidden_stride=64, weight=A, weight_stride=64, targets=A, bits=64, tokens=10, vocab=100, width=64,
               dtype=F16, ignore=-100, loss=A, lse=A, total=None, ws=A, ws_bytes=1 << 30)


@pytest.mark.parametrize("change", [
    dict(hidden=None), dict(weight=None), dict(targets=None), dict(loss=None), dict(lse=None), dict(ws=None),
    dict(hidden=A + 8), dict(weight=A + 2), dict(ws=A + 4), dict(targets=A + 4), dict(bits=16), dict(dtype=F32), dict(dtype=-1),
    dict(tokens=-1), dict(tokens=(1 << 20) + 1), dict(vocab=0), dict(vocab=(1 << 24) + 1), dict(width=0), dict(width=60),
    dict(hidden_stride=56), dict(hidden_stride=68), dict(weight_stride=60), dict(weight_stride=1 << 22), dict(ws_bytes=0),
])
def test_cross_entropy(lib, change):
    a = {**FORWARD, **change}
    assert lib.qwen_cross_entropy(*a.values(), None) == ERR_ARG
    b = dict(grad=A, grad_stride=1, divisor=None, **{k: v for k, v in a.items() if k not in ("loss", "lse", "total", "ws", "ws_bytes")},
             loss=a["loss"], lse=a["lse"], gh=A, gw=A, ws=a["ws"], ws_bytes=a["ws_bytes"])
    assert lib.qwen_cross_entropy_backward(*b.values(), None) == ERR_ARG


@pytest.mark.parametrize("change", [dict(grad=None), dict(grad_stride=-1), dict(gh=None, gw=None), dict(gh=A + 8), dict(gw=A + 2),
                                    dict(tokens=0)])
def test_cross_entropy_backward(lib, change):
    b = dict(grad=A, grad_stride=1, divisor=None, **{k: v for k, v in FORWARD.items() if k not in ("loss", "lse", "total", "ws", "ws_bytes")},
             loss=A, lse=A, gh=A, gw=A, ws=A, ws_bytes=1 << 40)
    b.update(change)
    assert lib.qwen_cross_entropy_backward(*b.values(), None) == ERR_ARG


def test_nothing_to_do_is_no_error(lib):
    assert lib.qwen_cross_entropy(*{**FORWARD, "tokens": 0, "hidden": None, "targets": None}.values(), None) == 0
    assert lib.qwen_quantize_rows(None, 64, 0, 64, F16, None, None, None) == 0
    assert lib.qwen_matmul_i8(None, None, None, None, None, F16, 0, 5, 64, None) == 0
    assert lib.qwen_matmul_i8(None, None, None, None, None, F16, 5, 0, 64, None) == 0


def test_workspaces(lib):
    # sizes only: enough for a workgroup's statistics, a piece of the logits' gradient below 128 MB and what goes with it
    assert lib.qwen_cross_entropy_workspace(0, 100, 64) == 0
    assert 0 < lib.qwen_cross_entropy_workspace(1, 151936, 1024) < 1 << 20
    assert lib.qwen_cross_entropy_workspace(4096, 151936, 1024) < 8 << 20
    full = lib.qwen_cross_entropy_backward_workspace(4096, 151936, 1024, 1, 1)
    assert 128 << 20 <= full < 256 << 20
    assert lib.qwen_cross_entropy_backward_workspace(4096, 151936, 1024, 0, 1) < full
    assert lib.qwen_cross_entropy_backward_workspace(1 << 20, 1 << 24, 64, 1, 1) < 2 << 30


@pytest.mark.parametrize("args", [
    (None, 64, 4, 64, F16, A, A), (A, 64, 4, 64, F16, None, A), (A, 64, 4, 64, F16, A, None), (A + 8, 64, 4, 64, F16, A, A),
    (A, 64, 4, 64, F16, A + 8, A), (A, 64, 4, 64, F32, A, A), (A, 64, -1, 64, F16, A, A), (A, 64, 4, 72, F16, A, A),
    (A, 48, 4, 64, F16, A, A), (A, 68, 4, 64, F16, A, A), (A, 64, 4, 0, F16, A, A),
])
def test_quantize_rows(lib, args):
    assert lib.qwen_quantize_rows(*args, None) == ERR_ARG


@pytest.mark.parametrize("args", [
    (None, A, A, A, A, F16, 4, 4, 64), (A, None, A, A, A, F16, 4, 4, 64), (A, A, None, A, A, F16, 4, 4, 64),
    (A, A, A, None, A, F16, 4, 4, 64), (A, A, A, A, None, F16, 4, 4, 64), (A + 4, A, A, A, A, F16, 4, 4, 64),
    (A, A, A + 4, A, A, F16, 4, 4, 64), (A, A, A, A, A + 4, F16, 4, 4, 64), (A, A, A, A, A, 3, 4, 4, 64),
    (A, A, A, A, A, F16, -1, 4, 64), (A, A, A, A, A, F16, 4, -1, 64), (A, A, A, A, A, F16, 4, 4, 24),
    (A, A, A, A, A, F16, 4, 4, 0), (A, A, A, A, A, F16, 4, 4, 65552), (A, A, A, A, A, F16, 4, (1 << 22) + 1, 64),
    (A, A, A, A, A, F16, (1 << 20) + 1, 4, 64),
])
def test_matmul_i8(lib, args):
    assert lib.qwen_matmul_i8(*args, None) == ERR_ARG


def test_prefill_hidden(lib):
    f = lib.qwen_prefill_hidden
    f.argtypes = [vp, i32] + [vp] * 9 + [i32, i32, i32, ctypes.c_float, vp]
    good = [A, 4, A, A, A, A, A, A, A, A, A, 2, 0, 64, 1.0, None]
    for at, value in ((0, None), (4, None), (4, A + 8), (10, None), (10, A + 2), (9, None), (1, 0), (1, 65), (11, 0), (13, 63)):
        args = list(good)
        args[at] = value
        assert f(*args) == ERR_ARG, (at, value)
