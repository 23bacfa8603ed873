"""linear_cross_entropy: what it refuses, without a GPU.  Nothing is launched."""

import ctypes

import pytest
import torch

from offload_adam_amd import _lib, linear_cross_entropy
from offload_adam_amd.qweight import FP8QWeight

BF16 = torch.bfloat16


def _args(t=4, h=16, v=10, dtype=BF16):
    return (torch.zeros(t, h, dtype=dtype), torch.zeros(v, h, dtype=dtype),
            torch.zeros(t, dtype=torch.int64))


def test_refused_arguments():
    x, w, y = _args()
    for bad, exc in [
        ((None, w, y), TypeError),
        ((x.float(), w.float(), y), TypeError),
        ((x, w.half(), y), TypeError),
        ((x, w, y.int()), TypeError),
        ((x, w, None), TypeError),
        ((x, w[:, :8], y), ValueError),
        ((x, w[0], y), ValueError),
        ((x, w, y[:3]), ValueError),
        ((x, w, y[:, None]), ValueError),
        ((x, w[:0], y), ValueError),
        ((x[:, :0], w[:, :0], y), ValueError),
        ((x, w, y), ValueError),  # CPU tensors: there is no CPU path
    ]:
        with pytest.raises(exc):
            linear_cross_entropy(*bad)
    with pytest.raises(ValueError, match="reduction"):
        linear_cross_entropy(x, w, y, reduction="average")


def test_autocast_casts_before_the_checks():
    x, w, y = _args(dtype=torch.float32)
    for dtype in (BF16, torch.float16):
        with torch.autocast("cpu", dtype=dtype):
            for head in (w, w.to(BF16), FP8QWeight.from_float(w)):
                with pytest.raises(ValueError, match="must be a GPU tensor"):  # only that is left
                    linear_cross_entropy(x, head, y)
            with pytest.raises(TypeError):
                linear_cross_entropy(x.double(), w.double(), y)
            with pytest.raises(TypeError):
                linear_cross_entropy(x, w.double(), y)
    with pytest.raises(TypeError):
        linear_cross_entropy(x, w, y)
    with pytest.raises(TypeError):
        linear_cross_entropy(x.to(BF16), FP8QWeight.from_float(w), y)


def test_ignore_index_is_an_int64():
    """Its low 64 bits would be another index."""
    for bad in (2**63, 2**64 - 100, -2**63 - 1):
        with pytest.raises(ValueError, match="ignore_index"):
            linear_cross_entropy(*_args(), ignore_index=bad)
    for good in (2**63 - 1, -2**63, torch.tensor(3), True):
        with pytest.raises(ValueError, match="must be a GPU tensor"):  # only that is left
            linear_cross_entropy(*_args(), ignore_index=good)


def test_the_meta_device_is_refused_too():
    with pytest.raises(ValueError, match="must be a GPU tensor"):
        linear_cross_entropy(*(t.to("meta") for t in _args()))


def test_the_c_entry_points_refuse_before_any_launch():
    lib = _lib.load()
    buf = (ctypes.c_char * 4096)()
    a = (ctypes.addressof(buf) + 255) // 256 * 256
    ok, odd = ctypes.c_void_p(a), ctypes.c_void_p(a + 2)
    big = ctypes.c_size_t(1 << 40)

    def fwd(x=ok, ldx=16, w=ok, ldw=16, dtype=1, y=ok, t=4, h=16, v=10, red=1, loss=ok, lse=ok,
            count=ok, ws=ok, wsb=big):
        return lib.oa_linear_ce_forward(x, ldx, w, ldw, dtype, y, t, h, v, -100, red, loss, lse,
                                        count, ws, wsb, None)

    def bwd(x=ok, ldx=16, w=ok, ldw=16, dtype=1, y=ok, t=4, h=16, v=10, red=1, lse=ok, count=ok,
            grad=ok, dx=ok, dw=ok, ws=ok, wsb=big):
        return lib.oa_linear_ce_backward(x, ldx, w, ldw, dtype, y, t, h, v, -100, red, lse, count,
                                         grad, dx, dw, ws, wsb, None)

    for f in (fwd, bwd):
        assert f(dtype=0) == -1 and f(dtype=7) == -1
        assert f(red=3) == -1
        assert f(t=-1) == -1 and f(h=0) == -1 and f(v=0) == -1
        assert f(x=None) == -1 and f(w=None) == -1 and f(y=None) == -1 and f(ws=None) == -1
        assert f(ldx=8) == -1 and f(ldw=8) == -1  # shorter than a row
        assert f(t=1, ldx=8) == -1
        assert f(h=12, ldx=16, ldw=16) == -2 and f(ldx=20) == -2 and f(ldw=20) == -2
        assert f(x=odd) == -2 and f(w=odd) == -2 and f(ws=odd) == -2
        assert f(ldx=1 << 21) == -3 and f(t=(1 << 22) + 1) == -3 and f(v=(1 << 24) + 1) == -3
        assert f(wsb=ctypes.c_size_t(8)) == -1
    assert fwd(loss=None) == -1 and fwd(lse=None) == -1 and fwd(count=None) == -1
    assert bwd(t=0) == -1 and bwd(grad=None) == -1 and bwd(dx=None, dw=None) == -1
    assert bwd(dx=odd) == -2
    assert lib.oa_linear_ce_workspace_bytes(-1, 16, 10, 0, 0, 0) == 0
    for sizes in ((1 << 40, 16, 1 << 40), (4, 1 << 62, 10), (4, 16, (1 << 24) + 1)):
        for backward in (0, 1):
            assert lib.oa_linear_ce_workspace_bytes(*sizes, backward, 1, 1) == 0
    assert lib.oa_linear_ce_workspace_bytes(0, 16, 10, 0, 0, 0) > 0
    # a backward pass holds far less than the logits of the 8B model's micro-batch in fp32
    assert lib.oa_linear_ce_workspace_bytes(4096, 4096, 128256, 1, 1, 1) < 4096 * 128256 * 4 // 3
