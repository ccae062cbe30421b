"""CPU tests of the Python binding's operator calls with handles, layers and tensors that do not fit."""
import ctypes

import pytest

from gyro_moe import abi

torch = pytest.importorskip("torch")


class Library:
    """Answers every call as the library answers an argument or state that it refuses."""

    def __init__(self, code):
        self.code, self.calls = code, []

    def __getattr__(self, name):
        def call(*args):
            self.calls.append(name)
            return self.code
        return call


def context(code):
    ctx = abi.Context.__new__(abi.Context)
    ctx.handle, ctx.lib, ctx.matrices, ctx.layers, ctx.device = None, Library(code), {0: (8, 64)}, {}, -1
    ctx._ticket = ctypes.c_uint64()
    ctx._ticket_ref = ctypes.byref(ctx._ticket)
    return ctx


def test_an_unknown_handle_or_layer_is_the_librarys_to_refuse():
    f = torch.zeros
    for code, call in [(-1, lambda c: c.linear(7, f(2, 64), f(2, 8))), (-1, lambda c: c.matvec(7, f(2, 64), f(2, 8))),
                       (-6, lambda c: c.upload_norms(3, {"pre": f(32).numpy()}))]:
        ctx = context(code)
        with pytest.raises(abi.GxError) as e:
            call(ctx)
        assert e.value.code == code and len(ctx.lib.calls) == 1


def test_matvec_checks_its_tensors():
    f = torch.zeros
    ctx = context(0)
    for x, y in [(f(2, 64), f(3, 8)), (f(2, 32), f(2, 8)), (f(2, 64), f(2, 9)), (f(2, 64).bfloat16(), f(2, 8)),
                 (f(2, 64), f(2, 8).bfloat16()), (f(2, 80)[:, :64], f(2, 8)), (f(2, 64), f(2, 16)[:, :8]), (f(64, 2).T, f(2, 8))]:
        with pytest.raises(ValueError):
            ctx.matvec(0, x, y)
    assert not ctx.lib.calls
    ctx.matvec(0, f(2, 64), f(2, 8))
    ctx.matvec(0, f(0, 64), f(0, 8))
    assert ctx.lib.calls == ["gx_matvec"] * 2
    ctx.device = 0
    with pytest.raises(ValueError, match="device"):
        ctx.matvec(0, f(2, 64), f(2, 8))
