"""GPU test of gx_matvec on 4-bit matrices: the argument rules are those of gx_linear."""
import numpy as np
import pytest

import operator_refs as refs
from gyro_moe import abi

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


def test_matvec_refuses_what_linear_refuses():
    packed, w, mag = refs.q4_matrix(8, refs.Q4_0, 24, 128)
    with abi.Context(device=0, max_tokens=16, max_layers=1) as ctx:
        h = ctx.upload_matrix(refs.Q4_0, 24, 128, packed)
        x = np.random.default_rng(2).normal(0, 1, (3, 128)).astype(np.float32)
        buf = torch.zeros(2048, device="cuda")
        buf[:384] = torch.from_numpy(x).reshape(-1).cuda()
        torch.cuda.synchronize()
        at, one = buf.data_ptr(), abi.ctypes.c_uint64()
        call = lambda xp, n, yp: ctx.lib.gx_matvec(ctx.handle, h, xp, n, yp, abi.ctypes.byref(one))  # noqa: E731
        # y over x, at its start and from its last value on; pointers that are not whole floats; too many tokens
        for xp, n, yp in [(at, 3, at), (at, 3, at + 4 * 383), (at + 4 * 100, 3, at + 4 * 80), (at, 3, at + 4 * 500 + 2),
                          (at + 2, 2, at + 4 * 500), (at, 65, at + 4 * 500), (None, 1, at), (at, 1, None)]:
            assert call(xp, n, yp) == -1, (xp, n, yp)
        torch.cuda.synchronize()
        assert bool((buf[384:] == 0).all()) and np.array_equal(buf[:384].cpu().numpy(), x.reshape(-1))
        assert call(at, 3, at + 4 * 384) == 0
        ctx.wait(one.value)
        y, (want, bound) = buf[384:456].view(3, 24).cpu().numpy(), refs.linear(x, w, mag, "f32")
        assert (np.abs(y - want) <= bound).all()
