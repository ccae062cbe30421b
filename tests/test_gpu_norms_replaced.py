"""GPU test of gx_upload_norms on a layer that has norms: the next gx_norm_block uses the new ones, and a refused
call leaves the ones before."""
import numpy as np
import pytest

from gyro_moe import abi, synth

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


def test_replaced_norms_are_used_at_once():
    E, n = 2048, 3
    rng = np.random.default_rng(0)
    res = torch.from_numpy(rng.normal(0, 2, (n, E)).astype(np.float32)).cuda()
    with abi.Context(device=0, max_tokens=16, max_layers=1) as ctx:
        ctx.upload_layer(0, synth.make_layer(1, n_expert=8, E=E, F=128, U=2))

        def block():
            r = res.clone()
            torch.cuda.synchronize()
            ctx.wait(ctx.norm_block(0, 1, r))
            return r

        def norms(k):
            g = np.random.default_rng(k)
            return dict(pre=g.normal(1, 0.2, E).astype(np.float32), post=g.normal(1, 0.2, E).astype(np.float32),
                        gate=g.normal(0, 0.02, E).astype(np.float32))

        want = []
        for k in range(8):
            ctx.upload_norms(0, None)
            ctx.upload_norms(0, norms(k))
            want.append(block())
        assert not torch.equal(want[0], want[1])
        for k in list(range(8)) * 5:
            ctx.upload_norms(0, norms(k))
            assert torch.equal(block(), want[k])
        with pytest.raises(abi.GxError) as e:
            ctx.upload_norms(0, dict(norms(3), eps=-1.0))
        assert e.value.code == -1 and torch.equal(block(), want[7])
