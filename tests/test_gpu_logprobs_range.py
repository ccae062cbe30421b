"""GPU test of gx_logprobs where a row has one certain token, or nearly: probabilities are at most 1 and the entropy
is at least 0, whatever the sums round to."""
import numpy as np
import pytest

import operator_refs as refs
from gyro_moe import abi

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

DT = {"f32": torch.float32, "bf16": torch.bfloat16}


@pytest.mark.parametrize("V,n", [(33, 600), (5000, 600), (40000, 40), (150001, 12)])
@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("n_top", [0, 3])
def test_certain_tokens(V, n, kind, n_top):
    """A token 0 to 120 above the others, at the row's start, middle and end, in every other row with a second one 4
    to 5.6 (8 ln 2 is 5.55, the most that the kernel's reference may lie below the largest) under it."""
    rng = np.random.default_rng(V)
    x = rng.normal(0, 0.01, (n, V)).astype(np.float32)
    at = rng.integers(0, V, n)
    at[::3], at[1::3] = 0, V - 1
    x[np.arange(n), at] += np.linspace(0, 120, n).astype(np.float32)
    other = (at + rng.integers(1, V, n)) % V
    x[np.arange(0, n, 2), other[::2]] = x[np.arange(0, n, 2), at[::2]] - rng.uniform(4, 5.6, len(other[::2])).astype(np.float32)
    x = refs.to_kind(x, kind)
    with abi.Context(device=0, max_tokens=16, max_layers=1) as ctx:
        lp, ent = torch.empty(n, device="cuda"), torch.empty(n, device="cuda")
        ids = torch.empty(n, n_top, dtype=torch.int32, device="cuda") if n_top else None
        top = torch.empty(n, n_top, device="cuda") if n_top else None
        xd, tok = torch.from_numpy(x).to(DT[kind]).cuda(), torch.from_numpy(at.astype(np.int32)).cuda()
        torch.cuda.synchronize()
        for scale in (1.0, 0.3, 7.0):
            ctx.wait(ctx.logprobs(xd, tok, logprob=lp, entropy=ent, n_top=n_top, top_ids=ids, top_logprobs=top, scale=scale))
            want, bounds = refs.logprobs(x, at.astype(np.uint32), n_top, scale)
            got = {"logprob": lp, "entropy": ent} | ({"top_logprobs": top} if n_top else {})
            for name, t in got.items():
                v = t.cpu().numpy().astype(np.float64)
                assert (np.abs(v - want[name]) <= bounds[name]).all(), name
                if name == "entropy":
                    assert v.min() >= 0, v.min()
                else:
                    assert v.max() <= 0, v.max()
