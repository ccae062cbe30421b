"""GPU tests of how exactly gx_linear sums: one rounding to the result's type, and errors of the batch product in
the 2-norm."""
import numpy as np
import pytest

import operator_refs as refs
from gyro_moe import abi

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    with abi.Context(device=0, max_tokens=16, max_layers=1) as c:
        yield c


def activations(seed, n, cols, kind):
    x = torch.from_numpy(refs.to_kind(np.random.default_rng(seed).standard_normal((n, cols)), kind))
    return x.to(torch.bfloat16 if kind == "bf16" else torch.float32).cuda()


def linear(ctx, h, x, rows, dtype):
    y = torch.empty(x.shape[0], rows, dtype=dtype, device="cuda")
    torch.cuda.synchronize()
    ctx.wait(ctx.linear(h, x, y))
    return y


@pytest.mark.parametrize("kind", [refs.Q4_0, refs.Q4_1])
@pytest.mark.parametrize("rows,cols,n,xk", [(300, 8192, 64, "bf16"), (2600, 4096, 33, "bf16"), (256, 10240, 13, "f32"),
                                            (20000, 1024, 20, "bf16"), (260, 6144, 30, "f32"), (500, 4096, 40, "f32"),
                                            (500, 2048, 1, "bf16"), (77, 4128, 2, "f32"), (500, 2048, 7, "f32")])
def test_bf16_results_are_the_f32_ones_rounded_once(ctx, kind, rows, cols, n, xk):
    packed, _, _ = refs.q4_matrix(rows, kind, rows, cols)
    h = ctx.upload_matrix(kind, rows, cols, packed)
    x = activations(cols, n, cols, xk)
    assert torch.equal(linear(ctx, h, x, rows, torch.bfloat16), linear(ctx, h, x, rows, torch.float32).bfloat16())


@pytest.mark.parametrize("kind", [refs.Q4_0, refs.Q4_1])
@pytest.mark.parametrize("n,xk", [(13, "f32"), (30, "f32"), (40, "f32"), (13, "bf16"), (64, "bf16")])
def test_batch_sums_are_kept_in_f32(ctx, kind, n, xk):
    """Whole positive numbers: weights up to 511 and activations up to 255, so that the sum of 128 columns is below
    2^24 and exact in f32, while 1792 columns pass 2^26 and a sum that is cut off after every 16 of them loses up to
    three bits each time (1.4e-6 of it and more). Added in f32, rounded to nearest, the 80 sums of 10240 columns in chains of 14
    and of 6 are off by at most 20 half steps."""
    rows, cols = 256, 10240
    rng = np.random.default_rng(n)
    g = cols // 32
    d = rng.integers(32, 74, (rows, g, 1)).astype(np.float16)
    q = rng.integers(9, 16, (rows, g, 32), dtype=np.uint8) if kind == refs.Q4_0 else rng.integers(1, 7, (rows, g, 32), dtype=np.uint8)
    parts = [d.view(np.uint8)]
    if kind == refs.Q4_1:
        parts.append(rng.integers(1, 74, (rows, g, 1)).astype(np.float16).view(np.uint8))
    packed = np.concatenate(parts + [q[..., :16] | (q[..., 16:] << 4)], axis=2).reshape(rows, -1)
    w, _ = refs.q4_weights(packed, kind, cols)
    assert w.min() >= 1 and w.max() <= 511
    h = ctx.upload_matrix(kind, rows, cols, packed)
    x = torch.from_numpy(rng.integers(128, 256, (n, cols)).astype(np.float32)).to(torch.bfloat16 if xk == "bf16" else torch.float32).cuda()
    exact = x.double() @ torch.from_numpy(w).cuda().T
    y = linear(ctx, h, x, rows, torch.float32).double()
    assert float(((y - exact).abs() / exact).max()) <= 20 * 2.0 ** -24
