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


@pytest.mark.parametrize("kind", [refs.Q4_0, refs.Q4_1])
@pytest.mark.parametrize("xk", ["f32", "bf16"])
@pytest.mark.parametrize("n", [1, 2, 3, 7, 20, 40])
def test_activations_near_the_end_of_the_range(ctx, kind, xk, n):
    """Activations up to the largest f32 by small weights: every sum of the definition is finite, and so are the results."""
    rows, cols = 70, 2080
    rng = np.random.default_rng(n)
    g = cols // 32
    q = rng.integers(0, 16, (rows, g, 32), dtype=np.uint8)
    half = [(rng.choice([-1, 1], (rows, g, 1)) * 2.0 ** rng.uniform(-23, -19, (rows, g, 1))).astype(np.float16) for _ in range(kind - 1)]
    packed = np.concatenate([h.view(np.uint8) for h in half] + [q[..., :16] | (q[..., 16:] << 4)], axis=2).reshape(rows, -1)
    w, mag = refs.q4_weights(packed, kind, cols)
    h = ctx.upload_matrix(kind, rows, cols, packed)
    for low, high in [(1e33, 1e35), (1e35, 3e37), (3e37, 3.38e38)]:
        x = rng.choice([-1, 1], (n, cols)) * np.exp(rng.uniform(np.log(low), np.log(high), (n, cols)))
        x[0] = np.abs(x[0])
        x = refs.to_kind(x.astype(np.float32), xk)
        assert np.isfinite(x).all()
        xd = torch.from_numpy(x).to(torch.bfloat16 if xk == "bf16" else torch.float32).cuda()
        want, bound = refs.linear(x, w, mag, "f32")
        assert np.abs(want).max() < 3e38
        y = linear(ctx, h, xd, rows, torch.float32).cpu().numpy().astype(np.float64)
        assert np.isfinite(y).all() and (np.abs(y - want) <= bound).all(), (low, high)


@pytest.mark.parametrize("kind", [refs.Q4_0, refs.Q4_1])
@pytest.mark.parametrize("xk", ["f32", "bf16"])
@pytest.mark.parametrize("n", [1, 2, 3, 7, 20, 40])
def test_activations_near_the_smallest(ctx, kind, xk, n):
    """Activations around the smallest normal f32 by large weights: results of ordinary relative error."""
    rows, cols = 70, 2080
    rng = np.random.default_rng(n)
    g = cols // 32
    q = rng.integers(0, 16, (rows, g, 32), dtype=np.uint8)
    half = [(rng.choice([-1, 1], (rows, g, 1)) * rng.uniform(3e4, 6.5e4, (rows, g, 1))).astype(np.float16) for _ in range(kind - 1)]
    packed = np.concatenate([h.view(np.uint8) for h in half] + [q[..., :16] | (q[..., 16:] << 4)], axis=2).reshape(rows, -1)
    w, mag = refs.q4_weights(packed, kind, cols)
    h = ctx.upload_matrix(kind, rows, cols, packed)
    for size in (1e-38, 1e-36, 1e-33):
        x = refs.to_kind((rng.standard_normal((n, cols)) * size).astype(np.float32), xk)
        xd = torch.from_numpy(x).to(torch.bfloat16 if xk == "bf16" else torch.float32).cuda()
        want, bound = refs.linear(x, w, mag, "f32")
        y = linear(ctx, h, xd, rows, torch.float32).cpu().numpy().astype(np.float64)
        # a sum is kept in steps of 2^-144 or less (32 times the smallest f32), one half a step lost for each group
        assert (np.abs(y - want) <= bound + cols / 32 * 2.0 ** -144).all(), size
