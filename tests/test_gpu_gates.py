"""GPU tests of the gates of gx_norm_residual over the whole range of their logits."""
import numpy as np
import pytest

from gyro_moe import abi

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

U32 = 2.0 ** -24
DT = {"f32": torch.float32, "bf16": torch.bfloat16}
SPECIAL = [0.0, -0.0, 87.0, 88.0, 88.5, 88.7, 88.73, 89.0, 90.5, 95.0, 100.0, 103.9, 104.0, 128.0, 500.0, 1e3, 9999.0, 1e4,
           10001.0, 1e30, 3e38, np.inf]


@pytest.fixture(scope="module")
def ctx():
    with abi.Context(device=0, max_tokens=16, max_layers=1) as c:
        yield c


def sweep(kind):
    g = np.concatenate([np.arange(-200.0, 200.0, 0.03), np.linspace(-11000.0, -89.0, 1500), SPECIAL, -np.array(SPECIAL)])
    return torch.from_numpy(g.astype(np.float32)).to(DT[kind]).float().numpy()


def check(got, logits):
    """res_out = gate where the block's output is 1 and the residual 0. The power of two is off by at most 2^-22 of
    itself (4 u), its correction, 1 + e and the product with block_scale by u, the quotient by 2 u; a gate below the
    smallest normal f32 may be 0."""
    with np.errstate(over="ignore"):
        want = 1.0 / (1.0 + np.exp(-logits.astype(np.float64)))
    got = got.cpu().numpy().astype(np.float64)
    assert not np.isnan(got).any(), logits[np.isnan(got)][:10]
    off = np.abs(got - want) - (9 * U32 * want + 2.0 ** -126)
    assert off.max() <= 0, (logits[off.argmax()], got[off.argmax()], want[off.argmax()])


# through 16-byte accesses and single ones, one, two and four vectors a thread, and the rows too long for registers
@pytest.mark.parametrize("width", [8, 31, 1000, 1023, 4096, 8192, 16384, 16400, 20001])
@pytest.mark.parametrize("kind", ["f32", "bf16"])
def test_element_gates_over_their_range(ctx, width, kind):
    g = sweep(kind)
    n = -(-len(g) // width)
    logits = np.concatenate([g, np.zeros(n * width - len(g), np.float32)])
    gate = torch.from_numpy(logits).to(DT[kind]).view(n, width).cuda()
    one, res = torch.ones(n, width, device="cuda"), torch.zeros(n, width, device="cuda")
    torch.cuda.synchronize()
    ctx.wait(ctx.norm_residual(one, res, post_norm=False, gate=gate))
    check(res.view(-1), logits)


@pytest.mark.parametrize("width", [8, 31, 2048, 16400])
def test_token_gates_over_their_range(ctx, width):
    g = sweep("f32") if width < 100 else np.concatenate([SPECIAL, -np.array(SPECIAL), np.linspace(-1000, -88, 60)]).astype(np.float32)
    one, res = torch.ones(len(g), width, device="cuda"), torch.zeros(len(g), width, device="cuda")
    gate = torch.from_numpy(g).cuda()
    torch.cuda.synchronize()
    ctx.wait(ctx.norm_residual(one, res, post_norm=False, gate=gate))
    assert bool((res == res[:, :1]).all())
    check(res[:, 0], g)


def test_closed_gates_leave_the_residual_and_a_nan_stays_a_nan(ctx):
    """Logits far below zero close their element, or their row; the next norm sees the residual alone."""
    rng = np.random.default_rng(0)
    for width in (64, 63, 16500):
        y = torch.from_numpy(rng.normal(0, 1, (6, width)).astype(np.float32)).cuda()
        res = torch.from_numpy(rng.normal(0, 1, (6, width)).astype(np.float32)).cuda()
        keep, out, plain = res.clone(), torch.empty_like(res), torch.empty_like(res)
        gate = torch.tensor([-95.0, -500.0, -1e3, -9999.0, -3e38, -np.inf], device="cuda")
        torch.cuda.synchronize()
        ctx.wait(ctx.norm_residual(y, res, gate=gate, out=out))
        ctx.wait(ctx.norm(keep, plain))
        assert torch.equal(res, keep)
        # two kernels may order the sum of squares differently: chains of width / 32 + 32 additions at most
        assert float(((out - plain).abs() / plain.abs()).max()) <= (width / 32 + 32 + 16) * U32
        el = torch.zeros(6, width, device="cuda")
        el[2, 5] = float("nan")
        torch.cuda.synchronize()
        ctx.wait(ctx.norm_residual(y, res, gate=el))
        nan = torch.isnan(res)
        assert int(nan.sum()) == 1 and bool(nan[2, 5])
