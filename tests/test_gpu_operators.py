"""GPU tests of the operators around the layer, through the C ABI, against their definitions in 64 bits
(operator_refs.py, which also derives the bounds)."""
import ctypes

import numpy as np
import pytest

import operator_refs as refs
from gyro_moe import abi, synth
from oracle import oracle

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

DT = {"f32": torch.float32, "bf16": torch.bfloat16}


@pytest.fixture(scope="module")
def ctx():
    with abi.Context(device=0, max_tokens=16, max_layers=1) as c:
        yield c


def dev(a, kind="f32", stride=None):
    """A device tensor of the rows of a; with a stride, rows of a wider buffer filled with NaN."""
    t = torch.from_numpy(np.ascontiguousarray(a)).to(DT[kind]).cuda()
    if stride is None:
        return t
    wide = torch.full((t.shape[0], stride), float("nan"), dtype=t.dtype, device="cuda")
    wide[:, :t.shape[1]] = t
    return wide[:, :t.shape[1]]


def out_rows(n, width, kind, stride=None, extra=3):
    """Rows of a larger buffer of a known value, so that writes outside them show."""
    stride = stride or width
    buf = torch.full(((n + extra), stride), 77.0, dtype=DT[kind], device="cuda")
    return buf[:n, :width], buf


def untouched(buf, n, width):
    assert bool((buf[n:] == 77.0).all()) and bool((buf[:, width:] == 77.0).all())


def near(got, want, bound, what=""):
    got = got.float().cpu().numpy().astype(np.float64) if isinstance(got, torch.Tensor) else got
    assert got.shape == want.shape
    fin = np.isfinite(want)
    assert np.array_equal(np.isnan(got), np.isnan(want)), what
    assert np.array_equal(got[~fin & ~np.isnan(want)], want[~fin & ~np.isnan(want)]), what
    off = np.abs(got[fin] - want[fin]) - np.broadcast_to(bound, want.shape)[fin]
    assert off.size == 0 or off.max() <= 0, (what, float(off.max()))


# ---- 4-bit matrices ---------------------------------------------------------------------------
SHAPES = [(1, 32), (3, 32), (8, 64), (15, 96), (16, 128), (17, 160), (33, 544), (130, 1024), (257, 2080), (640, 2560)]


def check_linear(ctx, kind, rows, cols, n, xk, yk, seed=0, xs=None, ys=None, x=None):
    packed, w, mag = refs.q4_matrix(seed + 1, kind, rows, cols)
    h = ctx.upload_matrix(kind, rows, cols, packed)
    if x is None:
        x = np.random.default_rng(seed + 2).normal(0, 1, (n, cols)) * 10.0 ** np.random.default_rng(seed + 3).uniform(-3, 3, (n, 1))
    x = refs.to_kind(x, xk)
    y, buf = out_rows(n, rows, yk, ys)
    ctx.wait(ctx.linear(h, dev(x, xk, xs), y))
    want, bound = refs.linear(x, w, mag, yk)
    near(y, want, bound, (kind, rows, cols, n, xk, yk))
    untouched(buf, n, rows)
    return h


@pytest.mark.parametrize("kind", [refs.Q4_0, refs.Q4_1])
@pytest.mark.parametrize("shape", SHAPES)
def test_linear_shapes(ctx, kind, shape):
    for i, (n, xk, yk) in enumerate([(1, "f32", "f32"), (2, "bf16", "f32"), (3, "f32", "bf16"), (5, "bf16", "bf16")]):
        check_linear(ctx, kind, *shape, n, xk, yk, seed=100 + i)


@pytest.mark.parametrize("n", [1, 4, 5, 8, 9, 12, 16, 17, 31, 32, 33, 48, 63, 64])
@pytest.mark.parametrize("xk", ["f32", "bf16"])
def test_linear_token_counts(ctx, n, xk):
    check_linear(ctx, refs.Q4_0, 200, 416, n, xk, "f32", seed=n)
    check_linear(ctx, refs.Q4_1, 72, 1056, n, xk, "bf16", seed=n + 50)


@pytest.mark.parametrize("rows,cols,n", [(5, 65536, 1), (40, 16384, 3), (33, 32768, 9), (16, 65536, 64), (70001, 64, 2)])
def test_linear_long(ctx, rows, cols, n):
    for xk in ("f32", "bf16"):
        check_linear(ctx, refs.Q4_0 if n != 3 else refs.Q4_1, rows, cols, n, xk, "f32", seed=cols)


@pytest.mark.parametrize("kind", [refs.Q4_0, refs.Q4_1])
@pytest.mark.parametrize("n,xk", [(12, "f32"), (30, "f32"), (64, "f32"), (20, "bf16"), (64, "bf16")])
def test_linear_more_row_blocks_than_multiprocessors(ctx, kind, n, xk):
    check_linear(ctx, kind, 40009, 160, n, xk, "f32", seed=n)


@pytest.mark.parametrize("n,xk", [(2, "f32"), (4, "f32"), (16, "f32"), (40, "bf16")])
@pytest.mark.parametrize("kind", [refs.Q4_0, refs.Q4_1])
def test_linear_scales_at_the_ends_of_fp16(ctx, kind, n, xk):
    """Group scales from the smallest subnormal to the largest fp16, and offsets of Q4_1 alike."""
    rng = np.random.default_rng(n)
    rows, cols = 150, 608
    packed, _, _ = refs.q4_matrix(3, kind, rows, cols)
    blocks = packed.reshape(rows, cols // 32, refs.BLOCK[kind]).copy()
    ends = np.array([2.0 ** -24, 3 * 2.0 ** -24, 1023 * 2.0 ** -24, 2.0 ** -14, 1.0, 2047.0, 65504.0, -65504.0, -2.0 ** -24, 0.0], np.float16)
    for at in range(0, refs.BLOCK[kind] - 16, 2):
        blocks[:, :, at:at + 2] = ends[rng.integers(0, len(ends), blocks.shape[:2] + (1,))].view(np.uint8)
    packed = blocks.reshape(rows, -1)
    w, mag = refs.q4_weights(packed, kind, cols)
    x = refs.to_kind(rng.standard_normal((n, cols)), xk)
    h = ctx.upload_matrix(kind, rows, cols, packed)
    y = torch.empty(n, rows, device="cuda")
    ctx.wait(ctx.linear(h, dev(x, xk), y))
    near(y, *refs.linear(x, w, mag, "f32"))


@pytest.mark.parametrize("n", [1, 7, 40])
def test_linear_strides_and_alignment(ctx, n):
    """Rows of wider buffers at odd strides, and buffers that start at an odd element."""
    for xk, yk in (("f32", "bf16"), ("bf16", "f32")):
        check_linear(ctx, refs.Q4_0, 45, 288, n, xk, yk, seed=n, xs=291, ys=53)
        check_linear(ctx, refs.Q4_1, 45, 288, n, xk, yk, seed=n, xs=296, ys=48)
    packed, w, mag = refs.q4_matrix(9, refs.Q4_0, 24, 96)
    h = ctx.upload_matrix(refs.Q4_0, 24, 96, packed)
    x = refs.to_kind(np.random.default_rng(1).normal(0, 1, (n, 96)), "bf16")
    src = torch.zeros(n * 96 + 1, dtype=torch.bfloat16, device="cuda")
    src[1:] = torch.from_numpy(x).reshape(-1).cuda()
    dst = torch.zeros(n * 24 + 1, dtype=torch.bfloat16, device="cuda")
    ctx.wait(ctx.linear(h, src[1:].view(n, 96), dst[1:].view(n, 24)))
    near(dst[1:].view(n, 24), *refs.linear(x, w, mag, "bf16"))


def test_linear_slices_of_a_fused_buffer(ctx):
    """x and y in columns of one buffer."""
    packed, w, mag = refs.q4_matrix(3, refs.Q4_0, 40, 64)
    h = ctx.upload_matrix(refs.Q4_0, 40, 64, packed)
    x = np.random.default_rng(4).normal(0, 1, (6, 64)).astype(np.float32)
    buf = torch.full((6, 112), 5.0, device="cuda")
    buf[:, 40:104] = torch.from_numpy(x).cuda()
    ctx.wait(ctx.linear(h, buf[:, 40:104], buf[:, :40]))
    near(buf[:, :40], *refs.linear(x, w, mag, "f32"))
    assert bool((buf[:, 104:] == 5.0).all()) and np.array_equal(buf[:, 40:104].cpu().numpy(), x)
    with pytest.raises(abi.GxError):
        ctx.linear(h, buf[:, 39:103], buf[:, :40])


@pytest.mark.parametrize("xk", ["f32", "bf16"])
@pytest.mark.parametrize("n", [1, 6, 24])
def test_linear_extreme_activations(ctx, xk, n):
    """Tokens of zeros, of the type's smallest and largest sizes, of very uneven ones, and one with an
    Inf or NaN next to others, which stay as they are."""
    rng = np.random.default_rng(n)
    packed, w, mag = refs.q4_matrix(5, refs.Q4_1, 37, 320)
    h = ctx.upload_matrix(refs.Q4_1, 37, 320, packed)
    base = rng.normal(0, 1, (6, 320))
    base[0] = 0.0
    base[1] *= 1e-37
    base[2] *= 1e33
    base[3] *= 10.0 ** rng.uniform(-12, 6, 320)
    base[4] = 0.0
    base[4, 300] = 2.5
    x = refs.to_kind(np.concatenate([base] * ((n + 5) // 6))[:n] if n > 1 else base[3:4], xk)
    y, _ = out_rows(n, 37, "f32")
    ctx.wait(ctx.linear(h, dev(x, xk), y))
    want, bound = refs.linear(x, w, mag, "f32")
    # sums below the smallest normal f32 may lose bits to its fixed step
    near(y, want, bound + 320 * 2.0 ** -126)
    if n > 1:
        for bad in (np.inf, -np.inf, np.nan):
            x2 = x.copy()
            x2[1, 77] = bad
            ctx.wait(ctx.linear(h, dev(x2, xk), y))
            got = y.cpu().numpy()
            assert np.isnan(got[1]).all()
            keep = [i for i in range(n) if i != 1]
            near(got[keep].astype(np.float64), want[keep], (bound + 320 * 2.0 ** -126)[keep])


def test_matvec_takes_4bit_matrices(ctx):
    packed, w, mag = refs.q4_matrix(8, refs.Q4_0, 24, 128)
    h = ctx.upload_matrix(refs.Q4_0, 24, 128, packed)
    x = np.random.default_rng(2).normal(0, 1, (3, 128)).astype(np.float32)
    y = torch.empty(3, 24, device="cuda")
    ctx.wait(ctx.matvec(h, dev(x), y))
    near(y, *refs.linear(x, w, mag, "f32"))


def test_linear_refusals(ctx):
    caps = ctx.caps().arena_bytes
    packed, _, _ = refs.q4_matrix(8, refs.Q4_0, 8, 64)
    for kind, rows, cols, p in [(2, 8, 64, packed[:, :-1]), (3, 8, 64, packed), (2, 8, 48, packed), (2, 0, 64, packed),
                                (2, 8, 65568, packed), (4, 8, 64, packed)]:
        with pytest.raises(abi.GxError) as e:
            ctx.upload_matrix(kind, rows, cols, p)
        assert e.value.code == -1
    h = ctx.upload_matrix(refs.Q4_0, 8, 64, packed)
    assert ctx.caps().arena_bytes > caps
    x, y = torch.zeros(65, 64, device="cuda"), torch.zeros(65, 8, device="cuda")
    with pytest.raises(abi.GxError):
        ctx.linear(h, x, y)
    rng = np.random.default_rng(0)
    gyro = ctx.upload_matrix(144, 8, 128, synth.packed_matrix(rng, 144, 8, 128))
    with pytest.raises(abi.GxError) as e:
        ctx.linear(gyro, torch.zeros(1, 128, device="cuda"), torch.zeros(1, 8, device="cuda"))
    assert e.value.code == -5
    assert ctx.lib.gx_linear(ctx.handle, 10 ** 6, x.data_ptr(), 0, 64, 1, y.data_ptr(), 0, 8, None) == -1
    ctx.wait(ctx.linear(h, x[:0], y[:0]))
    ctx.wait(ctx.linear(h, x[:64], y[:64]))


def test_linear_repeats_bit_for_bit(ctx):
    for rows, cols, n in [(300, 2048, 1), (64, 8192, 2), (100, 4096, 20), (50, 1024, 64)]:
        packed, _, _ = refs.q4_matrix(6, refs.Q4_0, rows, cols)
        h = ctx.upload_matrix(refs.Q4_0, rows, cols, packed)
        x = torch.randn(n, cols, device="cuda")
        torch.cuda.synchronize()
        ys = [torch.empty(n, rows, device="cuda") for _ in range(3)]
        for y in ys:
            ctx.wait(ctx.linear(h, x, y))
        assert torch.equal(ys[0], ys[1]) and torch.equal(ys[0], ys[2])


# ---- norms ------------------------------------------------------------------------------------
WIDTHS = [1, 3, 8, 31, 64, 100, 256, 1000, 2048, 2560, 4096, 5001, 8192, 16384, 65536]


@pytest.mark.parametrize("width", WIDTHS)
@pytest.mark.parametrize("xk,yk", [("f32", "f32"), ("bf16", "bf16"), ("f32", "bf16"), ("bf16", "f32")])
def test_norm(ctx, width, xk, yk):
    rng = np.random.default_rng(width)
    for n, with_w, with_g, eps in [(1, True, True, 1e-6), (5, True, False, 1e-5), (3, False, True, 0.0)]:
        x = refs.to_kind(rng.normal(0.3, 2, (n, width)), xk)
        w = (1 + 0.3 * rng.normal(0, 1, width)).astype(np.float32) if with_w else None
        gw = rng.normal(0, 1, width).astype(np.float32) if with_g else None
        y, buf = out_rows(n, width, yk)
        gate = torch.full((n + 1,), 77.0, device="cuda") if with_g else None
        ctx.wait(ctx.norm(dev(x, xk), y, None if w is None else dev(w), eps, None if gw is None else dev(gw),
                          None if gate is None else gate[:n]))
        want = refs.norm(x, w, eps, yk, gw)
        near(y, *want[0], (width, n))
        untouched(buf, n, width)
        if with_g:
            near(gate[:n], *want[1])
            assert float(gate[n]) == 77.0


def test_norm_many_rows_strides_and_in_place(ctx):
    rng = np.random.default_rng(3)
    for n, width, xs, ys in [(700, 96, 101, 97), (300, 256, 264, 256), (2000, 64, 64, 72), (40, 2048, 2051, 2048)]:
        for kind in ("f32", "bf16"):
            x = refs.to_kind(rng.normal(0, 1, (n, width)), kind)
            y, buf = out_rows(n, width, kind, ys)
            ctx.wait(ctx.norm(dev(x, kind, xs), y))
            near(y, *refs.norm(x, None, 1e-6, kind)[0], (n, width))
            untouched(buf, n, width)
            t = dev(x, kind)
            ctx.wait(ctx.norm(t, t))
            near(t, *refs.norm(x, None, 1e-6, kind)[0])


def test_norm_extreme_rows(ctx):
    """Zeros (eps decides), tiny and huge rows, and a NaN or Inf, which stays in its row. A row whose sum of
    squares passes f32 gives zeros, as the formula in f32 does."""
    x = np.random.default_rng(0).normal(0, 1, (6, 512)).astype(np.float32)
    x[0] = 0
    x[1] *= 1e-15
    x[2] *= 1e15
    x[3, 7] = np.nan
    x[4, 9] = np.inf
    y = torch.empty(6, 512, device="cuda")
    ctx.wait(ctx.norm(dev(x), y, None, 1e-6))
    want = refs.norm(x[[0, 1, 2, 5]], None, 1e-6, "f32")[0]
    got = y.cpu().numpy()
    near(got[[0, 1, 2, 5]].astype(np.float64), *want)
    assert np.isnan(got[3]).all() and np.isnan(got[4, 9]) and (got[4, :9] == 0).all()


RES_CASES = [dict(), dict(post_norm=False), dict(gate="token"), dict(gate="element"), dict(has_out=False),
             dict(has_out=False, gate="token", post_norm=False), dict(gate="token", next_gate=True), dict(w=False, next_gate=True)]


def check_residual(ctx, n, width, yk, rk, ok, gk, seed, gate=None, post_norm=True, has_out=True, next_gate=False, w=True,
                   strides=(None,) * 5, in_place=True):
    rng = np.random.default_rng(seed)
    ys, rs, os_, hs, gs = strides
    y = refs.to_kind(rng.normal(0, 1, (n, width)), yk)
    res = refs.to_kind(rng.normal(0, 3, (n, width)), rk)
    vec = lambda: (1 + 0.3 * rng.normal(0, 1, width)).astype(np.float32)  # noqa: E731
    post = vec() if w and post_norm else None
    nxt = vec() if w and has_out else None
    gw = vec() if next_gate else None
    g = None
    if gate == "token":
        g = rng.normal(0, 3, n).astype(np.float32)
    elif gate == "element":
        g = refs.to_kind(rng.normal(0, 3, (n, width)), gk)
    a, b, eps = 0.9, -0.7, 1e-5
    rt = dev(res, rk, rs)
    if in_place:
        ro, rbuf = rt, None
    else:
        ro, rbuf = out_rows(n, width, rk, os_)
    out, obuf = out_rows(n, width, ok, hs) if has_out else (None, None)
    ng = torch.full((n + 1,), 77.0, device="cuda") if next_gate else None
    t = lambda v: None if v is None else dev(v)  # noqa: E731
    ctx.wait(ctx.norm_residual(dev(y, yk, ys), rt, None if in_place else ro, t(post), post_norm, eps, a, b,
                               None if g is None else dev(g) if g.ndim == 1 else dev(g, gk, gs), out, t(nxt), t(gw),
                               None if ng is None else ng[:n]))
    want = refs.residual(y, res, post, post_norm, eps, np.float64(np.float32(a)), np.float64(np.float32(b)), g, nxt,
                         has_out, (rk, ok), gw)
    near(ro, *want[0], "res")
    if rbuf is not None:
        untouched(rbuf, n, width)
        assert np.array_equal(rt.float().cpu().numpy(), res)
    if has_out:
        near(out, *want[1], "out")
        untouched(obuf, n, width)
    if next_gate:
        near(ng[:n], *want[2], "next gate")
        assert float(ng[n]) == 77.0


@pytest.mark.parametrize("width", WIDTHS)
@pytest.mark.parametrize("case", range(len(RES_CASES)))
def test_norm_residual(ctx, width, case):
    kinds = [("f32", "f32", "f32", "f32"), ("bf16", "f32", "bf16", "bf16"), ("bf16", "bf16", "f32", "f32")]
    for i, k in enumerate(kinds):
        check_residual(ctx, 1 + 2 * i, width, *k, seed=width + i, **RES_CASES[case])


def test_norm_residual_strides(ctx):
    for n, width, strides in [(90, 96, (97, 99, 101, 103, 105)), (50, 1024, (1032, 1040, 1024, 1048, 1056)),
                              (33, 640, (641, 640, 648, 640, 642))]:
        for k in [("f32", "f32", "f32", "f32"), ("bf16", "f32", "bf16", "bf16"), ("f32", "bf16", "bf16", "bf16")]:
            check_residual(ctx, n, width, *k, seed=n, gate="element", next_gate=True, strides=strides, in_place=False)
            check_residual(ctx, n, width, *k, seed=n, gate="token", strides=strides)


def test_norm_residual_many_rows(ctx):
    check_residual(ctx, 3000, 128, "f32", "f32", "bf16", "f32", seed=1, gate="element", next_gate=True)
    check_residual(ctx, 1500, 520, "bf16", "bf16", "bf16", "bf16", seed=2, gate="token", in_place=False)


@pytest.mark.parametrize("width,n", [(1024, 9473), (2560, 4100), (8192, 1300)])
def test_norm_long_batches(ctx, width, n):
    """Enough rows for every CTA to take several."""
    rng = np.random.default_rng(width)
    w = (1 + 0.3 * rng.normal(0, 1, width)).astype(np.float32)
    for xk, yk, weight in (("bf16", "f32", w), ("f32", "bf16", None), ("f32", "f32", w), ("bf16", "bf16", w)):
        x = refs.to_kind(rng.standard_normal((n, width), np.float32), xk)
        y, buf = out_rows(n, width, yk, width + 8)
        ctx.wait(ctx.norm(dev(x, xk), y, None if weight is None else dev(weight)))
        want = refs.norm(x, weight, 1e-6, yk)[0]
        near(y, *want)
        untouched(buf, n, width)
        if xk == yk:
            t = dev(x, xk)
            ctx.wait(ctx.norm(t, t, None if weight is None else dev(weight)))
            near(t, *want)


@pytest.mark.parametrize("width,n", [(512, 7200), (2560, 1300), (4096, 700)])
def test_norm_residual_long_batches(ctx, width, n):
    for i, k in enumerate([("f32", "bf16", "bf16", "f32"), ("bf16", "f32", "f32", "bf16"), ("f32", "f32", "f32", "f32")]):
        check_residual(ctx, n, width, *k, seed=i, gate="element", next_gate=i == 0, in_place=i == 1)
        check_residual(ctx, n, width, *k, seed=i, gate="token" if i else None, next_gate=i == 1, post_norm=i != 2)
        check_residual(ctx, n, width, *k, seed=i, gate="token", has_out=False, strides=(width + 8,) * 5, in_place=False)


def test_norm_residual_refusals(ctx):
    y, r = torch.zeros(4, 64, device="cuda"), torch.ones(4, 64, device="cuda")
    for bad in [dict(out=y), dict(out=r), dict(res_out=y), dict(next_weight=torch.ones(64, device="cuda")),
                dict(eps=-1.0), dict(block_scale=float("nan")), dict(post=torch.ones(64, device="cuda"), post_norm=False)]:
        with pytest.raises(abi.GxError) as e:
            ctx.norm_residual(y, r, **bad)
        assert e.value.code == -1
    with pytest.raises(abi.GxError):
        ctx.norm(y[:3], y[1:])      # rows that lie over later ones
    assert bool((r == 1).all())
    ctx.wait(ctx.norm_residual(y[:0], r[:0]))


# ---- log probabilities ------------------------------------------------------------------------
def run_logprobs(ctx, x, kind, tokens, n_top, scale, stride=None):
    n = x.shape[0]
    o = dict(logprob=torch.full((n + 1,), 77.0, device="cuda"), entropy=torch.full((n + 1,), 77.0, device="cuda"),
             rank=torch.full((n + 1,), 77, dtype=torch.int32, device="cuda"),
             top_ids=torch.full((n * n_top + 1,), 77, dtype=torch.int32, device="cuda"),
             top_logprobs=torch.full((n * n_top + 1,), 77.0, device="cuda"))
    tok = torch.from_numpy(tokens.view(np.int32)).cuda()
    arg = {k: v[:-1] for k, v in o.items()}
    if not n_top:
        arg["top_ids"] = arg["top_logprobs"] = None
    t = ctx.logprobs(dev(x, kind, stride), tok, n_top=n_top, scale=scale, **arg)
    err = None
    try:
        ctx.wait(t)
    except abi.GxError as e:
        err = e.code
    assert all(float(v[-1]) == 77.0 for v in o.values())
    got = {k: v[:-1].cpu().numpy() for k, v in o.items()}
    got["top_ids"], got["top_logprobs"] = got["top_ids"].reshape(n, n_top), got["top_logprobs"].reshape(n, n_top)
    return got, err


def check_logprobs(ctx, x, kind, tokens, n_top, scale, stride=None):
    got, err = run_logprobs(ctx, x, kind, tokens, n_top, scale, stride)
    want, bounds = refs.logprobs(x, tokens, n_top, scale)
    assert np.array_equal(got["rank"], want["rank"])
    assert np.array_equal(got["top_ids"], want["top_ids"])
    for k, b in bounds.items():
        near(got[k].astype(np.float64), want[k], b, k)
    return err


def logits(seed, n, V, kind):
    rng = np.random.default_rng(seed)
    x = rng.normal(0, 2.5, (n, V))
    x[:, rng.integers(0, V, 5)] += 8
    return refs.to_kind(x, kind), rng.integers(0, V, n).astype(np.uint32)


@pytest.mark.parametrize("V", [1, 2, 7, 31, 33, 100, 1000, 1023, 4097, 32000, 50257, 131072, 150001, 262147, 524288])
@pytest.mark.parametrize("kind", ["f32", "bf16"])
def test_logprobs_widths(ctx, V, kind):
    for n, k, scale in [(1, 5, 1.0), (3, 20, 0.7)]:
        x, tok = logits(V + n, n, V, kind)
        assert check_logprobs(ctx, x, kind, tok, min(k, V), scale) is None


@pytest.mark.parametrize("n", [2, 17, 160, 600])
def test_logprobs_rows(ctx, n):
    for V, kind, k in [(1001, "bf16", 32), (2048, "f32", 1), (515, "f32", 0), (40003, "bf16", 3)]:
        if n * V > 8e6:
            continue
        x, tok = logits(n, n, V, kind)
        assert check_logprobs(ctx, x, kind, tok, k, 1.3) is None


@pytest.mark.parametrize("kind", ["f32", "bf16"])
def test_logprobs_strides(ctx, kind):
    for V, stride in [(1000, 1001), (1000, 1008), (4096, 4099), (33, 47), (50257, 50300)]:
        x, tok = logits(V, 5, V, kind)
        assert check_logprobs(ctx, x, kind, tok, 8, 1.0, stride) is None
    # a buffer that starts at an odd element
    x, tok = logits(1, 4, 777, kind)
    src = torch.zeros(4 * 777 + 1, dtype=DT[kind], device="cuda")
    src[1:] = torch.from_numpy(x).reshape(-1).cuda()
    lp = torch.empty(4, device="cuda")
    ctx.wait(ctx.logprobs(src[1:].view(4, 777), torch.from_numpy(tok.view(np.int32)).cuda(), logprob=lp))
    want, bounds = refs.logprobs(x, tok, 0, 1.0)
    near(lp, want["logprob"], bounds["logprob"])


@pytest.mark.parametrize("V", [40, 3001, 131080])
@pytest.mark.parametrize("kind", ["f32", "bf16"])
def test_logprobs_ties_and_orders(ctx, V, kind):
    """Equal logits, rising, falling and interleaved rows, few distinct values, -0 against 0, the best ones
    next to one another or one apart at every kind of distance."""
    rng = np.random.default_rng(V)
    rows = [np.zeros(V), np.full(V, -3.25), np.linspace(-40, 40, V), np.linspace(40, -40, V), np.arange(V) % 7,
            -(np.arange(V) % 5), np.where(np.arange(V) % 2, 0.0, -0.0), rng.integers(-2, 3, V),
            np.where(np.arange(V) < 32, 5.0, 0.0), np.where(np.arange(V) >= V - 32, 5.0, 0.0)]
    for step in (8, 32, 64, 256, 1024, 2048, 4096):
        r = rng.normal(0, 1, V)
        r[::step] += 30.0
        rows.append(r)
    x = refs.to_kind(np.stack(rows), kind)
    tok = rng.integers(0, V, len(rows)).astype(np.uint32)
    for k in (1, 32):
        assert check_logprobs(ctx, x, kind, tok, k, 1.0) is None


@pytest.mark.parametrize("V", [50, 9000, 150001])
@pytest.mark.parametrize("kind", ["f32", "bf16"])
def test_logprobs_masks(ctx, V, kind):
    """Masked tokens (-Inf and the type's lowest value), rows with one token left, none left, fewer left
    than alternatives asked for; a given token that is masked; NaN and +Inf."""
    rng = np.random.default_rng(V)
    low = float(torch.finfo(DT[kind]).min)
    x = rng.normal(0, 3, (14, V))
    x[0, V // 2:] = -np.inf
    x[1] = -np.inf
    x[2] = -np.inf
    x[2, V - 1] = 1.5
    x[3] = -np.inf
    x[3, [3, 7, V // 2]] = [1.0, 1.0, 0.5]
    x[4, : V // 3] = low
    x[5] = low
    x[6] = low
    x[6, 11] = -5.0
    x[7, 17] = np.nan
    x[8, 19] = np.inf
    x[9] = np.nan
    x[10] = -np.inf
    x[10, 5] = np.nan
    x[11, ::2] = -np.inf
    x[12] = low
    x[12, 4] = -low
    x[13, 8] = np.inf
    x[13, 12] = np.inf
    x = refs.to_kind(x, kind)
    with np.errstate(over="ignore"):
        x[4:7][x[4:7] < -1e38] = low
    tok = np.array([1, 2, V - 1, 4, 0, 9, 11, 17, 18, 4, 5, 2, 7, 12], np.uint32)
    # scaled, the lowest values differ from the rest by more than f32 holds: probability 0
    for k, scale in ((20, 1.0), (4, 0.5)):
        assert check_logprobs(ctx, x, kind, tok, k, scale) is None


def test_logprobs_tokens_not_given_and_out_of_range(ctx):
    x, tok = logits(5, 6, 3000, "f32")
    tok[[1, 4]] = 0xFFFFFFFF
    assert check_logprobs(ctx, x, "f32", tok, 3, 1.0) is None
    tok[3] = 3000
    assert check_logprobs(ctx, x, "f32", tok, 3, 1.0) == -9
    tok[3] = 5
    assert check_logprobs(ctx, x, "f32", tok, 3, 1.0) is None     # the context stays usable
    # only some of the outputs
    e = torch.empty(6, device="cuda")
    ids = torch.empty(6, 2, dtype=torch.int32, device="cuda")
    ctx.wait(ctx.logprobs(dev(x), entropy=e, n_top=2, top_ids=ids))
    want, bounds = refs.logprobs(x, tok, 2, 1.0)
    near(e, want["entropy"], bounds["entropy"])
    assert np.array_equal(ids.cpu().numpy(), want["top_ids"])
    ctx.wait(ctx.logprobs(dev(x)[:0]))


def test_logprobs_refusals(ctx):
    x = torch.zeros(2, 16, device="cuda")
    ids = torch.zeros(2 * 33, dtype=torch.int32, device="cuda")
    for bad in [dict(n_top=33, top_ids=ids), dict(n_top=17, top_ids=ids[:34]), dict(scale=0.0), dict(scale=float("inf")),
                dict(logprob=torch.zeros(2, device="cuda")), dict(entropy=x.view(-1)[:2])]:
        with pytest.raises(abi.GxError) as e:
            ctx.logprobs(x, **bad)
        assert e.value.code == -1


@pytest.mark.parametrize("scale", [1e-30, 1e-3, 30.0, 1e20, 1e30])
def test_logprobs_extreme_scales(ctx, scale):
    """Temperatures from flat to a single token; ties of the largest share it."""
    x, tok = logits(3, 5, 4001, "f32")
    x[2, [9, 90, 900]] = 40.0
    tok[:] = x.argmax(1)
    assert check_logprobs(ctx, x, "f32", tok, 4, scale) is None


def test_rows_far_apart(ctx):
    """Rows whose byte offsets pass 32 bits."""
    far = 1_200_000_000
    buf = torch.empty(far + 8192, dtype=torch.float32, device="cuda")
    rng = np.random.default_rng(0)

    def rows(width, values=None):
        v = buf.as_strided((2, width), (far, 1))
        if values is not None:
            v.copy_(torch.from_numpy(values))
        return v

    x = rng.normal(0, 1, (2, 2048)).astype(np.float32)
    y = torch.empty(2, 2048, device="cuda")
    src = rows(2048, x)
    torch.cuda.synchronize()
    ctx.wait(ctx.norm(src, y))
    near(y, *refs.norm(x, None, 1e-6, "f32")[0])
    ctx.wait(ctx.norm(src, src))
    near(rows(2048), *refs.norm(x, None, 1e-6, "f32")[0])
    z, tok = logits(1, 2, 8000, "f32")
    src = rows(8000, z)
    torch.cuda.synchronize()
    lp = torch.empty(2, device="cuda")
    ctx.wait(ctx.logprobs(src, torch.from_numpy(tok.view(np.int32)).cuda(), logprob=lp))
    want, bounds = refs.logprobs(z, tok, 0, 1.0)
    near(lp, want["logprob"], bounds["logprob"])
    packed, w, mag = refs.q4_matrix(7, refs.Q4_0, 40, 2048)
    h = ctx.upload_matrix(refs.Q4_0, 40, 2048, packed)
    src = rows(2048, x)
    y = torch.empty(2, 40, device="cuda")
    torch.cuda.synchronize()
    ctx.wait(ctx.linear(h, src, y))
    near(y, *refs.linear(x, w, mag, "f32"))
    out = buf[4096:].as_strided((2, 40), (far, 1))
    ctx.wait(ctx.linear(h, dev(x), out))
    near(out, *refs.linear(x, w, mag, "f32"))
    check = buf.as_strided((2, 2048), (far, 1))
    ctx.wait(ctx.norm_residual(dev(x), check, post_norm=False))
    near(check, 2.0 * x.astype(np.float64), np.abs(x) * 2.0 ** -21)


# ---- together ---------------------------------------------------------------------------------
def test_scoring_run(ctx):
    """Final norm, 4-bit head and log probabilities, as a host scores tokens, eagerly and as a graph that
    is replayed on new hidden states."""
    E, V, n, k = 256, 5003, 7, 6
    rng = np.random.default_rng(11)
    packed, w, mag = refs.q4_matrix(12, refs.Q4_0, V, E)
    h = ctx.upload_matrix(refs.Q4_0, V, E, packed)
    weight = (1 + 0.2 * rng.normal(0, 1, E)).astype(np.float32)
    wd, xd = dev(weight), torch.empty(n, E, device="cuda")
    hid, lg = torch.empty(n, E, device="cuda"), torch.empty(n, V, device="cuda")
    tok = torch.zeros(n, dtype=torch.int32, device="cuda")
    o = dict(logprob=torch.empty(n, device="cuda"), rank=torch.empty(n, dtype=torch.int32, device="cuda"),
             entropy=torch.empty(n, device="cuda"), top_ids=torch.empty(n, k, dtype=torch.int32, device="cuda"),
             top_logprobs=torch.empty(n, k, device="cuda"))

    def steps(ticket):
        ctx.norm(xd, hid, wd, ticket=ticket)
        ctx.linear(h, hid, lg, ticket=ticket)
        return ctx.logprobs(lg, tok, n_top=k, scale=0.05, ticket=ticket, **o)

    def check(x):
        hw = refs.norm(x, weight, 1e-6, "f32")[0]
        near(hid, *hw)
        got_h = hid.cpu().numpy()
        near(lg, *refs.linear(got_h, w, mag, "f32"))
        got_l = lg.cpu().numpy()
        want, bounds = refs.logprobs(got_l, tok.cpu().numpy().view(np.uint32), k, 0.05)
        assert np.array_equal(o["rank"].cpu().numpy(), want["rank"]) and np.array_equal(o["top_ids"].cpu().numpy(), want["top_ids"])
        for name, b in bounds.items():
            near(o[name], want[name], b, name)

    def load(seed):
        x = np.random.default_rng(seed).normal(0, 4, (n, E)).astype(np.float32)
        xd.copy_(torch.from_numpy(x))
        tok.copy_(torch.from_numpy(np.random.default_rng(seed).integers(0, V, n).astype(np.int32)))
        torch.cuda.synchronize()
        return x

    x = load(1)
    ctx.wait(steps(True))
    check(x)
    stream = torch.cuda.ExternalStream(ctx.stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream, capture_error_mode="thread_local"):
        with pytest.raises(abi.GxError) as e:
            ctx.norm(xd, hid, wd)
        assert e.value.code == -6
        steps(False)
    for seed in (2, 3):
        x = load(seed)
        with torch.cuda.stream(stream):
            graph.replay()
        torch.cuda.synchronize()
        check(x)
    x = load(4)
    ctx.wait(steps(True))
    check(x)


def test_batches_in_flight_share_a_workspace(ctx):
    """Batch products of different sizes one after another without a wait between them, each packing its
    activations where the one before did, eagerly and as a graph that is replayed on new ones."""
    work = []
    for i, (kind, rows, cols, n, xk) in enumerate([(refs.Q4_0, 700, 2048, 40, "f32"), (refs.Q4_1, 130, 4096, 12, "f32"),
                                                   (refs.Q4_0, 40, 8192, 64, "bf16"), (refs.Q4_1, 1000, 256, 20, "bf16"),
                                                   (refs.Q4_0, 129, 6144, 5, "f32"), (refs.Q4_0, 2100, 1024, 33, "bf16")]):
        packed, w, mag = refs.q4_matrix(70 + i, kind, rows, cols)
        work.append(dict(h=ctx.upload_matrix(kind, rows, cols, packed), w=w, mag=mag, n=n, cols=cols, xk=xk,
                         xd=dev(refs.to_kind(np.zeros((n, cols)), xk), xk), y=torch.empty(n, rows, device="cuda")))

    def load(seed):
        for i, s in enumerate(work):
            s["x"] = refs.to_kind(np.random.default_rng(seed + i).normal(0, 1, (s["n"], s["cols"])), s["xk"])
            s["xd"].copy_(dev(s["x"], s["xk"]))
            s["y"].fill_(float("nan"))
        torch.cuda.synchronize()

    def steps():
        for _ in range(3):
            for s in work:
                ctx.linear(s["h"], s["xd"], s["y"], ticket=False)

    def check():
        torch.cuda.synchronize()
        for s in work:
            near(s["y"], *refs.linear(s["x"], s["w"], s["mag"], "f32"))

    load(1)
    steps()
    check()
    stream = torch.cuda.ExternalStream(ctx.stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream, capture_error_mode="thread_local"):
        steps()
    for seed in (20, 40):
        load(seed)
        with torch.cuda.stream(stream):
            graph.replay()
        check()
    load(60)
    steps()
    check()


def test_two_contexts_at_once():
    """Two contexts' streams with calls in flight together share no workspace."""
    V, n, cols = 30011, 9, 4096
    with abi.Context(device=0, max_tokens=16, max_layers=1) as a, abi.Context(device=0, max_tokens=16, max_layers=1) as b:
        work = []
        for i, c in enumerate((a, b)):
            packed, w, mag = refs.q4_matrix(40 + i, refs.Q4_0, 64, cols)
            x, tok = logits(50 + i, n, V, "f32")
            v = np.random.default_rng(60 + i).normal(0, 1, (n, cols)).astype(np.float32)
            work.append(dict(c=c, h=c.upload_matrix(refs.Q4_0, 64, cols, packed), w=w, mag=mag, v=v, vd=dev(v), x=x, xd=dev(x),
                             tok=tok, td=torch.from_numpy(tok.view(np.int32)).cuda(), y=torch.empty(n, 64, device="cuda"),
                             hd=torch.empty(n, cols, device="cuda"), lp=torch.empty(n, device="cuda"),
                             ids=torch.empty(n, 4, dtype=torch.int32, device="cuda")))
        torch.cuda.synchronize()
        for _ in range(20):
            for s in work:
                s["c"].linear(s["h"], s["vd"], s["y"])
                s["c"].logprobs(s["xd"], s["td"], logprob=s["lp"], n_top=4, top_ids=s["ids"])
                s["t"] = s["c"].norm(s["vd"], s["hd"])
        for s in work:
            s["c"].wait(s["t"])
            near(s["y"], *refs.linear(s["v"], s["w"], s["mag"], "f32"))
            want, bounds = refs.logprobs(s["x"], s["tok"], 4, 1.0)
            near(s["lp"], want["logprob"], bounds["logprob"])
            assert np.array_equal(s["ids"].cpu().numpy(), want["top_ids"])
            near(s["hd"], *refs.norm(s["v"], None, 1e-6, "f32")[0])


# ---- the routed layer as a block of a residual stream -------------------------------------------
def norm_params(seed, E, gate=True, post=True):
    rng = np.random.default_rng(seed)
    v = lambda s: (1 + s * rng.normal(0, 1, E)).astype(np.float32)  # noqa: E731
    return dict(pre=v(0.2), post=v(0.2) if post else None, post_norm=post,
                gate=(rng.normal(0, 1, E) / np.sqrt(E)).astype(np.float32) if gate else None, eps=1e-6,
                res_scale=0.95, block_scale=0.6)


@pytest.mark.parametrize("n_tok", [1, 6, 80])
def test_norm_block(n_tok):
    """Two layers in a row, the second without gate and post-norm, against the norms in 64 bits around the
    layer as gx_moe_forward computes it on the same input (its own parity is tested elsewhere)."""
    E = 256
    layers = [synth.make_layer(800 + i, n_expert=16, E=E, F=128, U=4) for i in range(2)]
    norms = [norm_params(810, E), norm_params(811, E, gate=False, post=False)]
    res = np.random.default_rng(n_tok).normal(0, 2, (n_tok, E)).astype(np.float32)
    with abi.Context(device=0, max_tokens=128, max_layers=2) as ctx:
        for i in range(2):
            ctx.upload_layer(i, layers[i])
        rt = torch.from_numpy(res).cuda()
        with pytest.raises(abi.GxError) as e:
            ctx.norm_block(0, 2, rt)
        assert e.value.code == -6
        for i in range(2):
            ctx.upload_norms(i, norms[i])
        ctx.wait(ctx.norm_block(0, 2, rt))
        ctx.wait(ctx.norm_block(0, 1, rt[:0]))
        got = rt.cpu().numpy()
        # the same chain of separate calls
        st = torch.from_numpy(res).cuda()
        h, y, g = torch.empty_like(st), torch.empty_like(st), torch.empty(n_tok, device="cuda")
        d = [{k: (dev(v) if isinstance(v, np.ndarray) else v) for k, v in p.items()} for p in norms]
        ctx.norm(st, h, d[0]["pre"], 1e-6, d[0]["gate"], g)
        ctx.forward(0, h, y)
        ctx.norm_residual(y, st, post=d[0]["post"], eps=1e-6, res_scale=0.95, block_scale=0.6, gate=g, out=h,
                          next_weight=d[1]["pre"])
        ctx.wait(ctx.forward(1, h, y))
        h1 = h.cpu().numpy()
        ctx.wait(ctx.norm_residual(y, st, post_norm=False, res_scale=0.95, block_scale=0.6))
        assert np.array_equal(st.cpu().numpy(), got)
        with pytest.raises(abi.GxError):
            ctx.norm_block(0, 3, rt)
        ctx.upload_norms(1, None)
        with pytest.raises(abi.GxError):
            ctx.norm_block(0, 2, rt)
        ctx.upload_layer(0, layers[0])     # drops the norms with the layer
        with pytest.raises(abi.GxError):
            ctx.norm_block(0, 1, rt)
    # the first layer's input and the second's, against the oracle's layer
    (h0, b0), (g0, _) = refs.norm(res, norms[0]["pre"], 1e-6, "f32", norms[0]["gate"])
    y0, _, _ = oracle.moe_ffn(layers[0], h0.astype(np.float32))
    want = refs.residual(y0.astype(np.float64), res, norms[0]["post"], True, 1e-6, 0.95, 0.6, g0, norms[1]["pre"], True,
                         ("f32", "f32"))
    rel = np.linalg.norm(h1 - want[1][0]) / np.linalg.norm(want[1][0])
    assert rel <= 5e-3, rel       # the layer's own bound (f16 operands from 64 tokens)
