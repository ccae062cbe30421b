"""CPU checks of the operators around the layer: struct layouts, the argument rules (csrc/gx_checks.h,
compiled for the host), the Python binding's own checks, and the 64-bit references they are tested with."""
import ctypes
import math
import subprocess
from pathlib import Path

import numpy as np
import pytest

import operator_refs as refs
from gyro_moe import abi, build

ROOT = Path(__file__).resolve().parents[1]
torch = pytest.importorskip("torch")


@pytest.fixture(scope="module")
def chk(tmp_path_factory):
    so = tmp_path_factory.mktemp("chk") / "checks.so"
    subprocess.run(["g++", "-std=c++17", "-O1", "-shared", "-fPIC", str(ROOT / "tests" / "checks_emu.cpp"), "-o", str(so)],
                   check=True)
    lib = ctypes.CDLL(str(so))
    lib.chk_linear.argtypes = [ctypes.c_uint32, ctypes.c_uint32, ctypes.c_void_p, ctypes.c_uint32, ctypes.c_uint64,
                               ctypes.c_uint32, ctypes.c_void_p, ctypes.c_uint32, ctypes.c_uint64]
    return lib


def test_struct_layouts_match_c(tmp_path):
    names = {"gx_norm_desc": abi.NormDesc, "gx_residual_desc": abi.ResidualDesc, "gx_logprobs_desc": abi.LogprobsDesc,
             "gx_norms_desc": abi.NormsDesc}
    lines = []
    for c, py in names.items():
        lines.append(f'printf("%zu\\n", sizeof({c}));')
        lines += [f'printf("%zu\\n", offsetof({c}, {f}));' for f, _ in py._fields_]
    lines.append('printf("%d %d %d %d %d\\n", GX_Q4_0, GX_Q4_1, GX_RES_POST_NORM, GX_GATE_TOKEN, GX_GATE_ELEMENT);')
    src = tmp_path / "sz.c"
    src.write_text('#include "gyro_moe.h"\n#include <stdio.h>\n#include <stddef.h>\nint main(void){' + "".join(lines) +
                   "return 0;}\n")
    exe = tmp_path / "sz"
    subprocess.run(["gcc", "-I", str(ROOT / "include"), str(src), "-o", str(exe)], check=True)
    got = [int(v) for v in subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.split()]
    want = []
    for py in names.values():
        want += [ctypes.sizeof(py)] + [getattr(py, f).offset for f, _ in py._fields_]
    assert got == want + [abi.GX_Q4_0, abi.GX_Q4_1, abi.GX_RES_POST_NORM, abi.GX_GATE_TOKEN, abi.GX_GATE_ELEMENT]


A, B, C, D, E, F = (0x10000000 * i for i in range(1, 7))   # addresses far apart; nothing reads them


def test_linear_rules(chk):
    ok = dict(rows=48, cols=64, x=A, xd=0, xs=64, n=3, y=B, yd=0, ys=48)
    call = lambda **k: chk.chk_linear(*{**ok, **k}.values())  # noqa: E731
    assert call() and call(n=64) and call(n=0, x=None, y=None) and call(xd=30, x=A + 2) and call(xs=1000, ys=777)
    assert not call(n=65) and not call(xd=8) and not call(yd=1) and not call(x=None) and not call(y=None)
    assert not call(xs=63) and not call(ys=47) and not call(x=A + 2) and not call(yd=30, y=B + 1)
    assert not call(xs=(1 << 32) + 1)
    # y over x is refused; slices of one fused buffer are not
    assert not call(y=A) and not call(y=A + 4 * 60)
    assert call(xs=112, ys=112, y=A + 4 * 64) and not call(xs=112, ys=112, y=A + 4 * 63)
    assert call(xs=112, ys=112, x=A + 4 * 48, y=A) and not call(xs=112, ys=112, x=A + 4 * 47, y=A)


def test_norm_rules(chk):
    ok = dict(x=A, y=B, weight=C, gate_weight=D, gate=E, x_stride=96, y_stride=96, x_dtype=0, y_dtype=30, n_embd=96,
              eps=1e-6)

    def call(n=5, **k):
        d = abi.NormDesc(*{**ok, **k}.values())
        return bool(chk.chk_norm(ctypes.byref(d), n))

    assert call() and call(n=0, x=None, y=None) and call(weight=None, gate_weight=None, gate=None) and call(eps=0.0)
    assert call(n_embd=1) and call(x_stride=100)
    assert not call(n_embd=0) and not call(n_embd=65537, x_stride=70000, y_stride=70000) and not call(eps=-1e-6)
    assert not call(eps=math.nan) and not call(eps=math.inf) and not call(x_dtype=2) and not call(y_stride=95)
    assert not call(gate=None) and not call(gate_weight=None) and not call(weight=C + 2) and not call(x=None)
    assert not call(y=A)                                        # another encoding over the input
    assert call(y=A, y_dtype=0) and not call(y=A + 4, y_dtype=0) and not call(y=A, y_dtype=0, y_stride=97)
    assert not call(gate=A + 8) and not call(gate=B + 8) and not call(weight=B)
    assert not call(n=(1 << 24) + 1)


def test_residual_rules(chk):
    ok = dict(y=A, res=B, res_out=B, gate=C, post=D, out=E, next=F, next_gate_weight=F + 4096, next_gate=F + 8192,
              y_stride=32, res_stride=32, res_out_stride=32, gate_stride=0, out_stride=32, y_dtype=30, res_dtype=0,
              gate_dtype=0, out_dtype=30, n_embd=32, flags=1, gate_kind=1, eps=1e-5, res_scale=1.0, block_scale=0.5)

    def call(n=4, **k):
        d = abi.ResidualDesc(*{**ok, **k}.values())
        return bool(chk.chk_residual(ctypes.byref(d), n))

    assert call() and call(n=0) and call(res_out=A + 4096) and call(flags=0, post=None)
    assert call(gate_kind=0, gate=None) and call(gate_kind=2, gate_stride=32, gate_dtype=30)
    assert call(out=None, next=None, next_gate_weight=None, next_gate=None)
    assert not call(flags=2) and not call(flags=0) and not call(gate_kind=3) and not call(gate_kind=0)
    assert not call(gate=None) and not call(gate_kind=2, gate_stride=31) and not call(gate_kind=2, gate_stride=32, gate_dtype=7)
    assert not call(out=None) and not call(next_gate=None) and not call(next_gate_weight=None)
    assert not call(res_scale=math.inf) and not call(block_scale=math.nan) and not call(eps=-1.0)
    assert not call(res_out=B + 4) and not call(res_out=B, res_out_stride=33)
    assert not call(out=A) and not call(out=B) and not call(out=C) and not call(res_out=A) and not call(next_gate=C)
    assert not call(y=None) and not call(res=None) and not call(res_out=None)


def test_logprobs_rules(chk):
    ok = dict(logits=A, tokens=B, logprob=C, rank=C + 4096, entropy=C + 8192, top_ids=D, top_logprobs=E, stride=1000,
              dtype=0, n_vocab=1000, n_top=5, scale=1.0)

    def call(n=7, **k):
        d = abi.LogprobsDesc(*{**ok, **k}.values())
        return bool(chk.chk_logprobs(ctypes.byref(d), n))

    assert call() and call(n=0, logits=None) and call(dtype=30, logits=A + 2) and call(stride=1003)
    assert call(tokens=None, logprob=None, rank=None) and call(n_top=0, top_ids=None, top_logprobs=None)
    assert call(top_ids=None) and call(top_logprobs=None) and call(n_vocab=5) and call(n_top=32)
    assert not call(tokens=None) and not call(n_top=0) and not call(n_top=33) and not call(n_vocab=4)
    assert not call(n_vocab=0) and not call(n_vocab=524289, stride=524289) and not call(stride=999)
    assert not call(scale=0.0) and not call(scale=-1.0) and not call(scale=math.inf) and not call(scale=math.nan)
    assert call(scale=1e-40) and call(scale=1e29) and not call(scale=1e31)
    assert not call(dtype=8) and not call(logits=A + 2) and not call(logprob=C + 2)
    assert not call(logprob=A + 40) and not call(top_ids=E) and not call(entropy=C)


def test_norms_rules(chk):
    call = lambda *v: bool(chk.chk_norms(ctypes.byref(abi.NormsDesc(*v))))  # noqa: E731
    assert call(A, B, C, 1, 1e-6, 1.0, 0.5) and call(None, None, None, 0, 0.0, -1.0, 0.0)
    assert not call(A, B, C, 0, 1e-6, 1.0, 1.0) and not call(A, B, C, 2, 1e-6, 1.0, 1.0)
    assert not call(A, B, C, 1, -1.0, 1.0, 1.0) and not call(A, B, C, 1, 1e-6, math.nan, 1.0)


def test_null_contexts_are_refused():
    build.build()
    lib = abi.load()
    one = ctypes.c_uint64()
    assert lib.gx_linear(None, 0, A, 0, 32, 1, B, 0, 32, ctypes.byref(one)) == -1
    assert lib.gx_norm(None, None, 1, None) == -1 and lib.gx_norm_residual(None, None, 1, None) == -1
    assert lib.gx_logprobs(None, None, 1, None) == -1 and lib.gx_upload_norms(None, 0, None, 0) == -1
    assert lib.gx_norm_block(None, 0, 1, A, 1, None) == -1


def test_binding_checks_shapes():
    """What the binding refuses before any call reaches the library."""
    ctx = abi.Context.__new__(abi.Context)
    ctx.handle, ctx.lib, ctx.matrices, ctx.layers = None, None, {0: (8, 64)}, {0: {"n_embd": 32}}
    ctx.device = -1                     # where the host's tensors are, so that the shapes are what is refused
    f = torch.zeros
    bad = [lambda: ctx.linear(0, f(2, 64), f(3, 8)), lambda: ctx.linear(0, f(2, 32), f(2, 8)),
           lambda: ctx.linear(0, f(64, 2).T, f(2, 8)), lambda: ctx.linear(0, f(2, 64).half(), f(2, 8)),
           lambda: ctx.norm(f(2, 32), f(2, 31)), lambda: ctx.norm(f(2, 32), f(3, 32)),
           lambda: ctx.norm(f(2, 32), f(2, 32), f(31)), lambda: ctx.norm(f(2, 32), f(2, 32), f(32).bfloat16()),
           lambda: ctx.norm_residual(f(2, 32), f(3, 32)), lambda: ctx.norm_residual(f(2, 32), f(2, 32), gate=f(3)),
           lambda: ctx.norm_residual(f(2, 32), f(2, 32), gate=f(2, 31)),
           lambda: ctx.norm_residual(f(2, 32), f(2, 32), f(2, 32).bfloat16()),
           lambda: ctx.logprobs(f(2, 32), torch.zeros(3, dtype=torch.int32)),
           lambda: ctx.logprobs(f(2, 32), torch.zeros(2, dtype=torch.int64)),
           lambda: ctx.logprobs(f(2, 32), n_top=3, top_ids=torch.zeros(2, 2, dtype=torch.int32)),
           lambda: ctx.upload_norms(0, {"pre": np.ones(31)}), lambda: ctx.norm_block(0, 1, f(2, 31)),
           lambda: ctx.norm_block(0, 1, f(2, 40)[:, :32]), lambda: ctx.norm_block(1, 1, f(2, 32))]
    for i, call in enumerate(bad):
        with pytest.raises(ValueError):
            call()
            pytest.fail(f"call {i} was taken")


def test_binding_refuses_tensors_of_another_device():
    ctx = abi.Context.__new__(abi.Context)
    ctx.handle, ctx.lib, ctx.matrices, ctx.layers, ctx.device = None, None, {0: (8, 64)}, {0: {"n_embd": 32}}, 0
    f = torch.zeros
    for call in [lambda: ctx.linear(0, f(2, 64), f(2, 8)), lambda: ctx.norm(f(2, 32), f(2, 32)),
                 lambda: ctx.norm_residual(f(2, 32), f(2, 32)), lambda: ctx.logprobs(f(2, 32)),
                 lambda: ctx.norm_block(0, 1, f(2, 32))]:
        with pytest.raises(ValueError, match="device"):
            call()


def test_references_agree_with_plain_loops():
    rng = np.random.default_rng(1)
    for kind in (refs.Q4_0, refs.Q4_1):
        packed, w, mag = refs.q4_matrix(2, kind, 3, 64)
        for r in range(3):
            for g in range(2):
                b = packed[r, g * refs.BLOCK[kind]:(g + 1) * refs.BLOCK[kind]]
                d = float(b[:2].view(np.float16)[0])
                for j in range(32):
                    q = int(b[len(b) - 16 + j % 16]) >> (4 * (j // 16)) & 15
                    want = d * (q - 8) if kind == refs.Q4_0 else d * q + float(b[2:4].view(np.float16)[0])
                    assert w[r, 32 * g + j] == want and abs(want) <= mag[r, 32 * g + j]
    x = rng.normal(0, 2, (4, 50)).astype(np.float32)
    x[1, 10] = x[1, 20] = 9.0
    x[2, 5:] = -np.inf
    x[3] = -np.inf
    tok = np.array([3, 20, 7, 49], np.uint32)
    got, bounds = refs.logprobs(x, tok, 4, 0.5)
    lp = torch.log_softmax(torch.from_numpy(x[:3]).double() * 0.5, -1)
    assert np.allclose(got["logprob"][:2], lp[[0, 1], [3, 20]], rtol=1e-12) and got["logprob"][2] == -np.inf
    assert list(got["top_ids"][1][:2]) == [10, 20] and got["rank"][1] == 1 and list(got["top_ids"][3]) == [0, 1, 2, 3]
    assert got["rank"][2] == 6 and np.isclose(got["entropy"][3], np.log(50)) and got["logprob"][3] == -np.log(50)
    p = lp[0].exp()
    assert np.isclose(got["entropy"][0], float(-(p * lp[0]).sum()), rtol=1e-12)
    assert all((b >= 0).all() and (b < 1e-3).all() for b in bounds.values())
