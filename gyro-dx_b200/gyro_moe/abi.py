"""ctypes mirror of include/gyro_moe.h — the host-side binding a Python caller (tests, bench)
uses; the Zig host binds the same symbols through gyro-dx_b200/zig/gx_abi.zig.

It loads the in-tree libgyromoe.so and fails loudly when it is missing: there is no CPU
fallback for any entry point.
"""
from __future__ import annotations

import ctypes
import os
import struct
from pathlib import Path

import numpy as np

PKG = Path(__file__).resolve().parent
LIB_PATH = PKG / "libgyromoe.so"
CODEBOOK_PATH = PKG / "data" / "gyro_codebook.f16"

GX_OK = 0
ERRORS = {-1: "GX_E_INVALIDARG", -2: "GX_E_OUTOFMEMORY", -3: "GX_E_TIMEOUT", -4: "GX_E_DEVICE",
          -5: "GX_E_UNSUPPORTED", -6: "GX_E_STATE", -7: "GX_E_MISMATCH", -8: "GX_E_COMM", -9: "GX_E_KERNEL",
          -10: "GX_E_RANGE"}
GX_F32, GX_Q8_0, GX_BF16 = 0, 8, 30
GX_Q4_0, GX_Q4_1 = 2, 3                           # 4-bit matrices with group scales (upload_matrix)
GX_RES_POST_NORM = 1
GX_GATE_NONE, GX_GATE_TOKEN, GX_GATE_ELEMENT = 0, 1, 2
GX_NO_TOKEN, GX_MAX_TOP = 0xFFFFFFFF, 32
GX_FLAG_PROFILE = 1
GX_EP_NONE, GX_EP_NCCL, GX_EP_PEER = 0, 1, 2     # gx_caps.ep_exchange


class GxError(RuntimeError):
    def __init__(self, code: int, call: str):
        super().__init__(f"{call} failed: {ERRORS.get(code, code)}")
        self.code = code


class Options(ctypes.Structure):
    _fields_ = [("device", ctypes.c_uint32), ("rank", ctypes.c_uint32), ("world", ctypes.c_uint32),
                ("max_tokens", ctypes.c_uint32), ("max_layers", ctypes.c_uint32), ("flags", ctypes.c_uint32),
                ("codebook", ctypes.c_void_p), ("codebook_bytes", ctypes.c_uint64),
                ("nccl_id", ctypes.c_uint8 * 128)]


class Caps(ctypes.Structure):
    _fields_ = [("abi_version", ctypes.c_uint32), ("sm_count", ctypes.c_uint32), ("cc_major", ctypes.c_uint32),
                ("cc_minor", ctypes.c_uint32), ("rank", ctypes.c_uint32), ("world", ctypes.c_uint32),
                ("max_tokens", ctypes.c_uint32), ("max_layers", ctypes.c_uint32), ("hbm_bytes", ctypes.c_uint64),
                ("free_bytes", ctypes.c_uint64), ("l2_bytes", ctypes.c_uint64), ("arena_bytes", ctypes.c_uint64),
                ("device_name", ctypes.c_char * 120), ("ep_exchange", ctypes.c_uint32), ("ep_peer_layers", ctypes.c_uint32)]


class LayerDesc(ctypes.Structure):
    _fields_ = [("type_id", ctypes.c_uint32), ("n_expert", ctypes.c_uint32), ("n_embd", ctypes.c_uint32),
                ("n_ff", ctypes.c_uint32), ("n_used", ctypes.c_uint32), ("expert_weights_scale", ctypes.c_float),
                ("gate", ctypes.c_void_p), ("up", ctypes.c_void_p), ("down", ctypes.c_void_p),
                ("gate_bytes", ctypes.c_uint64), ("up_bytes", ctypes.c_uint64), ("down_bytes", ctypes.c_uint64),
                ("router", ctypes.c_void_p), ("gate_signs", ctypes.c_void_p), ("up_signs", ctypes.c_void_p),
                ("down_signs", ctypes.c_void_p), ("router_bias", ctypes.c_void_p)]


class SharedDesc(ctypes.Structure):
    _fields_ = [("type_id", ctypes.c_uint32), ("n_ff", ctypes.c_uint32), ("gate", ctypes.c_void_p),
                ("up", ctypes.c_void_p), ("down", ctypes.c_void_p), ("gate_bytes", ctypes.c_uint64),
                ("up_bytes", ctypes.c_uint64), ("down_bytes", ctypes.c_uint64), ("gate_inp", ctypes.c_void_p)]


class HcDesc(ctypes.Structure):
    _fields_ = [("n_streams", ctypes.c_uint32), ("rank", ctypes.c_uint32), ("type_id", ctypes.c_uint32),
                ("eps", ctypes.c_float), ("norm", ctypes.c_void_p), ("down", ctypes.c_void_p),
                ("up", ctypes.c_void_p), ("inject", ctypes.c_void_p), ("down_bytes", ctypes.c_uint64),
                ("up_bytes", ctypes.c_uint64), ("inject_bytes", ctypes.c_uint64)]


class GgufLayerInfo(ctypes.Structure):
    _fields_ = [("type_id", ctypes.c_uint32), ("n_expert", ctypes.c_uint32), ("n_embd", ctypes.c_uint32),
                ("n_ff", ctypes.c_uint32), ("n_used", ctypes.c_uint32), ("expert_weights_scale", ctypes.c_float),
                ("shared_type", ctypes.c_uint32), ("shared_ff", ctypes.c_uint32), ("rotated", ctypes.c_uint32),
                ("reserved", ctypes.c_uint32)]


GX_SHARED_NONE = 0xFFFFFFFF


class NormDesc(ctypes.Structure):
    _fields_ = [("x", ctypes.c_void_p), ("y", ctypes.c_void_p), ("weight", ctypes.c_void_p),
                ("gate_weight", ctypes.c_void_p), ("gate", ctypes.c_void_p), ("x_stride", ctypes.c_uint64),
                ("y_stride", ctypes.c_uint64), ("x_dtype", ctypes.c_uint32), ("y_dtype", ctypes.c_uint32),
                ("n_embd", ctypes.c_uint32), ("eps", ctypes.c_float)]


class ResidualDesc(ctypes.Structure):
    _fields_ = [("y", ctypes.c_void_p), ("res", ctypes.c_void_p), ("res_out", ctypes.c_void_p),
                ("gate", ctypes.c_void_p), ("post", ctypes.c_void_p), ("out", ctypes.c_void_p),
                ("next", ctypes.c_void_p), ("next_gate_weight", ctypes.c_void_p), ("next_gate", ctypes.c_void_p),
                ("y_stride", ctypes.c_uint64), ("res_stride", ctypes.c_uint64), ("res_out_stride", ctypes.c_uint64),
                ("gate_stride", ctypes.c_uint64), ("out_stride", ctypes.c_uint64), ("y_dtype", ctypes.c_uint32),
                ("res_dtype", ctypes.c_uint32), ("gate_dtype", ctypes.c_uint32), ("out_dtype", ctypes.c_uint32),
                ("n_embd", ctypes.c_uint32), ("flags", ctypes.c_uint32), ("gate_kind", ctypes.c_uint32),
                ("eps", ctypes.c_float), ("res_scale", ctypes.c_float), ("block_scale", ctypes.c_float)]


class LogprobsDesc(ctypes.Structure):
    _fields_ = [("logits", ctypes.c_void_p), ("tokens", ctypes.c_void_p), ("logprob", ctypes.c_void_p),
                ("rank", ctypes.c_void_p), ("entropy", ctypes.c_void_p), ("top_ids", ctypes.c_void_p),
                ("top_logprobs", ctypes.c_void_p), ("stride", ctypes.c_uint64), ("dtype", ctypes.c_uint32),
                ("n_vocab", ctypes.c_uint32), ("n_top", ctypes.c_uint32), ("scale", ctypes.c_float)]


class NormsDesc(ctypes.Structure):
    _fields_ = [("pre", ctypes.c_void_p), ("post", ctypes.c_void_p), ("gate", ctypes.c_void_p),
                ("post_norm", ctypes.c_uint32), ("eps", ctypes.c_float), ("res_scale", ctypes.c_float),
                ("block_scale", ctypes.c_float)]


class Timings(ctypes.Structure):
    _fields_ = [("router_ns", ctypes.c_uint64), ("gate_up_ns", ctypes.c_uint64), ("down_ns", ctypes.c_uint64),
                ("experts_ns", ctypes.c_uint64), ("total_ns", ctypes.c_uint64), ("layers", ctypes.c_uint64)]


assert ctypes.sizeof(Options) == 168 and ctypes.sizeof(Caps) == 192 and ctypes.sizeof(LayerDesc) == 112
assert ctypes.sizeof(SharedDesc) == 64 and ctypes.sizeof(GgufLayerInfo) == 40 and ctypes.sizeof(HcDesc) == 72

assert ctypes.sizeof(NormDesc) == 72 and ctypes.sizeof(ResidualDesc) == 152
assert ctypes.sizeof(LogprobsDesc) == 80 and ctypes.sizeof(NormsDesc) == 40

# (name, argtypes) of every exported entry point; include/gyro_moe.h declares exactly these.
_P, _U32, _U64, _F = ctypes.c_void_p, ctypes.c_uint32, ctypes.c_uint64, ctypes.c_float
SIGNATURES = {
    "gx_create": [ctypes.POINTER(Options), ctypes.POINTER(_P)],
    "gx_comm_unique_id": [ctypes.c_char_p, _U64],
    "gx_get_caps": [_P, ctypes.POINTER(Caps)],
    "gx_upload_layer": [_P, _U32, ctypes.POINTER(LayerDesc), _U32],
    "gx_upload_shared": [_P, _U32, ctypes.POINTER(SharedDesc), _U32],
    "gx_upload_hc": [_P, _U32, ctypes.POINTER(HcDesc), _U32],
    "gx_ffn_block": [_P, _U32, _P, _U32, _P, ctypes.POINTER(_U64)],
    "gx_gguf_inspect_layer": [ctypes.c_char_p, _U32, ctypes.POINTER(GgufLayerInfo)],
    "gx_upload_layer_gguf": [_P, _U32, ctypes.c_char_p, _U32, _U32],
    "gx_moe_forward": [_P, _U32, _P, _U32, _U32, _P, _U32, _P, _P, ctypes.POINTER(_U64)],
    "gx_moe_forward_host": [_P, _U32, _P, _U32, _U32, _P, _U32, _P, _P, _U32],
    "gx_stack_forward": [_P, _U32, _U32, _P, _U32, _U32, _P, _U32, ctypes.POINTER(_U64)],
    "gx_stack_forward_host": [_P, _U32, _U32, _P, _U32, _U32, _P, _U32, _U32],
    "gx_wait": [_P, _U64, _U32],
    "gx_poll": [_P, ctypes.POINTER(_U64)],
    "gx_get_stream": [_P, ctypes.POINTER(_P)],
    "gx_decode_blocks": [_P, _U32, _P, _U64, _P, _U32, _P, ctypes.POINTER(_F), _U32],
    "gx_upload_matrix": [_P, _U32, _U32, _U32, _P, _U64, ctypes.POINTER(_U32), _U32],
    "gx_matvec": [_P, _U32, _P, _U32, _P, ctypes.POINTER(_U64)],
    "gx_linear": [_P, _U32, _P, _U32, _U64, _U32, _P, _U32, _U64, ctypes.POINTER(_U64)],
    "gx_norm": [_P, _P, _U32, ctypes.POINTER(_U64)],
    "gx_norm_residual": [_P, _P, _U32, ctypes.POINTER(_U64)],
    "gx_logprobs": [_P, _P, _U32, ctypes.POINTER(_U64)],
    "gx_upload_norms": [_P, _U32, ctypes.POINTER(NormsDesc), _U32],
    "gx_norm_block": [_P, _U32, _U32, _P, _U32, ctypes.POINTER(_U64)],
    "gx_read_timings": [_P, ctypes.POINTER(Timings)],
    "gx_read_expert_counts": [_P, _U32, _P, _U32, _U32],
    "gx_replicate_experts": [_P, _U32, _P, _U32, _U32],
    "gx_moe_forward_noalloc": [_P, _U32, _P, _U32, _U32, _P, _U32, _P, _P, ctypes.POINTER(_U64)],
    "gx_set_flags": [_P, _U32],
    "gx_destroy": [_P, _U32],
}

NOALLOC_MAX_TOKENS = 16          # GX_NOALLOC_MAX_TOKENS

_LIB = None


def load(path: Path | str | None = None) -> ctypes.CDLL:
    """Loads libgyromoe.so (raises if it was not built). GYRO_MOE_LIB in the environment names
    another build of the same library (for side-by-side timing)."""
    global _LIB
    if _LIB is not None and path is None:
        return _LIB
    p = Path(path) if path else Path(os.environ.get("GYRO_MOE_LIB", "") or LIB_PATH)
    if not p.exists():
        raise RuntimeError(f"{p} is missing: build it with gyro-dx_b200/gyro_moe/build.py (no CPU fallback exists)")
    lib = ctypes.CDLL(str(p))
    for name, args in SIGNATURES.items():
        fn = getattr(lib, name)
        fn.argtypes = args
        fn.restype = ctypes.c_int32
    if path is None:
        _LIB = lib
    return lib


def _check(rc: int, call: str) -> None:
    if rc != GX_OK:
        raise GxError(rc, call)


def _ptr(a) -> int | None:
    """Device pointer of a torch tensor, host pointer of a numpy array, or None."""
    if a is None:
        return None
    if hasattr(a, "data_ptr"):
        return a.data_ptr()
    return a.ctypes.data


def _dtype_code(a) -> int:
    name = str(a.dtype)
    if "bfloat16" in name:
        return GX_BF16
    if "float32" in name:
        return GX_F32
    if name == "uint16":  # numpy bf16 bit patterns
        return GX_BF16
    raise ValueError(f"unsupported activation dtype {name}")


def gguf_layer_info(path, gguf_layer: int) -> GgufLayerInfo:
    """gx_gguf_inspect_layer: shapes and types of one layer of a GGUF file (no device needed)."""
    info = GgufLayerInfo()
    _check(load().gx_gguf_inspect_layer(str(path).encode(), gguf_layer, ctypes.byref(info)), "gx_gguf_inspect_layer")
    return info


def unique_id() -> bytes:
    """A fresh NCCL unique id for gx_options.nccl_id (rank 0 makes it, the others receive it)."""
    buf = ctypes.create_string_buffer(128)
    _check(load().gx_comm_unique_id(buf, 128), "gx_comm_unique_id")
    return buf.raw


def _packer(desc):
    """struct.Struct of a descriptor's fields: packing one costs a third of filling the ctypes structure."""
    codes = {ctypes.c_void_p: "Q", ctypes.c_uint64: "Q", ctypes.c_uint32: "I", ctypes.c_float: "f"}
    p = struct.Struct("=" + "".join(codes[t] for _, t in desc._fields_))
    assert p.size == ctypes.sizeof(desc)
    return p.pack


_PACK_NORM, _PACK_RESIDUAL, _PACK_LOGPROBS = _packer(NormDesc), _packer(ResidualDesc), _packer(LogprobsDesc)
_CODES: dict = {}                # dtype -> encoding, of the dtypes seen


def _rows(a) -> tuple[int, int, int, int, int]:
    """(rows, width, pointer, row stride in elements, encoding) of a device tensor of rows (1-D: one row)."""
    shape, stride = a.shape, a.stride()
    if len(shape) == 2:
        n, w = shape
        s = stride[0] if n > 1 else w
    elif len(shape) == 1:
        n, w = 1, shape[0]
        s = w
    else:
        raise ValueError("rows must lie in a tensor of one or two dimensions")
    if stride[-1] != 1 and w > 1:
        raise ValueError("rows must be contiguous")
    dt = a.dtype
    code = _CODES.get(dt)
    if code is None:
        code = _CODES[dt] = _dtype_code(a)
    return n, w, a.data_ptr(), s, code


_WORDS: dict = {}                # dtype -> whether it is f32 (True) or a 32-bit integer (False)


def _words(a, n: int, what: str, floats: bool = True) -> int:
    """Pointer of a contiguous device vector of n 32-bit words (floats or integers); 0 for None."""
    if a is None:
        return 0
    dt = a.dtype
    kind = _WORDS.get(dt)
    if kind is None:
        kind = _WORDS[dt] = {"float32": True, "int32": False, "uint32": False}.get(str(dt).removeprefix("torch."), str(dt))
    if kind is not floats or a.numel() != n or not a.is_contiguous():
        raise ValueError(f"{what}: {n} contiguous values of type {'f32' if floats else '32-bit integer'} are needed")
    return a.data_ptr()


class Context:
    """One device context (gx_create ... gx_destroy)."""

    def __init__(self, device: int = 0, max_tokens: int = 64, max_layers: int = 1, flags: int = 0,
                 rank: int = 0, world: int = 1, nccl_id: bytes | None = None):
        self.lib = load()
        table = CODEBOOK_PATH.read_bytes()
        self._codebook = ctypes.create_string_buffer(table, len(table))
        opts = Options(device, rank, world, max_tokens, max_layers, flags,
                       ctypes.cast(self._codebook, ctypes.c_void_p), len(table))
        if nccl_id:
            ctypes.memmove(opts.nccl_id, nccl_id, min(128, len(nccl_id)))
        h = ctypes.c_void_p()
        _check(self.lib.gx_create(ctypes.byref(opts), ctypes.byref(h)), "gx_create")
        self.handle = h
        self.device = device
        self._ticket = ctypes.c_uint64()                 # of the operator calls (one thread uses a context)
        self._ticket_ref = ctypes.byref(self._ticket)
        self.max_tokens = max_tokens
        self.layers: dict[int, dict] = {}
        self.matrices: dict[int, tuple[int, int]] = {}   # (rows, cols) by handle

    # --- lifecycle -----------------------------------------------------------------------
    def close(self, timeout_ms: int = 60000) -> None:
        if self.handle:
            _check(self.lib.gx_destroy(self.handle, timeout_ms), "gx_destroy")
            self.handle = None

    def __enter__(self):
        return self

    def __exit__(self, *exc):
        self.close()

    def caps(self) -> Caps:
        c = Caps()
        _check(self.lib.gx_get_caps(self.handle, ctypes.byref(c)), "gx_get_caps")
        return c

    def stream(self) -> int:
        s = ctypes.c_void_p()
        _check(self.lib.gx_get_stream(self.handle, ctypes.byref(s)), "gx_get_stream")
        return s.value or 0

    # --- upload ----------------------------------------------------------------------------
    def upload_layer(self, index: int, layer: dict, timeout_ms: int = 600000) -> None:
        keep = []

        def arr(a, dtype):
            if a is None:
                return None
            a = np.ascontiguousarray(a, dtype=dtype)
            keep.append(a)
            return a.ctypes.data

        gate, up, down = (np.ascontiguousarray(layer[k], dtype=np.uint8) for k in ("gate", "up", "down"))
        keep += [gate, up, down]
        gs = layer.get("gate_signs")
        desc = LayerDesc(layer["type_id"], layer["n_expert"], layer["n_embd"], layer["n_ff"], layer["n_used"],
                         layer.get("expert_weights_scale", 0.0), gate.ctypes.data, up.ctypes.data, down.ctypes.data,
                         gate.nbytes, up.nbytes, down.nbytes, arr(layer["router"], np.float32),
                         arr(gs, np.float32), arr(layer.get("up_signs", gs), np.float32),
                         arr(layer.get("down_signs"), np.float32), arr(layer.get("router_bias"), np.float32))
        _check(self.lib.gx_upload_layer(self.handle, index, ctypes.byref(desc), timeout_ms), "gx_upload_layer")
        self.layers[index] = {k: layer[k] for k in ("n_embd", "n_used", "n_expert")}
        if layer.get("shared") is not None:
            self.upload_shared(index, layer["shared"], timeout_ms)

    def upload_shared(self, index: int, shared: dict | None, timeout_ms: int = 600000) -> None:
        """gx_upload_shared: the layer's shared expert (synth.make_shared layout), or None to drop it."""
        if shared is None:
            _check(self.lib.gx_upload_shared(self.handle, index, None, timeout_ms), "gx_upload_shared")
            return
        mats = [np.ascontiguousarray(shared[k], dtype=np.uint8) for k in ("gate", "up", "down")]
        gi = np.ascontiguousarray(shared["gate_inp"], dtype=np.float32)
        desc = SharedDesc(shared["type_id"], shared["n_ff"], mats[0].ctypes.data, mats[1].ctypes.data,
                          mats[2].ctypes.data, mats[0].nbytes, mats[1].nbytes, mats[2].nbytes, gi.ctypes.data)
        _check(self.lib.gx_upload_shared(self.handle, index, ctypes.byref(desc), timeout_ms), "gx_upload_shared")

    def upload_hc(self, index: int, hc: dict | None, timeout_ms: int = 600000) -> None:
        """gx_upload_hc: the FFN block's hyper-connection mixer (synth.make_hc layout), or None."""
        if hc is None:
            _check(self.lib.gx_upload_hc(self.handle, index, None, timeout_ms), "gx_upload_hc")
            return
        mats = [np.ascontiguousarray(hc[k], dtype=np.uint8) for k in ("down", "up", "inject")]
        norm = np.ascontiguousarray(hc["norm"], dtype=np.float32)
        desc = HcDesc(hc["n_streams"], hc["rank"], hc["type_id"], hc["eps"], norm.ctypes.data, mats[0].ctypes.data,
                      mats[1].ctypes.data, mats[2].ctypes.data, mats[0].nbytes, mats[1].nbytes, mats[2].nbytes)
        _check(self.lib.gx_upload_hc(self.handle, index, ctypes.byref(desc), timeout_ms), "gx_upload_hc")

    def upload_layer_gguf(self, index: int, path, gguf_layer: int, timeout_ms: int = 600000) -> None:
        """gx_upload_layer_gguf: layer gguf_layer of a GGUF file into slot index."""
        _check(self.lib.gx_upload_layer_gguf(self.handle, index, str(path).encode(), gguf_layer, timeout_ms),
               "gx_upload_layer_gguf")
        info = gguf_layer_info(path, gguf_layer)
        self.layers[index] = {"n_embd": info.n_embd, "n_used": info.n_used, "n_expert": info.n_expert}

    # --- forward ---------------------------------------------------------------------------
    def forward(self, layer: int, x, y, ids=None, weights=None) -> int:
        """Device tensors (torch, on this context's device). Returns the ticket."""
        t = ctypes.c_uint64()
        n_tok = x.shape[0]
        _check(self.lib.gx_moe_forward(self.handle, layer, _ptr(x), _dtype_code(x), n_tok, _ptr(y), _dtype_code(y),
                                       _ptr(ids), _ptr(weights), ctypes.byref(t)), "gx_moe_forward")
        return t.value

    def ffn_block(self, layer: int, res, n_tok: int | None = None, mixed=None) -> int:
        """gx_ffn_block on a device f32 tensor res [n_tok, hc * n_embd], updated in place; mixed
        (optional device f32 [n_tok, n_embd]) receives the mixer's output. Returns the ticket."""
        t = ctypes.c_uint64()
        n = res.shape[0] if n_tok is None else n_tok
        _check(self.lib.gx_ffn_block(self.handle, layer, _ptr(res), n, _ptr(mixed), ctypes.byref(t)), "gx_ffn_block")
        return t.value

    def expert_counts(self, layer: int, reset: bool = False, timeout_ms: int = 60000) -> np.ndarray:
        """This rank's routed slots per global expert of a layer (expert-parallel contexts)."""
        n = self.layers[layer]["n_expert"]
        out = np.zeros(n, np.uint32)
        _check(self.lib.gx_read_expert_counts(self.handle, layer, out.ctypes.data, int(reset), timeout_ms),
               "gx_read_expert_counts")
        return out

    def replicate_experts(self, layer: int, experts, timeout_ms: int = 120000) -> None:
        """Collective: every rank serves the listed global experts of the layer for its own tokens."""
        ids = np.ascontiguousarray(np.asarray(experts, dtype=np.uint32))
        _check(self.lib.gx_replicate_experts(self.handle, layer, ids.ctypes.data if ids.size else None, ids.size,
                                             timeout_ms), "gx_replicate_experts")

    def forward_noalloc(self, layer: int, x, y, ids=None, weights=None) -> int:
        """gx_moe_forward_noalloc on device tensors: the decode layer on the library's static
        scratch, for at most NOALLOC_MAX_TOKENS tokens. Returns the ticket."""
        t = ctypes.c_uint64()
        _check(self.lib.gx_moe_forward_noalloc(self.handle, layer, _ptr(x), _dtype_code(x), x.shape[0], _ptr(y),
                                               _dtype_code(y), _ptr(ids), _ptr(weights), ctypes.byref(t)),
               "gx_moe_forward_noalloc")
        return t.value

    def forward_host(self, layer: int, x: np.ndarray, out_dtype=np.float32, timeout_ms: int = 60000,
                     want_routing: bool = False):
        """Host numpy in/out (bf16 passed as uint16 bit patterns)."""
        x = np.ascontiguousarray(x)
        n_tok, E = x.shape
        y = np.empty((n_tok, E), dtype=out_dtype)
        U = self.layers[layer]["n_used"]
        ids = np.empty((n_tok, U), np.uint32) if want_routing else None
        w = np.empty((n_tok, U), np.float32) if want_routing else None
        _check(self.lib.gx_moe_forward_host(self.handle, layer, x.ctypes.data, _dtype_code(x), n_tok, y.ctypes.data,
                                            _dtype_code(y), _ptr(ids), _ptr(w), timeout_ms), "gx_moe_forward_host")
        return (y, ids, w) if want_routing else y

    def stack_forward(self, first: int, n_layers: int, x, y) -> int:
        t = ctypes.c_uint64()
        _check(self.lib.gx_stack_forward(self.handle, first, n_layers, _ptr(x), _dtype_code(x), x.shape[0], _ptr(y),
                                         _dtype_code(y), ctypes.byref(t)), "gx_stack_forward")
        return t.value

    def stack_forward_host(self, first: int, n_layers: int, x: np.ndarray, out_dtype=np.float32,
                           timeout_ms: int = 60000) -> np.ndarray:
        x = np.ascontiguousarray(x)
        y = np.empty(x.shape, dtype=out_dtype)
        _check(self.lib.gx_stack_forward_host(self.handle, first, n_layers, x.ctypes.data, _dtype_code(x), x.shape[0],
                                              y.ctypes.data, _dtype_code(y), timeout_ms), "gx_stack_forward_host")
        return y

    def wait(self, ticket: int, timeout_ms: int = 60000) -> None:
        _check(self.lib.gx_wait(self.handle, ticket, timeout_ms), "gx_wait")

    def poll(self) -> int:
        t = ctypes.c_uint64()
        _check(self.lib.gx_poll(self.handle, ctypes.byref(t)), "gx_poll")
        return t.value

    def set_flags(self, flags: int) -> None:
        _check(self.lib.gx_set_flags(self.handle, flags), "gx_set_flags")

    def timings(self) -> Timings:
        t = Timings()
        _check(self.lib.gx_read_timings(self.handle, ctypes.byref(t)), "gx_read_timings")
        return t

    # --- conformance / standalone GEMV -----------------------------------------------------
    def decode_blocks(self, type_id: int, packed: bytes | np.ndarray, value_count: int,
                      expected: np.ndarray | None = None, timeout_ms: int = 60000):
        src = np.frombuffer(bytes(packed), dtype=np.uint8)
        out = np.empty(value_count, np.float32)
        err = ctypes.c_float(0.0)
        exp = None if expected is None else np.ascontiguousarray(expected, dtype=np.float32)
        rc = self.lib.gx_decode_blocks(self.handle, type_id, src.ctypes.data, src.size, out.ctypes.data, value_count,
                                       _ptr(exp), ctypes.byref(err), timeout_ms)
        return rc, out, err.value

    def upload_matrix(self, type_id: int, rows: int, cols: int, packed: np.ndarray, timeout_ms: int = 60000) -> int:
        p = np.ascontiguousarray(packed, dtype=np.uint8)
        h = ctypes.c_uint32()
        _check(self.lib.gx_upload_matrix(self.handle, type_id, rows, cols, p.ctypes.data, p.nbytes, ctypes.byref(h),
                                         timeout_ms), "gx_upload_matrix")
        self.matrices[h.value] = (rows, cols)
        return h.value

    def matvec(self, handle: int, x, y) -> int:
        """gx_matvec: y = W x on contiguous f32 rows, x [n, cols] and y [n, rows], n <= 64."""
        n, cols, xp, xs, xd = _rows(x)
        m, rows, yp, ys, yd = _rows(y)
        if n != m or self._other_shape(handle, rows, cols) or not (xd == yd == GX_F32 and xs == cols and ys == rows):
            raise ValueError("gx_matvec: contiguous f32 x [n, cols] and y [n, rows] are needed")
        self._here(x, y)
        t = ctypes.c_uint64()
        _check(self.lib.gx_matvec(self.handle, handle, xp, n, yp, ctypes.byref(t)), "gx_matvec")
        return t.value

    def _other_shape(self, handle: int, rows: int, cols: int) -> bool:
        """Whether the matrix has another shape (an unknown handle is the library's to refuse)."""
        return self.matrices.get(handle, (rows, cols)) != (rows, cols)

    # --- operators around the layer ----------------------------------------------------------
    # Device tensors of this context's device, rows in the last dimension; the work is enqueued on the
    # context's stream, which no stream of torch waits for or is waited for by: synchronise (or record and wait
    # for an event on ctx.stream()) between what torch enqueues on the tensors and the call, and wait for the
    # ticket before torch reads the results. Each returns the ticket, or 0 with ticket=False (calls captured into a graph).
    def _here(self, *tensors) -> None:
        """The tensors have to lie on this context's device: a kernel would fault on any other address."""
        dev = self.device
        for a in tensors:
            if a is not None and a.get_device() != dev:
                raise ValueError(f"a tensor does not lie on device {dev}")

    def _done(self, rc: int, call: str, ticket: bool) -> int:
        if rc != GX_OK:
            raise GxError(rc, call)
        return self._ticket.value if ticket else 0

    def linear(self, handle: int, x, y, ticket: bool = True) -> int:
        """gx_linear: y = W x for a 4-bit matrix, x [n, cols] and y [n, rows] in f32 or bf16, n <= 64."""
        n, cols, xp, xs, xd = _rows(x)
        m, rows, yp, ys, yd = _rows(y)
        if n != m or self._other_shape(handle, rows, cols):
            raise ValueError("gx_linear: x [n, cols] and y [n, rows] are needed")
        self._here(x, y)
        return self._done(self.lib.gx_linear(self.handle, handle, xp, xd, xs, n, yp, yd, ys,
                                             self._ticket_ref if ticket else None), "gx_linear", ticket)

    def norm(self, x, y, weight=None, eps: float = 1e-6, gate_weight=None, gate=None, ticket: bool = True) -> int:
        """gx_norm: y = norm(x) * weight, and gate = gate_weight . y for each row."""
        n, w, xp, xs, xd = _rows(x)
        m, v, yp, ys, yd = _rows(y)
        if n != m or v != w:
            raise ValueError("gx_norm: x and y of one shape are needed")
        d = _PACK_NORM(xp, yp, _words(weight, w, "weight"), _words(gate_weight, w, "gate_weight"), _words(gate, n, "gate"),
                       xs, ys, xd, yd, w, eps)
        self._here(x, y, weight, gate_weight, gate)
        return self._done(self.lib.gx_norm(self.handle, d, n, self._ticket_ref if ticket else None), "gx_norm", ticket)

    def norm_residual(self, y, res, res_out=None, post=None, post_norm: bool = True, eps: float = 1e-6,
                      res_scale: float = 1.0, block_scale: float = 1.0, gate=None, out=None, next_weight=None,
                      next_gate_weight=None, next_gate=None, ticket: bool = True) -> int:
        """gx_norm_residual: res_out = res_scale * res + block_scale * gate * norm(y; post) (y itself
        without post_norm), out = norm(res_out; next_weight). res_out None: res in place. gate: one f32
        logit per row (1-D) or one logit per element (2-D)."""
        n, w, yp, ys, yd = _rows(y)
        rn, rw, rp, rs, rd = _rows(res)
        on, ow, op, os_, od = _rows(res_out) if res_out is not None else (rn, rw, rp, rs, rd)
        gn, gw, gp, gs, gd, kind = n, w, 0, 0, GX_F32, GX_GATE_NONE
        if gate is not None and gate.ndim == 1:
            gp, kind = _words(gate, n, "gate"), GX_GATE_TOKEN
        elif gate is not None:
            (gn, gw, gp, gs, gd), kind = _rows(gate), GX_GATE_ELEMENT
        hn, hw, hp, hs, hd = _rows(out) if out is not None else (n, w, 0, 0, GX_F32)
        if not (n == rn == on == gn == hn and w == rw == ow == gw == hw and od == rd):
            raise ValueError("gx_norm_residual: rows of one shape, and res_out in the type of res, are needed")
        d = _PACK_RESIDUAL(yp, rp, op, gp, _words(post, w, "post"), hp, _words(next_weight, w, "next_weight"),
                           _words(next_gate_weight, w, "next_gate_weight"), _words(next_gate, n, "next_gate"),
                           ys, rs, os_, gs, hs, yd, rd, gd, hd, w, GX_RES_POST_NORM if post_norm else 0, kind,
                           eps, res_scale, block_scale)
        self._here(y, res, res_out, post, gate, out, next_weight, next_gate_weight, next_gate)
        return self._done(self.lib.gx_norm_residual(self.handle, d, n, self._ticket_ref if ticket else None),
                          "gx_norm_residual", ticket)

    def logprobs(self, logits, tokens=None, n_top: int = 0, scale: float = 1.0, logprob=None, rank=None, entropy=None,
                 top_ids=None, top_logprobs=None, ticket: bool = True) -> int:
        """gx_logprobs over rows of logits [n, vocab]; tokens, rank and top_ids are 32-bit integers."""
        n, v, p, s, dt = _rows(logits)
        if not n_top:       # empty outputs stand for none
            top_ids = None if top_ids is not None and top_ids.numel() == 0 else top_ids
            top_logprobs = None if top_logprobs is not None and top_logprobs.numel() == 0 else top_logprobs
        d = _PACK_LOGPROBS(p, _words(tokens, n, "tokens", False), _words(logprob, n, "logprob"),
                           _words(rank, n, "rank", False), _words(entropy, n, "entropy"),
                           _words(top_ids, n * n_top, "top_ids", False), _words(top_logprobs, n * n_top, "top_logprobs"),
                           s, dt, v, n_top, scale)
        self._here(logits, tokens, logprob, rank, entropy, top_ids, top_logprobs)
        return self._done(self.lib.gx_logprobs(self.handle, d, n, self._ticket_ref if ticket else None), "gx_logprobs",
                          ticket)

    def upload_norms(self, index: int, norms: dict | None, timeout_ms: int = 600000) -> None:
        """gx_upload_norms: pre, post and gate weights ([n_embd] f32 or None), post_norm, eps, res_scale and
        block_scale of a layer as a block of a residual stream, or None to drop them."""
        if norms is None:
            _check(self.lib.gx_upload_norms(self.handle, index, None, timeout_ms), "gx_upload_norms")
            return
        w = {}
        for k in ("pre", "post", "gate"):
            a = norms.get(k)
            w[k] = None if a is None else np.ascontiguousarray(a, dtype=np.float32)
            if a is not None and index in self.layers and w[k].shape != (self.layers[index]["n_embd"],):
                raise ValueError(f"{k}: one weight per hidden channel is needed")
        d = NormsDesc(_ptr(w["pre"]), _ptr(w["post"]), _ptr(w["gate"]), int(norms.get("post_norm", True)),
                      norms.get("eps", 1e-6), norms.get("res_scale", 1.0), norms.get("block_scale", 1.0))
        _check(self.lib.gx_upload_norms(self.handle, index, ctypes.byref(d), timeout_ms), "gx_upload_norms")

    def norm_block(self, first: int, n_layers: int, res) -> int:
        """gx_norm_block on a device f32 tensor res [n, n_embd], updated in place. Returns the ticket."""
        n, w, p, s, code = _rows(res)
        if s != w or code != GX_F32 or first not in self.layers or w != self.layers[first]["n_embd"]:
            raise ValueError("gx_norm_block: contiguous f32 rows of the layers' width are needed")
        self._here(res)
        t = ctypes.c_uint64()
        _check(self.lib.gx_norm_block(self.handle, first, n_layers, p, n, ctypes.byref(t)),
               "gx_norm_block")
        return t.value
