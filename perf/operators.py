"""The operators around the routed layer as timed cases: 4-bit matrix-vector products, the norms and
residual add around a block, and log probabilities of given tokens.

run(state) computes a case in plain torch operations, or, with `own` set, through the library's entry
points (gyro_moe.abi.Context). exact(case, seed) computes the same outputs in 64 bits.
"""
import math
import sys
from pathlib import Path

import numpy as np
import torch

own = False

DEVICE = "cuda"
Q4_0, Q4_1 = 2, 3          # GGUF type ids: groups of 32 weights, w = d (q - 8) and w = d q + m
BLOCK_BYTES = {Q4_0: 18, Q4_1: 20}
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16}
EPS = 1e-6


def listed():
    return [
        # one decode step's projection at the layer's hidden width: the smallest call, latency counts
        dict(name="matvec 1x2048x2048", op="matvec", type=Q4_0, rows=2048, cols=2048, n_tok=1, x="f32", y="f32"),
        # a few sequences through a fused projection, group minima, activations in bf16
        dict(name="matvec 5x5120x2560", op="matvec", type=Q4_1, rows=5120, cols=2560, n_tok=5, x="bf16", y="bf16"),
        # the output head of a wide vocabulary (an odd one) for one token
        dict(name="matvec 1x150001x2560", op="matvec", type=Q4_0, rows=150001, cols=2560, n_tok=1, x="bf16", y="f32"),
        # a projection down from four residual streams for a ragged batch, everything in f32
        dict(name="matvec 13x2560x10240", op="matvec", type=Q4_0, rows=2560, cols=10240, n_tok=13, x="f32", y="f32"),
        # a full decode batch through a large square projection
        dict(name="matvec 64x8192x8192", op="matvec", type=Q4_0, rows=8192, cols=8192, n_tok=64, x="bf16", y="bf16"),
        # the norm before a block for one token, with the block's gate logit
        dict(name="norm 1x2048", op="norm", n_tok=1, width=2048, x="f32", y="f32", gate=True),
        # between two blocks of a decode step: norm after, token gate, residual, next norm
        dict(name="residual 4x2560", op="residual", n_tok=4, width=2560, res="f32", y="bf16", out="bf16", gate="token",
             post=True, next=True),
        # between two blocks of a ragged continuous batch, a gate for every element
        dict(name="residual 4067x2048", op="residual", n_tok=4067, width=2048, res="f32", y="f32", out="bf16",
             gate="element", post=True, next=True),
        # the norm before a block of a long prefill
        dict(name="norm 16384x4096", op="norm", n_tok=16384, width=4096, x="bf16", y="bf16", gate=False),
        # the answer of one decode step, with a few alternatives
        dict(name="logprobs 1x32000", op="logprobs", n_rows=1, vocab=32000, x="f32", n_top=5, scale=1.0, masked=False),
        # a decode batch over a wide odd vocabulary, the most alternatives an interface offers
        dict(name="logprobs 64x150001", op="logprobs", n_rows=64, vocab=150001, x="bf16", n_top=20, scale=1.25,
             masked=False),
        # scoring a long prompt: every position, some of the vocabulary masked away
        dict(name="logprobs 1500x131073", op="logprobs", n_rows=1500, vocab=131073, x="f32", n_top=2, scale=1.0,
             masked=True),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["matvec", "matvec", "norm", "residual", "logprobs", "logprobs"])
    if op == "matvec":
        n_tok = _log_int(rng, 1, 64)
        cols = 32 * _log_int(rng, 4, 320)
        rows = _log_int(rng, 64, min(150001, 8192 * 8192 * 4 // cols, 8192 * 8192 * 64 // (cols * n_tok)))
        return dict(op=op, type=rng.choice([Q4_0, Q4_1]), rows=rows, cols=cols, n_tok=n_tok,
                    x=rng.choice(["f32", "bf16"]), y=rng.choice(["f32", "bf16"]))
    if op in ("norm", "residual"):
        width = _log_int(rng, 64, 8192)
        if rng.random() < 0.7:
            width = (width + 63) // 64 * 64
        n_tok = _log_int(rng, 1, min(16384, 4067 * 2048 // width))
        kinds = ["f32", "bf16"]
        if op == "norm":
            return dict(op=op, n_tok=n_tok, width=width, x=rng.choice(kinds), y=rng.choice(kinds),
                        gate=rng.random() < 0.5)
        return dict(op=op, n_tok=n_tok, width=width, res=rng.choice(kinds), y=rng.choice(kinds), out=rng.choice(kinds),
                    gate=rng.choice(["none", "token", "element"]), post=rng.random() < 0.7, next=rng.random() < 0.8)
    vocab = _log_int(rng, 2000, 262144)
    x = rng.choice(["f32", "bf16"])
    n_rows = _log_int(rng, 1, min(4096, 1500 * 131073 // vocab))
    return dict(op=op, n_rows=n_rows, vocab=vocab, x=x, n_top=rng.randint(0, 32), scale=rng.choice([1.0, 0.8, 1.25]),
                masked=rng.random() < 0.4)


def _randn(gen, *shape):
    return torch.randn(*shape, device=DEVICE, generator=gen)


def _packed(gen, kind, rows, cols):
    """Rows of groups as a model file holds them: fp16 d (and m), then 16 bytes of codes, weights j and
    j + 16 of a group in the low and high half of byte j. Codes of roughly normal weights."""
    groups = rows * cols // 32
    out = torch.empty(groups, BLOCK_BYTES[kind], dtype=torch.uint8, device=DEVICE)
    q = torch.empty(groups, 32, dtype=torch.uint8, device=DEVICE)
    step = 1 << 22
    for at in range(0, groups, step):
        n = min(step, groups - at)
        q[at:at + n] = (_randn(gen, n, 32) * 2.9 + 8.0).round().clamp(0, 15).to(torch.uint8)
    out[:, -16:] = q[:, :16] | (q[:, 16:] << 4)
    d = (0.02 / math.sqrt(cols)) * 20.0 * torch.exp(0.3 * _randn(gen, groups)) / 2.9
    if kind == Q4_0:       # the scale carries the sign of the group's largest weight
        d = torch.where(_randn(gen, groups) < 0, -d, d)
    d = d.half()
    out[:, 0:2] = d.view(torch.uint8).view(groups, 2)
    if kind == Q4_1:
        m = (-8.0 * d.float() + 0.5 * d.float() * _randn(gen, groups)).half()
        out[:, 2:4] = m.view(torch.uint8).view(groups, 2)
    return out.view(rows, cols // 32, BLOCK_BYTES[kind])


def _activations(gen, n, width, kind):
    """Rows of the sizes that hidden states have: unit scale, a few channels much larger."""
    x = _randn(gen, n, width)
    big = _randn(gen, width) > 2.4
    return torch.where(big, x * 12.0, x).to(DTYPES[kind]).contiguous()


class _Held:
    """A context that is closed with the state that holds it."""

    def __init__(self):
        pkg = str(Path(__file__).resolve().parents[1] / "gyro-dx_b200")
        if pkg not in sys.path:
            sys.path.insert(0, pkg)
        from gyro_moe import abi
        self.ctx = abi.Context(device=0, max_tokens=64, max_layers=1)

    def __del__(self):
        ctx = getattr(self, "ctx", None)
        if ctx is not None:
            ctx.close()


def _inputs(case, seed):
    gen = torch.Generator(device=DEVICE)
    gen.manual_seed(int(seed))
    op = case["op"]
    s = dict(case=case)
    if op == "matvec":
        s["w"] = _packed(gen, case["type"], case["rows"], case["cols"])
        s["x"] = _activations(gen, case["n_tok"], case["cols"], case["x"])
    elif op == "norm":
        s["x"] = _activations(gen, case["n_tok"], case["width"], case["x"])
        s["weight"] = 1.0 + 0.2 * _randn(gen, case["width"])
        s["gate_w"] = _randn(gen, case["width"]) / math.sqrt(case["width"]) if case["gate"] else None
    elif op == "residual":
        n, e = case["n_tok"], case["width"]
        s["block"] = (0.3 * _activations(gen, n, e, "f32")).to(DTYPES[case["y"]])
        s["res"] = (2.0 * _activations(gen, n, e, "f32")).to(DTYPES[case["res"]])
        s["post"] = 1.0 + 0.2 * _randn(gen, e) if case["post"] else None
        s["next"] = 1.0 + 0.2 * _randn(gen, e) if case["next"] else None
        s["gate"] = None
        if case["gate"] == "token":
            s["gate"] = _randn(gen, n)
        elif case["gate"] == "element":
            s["gate"] = _randn(gen, n, e).to(DTYPES[case["y"]])
    else:
        n, v = case["n_rows"], case["vocab"]
        x = _randn(gen, n, v) * 2.5
        x[:, :: max(1, v // 40)] += 6.0 * _randn(gen, n, 1).abs()      # a few likely tokens in each row
        if case["masked"]:
            x[:, v - v // 5:] = -math.inf
        s["logits"] = x.to(DTYPES[case["x"]])
        del x
        pick = torch.empty(n, v, device=DEVICE).exponential_(generator=gen).log_().neg_()
        drawn = (s["logits"].float() + pick).argmax(1)                   # tokens drawn from the rows
        any_ = torch.randint(0, v, (n,), device=DEVICE, generator=gen)
        s["tokens"] = torch.where(torch.rand(n, device=DEVICE, generator=gen) < 0.9, drawn, any_).to(torch.int32)
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    if not own:
        return s
    s["held"] = _Held()
    ctx = s["ctx"] = s["held"].ctx
    op = case["op"]
    new = lambda *shape, dtype: torch.empty(*shape, dtype=dtype, device=DEVICE)  # noqa: E731
    if op == "matvec":
        packed = s.pop("w").cpu().numpy().reshape(-1)
        s["handle"] = ctx.upload_matrix(case["type"], case["rows"], case["cols"], np.ascontiguousarray(packed))
        s["y"] = new(case["n_tok"], case["rows"], dtype=DTYPES[case["y"]])
    elif op == "norm":
        s["y"] = new(case["n_tok"], case["width"], dtype=DTYPES[case["y"]])
        s["gate_out"] = new(case["n_tok"], dtype=torch.float32) if case["gate"] else None
    elif op == "residual":
        s["res_out"] = torch.empty_like(s["res"])
        s["out"] = new(case["n_tok"], case["width"], dtype=DTYPES[case["out"]]) if case["next"] else None
    else:
        n, k = case["n_rows"], case["n_top"]
        s["logprob"], s["entropy"] = new(n, dtype=torch.float32), new(n, dtype=torch.float32)
        s["rank"] = new(n, dtype=torch.int32)
        s["top_ids"], s["top_logprobs"] = new(n, k, dtype=torch.int32), new(n, k, dtype=torch.float32)
    return s


def _run_own(s):
    ctx, case = s["ctx"], s["case"]
    op = case["op"]
    if op == "matvec":
        ctx.linear(s["handle"], s["x"], s["y"])
        return {"y": s["y"]}
    if op == "norm":
        ctx.norm(s["x"], s["y"], s["weight"], EPS, gate_weight=s["gate_w"], gate=s["gate_out"])
        return {"y": s["y"], "gate": s["gate_out"]} if case["gate"] else {"y": s["y"]}
    if op == "residual":
        ctx.norm_residual(s["block"], s["res"], s["res_out"], post=s["post"], post_norm=case["post"], eps=EPS,
                          res_scale=1.0, block_scale=0.7, gate=s["gate"], out=s["out"], next_weight=s["next"])
        return {"res": s["res_out"], "out": s["out"]} if case["next"] else {"res": s["res_out"]}
    ctx.logprobs(s["logits"], s["tokens"], n_top=case["n_top"], scale=case["scale"], logprob=s["logprob"],
                 rank=s["rank"], entropy=s["entropy"], top_ids=s["top_ids"], top_logprobs=s["top_logprobs"])
    return {k: s[k] for k in ("logprob", "rank", "entropy", "top_ids", "top_logprobs")}


def _dequantised(w, kind):
    d = w[..., 0:2].contiguous().view(torch.float16).float()
    code = w[..., -16:]
    q = torch.cat([code & 15, code >> 4], dim=-1).float()
    if kind == Q4_0:
        q = (q - 8.0) * d
    else:
        q = q * d + w[..., 2:4].contiguous().view(torch.float16).float()
    return q.view(w.shape[0], -1)


def _rms(x, weight):
    return x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * weight


def _plain_logprobs(s):
    case = s["case"]
    z = s["logits"].float() * case["scale"]
    top = z.amax(-1, keepdim=True)
    t = torch.where(z == top, torch.zeros_like(z), z - top)      # a row without any token left counts as even
    e = torch.exp(t)
    total = e.sum(-1, keepdim=True)
    entropy = torch.log(total)[:, 0] - torch.where(e > 0, e * t, torch.zeros_like(e)).sum(-1) / total[:, 0]
    given = z.gather(1, s["tokens"].long()[:, None])
    logprob = (given - top - torch.log(total))[:, 0]
    x = s["logits"].float()
    rank = ((x > x.gather(1, s["tokens"].long()[:, None])).sum(-1) + 1).to(torch.int32)
    # one whole number per logit that orders by value, then by lower id
    bits = (x + 0.0).view(torch.int32)
    bits = torch.where(bits < 0, bits ^ 0x7FFFFFFF, bits).long()
    key = bits * (1 << 32) + ((1 << 32) - 1 - torch.arange(z.shape[1], device=z.device))
    ids = ((1 << 32) - 1) - (key.topk(case["n_top"], dim=-1, sorted=True).values & ((1 << 32) - 1))
    return {"logprob": logprob, "rank": rank, "entropy": entropy, "top_ids": ids.to(torch.int32),
            "top_logprobs": z.gather(1, ids) - top - torch.log(total)}


def run(s):
    if own:
        return _run_own(s)
    case = s["case"]
    op = case["op"]
    if op == "matvec":
        y = s["x"].float() @ _dequantised(s["w"], case["type"]).T
        return {"y": y.to(DTYPES[case["y"]])}
    if op == "norm":
        h = _rms(s["x"].float(), s["weight"])
        y = h.to(DTYPES[case["y"]])
        return {"y": y, "gate": (h * s["gate_w"]).sum(-1)} if case["gate"] else {"y": y}
    if op == "residual":
        y = s["block"].float()
        if case["post"]:
            y = _rms(y, s["post"])
        if case["gate"] == "token":
            y = y / (1.0 + torch.exp(-s["gate"]))[:, None]
        elif case["gate"] == "element":
            y = y / (1.0 + torch.exp(-s["gate"].float()))
        r = s["res"].float() + 0.7 * y
        res = r.to(DTYPES[case["res"]])
        return {"res": res, "out": _rms(r, s["next"]).to(DTYPES[case["out"]])} if case["next"] else {"res": res}
    return _plain_logprobs(s)


def work(case):
    size = lambda kind: 4 if kind == "f32" else 2  # noqa: E731
    op = case["op"]
    if op == "matvec":
        r, c, n = case["rows"], case["cols"], case["n_tok"]
        return {"bytes": r * (c // 32) * BLOCK_BYTES[case["type"]] + n * c * size(case["x"]) + n * r * size(case["y"]),
                "flops": 2 * r * c * n}
    if op == "norm":
        n, e = case["n_tok"], case["width"]
        return {"bytes": n * e * (size(case["x"]) + size(case["y"])) + 4 * e * (2 if case["gate"] else 1),
                "flops": n * e * (6 if case["gate"] else 4)}
    if op == "residual":
        n, e = case["n_tok"], case["width"]
        per = size(case["y"]) + 2 * size(case["res"]) + (size(case["out"]) if case["next"] else 0)
        per += size(case["y"]) if case["gate"] == "element" else 0
        return {"bytes": n * e * per + 4 * e * (case["post"] + case["next"]) + (4 * n if case["gate"] == "token" else 0),
                "flops": n * e * (3 + 4 * case["post"] + 4 * case["next"] + 4 * (case["gate"] == "element"))}
    n, v = case["n_rows"], case["vocab"]
    return {"bytes": n * v * size(case["x"]) + n * 16 + n * case["n_top"] * 8, "flops": 6 * n * v}


def exact(case, seed):
    """The outputs of run() from the definitions, in 64 bits."""
    s = _inputs(case, seed)
    op = case["op"]
    if op == "matvec":
        w, x = s["w"], s["x"].double()
        j = torch.arange(32, device=DEVICE)
        y = torch.empty(case["n_tok"], case["rows"], dtype=torch.float64, device=DEVICE)
        step = max(1, (1 << 26) // case["cols"])
        for at in range(0, case["rows"], step):
            part = w[at:at + step]
            half = part[:, :, :-16].contiguous().view(torch.float16).double()
            code = (part[:, :, part.shape[2] - 16 + j % 16].int() >> (4 * (j // 16)).int()) & 15
            vals = half[..., :1] * (code.double() - 8) if case["type"] == Q4_0 else half[..., :1] * code.double() + half[..., 1:]
            y[:, at:at + step] = torch.einsum("tc,rc->tr", x, vals.reshape(part.shape[0], -1))
        return {"y": y}
    if op == "norm":
        x = s["x"].double()
        y = x / (x.pow(2).sum(1, keepdim=True) / case["width"] + EPS).sqrt() * s["weight"].double()
        return {"y": y, "gate": y @ s["gate_w"].double()} if case["gate"] else {"y": y}
    if op == "residual":
        y, r = s["block"].double(), s["res"].double()
        if case["post"]:
            y = y / (y.pow(2).sum(1, keepdim=True) / case["width"] + EPS).sqrt() * s["post"].double()
        if case["gate"] != "none":
            g = s["gate"].double()
            y = y * torch.sigmoid(g[:, None] if case["gate"] == "token" else g)
        r = r + 0.7 * y
        if not case["next"]:
            return {"res": r}
        return {"res": r, "out": r / (r.pow(2).sum(1, keepdim=True) / case["width"] + EPS).sqrt() * s["next"].double()}
    n, k = case["n_rows"], case["n_top"]
    got = {"logprob": [], "rank": [], "entropy": [], "top_logprobs": []}
    ids = []
    step = max(1, (1 << 27) // case["vocab"])
    for at in range(0, n, step):
        z = s["logits"][at:at + step].double() * case["scale"]
        own_z = z.gather(1, s["tokens"][at:at + step, None].long())
        got["rank"].append((z > own_z).sum(1).to(torch.int32) + 1)
        lp = z - torch.logsumexp(z, 1, keepdim=True)
        p = lp.exp()
        got["logprob"].append(lp.gather(1, s["tokens"][at:at + step, None].long())[:, 0])
        got["entropy"].append(-torch.where(p > 0, p * lp, 0.0).sum(1))
        best = torch.sort(z, dim=1, descending=True, stable=True)
        ids.append(best.indices[:, :k].to(torch.int32))
        got["top_logprobs"].append(lp.gather(1, best.indices[:, :k]))
    out = {name: torch.cat(v) for name, v in got.items()}
    return {**out, "top_ids": torch.cat(ids)}
