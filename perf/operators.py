"""The operators of a layer whose products run in 8-bit floating point (e4m3
with one fp32 scale per block of 128): the residual add + RMS norm that
quantises its output, the quantisation of activations and weights, and the
product with its epilogues.

Quantisation of a block with largest magnitude A: scale s = max(A / 448,
2^-126), q = e4m3(x / s).  Activations take a scale per row and 128 columns,
weights one per 128 rows and 128 columns.

``listed()`` names the cases, ``draw(rng)`` gives one more of the same ranges,
``prepare`` makes what a program holds before the call, ``run`` is one pass
(elementary torch in 32 bits, or with ``own`` the framework's entry points),
``work`` the bytes and operations a pass cannot do without and ``exact`` the
result in 64 bits.
"""

import math
import os
import sys

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
SIZES = {"bf16": 2, "fp16": 2, "fp32": 4, "e4m3": 1}
E4M3 = torch.float8_e4m3fn
E4M3_MAX = 448.0
MIN_SCALE = 2.0 ** -126
BLOCK = 128
WEIGHT_STD = 0.02
EPS = 1e-5


def listed():
    return [
        # The norm before a projection while single tokens of eight sequences
        # are processed: the latency of one call.
        dict(name="norm-tokens", kind="norm", rows=8, n=2048, res="bf16", delta="bf16"),
        # The norm between two blocks of the headline configuration (d 1024)
        # over the valid tokens of a ragged batch, fp32 residual stream.
        dict(name="norm-packed", kind="norm", rows=5430, n=1024, res="fp32", delta="bf16"),
        # The same for long prompts of a wide model with a bf16 residual
        # stream: a pure stream through memory.
        dict(name="norm-prompts", kind="norm", rows=32768, n=4096, res="bf16", delta="bf16"),
        # Activations that no norm comes before (the attention context, a
        # feed-forward intermediate), quantised per row.
        dict(name="quant-rows", kind="quant", rows=8192, n=8192, dtype="bf16", block_rows=1),
        # A weight matrix of an fp32 checkpoint, quantised when it is loaded;
        # neither dimension a whole number of blocks.
        dict(name="quant-weight", kind="quant", rows=2600, n=1008, dtype="fp32", block_rows=128),
        # A projection of single tokens of eight sequences: reads the weights
        # and little else.
        dict(name="gemm-tokens", kind="gemm", m=8, k=2048, n=8192, epilogue="bias", out="bf16"),
        # The small model's feed-forward up-projection on one short sequence.
        dict(name="gemm-short", kind="gemm", m=128, k=512, n=2048, epilogue="gelu", out="fp16"),
        # The headline model's feed-forward up-projection over a ragged
        # batch; its output goes straight into the next product, in 8 bits.
        dict(name="gemm-up", kind="gemm", m=5430, k=1024, n=4096, epilogue="gelu", out="e4m3"),
        # Its down-projection; the next norm adds the output to the residual.
        dict(name="gemm-down", kind="gemm", m=5430, k=4096, n=1024, epilogue="bias", out="bf16"),
        # Widths and a token count that are no multiple of any tile or block.
        dict(name="gemm-odd", kind="gemm", m=2443, k=1008, n=2600, epilogue="bias", out="fp16"),
        # The wide model's up-projection (d 2048, f 8192) over full sequences.
        dict(name="gemm-wide", kind="gemm", m=8192, k=2048, n=8192, epilogue="bias", out="bf16"),
        # The largest product in the range.
        dict(name="gemm-large", kind="gemm", m=8192, k=8192, n=8192, epilogue="bias", out="bf16"),
    ]


# ------------------------------------------------------------------ drawing

def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _width(rng, lo, hi, step):
    """A feature width: mostly whole matrix tiles, now and then not."""
    w = _log(rng, lo, hi)
    step = 64 if rng.random() < 0.6 else step
    return max(step, (w + step // 2) // step * step)


def _draw_norm(rng):
    return dict(kind="norm", rows=_log(rng, 1, 32768), n=_width(rng, 128, 8192, 8),
                res=rng.choice(["bf16", "fp16", "fp32", "fp32"]), delta=rng.choice(["bf16", "fp16", "none"]))


def _draw_quant(rng):
    return dict(kind="quant", rows=_log(rng, 1, 16384), n=_width(rng, 128, 8192, 8),
                dtype=rng.choice(["bf16", "bf16", "fp16", "fp32"]), block_rows=rng.choice([1, 1, 128]))


def _draw_gemm(rng):
    return dict(kind="gemm", m=_log(rng, 1, 16384), k=_width(rng, 128, 8192, 16), n=_width(rng, 128, 8192, 4),
                epilogue=rng.choice(["bias", "bias", "gelu"]), out=rng.choice(["bf16", "bf16", "fp16", "e4m3"]))


def draw(rng):
    make = rng.choice([_draw_norm, _draw_quant, _draw_gemm, _draw_gemm])
    while True:
        case = make(rng)
        w = work(case)
        if w["flops"] <= 8192.0 ** 3 and w["bytes"] <= 32768 * 4096 * 7:
            return case


# ------------------------------------------------------------------- inputs

class _Random:
    """Normal values on the GPU from one seed."""

    def __init__(self, seed):
        self.g = torch.Generator(device="cuda")
        self.g.manual_seed(seed)

    def normal(self, *shape, std=1.0, dtype=torch.float32):
        return (torch.randn(*shape, generator=self.g, device="cuda") * std).to(dtype)

    def activations(self, rows, n, dtype):
        """Rows of different magnitude, with a few columns that stand out, as
        the activations of a residual stream have them."""
        x = self.normal(rows, n)
        x *= torch.exp(0.5 * self.normal(rows, 1)) * torch.exp(0.7 * self.normal(1, n))
        return x.to(dtype)


def _blocks(n):
    return -(-n // BLOCK)


def prepare(case, seed):
    rng, kind = _Random(seed), case["kind"]
    s = {"kind": kind, "case": case}
    # the outputs of a layer are buffers that a program keeps
    if kind == "norm":
        rows, n, rdt = case["rows"], case["n"], DTYPES[case["res"]]
        s["res"] = rng.activations(rows, n, rdt)
        s["delta"] = None if case["delta"] == "none" else rng.normal(rows, n, std=0.5, dtype=DTYPES[case["delta"]])
        s["gamma"] = 1 + rng.normal(n, std=0.1)
        s["res_out"] = torch.empty(rows, n, dtype=rdt, device="cuda")
        s["q"] = torch.empty(rows, n, dtype=E4M3, device="cuda")
        s["scales"] = torch.empty(rows, _blocks(n), device="cuda")
        return s
    if kind == "quant":
        rows, n = case["rows"], case["n"]
        if case["block_rows"] == 1:
            s["x"] = rng.activations(rows, n, DTYPES[case["dtype"]])
        else:
            s["x"] = rng.normal(rows, n, std=WEIGHT_STD, dtype=DTYPES[case["dtype"]])
        s["q"] = torch.empty(rows, n, dtype=E4M3, device="cuda")
        s["scales"] = torch.empty(-(-rows // case["block_rows"]), _blocks(n), device="cuda")
        return s
    m, k, n = case["m"], case["k"], case["n"]
    s["a"], s["a_scales"] = _quantise(rng.activations(m, k, torch.bfloat16).float(), 1)
    w = rng.normal(n, k, std=WEIGHT_STD) * torch.exp(0.3 * rng.normal(n, 1))
    s["w"], s["w_scales"] = _quantise(w, BLOCK)
    s["bias"] = rng.normal(n, std=0.1, dtype=DTYPES.get(case["out"], torch.float32))
    if case["out"] == "e4m3":
        s["out"] = torch.empty(m, n, dtype=E4M3, device="cuda")
        s["out_scales"] = torch.empty(m, _blocks(n), device="cuda")
    else:
        s["out"] = torch.empty(m, n, dtype=DTYPES[case["out"]], device="cuda")
    return s


# --------------------------------------------------------------- plain form

def _in_blocks(x, block_rows):
    """x as [row blocks, block_rows, column blocks, 128], padded with zeros."""
    rows, n = x.shape
    rb, cb = -(-rows // block_rows), _blocks(n)
    if (rb * block_rows, cb * BLOCK) != (rows, n):
        whole = x.new_zeros(rb * block_rows, cb * BLOCK)
        whole[:rows, :n] = x
        x = whole
    return x.view(rb, block_rows, cb, BLOCK)


def _quantise(x, block_rows):
    """(q, scales) of an fp32 matrix."""
    rows, n = x.shape
    b = _in_blocks(x, block_rows)
    scales = (b.abs().amax(dim=(1, 3)) / E4M3_MAX).clamp(min=MIN_SCALE)
    q = (b / scales[:, None, :, None]).clamp(-E4M3_MAX, E4M3_MAX)
    return q.view(b.shape[0] * block_rows, -1)[:rows, :n].to(E4M3).contiguous(), scales


def _dequantise(q, scales, block_rows):
    rows, n = q.shape
    b = _in_blocks(q.float(), block_rows) * scales[:, None, :, None]
    return b.view(b.shape[0] * block_rows, -1)[:rows, :n]


def _plain_norm(s):
    x = s["res"].float()
    if s["delta"] is not None:
        x = x + s["delta"].float()
    y = x * torch.rsqrt((x * x).mean(dim=1, keepdim=True) + EPS) * s["gamma"]
    q, scales = _quantise(y, 1)
    return {"q": q, "scales": scales, "res": x.to(s["res"].dtype)}


def _plain_gemm(s):
    case = s["case"]
    v = torch.matmul(_dequantise(s["a"], s["a_scales"], 1), _dequantise(s["w"], s["w_scales"], BLOCK).t())
    v = v + s["bias"].float()
    if case["epilogue"] == "gelu":
        v = 0.5 * v * (1 + torch.erf(v * math.sqrt(0.5)))
    if case["out"] == "e4m3":
        q, scales = _quantise(v, 1)
        return {"out": q, "scales": scales}
    return {"out": v.to(DTYPES[case["out"]])}


def _ops():
    here = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    path = os.path.join(here if os.path.isdir(os.path.join(here, "tiktok-techjam-2026_amd")) else os.getcwd(),
                        "tiktok-techjam-2026_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    from tjkernels import ops
    return ops


def run(state):
    s, kind = state, state["kind"]
    if not own:
        if kind == "norm":
            return _plain_norm(s)
        if kind == "quant":
            q, scales = _quantise(s["x"].float(), s["case"]["block_rows"])
            return {"q": q, "scales": scales}
        return _plain_gemm(s)
    ops = sys.modules.get("tjkernels.ops") or _ops()
    if kind == "norm":
        ops.add_rmsnorm(s["res"], s["delta"], s["gamma"], EPS, s["q"], res_out=s["res_out"], scales=s["scales"])
        return {"q": s["q"], "scales": s["scales"], "res": s["res_out"]}
    if kind == "quant":
        ops.quantize_f8(s["x"], s["q"], s["scales"], block_rows=s["case"]["block_rows"])
        return {"q": s["q"], "scales": s["scales"]}
    epilogue = ops.EPI_BIAS_GELU if s["case"]["epilogue"] == "gelu" else ops.EPI_BIAS
    ops.gemm_f8(s["a"], s["a_scales"], s["w"], s["w_scales"], s["bias"], s["out"], epilogue,
                out_scales=s.get("out_scales"))
    return {"out": s["out"], "scales": s["out_scales"]} if "out_scales" in s else {"out": s["out"]}


# --------------------------------------------------------------------- work

def work(case):
    kind = case["kind"]
    if kind == "norm":
        rows, n = case["rows"], case["n"]
        each = 2 * SIZES[case["res"]] + (0 if case["delta"] == "none" else SIZES[case["delta"]]) + 1
        return {"bytes": rows * n * each + 4 * rows * _blocks(n) + 4 * n, "flops": 8.0 * rows * n}
    if kind == "quant":
        rows, n = case["rows"], case["n"]
        scales = -(-rows // case["block_rows"]) * _blocks(n)
        return {"bytes": rows * n * (SIZES[case["dtype"]] + 1) + 4 * scales, "flops": 3.0 * rows * n}
    m, k, n = case["m"], case["k"], case["n"]
    scales = m * _blocks(k) + _blocks(n) * _blocks(k) + (m * _blocks(n) if case["out"] == "e4m3" else 0)
    bias = n * (4 if case["out"] == "e4m3" else 2)
    return {"bytes": m * k + n * k + 4 * scales + bias + m * n * SIZES[case["out"]], "flops": 2.0 * m * n * k}


# ------------------------------------------------------------------ results

def _exact_quotient(y, block_rows):
    """(x / s, s) of a 64-bit matrix, the quotients not rounded."""
    rows, n = y.shape
    q, scales = torch.empty_like(y), []
    for c in range(0, n, BLOCK):
        col = y[:, c:c + BLOCK]
        top = col.abs().amax(dim=1)
        if block_rows > 1:
            top = torch.stack([t.amax() for t in top.split(block_rows)])
        sc = torch.clamp(top / E4M3_MAX, min=MIN_SCALE)
        scales.append(sc)
        q[:, c:c + BLOCK] = col / sc.repeat_interleave(block_rows)[:rows, None]
    return q, torch.stack(scales, dim=1)


def exact(case, seed):
    s, kind = prepare(case, seed), case["kind"]
    if kind == "quant":
        q, scales = _exact_quotient(s["x"].double(), case["block_rows"])
        return {"q": q, "scales": scales}
    if kind == "norm":
        x = s["res"].double()
        if s["delta"] is not None:
            x += s["delta"].double()
        root = (x.square().sum(dim=1) / case["n"] + EPS).sqrt()
        q, scales = _exact_quotient(x / root[:, None] * s["gamma"].double(), 1)
        return {"q": q, "scales": scales, "res": x}
    m, k, n = case["m"], case["k"], case["n"]
    v = s["bias"].double().expand(m, n).clone()
    for b in range(_blocks(k)):
        part = torch.matmul(s["a"][:, b * BLOCK:(b + 1) * BLOCK].double(),
                            s["w"][:, b * BLOCK:(b + 1) * BLOCK].double().t().contiguous())
        part *= s["a_scales"][:, b].double()[:, None]
        part *= s["w_scales"][:, b].double().repeat_interleave(BLOCK)[None, :n]
        v += part
    if case["epilogue"] == "gelu":
        v *= 0.5 * torch.special.erfc(-v * math.sqrt(0.5))
    if case["out"] == "e4m3":
        q, scales = _exact_quotient(v, 1)
        return {"out": q, "scales": scales}
    return {"out": v}
