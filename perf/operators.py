"""Cases that measure the 8-bit floating point (e4m3) operators of ``nanopointllm_b200.fp8``.

Five operators, all with one fp32 scale for each block of 128:

* ``tokens``  - activations quantised per token and 128 columns
* ``norm``    - (x + residual), its RMSNorm, quantised the same way
* ``silu``    - SiLU(gate) * up, quantised the same way
* ``weight``  - a weight quantised per 128 x 128 block
* ``linear``  - the matrix product of such activations and weights (+ residual)

``own`` False computes them in elementary torch operations, True calls the
package. Sizes are those of the repository's 7B shape (hidden 4096,
intermediate 11008, vocabulary 32003, packed QKV 12288, packed gate/up 22016)
at decode batches, one 560-token prompt and a 16000-token prefill batch.
"""
from __future__ import annotations

import importlib.util
import math
import pathlib
import sys

import torch

own = False

BLOCK = 128
E4M3 = torch.float8_e4m3fn
E4M3_MAX = 448.0
SCALE_MIN = 2.0 ** -126  # the smallest normal fp32: the scale of an all-zero block
EPS = 1e-6
TYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
BYTES = {"fp16": 2, "bf16": 2, "fp32": 4}


# ------------------------------------------------------------------- cases
def listed():
    return [
        # a decode step of 8 sequences: the attention rows before the O projection
        {"name": "tokens, 8 rows", "op": "tokens", "m": 8, "k": 4096, "type": "fp16"},
        # the same rows of a 20 x 800-token prefill batch
        {"name": "tokens, 16000 rows", "op": "tokens", "m": 16000, "k": 4096, "type": "bf16"},
        # one sequence decoding: the residual's addition and the norm before a projection
        {"name": "norm, 1 row", "op": "norm", "m": 1, "k": 4096, "type": "fp16", "residual": True},
        # the same of a prefill batch
        {"name": "norm, 16000 rows", "op": "norm", "m": 16000, "k": 4096, "type": "bf16", "residual": True},
        # the input of the down projection: a decode batch, and a prefill batch
        {"name": "silu, 8 rows", "op": "silu", "m": 8, "k": 11008, "type": "fp16"},
        {"name": "silu, 16000 rows", "op": "silu", "m": 16000, "k": 11008, "type": "fp16"},
        # loading: one O projection; the LM head, whose last block of rows is not full
        {"name": "weight, 4096 x 4096", "op": "weight", "n": 4096, "k": 4096, "type": "bf16"},
        {"name": "weight, 32003 x 4096", "op": "weight", "n": 32003, "k": 4096, "type": "fp16"},
        # packed QKV of a decode batch of 8
        {"name": "linear, 8 x 12288 x 4096", "op": "linear", "m": 8, "n": 12288, "k": 4096, "type": "fp16",
         "residual": False},
        # LM head of the largest decode batch: an odd number of columns
        {"name": "linear, 64 x 32003 x 4096", "op": "linear", "m": 64, "n": 32003, "k": 4096, "type": "bf16",
         "residual": False},
        # down projection of one prompt (513 point rows and 47 text tokens) with the residual
        {"name": "linear, 560 x 4096 x 11008", "op": "linear", "m": 560, "n": 4096, "k": 11008, "type": "fp16",
         "residual": True},
        # packed gate/up of a prefill batch
        {"name": "linear, 16000 x 22016 x 4096", "op": "linear", "m": 16000, "n": 22016, "k": 4096, "type": "bf16",
         "residual": False},
    ]


def _size(rng, lo, hi):
    """A size spread over the logarithm of [lo, hi]: any integer, or rounded to 16 or 128 as layer sizes are."""
    v = math.exp(rng.uniform(math.log(lo), math.log(hi)))
    step = rng.choice((1, 1, 16, 128))
    return max(lo, min(hi, int(round(v / step)) * step))


def draw(rng):
    op = rng.choice(("tokens", "norm", "silu", "weight", "linear", "linear"))
    if op == "weight":
        return {"op": op, "n": _size(rng, 64, 32003), "k": _size(rng, 64, 11008),
                "type": rng.choice(("fp16", "bf16", "fp32"))}
    if op == "linear":
        return {"op": op, "m": _size(rng, 1, 16000), "n": _size(rng, 64, 22016), "k": _size(rng, 64, 4096),
                "type": rng.choice(("fp16", "bf16")), "residual": rng.random() < 0.5}
    c = {"op": op, "m": _size(rng, 1, 16000), "k": _size(rng, 64, 11008)}
    c["type"] = rng.choice(("fp16", "bf16", "fp32") if op == "tokens" else ("fp16", "bf16"))
    if op == "norm":
        c["residual"] = rng.random() < 0.5
    return c


def _blocks(n):
    return -(-n // BLOCK)


def work(case):
    op, k, b = case["op"], case["k"], BYTES[case["type"]]
    kb = _blocks(k)
    if op == "weight":
        n = case["n"]
        return {"bytes": n * k * (b + 1) + 4 * _blocks(n) * kb, "flops": 3 * n * k}
    m = case["m"]
    out = m * (k + 4 * kb)  # codes and scales
    if op == "tokens":
        return {"bytes": m * k * b + out, "flops": 3 * m * k}
    if op == "norm":
        # x and the residual in, the sum, the codes and the scales out
        return {"bytes": m * k * b * (3 if case["residual"] else 1) + k * b + out, "flops": 8 * m * k}
    if op == "silu":
        return {"bytes": 2 * m * k * b + out, "flops": 8 * m * k}
    n = case["n"]
    return {"bytes": out + n * k + 4 * _blocks(n) * kb + m * n * b * (2 if case["residual"] else 1),
            "flops": 2 * m * n * k}


# ------------------------------------------------------------------ inputs
def _activations(g, m, k, dtype):
    """Rows ~N(0, 1) with 1% of the channels x20; the last of several rows is
    zero, as a padded row of a decode bucket."""
    x = torch.randn(m, k, generator=g, device="cuda")
    hot = torch.rand(k, generator=g, device="cuda") < 0.01
    x[:, hot] *= 20.0
    if m > 4:
        x[-1] = 0.0
    return x.to(dtype)


def _rows16(q):
    """The same codes with rows that start on 16-byte boundaries."""
    k = q.shape[1]
    if k % 16 == 0:
        return q.contiguous()
    store = torch.zeros(q.shape[0], -(-k // 16) * 16, dtype=q.dtype, device=q.device)
    store[:, :k] = q
    return store[:, :k]


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    op, k, dtype = case["op"], case["k"], TYPES[case["type"]]
    if op == "tokens":
        return {"op": op, "x": _activations(g, case["m"], k, dtype)}
    if op == "norm":
        return {"op": op, "x": _activations(g, case["m"], k, dtype),
                "w": (1.0 + 0.1 * torch.randn(k, generator=g, device="cuda")).to(dtype),
                "residual": _activations(g, case["m"], k, dtype) if case["residual"] else None}
    if op == "silu":
        # the halves of one packed projection's output
        y = torch.randn(case["m"], 2 * k, generator=g, device="cuda").mul_(2.0).to(dtype)
        return {"op": op, "gate": y[:, :k], "up": y[:, k:]}
    w = torch.randn(case["n"], k, generator=g, device="cuda").mul_(0.02)
    if op == "weight":
        return {"op": op, "w": w.to(dtype)}
    qw, sw = _plain_weight(w)
    qa, sa = _plain_tokens(_activations(g, case["m"], k, torch.float32))
    res = torch.randn(case["m"], case["n"], generator=g, device="cuda").to(dtype) if case["residual"] else None
    return {"op": op, "qa": _rows16(qa), "sa": sa, "qw": _rows16(qw), "sw": sw, "residual": res, "type": dtype}


# ------------------------------------------------------------- plain forms
def _plain_codes(v, scale):
    """Codes of blocks v [..., 128] under their scales [..., 1]."""
    return (v * (1.0 / scale)).to(E4M3)


def _plain_tokens(x):
    """fp32 values [M, K] -> (codes [M, K], scales [M, ceil(K / 128)])."""
    m, k = x.shape
    v = torch.nn.functional.pad(x, (0, _blocks(k) * BLOCK - k)).view(m, _blocks(k), BLOCK)
    scale = (v.abs().amax(-1, keepdim=True) / E4M3_MAX).clamp_min(SCALE_MIN)
    return _plain_codes(v, scale).view(m, -1)[:, :k], scale.squeeze(-1)


def _plain_weight(w):
    """fp32 weight [N, K] -> (codes [N, K], scales [ceil(N / 128), ceil(K / 128)])."""
    n, k = w.shape
    nb, kb = _blocks(n), _blocks(k)
    v = torch.nn.functional.pad(w, (0, kb * BLOCK - k, 0, nb * BLOCK - n)).view(nb, BLOCK, kb, BLOCK)
    scale = (v.abs().amax((1, 3), keepdim=True) / E4M3_MAX).clamp_min(SCALE_MIN)
    return _plain_codes(v, scale).view(nb * BLOCK, kb * BLOCK)[:n, :k], scale.view(nb, kb)


def _plain_norm(x, w, residual):
    s = x if residual is None else (x.float() + residual.float()).to(x.dtype)
    v = s.float()
    y = v * (1.0 / torch.sqrt(v.square().mean(-1, keepdim=True) + EPS)) * w.float()
    q, scale = _plain_tokens(y)
    return (q, scale) if residual is None else (q, scale, s)


def _plain_silu(gate, up):
    g = gate.float()
    return _plain_tokens(g / (1.0 + torch.exp(-g)) * up.float())


def _spread(scale, rows, cols, row_block):
    """Scales of blocks as a value for each element of [rows, cols]."""
    return scale.repeat_interleave(row_block, 0)[:rows].repeat_interleave(BLOCK, 1)[:, :cols]


def _plain_linear(qa, sa, qw, sw, residual, dtype):
    (m, k), n = qa.shape, qw.shape[0]
    a = qa.float() * _spread(sa, m, k, 1)
    w = qw.float() * _spread(sw, n, k, BLOCK)
    y = a @ w.t()
    if residual is not None:
        y = y + residual.float()
    return y.to(dtype)


# ----------------------------------------------------------------- one pass
_fp8 = None


def _package():
    """nanopointllm_b200.fp8; the package's folder has a hyphen, so it is registered by hand."""
    global _fp8
    if _fp8 is None:
        if "nanopointllm_b200" not in sys.modules:
            folder = pathlib.Path(__file__).resolve().parent.parent / "nano-pointllm_b200"
            spec = importlib.util.spec_from_file_location("nanopointllm_b200", folder / "__init__.py",
                                                          submodule_search_locations=[str(folder)])
            module = importlib.util.module_from_spec(spec)
            sys.modules["nanopointllm_b200"] = module
            spec.loader.exec_module(module)
        _fp8 = importlib.import_module("nanopointllm_b200.fp8")
    return _fp8


def run(state):
    op = state["op"]
    if own:
        f = _package()
        if op == "tokens":
            return f.quantize_token_blocks(state["x"])
        if op == "norm":
            q, scale, total = f.rmsnorm_quant_blocks(state["x"], state["w"], EPS, state["residual"])
            return (q, scale) if total is None else (q, scale, total)
        if op == "silu":
            return f.silu_mul_quant_blocks(state["gate"], state["up"])
        if op == "weight":
            return f.quantize_weight_blocks(state["w"])
        return f.linear_blocks(state["qa"], state["sa"], state["qw"], state["sw"], residual=state["residual"],
                               out_dtype=state["type"])
    if op == "tokens":
        return _plain_tokens(state["x"].float())
    if op == "norm":
        return _plain_norm(state["x"], state["w"], state["residual"])
    if op == "silu":
        return _plain_silu(state["gate"], state["up"])
    if op == "weight":
        return _plain_weight(state["w"].float())
    return _plain_linear(state["qa"], state["sa"], state["qw"], state["sw"], state["residual"], state["type"])


# -------------------------------------------------------------------- exact
def _exact_blocks(v, rows):
    """64-bit values [R, K] and the rows of a block -> (the quotients that the
    codes stand for before they are rounded, the scales)."""
    r, k = v.shape
    rb, kb = -(-r // rows), _blocks(k)
    full = torch.zeros(rb * rows, kb * BLOCK, dtype=torch.float64, device=v.device)
    full[:r, :k] = v
    tiles = full.reshape(rb, rows, kb, BLOCK).transpose(1, 2)
    scale = torch.clamp(tiles.abs().flatten(2).max(-1).values / 448.0, min=2.0 ** -126)
    codes = (tiles / scale[:, :, None, None]).transpose(1, 2).reshape(rb * rows, kb * BLOCK)
    return codes[:r, :k], scale


def exact(case, seed):
    s = prepare(case, seed)
    op = s["op"]
    if op == "tokens":
        return _exact_blocks(s["x"].double(), 1)
    if op == "weight":
        return _exact_blocks(s["w"].double(), 128)
    if op == "silu":
        g = s["gate"].double()
        return _exact_blocks(g * torch.sigmoid(g) * s["up"].double(), 1)
    if op == "norm":
        x = s["x"].double()
        total = None
        if s["residual"] is not None:  # the norm reads the sum as it is stored
            total = x + s["residual"].double()
            x = total.to(s["x"].dtype).double()
        y = x * torch.rsqrt((x * x).sum(-1, keepdim=True) / x.shape[-1] + EPS) * s["w"].double()
        q, scale = _exact_blocks(y, 1)
        return (q, scale) if total is None else (q, scale, total)
    # linear: one block of 128 columns after the other, scales applied to its sums
    qa, qw, k = s["qa"].double(), s["qw"].double(), case["k"]
    y = torch.zeros(case["m"], case["n"], dtype=torch.float64, device=qa.device)
    for b in range(_blocks(k)):
        at = slice(b * 128, min(k, b * 128 + 128))
        col = s["sw"][:, b].double().repeat_interleave(128)[: case["n"]]
        y += (qa[:, at] @ qw[:, at].t()) * s["sa"][:, b, None].double() * col
    return y if s["residual"] is None else y + s["residual"].double()
