"""Block-scaled 8-bit floating point (e4m3) linears and their activation
quantisers, beside the int8 contract of ``w8a8``.

One fp32 scale for each block of 128: 128 consecutive columns of a token, or a
128 x 128 tile of a weight (the last ones may be partial). For a block of
values v

    scale = max(max |v| / 448, 2^-126),  q = e4m3(v * (1 / scale)),  v ~ q * scale

in fp32 (448 is the largest e4m3 value), and a linear is

    out[m, n] = sum_b sa[m, b] * sw[n // 128, b] * sum_{k in block b} qa[m, k] * qw[n, k]

with fp32 sums and one rounding to fp16 or bf16. A block that holds a NaN or
an infinity reads back as NaN altogether; other blocks are not affected. The
reference project has no counterpart (its only 8-bit form is int8).

* ``quantize_token_blocks``   - activations, per token and 128 columns
* ``rmsnorm_quant_blocks``    - (x + residual), RMSNorm, quantised (cf. runner.rmsnorm_quant)
* ``silu_mul_quant_blocks``   - SiLU(gate) * up, quantised
* ``quantize_weight_blocks``  - a weight, per 128 x 128 block
* ``linear_blocks``           - the matrix product (+ bias, + residual)
* ``Fp8BlockLinear``          - a quantised Linear (cf. w8a8.W8A8Linear)

A decoder layer's MLP reads ``rmsnorm_quant_blocks`` -> ``linear_blocks``
(packed gate/up rows) -> ``silu_mul_quant_blocks`` on the two halves ->
``linear_blocks(..., residual=...)``. Every call runs kernels of libnpl_w8a8 on
the current stream of its tensors' device; none synchronises, keeps a
workspace or reads anything back, and every one can be captured into a CUDA
graph. CUDA tensors only. Codes come and go as torch.float8_e4m3fn.
"""
from __future__ import annotations

import torch

from . import _lib as L

BLOCK = 128

_E4M3 = torch.float8_e4m3fn
_DT16 = {torch.float16: L.NPL_F16, torch.bfloat16: L.NPL_BF16}
_DT = {torch.float32: L.NPL_F32, **_DT16}

_quant_rows, _quant_weight = L.lib.npl_fp8_quant_rows, L.lib.npl_fp8_quant_weight
_rmsnorm_quant, _silu_mul_quant = L.lib.npl_fp8_rmsnorm_quant, L.lib.npl_fp8_silu_mul_quant
_linear = L.lib.npl_fp8_linear


def _blocks(n: int) -> int:
    return -(-n // BLOCK)


def _same_device(first: torch.Tensor, *others: torch.Tensor | None) -> None:
    d = first.get_device()
    if d < 0:
        raise ValueError("the fp8 path runs on CUDA tensors only")
    for t in others:
        if t is not None and t.get_device() != d:
            raise ValueError(f"tensors on different devices: {first.device} and {t.device}")


# Raw queries and bound names below: a call on a few rows is bound by the host
# (torch.cuda.current_stream alone takes as long as the kernel). A torch build
# without the raw ones has the public ones.
_current_device = getattr(torch._C, "_cuda_getDevice", None) or torch.cuda.current_device
_current_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (
    lambda index: torch.cuda.current_stream(index).cuda_stream)
_empty = torch.empty_strided


def _call(fn, device: torch.device, *args) -> None:
    """fn(*args, stream) with ``device`` current, on its current stream."""
    i = device.index
    if i == _current_device():
        rc = fn(*args, _current_stream(i))
    else:
        with torch.cuda.device(i):
            rc = fn(*args, _current_stream(i))
    if rc:
        L.check(rc)


def _rows(t: torch.Tensor) -> torch.Tensor:
    """[..., K] as [rows, K] with contiguous columns and rows that do not
    overlap (a copy only where the strides do not allow a view)."""
    t = t if t.dim() == 2 else t.reshape(-1, t.shape[-1])
    if t.is_contiguous():
        return t
    r, k = t.shape
    if (k > 1 and t.stride(1) != 1) or (r > 1 and t.stride(0) < k):
        t = t.contiguous()
    return t


def _new_codes(rows: int, k: int, device: torch.device) -> torch.Tensor:
    """e4m3 [rows, K] whose rows start on 16-byte boundaries, as the linear reads them."""
    return _empty((rows, k), (-(-k // 16) * 16, 1), dtype=_E4M3, device=device)


def _outputs(rows: int, k: int, device: torch.device, scale_rows: int) -> tuple[torch.Tensor, torch.Tensor, int, int]:
    """New (codes [rows, K], scales [scale_rows, ceil(K / 128)]) and their row strides."""
    ld, kb = (k + 15) & ~15, (k + 127) // BLOCK
    return (_empty((rows, k), (ld, 1), dtype=_E4M3, device=device),
            _empty((scale_rows, kb), (kb, 1), dtype=torch.float32, device=device), ld, kb)


def _activation(name: str, t: torch.Tensor, types: dict) -> int:
    dt = types.get(t.dtype)
    if dt is None:
        raise ValueError(f"{name} must be one of {', '.join(str(d).replace('torch.', '') for d in types)}")
    if t.dim() == 0 or t.shape[-1] == 0:
        raise ValueError(f"{name} needs at least one column")
    return dt


def quantize_token_blocks(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """fp16, bf16 or fp32 [..., K] -> (codes e4m3 [..., K], scales fp32
    [..., ceil(K / 128)])."""
    _same_device(x)
    dt = _activation("x", x, _DT)
    v = _rows(x)
    m, k = v.shape
    dev = x.device
    q, s, ldq, kb = _outputs(m, k, dev, m)
    if m:
        _call(_quant_rows, dev, v.data_ptr(), dt, m, k, v.stride(0), q.data_ptr(), ldq, s.data_ptr(), kb)
    return (q, s) if x.dim() == 2 else (q.reshape(x.shape), s.reshape(*x.shape[:-1], kb))


def quantize_weight_blocks(weight: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """fp16, bf16 or fp32 [N, K] -> (codes e4m3 [N, K], scales fp32
    [ceil(N / 128), ceil(K / 128)])."""
    _same_device(weight)
    if weight.dim() != 2 or weight.shape[0] == 0:
        raise ValueError("weight must be [N, K] with N >= 1")
    dt = _activation("weight", weight, _DT)
    w = _rows(weight.detach())
    n, k = w.shape
    dev = w.device
    q, s, ldq, kb = _outputs(n, k, dev, _blocks(n))
    _call(_quant_weight, dev, w.data_ptr(), dt, n, k, w.stride(0), q.data_ptr(), ldq, s.data_ptr(), kb)
    return q, s


def rmsnorm_quant_blocks(x: torch.Tensor, weight: torch.Tensor, eps: float, residual: torch.Tensor | None = None, *,
                         sum_out: torch.Tensor | None = None):
    """RMSNorm (of x + residual when given) fused with the token quantiser.
    x, residual fp16 or bf16 [M, K], weight [K], one type. Returns (codes
    [M, K], scales [M, ceil(K / 128)], sum): the sum is x + residual in their
    type, which the norm reads, in ``sum_out`` when given (it may be x or
    residual itself), else in new rows that start 32 bytes aligned; None
    without a residual. The norm stays in fp32 up to the codes."""
    _same_device(x, weight, residual, sum_out)
    dt, shape = _activation("x", x, _DT16), x.shape
    if len(shape) != 2 or weight.shape != shape[1:] or weight.dtype is not x.dtype:
        raise ValueError("x must be [M, K] and weight [K], of one type")
    m, k = shape
    dev = x.device
    v = _rows(x)
    w = weight if weight.is_contiguous() else weight.contiguous()
    res = total = None
    ld_res = ld_sum = 0
    if residual is not None:
        if residual.shape != shape or residual.dtype is not x.dtype:
            raise ValueError("residual must have the shape and type of x")
        r = _rows(residual)
        if sum_out is None:
            ld_sum = (k + 15) & ~15
            sum_out = _empty(shape, (ld_sum, 1), dtype=x.dtype, device=dev)
        else:
            if sum_out.shape != shape or sum_out.dtype is not x.dtype:
                raise ValueError("sum_out must have the shape and type of x")
            if _rows(sum_out) is not sum_out:
                raise ValueError("sum_out needs contiguous columns and rows that do not overlap")
            if _overlap(sum_out, x, residual, itself=True) or _overlap(sum_out, weight):
                raise ValueError("sum_out may be x or residual itself, but not overlap an input otherwise")
            ld_sum = sum_out.stride(0)
        res, ld_res, total = r.data_ptr(), r.stride(0), sum_out.data_ptr()
    elif sum_out is not None:
        raise ValueError("sum_out needs a residual")
    q, s, ldq, kb = _outputs(m, k, dev, m)
    if m:
        _call(_rmsnorm_quant, dev, v.data_ptr(), v.stride(0), res, ld_res, w.data_ptr(), dt, eps, m, k, total, ld_sum,
              q.data_ptr(), ldq, s.data_ptr(), kb)
    return q, s, sum_out


def silu_mul_quant_blocks(gate: torch.Tensor, up: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """SiLU(gate) * up of fp16 or bf16 [M, K] rows (for a packed gate/up
    projection: its two column halves), in fp32 up to the codes. Returns
    (codes [M, K], scales [M, ceil(K / 128)])."""
    _same_device(gate, up)
    dt, shape = _activation("gate", gate, _DT16), gate.shape
    if len(shape) != 2 or up.shape != shape or up.dtype is not gate.dtype:
        raise ValueError("gate and up must be [M, K] of one shape and type")
    g, u = _rows(gate), _rows(up)
    m, k = shape
    dev = g.device
    q, s, ldq, kb = _outputs(m, k, dev, m)
    if m:
        _call(_silu_mul_quant, dev, g.data_ptr(), g.stride(0), u.data_ptr(), u.stride(0), dt, m, k, q.data_ptr(), ldq,
              s.data_ptr(), kb)
    return q, s


def _overlap(out: torch.Tensor, *others: torch.Tensor | None, itself: bool = False) -> bool:
    """Whether the memory of ``out`` and another tensor may meet: their spans
    do, and they are not different columns of one buffer's rows. With
    ``itself`` the same elements of the same memory do not count."""
    def span(t):
        if t.is_contiguous():
            n = t.numel()
        else:
            n = sum((d - 1) * abs(st) for d, st in zip(t.shape, t.stride())) + 1 if t.numel() else 0
        return t.data_ptr(), t.data_ptr() + n * t.element_size()

    def columns(a, b):
        ld, size = a.stride(0), a.element_size()
        at, off = divmod(b.data_ptr() - a.data_ptr(), size)
        return (a.dim() == b.dim() == 2 and a.stride() == b.stride() and a.stride(1) == 1 and size == b.element_size()
                and off == 0 and ld > 0 and at % ld >= a.shape[1] and at % ld + b.shape[1] <= ld)

    def same(a, b):  # the stride of a single row or column does not count
        return a.shape == b.shape and all(n == 1 or x == y for n, x, y in zip(a.shape, a.stride(), b.stride()))

    a0, a1 = span(out)
    for t in others:
        if t is None or (itself and t is out):
            continue
        b0, b1 = span(t)
        if a0 < b1 and b0 < a1 and not columns(out, t) and not (itself and a0 == b0 and same(t, out)):
            return True
    return False


def _code_rows(name: str, q: torch.Tensor) -> tuple[int, int, int]:
    """(rows, K, row stride) of codes; a single row's stride is K rounded up to 16."""
    if q.dtype is not _E4M3 or q.dim() != 2:
        raise ValueError(f"{name} must be float8_e4m3fn [rows, K]")
    rows, k = q.shape
    ld, step = q.stride()
    if rows <= 1:
        ld = -(-k // 16) * 16
    if (step != 1 and k > 1) or (ld | q.data_ptr()) & 15 or ld < k:
        raise ValueError(f"{name} needs contiguous columns and rows on 16-byte boundaries, as the quantisers return them")
    return rows, k, ld


def _scales(name: str, s: torch.Tensor, rows: int, cols: int) -> tuple[torch.Tensor, int]:
    if s.dtype is not torch.float32 or s.shape != (rows, cols):
        raise ValueError(f"{name} must be float32 [{rows}, {cols}], got {s.dtype} {tuple(s.shape)}")
    s = _rows(s)
    return s, s.stride(0) if rows > 1 else cols


def linear_blocks(q: torch.Tensor, scale: torch.Tensor, qweight: torch.Tensor, wscale: torch.Tensor, *,
                  bias: torch.Tensor | None = None, residual: torch.Tensor | None = None,
                  out: torch.Tensor | None = None, out_dtype: torch.dtype | None = None) -> torch.Tensor:
    """Codes [M, K] with scales [M, ceil(K / 128)] times weight codes [N, K]
    with scales [ceil(N / 128), ceil(K / 128)] -> [M, N] (+ bias fp32 [N])
    (+ residual [M, N]), rounded once to ``out_dtype``: fp16 or bf16, by default
    the type of ``out`` or ``residual``, else bf16. ``out`` may be ``residual``
    itself. The product of two scales is formed first, in fp32: below 2^-126 it
    loses bits (2^-125 of an output for each such block), above fp32's largest
    number it makes the outputs of that token and those weight rows infinite or
    NaN."""
    _same_device(q, scale, qweight, wscale, bias, residual, out)
    m, k, lda = _code_rows("q", q)
    n, kw, ldw = _code_rows("qweight", qweight)
    if kw != k or k == 0 or n == 0:
        raise ValueError("linear input/weight shapes do not match")
    kb = (k + 127) // BLOCK
    sa, ld_sa = _scales("scale", scale, m, kb)
    sw, ld_sw = _scales("wscale", wscale, (n + 127) // BLOCK, kb)
    if out_dtype is None:
        out_dtype = out.dtype if out is not None else residual.dtype if residual is not None else torch.bfloat16
    dt = _DT16.get(out_dtype)
    if dt is None:
        raise ValueError("out_dtype must be float16 or bfloat16")
    add = res = None
    ld_res, ld_out = 0, n
    if bias is not None:
        if bias.dtype is not torch.float32 or bias.shape != (n,) or not bias.is_contiguous():
            raise ValueError("bias must be contiguous float32 [N]")
        add = bias.data_ptr()
    if residual is not None:
        if residual.shape != (m, n) or residual.dtype is not out_dtype:
            raise ValueError("residual must be [M, N] of out_dtype")
        r = _rows(residual)
        res, ld_res = r.data_ptr(), r.stride(0) if m > 1 else n
    dev = q.device
    if out is None:
        out = _empty((m, n), (n, 1), dtype=out_dtype, device=dev)
    else:
        if out.shape != (m, n) or out.dtype is not out_dtype:
            raise ValueError("out must be [M, N] of out_dtype")
        if _rows(out) is not out:
            raise ValueError("out needs contiguous columns and rows that do not overlap")
        if _overlap(out, residual, itself=True) or _overlap(out, q, scale, qweight, wscale, bias):
            raise ValueError("out may be residual itself, but not overlap an input otherwise")
        if m > 1:
            ld_out = out.stride(0)
    if m:
        _call(_linear, dev, q.data_ptr(), lda, sa.data_ptr(), ld_sa, qweight.data_ptr(), ldw, sw.data_ptr(), ld_sw, add,
              m, n, k, res, ld_res, out.data_ptr(), ld_out, dt)
    return out


class Fp8BlockLinear:
    """A quantised Linear: e4m3 weight codes [N, K] with fp32 scales
    [ceil(N / 128), ceil(K / 128)] and an optional fp32 bias. Calling it
    quantises the input's tokens and multiplies; the output has the input's
    type (fp16 or bf16)."""

    def __init__(self, qweight: torch.Tensor, wscale: torch.Tensor, bias: torch.Tensor | None = None):
        if qweight.dtype != _E4M3 or qweight.dim() != 2 or 0 in qweight.shape:
            raise ValueError("qweight must be float8_e4m3fn [N, K]")
        n, k = qweight.shape
        if wscale.shape != (_blocks(n), _blocks(k)):
            raise ValueError(f"wscale must be [{_blocks(n)}, {_blocks(k)}], got {tuple(wscale.shape)}")
        if k % 16 == 0 and qweight.is_contiguous() and qweight.data_ptr() % 16 == 0:
            self.qweight = qweight
        else:  # a checkpoint's rows, laid out once as the linear reads them
            self.qweight = _new_codes(n, k, qweight.device)
            self.qweight.copy_(qweight)
        self.wscale = wscale.float().contiguous()
        self.bias = None if bias is None else bias.float().contiguous()

    @classmethod
    def from_float(cls, weight: torch.Tensor, bias: torch.Tensor | None = None) -> "Fp8BlockLinear":
        return cls(*quantize_weight_blocks(weight), bias)

    @property
    def out_features(self) -> int:
        return self.qweight.shape[0]

    @property
    def in_features(self) -> int:
        return self.qweight.shape[1]

    def __call__(self, x: torch.Tensor, residual: torch.Tensor | None = None) -> torch.Tensor:
        if x.dtype not in _DT16 or x.shape[-1] != self.in_features:
            raise ValueError("x must be float16 or bfloat16 [..., in_features]")
        q, s = quantize_token_blocks(x.reshape(-1, x.shape[-1]))
        res = None if residual is None else residual.reshape(-1, self.out_features)
        out = linear_blocks(q, s, self.qweight, self.wscale, bias=self.bias, residual=res, out_dtype=x.dtype)
        return out.reshape(*x.shape[:-1], self.out_features)
