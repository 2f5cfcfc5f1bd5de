"""The block-scaled e4m3 kernels against the numpy oracle in 64 bits.

Tolerances. The quantisers' own fp32 steps on given values are fixed, so
tokens and weights are compared bit for bit. Behind RMSNorm and SiLU * up the
fp32 values differ from the exact ones: by VAL = 2^-18 relative (RMSNorm: an
fp32 sum of squares in chains of at most 64 additions, 64 * 2^-24 = 2^-18,
halved by the square root, and five more roundings of 2^-24; SiLU: 1 + e^-g
within 2 ulps, three more roundings); so a scale is within VAL + 2^-23, and a
code within half a step of its exact quotient plus 2 VAL of it.
Linear: every fp32 addition is off by at most 2^-23 of the running magnitude
(2^-24 if it rounds to nearest; tensor cores may truncate), 128 inside a block
and one more for each block, rank, bias and residual, so an output is within
(128 + blocks + 12) * 2^-23 of the sum of magnitudes, and then half a step of
its type. Sums that are exact in fp32 are compared bit for bit.
"""
from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import fp8 as O

pytestmark = pytest.mark.gpu

E4M3 = torch.float8_e4m3fn
F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32
VAL = 2.0 ** -18


@pytest.fixture(scope="module")
def F(cuda_device):
    from nanopointllm_b200 import fp8
    return fp8


@pytest.fixture(autouse=True)
def _status():
    yield
    from nanopointllm_b200 import _lib
    torch.cuda.synchronize()
    assert _lib.device_status() == 0


def cpu(t: torch.Tensor) -> np.ndarray:
    return t.detach().float().cpu().numpy()


def rand(shape, dtype, seed, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(*shape, generator=g) * scale
    x[..., ::37] *= 20
    return x.to(dtype)


def laid_out(t: torch.Tensor, how: str, dev) -> torch.Tensor:
    """The same values on the GPU: contiguous, with a row stride, or with rows
    that start one element off any alignment."""
    t = t.to(dev)
    if how == "contiguous":
        return t
    pad = {"strided": (0, 24), "unaligned": (1, 2)}[how]
    wide = torch.full((t.shape[0], t.shape[1] + sum(pad)), 7.0, dtype=t.dtype, device=dev)
    wide[:, pad[0]:pad[0] + t.shape[1]] = t
    return wide[:, pad[0]:pad[0] + t.shape[1]]


SHAPES = [(1, 1), (1, 128), (3, 129), (5, 100), (7, 1000), (8, 4096), (33, 520), (300, 264)]


@pytest.mark.parametrize("how", ["contiguous", "strided", "unaligned"])
@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("m,k", SHAPES)
def test_tokens(F, cuda_device, m, k, dtype, how):
    x = rand((m, k), dtype, m * 1009 + k)
    if m > 3:
        x[2] = 0
    q, s = F.quantize_token_blocks(laid_out(x, how, cuda_device))
    oq, os = O.quant_fp32(cpu(x), 1)
    assert q.dtype == E4M3 and q.shape == (m, k) and s.dtype == F32
    np.testing.assert_array_equal(cpu(s), os)
    np.testing.assert_array_equal(cpu(q), oq)


@pytest.mark.parametrize("how", ["contiguous", "unaligned"])
@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("n,k", [(1, 1), (128, 128), (129, 257), (100, 1000), (1000, 512), (64, 4096)])
def test_weight(F, cuda_device, n, k, dtype, how):
    w = rand((n, k), dtype, n * 31 + k, 0.02)
    q, s = F.quantize_weight_blocks(laid_out(w, how, cuda_device))
    oq, os = O.quant_fp32(cpu(w), 128)
    assert s.shape == (-(-n // 128), -(-k // 128))
    np.testing.assert_array_equal(cpu(s), os)
    np.testing.assert_array_equal(cpu(q), oq)


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
def test_extreme_blocks(F, cuda_device, dtype):
    """The type's largest and smallest values, zeros of both signs, and blocks
    that hold a NaN or an infinity, which alone read back as NaN."""
    big, tiny = torch.finfo(dtype).max, torch.finfo(dtype).smallest_normal
    x = rand((10, 384), dtype, 5)
    x[0, :128] = 0.0
    x[1, :128] = -0.0
    x[2, 5] = big
    x[3, :128] = tiny / 4 if dtype != F32 else tiny
    x[4, :128], x[4, 7] = 0.0, tiny
    x[5, 130] = float("nan")
    x[6, 131] = float("inf")
    x[7, 132] = float("-inf")
    x[8, 256:] = float("inf")
    x[9] = big
    q, s = (cpu(t) for t in F.quantize_token_blocks(x.to(cuda_device)))
    with np.errstate(all="ignore"):
        oq, os = O.quant_fp32(cpu(x), 1)
        vals = q * O.spread(s, 1, q.shape)
    bad = np.zeros_like(vals, dtype=bool)
    bad[5:8, 128:256] = True
    bad[8, 256:] = True
    assert np.isnan(vals[bad]).all() and np.isfinite(vals[~bad]).all()
    np.testing.assert_array_equal(q[~bad], oq[~bad])
    np.testing.assert_array_equal(s[:5], os[:5])
    w, _ = F.quantize_weight_blocks(x[:5].to(cuda_device))
    np.testing.assert_array_equal(cpu(w), O.quant_fp32(cpu(x[:5]), 128)[0])


def check_codes(q, s, v, rows=1):
    es = O.block_scales(v, rows)
    np.testing.assert_allclose(cpu(s), es, rtol=VAL + 2.0 ** -23, atol=0)
    want = v / O.spread(es, rows, v.shape)
    off = np.abs(cpu(q) - want)
    assert (off <= O.half_step_e4m3(want) + 2 * VAL * np.abs(want)).all()


@pytest.mark.parametrize("how", ["contiguous", "strided", "unaligned"])
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("residual", [False, True])
@pytest.mark.parametrize("m,k", SHAPES + [(2, 5000), (3, 11008), (2, 16384), (2, 20000), (1, 33000)])
def test_rmsnorm(F, cuda_device, m, k, residual, dtype, how):
    x, r = rand((m, k), dtype, m + k), rand((m, k), dtype, m + k + 1)
    w = (1 + 0.1 * rand((1, k), F32, k)[0]).to(dtype)
    if m > 3:
        x[1], r[1] = 0, 0
    xd = laid_out(x, how, cuda_device)
    rd = laid_out(r, how, cuda_device) if residual else None
    q, s, total = F.rmsnorm_quant_blocks(xd, w.to(cuda_device), 1e-6, rd)
    t = (x.float() + r.float()).to(dtype) if residual else x
    if residual:
        assert torch.equal(total.cpu(), t)
    else:
        assert total is None
    check_codes(q, s, O.rmsnorm(cpu(t), cpu(w), 1e-6))


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("residual", [False, True])
@pytest.mark.parametrize("k", [5120, 5121, 6656, 6657, 8191, 8192, 8193, 11264, 11265, 16385])
def test_rmsnorm_row_lengths(F, cuda_device, k, residual, dtype):
    """Both sides of each length at which the kernel's registers a thread change."""
    test_rmsnorm(F, cuda_device, 2, k, residual, dtype, "strided")


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("m,k", [(1300, 2111), (6100, 520)])
def test_rmsnorm_many_rows(F, cuda_device, m, k, dtype):
    """More rows than the SMs hold at once."""
    test_rmsnorm(F, cuda_device, m, k, True, dtype, "contiguous")


@pytest.mark.parametrize("k", [256, 4096, 20000])
def test_rmsnorm_in_place(F, cuda_device, k):
    """The sum in place of x or of the residual, rows past the batch untouched."""
    x, r = rand((6, k), BF16, 1).to(cuda_device), rand((6, k), BF16, 2).to(cuda_device)
    w = torch.ones(k, dtype=BF16, device=cuda_device)
    q0, s0, t0 = F.rmsnorm_quant_blocks(x[:4], w, 1e-6, r[:4])
    for into in (0, 1):
        a, b = x.clone(), r.clone()
        tgt = (a, b)[into][:4]
        xs, rs = (tgt, b[:4]) if into == 0 else (a[:4], tgt)
        q, s, t = F.rmsnorm_quant_blocks(xs, w, 1e-6, rs, sum_out=tgt)
        assert t is tgt and torch.equal(t, t0) and torch.equal(s, s0) and torch.equal(q.float(), q0.float())
        assert torch.equal(a[4:], x[4:]) and torch.equal(b[4:], r[4:])


@pytest.mark.parametrize("how", ["contiguous", "strided", "unaligned"])
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("m,k", SHAPES + [(3, 11008)])
def test_silu_mul(F, cuda_device, m, k, dtype, how):
    g, u = rand((m, k), dtype, m + 2 * k), rand((m, k), dtype, m + 2 * k + 1)
    q, s = F.silu_mul_quant_blocks(laid_out(g, how, cuda_device), laid_out(u, how, cuda_device))
    check_codes(q, s, O.silu_mul(cpu(g), cpu(u)))


def test_silu_far_gates(F, cuda_device):
    """Gates whose e^-g overflows or vanishes in fp32, and infinite ones."""
    g = torch.tensor([-3e4, -120.0, -89.0, -88.0, -20.0, 0.0, 20.0, 89.0, 3e4], dtype=F16)
    g = g.repeat(15)[:128].reshape(1, 128)
    u = rand((1, 128), F16, 3)
    q, s = F.silu_mul_quant_blocks(g.to(cuda_device), u.to(cuda_device))
    check_codes(q, s, O.silu_mul(cpu(g), cpu(u)))
    g = torch.zeros(1, 256, dtype=F16)
    g[0, 3], g[0, 200] = float("-inf"), 1.0
    q, s = F.silu_mul_quant_blocks(g.to(cuda_device), torch.ones(1, 256, dtype=F16, device=cuda_device))
    vals = cpu(q) * np.repeat(cpu(s), 128, 1)
    assert np.isnan(vals[0, :128]).all() and np.isfinite(vals[0, 128:]).all()


def test_guarded_outputs(F, cuda_device):
    """The C entries write their rows and columns and nothing around them."""
    from nanopointllm_b200 import _lib as L
    m, k, ld = 5, 300, 320
    x = rand((m, k), F16, 9).to(cuda_device)
    w = torch.ones(k, dtype=F16, device=cuda_device)
    st = L.stream_ptr(cuda_device)

    def guarded(call):
        q = torch.full((m + 2, ld), 0x55, dtype=torch.uint8, device=cuda_device)
        s = torch.full((m + 2, 5), 3.25, device=cuda_device)
        L.check(call(q[1:], s[1:]))
        torch.cuda.synchronize()
        inner = torch.zeros_like(q, dtype=torch.bool)
        inner[1:m + 1, :k] = True
        assert (q[~inner] == 0x55).all()
        return q[1:m + 1, :k].view(E4M3), s

    q, s = guarded(lambda q, s: L.lib.npl_fp8_quant_rows(x.data_ptr(), L.NPL_F16, m, k, k, q.data_ptr(), ld,
                                                         s.data_ptr(), 5, st))
    assert (s[0] == 3.25).all() and (s[m + 1] == 3.25).all() and (s[1:m + 1, 3:] == 3.25).all()
    np.testing.assert_array_equal(cpu(q), O.quant_fp32(cpu(x), 1)[0])
    guarded(lambda q, s: L.lib.npl_fp8_silu_mul_quant(x.data_ptr(), k, x.data_ptr(), k, L.NPL_F16, m, k, q.data_ptr(),
                                                      ld, s.data_ptr(), 5, st))
    guarded(lambda q, s: L.lib.npl_fp8_rmsnorm_quant(x.data_ptr(), k, None, 0, w.data_ptr(), L.NPL_F16, 1e-6, m, k,
                                                     None, 0, q.data_ptr(), ld, s.data_ptr(), 5, st))
    q, s = guarded(lambda q, s: L.lib.npl_fp8_quant_weight(x.data_ptr(), L.NPL_F16, m, k, k, q.data_ptr(), ld,
                                                           s.data_ptr(), 5, st))
    assert (s[2:] == 3.25).all() and (s[1, 3:] == 3.25).all()


# ------------------------------------------------------------------- linear
def codes(rows, k, seed, dev, top=4):
    """Random small whole codes, rows on 16-byte boundaries."""
    g = torch.Generator().manual_seed(seed)
    v = torch.randint(-top, top + 1, (rows, k), generator=g).float()
    store = torch.zeros(rows, -(-k // 16) * 16, dtype=E4M3, device=dev)
    store[:, :k] = v.to(dev).to(E4M3)
    return store[:, :k]


def powers(rows, cols, seed, dev, lo=-2, hi=1):
    g = torch.Generator().manual_seed(seed)
    return (2.0 ** torch.randint(lo, hi, (rows, cols), generator=g).float()).to(dev)


LINEAR_SHAPES = [
    (1, 1, 1), (1, 8, 16), (2, 128, 128), (8, 1000, 512), (1, 4096, 1408), (16, 100, 77), (17, 129, 129),
    (33, 300, 640), (64, 1003, 500), (65, 257, 384), (128, 128, 256), (129, 513, 1000), (200, 640, 4096),
    (300, 264, 132), (513, 520, 896), (1000, 1001, 272), (2100, 700, 300),
]


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("m,n,k", LINEAR_SHAPES)
def test_linear_exact_sums(F, cuda_device, m, n, k, dtype):
    """Whole codes under power-of-two scales: every partial sum is exact in
    fp32 (terms are multiples of 2^-4 and sum to at most 16 K < 2^17), so the
    result is the exact sum rounded once, whatever the order."""
    kb, nb = -(-k // 128), -(-n // 128)
    qa, qw = codes(m, k, 1, cuda_device), codes(n, k, 2, cuda_device)
    sa, sw = powers(m, kb, 3, cuda_device), powers(nb, kb, 4, cuda_device)
    bias = torch.randint(-3, 4, (n,), generator=torch.Generator().manual_seed(5)).float()
    res = torch.randint(-9, 10, (m, n), generator=torch.Generator().manual_seed(6)).to(dtype)
    for b, r in ((None, None), (bias, None), (bias, res)):
        out = F.linear_blocks(qa, sa, qw, sw, bias=None if b is None else b.to(cuda_device),
                              residual=None if r is None else r.to(cuda_device), out_dtype=dtype)
        want, _ = O.linear(cpu(qa), cpu(sa), cpu(qw), cpu(sw), None if b is None else b.numpy(),
                           None if r is None else cpu(r))
        assert out.shape == (m, n) and out.dtype == dtype
        assert torch.equal(out.cpu(), torch.from_numpy(want).to(dtype))


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("m,n,k", [(1, 4096, 4096), (8, 12288, 4096), (40, 1000, 11008), (200, 1100, 4100),
                                   (560, 2000, 1000), (1500, 1300, 2048)])
def test_linear_random(F, cuda_device, m, n, k, dtype):
    x = rand((m, k), F32, m + n).to(cuda_device)
    w = rand((n, k), F32, n + k, 0.02).to(cuda_device)
    qa, sa = F.quantize_token_blocks(x)
    qw, sw = F.quantize_weight_blocks(w)
    res = rand((m, n), dtype, 8).to(cuda_device)
    bias = rand((1, n), F32, 9)[0].to(cuda_device)
    out = cpu(F.linear_blocks(qa, sa, qw, sw, bias=bias, residual=res))
    want, mag = O.linear(cpu(qa), cpu(sa), cpu(qw), cpu(sw), cpu(bias), cpu(res))
    tol = (128 + -(-k // 128) + 12) * 2.0 ** -23 * mag
    half = torch.finfo(dtype).eps / 2
    assert (np.abs(out - want) <= tol + half * (np.abs(want) + tol)).all()


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("m,n,k", [
    (150, 190, 200), (300, 193, 300), (260, 385, 130), (257, 4000, 260), (800, 4093, 300), (800, 4096, 300),
    (1025, 3900, 140), (140, 200, 3071), (300, 700, 2944), (300, 700, 2945), (129, 8448, 3200), (129, 8449, 3200),
    (200, 9472, 3200), (100, 300, 2432), (100, 300, 2433), (128, 5504, 2500), (65, 5505, 2500)])
def test_linear_tile_choices(F, cuda_device, m, n, k, dtype):
    """Tiles of 192 and 256 weight rows in one round or two, ragged or not, and
    tiles shared by two pairs of CTAs, up to more than fit on the device at
    once; 65 to 128 tokens in decode tiles or not. The sums are exact (K <= 2^13, as test_linear_exact_sums)."""
    test_linear_exact_sums(F, cuda_device, m, n, k, dtype)


def test_linear_layouts(F, cuda_device):
    """Strided scales, residual and output; the residual in place; columns and
    rows around the output untouched; odd output strides."""
    for m, n, k in ((5, 200, 300), (70, 200, 300), (300, 328, 640)):
        kb, nb = -(-k // 128), -(-n // 128)
        qa, qw = codes(m, k, 1, cuda_device), codes(n, k, 2, cuda_device)
        sa, sw = powers(m, kb, 3, cuda_device), powers(nb, kb, 4, cuda_device)
        res = torch.randint(-9, 10, (m, n), generator=torch.Generator().manual_seed(6)).to(F16).to(cuda_device)
        want = F.linear_blocks(qa, sa, qw, sw, residual=res)
        wide = torch.zeros(m, kb + 3, device=cuda_device)
        wide[:, 1:kb + 1] = sa
        turned = sw.t().contiguous().t()
        for off, pad in ((0, 8), (1, 1), (3, 2), (8, 0)):
            r = torch.full((m + 2, off + n + pad), 5.0, dtype=F16, device=cuda_device)
            r[1:m + 1, off:off + n] = res
            o = torch.full((m + 2, off + n + pad), -77.0, dtype=F16, device=cuda_device)
            inner = torch.zeros_like(o, dtype=torch.bool)
            inner[1:m + 1, off:off + n] = True
            view, rv = o[1:m + 1, off:off + n], r[1:m + 1, off:off + n]
            got = F.linear_blocks(qa, wide[:, 1:kb + 1], qw, turned, residual=rv, out=view)
            assert got is view and torch.equal(view, want) and (o[~inner] == -77.0).all()
            F.linear_blocks(qa, sa, qw, sw, residual=rv, out=rv)  # in place
            assert torch.equal(rv, want) and (r[~inner] == 5.0).all()


@pytest.mark.parametrize("m", [3, 70, 300])
def test_linear_bad_token_stays_in_its_row(F, cuda_device, m):
    x = rand((m, 512), F16, 1).to(cuda_device)
    x[1, 200] = float("inf")
    w = rand((300, 512), F16, 2, 0.02).to(cuda_device)
    out = F.linear_blocks(*F.quantize_token_blocks(x), *F.quantize_weight_blocks(w), out_dtype=F16)
    assert out[1].isnan().all() and out[0].isfinite().all() and out[2:].isfinite().all()


@pytest.mark.parametrize("m", [1, 8, 64, 65, 300])
def test_linear_repeats_bit_for_bit(F, cuda_device, m):
    qa, sa = F.quantize_token_blocks(rand((m, 4096), F16, 1).to(cuda_device))
    qw, sw = F.quantize_weight_blocks(rand((1000, 4096), F16, 2, 0.02).to(cuda_device))
    first = F.linear_blocks(qa, sa, qw, sw)
    for _ in range(20):
        assert torch.equal(F.linear_blocks(qa, sa, qw, sw), first)


def test_no_rows(F, cuda_device):
    x = torch.zeros(0, 256, dtype=F16, device=cuda_device)
    q, s = F.quantize_token_blocks(x)
    w = torch.ones(256, dtype=F16, device=cuda_device)
    assert F.rmsnorm_quant_blocks(x, w, 1e-6, x)[2].shape == (0, 256)
    assert F.silu_mul_quant_blocks(x, x)[1].shape == (0, 2)
    qw, sw = F.quantize_weight_blocks(torch.ones(100, 256, dtype=F16, device=cuda_device))
    assert F.linear_blocks(q, s, qw, sw).shape == (0, 100)


# ------------------------------------------------------------ used together
def mlp_weights(F, dev, hidden, inter, dtype):
    gu = rand((2 * inter, hidden), dtype, 11, 0.02).to(dev)
    dn = rand((hidden, inter), dtype, 12, 0.02).to(dev)
    nw = (1 + 0.1 * rand((1, hidden), F32, 13)[0]).to(dtype).to(dev)
    return F.quantize_weight_blocks(gu), F.quantize_weight_blocks(dn), nw


def mlp(F, h, delta, nw, gu, dn, inter):
    """A decoder layer's MLP: the residual's addition and norm, packed gate/up,
    SiLU * up, down with the residual."""
    q, s, h = F.rmsnorm_quant_blocks(h, nw, 1e-6, delta)
    y = F.linear_blocks(q, s, *gu, out_dtype=h.dtype)
    a, sa = F.silu_mul_quant_blocks(y[:, :inter], y[:, inter:])
    return F.linear_blocks(a, sa, *dn, residual=h), (q, s, h, y, a, sa)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("m,hidden,inter", [(1, 512, 1024), (8, 4096, 1100), (65, 500, 1000), (300, 512, 1376)])
def test_mlp_block(F, cuda_device, m, hidden, inter, dtype):
    """The operators of an MLP in a row, each checked in 64 bits on what the
    one before it gave."""
    gu, dn, nw = mlp_weights(F, cuda_device, hidden, inter, dtype)
    h, delta = (rand((m, hidden), dtype, i).to(cuda_device) for i in (1, 2))
    out, (q, s, total, y, a, sa) = mlp(F, h, delta, nw, gu, dn, inter)
    half = torch.finfo(dtype).eps / 2
    check_codes(q, s, O.rmsnorm(cpu(total), cpu(nw), 1e-6))
    for got, (codes_, scale), w, res in ((y, (q, s), gu, None), (out, (a, sa), dn, cpu(total))):
        want, mag = O.linear(cpu(codes_), cpu(scale), cpu(w[0]), cpu(w[1]), None, res)
        tol = (128 + scale.shape[1] + 12) * 2.0 ** -23 * mag
        assert (np.abs(cpu(got) - want) <= tol + half * (np.abs(want) + tol)).all()
    check_codes(a, sa, O.silu_mul(cpu(y[:, :inter]), cpu(y[:, inter:])))


def test_block_linear_module(F, cuda_device):
    w = rand((300, 500), F16, 1, 0.02).to(cuda_device)
    x = rand((6, 500), F16, 2).to(cuda_device).reshape(2, 3, 500)
    lin = F.Fp8BlockLinear.from_float(w, torch.ones(300, device=cuda_device))
    out = lin(x)
    q, s = F.quantize_token_blocks(x.reshape(6, 500))
    want = F.linear_blocks(q, s, *F.quantize_weight_blocks(w), bias=torch.ones(300, device=cuda_device), out_dtype=F16)
    assert out.shape == (2, 3, 300) and torch.equal(out.reshape(6, 300), want)
    assert torch.equal(lin(x, residual=out).reshape(6, 300),
                       F.linear_blocks(q, s, lin.qweight, lin.wscale, bias=lin.bias, residual=want))


@pytest.mark.parametrize("m", [4, 100])
def test_graphs_and_streams(F, cuda_device, m):
    """The same chain captured twice, replayed by turns and at once on two
    streams, on new inputs, gives what the eager calls give."""
    hidden, inter = 1024, 1408
    gu, dn, nw = mlp_weights(F, cuda_device, hidden, inter, F16)
    ins, outs, graphs, streams = [], [], [], []
    for i in range(2):
        h, d = (rand((m, hidden), F16, 20 + 2 * i + j).to(cuda_device) for j in (0, 1))
        st = torch.cuda.Stream()
        st.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(st):
            mlp(F, h, d, nw, gu, dn, inter)
        torch.cuda.current_stream().wait_stream(st)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out, _ = mlp(F, h, d, nw, gu, dn, inter)
        ins.append((h, d)), outs.append(out), graphs.append(g), streams.append(st)
    for turn in range(3):
        for i in range(2):
            for j in range(2):
                ins[i][j].copy_(rand((m, hidden), F16, 100 * turn + 10 * i + j).to(cuda_device))
        want = [mlp(F, *ins[i], nw, gu, dn, inter)[0].clone() for i in range(2)]
        torch.cuda.synchronize()
        for _ in range(5):
            for i in range(2):
                with torch.cuda.stream(streams[i]):
                    graphs[i].replay()
        torch.cuda.synchronize()
        for i in range(2):
            assert torch.equal(outs[i], want[i])


def test_weight_written_just_before(F, cuda_device):
    """A weight quantised right before the product that reads it."""
    qa, sa = F.quantize_token_blocks(rand((8, 2048), F16, 1).to(cuda_device))
    ws = [rand((4096, 2048), F16, 2 + i, 0.02).to(cuda_device) for i in range(6)]
    want = []
    for w in ws:
        qw, sw = F.quantize_weight_blocks(w)
        torch.cuda.synchronize()
        want.append(F.linear_blocks(qa, sa, qw, sw))
    torch.cuda.synchronize()
    got = [F.linear_blocks(qa, sa, *F.quantize_weight_blocks(w)) for w in ws]
    for g, e in zip(got, want):
        assert torch.equal(g, e)


def test_calls_at_once_on_streams(F, cuda_device):
    """Decode and prefill tiles, split and whole, quantisers and the int8
    linear on four streams at once: nothing is shared between calls."""
    from nanopointllm_b200 import w8a8 as W
    x = rand((300, 2048), F16, 1).to(cuda_device)
    q, s = F.quantize_token_blocks(x)
    weights = [F.quantize_weight_blocks(rand((n, 2048), F16, n, 0.02).to(cuda_device)) for n in (1000, 4096)]
    i8 = W.dynamic_per_token_quant(x[:40])
    i8w = W.per_output_weight_quant(rand((1024, 2048), F16, 5, 0.02).to(cuda_device))
    work = [
        lambda: F.linear_blocks(q[:8], s[:8], *weights[0]),     # decode tiles, split
        lambda: F.linear_blocks(q[:64], s[:64], *weights[1]),   # 64-token tiles, split
        lambda: F.linear_blocks(q, s, *weights[0]),             # prefill tiles, two pairs each
        lambda: F.quantize_token_blocks(x)[1],
        lambda: F.linear_blocks(q, s, *weights[1], out_dtype=F16),
        lambda: W.linear_q(i8[0], i8[1].reshape(-1), *i8w),
    ]
    want = [f().clone() for f in work]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(4)]
    got = []
    for turn in range(25):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                # the int8 linear has one workspace, so one stream
                j = (turn + i) % 5 if i else (5 if turn % 2 else 0)
                got.append((j, work[j]()))
    torch.cuda.synchronize()
    for j, g in got:
        assert torch.equal(g, want[j]), j


def test_far_rows(F, cuda_device):
    """Offsets past 2^31 elements: the last rows of large operands. The linear
    is held to the 64-bit sums and not to the bits of a call on these rows
    alone: 200 rows make two tiles, whose 64 blocks two pairs of CTAs share, so
    s0 + .. + s63 is there (s0 + .. + s31) + (s32 + .. + s63), another order of
    fp32 additions than that of 270000 rows."""
    m, k = 270000, 8192
    x = torch.zeros(m, k, dtype=F16, device=cuda_device)
    x[-200:] = rand((200, k), F16, 1).to(cuda_device)
    q, s = F.quantize_token_blocks(x)
    q1, s1 = F.quantize_token_blocks(x[-200:].clone())
    assert torch.equal(q[-200:].view(torch.uint8), q1.view(torch.uint8)) and torch.equal(s[-200:], s1)
    w = F.quantize_weight_blocks(rand((136, k), F16, 2, 0.02).to(cuda_device))
    for out in (F.linear_blocks(q, s, *w)[-200:], F.linear_blocks(q1, s1, *w)):
        want, mag = O.linear(cpu(q1), cpu(s1), cpu(w[0]), cpu(w[1]))
        tol = (128 + 64 + 12) * 2.0 ** -23 * mag
        assert (np.abs(cpu(out) - want) <= tol + torch.finfo(BF16).eps / 2 * (np.abs(want) + tol)).all()
    nw = torch.ones(k, dtype=F16, device=cuda_device)
    assert torch.equal(F.rmsnorm_quant_blocks(x, nw, 1e-6)[1][-200:], F.rmsnorm_quant_blocks(x[-200:], nw, 1e-6)[1])
    del x, q
    n = 32776
    q, s = F.quantize_token_blocks(rand((66000, 128), F16, 3).to(cuda_device))
    w = F.quantize_weight_blocks(rand((n, 128), F16, 4, 0.02).to(cuda_device))
    out = F.linear_blocks(q, s, *w)
    assert torch.equal(out[-300:], F.linear_blocks(q[-300:], s[-300:], *w))


@pytest.mark.parametrize("m", [1, 100, 300])
def test_operands_of_two_devices_are_refused(F, cuda_device, m):
    x = rand((m, 256), F16, 1).to(cuda_device)
    w = F.quantize_weight_blocks(rand((64, 256), F16, 2).to(cuda_device))
    q, s = F.quantize_token_blocks(x)
    with pytest.raises(ValueError, match="device"):
        F.linear_blocks(q, s.cpu(), *w)
    with pytest.raises(ValueError, match="device"):
        F.rmsnorm_quant_blocks(x, torch.ones(256, dtype=F16), 1e-6)


# ------------------------------------------------------------- far SiLU gates
@pytest.mark.parametrize("how", ["contiguous", "unaligned"])
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("lo,hi", [(-88.5, -87.4), (-89.0, -85.0), (-104.0, -88.8), (-170.0, -110.0), (-210.0, -165.0)])
def test_silu_blocks_of_far_gates(F, cuda_device, lo, hi, dtype, how):
    """Blocks whose gates are all far below 0, so that e^-g leaves fp32's
    normal range, under ups of any size. VAL, and 2^-13 in units of a code for
    p = e^(g / 2) once it is subnormal: 2^-149 |g| p up / scale with |g| < 2^8, p < 2^-126,
    up < 2^128 and scale >= 2^-126."""
    m, k = 6, 300
    gen = torch.Generator().manual_seed(int(-lo * 8))
    g = (lo + (hi - lo) * torch.rand(m, k, generator=gen)).to(dtype)
    u = torch.rand(m, k, generator=gen) * 0.5 + 0.25
    big = float(torch.finfo(dtype).max)
    u = (u * torch.tensor([big, big / 1e3, 3e4, 1.0, -big, 1e-3]).double()[:, None]).to(dtype)
    q, s = F.silu_mul_quant_blocks(laid_out(g, how, cuda_device), laid_out(u, how, cuda_device))
    v = O.silu_mul(cpu(g), cpu(u))
    es = O.block_scales(v, 1)
    np.testing.assert_allclose(cpu(s), es, rtol=VAL + 2.0 ** -23, atol=0)
    want = v / O.spread(es, 1, v.shape)
    off = np.abs(cpu(q) - want)
    assert (off <= O.half_step_e4m3(want) + 2 * VAL * np.abs(want) + 2.0 ** -13).all()


def test_silu_far_gates_beside_others(F, cuda_device):
    """A far gate changes no other value of its block, and an infinite or NaN
    one makes its block NaN."""
    u = rand((3, 256), BF16, 3)
    g = rand((3, 256), BF16, 4)
    plain = [cpu(t) for t in F.silu_mul_quant_blocks(g.to(cuda_device), u.to(cuda_device))]
    g[:, 5], g[:, 133] = -100.0, -300.0
    q, s = (cpu(t) for t in F.silu_mul_quant_blocks(g.to(cuda_device), u.to(cuda_device)))
    keep = np.ones(256, bool)
    keep[[5, 133]] = False
    old = np.abs(O.silu_mul(cpu(g), cpu(u))).reshape(3, 2, 128).argmax(2)
    assert not (old == 5).any()
    np.testing.assert_array_equal(s, plain[1])
    np.testing.assert_array_equal(q[:, keep], plain[0][:, keep])
    assert (q[:, ~keep] == 0).all()
    g[0, 6], g[1, 140] = float("-inf"), float("nan")
    q, s = (cpu(t) for t in F.silu_mul_quant_blocks(g.to(cuda_device), u.to(cuda_device)))
    vals = q * O.spread(s, 1, q.shape)
    bad = np.zeros((3, 256), bool)
    bad[0, :128] = bad[1, 128:] = True
    assert np.isnan(vals[bad]).all() and np.isfinite(vals[~bad]).all()


# ------------------------------------------------- products of far apart scales
@pytest.mark.parametrize("m", [5, 40, 100, 300])
def test_linear_products_of_tiny_scales(F, cuda_device, m):
    """Scales whose product is subnormal: it is off by 2^-150 at most, and a
    block's sum here at most 128 * 4 * 4 = 2^11 (128 * 448^2 < 2^25 in general),
    which is 2^-139 a block, beside the linear's own bound and half a step of bf16 (2^-134
    below its smallest normal number)."""
    n, k = 300, 640
    kb, nb = -(-k // 128), -(-n // 128)
    gen = torch.Generator().manual_seed(m)
    qa, qw = codes(m, k, 1, cuda_device), codes(n, k, 2, cuda_device)
    sa = (2.0 ** -70 * (1 + torch.rand(m, kb, generator=gen))).to(cuda_device)
    sw = (2.0 ** -66 * (1 + torch.rand(nb, kb, generator=gen))).to(cuda_device)
    sa[1], sw[1] = 2.0 ** -126, 2.0 ** -126  # blocks of zeros would have these; their product is 0
    out = cpu(F.linear_blocks(qa, sa, qw, sw, out_dtype=BF16))
    want, mag = O.linear(cpu(qa), cpu(sa), cpu(qw), cpu(sw))
    tol = (128 + kb + 12) * 2.0 ** -23 * mag + kb * 2.0 ** -139
    half = np.maximum(torch.finfo(BF16).eps / 2 * (np.abs(want) + tol), 2.0 ** -134)
    assert np.abs(want).max() > 2.0 ** -130 and (np.abs(out - want) <= tol + half).all()


@pytest.mark.parametrize("m", [5, 40, 100, 300])
def test_linear_products_of_huge_scales(F, cuda_device, m):
    """Scales whose product overflows make their token infinite or NaN in those
    128 columns, and nothing else."""
    n, k = 300, 640
    qa, qw = codes(m, k, 1, cuda_device), codes(n, k, 2, cuda_device)
    sa, sw = powers(m, 5, 3, cuda_device), powers(3, 5, 4, cuda_device)
    plain = F.linear_blocks(qa, sa, qw, sw)
    sa2, sw2 = sa.clone(), sw.clone()
    sa2[2, 1], sw2[1, 1] = 2.0 ** 70, 2.0 ** 70
    with_far = F.linear_blocks(qa, sa2, qw, sw2)
    assert not with_far[2, 128:256].isfinite().any()
    # the other tokens and columns by the oracle, whose terms stay finite
    want, mag = O.linear(cpu(qa), cpu(sa2), cpu(qw), cpu(sw2))
    tol = (128 + 5 + 12) * 2.0 ** -23 * mag
    ok = np.ones((m, n), bool)
    ok[2, 128:256] = False
    got = cpu(with_far)
    assert (np.abs(got - want) <= tol + torch.finfo(BF16).eps / 2 * (np.abs(want) + tol))[ok].all()
    rest = torch.ones(m, n, dtype=torch.bool)
    rest[2], rest[:, 128:256] = False, False
    assert torch.equal(with_far.cpu()[rest], plain.cpu()[rest])


# ------------------------------------ the paths that layers of real sizes take
# (M, N, K) -> (kernel, tokens or weight rows of a tile, CTAs or pairs that share one, blocks of each
# at most, tiles of a cluster at most); test_fp8_cpu.py holds these to the rules of the host code.
LINEAR_PATHS = {
    (8, 12288, 5000): ("decode", 16, 1, 40, 1),
    (24, 12291, 5000): ("decode", 32, 1, 40, 1),
    (50, 12288, 5000): ("decode", 64, 1, 40, 1),
    (3, 11137, 8300): ("decode", 16, 1, 65, 1),
    (8, 1000, 33000): ("decode", 16, 8, 33, 1),
    (100, 1003, 33000): ("decode", 64, 8, 33, 1),
    (800, 4096, 2300): ("prefill", 256, 1, 18, 1),
    (300, 14400, 2300): ("prefill", 256, 1, 18, 2),
    (150, 28501, 1300): ("prefill", 256, 1, 11, 2),
    (2100, 2100, 2300): ("prefill", 192, 1, 18, 2),
    (4200, 2101, 1300): ("prefill", 192, 1, 11, 3),
    (200, 1000, 8000): ("prefill", 256, 2, 32, 1),
}


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("m,n,k", LINEAR_PATHS)
def test_linear_long_sums(F, cuda_device, m, n, k, dtype):
    """More blocks than a CTA holds scales or ring stages for, and several tiles
    a cluster. Sums are exact: multiples of 2^-4 up to 16 K < 2^20."""
    test_linear_exact_sums(F, cuda_device, m, n, k, dtype)


def compare_with_bad_blocks(F, x, rows, call, dev, how):
    """Codes and scales bit for bit, a NaN and an infinite block apart, which read back as NaN."""
    q, s = (cpu(t) for t in call(laid_out(x, how, dev)))
    with np.errstate(all="ignore"):
        oq, os = O.quant_fp32(cpu(x), rows)
        vals = q * O.spread(s, rows, q.shape)
    bad_scale = ~np.isfinite(os)
    assert bad_scale.sum() == 2
    bad = O.spread(bad_scale.astype(np.float64), rows, q.shape) > 0
    assert np.isnan(vals[bad]).all()
    np.testing.assert_array_equal(s[~bad_scale], os[~bad_scale])
    np.testing.assert_array_equal(q[~bad], oq[~bad])


@pytest.mark.parametrize("how", ["contiguous", "unaligned"])
@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("n,k", [(4000, 2100), (8200, 1100), (20000, 1099)])
def test_weight_of_many_blocks(F, cuda_device, n, k, dtype, how):
    """More blocks than CTAs: each takes several, one after the other."""
    w = rand((n, k), dtype, n + k, 0.02)
    w[700, 300], w[n - 1, k - 1] = float("nan"), float("inf")
    compare_with_bad_blocks(F, w, 128, F.quantize_weight_blocks, cuda_device, how)


@pytest.mark.parametrize("how", ["contiguous", "strided", "unaligned"])
@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("m,k", [(3000, 1000), (1200, 2111), (2400, 1024), (4000, 513)])
def test_tokens_two_blocks_a_thread(F, cuda_device, m, k, dtype, how):
    """More than 128 blocks an SM: a thread takes two blocks of a row, four apart."""
    assert m * -(-k // 128) > 128 * 148
    x = rand((m, k), dtype, m + k)
    x[1] = 0
    x[7, 130], x[m - 1, k - 1] = float("nan"), float("-inf")
    compare_with_bad_blocks(F, x, 1, F.quantize_token_blocks, cuda_device, how)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("residual", [False, True])
@pytest.mark.parametrize("m,k", [(3, 40001), (2, 200000)])
def test_rmsnorm_of_long_rows(F, cuda_device, m, k, residual, dtype):
    """Rows that are read twice. A thread adds 16 squares in each of ceil(K /
    8192) steps and the sums are joined in 10 more: so many roundings of 2^-24,
    halved by the square root. The quotient and rsqrtf are within 2 ulps, 4
    roundings each, the former halved too; with eps and two products 8.5 more."""
    x, r = rand((m, k), dtype, m + k), rand((m, k), dtype, m + k + 1)
    w = (1 + 0.1 * rand((1, k), F32, k)[0]).to(dtype)
    q, s, total = F.rmsnorm_quant_blocks(x.to(cuda_device), w.to(cuda_device), 1e-6,
                                         r.to(cuda_device) if residual else None)
    t = (x.float() + r.float()).to(dtype) if residual else x
    if residual:
        assert torch.equal(total.cpu(), t)
    off = ((16 * -(-k // 8192) + 10) / 2 + 8.5) * 2.0 ** -24
    v = O.rmsnorm(cpu(t), cpu(w), 1e-6)
    es = O.block_scales(v, 1)
    np.testing.assert_allclose(cpu(s), es, rtol=off + 2.0 ** -23, atol=0)
    want = v / O.spread(es, 1, v.shape)
    assert (np.abs(cpu(q) - want) <= O.half_step_e4m3(want) + 2 * off * np.abs(want)).all()


def test_rmsnorm_of_squares_that_overflow(F, cuda_device):
    """Rows whose sum of squares is past fp32 read back as zeros, rows just
    below it as their norm."""
    x = rand((4, 512), BF16, 1)
    x[1] = (x[1].float() * 2.0 ** 70).to(BF16)
    x[2] = (x[2].float().clamp(-4, 4) * 2.0 ** 50).to(BF16)
    w = torch.ones(512, dtype=BF16)
    q, s, _ = F.rmsnorm_quant_blocks(x.to(cuda_device), w.to(cuda_device), 1e-6)
    assert (cpu(q)[1] == 0).all() and (cpu(s)[1] == 2.0 ** -126).all()
    keep = [0, 2, 3]
    check_codes(q[keep], s[keep], O.rmsnorm(cpu(x)[keep], cpu(w), 1e-6))
