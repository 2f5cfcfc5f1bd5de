"""Host side of tree attention, window attention and token log probabilities,
without a GPU: the refusals of the C entries and of the Python calls, what the
calls hand to the C entries, the tree's mask, and the oracles."""
from __future__ import annotations

import ctypes

import numpy as np
import pytest
import torch

from oracle import logprobs as OL
from oracle import masked_attention as OM

F16, BF16, F32, I32 = torch.float16, torch.bfloat16, torch.float32, torch.int32


@pytest.fixture(scope="module")
def L():
    from nanopointllm_b200 import _lib
    return _lib


@pytest.fixture
def PA(monkeypatch):
    """paged_attention on CPU tensors: the device check is off and the C call is
    written down instead of made."""
    from nanopointllm_b200 import paged_attention
    calls = []
    monkeypatch.setattr(paged_attention, "_same_device", lambda *a: None)
    monkeypatch.setattr(paged_attention, "_call", lambda fn, device, *args: calls.append((fn.__name__, args)))
    return paged_attention, calls


@pytest.fixture
def LP(monkeypatch):
    from nanopointllm_b200 import logprobs
    calls = []
    monkeypatch.setattr(logprobs, "_same_device", lambda *a: None)
    monkeypatch.setattr(logprobs, "_call", lambda fn, device, *args: calls.append((fn.__name__, args)))
    return logprobs, calls


def _buf(n=1 << 16):
    b = ctypes.create_string_buffer(n + 16)
    at = ctypes.addressof(b)
    return b, at + (-at) % 16


def test_c_entries_refuse_bad_arguments(L):
    keep, p = _buf()
    good = dict(q=p, dtype=1, ld_q=1024, total_q=4, H=8, Hkv=2, D=128, k=p, v=p, nb=10, bs=16, bt=p, bt_stride=5,
                max_blocks=5, ctx=p, lens=p, offs=p, B=2, most=2)
    tree_tail = dict(mask=p, ld_mask=4, cols=4, scale=0.1, out=p, ld_out=1024, stream=None)
    window_tail = dict(window=8, sinks=1, scale=0.1, out=p, ld_out=1024, stream=None)
    shared = [dict(q=None), dict(k=None), dict(v=None), dict(bt=None), dict(ctx=None), dict(out=None),
              dict(dtype=0), dict(dtype=7), dict(lens=None), dict(offs=None), dict(total_q=-1), dict(B=-1),
              dict(most=-1), dict(H=0), dict(Hkv=0), dict(Hkv=3), dict(nb=0), dict(bs=0), dict(max_blocks=0),
              dict(bt_stride=4), dict(ld_q=1023), dict(ld_q=1016), dict(ld_out=1016), dict(ld_out=1028),
              dict(scale=0.0), dict(scale=-1.0), dict(scale=float("nan")), dict(scale=float("inf")),
              dict(q=p + 2), dict(k=p + 8), dict(v=p + 4), dict(out=p + 2)]
    unsupported = [dict(D=80), dict(bs=12), dict(bs=7), dict(H=258, ld_q=1 << 16, ld_out=1 << 16),
                   dict(nb=1 << 27, bs=16), dict(max_blocks=1 << 27, bt_stride=1 << 27), dict(B=65536)]

    def tree(**kw):
        return L.lib.npl_paged_tree_attention(*{**good, **tree_tail, **kw}.values())

    def window(**kw):
        return L.lib.npl_paged_window_attention(*{**good, **window_tail, **kw}.values())

    for kw in shared:
        assert tree(**kw) == L.NPL_ERR_ARG, kw
        assert window(**kw) == L.NPL_ERR_ARG, kw
    for kw in unsupported:
        assert tree(**kw) == L.NPL_ERR_UNSUPPORTED, kw
        assert window(**kw) == L.NPL_ERR_UNSUPPORTED, kw
    for kw in (dict(mask=None), dict(lens=None, offs=None, total_q=2), dict(cols=1), dict(ld_mask=3)):
        assert tree(**kw) == L.NPL_ERR_ARG, kw
    for kw in (dict(window=0), dict(window=-3), dict(sinks=-1), dict(lens=None, offs=None)):
        assert window(**kw) == L.NPL_ERR_ARG, kw
    f = L.lib.npl_token_logprobs
    ok = dict(logits=p, dtype=0, ld=100, rows=2, vocab=100, ids=p, top=5, lp=p, ent=p, top_ids=p, top_lp=p, stream=None)
    for kw in (dict(dtype=3), dict(rows=-1), dict(vocab=0), dict(vocab=1 << 31, ld=1 << 31), dict(ld=99),
               dict(top=-1), dict(top=33), dict(vocab=4, ld=4), dict(logits=None), dict(ids=None), dict(lp=None),
               dict(ent=None), dict(top_ids=None), dict(top_lp=None), dict(logits=p + 2), dict(ids=p + 4),
               dict(lp=p + 2), dict(top_ids=p + 4)):
        assert f(*{**ok, **kw}.values()) == L.NPL_ERR_ARG, kw
    assert f(*{**ok, "dtype": 1, "logits": p + 1}.values()) == L.NPL_ERR_ARG


def _case(T=6, H=4, Hkv=2, D=64, B=2, dtype=F16):
    q = torch.zeros(T, H, D, dtype=dtype)
    k, v = torch.zeros(2, 7, 16, Hkv, D, dtype=dtype).unbind(0)
    i = torch.zeros(B, dtype=I32)
    return dict(q=q, k_cache=k, v_cache=v, block_tables=torch.zeros(B, 3, dtype=I32), context_lens=i, q_lens=i + 3,
                q_offsets=i, scale=0.125, num_kv_groups=H // Hkv)


def test_refusals_of_the_python_calls(PA):
    pa, calls = PA
    mask = torch.ones(6, 3, dtype=torch.bool)
    bad = [
        (dict(q=torch.zeros(6, 4, 64)), "float16 or bfloat16"),
        (dict(q=torch.zeros(6, 256, dtype=F16)), r"\[total_q, H, D\]"),
        (dict(k_cache=torch.zeros(7, 16, 2, 64, dtype=BF16)), "type of q"),
        (dict(v_cache=torch.zeros(7, 16, 1, 64, dtype=F16)), "num_blocks"),
        (dict(k_cache=torch.zeros(7, 16, 2, 128, dtype=F16)[..., :64]), "contiguous"),
        (dict(num_kv_groups=1), "geometry"),
        (dict(block_tables=torch.zeros(2, 3, dtype=torch.int64)), "block_tables"),
        (dict(block_tables=torch.zeros(6, dtype=I32)), "block_tables"),
        (dict(context_lens=torch.zeros(3, dtype=I32)), "context_lens"),
        (dict(context_lens=torch.zeros(2, dtype=torch.int64)), "context_lens"),
        (dict(q_lens=torch.zeros(2)), "q_lens"),
        (dict(q_offsets=torch.zeros(1, dtype=I32)), "q_offsets"),
        (dict(q_offsets=None), "q_offsets"),
        (dict(out=torch.zeros(6, 4, 64)), "shape and type"),
        (dict(out=torch.zeros(5, 4, 64, dtype=F16)), "shape and type"),
        (dict(out=torch.zeros(6, 64, 4, dtype=F16).transpose(1, 2)), "contiguous heads"),
        (dict(out=torch.zeros(1, 4, 64, dtype=F16).expand(6, 4, 64)), "contiguous heads"),
    ]
    for kw, match in bad:
        with pytest.raises(ValueError, match=match):
            pa.paged_tree_attention(**{**_case(), **kw}, tree_mask=mask)
        with pytest.raises(ValueError, match=match):
            pa.paged_window_attention(**{**_case(), **kw}, window=5)
    for m, match in ((mask.float(), "bool"), (mask[:5], "total_q"), (mask[:, :2], "max_q_len"), (mask[0], "total_q")):
        with pytest.raises(ValueError, match=match):
            pa.paged_tree_attention(**_case(), tree_mask=m)
    for w, sinks in ((0, 0), (-1, 0), (4, -1), (1 << 31, 0), (4, 1 << 31)):
        with pytest.raises(ValueError, match="window"):
            pa.paged_window_attention(**_case(), window=w, sinks=sinks)
    c = _case()
    with pytest.raises(ValueError, match="one token"):
        pa.paged_window_attention(**{**c, "q_lens": None, "q_offsets": None}, window=5)
    for out in (c["q"], c["k_cache"].view(-1)[64:64 + 6 * 256].view(6, 4, 64)):
        with pytest.raises(ValueError, match="overlap"):
            pa.paged_window_attention(**c, window=5, out=out)
    assert not calls


def test_cpu_tensors_are_refused():
    from nanopointllm_b200 import logprobs, paged_attention
    with pytest.raises(ValueError, match="CUDA"):
        paged_attention.paged_window_attention(**_case(), window=5)
    with pytest.raises(ValueError, match="CUDA"):
        paged_attention.paged_tree_attention(**_case(), tree_mask=torch.ones(6, 3, dtype=torch.bool))
    with pytest.raises(ValueError, match="CUDA"):
        logprobs.token_logprobs(torch.zeros(2, 9), torch.zeros(2, dtype=torch.int64))


def test_what_the_attention_calls_hand_over(PA, L):
    pa, calls = PA
    c = _case()
    packed = torch.zeros(6, 4 * 64 + 256, dtype=F16)
    c["q"] = packed[:, 128:128 + 256].view(6, 4, 64)
    wide = torch.zeros(6, 40, dtype=torch.bool)
    store = torch.zeros(6, 320, dtype=F16)
    out = store[:, 8:264].view(6, 4, 64)
    assert pa.paged_tree_attention(**c, tree_mask=wide[:, 3:20], max_q_len=11, out=out) is out
    name, a = calls.pop()
    assert name == "npl_paged_tree_attention"
    assert a == (c["q"].data_ptr(), L.NPL_F16, 512, 6, 4, 2, 64, c["k_cache"].data_ptr(), c["v_cache"].data_ptr(), 7, 16,
                 c["block_tables"].data_ptr(), 3, 3, c["context_lens"].data_ptr(), c["q_lens"].data_ptr(),
                 c["q_offsets"].data_ptr(), 2, 11, wide[:, 3:].data_ptr(), 40, 17, 0.125, out.data_ptr(), 320)
    # without max_q_len the lengths are read back; a q that the kernel cannot read is copied
    c["q"] = torch.zeros(4, 6, 64, dtype=F16).transpose(0, 1)
    got = pa.paged_window_attention(**c, window=9, sinks=2)
    name, a = calls.pop()
    assert name == "npl_paged_window_attention" and a[18:21] == (3, 9, 2) and a[2] == 256 and a[0] != c["q"].data_ptr()
    assert got.shape == (6, 4, 64) and got.is_contiguous() and a[-2:] == (got.data_ptr(), 256)
    one = _case(T=2)
    pa.paged_window_attention(**{**one, "q_lens": None, "q_offsets": None}, window=9)
    assert calls.pop()[1][15:19] == (None, None, 2, 1)
    # nothing to do: no call
    pa.paged_tree_attention(**{**c, "q_lens": c["q_lens"] * 0}, tree_mask=wide)
    pa.paged_window_attention(**{**_case(T=0), "q_lens": None, "q_offsets": None, "block_tables": torch.zeros(0, 3, dtype=I32),
                                 "context_lens": torch.zeros(0, dtype=I32)}, window=9)
    assert not calls


def test_tree_mask_from_parents():
    from nanopointllm_b200 import paged_attention as pa
    g = torch.Generator().manual_seed(0)
    lens = [5, 1, 12, 0, 8]
    order = [2, 0, 4, 1]  # rows need not follow the sequences
    parents, offs, at = {}, [0] * 5, 0
    for b in order:
        parents[b] = [int(torch.randint(-1, i, (1,), generator=g)) if i else -1 for i in range(lens[b])]
        offs[b] = at
        at += lens[b]
    offs[3] = at
    flat = sum((parents[b] for b in order), [])
    got = pa.tree_mask_from_parents(torch.tensor(flat), torch.tensor(offs), 12)
    want = torch.zeros(at, 12, dtype=torch.bool)
    for b in order:
        for i in range(lens[b]):
            j = i
            while j >= 0:
                want[offs[b] + i, j] = True
                j = parents[b][j]
    assert torch.equal(got, want)
    chain = pa.tree_mask_from_parents(torch.arange(-1, 6), torch.tensor([0]), 7)
    assert torch.equal(chain, torch.ones(7, 7).tril().bool())
    with pytest.raises(ValueError):
        pa.tree_mask_from_parents(torch.zeros(3), torch.tensor([0]), 3)


def test_strides_of_a_single_row(PA):
    """A tensor with one row may have any stride there: it is never used."""
    pa, calls = PA
    c = _case(T=1, B=1)
    c["q"] = torch.zeros(256, dtype=F16).as_strided((1, 4, 64), (259, 64, 1))
    c["block_tables"] = torch.zeros(3, dtype=I32).as_strided((1, 3), (0, 1))
    out = torch.zeros(256, dtype=F16).as_strided((1, 4, 64), (261, 64, 1))
    mask = torch.ones(5, dtype=torch.bool).as_strided((1, 5), (0, 1))
    assert pa.paged_tree_attention(**c, tree_mask=mask, max_q_len=1, out=out) is out
    _, a = calls.pop()
    assert (a[0], a[2], a[12], a[20], a[-2:]) == (c["q"].data_ptr(), 256, 3, 5, (out.data_ptr(), 256))
    for most in (-1, 1 << 31):
        with pytest.raises(ValueError, match="max_q_len"):
            pa.paged_window_attention(**c, window=5, max_q_len=most)
    assert not calls


def test_tree_mask_from_odd_parents():
    from nanopointllm_b200 import paged_attention as pa
    got = pa.tree_mask_from_parents(torch.tensor([-5, 0, 9, 4]), torch.tensor([0]), 4)
    assert torch.equal(got, torch.tensor([[1, 0, 0, 0], [1, 1, 0, 0], [0, 0, 1, 0], [0, 0, 0, 1]]).bool())
    assert pa.tree_mask_from_parents(torch.zeros(0, dtype=I32), torch.zeros(0, dtype=I32), 4).shape == (0, 4)
    with pytest.raises(ValueError, match="q_offsets"):
        pa.tree_mask_from_parents(torch.zeros(2, dtype=I32), torch.zeros(0, dtype=I32), 4)


def test_refusals_and_layouts_of_log_probabilities(LP, L):
    lp, calls = LP
    x, ids = torch.zeros(4, 50), torch.zeros(4, dtype=torch.int64)
    for args, match in (((x.double(), ids), "float32"), ((torch.zeros(4, 0), ids), "column"),
                        ((x, ids.int()), "int64"), ((x, ids[:3]), "shape"), ((x, ids, -1), "top_k"),
                        ((x, ids, 33), "top_k"), ((x[:, :5], ids, 6), "top_k")):
        with pytest.raises(ValueError, match=match):
            lp.token_logprobs(*args)
    store = torch.zeros(4, 64, dtype=BF16)
    r = lp.token_logprobs(store[:, 3:53], ids, 7)
    name, a = calls.pop()
    assert a[:5] == (store[:, 3:].data_ptr(), L.NPL_BF16, 64, 4, 50) and a[6] == 7
    assert [t.shape for t in r] == [(4,), (4,), (4, 7), (4, 7)] and r.top_ids.dtype == torch.int64
    r = lp.token_logprobs(torch.zeros(2, 3, 50, dtype=F16), torch.zeros(2, 3, dtype=torch.int64), 2)
    assert r.logprobs.shape == (2, 3) and r.top_logprobs.shape == (2, 3, 2) and calls.pop()[1][3] == 6
    r = lp.token_logprobs(x[0], ids[0], 2)
    assert r.logprobs.shape == () and r.top_ids.shape == (2,) and calls.pop()[1][2:5] == (50, 1, 50)
    lp.token_logprobs(x.t().contiguous().t(), ids)
    assert calls.pop()[1][2] == 50  # copied to rows
    lp.token_logprobs(x[:0], ids[:0], 3)
    assert not calls


def test_oracle_of_attention():
    """Against torch's softmax in 64 bits over gathered keys; bad values reach the rows that see them only."""
    g = torch.Generator().manual_seed(2)
    n, ctx, H, Hkv, D, bs = 5, 23, 4, 2, 8, 8
    q, k, v = (torch.randn(*s, generator=g) for s in ((n, H, D), (4, bs, Hkv, D), (4, bs, Hkv, D)))
    bt = torch.tensor([[2, 0, 3]])
    kk, vv = (t[bt[0]].reshape(-1, Hkv, D)[:ctx].double() for t in (k, v))
    seen = OM.window_seen(n, ctx, 6, 3)
    assert seen[0].tolist() == [i < 3 or 13 <= i <= 18 for i in range(ctx)]
    out, tol = OM.attention(q, k, v, bt.numpy(), [ctx], [n], [0], 0.3, 2, lambda b: seen, "float16")
    for h in range(H):
        s = (q[:, h].double() @ kk[:, h // 2].T * 0.3).masked_fill(~torch.from_numpy(seen), -float("inf"))
        np.testing.assert_allclose(out[:, h], (s.softmax(-1) @ vv[:, h // 2]).numpy(), atol=1e-12)
    v[3, 1, 0, 4] = float("nan")  # key 17
    bad, _ = OM.attention(q, k, v, bt.numpy(), [ctx], [n], [0], 0.3, 2, lambda b: seen, "float16")
    nan = np.isnan(bad)
    assert (nan[:, 0, 4] == seen[:, 17]).all() and nan.sum() == 2 * seen[:, 17].sum()
    # the same sums of 23 terms below 4 in another order: within 2 * 23 * 2^-53 * 4
    np.testing.assert_allclose(bad[~nan], out[~nan], rtol=0, atol=2 * 23 * 2.0 ** -53 * 4)


def test_oracle_of_log_probabilities():
    x = torch.randn(6, 40, generator=torch.Generator().manual_seed(1)) * 4
    x[1, 3] = -float("inf")
    x[2, 5] = x[2, 9] = x[2].max() + 1
    ids = torch.tensor([0, 3, 9, 39, -1, 40])
    lp, ent, order, top, _, _ = OL.token_logprobs(x.numpy(), ids.numpy(), 5)
    want = torch.log_softmax(x.double(), -1)
    np.testing.assert_allclose(lp[:4], want[torch.arange(4), ids[:4]].numpy(), atol=1e-12)
    assert lp[1] == -np.inf and lp[4] == 0 and np.isnan(lp[5]) and order[2, :2].tolist() == [5, 9]
    p = want.exp()
    np.testing.assert_allclose(ent, -(p * torch.where(p > 0, want, 0)).sum(-1).numpy(), atol=1e-12)
    np.testing.assert_allclose(top, want.gather(1, torch.from_numpy(order.copy())).numpy(), atol=1e-12)


def test_division_by_multiplication():
    """floor(n / d) as the kernels form it, for every d that a launch can have and the n around its multiples."""
    rng = np.random.default_rng(0)
    for d in [*range(1, 3000), 2 ** 20, 2 ** 20 + 1, 2 ** 30, 2 ** 31 - 1, *rng.integers(3000, 2 ** 31, 500).tolist()]:
        s = (d - 1).bit_length()
        mul = -(-(1 << (31 + s)) // d)
        assert mul < 1 << 32
        n = np.unique(np.concatenate([rng.integers(0, 2 ** 31, 20), [0, 1, d - 1, d, 2 ** 31 - 1],
                                      (np.arange(1, 4) * d)[np.arange(1, 4) * d < 2 ** 31] - 1]).astype(np.int64))
        for m in n.tolist():
            assert (m if s == 0 else (m * mul) >> (31 + s)) == m // d


def test_polynomial_exponential():
    """2^x as the kernels form it for a part of the exponentials, in fp32 step by step with the source's own
    coefficients: within 2^-22 relative down to 2^-126, and no more than 2^-126 below."""
    import re
    from conftest import REPO
    text = (REPO / "nano-pointllm_b200" / "csrc" / "masked_attention.cu").read_text()
    body = text[text.index("ma_exp2_poly(uint64_t x2) {"):]
    body = body[:body.index("return make_float2")]
    coeff = [np.float32(m) for m in re.findall(r"ma_pair\((\d\.\d+e[+-]\d+)f, ", body)]
    coeff += [np.float32(m) for m in re.findall(r"ma_pair\((1\.00\d+)f, ", body)]
    assert len(coeff) == 6
    rng = np.random.default_rng(0)
    x = np.concatenate([rng.uniform(-140, 16, 400000), np.arange(-140, 16), np.arange(-140, 16) + 0.5,
                        [-np.inf, -1e30, -127, -126.5]]).astype(np.float32)
    c = np.maximum(x, np.float32(-127))
    magic = np.float32(12582912)
    t = c + magic
    f = (c - (t - magic)).astype(np.float32)  # exact
    y = np.full_like(f, coeff[0])
    for a in coeff[1:]:
        y = (y.astype(np.float64) * f + a).astype(np.float32)  # a fused step
    r = (y.view(np.int32) + (t.view(np.int32) << 23)).view(np.float32).astype(np.float64)
    want = np.exp2(x.astype(np.float64))
    far = x < -126
    assert (np.abs(r - want) <= want * 2.0 ** -22)[~far].all()
    assert (r[far] >= 0).all() and (r[far] <= 2.0 ** -125).all()


def test_polynomial_exponential_by_a_product():
    """2^x as the kernels form it for a part of the exponentials, with 2^n from the bits of n as a factor: within
    2^-22 relative, 0 from x = -127 down (n = -127), and NaN where x is NaN."""
    import re
    from conftest import REPO
    text = (REPO / "nano-pointllm_b200" / "csrc" / "masked_attention.cu").read_text()
    body = text[text.index("ma_exp2_poly(uint64_t x2) {"):]
    body = body[:body.index("\n}")]
    assert "<< 23) + 0x3f800000" in body and "ma_mul2(y, power)" in body
    coeff = [np.float32(m) for m in re.findall(r"ma_pair\((\d\.\d+(?:e[+-]\d+)?)f, ", body) if m != "12582912."]
    coeff = [c for c in coeff if c < 2]
    assert len(coeff) == 6
    rng = np.random.default_rng(1)
    x = np.concatenate([rng.uniform(-140, 16, 400000), np.arange(-140, 128), np.arange(-140, 127) + 0.5,
                        [-np.inf, -1e30, -127, -126.5, -126.49, np.nan]]).astype(np.float32)
    with np.errstate(invalid="ignore", over="ignore"):
        c = np.where(np.isnan(x), x, np.maximum(x, np.float32(-127)))
        t = c + np.float32(12582912)
        f = (c - (t - np.float32(12582912))).astype(np.float32)  # exact
        y = np.full_like(f, coeff[0])
        for a in coeff[1:]:
            y = (y.astype(np.float64) * f + a).astype(np.float32)  # a fused step
        power = ((t.view(np.int32).astype(np.int64) << 23) + 0x3f800000).astype(np.uint32).view(np.float32)
        r = (y * power).astype(np.float64)
    want = np.exp2(x.astype(np.float64))
    assert (np.isnan(r) == np.isnan(x)).all()
    near = x >= -126.0
    assert (np.abs(r - want) <= want * 2.0 ** -22)[near].all()
    assert (r[x <= -127] == 0).all() and (r[x < -126.0] >= 0).all() and (r[x < -126.0] <= 2.0 ** -125).all()


@pytest.mark.parametrize("stages,lists", [(5, 4), (8, 8), (10, 8)])
def test_lists_of_bad_values_are_free_when_taken_again(stages, lists):
    """The order of a CTA's roles at its worst: a stream still reads its lists of item j, so that the products of the
    next item in which it has rows wait for it, and with them the stages of the tiles behind (two an item at the
    least). No item whose V tile may come meanwhile has the lists of item j: items of one stream and of two count
    apart. (Counted together, eight lists are not enough.)"""
    from conftest import REPO
    text = (REPO / "nano-pointllm_b200" / "csrc" / "masked_attention.cu").read_text()
    assert text.count(": MaBarriers<D == 128 ? 4 : 8> {") == 2
    assert "kStages = D == 128 ? 5 : 8;" in text and "kStages = D == 64 ? 10 : 5;" in text
    rng = np.random.default_rng(stages)
    together = 0
    for _ in range(200):
        two = rng.random(60) < rng.choice([0.1, 0.5, 0.9])
        count, lists_of = [0, 0], []
        for t in two.tolist():
            lists_of.append((t, count[t] % lists))
            count[t] += 1
        for j in range(60):
            for stream in ((0, 1) if two[j] else (0,)):
                next_item = next((i for i in range(j + 1, 60) if stream == 0 or two[i]), 1000)
                free = 2 * next_item  # K and V of item i are tiles 2 i and 2 i + 1 of the ring; K of the next is read
                meanwhile = [i for i in range(j + 1, 60) if 2 * i + 1 - stages <= free]
                assert all(lists_of[i] != lists_of[j] for i in meanwhile)
                together += any(i % 8 == j % 8 for i in meanwhile)
    assert together > 0


def test_tree_mask_leaves_out_sequences_without_drafts():
    """Their offsets may be any, inside other sequences' rows too."""
    from nanopointllm_b200 import paged_attention as pa
    parents = torch.tensor([-1, 0, 1, 0, -1, 0, 0])
    want = pa.tree_mask_from_parents(parents, torch.tensor([0, 4]), 4)
    for offs, lens in (([0, 2, 4], [4, 0, 3]), ([2, 0, 4, 5], [0, 4, 3, 0]), ([0, 100, 4], [4, 0, 3]),
                       ([4, -3, 0, 3, 6, 7], [3, 0, 4, 0, 0, 0])):
        o, n = torch.tensor(offs, dtype=I32), torch.tensor(lens, dtype=I32)
        assert torch.equal(pa.tree_mask_from_parents(parents, o, 4, n), want), (offs, lens)
    assert torch.equal(pa.tree_mask_from_parents(parents, torch.tensor([4, 0]), 4, torch.tensor([3, 4])), want)
    for wrong in (torch.tensor([4]), torch.tensor([4.0, 3.0])):
        with pytest.raises(ValueError, match="q_lens"):
            pa.tree_mask_from_parents(parents, torch.tensor([0, 4]), 4, wrong)
