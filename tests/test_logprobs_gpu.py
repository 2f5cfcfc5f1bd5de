"""Log probabilities of tokens, entropy and top alternatives on the GPU, against
the 64-bit oracle (oracle/logprobs.py, where the tolerances are derived)."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import logprobs as O

pytestmark = pytest.mark.gpu

TYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}


@pytest.fixture
def P(cuda_device):
    from nanopointllm_b200 import _lib, logprobs
    yield logprobs
    torch.cuda.synchronize()
    _lib.device_status()


def check(r, logits, ids, k):
    v = logits.shape[-1]
    x = logits.reshape(-1, v).float().cpu().numpy()
    i = ids.reshape(-1).cpu().numpy()
    lp, ent, order, top_lp, tol, ent_tol = O.token_logprobs(x, i, k)
    got = [t.reshape(len(i), -1).cpu().numpy() for t in r]
    np.testing.assert_array_equal(got[2], order)

    def close(a, b, t, what):
        same = (np.isnan(a) & np.isnan(b)) | (a == b)
        err = np.where(same, 0.0, np.abs(a.astype(np.float64) - b))
        assert (same | (err <= t)).all(), f"{what}: {np.nanmax(err)} {np.nanmax(err / t)} times its bound"

    close(got[0][:, 0], lp, O.value_tol(tol, lp), "logprobs")
    close(got[1][:, 0], ent, ent_tol, "entropy")
    close(got[3], top_lp, O.value_tol(tol[:, None], top_lp), "top")


def rows(n, v, dtype, seed=0, spread=2.5):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(n, v, generator=g) * spread
    x[torch.arange(n), torch.randint(0, v, (n,), generator=g)] += 9.0
    ids = torch.randint(0, v, (n,), generator=g)
    return x.to(dtype).cuda(), ids.cuda()


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("n,v,k", [
    (1, 1, 1), (3, 2, 2), (2, 7, 0), (5, 31, 31), (4, 33, 32), (1, 1000, 5), (9, 1003, 20), (8, 32003, 5),
    (64, 32003, 20), (300, 4099, 1), (700, 2049, 32), (2, 160001, 20), (1, 300007, 32), (37, 50257, 3), (150, 8192, 10),
    (149, 40000, 0),
])
def test_rows(P, n, v, k, kind):
    x, ids = rows(n, v, TYPES[kind], seed=n + v)
    check(P.token_logprobs(x, ids, k), x, ids, k)


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("v", [257, 32003, 70001])
@pytest.mark.parametrize("n", [2, 400])
def test_ties_go_to_the_lowest(P, n, v, kind):
    """Few different values, whole rows of one value, zeros of both signs."""
    g = torch.Generator().manual_seed(v)
    x = torch.randint(-2, 3, (n, v), generator=g).float()
    x[0] = 0.5
    x[1] = torch.where(torch.rand(v, generator=g) < 0.5, 0.0, -0.0)
    x = x.to(TYPES[kind]).cuda()
    ids = torch.randint(0, v, (n,), generator=g).cuda()
    check(P.token_logprobs(x, ids, 20), x, ids, 20)


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("n", [12, 310])
@pytest.mark.parametrize("v", [100, 5001, 32003])
def test_barred_infinite_and_nan(P, n, v, kind):
    """Minus infinity and the type's lowest value (barred tokens), rows of
    nothing else, plus infinity and NaN: each stays in its row."""
    dt = TYPES[kind]
    x, ids = rows(n, v, dt, seed=v)
    low = torch.finfo(dt).min
    x[0, 5:] = -float("inf")
    x[1, :-3] = low
    x[2] = -float("inf")
    x[3] = low
    x[4, 17] = float("nan")
    x[5, 3], x[5, 60] = float("inf"), float("inf")
    x[6, 90] = float("inf")
    x[6, 91] = float("nan")
    x[7, ::2] = -float("inf")
    x[8] = -float("inf")
    x[8, 77] = 3.0
    x[9] = torch.finfo(dt).max
    x[10, 1:] = low
    ids[0], ids[1], ids[7], ids[8] = 40, 2, 6, 5
    check(P.token_logprobs(x, ids, 20), x, ids, 20)


def test_padding_and_bad_tokens(P):
    from nanopointllm_b200 import _lib
    x, ids = rows(6, 500, torch.float16)
    ids[1] = ids[4] = -1
    r = P.token_logprobs(x, ids, 2)
    check(r, x, ids, 2)
    assert r.logprobs[1] == 0 and r.logprobs[4] == 0
    torch.cuda.synchronize()
    _lib.device_status()
    for wrong in (-2, 500, 1 << 40, -(1 << 62)):
        ids[3] = wrong
        r = P.token_logprobs(x, ids, 2)
        torch.cuda.synchronize()
        with pytest.raises(_lib.NplTimeout):
            _lib.device_status()
        check(r, x, ids, 2)


@pytest.mark.parametrize("kind", TYPES)
def test_layouts(P, kind):
    """Leading dimensions, strided rows at every alignment, ids of another stride."""
    x, ids = rows(24, 1001, TYPES[kind], seed=4)
    check(P.token_logprobs(x.view(2, 3, 4, 1001), ids.view(2, 3, 4), 4), x, ids, 4)
    check(P.token_logprobs(x[3], ids[3], 4), x[3:4], ids[3:4], 4)
    for off in range(9):
        store = torch.full((24, 1030), float("nan"), dtype=x.dtype, device="cuda")
        store[:, off:off + 1001] = x
        view = store[:, off:off + 1001]
        check(P.token_logprobs(view, ids, 4), x, ids, 4)
        check(P.token_logprobs(view[::2], ids[::2], 4), x[::2], ids[::2], 4)
    check(P.token_logprobs(x.t().contiguous().t(), ids, 4), x, ids, 4)
    r = P.token_logprobs(x[:0], ids[:0], 3)
    assert r.logprobs.shape == (0,) and r.top_ids.shape == (0, 3)


def test_confident_rows(P):
    """Probabilities near one: the absolute error stays at fp32's half steps."""
    x = torch.zeros(4, 32003)
    x[:, 9] = torch.tensor([12.0, 20.0, 40.0, 100.0])
    ids = torch.full((4,), 9)
    check(P.token_logprobs(x.cuda(), ids.cuda(), 3), x, ids, 3)


def test_graphs_streams_and_calls_at_once(P):
    xs = [rows(8, 32003, torch.float16, seed=1), rows(2, 160001, torch.float32, seed=2),
          rows(400, 8000, torch.bfloat16, seed=3)]
    refs = [P.token_logprobs(x, i, 20) for x, i in xs]
    streams = [torch.cuda.Stream() for _ in xs]
    graphs = []
    for s, (x, i) in zip(streams, xs):
        s.wait_stream(torch.cuda.current_stream())
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            out = P.token_logprobs(x, i, 20)
        graphs.append((g, out))
    torch.cuda.synchronize()
    for _ in range(10):
        for s, (g, out) in zip(streams, graphs):
            with torch.cuda.stream(s):
                for t in out:
                    t.zero_()
                g.replay()
        eager = [P.token_logprobs(x, i, 20) for x, i in xs]
        torch.cuda.synchronize()
        for ref, (_, out), e in zip(refs, graphs, eager):
            for a, b, c in zip(ref, out, e):
                assert torch.equal(a, b) and torch.equal(a, c)


def test_far_rows(P):
    """Rows whose offsets pass 32 bits."""
    n, v = 70000, 32003  # 2^31 elements and more
    x = torch.zeros(n, v, dtype=torch.float16, device="cuda")
    near, ids = rows(300, v, torch.float16, seed=8)
    x[-300:] = near
    all_ids = torch.zeros(n, dtype=torch.int64, device="cuda")
    all_ids[-300:] = ids
    r = P.token_logprobs(x, all_ids, 4)
    check([t[-300:] for t in r], near, ids, 4)
    check([t[:300] for t in r], x[:300], all_ids[:300], 4)


def test_written_just_before(P):
    x, ids = rows(16, 32003, torch.float16, seed=6)
    want = P.token_logprobs(x, ids, 5)
    keep = x.clone()
    for _ in range(10):
        x.zero_()
        torch.cuda.synchronize()
        x.copy_(keep)
        for a, b in zip(P.token_logprobs(x, ids, 5), want):
            assert torch.equal(a, b)


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("n", [3, 330])
def test_large_logits_that_share_their_places(P, n, kind):
    """Rows whose largest logits stand where one thread reads them all, more
    than any list of candidates holds; few of them, many equal ones, and equal
    ones that end within the row."""
    v = 70000
    x = torch.zeros(n, v)
    for i in range(n):
        lo = 2048 * (1 + i % 5) + 16 * (i % 3)
        at = torch.cat([torch.arange(lo + 2048 * j, lo + 2048 * j + 64) for j in range(28)])
        x[i, at] = 50.0 + (torch.arange(at.numel()) % (3, 40, 1000)[i % 3]).float() / 16
    x = x.to(TYPES[kind]).cuda()
    ids = torch.arange(n).cuda()
    check(P.token_logprobs(x, ids, 32), x, ids, 32)


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("n", [7, 310])
@pytest.mark.parametrize("v", [600, 5001, 70001])
def test_nan_before_all_others(P, n, v, kind):
    """A NaN in the first place, with more equal logits than any list of candidates holds, beside it or behind it."""
    x, ids = rows(n, v, TYPES[kind], seed=v)
    nan = float("nan")
    x[0] = nan
    x[1] = 0.0
    x[1, 0] = nan
    x[2, 0] = nan
    x[3] = 1.0
    x[3, 0] = x[3, 7] = x[3, v - 1] = nan
    x[4] = -x[0]  # with the sign set
    x[5] = nan
    x[5, 0] = float("inf")
    x[6] = -float("inf")
    x[6, 0] = nan
    for k in (1, 5, 20):
        check(P.token_logprobs(x, ids, k), x, ids, k)
