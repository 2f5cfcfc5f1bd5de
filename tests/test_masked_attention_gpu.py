"""Tree attention and sliding-window attention with sinks on the GPU, against
the 64-bit oracle (oracle/masked_attention.py, where the tolerance is derived)."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import masked_attention as O

pytestmark = pytest.mark.gpu

F16, BF16 = torch.float16, torch.bfloat16
NAME = {F16: "float16", BF16: "bfloat16"}


@pytest.fixture
def PA(cuda_device):
    from nanopointllm_b200 import _lib, paged_attention
    yield paged_attention
    torch.cuda.synchronize()
    _lib.device_status()


class Case:
    """Sequences [(new tokens, context)] over a shuffled pool, on the GPU."""

    def __init__(self, seqs, H, Hkv, D, bs, dtype, seed=0, dev="cuda", gaps=0):
        g = torch.Generator().manual_seed(seed)
        self.seqs, self.H, self.Hkv, self.D, self.bs, self.dtype = seqs, H, Hkv, D, bs, dtype
        self.groups, self.scale = H // Hkv, D ** -0.5
        new = [n for n, _ in seqs]
        offs, at = [], gaps
        for n in new:
            offs.append(at)
            at += n + gaps
        self.total = at
        width = max(1, max(-(-c // bs) for _, c in seqs)) + 1
        nb = sum(-(-c // bs) for _, c in seqs) + 3
        perm = torch.randperm(nb, generator=g).int()
        bt = torch.full((len(seqs), width), -1, dtype=torch.int32)
        j = 0
        for i, (_, c) in enumerate(seqs):
            m = -(-c // bs)
            bt[i, :m] = perm[j:j + m]
            j += m
        self.bt = bt
        rnd = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
        q = rnd(self.total, H, D) * torch.exp(0.7 * rnd(self.total, H, 1))
        self.q = q.to(dtype).to(dev)
        self.k = rnd(nb, bs, Hkv, D).to(dtype).to(dev)
        self.v = rnd(nb, bs, Hkv, D).to(dtype).to(dev)
        self.ctx = torch.tensor([c for _, c in seqs], dtype=torch.int32)
        self.new = torch.tensor(new, dtype=torch.int32)
        self.offs = torch.tensor(offs, dtype=torch.int32)
        self.dev = dev
        self.g = g

    def slot(self, b, i):
        return int(self.bt[b, i // self.bs]), i % self.bs

    def args(self):
        d = self.dev
        return (self.q, self.k, self.v, self.bt.to(d), self.ctx.to(d), self.new.to(d), self.offs.to(d), self.scale,
                self.groups)

    def oracle(self, seen_of):
        f = lambda t: t.float().cpu().numpy()  # noqa: E731
        return O.attention(f(self.q), f(self.k), f(self.v), self.bt.numpy(), self.ctx.numpy(), self.new.numpy(),
                           self.offs.numpy(), self.scale, self.groups, seen_of, NAME[self.dtype])

    def rows(self, b):
        return slice(int(self.offs[b]), int(self.offs[b] + self.new[b]))

    def tree_oracle(self, mask):
        m = mask.cpu().numpy()
        return self.oracle(lambda b: O.tree_seen(m[self.rows(b)], int(self.new[b]), int(self.ctx[b])))

    def window_oracle(self, window, sinks):
        return self.oracle(lambda b: O.window_seen(int(self.new[b]), int(self.ctx[b]), window, sinks))


def check(got, want, what=""):
    out, tol = want
    g = got.double().cpu().numpy()
    of_some = ~np.isnan(tol)
    bad = of_some & ~np.isfinite(out)
    assert (np.isnan(g) == np.isnan(out))[bad].all() and (g[bad & np.isinf(out)] == out[bad & np.isinf(out)]).all(), \
        f"{what}: infinities or NaN differ"
    ok = of_some & np.isfinite(out)
    err = np.abs(g - out)
    assert np.isfinite(g[ok]).all(), f"{what}: not finite"
    worst = (err[ok] / np.maximum(tol[ok], 1e-300)).max(initial=0.0)
    assert worst <= 1.0, f"{what}: error {err[ok].max()} is {worst} times its bound"


def tree(case, g=None, density=None, cols=None):
    """A tree's mask (or, with a density, any mask) for every sequence."""
    g = g or case.g
    cols = cols or max(1, int(case.new.max()))
    mask = torch.zeros(case.total, cols, dtype=torch.bool)
    for b, (n, _) in enumerate(case.seqs):
        r0 = int(case.offs[b])
        if density is not None:
            mask[r0:r0 + n] = torch.rand(n, cols, generator=g) < density
            continue
        for i in range(n):
            p = i - 1 - int(torch.randint(0, 5, (1,), generator=g))
            if p >= 0:
                mask[r0 + i] = mask[r0 + p]
            mask[r0 + i, i] = True
    return mask.to(case.dev)


TREES = [
    ([(1, 1)], 4, 4, 128, 16),
    ([(16, 1040)], 8, 8, 128, 256),
    ([(64, 700), (64, 64), (64, 65), (64, 1999)], 4, 4, 128, 256),
    ([(7, 500), (1, 3), (0, 40), (25, 1025), (12, 12)], 8, 2, 128, 16),
    ([(61, 900), (33, 2000)], 14, 2, 64, 32),
    ([(128, 128), (100, 1300)], 2, 2, 64, 8),
    ([(129, 400), (300, 300), (257, 2500), (2, 130)], 2, 1, 128, 64),
    ([(40, 3000)], 16, 1, 128, 48),
    ([(3, 127), (3, 128), (3, 129), (3, 131), (1, 0), (2, 9000)], 6, 2, 128, 8),
    ([(5, 260)] * 40, 4, 4, 64, 128),
    ([(32, 500), (17, 900), (1, 40)], 4, 4, 128, 256),
    ([(31, 1500), (24, 333)], 3, 3, 64, 16),
    ([(6, 700), (5, 2000)], 10, 2, 128, 32),
    ([(33, 600), (9, 64)], 4, 4, 128, 16),
    ([(50, 400), (1, 700)], 3, 3, 128, 16),
    ([(3, 200), (2, 900)], 100, 1, 64, 16),
    ([(2, 300)], 128, 1, 128, 32),
    ([((7 * i) % 300, (7 * i) % 300 + 40 * (i % 5)) for i in range(60)], 4, 4, 64, 16),
]


@pytest.mark.parametrize("dtype", [F16, BF16], ids=["fp16", "bf16"])
@pytest.mark.parametrize("seqs,H,Hkv,D,bs", TREES, ids=[str(i) for i in range(len(TREES))])
def test_tree(PA, seqs, H, Hkv, D, bs, dtype):
    c = Case(seqs, H, Hkv, D, bs, dtype, seed=len(seqs) + bs)
    m = tree(c)
    got = PA.paged_tree_attention(*c.args(), m, max_q_len=int(c.new.max()))
    check(got, c.tree_oracle(m))
    assert torch.equal(got, PA.paged_tree_attention(*c.args(), m))  # the length read back, the same bits


@pytest.mark.parametrize("density", [0.0, 0.1, 0.9])
def test_any_mask_and_empty_rows(PA, density):
    """Masks that are no trees; without a prefix, rows that see nothing are zeros."""
    c = Case([(30, 30), (90, 90), (200, 200), (30, 500)], 4, 2, 128, 16, F16, seed=3)
    m = tree(c, density=density, cols=230)
    m[c.rows(0)][4:7] = False
    got = PA.paged_tree_attention(*c.args(), m.to(torch.uint8) * 255, max_q_len=200)
    check(got, c.tree_oracle(m))
    assert (got[4:7] == 0).all()


def test_tree_layouts(PA):
    """Rows in another order with rows of no sequence between them, q inside a
    packed projection, a strided mask and output."""
    c = Case([(9, 77), (31, 431), (4, 260)], 8, 4, 128, 16, F16, seed=5, gaps=2)
    packed = torch.zeros(c.total, 16 * 128, dtype=F16, device="cuda")
    packed[:, 256:256 + 1024] = c.q.flatten(1)
    q = packed[:, 256:256 + 1024].view(c.total, 8, 128)
    order = [2, 0, 1]
    a = list(c.args())
    a[0] = q
    for i in (3, 4, 5, 6):
        a[i] = a[i][order]
    wide = torch.ones(c.total, 70, dtype=torch.bool, device="cuda")
    m = tree(c, cols=33)
    wide[:, 5:38] = m
    store = torch.full((c.total, 1200), 7.0, dtype=F16, device="cuda")
    out = store[:, 16:16 + 1024].view(c.total, 8, 128)
    got = PA.paged_tree_attention(*a, wide[:, 5:38], max_q_len=33, out=out)
    assert got is out
    want = c.tree_oracle(m)
    check(got, want)
    free = torch.from_numpy(np.isnan(want[1])[:, 0, 0])
    assert (out[free.cuda()] == 7).all() and (store[:, :16] == 7).all() and (store[:, 1040:] == 7).all()


WINDOWS = [
    ([(1, 4001)], 8, 8, 128, 256, 1024, 4),
    ([(1, 1), (1, 200), (1, 1024), (1, 1025), (1, 1028), (1, 1029), (1, 0), (1, 3500)], 4, 4, 128, 16, 1024, 4),
    ([(1, 5000), (1, 700), (1, 90)], 16, 2, 128, 16, 300, 16),
    ([(1, 777)], 7, 1, 64, 8, 1, 0),
    ([(800, 800), (300, 900), (1, 400), (0, 10), (129, 129)], 4, 4, 128, 256, 256, 4),
    ([(1000, 1000)], 8, 2, 128, 16, 129, 1),
    ([(500, 2000), (40, 41)], 4, 1, 64, 32, 2000, 0),
    ([(513, 700), (2, 300)], 6, 2, 128, 24, 16, 65),
    ([(260, 260)], 2, 2, 64, 64, 1, 0),
    ([(260, 1260)], 2, 2, 128, 64, 1, 1),
    ([(333, 1333), (20, 20)], 3, 1, 128, 40, 100, 200),
    ([(128, 600), (127, 600), (3, 600)], 2, 2, 128, 128, 5000, 10000),
    ([(1, 900), (1, 5)], 32, 1, 128, 16, 200, 3),
    ([(1, 900), (1, 5)], 34, 1, 64, 64, 200, 3),
    ([(20, 300), (3, 3000)], 3, 3, 128, 256, 256, 4),
    ([(1, 3000)], 80, 1, 128, 16, 1000, 0),
    ([(1, (i * 37) % 900) for i in range(600)], 3, 3, 64, 16, 200, 4),
    ([((11 * i) % 260, (11 * i) % 260 + 70 * (i % 4)) for i in range(70)], 4, 2, 128, 8, 64, 9),
    ([(3, 200), (5, 40)], 128, 1, 64, 8, 30, 2),
]


@pytest.mark.parametrize("dtype", [F16, BF16], ids=["fp16", "bf16"])
@pytest.mark.parametrize("seqs,H,Hkv,D,bs,window,sinks", WINDOWS, ids=[str(i) for i in range(len(WINDOWS))])
def test_window(PA, seqs, H, Hkv, D, bs, window, sinks, dtype):
    c = Case(seqs, H, Hkv, D, bs, dtype, seed=window + bs)
    want = c.window_oracle(window, sinks)
    got = PA.paged_window_attention(*c.args(), window, sinks, max_q_len=int(c.new.max()))
    check(got, want)
    if all(n == 1 for n, _ in seqs):
        a = list(c.args())
        a[5] = a[6] = None
        check(PA.paged_window_attention(*a, window, sinks), want, "one token each")


@pytest.mark.parametrize("at", [0, 8, 16], ids=["32-byte", "16-byte", "32-byte, within a row"])
@pytest.mark.parametrize("D,bs", [(128, 16), (64, 64)])
def test_window_outputs_inside_wider_rows(PA, at, D, bs):
    """Rows that one CTA finishes are stored 32 bytes at a time, or 16 where they start between such boundaries;
    what lies beside them stays."""
    c = Case([(700, 900), (150, 150)] * 12, 8, 4, D, bs, F16, seed=at)
    store = torch.full((c.total, 8 * D + 32), 7.0, dtype=F16, device="cuda")
    out = store[:, at:at + 8 * D].view(c.total, 8, D)
    PA.paged_window_attention(*c.args(), 100, 4, max_q_len=700, out=out)
    check(out, c.window_oracle(100, 4))
    assert (store[:, :at] == 7).all() and (store[:, at + 8 * D:] == 7).all()


def test_loose_bounds_and_a_single_row(PA):
    """A bound far above the lengths gives what the exact one gives; one row may have any stride."""
    c = Case([(150, 400), (3, 90)], 4, 2, 128, 16, F16, seed=41)
    want = PA.paged_window_attention(*c.args(), 70, 4, max_q_len=c.total)
    for most in (c.total + 1, 5000, 2 ** 31 - 1):
        assert torch.equal(PA.paged_window_attention(*c.args(), 70, 4, max_q_len=most), want)
    c = Case([(1, 333)], 4, 2, 64, 8, BF16, seed=43)
    a = list(c.args())
    a[0] = c.q.as_strided((1, 4, 64), (259, 64, 1))
    a[3] = a[3].as_strided(a[3].shape, (0, 1))
    out = torch.zeros(256, dtype=BF16, device="cuda").as_strided((1, 4, 64), (261, 64, 1))
    check(PA.paged_window_attention(*a, 100, 3, max_q_len=1, out=out), c.window_oracle(100, 3))
    mask = torch.ones(3, dtype=torch.bool, device="cuda").as_strided((1, 3), (0, 1))
    check(PA.paged_tree_attention(*a, mask, max_q_len=1), c.tree_oracle(mask))


def test_window_of_everything_is_causal(PA):
    """A window longer than the context: the causal kernel's results, within both kernels' roundings."""
    c = Case([(300, 300), (129, 700)], 8, 2, 128, 16, F16, seed=2)
    a = PA.paged_window_attention(*c.args(), 1 << 30, 0)
    b = PA.paged_varlen_attention(*c.args())
    tol = torch.from_numpy(2 * c.window_oracle(1 << 30, 0)[1]).cuda()
    assert ((a.double() - b.double()).abs() <= tol).all()


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")], ids=["nan", "inf", "-inf"])
@pytest.mark.parametrize("new", [1, 40, 300])
def test_freed_pages_are_not_read(PA, new, bad):
    """Behind the window and before the sinks end: table entries of freed pages
    are -1 or name pages of others, and their slots hold anything."""
    from nanopointllm_b200 import _lib
    c = Case([(new, 1500)], 4, 2, 128, 16, F16, seed=7)
    want = c.window_oracle(256, 20)
    first = 1500 - new - 256 + 1  # the first key that a window holds
    for i in range(1500):
        if 20 <= i < first:
            blk, at = c.slot(0, i)
            c.k[blk, at], c.v[blk, at] = bad, bad
    for i in range(1500, c.bt.shape[1] * 16):  # behind the context, in its last page
        if c.bt[0, i // 16] >= 0:
            blk, at = c.slot(0, i)
            c.k[blk, at], c.v[blk, at] = bad, bad
    gone = [p for p in range(c.bt.shape[1]) if p * 16 >= 20 and (p + 1) * 16 <= first]
    assert gone
    c.bt[0, gone[::2]] = -1
    c.bt[0, gone[1::2]] = 1 << 30
    check(PA.paged_window_attention(*c.args(), 256, 20), want)
    torch.cuda.synchronize()
    _lib.device_status()  # no entry was called bad


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")], ids=["nan", "inf", "-inf"])
@pytest.mark.parametrize("what", ["k", "v", "kv"])
def test_bad_values_reach_their_rows_only(PA, what, bad):
    """A slot that some rows see and others do not."""
    for seqs, D in (([(20, 300), (140, 400)], 128), ([(64, 64)], 64)):
        c = Case(seqs, 4, 2, D, 16, F16, seed=11)
        m = tree(c)
        for b, (n, ctx) in enumerate(seqs):
            blk, at = c.slot(b, ctx - n + n // 2)
            if "k" in what:
                c.k[blk, at, 0, 3] = bad
            if "v" in what:
                c.v[blk, at, 0, 5] = bad
                c.v[blk, at, 1] = bad
        if what == "v":
            check(PA.paged_tree_attention(*c.args(), m), c.tree_oracle(m))
        else:  # rows that see the slot are not determined where the score is infinite or NaN: the others are
            out, tol = c.tree_oracle(m)
            got = PA.paged_tree_attention(*c.args(), m)
            seen = np.zeros(c.total, bool)
            for b, (n, ctx) in enumerate(seqs):
                seen[c.rows(b)] = m[c.rows(b), n // 2].cpu().numpy()
            tol[seen] = np.nan
            assert (~seen).sum() > 10
            check(got, (out, tol))
    c = Case([(300, 600), (1, 900)], 4, 2, 128, 16, F16, seed=12)
    for b, i in ((0, 450), (0, 301), (1, 700)):
        blk, at = c.slot(b, i)
        c.v[blk, at, 0, 9] = bad
        c.v[blk, at, 1, 100:] = bad
    check(PA.paged_window_attention(*c.args(), 100, 4), c.window_oracle(100, 4))


def test_many_bad_values(PA):
    """More of them than any list would hold."""
    c = Case([(400, 800)], 2, 1, 64, 16, F16, seed=13)
    for i in range(350, 790):
        blk, at = c.slot(0, i)
        c.v[blk, at, 0, i % 64] = float("inf")
    check(PA.paged_window_attention(*c.args(), 60, 2), c.window_oracle(60, 2))


def test_large_scores(PA):
    """Scores far apart: the running maximum moves by more than the exponential's range, up and down."""
    c = Case([(16, 2000), (200, 1000)], 2, 2, 128, 16, F16, seed=17)
    c.q *= 8
    for step in (2.0, 0.5):
        grow = step ** (torch.arange(2000) // 128).clamp(max=6).float()
        for b in range(2):
            for i in range(int(c.ctx[b])):
                blk, at = c.slot(b, i)
                c.k[blk, at] *= float(grow[i])
        m = tree(c)
        check(PA.paged_tree_attention(*c.args(), m), c.tree_oracle(m), f"tree {step}")
        check(PA.paged_window_attention(*c.args(), 700, 8), c.window_oracle(700, 8), f"window {step}")


def test_bad_tables_and_offsets(PA):
    """Entries outside the pool read as zeros, offsets and lengths outside the
    rows are skipped; each is recorded, and nothing else is touched."""
    from nanopointllm_b200 import _lib
    c = Case([(5, 100), (6, 200)], 4, 2, 128, 16, F16, seed=19)
    m = tree(c)
    c.bt[0, 2] = c.k.shape[0]
    got = PA.paged_tree_attention(*c.args(), m)
    torch.cuda.synchronize()
    with pytest.raises(_lib.NplTimeout):
        _lib.device_status()
    saved_k, saved_v = c.k, c.v
    c.k = torch.cat([c.k, torch.zeros_like(c.k[:1])])
    c.v = torch.cat([c.v, torch.zeros_like(c.v[:1])])
    check(got, c.tree_oracle(m))
    c.k, c.v, c.bt[0, 2] = saved_k, saved_v, 0
    room = c.bt.shape[1] * 16
    for field, value in (("offs", -1), ("offs", c.total - 5), ("new", 7), ("ctx", 3), ("ctx", -1), ("ctx", -2 ** 31),
                         ("ctx", room + 1), ("ctx", 2 ** 31 - 1), ("new", 2 ** 31 - 1), ("offs", 2 ** 31 - 1)):
        t = getattr(c, field)
        keep = int(t[1])
        t[1] = value
        out = torch.full_like(c.q, 3.0)
        PA.paged_tree_attention(*c.args(), m, max_q_len=6, out=out)
        torch.cuda.synchronize()
        with pytest.raises(_lib.NplTimeout):
            _lib.device_status()
        t[1] = keep
        assert (out[5:] == (0.0 if value == 3 else 3.0)).all(), field
        out, tol = out, c.tree_oracle(m)
        tol[1][5:] = np.nan
        check(out, tol, field)


def test_no_rows(PA):
    c = Case([(3, 40), (2, 50)], 4, 2, 64, 16, F16)
    a = list(c.args())
    none = torch.zeros(0, dtype=torch.int32, device="cuda")
    assert PA.paged_window_attention(a[0][:0], a[1], a[2], a[3][:0], none, None, None, 1.0, 2, 5).shape == (0, 4, 64)
    a[5] = torch.zeros_like(a[5])
    out = torch.full_like(c.q, 2.0)
    PA.paged_window_attention(*a, 5, 1, out=out)
    PA.paged_window_attention(*a, 5, 1, max_q_len=7, out=out)
    PA.paged_tree_attention(*a, tree(c), max_q_len=3, out=out)
    assert (out == 2).all()


def test_graphs_streams_and_calls_at_once(PA):
    """Two captured graphs replayed at once on two streams, beside eager calls:
    equal bits each time; a captured call reads the lengths of the replay."""
    tc = Case([(24, 600), (9, 1300)], 8, 4, 128, 16, F16, seed=23)
    wc = Case([(1, 2000), (1, 300), (1, 0)], 8, 8, 128, 256, F16, seed=24)
    m = tree(tc)
    ta, wa = tc.args(), list(wc.args())
    wa[5] = wa[6] = None
    t_ref = PA.paged_tree_attention(*ta, m, max_q_len=24)
    w_ref = PA.paged_window_attention(*wa, 512, 4)
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    graphs = []
    for s, fn in ((s1, lambda: PA.paged_tree_attention(*ta, m, max_q_len=24)),
                  (s2, lambda: PA.paged_window_attention(*wa, 512, 4))):
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            fn()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            out = fn()
        graphs.append((g, s, out))
    torch.cuda.synchronize()
    for _ in range(20):
        for g, s, out in graphs:
            with torch.cuda.stream(s):
                out.zero_()
                g.replay()
        e1, e2 = PA.paged_tree_attention(*ta, m, max_q_len=24), PA.paged_window_attention(*wa, 512, 4)
        torch.cuda.synchronize()
        assert torch.equal(graphs[0][2], t_ref) and torch.equal(graphs[1][2], w_ref)
        assert torch.equal(e1, t_ref) and torch.equal(e2, w_ref)
    wa[4].copy_(torch.tensor([1500, 1, 299], dtype=torch.int32))
    wc.ctx = torch.tensor([1500, 1, 299], dtype=torch.int32)
    wc.bt[2] = wc.bt[1]
    wa[3].copy_(wc.bt)
    graphs[1][0].replay()
    torch.cuda.synchronize()
    check(graphs[1][2], wc.window_oracle(512, 4))


def test_far_slots(PA):
    """Cache slots whose offsets pass 32 bits."""
    bs, hkv, d = 256, 8, 128
    nb = (1 << 32) // (bs * hkv * d) + 9  # elements past 2^32
    k = torch.empty(nb, bs, hkv, d, dtype=F16, device="cuda")
    v = torch.empty_like(k)
    c = Case([(4, 500), (1, 700)], 16, 8, 128, bs, F16, seed=29)
    move = {int(p): nb - 1 - i for i, p in enumerate(c.bt[c.bt >= 0].unique())}
    for p, to in move.items():
        k[to], v[to] = c.k[p], c.v[p]
    far = c.bt.clone()
    for p, to in move.items():
        far[c.bt == p] = to
    a = list(c.args())
    m = tree(c)
    near_t, near_w = PA.paged_tree_attention(*a, m), PA.paged_window_attention(*a, 300, 4)
    check(near_t, c.tree_oracle(m))
    a[1], a[2], a[3] = k, v, far.cuda()
    assert torch.equal(PA.paged_tree_attention(*a, m), near_t)
    assert torch.equal(PA.paged_window_attention(*a, 300, 4), near_w)


def test_repeats_bit_for_bit(PA):
    c = Case([(64, 3000), (10, 200)], 8, 2, 128, 16, BF16, seed=31)
    m = tree(c)
    first = PA.paged_tree_attention(*c.args(), m), PA.paged_window_attention(*c.args(), 500, 4)
    for _ in range(5):
        assert torch.equal(PA.paged_tree_attention(*c.args(), m), first[0])
        assert torch.equal(PA.paged_window_attention(*c.args(), 500, 4), first[1])


def test_written_just_before(PA):
    """Inputs that the kernel before, on the same stream, has written."""
    c = Case([(16, 1000)] * 4, 8, 8, 128, 16, F16, seed=37)
    m = tree(c)
    a = list(c.args())
    want = PA.paged_tree_attention(*a, m, max_q_len=16)
    q0, k0, v0 = a[0].clone(), a[1].clone(), a[2].clone()
    for _ in range(10):
        for t in a[:3]:
            t.zero_()
        torch.cuda.synchronize()
        a[0].copy_(q0), a[1].copy_(k0), a[2].copy_(v0)
        assert torch.equal(PA.paged_tree_attention(*a, m, max_q_len=16), want)


def test_mask_from_parents(PA):
    """On the GPU as on the CPU: ancestors and the draft itself."""
    g = torch.Generator().manual_seed(1)
    lens, parents = [7, 1, 20, 5], []
    for n in lens:
        parents += [int(torch.randint(-1, i, (1,), generator=g)) if i else -1 for i in range(n)]
    offs = torch.tensor([0, 7, 8, 28], dtype=torch.int32)
    p = torch.tensor(parents)
    cpu = PA.tree_mask_from_parents(p, offs, 20)
    gpu = PA.tree_mask_from_parents(p.cuda(), offs.cuda(), 20)
    assert torch.equal(cpu, gpu.cpu())


@pytest.mark.parametrize("new,heads", [(20, 2), (90, 2), (150, 2)])
def test_scores_of_minus_infinity(PA, new, heads):
    """Keys whose scores are all minus infinity count as unseen: rows of nothing else give zeros."""
    c = Case([(new, new + 300)], heads, heads, 64, 16, BF16, seed=41)
    c.q.abs_()
    c.k[...] = -float("inf")
    got = PA.paged_window_attention(*c.args(), 200, 4)
    assert (got == 0).all()
    blk, at = c.slot(0, new + 150)
    c.k[blk, at] = 0.25  # seen by the rows from new + 150 on
    got = PA.paged_window_attention(*c.args(), 200, 4)
    first = max(0, 150 - 300 + new)
    assert (got[:first] == 0).all() and first < new
    assert (got[first:] == c.v[blk, at]).all()


def test_many_bad_values_over_a_long_context(PA):
    """The rare path is bounded: every key in tiles that are seen in part is bad, beside a long context."""
    c = Case([(300, 12000), (3, 9000)], 2, 1, 128, 16, F16, seed=43)
    m = tree(c)
    for b, (n, ctx) in enumerate(c.seqs):
        for i in range(ctx - n, ctx):
            blk, at = c.slot(b, i)
            c.v[blk, at, 0, i % 128] = float("nan")
    check(PA.paged_tree_attention(*c.args(), m), c.tree_oracle(m))


def test_first_call_in_a_capture(cuda_device):
    """A process whose first call of each operator is captured into a graph."""
    import subprocess
    import sys
    from conftest import REPO
    code = """
import sys; sys.path.insert(0, 'tests')
import conftest, torch
from nanopointllm_b200 import logprobs, paged_attention as PA
from test_masked_attention_gpu import Case, check, tree
c = Case([(9, 900), (20, 300)], 4, 2, 128, 16, torch.float16)
a, m = c.args(), tree(c)
x, ids = torch.randn(3, 5000, device='cuda'), torch.zeros(3, dtype=torch.int64, device='cuda')
torch.cuda.synchronize()
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    t = PA.paged_tree_attention(*a, m, max_q_len=20)
    w = PA.paged_window_attention(*a, 100, 4, max_q_len=20)
    r = logprobs.token_logprobs(x, ids, 4)
g.replay()
torch.cuda.synchronize()
check(t, c.tree_oracle(m))
check(w, c.window_oracle(100, 4))
assert torch.equal(r.top_ids, x.topk(4).indices)
"""
    subprocess.run([sys.executable, "-c", code], cwd=REPO, check=True, timeout=300)


def test_bad_values_ahead_of_full_tiles(PA):
    """Sequences whose tiles need no cleaning behind ones with a bad value that one of two tokens sees: the warp that
    cleans may run ahead through all of them."""
    first = 148
    c = Case([(2, 130)] * first + [(1, 128)] * (9 * first), 1, 1, 64, 128, F16, seed=47)
    for b in range(first):
        blk, at = c.slot(b, 129)
        c.v[blk, at, 0, b % 64] = float("inf")
    check(PA.paged_window_attention(*c.args(), 1000, 0), c.window_oracle(1000, 0))


@pytest.mark.parametrize("dtype", [F16, BF16], ids=["fp16", "bf16"])
@pytest.mark.parametrize("new,before", [(12, 400), (20, 400), (40, 400), (150, 400), (300, 300), (40, 6000)])
def test_scores_that_are_no_numbers(PA, new, before, dtype):
    """A key that is NaN or infinite makes the rows that see it with a score of NaN or plus infinity NaN as a whole,
    wherever it stands in its tile; a score of minus infinity has no weight."""
    for i, bad in enumerate([float("nan"), float("inf"), -float("inf")]):
        c = Case([(new, new + before)], 4, 2, 128, 16, dtype, seed=51 + i)
        for place in range(8):
            blk, at = c.slot(0, before + place)  # some rows of a window of 60 see it, others do not
            keep = c.k[blk, at].clone()
            c.k[blk, at, place % 2, 3] = bad
            for what, got, want in (
                    ("window", PA.paged_window_attention(*c.args(), 60, 4), c.window_oracle(60, 4)),
                    ("all", PA.paged_window_attention(*c.args(), 1 << 20, 0), c.window_oracle(1 << 20, 0))):
                none = np.isnan(want[0])
                assert none.any() and not none.all()
                assert np.isnan(got.float().cpu().numpy()[none]).all(), (what, bad, place)
                check(got, want, f"{what}, {bad} at {place}")
            c.k[blk, at] = keep


@pytest.mark.parametrize("bad", [12, 72])
@pytest.mark.parametrize("Hkv,D", [(1, 64), (5, 128)])
def test_bad_values_of_a_stream_that_falls_behind(PA, Hkv, D, bad):
    """Sequences of two row tiles, whose bad values only the second tile's rows see, ahead of many sequences of one:
    the first tile's stream goes on to those while the second still adds its bad values. Few, and more than a list
    holds."""
    first, later = 148, 12 * 148
    c = Case([(200, 200)] * first + [(3, 100)] * (later if Hkv == 1 else later // 3), Hkv, Hkv, D, 16, F16, seed=53)
    for b in range(len(c.seqs)):
        for i in (range(128, 128 + bad) if b < first else [98, 99]):
            blk, at = c.slot(b, i)
            c.v[blk, at, :, (b + 5 * i) % D] = float("inf") if i % 2 else -float("inf")
    check(PA.paged_window_attention(*c.args(), 1000, 0, max_q_len=200), c.window_oracle(1000, 0))
    check(PA.paged_tree_attention(*c.args(), m := tree(c), max_q_len=200), c.tree_oracle(m))


def test_mask_of_sequences_without_drafts(PA):
    """A sequence without drafts whose offset lies inside another's rows, through the mask and the attention."""
    c = Case([(6, 200), (0, 70), (4, 90)], 4, 2, 128, 16, F16, seed=61)
    c.offs[1] = 3
    parents = torch.tensor([-1, 0, 0, 1, 2, 4, -1, 0, 1, -1])
    offs, lens = c.offs.cuda(), c.new.cuda()
    g = torch.cuda.CUDAGraph()
    p = parents.cuda()
    torch.cuda.synchronize()
    with torch.cuda.graph(g):
        m = PA.tree_mask_from_parents(p, offs, 6, lens)
    g.replay()
    assert torch.equal(m.cpu(), PA.tree_mask_from_parents(parents, torch.tensor([0, 6]), 6))
    check(PA.paged_tree_attention(*c.args(), m, max_q_len=6), c.tree_oracle(m))


@pytest.mark.parametrize("most", [150, 153, 2 ** 31 - 1])
def test_bounds_on_the_lengths(PA, most):
    """The longest length itself and bounds above it, which may select another kernel and split: each within the
    oracle's bounds. Single tokens under a loose bound too."""
    c = Case([(150, 400), (3, 90)], 4, 2, 128, 16, F16, seed=41)
    check(PA.paged_window_attention(*c.args(), 70, 4, max_q_len=most), c.window_oracle(70, 4))
    check(PA.paged_tree_attention(*c.args(), m := tree(c, cols=160 if most < 160 else c.total), max_q_len=min(most, c.total)),
          c.tree_oracle(m))
    c = Case([(1, 40 * i) for i in range(1, 65)], 4, 4, 64, 16, BF16, seed=42)
    check(PA.paged_window_attention(*c.args(), 300, 4, max_q_len=1 if most == 150 else most), c.window_oracle(300, 4))


@pytest.mark.parametrize("dtype", [F16, BF16], ids=["fp16", "bf16"])
@pytest.mark.parametrize("new,heads,kv_heads,D,ctx", [(1, 2, 2, 64, 300), (1, 8, 1, 128, 5000), (12, 4, 2, 128, 700),
                                                      (5, 3, 3, 64, 90)])
def test_probabilities_of_few_rows(PA, new, heads, kv_heads, D, ctx, dtype):
    """Single tokens and small trees (at most 32 rows of a kv head) keep the probabilities to twice the bits of their
    type. Key 0 scores 0, all others x, a single product; V is 0 and 1: every product p v of a row is off by the same
    factor, so that a p rounded once shows whole in the result. With u half a step of the type, a right one is off by
    u for the output, u^2 for p, 2 e_s + 2^-21 for scores of two fp32 steps and exp2, 2 n 2^-24 for the sums, and in
    fp16 by 2^-31 a key where the second part of p is subnormal."""
    c = Case([(new, ctx + i) for i in range(40)], heads, kv_heads, D, 16, dtype, seed=67)
    c.scale = 1.0
    g = torch.Generator().manual_seed(5)
    c.q.zero_()
    c.q[:, :, 0] = (-torch.rand(c.total, heads, generator=g) * 3 - float(np.log(ctx)) + 2).to(dtype).cuda()
    c.k.zero_()
    c.k[..., 0] = 1.0
    c.v.fill_(1.0)
    for b in range(len(c.seqs)):
        blk, at = c.slot(b, 0)
        c.k[blk, at] = 0.0
        c.v[blk, at] = 0.0
    u = O.HALF_STEP[NAME[dtype]]
    x = c.q[:, :, :1].double().abs().cpu().numpy()
    m = tree(c, density=0.5)
    for got, (out, _) in ((PA.paged_tree_attention(*c.args(), m), c.tree_oracle(m)),
                          (PA.paged_window_attention(*c.args(), 1 << 20, 0), c.window_oracle(1 << 20, 0))):
        n = ctx + 40
        tol = out * (u + u * u + 4 * 2.0 ** -23 * x + 2.0 ** -21 + 2 * n * 2.0 ** -24)
        if dtype == F16:
            tol = tol + n * 2.0 ** -31 + 2.0 ** -25
        err = np.abs(got.double().cpu().numpy() - out)
        assert (err <= tol).all(), f"{(err / tol).max()} times its bound"
