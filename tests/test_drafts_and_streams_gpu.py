"""Drafts verified as a tree, streams under a window, and scored tokens, as a
serving loop uses them: through the runner and the engine, on the tiny model.

Two attention kernels of one step agree to an fp16 ulp, and a ulp can flip an
int8 rounding of the O projection's input, which this model amplifies without a
useful bound. So the two halves are shown apart, each exactly: with attention
computed in 64 bits in every kernel's place, rounded once, the steps compared
here have equal bits (everything else of the runner is batch-invariant); and the
kernels, on what a step really passes them, stay within their derived bounds.
"""
from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import logprobs as OL
from oracle import masked_attention as OM

pytestmark = pytest.mark.gpu


@pytest.fixture
def setup(cuda_device):
    from nanopointllm_b200 import _lib, runner as R, synthetic as S
    sd = S.llama_weights(S.TINY, seed=0)

    def make(**kw):
        return R.W8A8LlamaRunner(S.TINY, sd, device=cuda_device, num_blocks=40, block_size=16, **kw)

    yield R, S, make, cuda_device
    torch.cuda.synchronize()
    _lib.device_status()


BT = torch.arange(40, dtype=torch.int32).flip(0).reshape(2, 20)


def step(R, run, dev, ids, positions, seqs, ctx, mask=None):
    """One forward; ids, positions and the places in the cache of each sequence's new tokens."""
    slots = [int(BT[b, p // 16]) * 16 + p % 16 for b, places in enumerate(seqs) for p in places]
    pos = torch.tensor(positions, device=dev)
    R.set_forward_context(R.ForwardContext(
        slot_mapping=torch.tensor(slots, dtype=torch.int32, device=dev), block_tables=BT.to(dev),
        context_lens=torch.tensor(ctx, dtype=torch.int32, device=dev), position_ids=pos,
        seq_lens=[len(p) for p in seqs], tree_mask=mask))
    try:
        return run.forward(torch.tensor(ids, device=dev), position_ids=pos)[0]
    finally:
        R.clear_forward_context()


def _seen_of(mask, offs, window, sinks):
    def of(b, n, ctx):
        if mask is not None:
            return OM.tree_seen(mask[offs[b]:offs[b] + n], n, ctx)
        return OM.window_seen(n, ctx, window, sinks)
    return of


def _oracle(args, kw, kind):
    """The oracle's (out, tol) of a call of an attention function, from the arguments it was given."""
    q, k, v, bt, ctx = (t.float().cpu().numpy() for t in args[:5])
    lens = offs = None
    window, sinks, mask = 1 << 30, 0, None
    if kind == "decode":
        scale, groups = args[5:7]
    else:
        lens, offs, scale, groups = args[5:9]
        if kind == "tree":
            mask = args[9].cpu().numpy()
        elif kind == "window":
            window, sinks = args[9:11]
    n = [1] * len(ctx) if lens is None else lens.tolist()
    o = list(range(len(ctx))) if offs is None else offs.tolist()
    seen = _seen_of(mask, o, window, sinks)
    return OM.attention(q, k, v, bt.astype(int), ctx.astype(int), n, o, scale, groups,
                        lambda b: seen(b, n[b], int(ctx[b])), "float16")


class Attention:
    """Takes the place of the runner's attention functions: exact (64 bits, rounded
    once), or the kernels themselves, each call checked against the oracle."""

    NAMES = {"paged_tree_attention": "tree", "paged_window_attention": "window", "paged_decode_attention": "decode",
             "paged_varlen_attention": "varlen"}

    def __init__(self, monkeypatch, exact):
        from nanopointllm_b200 import paged_attention as PA, w8a8 as W
        self.calls = dict.fromkeys(self.NAMES.values(), 0)
        for name, kind in self.NAMES.items():
            monkeypatch.setattr(PA, name, self.stand_in(getattr(PA, name), kind, exact, W))

    def stand_in(self, real, kind, exact, W):
        def call(*args, **kw):
            self.calls[kind] += 1
            want, tol = _oracle(args, kw, kind)
            if not exact:
                got = real(*args, **kw)
                if kind in ("tree", "window"):
                    assert (np.abs(got.double().cpu().numpy() - want) <= tol).all()
                return got
            out = torch.from_numpy(np.nan_to_num(want)).half().cuda()
            if kw.get("out") is not None:
                out = kw["out"].copy_(out)
            if kw.get("quant_out") is not None:
                q8, qs = W.dynamic_per_token_quant(out.reshape(out.shape[0], -1))
                kw["quant_out"][0].copy_(q8)
                kw["quant_out"][1].copy_(qs.reshape(-1))
            return out
        return call


def _verify(R, run, dev, prompts, parents, drafts):
    """Prefills the prompts and verifies the drafts: their logits [all drafts, V]."""
    from nanopointllm_b200 import paged_attention as PA
    n = [len(p) for p in prompts]
    step(R, run, dev, sum(prompts, []), [i for k in n for i in range(k)], [range(k) for k in n], n)
    depth = [[0] * len(p) for p in parents]
    for d, p in zip(depth, parents):
        for i, j in enumerate(p):
            d[i] = 0 if j < 0 else d[j] + 1
    sizes = [len(p) for p in parents]
    mask = PA.tree_mask_from_parents(torch.tensor(sum(parents, []), device=dev),
                                     torch.tensor([0, sizes[0]], dtype=torch.int32, device=dev), max(sizes))
    return step(R, run, dev, sum(drafts, []), [len(p) + x for p, d in zip(prompts, depth) for x in d],
                [range(k, k + m) for k, m in zip(n, sizes)], [k + m for k, m in zip(n, sizes)], mask)


PARENTS = [[-1, -1, 0, 0, 1, 2, 5], [-1, 0, 1, 1]]


def _prompts(S):
    g = torch.Generator().manual_seed(3)
    prompts = [torch.randint(0, S.TINY.vocab, (n,), generator=g).tolist() for n in (37, 90)]
    return prompts, [torch.randint(0, S.TINY.vocab, (len(p),), generator=g).tolist() for p in PARENTS]


def test_tree_step_equals_its_paths(setup, monkeypatch):
    """Every draft's logits are those of decoding its path token by token."""
    R, S, make, dev = setup
    run = make()
    attention = Attention(monkeypatch, exact=True)
    prompts, drafts = _prompts(S)
    n = [len(p) for p in prompts]
    logits = _verify(R, run, dev, prompts, PARENTS, drafts)
    assert attention.calls["tree"] == S.TINY.layers
    row = 0
    for b in (0, 1):
        for i in range(len(PARENTS[b])):
            path, j = [], i
            while j >= 0:
                path.insert(0, j)
                j = PARENTS[b][j]
            # the prompts again, which drops the drafts' keys
            step(R, run, dev, sum(prompts, []), [i for k in n for i in range(k)], [range(k) for k in n], n)
            for k, j in enumerate(path):
                ids, pos, seqs, ctx = [0, 0], [0, 0], [[300], [300]], [0, 0]  # a padding row beside it
                ids[b], pos[b], seqs[b], ctx[b] = drafts[b][j], n[b] + k, [n[b] + k], n[b] + k + 1
                out = step(R, run, dev, ids, pos, seqs, ctx)
            assert torch.equal(logits[row], out[b]), f"sequence {b}, draft {i}"
            row += 1


def test_tree_step_and_scores(setup, monkeypatch):
    """The kernels within their bounds in a step as it runs, and the scores of its
    drafts' children by which a serving loop accepts or rejects them."""
    from nanopointllm_b200 import logprobs as LP
    R, S, make, dev = setup
    run = make()
    attention = Attention(monkeypatch, exact=False)
    prompts, drafts = _prompts(S)
    logits = _verify(R, run, dev, prompts, PARENTS, drafts)
    assert attention.calls["tree"] == S.TINY.layers
    children = [next((d[c] for c, q in enumerate(p) if q == i), -1) for p, d in zip(PARENTS, drafts)
                for i in range(len(p))]
    asked = torch.tensor(children, device=dev)
    scores = LP.token_logprobs(logits, asked, top_k=3)
    lp, ent, order, top_lp, tol, ent_tol = OL.token_logprobs(logits.float().cpu().numpy(), asked.cpu().numpy(), 3)
    assert (np.abs(scores.logprobs.cpu().numpy() - lp) <= OL.value_tol(tol, lp)).all()
    assert (np.abs(scores.entropy.cpu().numpy() - ent) <= ent_tol).all()
    np.testing.assert_array_equal(scores.top_ids.cpu().numpy(), order)


@pytest.mark.parametrize("window,sinks", [(1000, 0), (40, 4), (7, 20)])
def test_window_runner(setup, monkeypatch, window, sinks):
    """The prompt's last token in a prefill has the logits of decoding it alone,
    with pages that have left the window used for other things."""
    R, S, make, dev = setup
    attention = Attention(monkeypatch, exact=True)
    g = torch.Generator().manual_seed(5)
    prompts = [torch.randint(0, S.TINY.vocab, (n,), generator=g).tolist() for n in (200, 33)]
    n = [len(p) for p in prompts]
    run = make(window=window, sinks=sinks)

    def prefill(k):
        return step(R, run, dev, sum((p[:x] for p, x in zip(prompts, k)), []), [i for x in k for i in range(x)],
                    [range(x) for x in k], k)

    whole = prefill(n)
    causal = make()
    same = step(R, causal, dev, sum(prompts, []), [i for x in n for i in range(x)], [range(x) for x in n], n)
    assert torch.equal(whole[:min(window, 200)], same[:min(window, 200)])
    assert torch.equal(whole[199], same[199]) == (window >= 200)
    run.kv_pool.zero_()
    prefill([x - 1 for x in n])
    for page in range(-(-sinks // 16), max(0, 200 - window) // 16):
        run.kv_pool[:, :, int(BT[0, page])] = float("nan")
    last = step(R, run, dev, [p[-1] for p in prompts], [x - 1 for x in n], [[x - 1] for x in n], n)
    assert torch.equal(last, whole[[199, 232]])
    assert attention.calls["window"] == 3 * S.TINY.layers


def test_window_step_within_bounds(setup, monkeypatch):
    """The kernels within their bounds in a mixed step as it runs."""
    R, S, make, dev = setup
    run = make(window=40, sinks=4)
    attention = Attention(monkeypatch, exact=False)
    g = torch.Generator().manual_seed(7)
    ids = torch.randint(0, S.TINY.vocab, (150,), generator=g).tolist()
    step(R, run, dev, ids[:120], list(range(120)) , [range(120), []], [120, 0])
    step(R, run, dev, ids[120:], [120, *range(29)], [[120], range(29)], [121, 29])  # one decodes, one is a prompt
    step(R, run, dev, [1, 2], [121, 29], [[121], [29]], [122, 30])
    assert attention.calls["window"] == 3 * S.TINY.layers


def test_window_and_tree_are_refused(setup):
    R, S, make, dev = setup
    run = make(window=64)
    mask = torch.ones(2, 1, dtype=torch.bool, device=dev)
    with pytest.raises(ValueError, match="window"):
        step(R, run, dev, [1, 2], [0, 0], [[0], [0]], [1, 1], mask)
    with pytest.raises(ValueError, match="window"):
        make(window=0)


@pytest.mark.parametrize("kw", [{}, {"window": 24, "sinks": 2}])
def test_serving_reports_scores(setup, kw):
    """The engine's scores: one for each token, the chosen token on top, the same
    whether a step was replayed from a graph or ran eagerly."""
    from nanopointllm_b200 import serving
    R, S, make, dev = setup
    run = make(**kw)
    g = torch.Generator().manual_seed(11)
    reqs = [serving.Request(rid=i, text_ids=torch.randint(0, S.TINY.vocab, (t,), generator=g).tolist(), max_tokens=m)
            for i, (t, m) in enumerate([(12, 9), (40, 5), (3, 12)])]
    a = serving.ServingEngine(run, max_blocks_per_seq=6, logprobs=4).run(reqs)
    b = serving.ServingEngine(run, max_blocks_per_seq=6, logprobs=4, use_graphs=False).run(reqs)
    c = serving.ServingEngine(run, max_blocks_per_seq=6).run(reqs)
    assert "scores" not in c and a["outputs"] == b["outputs"] == c["outputs"]
    for r in reqs:
        tokens, scores = a["outputs"][r.rid], a["scores"][r.rid]
        assert len(scores) == len(tokens) == r.max_tokens
        for t, s in zip(tokens, scores):
            assert s.top_ids[0] == t and s.top_logprobs[0] == s.logprob and len(s.top_ids) == 4
            assert s.logprob < 0 < s.entropy and s.top_logprobs == sorted(s.top_logprobs, reverse=True)
        if not kw:  # the causal kernels do not depend on the batch
            assert [s.logprob for s in scores] == [s.logprob for s in b["scores"][r.rid]]
    with pytest.raises(ValueError, match="logprobs"):
        serving.ServingEngine(run, max_blocks_per_seq=6, logprobs=33)
