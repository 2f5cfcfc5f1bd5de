"""Paged-KV operators on the GPU, mirroring ``nanopointllm.llama.paged_attention``.

* ``store_kvcache``          - paged_attention.py:353-383 (same signature)
* ``paged_decode_attention`` - paged_attention.py:872-1030 (same signature)
* ``paged_varlen_attention`` - paged_attention.py:1142-1207 (same signature;
                               causal prefill / suffix prefill from the pool)
* ``rope_store_kvcache``     - paged_attention.py:1284-1294 (rotary_fn on q/k of
                               the packed QKV projection, then store_kvcache)

Beside them, without a counterpart in the reference, on fp16 or bf16 tensors:

* ``paged_tree_attention``   - every draft of a tree of drafted tokens sees the
                               cache and the drafts that it follows
* ``tree_mask_from_parents`` - that tree's mask from each draft's parent
* ``paged_window_attention`` - causal attention with a sliding window and a few
                               first tokens that stay visible (sinks), for
                               prompts and single tokens

KV pool layout per layer (kv_pool.py:9-24): fp16 [num_blocks, block_size,
Hkv, D]; ``slot_mapping`` int32 (-1 = padding, skipped); ``block_tables`` int32
[B, max_blocks]; ``context_lens`` int32 [B]. CUDA tensors only.
"""
from __future__ import annotations

import torch

from . import _lib as L
from .fp8 import _call, _overlap


def _same_device(first: torch.Tensor, *others: torch.Tensor | None) -> None:
    d = first.get_device()
    if d < 0:
        raise ValueError("the paged path runs on CUDA tensors only")
    for t in others:
        if t is not None and t.get_device() != d:
            raise ValueError(f"tensors on different devices: {first.device} and {t.device}")


def _check_cache(k_cache: torch.Tensor, v_cache: torch.Tensor) -> None:
    if not (k_cache.is_cuda and v_cache.is_cuda):
        raise ValueError("the paged path runs on CUDA tensors only")
    if k_cache.dtype != torch.float16 or v_cache.dtype != torch.float16:
        raise ValueError("KV caches must be float16")
    if k_cache.shape != v_cache.shape or k_cache.dim() != 4:
        raise ValueError("KV caches must be [num_blocks, block_size, Hkv, D]")
    if not (k_cache.is_contiguous() and v_cache.is_contiguous()):
        raise ValueError("KV caches must be contiguous")


def store_kvcache(key: torch.Tensor, value: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                  slot_mapping: torch.Tensor) -> None:
    """Write key/value [T, Hkv, D] into the pool at ``slot_mapping`` (int32)."""
    _check_cache(k_cache, v_cache)
    t, hkv, d = key.shape
    key = key.reshape(t, hkv * d)
    value = value.reshape(t, hkv * d)
    if key.stride(-1) != 1 or value.stride(-1) != 1 or key.stride(0) != value.stride(0):
        key, value = key.contiguous(), value.contiguous()
    nb, bs = k_cache.shape[:2]
    L.check(L.lib.npl_store_kv(key.data_ptr(), value.data_ptr(), key.stride(0), t, hkv, d,
                               slot_mapping.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), nb, bs,
                               L.stream_ptr(key.device)))


def rope_store_kvcache(qkv: torch.Tensor, num_heads: int, num_kv_heads: int, head_dim: int,
                       cos_table: torch.Tensor, sin_table: torch.Tensor, positions: torch.Tensor,
                       slot_mapping: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                       q_out: torch.Tensor | None = None) -> torch.Tensor:
    """Packed QKV projection output [T, (H + 2*Hkv) * D] -> rotated q [T, H, D];
    rotated k and v stored into the pool. cos/sin: fp16 [max_position, D]."""
    _check_cache(k_cache, v_cache)
    t = qkv.shape[0]
    if q_out is None:
        q_out = torch.empty((t, num_heads, head_dim), dtype=torch.float16, device=qkv.device)
    nb, bs = k_cache.shape[:2]
    L.check(L.lib.npl_rope_store_kv(
        qkv.data_ptr(), qkv.stride(0), t, num_heads, num_kv_heads, head_dim, cos_table.data_ptr(),
        sin_table.data_ptr(), cos_table.shape[0], positions.data_ptr(), slot_mapping.data_ptr(), q_out.data_ptr(),
        k_cache.data_ptr(), v_cache.data_ptr(), nb, bs, L.stream_ptr(qkv.device)))
    return q_out


def decode_attention_workspace(device: torch.device, b: int, h: int, d: int, max_blocks: int,
                               block_size: int) -> torch.Tensor:
    nbytes = int(L.lib.npl_decode_attention_workspace_bytes(b, h, d, max_blocks, block_size))
    return L.workspaces.get(device, "decode_attention", nbytes)


def paged_decode_attention(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                           block_tables: torch.Tensor, context_lens: torch.Tensor, scale: float,
                           num_kv_groups: int, block_n: int | None = None,
                           out: torch.Tensor | None = None, quant_out: tuple | None = None) -> torch.Tensor:
    """Decode-only paged attention (q_len = 1): q fp16 [B, H, D] -> [B, H, D].

    ``block_n`` is accepted for signature compatibility with the reference
    (its Triton tile size); the kernel chooses its own context split.
    ``quant_out = (q8 int8 [B, H*D], scale fp32 [B])`` also receives the
    per-token int8 quantisation of each output row (the O projection input).
    """
    del block_n
    _check_cache(k_cache, v_cache)
    b, h, d = q.shape
    nb, bs, hkv, dk = k_cache.shape
    if dk != d or hkv * num_kv_groups != h:
        raise ValueError("q / KV cache head geometry mismatch")
    if b == 0:
        return q.new_empty((0, h, d))
    q = q.contiguous()
    if out is None:
        out = torch.empty_like(q)
    if block_tables.dtype != torch.int32 or context_lens.dtype != torch.int32:
        raise ValueError("block_tables and context_lens must be int32")
    max_blocks = block_tables.shape[1]
    ws = decode_attention_workspace(q.device, b, h, d, max_blocks, bs)
    q8, qs = quant_out if quant_out is not None else (None, None)
    L.check(L.lib.npl_paged_decode_attention(
        q.data_ptr(), b, h, hkv, d, k_cache.data_ptr(), v_cache.data_ptr(), nb, bs, block_tables.data_ptr(),
        block_tables.stride(0), max_blocks, context_lens.data_ptr(), float(scale), out.data_ptr(), L.ptr(q8),
        L.ptr(qs), ws.data_ptr(), ws.numel(), L.stream_ptr(q.device)))
    return out


def paged_varlen_attention(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                           block_tables: torch.Tensor, context_lens: torch.Tensor, q_lens: torch.Tensor,
                           q_offsets: torch.Tensor, scale: float, num_kv_groups: int,
                           block_m: int | None = None, block_n: int | None = None, *,
                           max_q_len: int | None = None, out: torch.Tensor | None = None) -> torch.Tensor:
    """Varlen paged attention for q_len > 1 prefill / suffix prefill
    (paged_attention.py:1142-1207): q fp16 [total_q, H, D] -> [total_q, H, D].

    ``block_m`` / ``block_n`` are accepted for signature compatibility with the
    reference (its Triton tile sizes); the kernel uses 128 x 128 tiles.
    ``max_q_len`` (>= every q_lens) avoids reading q_lens back to the host.
    """
    del block_m, block_n
    _check_cache(k_cache, v_cache)
    total_q, h, d = q.shape
    nb, bs, hkv, dk = k_cache.shape
    if dk != d or hkv * num_kv_groups != h:
        raise ValueError("q / KV cache head geometry mismatch")
    if total_q == 0:
        return q.new_empty((0, h, d))
    if q.dtype != torch.float16:
        raise ValueError("q must be float16")
    if q.stride(2) != 1 or q.stride(1) != d:
        q = q.contiguous()
    for t in (block_tables, context_lens, q_lens, q_offsets):
        if t.dtype != torch.int32:
            raise ValueError("block_tables, context_lens, q_lens and q_offsets must be int32")
    block_tables = block_tables if block_tables.stride(1) == 1 else block_tables.contiguous()
    context_lens, q_lens, q_offsets = context_lens.contiguous(), q_lens.contiguous(), q_offsets.contiguous()
    if out is None:
        out = torch.empty((total_q, h, d), dtype=torch.float16, device=q.device)
    if max_q_len is None:
        max_q_len = int(q_lens.max().item()) if q_lens.numel() else 0
    L.check(L.lib.npl_paged_prefill_attention(
        q.data_ptr(), q.stride(0), total_q, h, hkv, d, k_cache.data_ptr(), v_cache.data_ptr(), nb, bs,
        block_tables.data_ptr(), block_tables.stride(0), block_tables.shape[1], context_lens.data_ptr(),
        q_lens.data_ptr(), q_offsets.data_ptr(), q_lens.numel(), int(max_q_len), float(scale), out.data_ptr(),
        out.stride(0), L.stream_ptr(q.device)))
    return out



_DT16 = {torch.float16: L.NPL_F16, torch.bfloat16: L.NPL_BF16}
_tree_attention, _window_attention = L.lib.npl_paged_tree_attention, L.lib.npl_paged_window_attention


def _masked_arguments(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, block_tables: torch.Tensor,
                      context_lens: torch.Tensor, q_lens: torch.Tensor | None, q_offsets: torch.Tensor | None,
                      num_kv_groups: int, max_q_len: int | None, out: torch.Tensor | None,
                      mask: torch.Tensor | None = None):
    """Checks what tree and window attention share. Returns (the C entries'
    leading arguments up to max_q_len, out and its stride, the tensors that
    they point to). Few steps: a call on single tokens is bound by the host."""
    _same_device(q, k_cache, v_cache, block_tables, context_lens, q_lens, q_offsets, mask, out)
    dt = q.dtype
    code = _DT16.get(dt)
    if code is None:
        raise ValueError("q must be float16 or bfloat16")
    if k_cache.dtype is not dt or v_cache.dtype is not dt:
        raise ValueError("KV caches must have the type of q")
    shape = k_cache.shape
    if len(shape) != 4 or v_cache.shape != shape:
        raise ValueError("KV caches must be [num_blocks, block_size, Hkv, D]")
    if not (k_cache.is_contiguous() and v_cache.is_contiguous()):
        raise ValueError("KV caches must be contiguous")
    if q.dim() != 3:
        raise ValueError("q must be [total_q, H, D]")
    total_q, h, d = q.shape
    nb, bs, hkv, dk = shape
    if dk != d or hkv * num_kv_groups != h:
        raise ValueError("q / KV cache head geometry mismatch")
    if block_tables.dtype is not torch.int32 or block_tables.dim() != 2:
        raise ValueError("block_tables must be int32 [B, max_blocks]")
    b, width = block_tables.shape
    if context_lens.dtype is not torch.int32 or context_lens.dim() != 1 or context_lens.numel() != b:
        raise ValueError("context_lens must be int32 [B]")
    if q_lens is None:
        if q_offsets is not None:
            raise ValueError("q_lens and q_offsets go together")
        if total_q != b:
            raise ValueError("without q_lens every sequence has one token: q must be [B, H, D]")
        max_q_len, lens, offsets = 1, None, None
    else:
        if q_offsets is None:
            raise ValueError("q_lens and q_offsets go together")
        for name, t in (("q_lens", q_lens), ("q_offsets", q_offsets)):
            if t.dtype is not torch.int32 or t.dim() != 1 or t.numel() != b:
                raise ValueError(f"{name} must be int32 [B]")
        q_lens, q_offsets = q_lens.contiguous(), q_offsets.contiguous()
        if max_q_len is None:
            max_q_len = int(q_lens.max().item()) if b else 0
        if not 0 <= max_q_len < 2 ** 31:
            raise ValueError("max_q_len must be at least 0, below 2^31")
        lens, offsets = q_lens.data_ptr(), q_offsets.data_ptr()
    if not q.is_contiguous():
        ld, step, one = q.stride()
        if one != 1 or step != d or ld % 8 or ld < h * d:
            q = q.contiguous()
    if q.data_ptr() % 16:
        q = q.clone(memory_format=torch.contiguous_format)
    if not block_tables.is_contiguous():
        ld, one = block_tables.stride()
        if one != 1 or ld < width:
            block_tables = block_tables.contiguous()
    ld_table = block_tables.stride(0) if b > 1 else width  # one row's stride may be anything
    context_lens = context_lens.contiguous()
    if out is None:
        ld_out = h * d
        out = torch.empty_strided((total_q, h, d), (ld_out, d, 1), dtype=dt, device=q.device)
    else:
        if out.shape != (total_q, h, d) or out.dtype is not dt:
            raise ValueError("out must have the shape and type of q")
        ld_out, step, one = out.stride()
        if total_q == 1:
            ld_out = h * d
        if out.numel() and (one != 1 or step != d or ld_out % 8 or ld_out < h * d or out.data_ptr() % 16):
            raise ValueError("out needs contiguous heads and tokens on 16-byte boundaries that do not overlap")
        if _overlap(out, q, k_cache, v_cache):
            raise ValueError("out may not overlap q or the caches")
    args = (q.data_ptr(), code, q.stride(0) if total_q > 1 else h * d, total_q, h, hkv, d, k_cache.data_ptr(), v_cache.data_ptr(), nb, bs,
            block_tables.data_ptr(), ld_table, width, context_lens.data_ptr(), lens, offsets, b,
            max_q_len)
    return args, out, ld_out, (q, block_tables, context_lens, q_lens, q_offsets)


def paged_tree_attention(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, block_tables: torch.Tensor,
                         context_lens: torch.Tensor, q_lens: torch.Tensor, q_offsets: torch.Tensor, scale: float,
                         num_kv_groups: int, tree_mask: torch.Tensor, *, max_q_len: int | None = None,
                         out: torch.Tensor | None = None) -> torch.Tensor:
    """Attention of a tree of drafted tokens: q fp16 or bf16 [total_q, H, D] ->
    [total_q, H, D]; the arguments of ``paged_varlen_attention`` and the mask.

    The rows of sequence b, q[q_offsets[b] : q_offsets[b] + q_lens[b]], are its
    drafts, and their keys and values the last q_lens[b] of the context_lens[b]
    that its block table holds. Every draft sees all keys before the drafts,
    and draft j of its sequence where ``tree_mask`` [total_q, >= max_q_len]
    (bool or uint8) says so: itself and those that it follows
    (``tree_mask_from_parents``). A draft that sees nothing gets zeros. What a
    masked slot holds, infinities and NaN included, never reaches a row that
    does not see it. Probabilities are rounded to the type of the caches where
    max_q_len times num_kv_groups is above 32; up to there twice its bits are
    kept. ``max_q_len`` (>= every q_lens) avoids reading q_lens back to the host; the
    nearer it is, the less work is looked at in vain, and a row's last bits may
    change with it. How keys are split over CTAs goes by the width of
    ``block_tables``: pass its first columns, as many as the longest context
    needs (any stride will do)."""
    if tree_mask.dtype not in (torch.bool, torch.uint8):
        raise ValueError("tree_mask must be bool or uint8")
    if q_lens is None or q_offsets is None:
        raise ValueError("tree attention needs q_lens and q_offsets")
    args, out, ld_out, _held = _masked_arguments(q, k_cache, v_cache, block_tables, context_lens, q_lens, q_offsets,
                                                 num_kv_groups, max_q_len, out, tree_mask)
    total_q, most = args[3], args[-1]
    if tree_mask.dim() != 2 or tree_mask.shape[0] != total_q or tree_mask.shape[1] < most:
        raise ValueError("tree_mask must be [total_q, at least max_q_len]")
    cols = tree_mask.shape[1]
    if tree_mask.stride(1) != 1 or (tree_mask.stride(0) < cols and total_q > 1):
        tree_mask = tree_mask.clone(memory_format=torch.contiguous_format)
    ld_mask = tree_mask.stride(0) if total_q > 1 else cols
    if total_q and most and args[-2]:
        _call(_tree_attention, out.device, *args, tree_mask.data_ptr(), ld_mask, cols, scale,
              out.data_ptr(), ld_out)
    return out


def tree_mask_from_parents(parents: torch.Tensor, q_offsets: torch.Tensor, max_q_len: int,
                           q_lens: torch.Tensor | None = None) -> torch.Tensor:
    """bool [total_q, max_q_len] for ``paged_tree_attention``: each draft sees
    itself and the drafts that it follows. ``parents`` [total_q] holds the
    place of each draft's parent within its sequence (0 to max_q_len - 1), -1
    where it follows the last token of the cache; one outside that range ends
    the path as -1 does. Parents come before their children. Rows of no sequence come out as if they belonged to the one
    before. ``q_lens`` [B] says which sequences have no drafts: their offsets, which may be any, are left out; without
    it every offset begins a sequence's rows. Elementary torch operations, on any device, none of which waits for it:
    built once per tree."""
    total = parents.shape[0]
    if parents.dim() != 1 or parents.is_floating_point() or q_offsets.dim() != 1 or max_q_len < 1:
        raise ValueError("parents must be whole numbers [total_q], q_offsets [B], max_q_len at least 1")
    if total and not q_offsets.numel():
        raise ValueError("q_offsets must hold each sequence's first row")
    if q_lens is not None:
        if q_lens.is_floating_point() or q_lens.shape != q_offsets.shape:
            raise ValueError("q_lens must be whole numbers [B], as q_offsets")
        q_offsets = torch.where(q_lens > 0, q_offsets.long(), total)  # behind all rows
    row = torch.arange(total, device=parents.device)
    order = torch.sort(q_offsets.long()).values
    first = order[(torch.searchsorted(order, row, right=True) - 1).clamp_min(0)]  # each draft's first row
    place = (row - first).clamp_(0, max_q_len - 1)
    mask = torch.zeros((total, max_q_len + 1), dtype=torch.bool, device=parents.device)
    at = place
    for _ in range(max_q_len):
        # a finished path stays where it is, in the spare last column
        done = (at < 0) | (at >= max_q_len)
        mask.scatter_(1, torch.where(done, max_q_len, at)[:, None], True)
        at = torch.where(done, at, parents.long()[(first + at).clamp(0, total - 1)])
    return mask[:, :max_q_len]


def paged_window_attention(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, block_tables: torch.Tensor,
                           context_lens: torch.Tensor, q_lens: torch.Tensor | None, q_offsets: torch.Tensor | None,
                           scale: float, num_kv_groups: int, window: int, sinks: int = 0, *,
                           max_q_len: int | None = None, out: torch.Tensor | None = None) -> torch.Tensor:
    """Causal attention with a sliding window and sinks: q fp16 or bf16
    [total_q, H, D] -> [total_q, H, D]; the arguments of
    ``paged_varlen_attention``, and ``window`` >= 1 and ``sinks`` >= 0.

    Query j of sequence b stands at position p = context_lens[b] - q_lens[b] + j
    and sees key i where i <= p and (i > p - window or i < sinks). ``q_lens`` and
    ``q_offsets`` None: q [B, H, D] holds the one new token of each sequence, as
    in ``paged_decode_attention``. Table entries of pages that no query sees are
    not read, so those pages may have been freed. What a masked slot holds,
    infinities and NaN included, never reaches a row that does not see it.
    Probabilities are rounded as in ``paged_tree_attention`` (single tokens of
    up to 32 query heads for each kv head: not, but to twice the bits of the type).
    ``max_q_len`` (>= every q_lens) avoids reading q_lens back to the host, as in
    ``paged_tree_attention``."""
    if not 1 <= window < 2 ** 31 or not 0 <= sinks < 2 ** 31:
        raise ValueError("window must be at least 1 and sinks at least 0, below 2^31")
    args, out, ld_out, _held = _masked_arguments(q, k_cache, v_cache, block_tables, context_lens, q_lens, q_offsets,
                                                 num_kv_groups, max_q_len, out)
    if args[3] and args[-1] and args[-2]:
        _call(_window_attention, out.device, *args, window, sinks, scale, out.data_ptr(), ld_out)
    return out
