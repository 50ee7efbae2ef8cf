"""The 8-bit latent KV cache on MI355X: append, attention, eviction.

Requests whose history stays in HBM (``num_cache_tokens == 0`` on the offload
path, or a whole model's on 288 GB) can hold it in half the bytes: one row of
576 e4m3 values per token and latent head (512 latent ++ 64 rope), in pages of
128 tokens, with one fp32 scale per page and latent head.  Three operators,
registered as ``torch.ops.nanovllm_dsa.latent8_*`` next to the 16-bit ones:

* :func:`latent8_append` quantises new rows into the pages (a prompt's, a
  chunk's, or one token per request);
* :func:`latent8_attention` is absorbed-MLA attention over them: decode, a few
  rows per request (speculative verify), or a prompt's chunk, over every cached
  token or over the indexer's list; on request it adds up the attention weight
  that each cached token receives;
* :func:`latent8_evict` brings requests back under a budget: it keeps their
  most attended tokens and moves those beyond the budget into the holes.

As everywhere in this package the caller owns every buffer, calls launch on
the current stream without a host sync and can be captured into a HIP graph,
rows or pages that name nothing are skipped on the device, and a rejected call
raises ``RuntimeError``.  The reference has no counterpart: its caches are
16-bit (nanovllm/engine/model_runner.py:640-660).

Shapes (B requests, T packed rows, G latent heads, N heads, C table columns):

====================  ==========================  =======================================
latent_cache          [blocks, 128, G, 576]       float8_e4m3fn, value = code * scale
cache_scale           [blocks, G]                 float32, positive and finite
block_table           [B, C]                      int32 pages of each request
..._lengths_query     [B]                         int32 end of each request's packed rows
..._lengths_kv        [B]                         int32 cached tokens, new ones included
token_positions       [pool rows, C * 128]        int32, row ``req_pool_entries[b]``
token_weights         [pool rows, C * 128]        float32, likewise
====================  ==========================  =======================================

Two requests of one call must not share a page or a pool row that the call
writes, and the ends of packed rows must not decrease.  Packed rows behind the
last request are neither read nor written.
"""

from __future__ import annotations

from contextlib import nullcontext

import torch
from torch.autograd.graph import increment_version  # what torch's own in-place operators do to their outputs

from . import BLOCK_SIZE, CKV_DIM, KPE_DIM, _lib
from .ops import _C, _L, _pack, _stream_of, _workspace

LATENT_ROW = CKV_DIM + KPE_DIM

SCHEMAS = {
    "latent8_append": (
        "latent8_append(Tensor kv, Tensor k_rope, Tensor actual_seq_lengths_query,"
        " Tensor actual_seq_lengths_kv, Tensor block_table, Tensor(a!) latent_cache,"
        " Tensor(b!) cache_scale, Tensor? positions=None, Tensor? req_pool_entries=None,"
        " Tensor(c!)? token_positions=None, Tensor(d!)? token_weights=None) -> ()"
    ),
    "latent8_attention": (
        "latent8_attention(Tensor query_rope, Tensor query, Tensor actual_seq_lengths_query,"
        " Tensor actual_seq_lengths_kv, Tensor block_table, Tensor latent_cache, Tensor cache_scale,"
        " float scale_value, Tensor(a!) attention_out, Tensor? topk_ids=None,"
        " Tensor? req_pool_entries=None, Tensor(b!)? token_weights=None) -> ()"
    ),
    "latent8_evict": (
        "latent8_evict(Tensor actual_seq_lengths_kv, Tensor budgets, Tensor block_table,"
        " Tensor req_pool_entries, Tensor(a!) latent_cache, Tensor(b!) cache_scale,"
        " Tensor(c!) token_positions, Tensor(d!) token_weights, Tensor(e!) move_src_slots,"
        " Tensor(f!) move_dst_slots, Tensor(g!) move_counts, Tensor(h!) kept_lengths,"
        " int protect_first, int protect_last) -> ()"
    ),
}


def empty_latent_cache(blocks: int, latent_heads: int = 1, device=None) -> tuple[torch.Tensor, torch.Tensor]:
    """``(latent_cache, cache_scale)`` for that many pages; the scales are 1."""
    cache = torch.empty(blocks, BLOCK_SIZE, latent_heads, LATENT_ROW, dtype=torch.float8_e4m3fn, device=device)
    return cache, torch.ones(blocks, latent_heads, dtype=torch.float32, device=device)


def _device_of(t: torch.Tensor):
    """The tensor's device as the current one: kernels launch on its stream."""
    return nullcontext() if t.get_device() == torch.cuda.current_device() else torch.cuda.device(t.device)


def _written(*outputs) -> None:
    """Outputs count as written for autograd: a backward pass through values
    that a call overwrote is refused."""
    increment_version([t for t in outputs if t is not None])


def _append(kv, k_rope, actual_seq_lengths_query, actual_seq_lengths_kv, block_table, latent_cache, cache_scale,
            positions=None, req_pool_entries=None, token_positions=None, token_weights=None) -> None:
    buf, at = _pack(kv, k_rope, actual_seq_lengths_query, actual_seq_lengths_kv, block_table, latent_cache, cache_scale,
                    positions, req_pool_entries, token_positions, token_weights)
    with _device_of(latent_cache):
        _lib.check(_C.nvdsa_latent8_append(*at, _stream_of(latent_cache)))
    _written(latent_cache, cache_scale, token_positions, token_weights)


def _attention(query_rope, query, actual_seq_lengths_query, actual_seq_lengths_kv, block_table, latent_cache,
               cache_scale, scale_value, attention_out, topk_ids=None, req_pool_entries=None,
               token_weights=None) -> None:
    buf, at = _pack(query_rope, query, actual_seq_lengths_query, actual_seq_lengths_kv, block_table, latent_cache,
                    cache_scale, topk_ids, req_pool_entries, token_weights, attention_out)
    rows, heads = query.shape[:2] if query.dim() == 3 else (0, 0)
    ws = _workspace(latent_cache.device, _L.nvdsa_latent8_attention_workspace_size(rows, heads, token_weights is not None))
    with _device_of(latent_cache):
        _lib.check(_C.nvdsa_latent8_attention(*at[:-1], float(scale_value), at[-1], ws.data_ptr(), ws.numel(),
                                              _stream_of(latent_cache)))
    _written(attention_out, token_weights)


def _evict(actual_seq_lengths_kv, budgets, block_table, req_pool_entries, latent_cache, cache_scale, token_positions,
           token_weights, move_src_slots, move_dst_slots, move_counts, kept_lengths, protect_first,
           protect_last) -> None:
    buf, at = _pack(actual_seq_lengths_kv, budgets, block_table, req_pool_entries, latent_cache, cache_scale,
                    token_positions, token_weights, move_src_slots, move_dst_slots, move_counts, kept_lengths)
    batch, cols = block_table.shape if block_table.dim() == 2 else (0, 0)
    heads = latent_cache.shape[2] if latent_cache.dim() == 4 else 0
    ws = _workspace(latent_cache.device, _L.nvdsa_latent8_evict_workspace_size(batch, cols, heads))
    with _device_of(latent_cache):
        _lib.check(_C.nvdsa_latent8_evict(*at[:8], int(protect_first), int(protect_last), *at[8:], ws.data_ptr(),
                                          ws.numel(), _stream_of(latent_cache)))
    _written(latent_cache, cache_scale, token_positions, token_weights, move_src_slots, move_dst_slots, move_counts,
             kept_lengths)


IMPLS = {"latent8_append": _append, "latent8_attention": _attention, "latent8_evict": _evict}


def _meta(*args, **kwargs) -> None:
    return None


def _register() -> torch.library.Library:
    library = torch.library.Library("nanovllm_dsa", "FRAGMENT")
    for name, schema in SCHEMAS.items():
        library.define(schema)
        library.impl(name, IMPLS[name], "CUDA")
        library.impl(name, _meta, "Meta")
    return library


_LIBRARY = _register()


# (By the dispatcher, which resolves negated views and hands the calls to whatever
# traces or wraps tensors.)
_append_op = torch.ops.nanovllm_dsa.latent8_append.default
_attention_op = torch.ops.nanovllm_dsa.latent8_attention.default
_evict_op = torch.ops.nanovllm_dsa.latent8_evict.default


def latent8_append(kv, k_rope, actual_seq_lengths_query, actual_seq_lengths_kv, block_table, latent_cache, cache_scale,
                   *, positions=None, req_pool_entries=None, token_positions=None, token_weights=None) -> None:
    """Quantise new rows (``kv`` [T, G, 512], ``k_rope`` [T, G, 64], 16-bit)
    into the cache: row i of a request's n goes to slot
    ``actual_seq_lengths_kv - n + i``.

    A page's scale is the least power of two under which its rows' largest
    finite magnitude is at most 448; a page with older rows keeps its scale
    while that suffices, and otherwise the older codes are shifted to the
    larger one.  Infinities and NaN are stored as NaN.  With token records, the
    new slots' positions are noted (``positions`` [T]) and their weights set to
    0."""
    _append_op(kv, k_rope, actual_seq_lengths_query, actual_seq_lengths_kv, block_table, latent_cache, cache_scale,
               positions, req_pool_entries, token_positions, token_weights)


def latent8_attention(query_rope, query, actual_seq_lengths_query, actual_seq_lengths_kv, block_table, latent_cache,
                      cache_scale, scale_value, attention_out, *, topk_ids=None, req_pool_entries=None,
                      token_weights=None) -> None:
    """``attention_out[r] = softmax(scale_value * q[r] . k) . k[:512]`` over
    what row r sees: row i of a request's n sees the first
    ``actual_seq_lengths_kv - (n - 1 - i)`` slots, or, with ``topk_ids``
    [T, K], the slots of its list within them.  A row that sees nothing is
    zero.  ``query`` [T, N, 512] and ``query_rope`` [T, N, 64] are 16-bit, and
    head h attends latent head ``h // (N // G)``.

    With ``token_weights`` (and ``req_pool_entries``; not with a list) the
    attention weight of every slot, summed over the request's rows and heads,
    is added to its record."""
    _attention_op(query_rope, query, actual_seq_lengths_query, actual_seq_lengths_kv, block_table, latent_cache,
                  cache_scale, float(scale_value), attention_out, topk_ids, req_pool_entries, token_weights)


def latent8_evict(actual_seq_lengths_kv, budgets, block_table, req_pool_entries, latent_cache, cache_scale,
                  token_positions, token_weights, move_src_slots, move_dst_slots, move_counts, kept_lengths, *,
                  protect_first: int = 0, protect_last: int = 0) -> None:
    """Bring every request with more than ``budgets[b]`` cached tokens down to
    that many.

    Kept are the tokens at a position below ``protect_first`` or among the
    ``protect_last`` latest positions, then those of the largest weight, ties
    to the lower slot.  Where more tokens are protected than the budget holds,
    those at the lower slots stay, which are the earliest of a request that
    nothing was evicted from: budgets of at least ``protect_first +
    protect_last`` keep every protected token.  The kept tokens at slots >=
    budget move, in order, into the slots below it that were given up, with their positions and weights;
    the slots of a request are then in no order, which attention does not mind
    (rope is in the rows) as long as the next rows are appended behind them.
    ``move_src_slots`` / ``move_dst_slots`` [B, C * 128] and ``move_counts``
    [B] list the moves, for other caches that follow the same slots, and
    ``kept_lengths`` [B] receives the new lengths (it may be
    ``actual_seq_lengths_kv`` itself).  Of tokens on pages that name no block
    the records move but no rows."""
    _evict_op(actual_seq_lengths_kv, budgets, block_table, req_pool_entries, latent_cache, cache_scale,
              token_positions, token_weights, move_src_slots, move_dst_slots, move_counts, kept_lengths,
              int(protect_first), int(protect_last))


__all__ = ["LATENT_ROW", "empty_latent_cache", "latent8_append", "latent8_attention", "latent8_evict"]
