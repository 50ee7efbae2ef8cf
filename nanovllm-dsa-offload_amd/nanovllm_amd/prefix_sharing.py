"""Many continuations of one prefix on the 16-bit latent cache: attention, the
rows it reads, and the pages that requests share.

Requests whose history stays in HBM (``num_cache_tokens == 0``) often continue
the same tokens: samples and beams of one prompt, conversations behind one
system prompt, questions about one document.  They can hold the prefix's pages
together, and then need, beside the operators of the other modules:

* :func:`norm_rope_append` makes a step's new cache rows (norm of the latent,
  rotation of the rope part) and writes them to their pages, and rotates, on
  request also normalises, the queries in the same pass;
* :func:`shared_prefix_attention` is absorbed-MLA attention that can read a page
  shared by a group of requests once for all of them;
* :func:`pages_branch` lets requests go on from others (a page is held by
  several until someone writes to it) and gives every request pages of its own
  for its next tokens; :func:`pages_compact` brings a cache's held pages
  together; :func:`pages_copy` does the copies that either asks for, once per
  layer.

As everywhere in this package the caller owns every buffer, calls launch on
the current stream without a host sync and can be captured into a HIP graph,
rows or pages that name nothing are skipped on the device, and a rejected call
raises ``RuntimeError``.  The reference's operators have no counterpart.

Shapes (B requests, T packed rows, N heads, C table columns, P pages):

====================  ====================  ==============================================
kv_cache, k_rope      [P, 128, 1, 512], 64  16-bit
block_table           [B, C]                int32 pages of each request, -1: none
..._lengths_query     [B]                   int32 end of each request's packed rows
..._lengths_kv        [B]                   int32 cached tokens, new ones included
page_refs             [P]                   int32 holders of each page, 0: free
====================  ====================  ==============================================

The ends of packed rows must not decrease, and count as the number of rows where
they lie past it.  Packed rows behind the last request are neither read nor
written.  A call's outputs must not overlap its inputs.
"""

from __future__ import annotations

import torch

from . import _lib
from .latent_cache import _device_of, _written
from .ops import _C, _L, _pack, _stream_of, _workspace

SCHEMAS = {
    "norm_rope_append": (
        "norm_rope_append(Tensor query, Tensor kv, Tensor cos, Tensor sin, Tensor kv_norm_weight,"
        " Tensor actual_seq_lengths_query, Tensor actual_seq_lengths_kv, Tensor block_table, Tensor(a!) k_rope,"
        " Tensor(b!) kv_cache, Tensor(c!) query_rope, Tensor? query_norm_weight=None, Tensor(d!)? query_nope=None,"
        " float eps=1e-06) -> ()"
    ),
    "shared_prefix_attention": (
        "shared_prefix_attention(Tensor query_rope, Tensor query, Tensor actual_seq_lengths_query,"
        " Tensor actual_seq_lengths_kv, Tensor block_table, Tensor k_rope, Tensor kv_cache, float scale_value,"
        " Tensor(a!) attention_out, Tensor? prefix_request_ends=None, Tensor? prefix_lengths=None) -> ()"
    ),
    "pages_branch": (
        "pages_branch(Tensor(a!) seq_lens, Tensor new_tokens, Tensor(b!) block_table, Tensor(c!) page_refs,"
        " Tensor(d!) copy_src, Tensor(e!) copy_dst, Tensor(f!) copy_tokens, Tensor(g!) missing,"
        " Tensor? parents=None) -> ()"
    ),
    "pages_compact": (
        "pages_compact(Tensor(a!) block_table, Tensor(b!) page_refs, Tensor(c!) move_src, Tensor(d!) move_dst,"
        " Tensor(e!) move_count) -> ()"
    ),
    "pages_copy": (
        "pages_copy(Tensor src_ids, Tensor dst_ids, Tensor(a!)[] caches, Tensor? tokens=None,"
        " Tensor? count=None) -> ()"
    ),
}


def _norm_rope_append(query, kv, cos, sin, kv_norm_weight, actual_seq_lengths_query, actual_seq_lengths_kv, block_table,
                      k_rope, kv_cache, query_rope, query_norm_weight=None, query_nope=None, eps=1e-6) -> None:
    buf, at = _pack(query, kv, cos, sin, kv_norm_weight, actual_seq_lengths_query, actual_seq_lengths_kv, block_table,
                    k_rope, kv_cache, query_rope, query_norm_weight, query_nope)
    with _device_of(kv_cache):
        _lib.check(_C.nvdsa_norm_rope_append(*at, float(eps), _stream_of(kv_cache)))
    _written(k_rope, kv_cache, query_rope, query_nope)


def _shared_prefix_attention(query_rope, query, actual_seq_lengths_query, actual_seq_lengths_kv, block_table, k_rope,
                             kv_cache, scale_value, attention_out, prefix_request_ends=None, prefix_lengths=None) -> None:
    buf, at = _pack(query_rope, query, actual_seq_lengths_query, actual_seq_lengths_kv, block_table, k_rope, kv_cache,
                    attention_out, prefix_request_ends, prefix_lengths)
    rows, heads = query.shape[:2] if query.dim() == 3 else (0, 0)
    groups = 0 if prefix_request_ends is None else prefix_request_ends.numel()
    ws = _workspace(kv_cache.device, _L.nvdsa_shared_prefix_attention_workspace_size(
        rows, heads, actual_seq_lengths_query.numel(), groups))
    with _device_of(kv_cache):
        _lib.check(_C.nvdsa_shared_prefix_attention(*at[:7], float(scale_value), *at[7:], ws.data_ptr(), ws.numel(),
                                                    _stream_of(kv_cache)))
    _written(attention_out)


def _pages_branch(seq_lens, new_tokens, block_table, page_refs, copy_src, copy_dst, copy_tokens, missing,
                  parents=None) -> None:
    buf, at = _pack(seq_lens, new_tokens, block_table, page_refs, copy_src, copy_dst, copy_tokens, missing, parents)
    ws = _workspace(page_refs.device, _L.nvdsa_pages_branch_workspace_size(page_refs.numel()))
    with _device_of(page_refs):
        _lib.check(_C.nvdsa_pages_branch(*at, ws.data_ptr(), ws.numel(), _stream_of(page_refs)))
    _written(seq_lens, block_table, page_refs, copy_src, copy_dst, copy_tokens, missing)


def _pages_compact(block_table, page_refs, move_src, move_dst, move_count) -> None:
    buf, at = _pack(block_table, page_refs, move_src, move_dst, move_count)
    ws = _workspace(page_refs.device, _L.nvdsa_pages_compact_workspace_size(page_refs.numel()))
    with _device_of(page_refs):
        _lib.check(_C.nvdsa_pages_compact(*at, ws.data_ptr(), ws.numel(), _stream_of(page_refs)))
    _written(block_table, page_refs, move_src, move_dst, move_count)


MOST_CACHES = 16  # of one pages_copy call


def _pages_copy(src_ids, dst_ids, caches, tokens=None, count=None) -> None:
    if not 1 <= len(caches) <= MOST_CACHES:
        raise RuntimeError(f"[nvdsa ARG] pages_copy: 1 to {MOST_CACHES} caches")
    buf, at = _pack(*caches, src_ids, dst_ids, tokens, count)
    n = len(caches)
    with _device_of(src_ids):
        _lib.check(_C.nvdsa_pages_copy(at[n], at[n + 1], at[0], n, at[n + 2], at[n + 3], _stream_of(src_ids)))
    _written(*caches)


IMPLS = {"norm_rope_append": _norm_rope_append, "shared_prefix_attention": _shared_prefix_attention,
         "pages_branch": _pages_branch,
         "pages_compact": _pages_compact, "pages_copy": _pages_copy}


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

_norm_rope_append_op = torch.ops.nanovllm_dsa.norm_rope_append.default
_shared_prefix_attention_op = torch.ops.nanovllm_dsa.shared_prefix_attention.default
_pages_branch_op = torch.ops.nanovllm_dsa.pages_branch.default
_pages_compact_op = torch.ops.nanovllm_dsa.pages_compact.default
_pages_copy_op = torch.ops.nanovllm_dsa.pages_copy.default


def norm_rope_append(query, kv, cos, sin, kv_norm_weight, actual_seq_lengths_query, actual_seq_lengths_kv, block_table,
                     k_rope, kv_cache, query_rope, *, query_norm_weight=None, query_nope=None, eps=1e-6) -> None:
    """New rows of the cache from their projection ``kv`` [T, 576], and the
    queries [T, N, nope + 64] beside them: row i of a request's n goes to slot
    ``actual_seq_lengths_kv - n + i``.

    ``kv_cache`` receives ``kv[:, :512]`` divided by its root mean square (of
    512 values, ``eps`` added to the mean) times ``kv_norm_weight`` [512],
    ``k_rope`` the rotated ``kv[:, 512:]``, and ``query_rope`` [T, N, 64] the
    rotated last 64 dims of the queries.  With ``query_norm_weight``
    [nope + 64] and ``query_nope`` [T, N, nope] every head's query is
    normalised over all its dims first, and the others written to
    ``query_nope``.  ``cos`` and ``sin`` [T, 64 or more] turn neighbouring
    pairs, as in ``dsa_indexer_query_rope_inplace``.  All tensors share the
    cache's 16-bit dtype; values are computed in fp32 and rounded once.  nope is
    a multiple of 8, up to 512."""
    _norm_rope_append_op(query, kv, cos, sin, kv_norm_weight, actual_seq_lengths_query, actual_seq_lengths_kv, block_table,
                         k_rope, kv_cache, query_rope, query_norm_weight, query_nope, float(eps))


def shared_prefix_attention(query_rope, query, actual_seq_lengths_query, actual_seq_lengths_kv, block_table, k_rope,
                            kv_cache, scale_value, attention_out, *, prefix_request_ends=None,
                            prefix_lengths=None) -> None:
    """``attention_out[r] = softmax(scale_value * q[r] . k) . k[:512]`` over the
    slots that row r sees: row i of a request's n sees the first
    ``actual_seq_lengths_kv - (n - 1 - i)``.  A row that sees nothing is zero.
    ``query`` [T, N, 512] and ``query_rope`` [T, N, 64] have the cache's dtype.
    Scores, their sums and the output's are fp32; the weights are rounded to the
    cache's 16 bits (they still sum to one), so that an output is off by half a
    step of its values' mean distance from it beside the store's half step.

    ``prefix_request_ends`` [S] and ``prefix_lengths`` [S] name the groups:
    requests ``[prefix_request_ends[s-1], prefix_request_ends[s])`` hold the same
    pages for their first ``prefix_lengths[s]`` tokens (the whole pages among
    them; what is left counts as their own).  Where that saves enough time, those
    pages are taken from the table of the first request that has rows, read once,
    and multiplied with the queries of all of them; small calls read every
    request's own.  A group's requests without rows may hold anything.
    Results are those of a call without groups, up to the order of sums and the
    rounding of the weights.
    Requests behind the last end, and a group of one, share nothing.

    What a row does not see may hold anything.  A row that sees a NaN, or a score
    of +inf, is NaN.  An infinite value under a score of -inf has no weight: its
    dims are NaN, or what the row's other keys make of them, as the work is cut."""
    _shared_prefix_attention_op(query_rope, query, actual_seq_lengths_query, actual_seq_lengths_kv, block_table, k_rope,
                                kv_cache, float(scale_value), attention_out, prefix_request_ends, prefix_lengths)


def pages_branch(seq_lens, new_tokens, block_table, page_refs, copy_src, copy_dst, copy_tokens, missing, *,
                 parents=None) -> None:
    """Rows of the batch go on from others, and get pages for their next tokens.

    With ``parents`` [B], row b takes over the table and length that row
    ``parents[b]`` had before the call (all at once: rows may swap), and
    ``page_refs`` follow; a parent that names no row (-1) leaves it empty, its
    pages given back.  Then every row gets the pages that tokens ``seq_lens[b]``
    to ``seq_lens[b] + new_tokens[b]`` fall into, as far as the table goes: new
    ones where it has none, and in the place of pages that others hold too.  A
    page with older rows of several rows that all write on, held by nobody else,
    stays with the lowest of them.  New pages are the lowest free ones, given
    out by row and column.  Pages that the rows' old tables give back are among
    them; those that a row gives up for a new one are free for the next call.

    ``copy_src`` / ``copy_dst`` / ``copy_tokens`` [B] list what
    :func:`pages_copy` has to do before the rows are written (-1, -1, 0 for a
    row without).  All rows get their pages, or, where too few are free, none
    does, and ``missing`` [1] holds the number that lacks (else 0).  The parents'
    tables and lengths have been taken over then all the same: when pages are
    free again, the call is to be repeated with ``parents=None``, or with parents
    that go by the rows as they are now (-1 gives a row's pages back)."""
    _pages_branch_op(seq_lens, new_tokens, block_table, page_refs, copy_src, copy_dst, copy_tokens, missing, parents)


def pages_compact(block_table, page_refs, move_src, move_dst, move_count) -> None:
    """Bring the held pages together at the low end: with L pages held, those at
    or behind L go, in ascending order, to the free ones below L.

    ``block_table`` and ``page_refs`` name the new places when the call returns;
    ``move_src`` / ``move_dst`` [P] and ``move_count`` [1] list the moves for
    :func:`pages_copy` and for holders outside the table."""
    _pages_compact_op(block_table, page_refs, move_src, move_dst, move_count)


def pages_copy(src_ids, dst_ids, caches, *, tokens=None, count=None) -> None:
    """Copy pages ``src_ids[k]`` to ``dst_ids[k]`` of every cache in ``caches``
    (1 to 16 tensors [P, ...]: latent rows, rope, index keys, 8-bit codes and
    scales).

    ``tokens`` [pairs]: only the first ``tokens[k]`` rows of caches
    [P, 128, ...] (of others whole pages, where there are any rows).  ``count``
    [1]: only the first ``count[0]`` pairs.  Pairs that name no page are
    skipped.  A page must not be a source and a destination of one call, nor a
    destination twice.  Pages, and the rows of caches [P, 128, ...], are whole
    multiples of 4 bytes."""
    _pages_copy_op(src_ids, dst_ids, list(caches), tokens, count)


__all__ = ["MOST_CACHES", "norm_rope_append", "pages_branch", "pages_compact", "pages_copy",
           "shared_prefix_attention"]
