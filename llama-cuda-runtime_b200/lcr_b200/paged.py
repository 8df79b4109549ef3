"""Ragged steps over a paged KV cache, on torch tensors (the C ABI's
``lcr_plan_step``, ``lcr_qk_norm_rope_kv``, ``lcr_chunk_attention``,
``lcr_token_probs`` and ``lcr_verify_drafts``; include/lcr_b200.h has their
definitions).

In a step every request brings its own number of new tokens -- one, a few
drafted tokens, a chunk of its prompt -- and the rows of all requests are
packed: request ``b`` owns rows ``row_starts[b]`` to ``row_starts[b + 1]``.
The cache is a pair of pools ``[pages, kv_heads, page_size, head_dim]`` and
the requests' block tables ``[requests, max_pages]``. ``speculate.py`` runs
them together.

Every function writes into tensors of the caller, on torch's current stream,
and allocates nothing (``chunk_attention`` keeps one workspace for each device
and stream unless it is given one). Tensors must be on torch's current device;
what does not fit raises ``ValueError`` (``csrc/tensors.cpp`` checks them), what
the library refuses ``runtime.LcrError``.
"""
from __future__ import annotations

import ctypes
from typing import Optional

import torch

from . import runtime as rt

try:
    from ._tensors import pointers as _pointers
except ImportError as e:  # like the library itself: no other path
    raise RuntimeError(f"lcr_b200/_tensors.so is not built; run `make -C {rt.PKG_DIR}`") from e


def _need(ok: bool, text: str) -> None:
    if not ok:
        raise ValueError(text)


def kv_view(keys, values, block_tables=None) -> rt.KvView:
    """The ``lcr_kv_view`` of a pair of pools [pages, kv_heads, page_size,
    head_dim] (any page and head strides, dense slots) and, for attention, the
    block tables."""
    k, ps, hs, v, ps2, hs2, _ = _pointers(("keys", "values"), "KK", keys, 0, values, 0)
    return _view(keys, values, k, ps, hs, v, ps2, hs2, None if block_tables is None else block_tables.data_ptr())


def _view(keys, values, k, page_stride, head_stride, v, page_stride_v, head_stride_v, table) -> rt.KvView:
    shape = keys.shape
    _need(shape == values.shape and page_stride == page_stride_v and head_stride == head_stride_v,
          "keys and values differ in shape or strides")
    _need(page_stride < 2 ** 31 and head_stride < 2 ** 31, "page and head strides must fit in 31 bits")
    return rt.KvView(k, v, table, shape[2], page_stride, head_stride, shape[1], shape[3])


_PLAN = ("block_tables", "held", "held_out", "free_pages", "free_count", "free_count_out", "cached", "new_tokens",
         "finished", "row_starts", "kv_lengths", "positions", "slots", "row_sequence")


def plan_step(block_tables, held, free_pages, free_count, cached, new_tokens, finished=None, *, page_size: int,
              held_out, free_count_out, row_starts, kv_lengths, positions, slots, row_sequence) -> None:
    """Block tables, slot map and row map of a step from the requests' lengths
    (``lcr_plan_step``). ``block_tables`` [requests, max_pages] and
    ``free_pages`` [pool pages] are updated in place; ``held_out`` may be
    ``held`` and ``free_count_out`` ``free_count``."""
    n, width = block_tables.shape
    rows = positions.numel()
    (table, h, ho, stack, count, count_out, c, new, done, starts, kv, pos, slot, seq, stream) = _pointers(
        _PLAN, "iiiiiiiiiiiiii", block_tables, n * width, held, n, held_out, n, free_pages, 1, free_count, 1,
        free_count_out, 1, cached, n, new_tokens, n, finished, n, row_starts, n + 1, kv_lengths, n, positions, rows,
        slots, rows, row_sequence, rows)
    status = rt.lib().lcr_plan_step(table, width, h, ho, stack, count, count_out, free_pages.numel(), c, new, done, n,
                                    page_size, rows, starts, kv, pos, slot, seq, stream)
    if status:
        rt.check(status)


_ROPE = ("q_out", "keys", "values", "qkv", "positions", "slots", "inv_freq", "q_gain", "k_gain")


def qk_norm_rope_kv(q_out, keys, values, qkv, positions, slots, inv_freq, q_gain=None, k_gain=None, *,
                    eps: float = 1e-5) -> None:
    """Per-head norms of q and k (where a gain is given), rotary positions and
    the cache write of the rows of ``qkv`` [rows, (heads + 2 kv_heads) *
    head_dim] (``lcr_qk_norm_rope_kv``)."""
    rows, width = qkv.shape
    pages, kv_heads, _, d = keys.shape
    heads = width // d - 2 * kv_heads
    _need(heads > 0 and width % d == 0 and q_out.shape[0] == rows and inv_freq.numel() == d // 2,
          f"qkv {tuple(qkv.shape)}, q_out {tuple(q_out.shape)} and inv_freq {tuple(inv_freq.shape)} do not fit heads "
          f"of {d} on {kv_heads} KV heads")
    (q, q_stride, k, ps, hs, v, ps2, hs2, x, x_stride, pos, slot, freq, gq, gk, stream) = _pointers(
        _ROPE, "HKKHiifhh", q_out, heads * d, keys, 0, values, 0, qkv, width, positions, rows, slots, rows, inv_freq,
        d // 2, q_gain, d, k_gain, d)
    view = _view(keys, values, k, ps, hs, v, ps2, hs2, None)
    status = rt.lib().lcr_qk_norm_rope_kv(q, q_stride, ctypes.byref(view), pages, x, x_stride, rows, heads, gq or None,
                                          gk or None, eps, freq, pos, slot, stream)
    if status:
        rt.check(status)


_workspaces: dict = {}


def attention_workspace(heads: int, head_dim: int, device=None) -> torch.Tensor:
    """A zeroed workspace for ``chunk_attention``."""
    return torch.zeros(rt.lib().lcr_chunk_attention_scratch_bytes(heads, head_dim), dtype=torch.uint8,
                       device=device if device is not None else torch.cuda.current_device())


_ATTENTION = ("out", "q", "keys", "values", "block_tables", "row_starts", "kv_lengths")


def chunk_attention(out, q, keys, values, block_tables, row_starts, kv_lengths, *, scale: float,
                    workspace: Optional[torch.Tensor] = None) -> None:
    """Attention of each request's new rows (``q`` [rows, heads * head_dim],
    packed) over its pages (``lcr_chunk_attention``)."""
    rows, width = q.shape
    n = kv_lengths.numel()
    requests, max_pages = block_tables.shape
    d = keys.shape[3]
    heads = width // d
    _need(width == heads * d and out.shape[0] == rows and requests >= n,
          f"q {tuple(q.shape)}, out {tuple(out.shape)} and block_tables {tuple(block_tables.shape)} do not fit {n} "
          f"requests and heads of {d}")
    (o, o_stride, x, x_stride, k, ps, hs, v, ps2, hs2, table, starts, kv, stream) = _pointers(
        _ATTENTION, "HHKKiii", out, width, q, width, keys, 0, values, 0, block_tables, requests * max_pages, row_starts,
        n + 1, kv_lengths, n)
    if workspace is None:
        key = (q.get_device(), stream, d)
        workspace = _workspaces.get(key)
        if workspace is None:
            workspace = _workspaces[key] = attention_workspace(heads, d)
    view = _view(keys, values, k, ps, hs, v, ps2, hs2, table)
    status = rt.lib().lcr_chunk_attention(o, o_stride, x, x_stride, ctypes.byref(view), max_pages, keys.shape[0], starts,
                                          kv, n, rows, heads, scale, workspace.data_ptr(), workspace.numel(), stream)
    if status:
        rt.check(status)


def attention_status(workspace: Optional[torch.Tensor] = None) -> None:
    """Waits for the current stream and raises what the attention calls on
    this workspace (default: the current device's and stream's) reported."""
    stream = torch.cuda.current_stream().cuda_stream
    spaces = [workspace] if workspace is not None else [
        w for k, w in _workspaces.items() if k[:2] == (torch.cuda.current_device(), stream)]
    for w in spaces:
        rt.check(rt.lib().lcr_chunk_attention_status(w.data_ptr(), stream))


_PROBS = ("probs", "logits", "temperature", "row_sequence")


def token_probs(probs, logits, temperature=None, row_sequence=None) -> None:
    """Rows of fp32 logits to rows of probabilities (``lcr_token_probs``), by
    the temperature of each row, or of each row's request (an entry of
    ``row_sequence`` past ``temperature`` is not checked)."""
    rows, vocab = logits.shape
    _need(probs.shape[0] == rows, "probs and logits have the same shape")
    p, p_stride, x, x_stride, t, seq, stream = _pointers(
        _PROBS, "FFfi", probs, vocab, logits, vocab, temperature, 1 if row_sequence is not None else rows, row_sequence,
        rows)
    status = rt.lib().lcr_token_probs(p, p_stride, x, x_stride, rows, vocab, t or None, seq or None, stream)
    if status:
        rt.check(status)


_VERIFY = ("tokens", "accepted", "target_probs", "target_starts", "drafts", "draft_counts", "draft_probs", "uniforms")


def verify_drafts(tokens, accepted, target_probs, target_starts, drafts, draft_counts, draft_probs, uniforms) -> None:
    """Keeps each request's drafts as far as the given uniforms allow and draws
    its next token (``lcr_verify_drafts``). ``draft_probs`` [requests,
    max_drafts, vocab], or None for drafts that were certain."""
    n, k = drafts.shape
    vocab = target_probs.shape[1]
    _need(tokens.shape == (n, k + 1) and uniforms.shape == tokens.shape,
          "tokens and uniforms: [requests, max_drafts + 1]")
    _need(draft_probs is None or draft_probs.shape == (n, k, vocab), "draft_probs: [requests, max_drafts, vocab]")
    t, got, p, p_stride, starts, d, counts, q, u, stream = _pointers(
        _VERIFY, "iiFiiiff", tokens, n * (k + 1), accepted, n, target_probs, vocab, target_starts, n + 1, drafts, n * k,
        draft_counts, n, draft_probs, n * k * vocab, uniforms, n * (k + 1))
    status = rt.lib().lcr_verify_drafts(t, got, p, p_stride, starts, d, counts, q or None, u, n, k, vocab, stream)
    if status:
        rt.check(status)
