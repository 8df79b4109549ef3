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
and stream unless it is given one). Tensors must be on torch's current
device; int32 ones contiguous.
"""
from __future__ import annotations

import ctypes
from typing import Optional

import torch

from . import runtime as rt

_I32 = torch.int32
_BF16 = torch.bfloat16
_F32 = torch.float32


def _need(ok: bool, text: str) -> None:
    if not ok:
        raise ValueError(text)


def _vector(t, n: int, name: str) -> int:
    """Pointer of a contiguous int32 tensor of at least n elements."""
    if t.dtype is not _I32 or not t.is_cuda or not t.is_contiguous() or t.numel() < n:
        raise ValueError(f"{name}: a contiguous int32 CUDA tensor of {n} elements, got {t.dtype} {tuple(t.shape)} "
                         f"on {t.device}")
    return t.data_ptr()


def _rows(t, dtype, name: str) -> int:
    """Pointer of a 2-D tensor whose rows are dense."""
    if t.dtype is not dtype or not t.is_cuda or t.dim() != 2 or (t.stride(1) != 1 and t.shape[1] > 1):
        raise ValueError(f"{name}: a CUDA tensor of dense {dtype} rows, got {t.dtype} {tuple(t.shape)} with strides "
                         f"{t.stride()} on {t.device}")
    return t.data_ptr()


def _stream(t) -> int:
    if t.device.index != torch.cuda.current_device():
        raise ValueError(f"tensors are on {t.device}, the current device is cuda:{torch.cuda.current_device()}")
    return torch.cuda.current_stream().cuda_stream


def kv_view(keys, values, block_tables=None) -> rt.KvView:
    """The ``lcr_kv_view`` of a pair of pools [pages, kv_heads, page_size,
    head_dim] (any page and head strides, dense slots) and, for attention, the
    block tables."""
    s = keys.stride()
    if (keys.dtype is not _BF16 or values.dtype is not _BF16 or not keys.is_cuda or keys.dim() != 4
            or keys.shape != values.shape or s != values.stride() or s[3] != 1 or s[2] != keys.shape[3]):
        raise ValueError(f"keys and values: bf16 CUDA pools [pages, kv_heads, page_size, head_dim] with dense slots and "
                         f"equal strides, got {keys.dtype} {tuple(keys.shape)} {s} and {values.dtype} "
                         f"{tuple(values.shape)} {values.stride()}")
    _need(s[0] < 2 ** 31 and s[1] < 2 ** 31, "page and head strides must fit in 31 bits")
    return rt.KvView(keys.data_ptr(), values.data_ptr(), None if block_tables is None else block_tables.data_ptr(),
                     keys.shape[2], s[0], s[1], keys.shape[1], keys.shape[3])


def plan_step(block_tables, held, free_pages, free_count, cached, new_tokens, finished=None, *, page_size: int,
              held_out, free_count_out, row_starts, kv_lengths, positions, slots, row_sequence) -> None:
    """Block tables, slot map and row map of a step from the requests' lengths
    (``lcr_plan_step``). ``block_tables`` [requests, max_pages] and
    ``free_pages`` [pool pages] are updated in place; ``held_out`` may be
    ``held`` and ``free_count_out`` ``free_count``."""
    _need(block_tables.dim() == 2, "block_tables: [requests, max_pages]")
    n, width = block_tables.shape
    rows = positions.numel()
    rt.check(rt.lib().lcr_plan_step(
        _vector(block_tables, n * width, "block_tables"), width, _vector(held, n, "held"),
        _vector(held_out, n, "held_out"), _vector(free_pages, 1, "free_pages"), _vector(free_count, 1, "free_count"),
        _vector(free_count_out, 1, "free_count_out"), free_pages.numel(), _vector(cached, n, "cached"),
        _vector(new_tokens, n, "new_tokens"), None if finished is None else _vector(finished, n, "finished"), n,
        page_size, rows, _vector(row_starts, n + 1, "row_starts"), _vector(kv_lengths, n, "kv_lengths"),
        _vector(positions, rows, "positions"), _vector(slots, rows, "slots"),
        _vector(row_sequence, rows, "row_sequence"), _stream(block_tables)))


def qk_norm_rope_kv(q_out, keys, values, qkv, positions, slots, inv_freq, q_gain=None, k_gain=None, *,
                    eps: float = 1e-5) -> None:
    """Per-head norms of q and k (where a gain is given), rotary positions and
    the cache write of the rows of ``qkv`` [rows, (heads + 2 kv_heads) *
    head_dim] (``lcr_qk_norm_rope_kv``)."""
    view = kv_view(keys, values)
    d = view.head_dim
    rows, width = qkv.shape
    heads = width // d - 2 * view.num_kv_heads
    _need(heads > 0 and width % d == 0 and q_out.shape[0] == rows and q_out.shape[1] == heads * d,
          f"qkv {tuple(qkv.shape)} and q_out {tuple(q_out.shape)} do not fit heads of {d} on {view.num_kv_heads} "
          "KV heads")
    _need(inv_freq.dtype is _F32 and inv_freq.is_cuda and inv_freq.is_contiguous() and inv_freq.numel() == d // 2,
          "inv_freq: head_dim / 2 fp32 values")
    for g in (q_gain, k_gain):
        _need(g is None or (g.dtype is _BF16 and g.is_cuda and g.is_contiguous() and g.numel() == d),
              "gains: head_dim bf16 values")
    rt.check(rt.lib().lcr_qk_norm_rope_kv(
        _rows(q_out, _BF16, "q_out"), q_out.stride(0), ctypes.byref(view), keys.shape[0], _rows(qkv, _BF16, "qkv"),
        qkv.stride(0), rows, heads, None if q_gain is None else q_gain.data_ptr(),
        None if k_gain is None else k_gain.data_ptr(), eps, inv_freq.data_ptr(), _vector(positions, rows, "positions"),
        _vector(slots, rows, "slots"), _stream(qkv)))


_workspaces: dict = {}


def attention_workspace(heads: int, head_dim: int, device=None) -> torch.Tensor:
    """A zeroed workspace for ``chunk_attention``."""
    return torch.zeros(rt.lib().lcr_chunk_attention_scratch_bytes(heads, head_dim), dtype=torch.uint8,
                       device=device if device is not None else torch.cuda.current_device())


def chunk_attention(out, q, keys, values, block_tables, row_starts, kv_lengths, *, scale: float,
                    workspace: Optional[torch.Tensor] = None) -> None:
    """Attention of each request's new rows (``q`` [rows, heads * head_dim],
    packed) over its pages (``lcr_chunk_attention``)."""
    view = kv_view(keys, values, block_tables)
    rows, width = q.shape
    n = kv_lengths.numel()
    heads = width // view.head_dim
    _need(width == heads * view.head_dim and out.shape == q.shape, f"q {tuple(q.shape)} and out {tuple(out.shape)} do "
          f"not fit heads of {view.head_dim}")
    _need(block_tables.dim() == 2 and block_tables.shape[0] >= n, "block_tables: [requests, max_pages]")
    stream = _stream(q)
    if workspace is None:
        key = (q.device.index, stream, heads, view.head_dim)
        workspace = _workspaces.get(key)
        if workspace is None:
            workspace = _workspaces[key] = attention_workspace(heads, view.head_dim)
    _vector(block_tables, 1, "block_tables")
    rt.check(rt.lib().lcr_chunk_attention(
        _rows(out, _BF16, "out"), out.stride(0), _rows(q, _BF16, "q"), q.stride(0), ctypes.byref(view),
        block_tables.shape[1], keys.shape[0], _vector(row_starts, n + 1, "row_starts"),
        _vector(kv_lengths, n, "kv_lengths"), n, rows, heads, scale, workspace.data_ptr(), workspace.numel(), stream))


def attention_status(workspace: Optional[torch.Tensor] = None) -> None:
    """Waits for the current stream and raises what the attention calls on
    this workspace (default: the current device's and stream's) reported."""
    stream = torch.cuda.current_stream().cuda_stream
    spaces = [workspace] if workspace is not None else [
        w for k, w in _workspaces.items() if k[:2] == (torch.cuda.current_device(), stream)]
    for w in spaces:
        rt.check(rt.lib().lcr_chunk_attention_status(w.data_ptr(), stream))


def token_probs(probs, logits, temperature=None, row_sequence=None) -> None:
    """Rows of fp32 logits to rows of probabilities (``lcr_token_probs``), by
    the temperature of each row, or of each row's request."""
    _need(probs.shape == logits.shape, "probs and logits have the same shape")
    rows, vocab = logits.shape
    _need(temperature is None or (temperature.dtype is _F32 and temperature.is_cuda and temperature.is_contiguous()
                                  and (row_sequence is not None or temperature.numel() >= rows)),
          "temperature: one fp32 value for each row (or request, with row_sequence)")
    rt.check(rt.lib().lcr_token_probs(
        _rows(probs, _F32, "probs"), probs.stride(0), _rows(logits, _F32, "logits"), logits.stride(0), rows, vocab,
        None if temperature is None else temperature.data_ptr(),
        None if row_sequence is None else _vector(row_sequence, rows, "row_sequence"), _stream(logits)))


def verify_drafts(tokens, accepted, target_probs, target_starts, drafts, draft_counts, draft_probs, uniforms) -> None:
    """Keeps each request's drafts as far as the given uniforms allow and draws
    its next token (``lcr_verify_drafts``). ``draft_probs`` [requests,
    max_drafts, vocab], or None for drafts that were certain."""
    _need(drafts.dim() == 2 and tokens.dim() == 2, "drafts: [requests, max_drafts], tokens: [requests, max_drafts + 1]")
    n, k = drafts.shape
    _need(tokens.shape[0] == n and tokens.shape[1] == k + 1, "tokens: [requests, max_drafts + 1]")
    _need(uniforms.dtype is _F32 and uniforms.is_cuda and uniforms.is_contiguous() and uniforms.shape == tokens.shape,
          "uniforms: fp32 [requests, max_drafts + 1]")
    vocab = target_probs.shape[1]
    _need(draft_probs is None or (draft_probs.dtype is _F32 and draft_probs.is_cuda and draft_probs.is_contiguous()
                                  and draft_probs.shape == (n, k, vocab)), "draft_probs: fp32 [requests, max_drafts, vocab]")
    rt.check(rt.lib().lcr_verify_drafts(
        _vector(tokens, n * (k + 1), "tokens"), _vector(accepted, n, "accepted"),
        _rows(target_probs, _F32, "target_probs"), target_probs.stride(0), _vector(target_starts, n + 1, "target_starts"),
        _vector(drafts, n * k, "drafts"), _vector(draft_counts, n, "draft_counts"),
        None if draft_probs is None else draft_probs.data_ptr(), uniforms.data_ptr(), n, k, vocab, _stream(tokens)))
