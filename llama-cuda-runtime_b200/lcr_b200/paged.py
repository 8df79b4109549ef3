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
and stream unless it is given one, which a capture has to do). Tensors must be
on torch's current device;
what does not fit raises ``ValueError`` (``csrc/tensors.cpp`` checks them and calls
the C ABI), what the library refuses ``runtime.LcrError``.
"""
from __future__ import annotations

from typing import Optional

import torch

from . import runtime as rt

try:
    from . import _tensors
except ImportError as e:  # like the library itself: no other path
    raise RuntimeError(f"lcr_b200/_tensors.so is not built; run `make -C {rt.PKG_DIR}`") from e

_lib = None


def _operators():
    """The operators, bound to the library (which has to be there)."""
    global _lib
    if _lib is None:
        rt.lib()
        _tensors.open(rt.LIB_PATH)
        _lib = _tensors
    return _lib


def plan_step(block_tables, held, free_pages, free_count, cached, new_tokens, finished=None, *, page_size: int,
              held_out, free_count_out, row_starts, kv_lengths, positions, slots, row_sequence) -> None:
    """Block tables, slot map and row map of a step from the requests' lengths
    (``lcr_plan_step``). ``block_tables`` [requests, max_pages] and
    ``free_pages`` [pool pages] are updated in place; ``held_out`` may be
    ``held`` and ``free_count_out`` ``free_count``. The step has
    ``positions.numel()`` rows at most; those left over belong to nobody."""
    status = (_lib or _operators()).plan_step(block_tables, held, free_pages, free_count, cached, new_tokens, finished,
                                              page_size, held_out, free_count_out, row_starts, kv_lengths, positions,
                                              slots, row_sequence)
    if status:
        rt.check(status)


def qk_norm_rope_kv(q_out, keys, values, qkv, positions, slots, inv_freq, q_gain=None, k_gain=None, *,
                    eps: float = 1e-5) -> None:
    """Per-head norms of q and k (where a gain is given), rotary positions and
    the cache write of the rows of ``qkv`` [rows, (heads + 2 kv_heads) *
    head_dim] (``lcr_qk_norm_rope_kv``). The pools may have any page and head
    strides; their slots are dense."""
    status = (_lib or _operators()).qk_norm_rope_kv(q_out, keys, values, qkv, positions, slots, inv_freq, q_gain, k_gain,
                                                    eps)
    if status:
        rt.check(status)


_workspaces: dict = {}


def attention_workspace(heads: int, head_dim: int, device=None) -> torch.Tensor:
    """A zeroed workspace for ``chunk_attention``."""
    return torch.zeros(rt.lib().lcr_chunk_attention_scratch_bytes(heads, head_dim), dtype=torch.uint8,
                       device=device if device is not None else torch.cuda.current_device())


def chunk_attention(out, q, keys, values, block_tables, row_starts, kv_lengths, *, scale: float,
                    workspace: Optional[torch.Tensor] = None) -> None:
    """Attention of each request's new rows (``q`` [rows, heads * head_dim],
    packed) over its pages (``lcr_chunk_attention``). Without a ``workspace``
    each stream keeps one of its own from its first call on; a call in a
    capture has to pass one, as the graph may be replayed beside calls on the
    stream that it was captured on."""
    operators = _lib or _operators()
    if workspace is None:
        if torch.cuda.is_current_stream_capturing():
            raise RuntimeError("chunk_attention: a graph needs a workspace of its own; pass a workspace")
        head_dim = keys.shape[-1] if isinstance(keys, torch.Tensor) and keys.dim() == 4 else 0
        key = (operators.current(), head_dim)
        workspace = _workspaces.get(key)
        if workspace is None:
            if head_dim in (64, 128):  # (whatever the number of heads)
                workspace = _workspaces[key] = attention_workspace(1, head_dim)
            else:  # refused below
                workspace = torch.empty(16, dtype=torch.uint8, device=torch.cuda.current_device())
    status = operators.chunk_attention(out, q, keys, values, block_tables, row_starts, kv_lengths, scale, workspace)
    if status:
        rt.check(status)


def attention_status(workspace: Optional[torch.Tensor] = None) -> None:
    """Waits for the current stream and raises what the attention calls on
    this workspace (default: the current device's and stream's) reported."""
    here = _operators().current()
    spaces = [workspace] if workspace is not None else [w for k, w in _workspaces.items() if k[0] == here]
    for w in spaces:
        rt.check(rt.lib().lcr_chunk_attention_status(w.data_ptr(), here[0]))


def token_probs(probs, logits, temperature=None, row_sequence=None) -> None:
    """Rows of fp32 logits to rows of probabilities (``lcr_token_probs``), by
    the temperature of each row, or of each row's request (zeros for a row of
    no request: an entry of ``row_sequence`` outside ``temperature``)."""
    status = (_lib or _operators()).token_probs(probs, logits, temperature, row_sequence)
    if status:
        rt.check(status)


def verify_drafts(tokens, accepted, target_probs, target_starts, drafts, draft_counts, draft_probs, uniforms) -> None:
    """Keeps each request's drafts as far as the given uniforms allow and draws
    its next token (``lcr_verify_drafts``). ``draft_probs`` [requests,
    max_drafts, vocab], or None for drafts that were certain. A request whose
    ``target_starts`` are not among ``target_probs``' rows counts as idle."""
    status = (_lib or _operators()).verify_drafts(tokens, accepted, target_probs, target_starts, drafts, draft_counts,
                                                  draft_probs, uniforms)
    if status:
        rt.check(status)
