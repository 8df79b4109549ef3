"""Argument checks of the ragged step's C entry points: they need no device."""
import ctypes

import pytest

from lcr_b200 import runtime as rt


@pytest.fixture(scope="module")
def L():
    return rt.lib()


P = 4096  # any aligned, never dereferenced address


def view(head_dim=64, page_size=16, kv_heads=2, page_stride=2048, head_stride=1024, table=P):
    return rt.KvView(P, P, table, page_size, page_stride, head_stride, kv_heads, head_dim)


def attention(L, v, *, q=P, q_stride=256, max_pages=4, pool=8, sequences=1, rows=1, heads=4, scratch=P, size=1 << 30):
    return L.lcr_chunk_attention(P, 256, q, q_stride, ctypes.byref(v), max_pages, pool, P, P, sequences, rows, heads, 0.1,
                                 scratch, size, None)


def test_empty_calls_do_nothing(L):
    assert attention(L, view(), rows=0) == 0 and attention(L, view(), sequences=0) == 0
    assert L.lcr_token_probs(None, 0, None, 0, 0, 5, None, 0, None, None) == 0
    assert L.lcr_verify_drafts(None, None, None, 0, None, None, None, None, None, 0, 1, 5, None) == 0
    assert L.lcr_qk_norm_rope_kv(None, 0, None, 0, None, 0, 0, 1, None, None, 0.0, None, None, None, None) == 0


@pytest.mark.parametrize("kw,status", [
    (dict(q=None), 1), (dict(scratch=None), 1), (dict(q_stride=128), 1), (dict(max_pages=0), 1), (dict(pool=0), 1),
    (dict(size=16), 1), (dict(q=P + 2), 2), (dict(q_stride=260), 2), (dict(heads=3), 2), (dict(rows=-1), 1),
    (dict(pool=1 << 28), 2), (dict(max_pages=1 << 28), 2)])
def test_attention_refuses(L, kw, status):
    assert attention(L, view(), **kw) == status
    assert b"chunk_attention" in L.lcr_last_error_string()


@pytest.mark.parametrize("v,status", [
    (dict(head_dim=96), 2), (dict(page_size=0), 1), (dict(kv_heads=0), 1), (dict(page_stride=12), 2),
    (dict(head_stride=0), 2), (dict(table=None), 1)])
def test_attention_refuses_views(L, v, status):
    assert attention(L, view(**v)) == status


def test_rope_refuses(L):
    def call(q_out=P, q_stride=256, v=None, qkv_stride=512, heads=4, gain=None, eps=1e-5):
        return L.lcr_qk_norm_rope_kv(q_out, q_stride, ctypes.byref(v or view()), 8, P, qkv_stride, 3, heads, gain, None,
                                     eps, P, P, P, None)
    assert call(q_out=None) == 1 and call(q_stride=128) == 1 and call(qkv_stride=504) == 1 and call(heads=0) == 1
    assert call(eps=-1.0) == 1 and call(gain=P + 2) == 2 and call(qkv_stride=516) == 2
    assert call(v=view(head_dim=80)) == 2


def test_plan_refuses(L):
    def call(tables=P, n=2, width=4, pool=16, ps=16, rows=8, positions=P):
        return L.lcr_plan_step(tables, width, P, P, P, P, P, pool, P, P, None, n, ps, rows, P, P, positions, P, P, None)
    assert call(tables=None) == 1 and call(n=0) == 1 and call(ps=0) == 1 and call(rows=-1) == 1
    assert call(positions=None) == 1 and call(n=8193) == 2 and call(pool=1 << 28) == 2
    assert call(n=8192, width=1 << 20) == 2


def test_probs_and_verify_refuse(L):
    assert L.lcr_token_probs(P, 5, None, 5, 1, 5, None, 0, None, None) == 1
    assert L.lcr_token_probs(P, 4, P, 5, 1, 5, None, 0, None, None) == 1
    assert L.lcr_token_probs(P, 5, P, 5, 1, 0, None, 0, None, None) == 1
    assert L.lcr_token_probs(P, 5, P, 5, 2, 5, P, 1, None, None) == 1  # fewer temperatures than rows
    assert L.lcr_token_probs(P, 5, P, 5, 2, 5, P, 0, P, None) == 1
    verify = lambda tokens=P, stride=9, k=2, vocab=9, drafts=P: L.lcr_verify_drafts(  # noqa: E731
        tokens, P, P, stride, P, drafts, P, None, P, 1, k, vocab, None)
    assert verify(tokens=None) == 1 and verify(stride=8) == 1 and verify(vocab=0) == 1 and verify(drafts=None) == 1
    assert verify(k=-1) == 1


def test_scratch_size(L):
    assert 0 < L.lcr_chunk_attention_scratch_bytes(32, 64) < 1 << 28
    assert 0 < L.lcr_chunk_attention_scratch_bytes(32, 128) < 1 << 28
