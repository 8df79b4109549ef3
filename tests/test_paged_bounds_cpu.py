"""Argument checks of the ragged step's C entry points that bound what a call
may reach: they need no device."""
from lcr_b200 import runtime as rt

P = 4096  # any aligned, never dereferenced address


def test_verify_drafts_bounded_refuses():
    L = rt.lib()

    def call(tokens=P, stride=9, rows=4, k=2, vocab=9, sequences=1):
        return L.lcr_verify_drafts_bounded(tokens, P, P, stride, rows, P, P, P, None, P, sequences, k, vocab, None)
    assert call(rows=-1) == 1 and call(tokens=None) == 1 and call(stride=8) == 1 and call(k=-1) == 1
    assert call(sequences=0) == 0
