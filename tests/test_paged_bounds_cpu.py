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


def test_plan_step_refuses_tables_past_31_bits():
    """Positions are 32-bit: a row of block_tables holds at most 2^31 - 1, as
    for the attention that reads it."""
    L = rt.lib()

    def call(width, ps):
        return L.lcr_plan_step(P, width, P, P, P, P, P, 4, P, P, None, 2, ps, 8, P, P, P, P, P, None)
    assert call(1 << 20, 1 << 11) == 2 and b"plan_step" in L.lcr_last_error_string()
    assert call(1 << 16, 1 << 28) == 2
