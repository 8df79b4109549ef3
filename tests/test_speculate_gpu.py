"""Speculative decoding through the ragged-step operators (lcr_b200.speculate):
greedy tokens are the model's own, with and without drafts, for prompts of one
token up to several chunks, slots that turn over, and pages that do not divide
the lengths; a pool too small is an error."""
import numpy as np
import pytest

import oracle
from lcr_b200 import checkpoint as ck

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
if not torch.cuda.is_available():
    pytest.skip("needs a CUDA device", allow_module_level=True)

from lcr_b200 import paged, runtime as rt, speculate as sp  # noqa: E402

MARGIN = 3e-2  # logits this close may swap places in bf16


@pytest.fixture(scope="module")
def tiny():
    block = ck.cached(ck.TINY, 0)
    return block, rt.upload_block(block)


def check_greedy(block, prompt, tokens):
    """Each token is the fp32 host evaluation's argmax, given those before it
    (or within bf16's reach of it)."""
    ref = oracle.Model(block, len(prompt) + len(tokens) + 1)
    for p, t in enumerate(prompt):
        want = ref.decode(int(t), p, oracle.MODE_FP32)
    for i, t in enumerate(tokens):
        assert want[int(t)] >= want.max() - MARGIN, i
        want = ref.decode(int(t), len(prompt) + i, oracle.MODE_FP32)


@pytest.mark.parametrize("drafts,page_size", [(0, 16), (4, 16), (3, 5), (8, 64)])
def test_greedy_tokens(tiny, drafts, page_size):
    block, wdev = tiny
    passage = [int(t) for t in ck.prompt_ids(3, 9)]
    prompts = [passage * 4, passage[:1], [int(t) for t in ck.prompt_ids(4, 70)], passage[:5] * 3, passage * 2]
    model = sp.RaggedModel(block, wdev, slots=3, max_seq=96, pages=3 * (-(-96 // page_size)), page_size=page_size)
    requests = [sp.Request(p, 12) for p in prompts]
    spec = sp.Speculator(model, drafts=drafts, chunk=32)
    spec.run(requests)
    paged.attention_status()
    for r in requests:
        assert len(r.generated) == 12 and r.accepted <= r.drafted
        check_greedy(block, r.prompt, r.generated)
    if drafts:
        # A random-init model falls into loops, which look-up drafts follow.
        assert sum(r.accepted for r in requests) > 0
    # The last step's requests gave their pages back once a step told so: run one more.
    tail = sp.Request(passage, 2)
    spec.run([tail])
    held = int(model.held.sum())
    assert int(model.free_count) + held == model.free_pages.numel()


def test_sampled_tokens_repeat_with_the_seed(tiny):
    block, wdev = tiny
    passage = [int(t) for t in ck.prompt_ids(5, 11)]

    def go(seed):
        model = sp.RaggedModel(block, wdev, slots=2, max_seq=64, pages=8)
        requests = [sp.Request(passage * 2, 10, temperature=0.9) for _ in range(3)]
        sp.Speculator(model, drafts=2, seed=seed).run(requests)
        return [r.generated for r in requests]

    a, b, c = go(1), go(1), go(2)
    assert a == b and a != c
    assert all(0 <= t < ck.TINY.vocab_size for r in a for t in r)


def test_pool_exhausted(tiny):
    block, wdev = tiny
    model = sp.RaggedModel(block, wdev, slots=2, max_seq=64, pages=3)
    with pytest.raises(MemoryError):
        sp.Speculator(model, drafts=0).run([sp.Request(list(range(40)), 4), sp.Request(list(range(30)), 4)])


def test_lookup_drafts():
    assert sp.lookup_drafts([1, 2, 3, 4, 1, 2], 3) == [3, 4, 1]
    assert sp.lookup_drafts([1, 2, 9, 1, 2, 8, 1, 2], 1) == [8]
    assert sp.lookup_drafts([1, 2, 3], 4) == [] and sp.lookup_drafts([5], 4) == []
    assert sp.lookup_drafts([7, 7, 7], 2) == [7]
