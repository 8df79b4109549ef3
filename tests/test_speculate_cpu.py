"""The host side of lcr_b200.speculate over a model of plain Python: which rows
a step brings, and what is refused."""
import types

import pytest

torch = pytest.importorskip("torch")

from lcr_b200 import paged, speculate as sp  # noqa: E402

VOCAB = 61


class Rows:
    """Stands for RaggedModel: the next token after t at position p is
    (t + p + 1) % VOCAB. A row is (request, position, token)."""

    def __init__(self, slots=2, max_seq=48, page_size=16):
        self.w = types.SimpleNamespace(device=torch.device("cpu"))
        self.geom = types.SimpleNamespace(vocab_size=VOCAB)
        self.slots, self.page_size = slots, page_size
        self.tables = torch.zeros(slots, -(-max_seq // page_size), dtype=torch.int32)
        self.kv_lengths = torch.zeros(slots, dtype=torch.int32)
        self.steps = []

    def forward(self, tokens, cached, new_tokens, finished, wanted):
        rows = []
        for b, (c, n) in enumerate(zip(cached.tolist(), new_tokens.tolist())):
            for i in range(n):
                rows.append((b, c + i, int(tokens[len(rows)])))
        assert len(rows) == tokens.numel() and all(0 <= w < len(rows) for w in wanted.tolist())
        self.kv_lengths = cached + new_tokens
        self.steps.append(rows)
        logits = torch.zeros(wanted.numel(), VOCAB)
        for i, w in enumerate(wanted.tolist()):
            logits[i, (rows[w][2] + rows[w][1] + 1) % VOCAB] = 1.0
        return logits


def greedy(prompt, n):
    t = list(prompt)
    for _ in range(n):
        t.append((t[-1] + len(t)) % VOCAB)
    return t[len(prompt):]


@pytest.fixture(autouse=True)
def plain_operators(monkeypatch):
    def verify(tokens, accepted, probs, starts, drafts, counts, draft_probs, uniforms):
        tokens.fill_(-1)
        accepted.zero_()
        for b in range(drafts.shape[0]):
            if starts[b + 1] > starts[b]:
                best = probs[starts[b + 1] - 1 - counts[b]:starts[b + 1]].argmax(1)
                while accepted[b] < counts[b] and drafts[b, accepted[b]] == best[accepted[b]]:
                    accepted[b] += 1
                tokens[b, :accepted[b] + 1] = best[:accepted[b] + 1]
                if probs[starts[b + 1] - 1 - counts[b] + accepted[b]].isnan().all():
                    tokens[b, accepted[b]] = -1

    monkeypatch.setattr(paged, "token_probs", lambda *a: None)
    monkeypatch.setattr(paged, "verify_drafts", verify)


@pytest.mark.parametrize("drafts", [0, 3])
def test_tokens_of_requests(drafts):
    model = Rows()
    requests = [sp.Request(list(range(p)), n) for p, n in ((1, 9), (20, 5), (7, 12), (40, 9))]
    sp.Speculator(model, drafts=drafts, chunk=8).run(requests)
    for r in requests:
        assert r.generated == greedy(r.prompt, r.new_tokens)


def test_an_empty_prompt_is_refused():
    """It has no last token to continue: nothing of the call runs, and the
    requests beside it stay as they were."""
    for requests in ([sp.Request([], 4)], [sp.Request([1, 2], 4), sp.Request([], 4)]):
        model = Rows()
        with pytest.raises(ValueError, match="request .*prompt"):
            sp.Speculator(model).run(requests)
        assert not model.steps and not requests[0].tokens


def test_a_request_longer_than_its_table_is_refused():
    """The last token needs no place in the cache: 48 positions hold 40 and 9."""
    sp.Speculator(Rows()).run([sp.Request([3] * 40, 9)])
    model = Rows()
    with pytest.raises(ValueError, match="request 1 .*49 positions.*48"):
        sp.Speculator(model).run([sp.Request([1], 2), sp.Request([3] * 40, 10)])
    assert not model.steps


def test_a_request_runs_again():
    r = sp.Request([5, 6, 7, 5, 6], 6)
    for drafts in (4, 0):
        sp.Speculator(Rows(), drafts=drafts).run([r])
        assert r.generated == greedy([5, 6, 7, 5, 6], 6) and (r.drafted == 0) == (drafts == 0)


def test_a_prompt_may_be_an_array():
    numpy = pytest.importorskip("numpy")
    r = sp.Request(numpy.arange(1, 6), 3)
    sp.Speculator(Rows()).run([r])
    assert r.generated == greedy([1, 2, 3, 4, 5], 3)


@pytest.mark.parametrize("token", [-1, VOCAB, 2 ** 31 - 1])
def test_a_prompt_outside_the_vocabulary_is_refused(token):
    """The embedding's table has no row for it."""
    model = Rows()
    with pytest.raises(ValueError, match="request 1 .*vocabulary"):
        sp.Speculator(model).run([sp.Request([1], 2), sp.Request([3, token, 4], 2)])
    assert not model.steps


def test_a_row_without_a_token_is_an_error():
    """Logits of NaN leave nothing to draw from: a token of -1 is not gone on
    from, and not handed out."""
    class Broken(Rows):
        def forward(self, *a):
            logits = super().forward(*a)
            return logits * float("nan") if len(self.steps) == 3 else logits

    requests = [sp.Request([1, 2], 8), sp.Request([4], 8)]
    with pytest.raises(ArithmeticError, match="request .*nothing to draw"):
        sp.Speculator(Broken(), drafts=0).run(requests)
    assert all(0 <= t < VOCAB for r in requests for t in r.tokens)
    assert [len(r.generated) for r in requests] == [2, 2]
