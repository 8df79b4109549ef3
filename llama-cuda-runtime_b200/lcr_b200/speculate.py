"""Speculative decoding of many requests with prompt look-up drafts, on ragged
steps over one paged cache (``paged.py``).

Every step mixes what the requests need: a chunk of a prompt, or a request's
last token with up to ``drafts`` tokens after it that its own text suggests
(what followed the last occurrence of its trailing pair of tokens). One pass
of the model scores all rows; ``verify_drafts`` keeps each request's drafts
as far as the model agrees and draws its next token, so that a request's
tokens are distributed as without drafts -- at temperature 0, they are the
greedy ones.

  python -m lcr_b200.speculate --layers 2 --requests 16 --drafts 4

Per step: ``lcr_plan_step`` (pages, slots and positions on the device); per
layer the projections (``lcr_gemm_nt``), ``lcr_qk_norm_rope_kv`` and
``lcr_chunk_attention``; then ``lcr_token_probs`` and ``lcr_verify_drafts``
on the rows that drafts are checked against. The host keeps only the token
histories and reads back the tokens kept.
"""
from __future__ import annotations

import argparse
import dataclasses
import json
import sys
import time
from typing import List, Optional, Sequence

import numpy as np
import torch

from . import checkpoint as ck
from . import paged
from . import runtime as rt


def lookup_drafts(tokens: Sequence[int], most: int) -> List[int]:
    """Up to ``most`` tokens that followed the last earlier occurrence of the
    trailing pair of ``tokens``."""
    n = len(tokens)
    for at in range(n - 3, -1, -1):
        if tokens[at] == tokens[n - 2] and tokens[at + 1] == tokens[n - 1]:
            return [int(t) for t in tokens[at + 2:at + 2 + most]]
    return []


class RaggedModel:
    """A forward pass over packed rows of many requests. ``pages`` pages of
    ``page_size`` positions are shared by ``slots`` requests of up to
    ``max_seq`` positions; a page holds its positions of every layer."""

    def __init__(self, block: ck.WeightBlock, weights_dev=None, *, slots: int, max_seq: int, pages: int,
                 page_size: int = 16):
        g = self.geom = block.geom
        self.w = weights_dev if weights_dev is not None else rt.upload_block(block, torch.cuda.current_device())
        dev = self.w.device
        at = lambda name: self.w.data_ptr() + 2 * block.offsets[name][0]  # noqa: E731
        self.embed, self.final_norm, self.lm_head = at("embed"), at("final_norm"), at(block.lm_head_group)
        self.layers = [[at(n) for n in block.layer_groups(l)] for l in range(g.num_layers)]
        self.inv_freq = torch.from_numpy(rt.rope_inv_freq(g)).to(dev)
        self.slots, self.page_size = slots, page_size
        pool = (g.num_layers, pages, g.num_kv_heads, page_size, g.head_dim)
        self.keys = torch.zeros(pool, dtype=torch.bfloat16, device=dev)
        self.values = torch.zeros(pool, dtype=torch.bfloat16, device=dev)
        i32 = lambda *shape: torch.zeros(shape, dtype=torch.int32, device=dev)  # noqa: E731
        self.tables, self.held = i32(slots, -(-max_seq // page_size)), i32(slots)
        self.free_pages = torch.arange(pages, dtype=torch.int32, device=dev)
        self.free_count = torch.full((1,), pages, dtype=torch.int32, device=dev)
        self.row_starts, self.kv_lengths = i32(slots + 1), i32(slots)

    def forward(self, tokens: torch.Tensor, cached, new_tokens, finished, wanted: torch.Tensor) -> torch.Tensor:
        """fp32 logits of the rows ``wanted`` (indices into the step's rows) of
        a step with the packed ``tokens``."""
        g, L, check = self.geom, rt.lib(), rt.check
        rows, dev = tokens.numel(), tokens.device
        s = torch.cuda.current_stream().cuda_stream
        empty = lambda *shape: torch.empty(shape, dtype=torch.bfloat16, device=dev)  # noqa: E731
        positions, slots, row_sequence = (torch.empty(rows, dtype=torch.int32, device=dev) for _ in range(3))
        paged.plan_step(self.tables, self.held, self.free_pages, self.free_count, cached, new_tokens, finished,
                        page_size=self.page_size, held_out=self.held, free_count_out=self.free_count,
                        row_starts=self.row_starts, kv_lengths=self.kv_lengths, positions=positions, slots=slots,
                        row_sequence=row_sequence)
        h, f = g.hidden_size, g.intermediate_size
        x, xn, out = empty(rows, h), empty(rows, h), empty(rows, h)
        qkv, q, attn = empty(rows, g.qkv_rows), empty(rows, g.q_dim), empty(rows, g.q_dim)
        gate_up, act = empty(rows, 2 * f), empty(rows, f)
        check(L.lcr_embedding_lookup(x.data_ptr(), self.embed, tokens.data_ptr(), rows, h, s))
        check(L.lcr_rmsnorm(xn.data_ptr(), x.data_ptr(), self.layers[0][0], rows, h, g.rms_norm_eps, s))
        for l, (_, w_qkv, w_o, post_norm, w_gate_up, w_down) in enumerate(self.layers):
            check(L.lcr_gemm_nt(qkv.data_ptr(), 0, xn.data_ptr(), w_qkv, rows, h, g.qkv_rows, s))
            paged.qk_norm_rope_kv(q, self.keys[l], self.values[l], qkv, positions, slots, self.inv_freq)
            paged.chunk_attention(attn, q, self.keys[l], self.values[l], self.tables, self.row_starts, self.kv_lengths,
                                  scale=g.head_dim ** -0.5)
            check(L.lcr_gemm_nt(out.data_ptr(), 0, attn.data_ptr(), w_o, rows, g.q_dim, h, s))
            check(L.lcr_add_residual_rmsnorm(xn.data_ptr(), x.data_ptr(), out.data_ptr(), post_norm, rows, h,
                                             g.rms_norm_eps, s))
            check(L.lcr_gemm_nt(gate_up.data_ptr(), 0, xn.data_ptr(), w_gate_up, rows, h, 2 * f, s))
            check(L.lcr_swiglu_strided(act.data_ptr(), gate_up.data_ptr(), gate_up.data_ptr() + 2 * f, rows, f, 2 * f, s))
            check(L.lcr_gemm_nt(out.data_ptr(), 0, act.data_ptr(), w_down, rows, f, h, s))
            norm = self.layers[l + 1][0] if l + 1 < g.num_layers else self.final_norm
            check(L.lcr_add_residual_rmsnorm(xn.data_ptr(), x.data_ptr(), out.data_ptr(), norm, rows, h,
                                             g.rms_norm_eps, s))
        last = xn.index_select(0, wanted)
        logits = torch.empty(last.shape[0], g.vocab_size, dtype=torch.float32, device=dev)
        check(L.lcr_gemm_nt(logits.data_ptr(), 1, last.data_ptr(), self.lm_head, last.shape[0], h, g.vocab_size, s))
        return logits


@dataclasses.dataclass
class Request:
    prompt: List[int]
    new_tokens: int
    temperature: float = 0.0
    tokens: List[int] = dataclasses.field(default_factory=list)  # prompt, then what was kept
    cached: int = 0
    drafted: int = 0
    accepted: int = 0

    @property
    def generated(self) -> List[int]:
        return self.tokens[len(self.prompt):len(self.prompt) + self.new_tokens]


class Speculator:
    """Runs requests to their ends, up to ``slots`` at a time."""

    def __init__(self, model: RaggedModel, *, drafts: int = 4, chunk: int = 512, seed: int = 0):
        self.model, self.drafts, self.chunk = model, drafts, chunk
        self.rng = torch.Generator(device=model.w.device).manual_seed(seed)
        self.slots: List[Optional[Request]] = [None] * model.slots
        self.turned = [False] * model.slots  # its last request has ended: the pages go back with the next step
        self.steps = 0

    def run(self, requests: List[Request]) -> None:
        for i, r in enumerate(requests):
            if len(r.prompt) == 0:
                raise ValueError(f"request {i} has an empty prompt")
            if not all(0 <= t < self.model.geom.vocab_size for t in r.prompt):
                raise ValueError(f"request {i} has tokens outside the vocabulary of {self.model.geom.vocab_size}")
            # (The last token needs no place in the cache.)
            longest, holds = len(r.prompt) + max(1, r.new_tokens) - 1, self.model.tables.shape[1] * self.model.page_size
            if longest > holds:
                raise ValueError(f"request {i} has up to {longest} positions; a slot's table holds {holds}")
        waiting = list(requests)
        while waiting or any(self.slots):
            for i, r in enumerate(self.slots):
                if r is None and waiting:
                    r = self.slots[i] = waiting.pop(0)
                    r.tokens, r.cached, r.drafted, r.accepted = list(r.prompt), 0, 0, 0
            self.step()

    def step(self) -> None:
        n, dev = len(self.slots), self.model.w.device
        tokens, new, counts = [], [0] * n, [0] * n
        drafts = np.zeros((n, max(1, self.drafts)), dtype=np.int32)
        wanted, target_starts = [], [0]
        for b, r in enumerate(self.slots):
            if r is not None:
                mine = r.tokens[r.cached:r.cached + self.chunk]
                if r.cached + len(mine) == len(r.tokens):  # the step reaches the request's last token
                    room = r.new_tokens - (len(r.tokens) - len(r.prompt)) - 1
                    guess = lookup_drafts(r.tokens, min(self.drafts, room)) if room > 0 else []
                    drafts[b, :len(guess)] = guess
                    counts[b] = len(guess)
                    mine = mine + guess
                    end = len(tokens) + len(mine)
                    wanted += range(end - 1 - len(guess), end)
                new[b] = len(mine)
                tokens += mine
            target_starts.append(len(wanted))
        i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=dev)  # noqa: E731
        logits = self.model.forward(i32(tokens), i32([r.cached if r else 0 for r in self.slots]), i32(new),
                                    i32([int(t) for t in self.turned]),
                                    torch.tensor(wanted, dtype=torch.int64, device=dev))
        self.turned = [False] * n
        kept = accepted = None
        if wanted:
            owner = np.repeat(np.arange(n), np.diff(target_starts))
            heat = torch.tensor([r.temperature if r else 0.0 for r in self.slots], dtype=torch.float32, device=dev)
            paged.token_probs(logits, logits, heat, i32(owner))
            out = torch.empty(n, drafts.shape[1] + 1, dtype=torch.int32, device=dev)
            got = torch.empty(n, dtype=torch.int32, device=dev)
            u = torch.rand(out.shape, generator=self.rng, device=dev)
            paged.verify_drafts(out, got, logits, i32(target_starts), i32(drafts), i32(counts), None, u)
            kept, accepted = out.cpu().numpy(), got.cpu().numpy()
        lengths = self.model.kv_lengths.cpu().numpy()
        for b, r in enumerate(self.slots):
            if r is None:
                continue
            if new[b] and lengths[b] == 0:
                raise MemoryError(f"the pool has no pages for request {b}: {new[b]} tokens at {r.cached}")
            if target_starts[b + 1] == target_starts[b]:  # more of the prompt to come
                r.cached += new[b]
                continue
            a = int(accepted[b])
            if kept[b, a] < 0:
                raise ArithmeticError(f"request {b} has nothing to draw from at {len(r.tokens) + a}: its logits are not finite")
            r.cached = len(r.tokens) + a
            r.tokens += [int(t) for t in kept[b, :a + 1]]
            r.drafted += counts[b]
            r.accepted += a
            if len(r.tokens) - len(r.prompt) >= r.new_tokens:
                self.slots[b], self.turned[b] = None, True
        self.steps += 1


def main(argv=None) -> int:
    ap = argparse.ArgumentParser(description=__doc__.split("\n")[0])
    ap.add_argument("--layers", type=int, default=0, help="override the model's layer count")
    ap.add_argument("--requests", type=int, default=16)
    ap.add_argument("--slots", type=int, default=8)
    ap.add_argument("--drafts", type=int, default=4)
    ap.add_argument("--prompt", type=int, default=256, help="prompt tokens: a repeated passage, so that drafts hit")
    ap.add_argument("--tokens", type=int, default=64, help="tokens each request decodes")
    ap.add_argument("--temperature", type=float, default=0.0)
    ap.add_argument("--json", action="store_true")
    args = ap.parse_args(argv)
    geom = ck.LLAMA_3_2_1B
    if args.layers:
        geom = dataclasses.replace(geom, num_layers=args.layers)
    block = ck.generate(geom, 1)
    longest = args.prompt + args.tokens + args.drafts + 1
    model = RaggedModel(block, slots=args.slots, max_seq=longest, pages=args.slots * -(-longest // 16))
    report = {"layers": geom.num_layers, "requests": args.requests, "slots": args.slots}
    for drafts in (0, args.drafts):
        requests = []
        for i in range(args.requests):
            passage = [int(t) for t in ck.prompt_ids(100 + i, max(2, args.prompt // 4))]
            requests.append(Request((passage * 5)[:args.prompt], args.tokens, args.temperature))
        spec = Speculator(model, drafts=drafts)
        model.free_count.fill_(model.free_pages.numel())
        model.free_pages.copy_(torch.arange(model.free_pages.numel(), dtype=torch.int32))
        model.held.zero_()
        torch.cuda.synchronize()
        t0 = time.perf_counter()
        spec.run(requests)
        torch.cuda.synchronize()
        dt = time.perf_counter() - t0
        report[f"drafts_{drafts}"] = {"steps": spec.steps, "seconds": dt,
                                      "tokens_per_second": args.requests * args.tokens / dt,
                                      "drafted": sum(r.drafted for r in requests),
                                      "accepted": sum(r.accepted for r in requests)}
    paged.attention_status()
    print(json.dumps(report) if args.json else "\n".join(f"{k}: {v}" for k, v in report.items()))
    return 0


if __name__ == "__main__":
    sys.exit(main())
