"""Cases of the operators of a ragged step over the paged KV cache: every
request brings its own number of new tokens (one, a few drafted tokens, a
chunk of its prompt), and drafted tokens are verified against the model's
probabilities.

  plan    block tables, slot map and row map of a step from request lengths
  rope    per-head norms of q and k, rotary positions, K/V into the cache
  attn    attention of each request's new rows over its pages
  probs   rows of logits to rows of probabilities
  verify  drafted tokens against the target's probabilities

Sizes: 64 slots with contexts of 128 to 4096 positions, 16-position pages,
32 query and 8 KV heads of 64 (or 128), vocabulary 128256, prompt chunks of
2048, requests of up to 32768 positions -- the continuous-batching, prefill
and long-request workloads this repository measures elsewhere -- with four
drafted tokens per request.
"""
import math
import os
import sys

import torch

own = False

DEV = "cuda"
SCALE = 2.0 ** 38  # fixed point of the verification


def _paged():
    """The framework's operators (own = True only)."""
    pkg = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "llama-cuda-runtime_b200")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    from lcr_b200 import paged

    return paged


# ---------------------------------------------------------------------------
# Cases
# ---------------------------------------------------------------------------

def listed():
    return [
        # One step of 64 slots that decode with up to four drafts each: a few
        # slots cross into a new page.
        dict(name="plan_drafts", op="plan", sequences=64, ctx_lo=128, ctx_hi=4096, new=5, chunked=0, page=16),
        # A step of 512 requests of which one in eight brings a prompt chunk
        # and one in eight has finished and hands its pages back.
        dict(name="plan_admit", op="plan", sequences=512, ctx_lo=128, ctx_hi=4096, new=2048, chunked=64, page=16),
        # The rows of one drafting step of 64 slots.
        dict(name="rope_drafts", op="rope", rows=320, heads=32, kv_heads=8, dim=64, norm=True, page=16, max_pos=4096),
        # Four prompt chunks of 2048 rows, heads of 128.
        dict(name="rope_chunks", op="rope", rows=8192, heads=32, kv_heads=8, dim=128, norm=True, page=16,
             max_pos=32768),
        # The smallest call: one request verifies four drafts on a short context.
        dict(name="attn_one", op="attn", sequences=1, new=5, chunked=0, ctx_lo=250, ctx_hi=250, heads=32, kv_heads=8,
             dim=64, page=16),
        # 64 slots, up to four drafts each, contexts of 128 to 4096.
        dict(name="attn_drafts", op="attn", sequences=64, new=5, chunked=0, ctx_lo=128, ctx_hi=4096, heads=32,
             kv_heads=8, dim=64, page=16),
        # A mixed step: one prompt chunk beside fifteen decoding requests, heads of 128.
        dict(name="attn_mixed", op="attn", sequences=16, new=509, chunked=1, ctx_lo=128, ctx_hi=3500, heads=32,
             kv_heads=8, dim=128, page=16),
        # The last chunk of the longest prompt: 2048 rows that end at position 32768.
        dict(name="attn_chunk", op="attn", sequences=1, new=2048, chunked=1, ctx_lo=30720, ctx_hi=30720, heads=32,
             kv_heads=8, dim=64, page=16),
        # One request's five rows of logits.
        dict(name="probs_one", op="probs", rows=5, vocab=128256),
        # The rows of one drafting step of 64 slots.
        dict(name="probs_drafts", op="probs", rows=320, vocab=128256),
        # One request with four drafts and the drafting model's probabilities.
        dict(name="verify_one", op="verify", sequences=1, drafts=4, vocab=128256, point=False),
        # 64 of them.
        dict(name="verify_drafts", op="verify", sequences=64, drafts=4, vocab=128256, point=False),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.5)))))))


def draw(rng):
    """One more case of the same ranges."""
    op = rng.choice(["plan", "rope", "attn", "attn", "attn", "probs", "verify", "verify"])
    page = rng.choice([8, 16, 16, 32, 64])
    heads, kv_heads = rng.choice([(32, 8), (32, 8), (4, 2), (8, 8), (16, 2), (32, 32)])
    dim = rng.choice([64, 64, 128])
    if op == "plan":
        s = _log(rng, 1, 512)
        lo = _log(rng, 1, 2048)
        return dict(op=op, sequences=s, ctx_lo=lo, ctx_hi=lo + _log(rng, 1, 2048), new=_log(rng, 1, 2048),
                    chunked=rng.randint(0, max(0, s // 8)), page=page)
    if op == "rope":
        return dict(op=op, rows=_log(rng, 1, 8192), heads=heads, kv_heads=kv_heads if heads < 32 else 8, dim=dim,
                    norm=rng.random() < 0.7, page=page, max_pos=_log(rng, 64, 32768))
    if op == "probs":
        return dict(op=op, rows=_log(rng, 1, 320), vocab=_log(rng, 8000, 128256))
    if op == "verify":
        return dict(op=op, sequences=_log(rng, 1, 64), drafts=rng.randint(1, 4), vocab=_log(rng, 8000, 128256),
                    point=rng.random() < 0.4)
    most = {k: max(work(c)[k] for c in listed()) for k in ("bytes", "flops")}
    while True:
        s = _log(rng, 1, 64)
        new = _log(rng, 1, 2048)
        lo = _log(rng, 1, 24000)
        c = dict(op=op, sequences=s, new=new, chunked=rng.randint(0, min(s, 2)) if new > 8 else 0, ctx_lo=lo,
                 ctx_hi=lo + _log(rng, 1, 8000), heads=heads, kv_heads=kv_heads, dim=dim, page=page)
        w = work(c)
        cells = s * new * heads * (c["ctx_hi"] + new)  # padded scores of the plain form
        cache = s * (c["ctx_hi"] + new) * kv_heads * dim
        if cells <= 2.2e9 and cache <= 2.0e8 and w["bytes"] <= most["bytes"] and w["flops"] <= most["flops"]:
            return c


def _lengths(case):
    """(context, new tokens) of each request, fixed by the case: contexts
    evenly spread, `chunked` requests with a whole chunk (all, when it is 0
    and the chunk is short, have 1 .. new), the rest decoding with up to four
    drafts."""
    s, new = case["sequences"], case["new"]
    ctx, got = [], []
    for i in range(s):
        ctx.append(case["ctx_lo"] + (case["ctx_hi"] - case["ctx_lo"]) * i // max(1, s - 1))
        if case["chunked"] and i % max(1, s // case["chunked"]) == 0 and i // max(1, s // case["chunked"]) < case["chunked"]:
            got.append(new)
        elif case["chunked"] or new <= 8:
            got.append(1 + (new - 1 + 3 * i) % min(new, 5))
        else:
            got.append(1 + (new - 1 + 37 * i) % new)
    return ctx, got


def work(case):
    op = case["op"]
    if op == "plan":
        ctx, new = _lengths(case)
        rows = sum(new)
        pages = sum((c + n + case["page"] - 1) // case["page"] - (c + case["page"] - 1) // case["page"]
                    for c, n in zip(ctx, new))
        return {"bytes": 4 * (6 * case["sequences"] + 3 * rows + 2 * pages), "flops": 0}
    if op == "rope":
        n = case["rows"] * (case["heads"] + 2 * case["kv_heads"]) * case["dim"]
        return {"bytes": 4 * n + 8 * case["rows"], "flops": 10 * n}
    if op == "attn":
        ctx, new = _lengths(case)
        kv = sum(c + n for c, n in zip(ctx, new)) * case["kv_heads"] * case["dim"] * 4
        rows = sum(new) * case["heads"] * case["dim"] * 4
        seen = sum(n * c + n * (n + 1) // 2 for c, n in zip(ctx, new))
        return {"bytes": kv + rows, "flops": 4 * seen * case["heads"] * case["dim"]}
    if op == "probs":
        return {"bytes": 8 * case["rows"] * case["vocab"], "flops": 4 * case["rows"] * case["vocab"]}
    # verify: one row of the target for each request, and one of the drafting
    # model for about half of them (a draft was refused); point proposals have none.
    rows = case["sequences"] * (1.0 if case["point"] else 1.5)
    return {"bytes": 4 * rows * case["vocab"], "flops": 4 * rows * case["vocab"]}


# ---------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------

def _gen(seed, salt):
    return torch.Generator(device=DEV).manual_seed((seed * 1000003 + salt) % (2 ** 62))


def _int(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def _requests(case, seed):
    """The lengths in an order of the seed."""
    ctx, new = _lengths(case)
    order = torch.randperm(case["sequences"], generator=torch.Generator().manual_seed(seed + 7)).tolist()
    return [ctx[i] for i in order], [new[i] for i in order], order


def _tables(pages, spare, seed):
    """Block tables of requests holding `pages` pages each, scattered over a
    pool with `spare` pages left over: tables [requests][width], free stack."""
    used = sum(pages)
    perm = torch.randperm(used + spare, generator=_gen(seed, 1), device=DEV).to(torch.int32)
    width = max(1, max(pages))
    held = torch.tensor(pages, device=DEV)
    start = held.cumsum(0) - held
    col = torch.arange(width, device=DEV)
    at = (start[:, None] + col).clamp(max=used + spare - 1)
    table = torch.where(col < held[:, None], perm[at], torch.full_like(perm[at], -1))
    return table.contiguous(), perm[used:].contiguous()


def prepare(case, seed):
    op = case["op"]
    s = dict(case)
    if op == "plan":
        ctx, new, order = _requests(case, seed)
        ps, n = case["page"], case["sequences"]
        # With prompt chunks in the step, one request in eight has just
        # finished: its slot is empty and its pages go back.
        done = [1 if case["chunked"] and i % 8 == 5 and k <= 5 else 0 for i, k in zip(order, new)]
        pages = [(c + ps - 1) // ps for c in ctx]
        cached = [0 if d else c for c, d in zip(ctx, done)]
        new = [0 if d else k for k, d in zip(new, done)]
        need = [max(0, (c + k + ps - 1) // ps - p) for c, k, p in zip(cached, new, pages)]
        width = max(1, max(p + k for p, k in zip(pages, need)))
        table, free = _tables(pages, sum(need) + 8, seed)
        wide = torch.full((n, width), -1, dtype=torch.int32, device=DEV)
        wide[:, :table.shape[1]] = table
        total = sum(pages) + sum(need) + 8
        stack = torch.full((total,), -1, dtype=torch.int32, device=DEV)
        stack[:free.numel()] = free
        rows = sum(new)
        out = lambda k: torch.empty(k, dtype=torch.int32, device=DEV)  # noqa: E731
        s.update(tables=wide, held=_int(pages), free_pages=stack, free_count=_int([free.numel()]), cached=_int(cached),
                 new_tokens=_int(new), finished=_int(done), rows=rows, held_out=out(n), free_count_out=out(1),
                 row_starts=out(n + 1), kv_lengths=out(n), positions=out(rows), slots=out(rows), row_sequence=out(rows))
    elif op == "rope":
        g = _gen(seed, 2)
        rows, d, ps = case["rows"], case["dim"], case["page"]
        width = (case["heads"] + 2 * case["kv_heads"]) * d
        pages = (rows + ps - 1) // ps + 4
        pool = lambda: torch.randn(pages, case["kv_heads"], ps, d, generator=g, device=DEV).bfloat16()  # noqa: E731
        slots = torch.randperm(pages * ps, generator=g, device=DEV)[:rows].to(torch.int32)
        slots[torch.rand(rows, generator=g, device=DEV) < 0.01] = -1  # rows of requests that got no pages
        first = torch.randint(0, max(1, case["max_pos"] - rows // 4), (4,), generator=g, device=DEV)
        r = torch.arange(rows, device=DEV)
        per = (rows + 3) // 4
        gain = lambda: (1.0 + 0.2 * torch.randn(d, generator=g, device=DEV)).bfloat16()  # noqa: E731
        s.update(qkv=torch.randn(rows, width, generator=g, device=DEV).bfloat16(), keys=pool(), values=pool(),
                 slots=slots, positions=(first[r // per] + r % per).to(torch.int32),
                 inv_freq=(500000.0 ** (-torch.arange(0, d, 2, dtype=torch.float64) / d)).float().to(DEV),
                 q_gain=gain() if case["norm"] else None, k_gain=gain() if case["norm"] else None, eps=1e-5,
                 q_out=torch.empty(rows, case["heads"] * d, dtype=torch.bfloat16, device=DEV))
    elif op == "attn":
        g = _gen(seed, 3)
        ctx, new, _ = _requests(case, seed)
        d, ps = case["dim"], case["page"]
        kv = [c + n for c, n in zip(ctx, new)]
        table, free = _tables([(k + ps - 1) // ps for k in kv], 8, seed)
        pages = sum((k + ps - 1) // ps for k in kv) + 8
        starts = [0]
        for n in new:
            starts.append(starts[-1] + n)
        q = torch.randn(starts[-1], case["heads"] * d, generator=g, device=DEV).mul_(1.5).bfloat16()
        s.update(q=q, keys=torch.randn(pages, case["kv_heads"], ps, d, generator=g, device=DEV, dtype=torch.bfloat16),
                 values=torch.randn(pages, case["kv_heads"], ps, d, generator=g, device=DEV, dtype=torch.bfloat16),
                 tables=table, row_starts=_int(starts), kv_lengths=_int(kv), most_new=max(new), most_kv=max(kv),
                 scale=1.0 / math.sqrt(d), out=torch.empty_like(q))
    elif op == "probs":
        g = _gen(seed, 4)
        rows, v = case["rows"], case["vocab"]
        logits = torch.randn(rows, v, generator=g, device=DEV).mul_(2.5)
        logits[:, v - 256:] = -math.inf  # ids that no text uses
        t = 0.6 + 0.6 * torch.rand(rows, generator=g, device=DEV)
        t[torch.rand(rows, generator=g, device=DEV) < 0.1] = 0.0  # greedy requests
        s.update(logits=logits, temperature=t, probs=torch.empty_like(logits))
    else:
        g = _gen(seed, 5)
        n, k, v = case["sequences"], case["drafts"], case["vocab"]
        counts = torch.randint(0, k + 1, (n,), generator=torch.Generator().manual_seed(seed + 11))
        counts[0] = k
        starts = torch.zeros(n + 1, dtype=torch.int64)
        starts[1:] = (counts + 1).cumsum(0)
        # The drafting model: the target's logits, disturbed; it drafted by
        # its own probabilities (or, as a point, the target's likely token).
        logits = torch.randn(n, k + 1, v, generator=g, device=DEV).mul_(2.5)
        near = logits[:, :k] + 0.6 * torch.randn(n, k, v, generator=g, device=DEV)
        draft = torch.softmax(near, -1)
        if case["point"]:
            drafts = near.argmax(-1)
        else:
            drafts = torch.multinomial(draft.view(n * k, v), 1, generator=g).view(n, k)
        rows = torch.repeat_interleave(torch.arange(n), counts + 1)
        col = torch.arange(int(starts[-1])) - starts[:-1][rows]
        target = torch.softmax(logits, -1)[rows.to(DEV), col.to(DEV)].contiguous()
        s.update(target_probs=target, draft_probs=None if case["point"] else draft, drafts=drafts.to(torch.int32),
                 draft_counts=counts.to(torch.int32).to(DEV), target_starts=starts.to(torch.int32).to(DEV),
                 uniforms=torch.rand(n, k + 1, generator=g, device=DEV),
                 tokens=torch.empty(n, k + 1, dtype=torch.int32, device=DEV),
                 accepted=torch.empty(n, dtype=torch.int32, device=DEV))
    return s


# ---------------------------------------------------------------------------
# One pass
# ---------------------------------------------------------------------------

def run(state):
    s = state
    return (_own if own else _plain)[s["op"]](s)


def _own_plan(s):
    _paged().plan_step(s["tables"], s["held"], s["free_pages"], s["free_count"], s["cached"], s["new_tokens"],
                       s["finished"], page_size=s["page"], held_out=s["held_out"],
                       free_count_out=s["free_count_out"], row_starts=s["row_starts"], kv_lengths=s["kv_lengths"],
                       positions=s["positions"], slots=s["slots"], row_sequence=s["row_sequence"])
    return {"tables": s["tables"], "held": s["held_out"], "free_pages": s["free_pages"],
            "free_count": s["free_count_out"], "row_starts": s["row_starts"], "kv_lengths": s["kv_lengths"],
            "positions": s["positions"], "slots": s["slots"], "row_sequence": s["row_sequence"]}


def _own_rope(s):
    _paged().qk_norm_rope_kv(s["q_out"], s["keys"], s["values"], s["qkv"], s["positions"], s["slots"], s["inv_freq"],
                             s["q_gain"], s["k_gain"], eps=s["eps"])
    return {"q": s["q_out"], "keys": s["keys"], "values": s["values"]}


def _own_attn(s):
    _paged().chunk_attention(s["out"], s["q"], s["keys"], s["values"], s["tables"], s["row_starts"], s["kv_lengths"],
                             scale=s["scale"])
    return s["out"]


def _own_probs(s):
    _paged().token_probs(s["probs"], s["logits"], s["temperature"])
    return s["probs"]


def _own_verify(s):
    _paged().verify_drafts(s["tokens"], s["accepted"], s["target_probs"], s["target_starts"], s["drafts"],
                           s["draft_counts"], s["draft_probs"], s["uniforms"])
    return {"tokens": s["tokens"], "accepted": s["accepted"]}


def _plain_plan(s):
    ps, width = s["page"], s["tables"].shape[1]
    cached, new, done = s["cached"].long(), s["new_tokens"].long(), s["finished"] != 0
    released = torch.where(done, s["held"].long(), 0)
    held = torch.where(done, 0, s["held"].long())
    want = (cached + new + ps - 1) // ps
    need = (want - held).clamp(min=0)
    ends = need.cumsum(0)
    count = s["free_count"].long()
    total = count + released.sum()
    granted = (need == 0) | (ends <= total)
    used = torch.where(granted, ends, 0).max()
    col = torch.arange(width, device=DEV)
    # Pages handed back, on top of the free ones in request order.
    stack = s["free_pages"].clone()
    back = col < released[:, None]
    at = count + (released.cumsum(0) - released)[:, None] + col
    stack[at[back]] = s["tables"][back]
    # Pages handed out, from the top.
    fresh = (col >= held[:, None]) & (col < want[:, None]) & granted[:, None]
    take = (total - 1 - (ends - need)[:, None] - (col - held[:, None])).clamp(min=0, max=stack.numel() - 1)
    tables = torch.where(fresh, stack[take], s["tables"])
    starts = torch.zeros(new.numel() + 1, dtype=torch.long, device=DEV)
    starts[1:] = new.cumsum(0)
    seq = torch.repeat_interleave(torch.arange(new.numel(), device=DEV), new, output_size=s["rows"])
    pos = cached[seq] + torch.arange(s["rows"], device=DEV) - starts[seq]
    slot = tables[seq, pos // ps].long() * ps + pos % ps
    out = {"tables": tables, "held": torch.where(granted, torch.maximum(held, want), held), "free_pages": stack,
           "free_count": total - used, "row_starts": starts, "kv_lengths": torch.where(granted, cached + new, 0),
           "positions": pos, "slots": torch.where(granted[seq], slot, -1), "row_sequence": seq}
    return {k: v.to(torch.int32) for k, v in out.items()}


def _plain_rope(s):
    rows, d, h, kvh = s["qkv"].shape[0], s["dim"], s["heads"], s["kv_heads"]
    x = s["qkv"].view(rows, h + 2 * kvh, d)
    angle = s["positions"].float()[:, None] * s["inv_freq"]
    cos, sin = angle.cos()[:, None], angle.sin()[:, None]

    def turned(y, gain):
        y = y.float()
        if gain is not None:
            y = y * torch.rsqrt((y * y).mean(-1, keepdim=True) + s["eps"]) * gain.float()
        lo, hi = y[..., :d // 2], y[..., d // 2:]
        return torch.cat((lo * cos - hi * sin, hi * cos + lo * sin), -1).bfloat16()

    there = s["slots"] >= 0
    at = s["slots"][there].long()
    page, slot = at // s["page"], at % s["page"]
    s["keys"][page, :, slot] = turned(x[:, h:h + kvh], s["k_gain"])[there]
    s["values"][page, :, slot] = x[:, h + kvh:][there]
    return {"q": turned(x[:, :h], s["q_gain"]).view(rows, h * d), "keys": s["keys"], "values": s["values"]}


def _plain_attn(s):
    ps, d, h, kvh = s["page"], s["dim"], s["heads"], s["kv_heads"]
    starts, kv = s["row_starts"].long(), s["kv_lengths"].long()
    new = starts[1:] - starts[:-1]
    i = torch.arange(s["most_new"], device=DEV)
    j = torch.arange(s["most_kv"], device=DEV)
    live = i < new[:, None]
    q = s["q"][(starts[:-1, None] + i).clamp(max=s["q"].shape[0] - 1)].float()
    q = q.view(-1, s["most_new"], kvh, h // kvh, d).permute(0, 2, 3, 1, 4)
    page = s["tables"].long()[:, j // ps].clamp(min=0)
    k = s["keys"][page, :, (j % ps).expand_as(page)].float().permute(0, 2, 3, 1).unsqueeze(2)
    scores = torch.matmul(q, k).mul_(s["scale"])
    seen = j <= ((kv - new)[:, None] + i)[:, :, None]
    scores.masked_fill_(~seen[:, None, None], -math.inf)
    scores -= scores.amax(-1, keepdim=True)
    scores.exp_()
    v = s["values"][page, :, (j % ps).expand_as(page)].float().permute(0, 2, 1, 3).unsqueeze(2)
    o = torch.matmul(scores, v) / scores.sum(-1, keepdim=True)
    return o.permute(0, 3, 1, 2, 4)[live].reshape(-1, h * d).bfloat16()


def _plain_probs(s):
    t = s["temperature"][:, None]
    x = s["logits"]
    z = (x - x.amax(-1, keepdim=True)) / torch.where(t > 0, t, 1.0)
    e = z.exp()
    one = torch.zeros_like(x).scatter_(1, x.argmax(-1, keepdim=True), 1.0)
    return torch.where(t > 0, e / e.sum(-1, keepdim=True), one)


def _plain_verify(s):
    p, k = s["target_probs"], s["drafts"].shape[1]
    n = s["drafts"].shape[0]
    starts, counts, drafts = s["target_starts"].long(), s["draft_counts"].long(), s["drafts"].long()
    fixed = lambda x: (x.clamp(0, 1) * SCALE).round().long()  # noqa: E731
    u = (s["uniforms"] * 2.0 ** 24).long()
    first = starts[1:] - 1 - counts
    j = torch.arange(k, device=DEV)
    rows = (first[:, None] + j).clamp(max=p.shape[0] - 1)
    pd = fixed(p[rows, drafts])
    qd = torch.full_like(pd, int(SCALE)) if s["point"] else fixed(s["draft_probs"].gather(2, drafts[..., None])[..., 0])
    ok = (u[:, :k] * qd < pd * 2 ** 24) & (j < counts[:, None])
    a = ok.long().cumprod(1).sum(1)
    refused = a < counts
    each = torch.arange(n, device=DEV)
    last = a.clamp(max=k - 1)
    pr = fixed(p[first + a])
    if s["point"]:
        qr = torch.zeros_like(pr)
        qr[each, drafts[each, last]] = int(SCALE)
    else:
        qr = fixed(s["draft_probs"][each, last])
    r = torch.where(refused[:, None], (pr - qr).clamp(min=0), pr)
    r = torch.where(r.sum(1, keepdim=True) > 0, r, pr)
    t = (u[:, k] * r.sum(1)) >> 24
    pick = (r.cumsum(1) <= t[:, None]).sum(1)
    i = torch.arange(k + 1, device=DEV)
    padded = torch.cat((drafts, drafts[:, :1]), 1)
    tokens = torch.where(i < a[:, None], padded, torch.where(i == a[:, None], pick[:, None], -1))
    return {"tokens": tokens.to(torch.int32), "accepted": a.to(torch.int32)}


_own = {"plan": _own_plan, "rope": _own_rope, "attn": _own_attn, "probs": _own_probs, "verify": _own_verify}
_plain = {"plan": _plain_plan, "rope": _plain_rope, "attn": _plain_attn, "probs": _plain_probs,
          "verify": _plain_verify}


# ---------------------------------------------------------------------------
# The definitions in 64 bits
# ---------------------------------------------------------------------------

def exact(case, seed):
    op = case["op"]
    if op in ("plan", "verify"):
        return None  # whole numbers
    s = prepare(case, seed)
    if op == "probs":
        z = s["logits"].double()
        out = torch.zeros_like(z)
        for r in range(z.shape[0]):
            t = float(s["temperature"][r])
            if t == 0.0:
                out[r, int((z[r] == z[r].max()).nonzero()[0])] = 1.0
            else:
                out[r] = torch.softmax(z[r] / t, 0)
        return out
    d, h, kvh, ps = case["dim"], case["heads"], case["kv_heads"], case["page"]
    if op == "rope":
        f = s["inv_freq"].double()
        c = torch.polar(torch.ones((), dtype=torch.float64, device=DEV),
                        s["positions"].double()[:, None] * f[None]).unsqueeze(1)

        def turned(lo_head, heads, gain):
            y = s["qkv"][:, lo_head * d:(lo_head + heads) * d].double().unflatten(1, (heads, d))
            if gain is not None:
                y = y / (y.square().mean(2, keepdim=True) + s["eps"]).sqrt() * gain.double()
            z = torch.complex(y[..., :d // 2], y[..., d // 2:]) * c
            return torch.cat((z.real, z.imag), 2)

        keys, values = s["keys"].double(), s["values"].double()
        k, v = turned(h, kvh, s["k_gain"]), s["qkv"][:, (h + kvh) * d:].double().unflatten(1, (kvh, d))
        rows = (s["slots"] >= 0).nonzero()[:, 0]
        at = s["slots"].long()[rows]
        for head in range(kvh):
            keys[at // ps, head, at % ps] = k[rows, head]
            values[at // ps, head, at % ps] = v[rows, head]
        return {"q": turned(0, h, s["q_gain"]).flatten(1), "keys": keys, "values": values}
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=DEV)
    starts, kv, table = s["row_starts"].tolist(), s["kv_lengths"].tolist(), s["tables"].tolist()
    for b in range(case["sequences"]):
        r0, r1, n = starts[b], starts[b + 1], kv[b]
        pages = torch.tensor(table[b][:(n + ps - 1) // ps], device=DEV)
        own_pos = torch.arange(n - (r1 - r0), n, device=DEV)
        late = torch.arange(n, device=DEV)[None] > own_pos[:, None]
        for g in range(kvh):
            k = s["keys"][pages, g].double().reshape(-1, d)[:n]
            v = s["values"][pages, g].double().reshape(-1, d)[:n]
            for x in range(g * (h // kvh), (g + 1) * (h // kvh)):
                w = s["q"][r0:r1, x * d:(x + 1) * d].double() @ k.T / math.sqrt(d)
                w[late] = -math.inf
                out[r0:r1, x * d:(x + 1) * d] = torch.softmax(w, 1) @ v
    return out
