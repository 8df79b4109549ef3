"""The operators of a ragged step over the paged cache (lcr_b200.paged) against
plain 64-bit implementations, at the sizes, masks and layouts where they can go
wrong."""
import math

import numpy as np
import pytest

from lcr_b200 import runtime as rt

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
if not torch.cuda.is_available():
    pytest.skip("needs a CUDA device", allow_module_level=True)

from lcr_b200 import paged  # noqa: E402

DEV = "cuda"


def i32(x):
    return torch.tensor(np.asarray(x, dtype=np.int32), device=DEV)


# ---------------------------------------------------------------------------
# plan_step
# ---------------------------------------------------------------------------

def plan_reference(tables, held, stack, count, cached, new, done, ps, pool, max_rows):
    """The definition, request by request."""
    tables, stack = tables.copy(), stack.copy()
    n, width = tables.shape
    held = held.copy()
    for b in range(n):
        if done[b]:
            stack[count:count + held[b]] = tables[b, :held[b]]
            count += held[b]
            held[b] = 0
    height, ends = count, 0
    granted = np.zeros(n, bool)
    for b in range(n):
        want = -(-(cached[b] + new[b]) // ps)
        if want > width:
            continue
        need = max(0, want - held[b])
        ends += need
        granted[b] = need == 0 or ends <= height
        if granted[b] and need:
            for i in range(held[b], want):
                count -= 1
                tables[b, i] = stack[count]
            held[b] = want
    starts = np.minimum(np.concatenate(([0], np.cumsum(new.astype(np.int64)))), max_rows).astype(np.int32)
    pos, slots, seq = [], [], []
    for b in range(n):
        for i in range(starts[b + 1] - starts[b]):
            p = cached[b] + i
            pos.append(p)
            seq.append(b)
            page = tables[b, p // ps] if granted[b] else -1
            slots.append(page * ps + p % ps if 0 <= page < pool else -1)
    return dict(tables=tables, held=held, stack=stack, count=count, starts=starts,
                kv=np.where(granted, cached + new, 0), pos=pos, slots=slots, seq=seq)


def run_plan(tables, held, stack, count, cached, new, done, ps, max_rows, alias):
    n = len(held)
    t, h, s, c = i32(tables), i32(held), i32(stack), i32([count])
    ho, co = (h, c) if alias else (torch.full_like(h, -7), torch.full_like(c, -7))
    starts, kv = torch.full((n + 1,), -7, dtype=torch.int32, device=DEV), torch.full_like(h, -7)
    pos, slots, seq = (torch.full((max_rows,), -7, dtype=torch.int32, device=DEV) for _ in range(3))
    paged.plan_step(t, h, s, c, i32(cached), i32(new), None if done is None else i32(done), page_size=ps, held_out=ho,
                    free_count_out=co, row_starts=starts, kv_lengths=kv, positions=pos, slots=slots, row_sequence=seq)
    host = lambda x: x.cpu().numpy()  # noqa: E731
    rows = int(starts[-1])
    assert (host(pos)[rows:] == 0).all() and (host(slots)[rows:] == -1).all() and (host(seq)[rows:] == -1).all()
    return dict(tables=host(t), held=host(ho), stack=host(s), count=int(co), starts=host(starts), kv=host(kv),
                pos=host(pos)[:rows].tolist(), slots=host(slots)[:rows].tolist(), seq=host(seq)[:rows].tolist())


def same_plan(got, want):
    for k in want:
        assert np.array_equal(got[k], want[k]), k


@pytest.mark.parametrize("alias", [False, True])
@pytest.mark.parametrize("n,ps,most_new,spare", [
    (1, 16, 1, 4), (1, 1, 5, 40), (7, 3, 9, 30), (64, 16, 5, 100), (33, 16, 300, 50), (512, 8, 40, 1000),
    (1500, 16, 20, 4000), (5000, 4, 6, 9000)])
def test_plan_step(n, ps, most_new, spare, alias):
    rng = np.random.default_rng(n * 131 + ps)
    cached = rng.integers(0, 200, n).astype(np.int32)
    new = rng.integers(0, most_new + 1, n).astype(np.int32)
    extra = rng.integers(0, 3, n)  # pages left over from refused drafts
    held = (-(-cached // ps) + extra).astype(np.int32)
    done = (rng.random(n) < 0.15).astype(np.int32)
    # A turned-over slot is empty, or takes a new request at once.
    cached[done == 1] = 0
    new[(done == 1) & (rng.random(n) < 0.5)] = 0
    width = int(max(held.max(), (-(-(cached + new) // ps)).max()))
    width = max(1, width)
    pool = int(held.sum()) + spare
    perm = rng.permutation(pool).astype(np.int32)
    tables = np.full((n, width), -1, np.int32)
    at = 0
    for b in range(n):
        tables[b, :held[b]] = perm[at:at + held[b]]
        at += held[b]
    stack = np.full(pool, -1, np.int32)
    stack[:spare] = perm[at:]
    rows = int(new.sum())
    want = plan_reference(tables, held, stack, spare, cached, new, done, ps, pool, rows)
    same_plan(run_plan(tables, held, stack, spare, cached, new, done, ps, rows, alias), want)
    if rows > 3:  # rows cut off
        want = plan_reference(tables, held, stack, spare, cached, new, done, ps, pool, rows - 3)
        same_plan(run_plan(tables, held, stack, spare, cached, new, done, ps, rows - 3, alias), want)


def test_plan_step_refuses_in_order():
    """Three free pages: the first request takes two, the second lacks two and
    is refused, the third would fit but comes later, the fourth lacks none;
    the fifth wants more pages than a table row holds."""
    tables = np.array([[9, -1, -1], [8, -1, -1], [7, -1, -1], [6, 5, -1], [4, -1, -1]], np.int32)
    held = np.array([1, 1, 1, 2, 1], np.int32)
    cached = np.array([16, 16, 16, 20, 16], np.int32)
    new = np.array([17, 20, 1, 2, 40], np.int32)
    stack = np.full(10, -1, np.int32)
    stack[:3] = [0, 1, 2]
    got = run_plan(tables, held, stack, 3, cached, new, None, 16, 80, False)
    want = plan_reference(tables, held, stack, 3, cached, new, np.zeros(5, int), 16, 10, 80)
    same_plan(got, want)
    assert got["kv"].tolist() == [33, 0, 0, 22, 0] and got["count"] == 1
    assert got["slots"][17:38] == [-1] * 21 and got["held"].tolist() == [3, 1, 1, 2, 1]


def test_plan_step_turns_a_slot_over_at_once():
    """A finished request's pages serve the slot's next request in the same
    step, tables and counts updated in place."""
    tables = np.array([[3, 1, 0, 2]], np.int32)
    got = run_plan(tables, np.array([4], np.int32), np.full(4, -1, np.int32), 0, np.array([0], np.int32),
                   np.array([33], np.int32), np.array([1]), 16, 33, True)
    assert got["tables"].tolist() == [[2, 0, 1, 2]] and got["held"].tolist() == [3] and got["count"] == 1
    assert got["slots"][:2] == [32, 33] and got["slots"][32] == 16 and got["kv"].tolist() == [33]


def test_plan_step_negative_lengths_and_foreign_pages():
    """Negative lengths count as 0; a page outside the pool gives no slots."""
    got = run_plan(np.array([[50, 1], [2, 3]], np.int32), np.array([2, 2], np.int32), np.full(8, -1, np.int32), 0,
                   np.array([0, -5], np.int32), np.array([18, -1], np.int32), None, 16, 18, False)
    assert got["starts"].tolist() == [0, 18, 18] and got["kv"].tolist() == [18, 0]
    assert got["slots"] == [-1] * 16 + [16, 17]


# ---------------------------------------------------------------------------
# qk_norm_rope_kv
# ---------------------------------------------------------------------------

def pools(pages, kv_heads, ps, d, gen, page_pad=0):
    """A pair of pools, with page_pad unused elements after each page."""
    def one():
        flat = torch.randn(pages, kv_heads * ps * d + page_pad, generator=gen, device=DEV).bfloat16()
        return flat.as_strided((pages, kv_heads, ps, d), (flat.stride(0), ps * d, d, 1))
    return one(), one()


@pytest.mark.parametrize("rows,heads,kv_heads,d,ps,norm,pad", [
    (1, 4, 2, 64, 16, True, 0), (1, 1, 1, 128, 1, True, 0), (7, 3, 1, 64, 5, True, 8), (300, 32, 8, 64, 16, True, 0),
    (300, 32, 8, 64, 16, False, 16), (129, 32, 8, 128, 16, True, 24), (33, 8, 8, 128, 7, False, 0),
    (1025, 4, 2, 64, 32, True, 0), (2400, 16, 2, 128, 16, True, 0)])
def test_qk_norm_rope_kv(rows, heads, kv_heads, d, ps, norm, pad):
    g = torch.Generator(device=DEV).manual_seed(rows * 7 + d)
    pages = -(-rows // ps) + 3
    keys, values = pools(pages, kv_heads, ps, d, g, pad)
    width = (heads + 2 * kv_heads) * d
    qkv = torch.randn(rows, width + pad, generator=g, device=DEV).bfloat16()[:, :width]
    q_out = torch.full((rows, heads * d + pad), 7.0, dtype=torch.bfloat16, device=DEV)[:, :heads * d]
    slots = torch.randperm(pages * ps, generator=g, device=DEV)[:rows].to(torch.int32)
    if rows > 4:
        slots[2], slots[3] = -1, pages * ps  # no slot: q only
    pos = torch.randint(0, 100000, (rows,), generator=g, device=DEV).to(torch.int32)
    pos[0] = 0
    inv = (500000.0 ** (-torch.arange(0, d, 2, dtype=torch.float64) / d)).float().to(DEV)
    gains = [(1 + 0.3 * torch.randn(d, generator=g, device=DEV)).bfloat16() if norm else None for _ in range(2)]
    want_k, want_v = keys.double(), values.clone()
    x = qkv.double().reshape(rows, heads + 2 * kv_heads, d)
    ang = pos.double()[:, None, None] * inv.double()

    def turn(y, gain):
        if gain is not None:
            y = y / (y.square().mean(-1, keepdim=True) + 1e-5).sqrt() * gain.double()
        lo, hi = y[..., :d // 2], y[..., d // 2:]
        return torch.cat((lo * ang.cos() - hi * ang.sin(), hi * ang.cos() + lo * ang.sin()), -1)

    wq, wk = turn(x[:, :heads], gains[0]), turn(x[:, heads:heads + kv_heads], gains[1])
    for r in range(rows):
        s = int(slots[r])
        if 0 <= s < pages * ps:
            want_k[s // ps, :, s % ps] = wk[r]
            want_v[s // ps, :, s % ps] = x[r, heads + kv_heads:].bfloat16()
    paged.qk_norm_rope_kv(q_out, keys, values, qkv, pos, slots, inv, *gains, eps=1e-5)
    # One rounding to bf16 (2^-9 of the value, taken twice over) and fp32
    # arithmetic on two terms of at most the head's largest value times 3
    # (2^-24 each, a dozen operations, the angle's error of 1e-5 at most).
    top = float(wq.abs().max())
    bound = lambda w: w.abs() * 2.0 ** -8 + 2e-5 * top  # noqa: E731
    got = q_out.double().reshape(rows, heads, d)
    assert bool(((got - wq).abs() <= bound(wq)).all())
    assert bool(((keys.double() - want_k).abs() <= bound(want_k)).all())
    assert torch.equal(values, want_v)


def test_qk_norm_rope_kv_in_place():
    """q_out may be the projection's own buffer."""
    g = torch.Generator(device=DEV).manual_seed(5)
    keys, values = pools(4, 2, 16, 64, g)
    qkv = torch.randn(9, 8 * 64, generator=g, device=DEV).bfloat16()
    args = (torch.arange(9, dtype=torch.int32, device=DEV), torch.arange(9, dtype=torch.int32, device=DEV),
            torch.linspace(1, 0.1, 32, device=DEV))
    out = torch.empty(9, 4 * 64, dtype=torch.bfloat16, device=DEV)
    k2, v2 = keys.clone(), values.clone()
    paged.qk_norm_rope_kv(out, keys, values, qkv, *args)
    L = rt.lib()
    import ctypes
    view = rt.KvView(k2.data_ptr(), v2.data_ptr(), None, 16, 2 * 16 * 64, 16 * 64, 2, 64)
    rt.check(L.lcr_qk_norm_rope_kv(qkv.data_ptr(), 512, ctypes.byref(view), 4, qkv.data_ptr(), 512, 9, 4, None, None,
                                   1e-5, args[2].data_ptr(), args[0].data_ptr(), args[1].data_ptr(), rt.stream_ptr()))
    assert torch.equal(qkv[:, :256], out) and torch.equal(keys, k2) and torch.equal(values, v2)


# ---------------------------------------------------------------------------
# chunk_attention
# ---------------------------------------------------------------------------

def attention_case(lens, heads, kv_heads, d, ps, *, seed=0, gain=1.0, pad=0, q_pad=0, poison=True):
    """lens: (new rows, kv length) of each request; cache positions past the
    lengths hold NaN."""
    g = torch.Generator(device=DEV).manual_seed(seed + 17)
    need = [-(-kv // ps) for _, kv in lens]
    pages = sum(need) + 2
    keys, values = pools(pages, kv_heads, ps, d, g, pad)
    width = max(1, max(need))
    perm = torch.randperm(pages, generator=g, device=DEV).cpu().numpy().astype(np.int32)
    tables = np.full((len(lens), width), -1, np.int32)
    at = 0
    for b, k in enumerate(need):
        tables[b, :k] = perm[at:at + k]
        at += k
    if poison:
        live = torch.zeros(pages, ps, dtype=torch.bool, device=DEV)
        for b, (_, kv) in enumerate(lens):
            for i in range(need[b]):
                live[int(tables[b, i]), :min(ps, kv - i * ps)] = True
        dead = (~live)[:, None, :, None].expand_as(keys)
        keys.masked_fill_(dead, math.nan)
        values.masked_fill_(dead, math.nan)
    starts = np.concatenate(([0], np.cumsum([n for n, _ in lens])))
    rows = int(starts[-1])
    q = (gain * torch.randn(rows, heads * d + q_pad, generator=g, device=DEV)).bfloat16()[:, :heads * d]
    return dict(q=q, keys=keys, values=values, tables=i32(tables), starts=i32(starts),
                kv=i32([kv for _, kv in lens]), lens=lens, heads=heads, kv_heads=kv_heads, d=d, ps=ps,
                host_tables=tables, host_starts=starts)


def attention_reference(c):
    """(out, bound): the 64-bit result and how far a result may be off. The
    weights are rounded to bf16 before they multiply the values (2^-9 of each,
    so of sum p|v|) and the output once (2^-9); both taken twice over for the
    fp32 sums, exponentials and their scores: a score's error is up to 2^-22
    of the sum of its terms' sizes, which shifts the weights by that share."""
    out = torch.zeros(c["q"].shape, dtype=torch.float64, device=DEV)
    bound = torch.zeros_like(out)
    d, group = c["d"], c["heads"] // c["kv_heads"]
    for b, (n, kv) in enumerate(c["lens"]):
        if n == 0 or kv == 0:
            continue
        r0 = int(c["host_starts"][b])
        pages = torch.tensor(c["host_tables"][b][:-(-kv // c["ps"])].astype(np.int64), device=DEV)
        k = c["keys"][pages].double().permute(1, 0, 2, 3).reshape(c["kv_heads"], -1, d)[:, :kv]
        v = c["values"][pages].double().permute(1, 0, 2, 3).reshape(c["kv_heads"], -1, d)[:, :kv]
        q = c["q"][r0:r0 + n].double().reshape(n, c["kv_heads"], group, d).permute(1, 2, 0, 3)
        s = q @ k.unsqueeze(1).transpose(-1, -2) / math.sqrt(d)
        size = q.abs() @ k.unsqueeze(1).transpose(-1, -2).abs() / math.sqrt(d)
        seen = torch.arange(kv, device=DEV)[None] <= (torch.arange(n, device=DEV) + kv - n)[:, None]
        s = s.masked_fill(~seen, -math.inf)
        some = seen.any(1)
        p = torch.zeros_like(s)
        p[:, :, some] = torch.softmax(s[:, :, some], -1)
        o = p @ v.unsqueeze(1)
        off = (p @ v.unsqueeze(1).abs()) * (2.0 ** -8 + 2.0 ** -21 * float(size.max())) + o.abs() * 2.0 ** -8
        put = lambda t: t.permute(2, 0, 1, 3).reshape(n, -1)  # noqa: E731
        out[r0:r0 + n], bound[r0:r0 + n] = put(o), put(off)
    return out, bound + 1e-30


def run_attention(c, workspace=None):
    out = torch.full((c["q"].shape[0], c["heads"] * c["d"]), 7.0, dtype=torch.bfloat16, device=DEV)
    paged.chunk_attention(out, c["q"], c["keys"], c["values"], c["tables"], c["starts"], c["kv"],
                          scale=1.0 / math.sqrt(c["d"]), workspace=workspace)
    torch.cuda.synchronize()
    paged.attention_status(workspace)
    return out


def check_attention(c, got=None):
    want, bound = attention_reference(c)
    got = run_attention(c) if got is None else got
    off = (got.double() - want).abs()
    assert bool(torch.isfinite(got).all())
    assert bool((off <= bound).all()), f"off by up to {float((off / bound).max()):.3g} of the bound"


LENS = {
    "one": [(1, 1)],
    "two_keys": [(1, 2)],
    "single_rows": [(1, 1), (1, 63), (1, 64), (1, 65), (1, 700), (1, 16)],
    "drafts": [(5, 255), (1, 64), (3, 130), (4, 4), (2, 1000), (5, 5)],
    "chunks": [(70, 70), (33, 200), (128, 128), (129, 129), (1, 500), (257, 1111)],
    "idle": [(0, 50), (3, 60), (0, 0), (0, 7), (2, 2), (0, 12)],
    "empty_rows": [(4, 0), (6, 2), (3, 3), (40, 7), (1, 0), (200, 130)],
    "long": [(1, 9000), (4, 4097), (17, 6000)],
}


@pytest.mark.parametrize("heads,kv_heads,d,ps", [
    (4, 2, 64, 16), (8, 8, 64, 16), (32, 8, 64, 16), (16, 2, 64, 5), (6, 2, 64, 1), (32, 8, 128, 16), (4, 4, 128, 3),
    (16, 1, 128, 24)])
@pytest.mark.parametrize("lens", list(LENS))
def test_chunk_attention(lens, heads, kv_heads, d, ps):
    check_attention(attention_case(LENS[lens], heads, kv_heads, d, ps, seed=heads + d))


@pytest.mark.parametrize("heads,kv_heads", [(128, 1), (66, 2), (5, 1), (7, 7), (64, 1)])
def test_chunk_attention_groups(heads, kv_heads):
    check_attention(attention_case([(3, 200), (20, 100), (1, 65)], heads, kv_heads, 64, 16, seed=heads))


@pytest.mark.parametrize("d", [64, 128])
def test_chunk_attention_strides_and_sharp_scores(d):
    """Padded pages and rows; scores up to +-100, where one key takes all and
    the running maximum keeps moving."""
    check_attention(attention_case([(9, 500), (40, 333), (1, 2000)], 8, 2, d, 16, pad=64, q_pad=24, gain=8.0))


def test_chunk_attention_many_requests():
    rng = np.random.default_rng(3)
    lens = [(int(n), int(n + c)) for n, c in zip(rng.integers(0, 6, 700), rng.integers(0, 90, 700))]
    check_attention(attention_case(lens, 4, 2, 64, 16, seed=9))


def test_chunk_attention_long_split():
    """One request on one KV head: its keys are shared out over the whole GPU
    and the parts joined, for a few rows and for a full tile of them."""
    check_attention(attention_case([(1, 33000)], 1, 1, 64, 16, seed=1))
    check_attention(attention_case([(5, 30001)], 4, 1, 128, 16, seed=2))
    check_attention(attention_case([(130, 20011)], 4, 1, 64, 16, seed=3))


def test_chunk_attention_repeats_and_shares_nothing():
    """Equal inputs give equal bits, whatever ran on the workspace before, and
    on another stream."""
    a = attention_case([(5, 3000), (64, 900), (1, 7777)], 8, 2, 64, 16, seed=4)
    b = attention_case([(3, 12000)], 4, 1, 128, 16, seed=5)
    first = run_attention(a)
    other = run_attention(b)
    assert torch.equal(run_attention(a), first) and torch.equal(run_attention(b), other)
    space = paged.attention_workspace(8, 64)
    s = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(s):
        out = run_attention(a, space)
    assert torch.equal(out, first)
    check_attention(a, first)


def test_chunk_attention_in_a_graph():
    """The call is capturable, and a replay sees lengths changed on the device."""
    c = attention_case([(5, 400), (2, 90)], 8, 2, 64, 16, seed=6, poison=False)
    out = torch.zeros(7, 8 * 64, dtype=torch.bfloat16, device=DEV)
    space = paged.attention_workspace(8, 64)
    args = (out, c["q"], c["keys"], c["values"], c["tables"], c["starts"], c["kv"])
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        paged.chunk_attention(*args, scale=0.125, workspace=space)
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        paged.chunk_attention(*args, scale=0.125, workspace=space)
    c["kv"].copy_(i32([333, 64]))
    c["lens"] = [(5, 333), (2, 64)]
    graph.replay()
    torch.cuda.synchronize()
    check_attention(c, out)


def test_chunk_attention_keeps_no_workspace_of_a_graph():
    """A stream whose first call is captured has to pass a workspace."""
    c = attention_case([(2, 70)], 4, 2, 64, 16)
    stream = torch.cuda.Stream()
    kept = dict(paged._workspaces)
    paged._workspaces.clear()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        with pytest.raises(RuntimeError, match="pass a workspace"):
            run_attention(c)
    assert not paged._workspaces
    paged._workspaces.update(kept)


def test_chunk_attention_page_outside_the_pool():
    """Reads as zeros and is reported once; the other requests are right."""
    c = attention_case([(2, 100), (3, 80)], 4, 2, 64, 16, seed=7, poison=False)
    want, bound = attention_reference(c)
    c["tables"][0, 1] = 10 ** 6
    space = paged.attention_workspace(4, 64)
    out = torch.empty_like(c["q"])
    paged.chunk_attention(out, c["q"], c["keys"], c["values"], c["tables"], c["starts"], c["kv"], scale=0.125,
                          workspace=space)
    with pytest.raises(rt.LcrError) as e:
        paged.attention_status(space)
    assert e.value.status == 5
    paged.attention_status(space)
    assert bool(torch.isfinite(out).all()) and bool(((out.double() - want).abs() <= bound)[2:].all())


def test_chunk_attention_lengths_past_the_tables():
    """kv lengths are cut to what a table row can hold."""
    c = attention_case([(2, 64)], 4, 2, 64, 16, seed=8, poison=False)
    want, bound = attention_reference(c)
    c["kv"].fill_(2 ** 31 - 1)
    got = run_attention(c)
    assert bool(((got.double() - want).abs() <= bound).all())


@pytest.mark.parametrize("ps", [16, 5])
def test_offsets_past_32_bits(ps):
    """Pools of more than 2^31 elements: rows are written to and read from
    their last pages (page sizes with and without tensor copies)."""
    kv_heads, d, heads = 8, 64, 16
    pages = (2 ** 31 + 2 ** 28) // (kv_heads * ps * d)
    keys = torch.empty(pages, kv_heads, ps, d, dtype=torch.bfloat16, device=DEV)
    values = torch.empty_like(keys)
    n, g = 37, torch.Generator(device=DEV).manual_seed(21)
    used = -(-n // ps)
    table = torch.arange(pages - used, pages, dtype=torch.int32, device=DEV).flip(0)[None].contiguous()
    assert (pages - used) * kv_heads * ps * d > 2 ** 31
    pos = torch.arange(n, dtype=torch.int32, device=DEV)
    slots = table[0, (pos // ps).long()] * ps + pos % ps
    qkv = torch.randn(n, (heads + 2 * kv_heads) * d, generator=g, device=DEV).bfloat16()
    q = torch.empty(n, heads * d, dtype=torch.bfloat16, device=DEV)
    paged.qk_norm_rope_kv(q, keys, values, qkv, torch.zeros_like(pos), slots, torch.ones(d // 2, device=DEV))
    assert torch.equal(q, qkv[:, :heads * d])  # position 0: no turn
    c = dict(q=q, keys=keys, values=values, tables=table, starts=i32([0, n]), kv=i32([n]), lens=[(n, n)], heads=heads,
             kv_heads=kv_heads, d=d, ps=ps, host_tables=table.cpu().numpy(), host_starts=np.array([0, n]))
    flat = qkv.view(n, -1, d)
    assert torch.equal(keys[table[0].long()].permute(0, 2, 1, 3).reshape(-1, kv_heads, d)[:n], flat[:, heads:heads + kv_heads])
    assert torch.equal(values[table[0].long()].permute(0, 2, 1, 3).reshape(-1, kv_heads, d)[:n], flat[:, heads + kv_heads:])
    check_attention(c)


# ---------------------------------------------------------------------------
# token_probs
# ---------------------------------------------------------------------------

@pytest.mark.parametrize("rows,vocab", [(1, 1), (3, 2), (5, 1000), (2, 4099), (9, 128256), (40, 32001), (2, 131072),
                                        (3, 131073), (2, 300007)])
@pytest.mark.parametrize("pad", [0, 4, 5])
def test_token_probs(rows, vocab, pad):
    g = torch.Generator(device=DEV).manual_seed(vocab + rows)
    logits = (4 * torch.randn(rows, vocab + pad, generator=g, device=DEV))[:, :vocab]
    t = 0.5 + torch.rand(rows, generator=g, device=DEV)
    t[0] = 0.0
    if vocab > 4:
        logits[:, vocab // 2] = -math.inf
        logits[0, 3] = logits[0, vocab - 1] = 99.0  # a tie: the lowest id
    if rows > 2:
        logits[2] = -math.inf
    probs = torch.full((rows, vocab + pad), 7.0, device=DEV)[:, :vocab]
    want = torch.zeros(rows, vocab, dtype=torch.float64, device=DEV)
    for r in range(rows):
        x = logits[r].double()
        if bool((x == -math.inf).all()):
            continue
        if float(t[r]) <= 0:
            want[r, int((x == x.max()).nonzero()[0])] = 1.0
        else:
            want[r] = torch.softmax(x / t[r].double(), 0)
    paged.token_probs(probs, logits, t)
    # The exponent (x - max) / t has three roundings of 2^-24 of its size, up
    # to 150 here, the exponential and the sum a few more; below 2^-126 nothing.
    bound = want * (150 * 3 * 2.0 ** -24 + 1e-6) + 2.0 ** -126
    assert bool(((probs.double() - want).abs() <= bound).all())
    logits_copy = logits.clone() if pad else logits
    paged.token_probs(logits_copy, logits_copy, t)  # in place
    assert torch.equal(logits_copy, probs)


def test_token_probs_by_request_and_without_temperature():
    g = torch.Generator(device=DEV).manual_seed(1)
    x = torch.randn(6, 999, generator=g, device=DEV)
    seq = i32([0, 0, 1, 2, 2, 2])
    t = torch.tensor([0.7, 0.0, 1.3], device=DEV)
    a, b = torch.empty_like(x), torch.empty_like(x)
    paged.token_probs(a, x, t, seq)
    paged.token_probs(b, x, t[seq.long()].contiguous())
    assert torch.equal(a, b)
    paged.token_probs(b, x, t, i32([0, -1, 1, 2, 3, 2]))  # rows of no request
    assert torch.equal(b[[0, 2, 3, 5]], a[[0, 2, 3, 5]]) and not b[[1, 4]].any()
    paged.token_probs(a, x)
    assert float((a.double() - torch.softmax(x.double(), 1)).abs().max()) < 1e-6


def test_token_probs_at_the_ends_of_the_temperature():
    """1e-40: everything on the largest logits; inf: the same on all that are
    not -inf; NaN and below 0: the lowest of the largest."""
    x = torch.tensor([[1.0, 3.0, -math.inf, 3.0, 2.0, -1e30, 0.0]], device=DEV).repeat(4, 1)
    p = torch.empty_like(x)
    paged.token_probs(p, x, torch.tensor([1e-40, math.inf, math.nan, -1.0], device=DEV))
    want = torch.tensor([[0, 0.5, 0, 0.5, 0, 0, 0], [1 / 6, 1 / 6, 0, 1 / 6, 1 / 6, 1 / 6, 1 / 6],
                         [0, 1, 0, 0, 0, 0, 0], [0, 1, 0, 0, 0, 0, 0]], device=DEV)
    assert float((p[[0, 2, 3]] - want[[0, 2, 3]]).abs().max()) == 0
    assert float((p[1] - want[1]).abs().max()) < 1e-6


# ---------------------------------------------------------------------------
# verify_drafts
# ---------------------------------------------------------------------------

def fixed(p):
    p = np.where(np.isnan(p), 0, p).astype(np.float64)
    return np.rint(np.clip(p, 0, 1) * 2.0 ** 38).astype(np.int64).astype(object)  # Python integers


def verify_reference(target, starts, drafts, counts, draft_probs, uniforms):
    n, k = drafts.shape
    vocab = target.shape[1]
    tokens, accepted = np.full((n, k + 1), -1, np.int64), np.zeros(n, np.int64)
    for b in range(n):
        rows = starts[b + 1] - starts[b]
        if rows <= 0:
            continue
        c = max(0, min(counts[b], k, rows - 1))
        first = starts[b + 1] - 1 - c
        u = [int(math.floor(float(x) * 2 ** 24)) for x in uniforms[b]]
        a = 0
        while a < c:
            d = drafts[b, a]
            if not 0 <= d < vocab:
                break
            p = fixed(target[first + a, d:d + 1])[0]
            q = 2 ** 38 if draft_probs is None else fixed(draft_probs[b, a, d:d + 1])[0]
            if not u[a] * q < p * 2 ** 24:
                break
            tokens[b, a] = d
            a += 1
        r = p = fixed(target[first + a])
        if a < c:
            if draft_probs is not None:
                r = np.maximum(p - fixed(draft_probs[b, a]), 0)
            elif 0 <= drafts[b, a] < vocab:
                r = p.copy()
                r[drafts[b, a]] = max(0, r[drafts[b, a]] - 2 ** 38)
        if sum(r) == 0:
            r = p
        total = sum(r)
        t = u[k] * total // 2 ** 24
        accepted[b] = a
        run = np.cumsum(r)
        over = np.nonzero(run > t)[0]
        tokens[b, a] = over[0] if total else -1
    return tokens, accepted


def run_verify(target, starts, drafts, counts, draft_probs, uniforms):
    n, k = drafts.shape
    tokens, accepted = torch.full((n, k + 1), -9, dtype=torch.int32, device=DEV), torch.full((n,), -9, dtype=torch.int32,
                                                                                            device=DEV)
    paged.verify_drafts(tokens, accepted, target, i32(starts), i32(drafts).reshape(n, k), i32(counts), draft_probs,
                        uniforms)
    return tokens.cpu().numpy(), accepted.cpu().numpy()


@pytest.mark.parametrize("point", [False, True])
@pytest.mark.parametrize("n,k,vocab,pad", [(1, 0, 7, 0), (1, 1, 1, 0), (9, 4, 5, 3), (40, 3, 1000, 0), (64, 8, 333, 1),
                                           (6, 4, 128256, 0), (3, 2, 131073, 4), (2, 2, 300007, 0), (300, 1, 50, 0)])
def test_verify_drafts(n, k, vocab, pad, point):
    rng = np.random.default_rng(n * 1009 + vocab)
    g = torch.Generator(device=DEV).manual_seed(n + vocab)
    counts = rng.integers(0, k + 1, n)
    extra = rng.integers(0, 3, n)  # earlier rows of the step that nothing is drawn from
    rows = counts + 1 + extra
    rows[rng.random(n) < 0.1] = 0
    if n == 1:
        rows[0] = counts[0] + 1
    starts = np.concatenate(([0], np.cumsum(rows)))
    logits = 2.0 * torch.randn(int(starts[-1]) + 1, vocab + pad, generator=g, device=DEV)
    target = torch.softmax(logits, -1)[:, :vocab]
    draft_probs = torch.softmax(2.0 * torch.randn(n, k, vocab, generator=g, device=DEV), -1)
    for b in range(n):  # drafting rows near the target's
        for j in range(counts[b]):
            if rows[b] and rng.random() < 0.7:
                row = int(starts[b + 1]) - 1 - counts[b] + j
                draft_probs[b, j] = 0.9 * target[row] + 0.1 * draft_probs[b, j]
    drafts = np.zeros((n, k), np.int64)
    for b in range(n):
        for j in range(k):
            drafts[b, j] = int(torch.multinomial(draft_probs[b, j], 1, generator=g))
    if n > 4 and k > 1:
        drafts[1, 0], drafts[2, 1] = vocab, -1  # outside the vocabulary
    u = torch.rand(n, k + 1, generator=g, device=DEV)
    u[0, k] = 0.0
    u[n - 1, k] = 1.0 - 2.0 ** -24
    q = None if point else draft_probs
    want = verify_reference(target.cpu().numpy(), starts, drafts, counts, None if point else draft_probs.cpu().numpy(),
                            u.cpu().numpy())
    got = run_verify(target, starts, drafts, counts, q, u)
    assert np.array_equal(got[1], want[1])
    assert np.array_equal(got[0], want[0])


def test_verify_drafts_corner_values():
    """Equal rows (never refused), disjoint rows (always), a residual of
    nothing, rows of zeros, NaN and numbers outside [0, 1], counts that pass
    the rows."""
    v = 40
    p = torch.zeros(9, v, device=DEV)
    p[0, 3] = 1.0                      # request 0: equal rows
    p[1, 5] = 0.25
    p[1, 7] = 0.75
    p[2, 9] = 1.0                      # request 1: refused, drawn from the target alone
    p[3, 1] = 1.0
    p[4, 2] = 0.5                      # request 2: P <= Q everywhere and U at its largest: R is 0
    p[5, 0] = 1.0
    #      6                             request 3: a row of zeros
    p[7] = math.nan                    # request 4: only id 11 counts (as 1), twice its size
    p[7, 11] = 2.0
    p[7, 12] = -3.0
    p[8, 30] = 1.0                     # request 5: more drafts counted than rows
    starts = [0, 2, 4, 6, 7, 8, 9]
    q = torch.zeros(6, 1, v, device=DEV)
    q[0, 0, 3] = 1.0
    q[1, 0, 8] = 1.0
    q[2, 0, 2] = 1.0
    q[5, 0, 1] = 1.0
    drafts = np.array([[3], [8], [2], [0], [0], [1]])
    counts = np.array([1, 1, 1, 0, 0, 7])
    u = torch.tensor([[1 - 2.0 ** -24, 0.3], [0.0, 0.5], [1 - 2.0 ** -24, 0.9], [0.5, 0.5], [0.5, 0.5], [0.1, 0.1]],
                     device=DEV)
    got = run_verify(p, starts, drafts, counts, q, u)
    assert got[1].tolist() == [1, 0, 0, 0, 0, 0]
    assert got[0].tolist() == [[3, 7], [9, -1], [2, -1], [-1, -1], [11, -1], [30, -1]]
    want = verify_reference(p.cpu().numpy(), starts, drafts, counts, q.cpu().numpy(), u.cpu().numpy())
    assert np.array_equal(got[0], want[0]) and np.array_equal(got[1], want[1])


def test_verify_drafts_keeps_the_target_distribution():
    """Over many uniforms the first token is distributed as the target's row:
    each id's share is within five standard deviations of its probability."""
    n, v = 20000, 6
    p = torch.tensor([0.35, 0.05, 0.2, 0.0, 0.3, 0.1], device=DEV)
    q = torch.tensor([0.1, 0.3, 0.2, 0.2, 0.1, 0.1], device=DEV)
    g = torch.Generator(device=DEV).manual_seed(12)
    drafts = torch.multinomial(q.expand(n, v), 1, generator=g).cpu().numpy()
    starts = np.arange(0, 2 * n + 1, 2)
    got, _ = run_verify(p.expand(2 * n, v).contiguous(), starts, drafts, np.ones(n, int),
                        q.expand(n, 1, v).contiguous(), torch.rand(n, 2, generator=g, device=DEV))
    share = np.bincount(got[:, 0], minlength=v) / n
    pp = p.cpu().numpy().astype(np.float64)
    assert (np.abs(share - pp) <= 5 * np.sqrt(pp * (1 - pp) / n) + 1e-12).all()


# ---------------------------------------------------------------------------
# refusals
# ---------------------------------------------------------------------------

def test_a_captured_step_runs_with_fewer_rows():
    """Plan, cache write, attention and probabilities in one graph of 12 rows:
    replayed for steps of 12, 5 and 0 rows it gives what the entries give for
    exactly those rows, and touches nothing else."""
    g = torch.Generator(device=DEV).manual_seed(7)
    heads, kvh, d, ps, pool, n, most = 4, 2, 64, 16, 24, 3, 12
    inv = 10000.0 ** (-torch.arange(32, device=DEV) / 32.0)
    qkv = torch.randn(most, (heads + 2 * kvh) * d, generator=g, device=DEV).bfloat16()
    heat = torch.tensor([0.5, 1.0, 2.0], device=DEV)

    def state():
        rows = lambda: torch.full((most,), -7, dtype=torch.int32, device=DEV)  # noqa: E731
        z = lambda *shape: torch.zeros(*shape, dtype=torch.bfloat16, device=DEV)  # noqa: E731
        return dict(tables=torch.zeros(n, 8, dtype=torch.int32, device=DEV), held=i32([0] * n), stack=i32(range(pool)),
                    count=i32([pool]), cached=i32([0] * n), new=i32([5, 1, 6]), starts=i32([0] * (n + 1)), kv=i32([0] * n),
                    pos=rows(), slots=rows(), seq=rows(), keys=z(pool, kvh, ps, d), values=z(pool, kvh, ps, d),
                    q=z(most, heads * d), out=torch.full((most, heads * d), 3.0, dtype=torch.bfloat16, device=DEV),
                    probs=torch.full((most, d), 3.0, device=DEV), work=paged.attention_workspace(heads, d))

    def step(s, rows):
        pos, slots, seq = s["pos"][:rows], s["slots"][:rows], s["seq"][:rows]
        paged.plan_step(s["tables"], s["held"], s["stack"], s["count"], s["cached"], s["new"], page_size=ps,
                        held_out=s["held"], free_count_out=s["count"], row_starts=s["starts"], kv_lengths=s["kv"],
                        positions=pos, slots=slots, row_sequence=seq)
        paged.qk_norm_rope_kv(s["q"][:rows], s["keys"], s["values"], qkv[:rows], pos, slots, inv)
        paged.chunk_attention(s["out"][:rows], s["q"][:rows], s["keys"], s["values"], s["tables"], s["starts"], s["kv"],
                              scale=0.125, workspace=s["work"])
        paged.token_probs(s["probs"][:rows], qkv[:rows, :d].float(), heat, seq)

    a, b = state(), state()
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        step(a, most)
    cached = np.zeros(n, int)
    for new in ([5, 1, 6], [2, 0, 3], [0, 0, 0], [0, 12, 0]):
        rows = sum(new)
        for s in (a, b):
            s["cached"].copy_(i32(cached))
            s["new"].copy_(i32(new))
            s["out"].fill_(3.0)
        graph.replay()
        step(b, rows)
        paged.attention_status(a["work"])
        for k in ("tables", "held", "stack", "count", "starts", "kv", "keys", "values"):
            assert torch.equal(a[k], b[k]), (new, k)
        for k in ("pos", "slots", "seq", "q", "out", "probs"):
            assert torch.equal(a[k][:rows], b[k][:rows]), (new, k)
        assert (a["out"][rows:] == 3.0).all() and not a["probs"][rows:].any()
        assert (a["slots"][rows:] == -1).all() and (a["seq"][rows:] == -1).all()
        cached += np.array(new)


def test_refusals():
    c = attention_case([(2, 20)], 4, 2, 64, 16)
    out = torch.empty_like(c["q"])
    args = [out, c["q"], c["keys"], c["values"], c["tables"], c["starts"], c["kv"]]

    def attempt(i, t):
        a = list(args)
        a[i] = t
        with pytest.raises((ValueError, rt.LcrError)):
            paged.chunk_attention(*a, scale=0.1)

    attempt(0, out.float())
    attempt(0, out[:, :64])
    attempt(1, c["q"].cpu())
    attempt(2, c["keys"].float())
    attempt(2, c["keys"].transpose(1, 2))
    attempt(4, c["tables"].long())
    attempt(5, c["starts"][:1])
    attempt(6, c["kv"].float())
    with pytest.raises(rt.LcrError) as e:  # three query heads on two KV heads
        paged.chunk_attention(torch.empty_like(out[:, :192]), c["q"][:, :192], *args[2:], scale=0.1)
    assert e.value.status == 2
    with pytest.raises(rt.LcrError) as e:  # a scratch too small
        paged.chunk_attention(*args, scale=0.1, workspace=torch.zeros(16, dtype=torch.uint8, device=DEV))
    assert e.value.status == 1
    with pytest.raises(rt.LcrError) as e:  # rows off a 16-byte boundary
        flat = torch.zeros(2 * 256 + 1, dtype=torch.bfloat16, device=DEV)
        paged.chunk_attention(flat[1:].view(2, 256), *args[1:], scale=0.1)
    assert e.value.status == 2
    with pytest.raises(ValueError):
        paged.token_probs(torch.empty(2, 5, device=DEV), torch.empty(2, 6, device=DEV))
    with pytest.raises(ValueError):
        paged.verify_drafts(i32([[0, 0]]), i32([0]), torch.zeros(1, 5, device=DEV), i32([0, 1]), i32([[0, 0]]), i32([0]),
                            None, torch.zeros(1, 2, device=DEV))
    with pytest.raises(ValueError):
        paged.qk_norm_rope_kv(out, c["keys"], c["values"], c["q"], i32([0, 1]), i32([0, 1]),
                              torch.zeros(32, device=DEV))
