"""Corners of the ragged step's operators (lcr_b200.paged): what a call among
others, on odd values or with odd tensors, once got wrong or could."""
import math
import threading

import numpy as np
import pytest

from lcr_b200 import runtime as rt

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
if not torch.cuda.is_available():
    pytest.skip("needs a CUDA device", allow_module_level=True)

from lcr_b200 import paged  # noqa: E402
from test_paged_gpu import DEV, attention_case, check_attention, i32, pools, run_attention, run_verify  # noqa: E402


def test_chunk_attention_in_a_capture_needs_a_workspace():
    """A graph may be replayed on any stream, beside calls on the one it was
    captured on: what a stream keeps must not get into it."""
    c = attention_case([(2, 70)], 4, 2, 64, 16)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        first = run_attention(c)  # the stream keeps a workspace from here on
    out = torch.empty_like(first)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        with pytest.raises(RuntimeError, match="pass a workspace"):
            paged.chunk_attention(out, c["q"], c["keys"], c["values"], c["tables"], c["starts"], c["kv"], scale=0.125)
    with torch.cuda.stream(stream):
        assert torch.equal(run_attention(c), first)


@pytest.mark.parametrize("vocab", [3, 999, 128256])
def test_token_probs_zeros_of_either_sign_tie(vocab):
    """Greedy: -0.0 and 0.0 are equal, so the lower id of them is taken."""
    x = torch.full((3, vocab), -1.0, device=DEV)
    x[0, 0], x[0, vocab - 1] = -0.0, 0.0
    x[1, 0], x[1, vocab - 1] = 0.0, -0.0
    x[2, 1], x[2, vocab - 1] = -0.0, -0.0
    p = torch.empty_like(x)
    paged.token_probs(p, x, torch.zeros(3, device=DEV))
    want = torch.zeros_like(x)
    want[[0, 1, 2], [0, 0, 1]] = 1.0
    assert torch.equal(p, want)


@pytest.mark.parametrize("vocab", [4, 5000, 128256, 300007])
def test_token_probs_of_a_row_with_nan(vocab):
    """A NaN among the logits makes the whole row NaN, as in the formula, also
    where its neighbours are -inf; rows beside it are untouched."""
    x = torch.randn(3, vocab, generator=torch.Generator(device=DEV).manual_seed(vocab), device=DEV)
    x[1, :vocab // 2] = -math.inf
    x[1, 1] = math.nan
    p = torch.empty_like(x)
    paged.token_probs(p, x, torch.ones(3, device=DEV))
    assert bool(p[1].isnan().all())
    q = torch.empty_like(x[:1])
    for r in (0, 2):
        paged.token_probs(q, x[r:r + 1], torch.ones(1, device=DEV))
        # (A single row may go to another number of blocks: sums in another order.)
        assert float((q[0] - p[r]).abs().max()) <= 1e-6 * float(q.max())


def test_verify_drafts_refuses_other_layouts():
    """draft_probs and uniforms are read densely as [requests][max_drafts]
    [vocab] and [requests][max_drafts + 1]: padded or transposed ones would be
    misread. Room for more requests, and flat buffers, are as good."""
    n, k, v = 3, 2, 10
    g = torch.Generator(device=DEV).manual_seed(8)
    p, q = (torch.softmax(torch.randn(m, v, generator=g, device=DEV), 1) for m in (n * (k + 1), n * k))
    u = torch.rand(n, k + 1, generator=g, device=DEV)
    args = dict(target_probs=p, target_starts=i32([0, 3, 6, 9]), drafts=i32(np.ones((n, k))), draft_counts=i32([2, 1, 0]),
                draft_probs=q.view(n, k, v), uniforms=u)

    def run(**kw):
        tokens, accepted = i32(np.zeros((n, k + 1))), i32(np.zeros(n))
        paged.verify_drafts(tokens, accepted, **{**args, **kw})
        return tokens

    want = run()
    for kw in [dict(draft_probs=q), dict(draft_probs=q.view(n, k * v)), dict(draft_probs=q.flatten()),
               dict(draft_probs=torch.cat((q, q)).view(2 * n, k, v)), dict(uniforms=u.flatten()),
               dict(uniforms=torch.cat((u, u))), dict(uniforms=u[..., None])]:
        assert torch.equal(run(**kw), want)
    for name, shape in [("draft_probs", (n, k, v + 2)), ("draft_probs", (n, k + 1, v)), ("draft_probs", (n, v, k)),
                        ("draft_probs", (n * k, v + 1)), ("draft_probs", (n, k, v - 1)), ("uniforms", (n, k + 2)),
                        ("uniforms", (k + 1, n + 1)), ("uniforms", (n - 1, k + 1))]:
        with pytest.raises(ValueError, match=name):
            run(**{name: torch.full(shape, 0.5, device=DEV)})


def test_qk_norm_rope_kv_refuses_gains_of_several_heads():
    """Gains are one per element of a head, the same for all heads: a gain for
    each head is not taken in part."""
    g = torch.Generator(device=DEV).manual_seed(3)
    keys, values = pools(2, 2, 16, 64, g)
    qkv = torch.randn(2, 8 * 64, generator=g, device=DEV).bfloat16()
    q, at = torch.empty(2, 4 * 64, dtype=torch.bfloat16, device=DEV), i32([0, 1])
    inv, gain = torch.ones(32, device=DEV), torch.ones(64, dtype=torch.bfloat16, device=DEV)
    paged.qk_norm_rope_kv(q, keys, values, qkv, at, at, inv, gain, gain[None])
    for bad in [dict(q_gain=gain.repeat(4)), dict(k_gain=gain.repeat(2).view(2, 64)), dict(k_gain=gain[:32])]:
        with pytest.raises(ValueError, match=next(iter(bad))):
            paged.qk_norm_rope_kv(q, keys, values, qkv, at, at, inv, **{**dict(q_gain=gain, k_gain=gain), **bad})


@pytest.mark.parametrize("d", [64, 128])
def test_qk_norm_rope_kv_far_positions(d):
    """Positions up to 2^20. One rounding to bf16 (2^-8 of the value); the
    turn's pair is off by 1e-5 at most there, on two terms."""
    g = torch.Generator(device=DEV).manual_seed(d)
    rows, heads, kvh = 512, 6, 2
    keys, values = pools(rows // 16, kvh, 16, d, g)
    qkv = torch.randn(rows, (heads + 2 * kvh) * d, generator=g, device=DEV).bfloat16()
    pos = torch.randint(2 ** 17, 2 ** 20, (rows,), generator=g, device=DEV).to(torch.int32)
    pos[0] = 2 ** 20 - 1
    inv = (500000.0 ** (-torch.arange(0, d, 2, dtype=torch.float64) / d)).float().to(DEV)
    q = torch.empty(rows, heads * d, dtype=torch.bfloat16, device=DEV)
    paged.qk_norm_rope_kv(q, keys, values, qkv, pos, torch.arange(rows, dtype=torch.int32, device=DEV), inv)
    x = qkv.double().view(rows, -1, d)[:, :heads + kvh]
    a = pos.double()[:, None, None] * inv.double()
    lo, hi = x[..., :d // 2], x[..., d // 2:]
    want = torch.cat((lo * a.cos() - hi * a.sin(), hi * a.cos() + lo * a.sin()), -1)
    k = keys.permute(0, 2, 1, 3).reshape(rows, kvh, d)
    got = torch.cat((q.view(rows, heads, d), k), 1).double()
    assert bool(((got - want).abs() <= want.abs() * 2.0 ** -8 + 2e-5 * float(want.abs().max())).all())


def test_plan_step_from_several_threads():
    """Host threads plan steps of different sizes at the same time."""
    L = rt.lib()
    bad = {}

    def go(n):
        ints = lambda k: torch.zeros(k, dtype=torch.int32, device=DEV)  # noqa: E731
        t, h, s, c, cached, new, starts, kv, row = (ints(k) for k in (n, n, 4, 1, n, n, n + 1, n, 4))
        ptr = [x.data_ptr() for x in (t, h, s, c, cached, new, starts, kv, row)]
        t, h, s, c, cached, new, starts, kv, row = ptr
        torch.cuda.synchronize()
        start.wait()
        bad[n] = sum(L.lcr_plan_step(t, 1, h, h, s, c, c, 4, cached, new, None, n, 16, 4, starts, kv, row, row, row,
                                     None) != 0 for _ in range(4000))
        torch.cuda.synchronize()

    sizes = [8192, 1, 64, 3000]
    start = threading.Barrier(len(sizes))
    threads = [threading.Thread(target=go, args=(n,)) for n in sizes]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert bad == {n: 0 for n in sizes}


def test_chunk_attention_scratch_serves_both_head_sizes():
    """Every call leaves a workspace ready for the next, whatever its head
    size: tiles split over the whole GPU, in turn, on one workspace."""
    a = attention_case([(5, 9000), (64, 3000)], 8, 2, 64, 16, seed=4)
    b = attention_case([(3, 12000), (40, 2500)], 4, 1, 128, 16, seed=5)
    space = max((paged.attention_workspace(8, d) for d in (64, 128)), key=torch.Tensor.numel)
    for _ in range(2):
        check_attention(b, run_attention(b, space))
        check_attention(a, run_attention(a, space))


def test_chunk_attention_checks_before_it_keeps_a_workspace():
    c = attention_case([(2, 20)], 4, 2, 64, 16)
    wide = torch.zeros(2, 2, 16, 96, dtype=torch.bfloat16, device=DEV)
    out = torch.empty_like(c["q"])
    rest = (c["tables"], c["starts"], c["kv"])
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        kept = len(paged._workspaces)
        for keys in ([1, 2], None, torch.zeros(0, dtype=torch.bfloat16, device=DEV), wide[..., :0]):
            with pytest.raises(ValueError):
                paged.chunk_attention(out, c["q"], keys, keys, *rest, scale=0.1)
        rows = torch.empty(2, 4 * 96, dtype=torch.bfloat16, device=DEV)
        with pytest.raises(rt.LcrError) as e:
            paged.chunk_attention(rows, rows.clone(), wide, wide, *rest, scale=0.1)
        assert e.value.status == 2 and len(paged._workspaces) == kept


@pytest.mark.parametrize("n,k,vocab", [(4, 2, 40), (4, 2, 128256), (300, 1, 50)])
def test_verify_drafts_rows_outside_the_target(n, k, vocab):
    """A request whose rows are not all among the target's is idle; the others
    are as without it."""
    g = torch.Generator(device=DEV).manual_seed(vocab)
    p = torch.softmax(torch.randn(n * (k + 1), vocab, generator=g, device=DEV), 1)
    starts = np.arange(n + 1) * (k + 1)
    drafts, counts = np.full((n, k), 3), np.full(n, k)
    u = torch.rand(n, k + 1, generator=g, device=DEV)
    want = run_verify(p, starts, drafts, counts, None, u)
    for where, bad in [(n, n * (k + 1) + 1), (n, 2 ** 30), (n, 2 ** 31 - 1), (0, -1), (0, -2 ** 31)]:
        at = starts.copy()
        at[where] = bad  # the last request passes the target's end, or the first begins before it
        got = run_verify(p, at, drafts, counts, None, u)
        idle = max(0, where - 1)
        others = np.arange(n) != idle
        assert (got[0][idle] == -1).all() and got[1][idle] == 0
        assert np.array_equal(got[0][others], want[0][others]) and np.array_equal(got[1][others], want[1][others])


def counting_case(lens, heads, kv_heads, d, ps, *, left_out=None):
    """Queries of zeros weigh all visible keys alike (1 each, exact), and key j
    has a one in dimension j // width: a dimension of the result is the share
    of the visible keys that fall to it. Returns the case and the 64-bit
    result, without the keys `left_out` of each request."""
    c = attention_case(lens, heads, kv_heads, d, ps)
    c["q"].zero_()
    want = torch.zeros(c["q"].shape[0], d, dtype=torch.float64, device=DEV)
    for b, (n, kv) in enumerate(lens):
        width = -(-kv // d)
        j = torch.arange(kv, device=DEV)
        page = torch.tensor(c["host_tables"][b].astype(np.int64), device=DEV)[j // ps]
        v = torch.nn.functional.one_hot(j // width, d)
        c["values"][page, :, j % ps] = v[:, None].bfloat16()
        if left_out is not None:
            v[left_out] = 0
        sums = v.double().cumsum(0)[kv - n:]
        r0 = int(c["host_starts"][b])
        want[r0:r0 + n] = sums / sums.sum(1, keepdim=True)
    return c, want[:, None].expand(-1, heads, -1).reshape(-1, heads * d)


@pytest.mark.parametrize("lens,heads,kv_heads,d,ps", [
    ([(1, 33000)], 1, 1, 64, 16), ([(1, 33000)], 1, 1, 128, 16), ([(1, 29001)], 1, 1, 64, 5),
    ([(5, 30001)], 4, 1, 128, 16), ([(130, 20011)], 4, 1, 64, 16), ([(3, 9000), (1, 15000), (300, 4000)], 8, 2, 64, 16),
    ([(2, 7000), (77, 5000)], 8, 2, 128, 16)])
def test_chunk_attention_counts_every_key(lens, heads, kv_heads, d, ps):
    """Sums of ones: the only roundings are those of 1 / l (2^-23), of the
    product with it (2^-24) and to bf16 (2^-8), so a result is within 2^-7.9 of
    the exact one (masked keys weigh 2^-125 at most); a block of keys left out,
    planted in the reference, is far outside that."""
    c, want = counting_case(lens, heads, kv_heads, d, ps)
    near = lambda x: bool(((x.double() - want).abs() <= want * 2.0 ** -7.9 + 2.0 ** -115).all())  # noqa: E731
    assert near(run_attention(c))
    assert not near(counting_case(lens, heads, kv_heads, d, ps, left_out=slice(1024, 1088))[1])


def one_request_reference(c, left_out=slice(0)):
    """The 64-bit result of a case of one request, without the keys left out."""
    (n, kv), d, group = c["lens"][0], c["d"], c["heads"] // c["kv_heads"]
    page = torch.tensor(c["host_tables"][0].astype(np.int64), device=DEV)
    k, v = (x[page].double().transpose(1, 2).reshape(-1, c["kv_heads"], d)[:kv] for x in (c["keys"], c["values"]))
    seen = torch.arange(kv, device=DEV)[None] <= torch.arange(kv - n, kv, device=DEV)[:, None]
    seen[:, left_out] = False
    out = []
    for h in range(c["heads"]):
        s = c["q"][:, h * d:(h + 1) * d].double() @ k[:, h // group].T / math.sqrt(d)
        out.append(torch.softmax(s.masked_fill(~seen, -math.inf), 1) @ v[:, h // group])
    return torch.cat(out, 1)


@pytest.mark.parametrize("lens,heads,kv_heads,d", [
    ([(1, 33000)], 1, 1, 64), ([(5, 30001)], 4, 1, 128), ([(130, 20011)], 4, 1, 64)])
def test_chunk_attention_rms_error(lens, heads, kv_heads, d):
    """With random values the roundings are random too. To bf16 each is half a
    unit in the last place at most, evenly spread: with leading digits m in
    [1, 2) 2^-8 / (sqrt(3) m), 2^-9.2 rms. The weights' and the output's own
    make 2^-8.7 of the result's rms together; 2^-8 is allowed. A bound on the largest error, which lets all roundings of a long
    row point one way, would hide a lost range; 320 keys left out of the
    reference show that this one does not."""
    c = attention_case(lens, heads, kv_heads, d, 16, seed=31)
    want = one_request_reference(c)
    rms = lambda x: float(x.square().mean().sqrt())  # noqa: E731
    assert rms(run_attention(c).double() - want) <= 2.0 ** -8 * rms(want)
    assert rms(one_request_reference(c, slice(1024, 1344)) - want) > 2.0 ** -8 * rms(want)
