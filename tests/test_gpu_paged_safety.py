"""What the paged cache's operators do where a caller or the cache's contents go wrong: values
that no row sees, bounds that are too small, tokens that belong to nobody, memory that overlaps.

Tolerances are those of test_gpu_paged.py (derived there)."""

import math

import pytest
import torch

from test_gpu_batch_decoder import close, decoder, model, prompt  # noqa: F401 (a fixture)
from test_gpu_paged import BF16, F16, F32, check, make, restate, run
from wisp_b200 import paged

pytestmark = pytest.mark.gpu


# ------------------------------------------------------------------------ hidden values
@pytest.mark.parametrize("dim,cache", [(64, F16), (128, BF16)])
@pytest.mark.parametrize("heads,window,sinks", [((8, 2), 0, 0), ((4, 4), 100, 70)])
def test_two_row_tiles_behind_one_tile_of_hidden_nans(cuda, dim, cache, heads, window, sinks):
    """Row tiles of more than 128 rows share each V tile: infinities and NaNs that no row sees
    (the ends of pages) are taken out of it before either half's product reads it."""
    for fill in (math.nan, math.inf):
        args = make([(260, 300), (129, 129), (64, 1000), (200, 333)], heads=heads, dim=dim,
                    page=48, cache=cache, fill=fill)
        first, _ = run(args, window=window, sinks=sinks)
        for _ in range(20):
            again = paged.attention(*args, window=window, sinks=sinks)
            assert torch.equal(again, first)


# ------------------------------------------------------------------------ waits that run out
def test_a_call_whose_waits_run_out_returns_and_says_so(cuda):
    """With no time to wait every role of the kernels gives up at some point of its work, whichever
    comes first: the call still ends, its status says it (or its result is right), and the next
    call with time finds everything in order."""
    decode = make([(1, 40000), (1, 17), (1, 9000), (3, 500)], heads=(32, 8), dim=128)
    rows32 = make([(1, 20000), (2, 300)], heads=(8, 2), dim=64, dtype=F32)
    prompt = make([(900, 3000), (70, 333), (4, 20000)], heads=(32, 8), dim=128, cache=BF16)
    split = make([(300, 2000)], heads=(8, 2), dim=64, dtype=F32, cache=BF16)
    seen = set()
    for args in (decode, rows32, prompt, split):
        q, k, v, batch = args
        ws = torch.empty(paged.workspace_bytes(q, k, v, batch), dtype=torch.uint8, device="cuda")
        want = restate(q, k, v, batch)
        before = paged.wait_limit(0)
        assert before == 2.0
        try:
            for _ in range(4):
                out, lse = paged.attention(q, k, v, batch, return_lse=True, workspace=ws)
                seen.add(paged.status(ws))
                if paged.status(ws) == 0:
                    check(out, lse, want, q.dtype, k.dtype)
        finally:
            assert paged.wait_limit(before) == 0.0
        run(args)
    assert seen <= {0, 8} and 8 in seen
    for bad in (-1.0, math.inf, math.nan):
        with pytest.raises(ValueError, match="wait_limit"):
            paged.wait_limit(bad)


# ------------------------------------------------------------------------ a step that fails
@pytest.mark.parametrize("where", ["attention", "rope_append", "stack"])
def test_a_step_that_failed_can_be_repeated(model, monkeypatch, where):  # noqa: F811
    """A failure in the second layer: the repeated step gives what a decoder gives that never failed."""
    p, q = prompt(40, 21), prompt(9, 22)
    fresh, dec = decoder(model), decoder(model)
    a, b = fresh.open(), fresh.open()
    fresh.step([(a, p[:20]), (b, q[:5])])
    want = fresh.step([(a, p[20:]), (b, q[5:])])
    a, b = dec.open(), dec.open()
    dec.step([(a, p[:20]), (b, q[:5])])
    owner = dec.stack if where == "stack" else paged
    real, calls = getattr(owner, where), []

    def fail(*args, **kw):
        calls.append(0)
        if len(calls) == 2:
            raise torch.cuda.OutOfMemoryError("no memory left")
        return real(*args, **kw)

    with monkeypatch.context() as m:
        m.setattr(owner, where, fail)
        with pytest.raises(torch.cuda.OutOfMemoryError):
            dec.step([(a, p[20:]), (b, q[5:])])
    assert len(calls) == 2 and dec.pool.length(a) == 20 and dec.pool.length(b) == 5
    close(dec.step([(a, p[20:]), (b, q[5:])]), want)


# ------------------------------------------------------------------------ bounds that are too small
@pytest.mark.parametrize("dim,heads,lens,max_q", [
    (64, (8, 2), [(1, 200 + 13 * i) for i in range(180)] + [(4, 9000)], 1),  # few rows, planned
    (64, (8, 2), [(1, 300), (4, 9000), (2, 40)], 1),                         # few rows
    (128, (8, 2), [(60, 20000), (3, 100)], 20),                              # tcgen05
    (128, (8, 2), [(300, 9000)], 33),
    (256, (8, 2), [(60, 20000), (3, 100)], 20),                              # wide heads
    (256, (8, 8), [(64, 9000)], 24)])
def test_more_tokens_than_max_q_are_done_or_reported(cuda, dim, heads, lens, max_q):
    q, k, v, good = make(lens, heads=heads, dim=dim)
    want = restate(q, k, v, good)
    batch = paged.TokenBatch(good.q_start, good.kv_len, good.table, max_q)
    ws = torch.empty(paged.workspace_bytes(q, k, v, batch), dtype=torch.uint8, device="cuda")
    out = torch.full_like(q, math.nan)
    _, lse = paged.attention(q, k, v, batch, out=out, return_lse=True, workspace=ws)
    assert paged.status(ws) in (0, 2)
    if paged.status(ws) == 0:
        check(out, lse, want, q.dtype, k.dtype)
    # what lies within the bound is done in any case
    starts = good.q_start.tolist()
    for s, (n, kv) in enumerate(lens):
        if n <= max_q:
            a, b = starts[s], starts[s + 1]
            check(out[a:b], lse[a:b], (want[0][a:b], want[1][a:b], *want[2:]), q.dtype, k.dtype)


def test_a_replayed_step_whose_tokens_pass_max_q_says_so(cuda):
    q, k, v, batch = make([(20, 9000), (20, 9000), (20, 9000)], heads=(8, 2), dim=128)
    ws = torch.empty(paged.workspace_bytes(q, k, v, batch), dtype=torch.uint8, device="cuda")
    out = torch.full_like(q, math.nan)
    graph = torch.cuda.CUDAGraph()
    paged.attention(q, k, v, batch, out=out, workspace=ws)
    with torch.cuda.graph(graph):
        paged.attention(q, k, v, batch, out=out, workspace=ws)
    graph.replay()
    assert paged.status(ws) == 0
    batch.q_start.copy_(torch.tensor([0, 1, 2, 60], dtype=torch.int32))
    graph.replay()
    if paged.status(ws) == 0:
        check(out, None, restate(q, k, v, batch), F16, F16)
    else:
        assert paged.status(ws) == 2


# ------------------------------------------------------------------------ tokens of nobody
@pytest.mark.parametrize("lens,dim,dtype", [
    ([(1, 30), (1, 2000)], 128, F32), ([(3, 90), (2, 700)], 64, F16), ([(70, 90), (200, 3000)], 128, F16),
    ([(70, 90), (200, 3000)], 64, F32), ([(70, 90), (40, 3000)], 256, F16)])
@pytest.mark.parametrize("groups", [False, True])
def test_rows_that_no_sequence_owns_are_zeros(cuda, lens, dim, dtype, groups):
    q, k, v, batch = make(lens, dim=dim, dtype=dtype)
    n = q.shape[0]
    q = torch.cat([q.new_full((3, *q.shape[1:]), math.nan), q, q.new_full((70, *q.shape[1:]), math.inf)])
    res = torch.full((n + 73, 10 * dim), 7.0, dtype=dtype, device="cuda")
    out = res[:, dim:9 * dim].unflatten(1, (8, dim))
    batch.q_start.add_(3)
    kw = {}
    call = paged.attention
    if groups:
        call = paged.prefix_attention
        kw = dict(groups=torch.tensor([0, 1], dtype=torch.int32, device="cuda"),
                  prefix_len=torch.tensor([16], dtype=torch.int32, device="cuda"))
    _, lse = call(q, k, v, batch, out=out, return_lse=True, **kw)
    for rows in (slice(0, 3), slice(n + 3, None)):
        assert not out[rows].any() and (lse[rows] == -math.inf).all()
    batch.q_start.sub_(3)
    check(out[3:n + 3], lse[3:n + 3], restate(q[3:n + 3], k, v, batch), dtype, k.dtype)
    assert (res[:, :dim] == 7).all() and (res[:, 9 * dim:] == 7).all()


def test_a_replayed_step_with_fewer_tokens_clears_the_rest(cuda):
    q, k, v, batch = make([(30, 300), (70, 500)], dim=128)
    ws = torch.empty(paged.workspace_bytes(q, k, v, batch), dtype=torch.uint8, device="cuda")
    out = torch.empty_like(q)
    graph = torch.cuda.CUDAGraph()
    paged.attention(q, k, v, batch, out=out, workspace=ws)
    with torch.cuda.graph(graph):
        paged.attention(q, k, v, batch, out=out, workspace=ws)
    graph.replay()
    batch.q_start[-1] -= 45
    graph.replay()
    assert paged.status(ws) == 0 and not out[55:].any()
    want = restate(q, k, v, batch)
    check(out[:55], None, (want[0][:55], want[1][:55], *want[2:]), F16, F16)


def test_a_call_without_tokens_has_a_status_of_its_own(cuda):
    q, k, v, batch = make([(1, 300), (70, 200)])
    ws = torch.empty(paged.workspace_bytes(q, k, v, batch), dtype=torch.uint8, device="cuda")
    batch.table[0, 3] = -1
    paged.attention(q, k, v, batch, workspace=ws)
    assert paged.status(ws) == 1
    none = paged.TokenBatch(batch.q_start[:1], batch.kv_len[:0], batch.table[:0], 0)
    paged.attention(q[:0], k, v, none, workspace=ws)
    assert paged.status(ws) == 0
    paged.attention(q[:0], k, v, none, workspace=ws[:0])


@pytest.mark.parametrize("dim,tokens", [(64, 1), (128, 200), (128, 3), (256, 40)])
@pytest.mark.parametrize("seen_inf", [False, True])
def test_positions_of_a_bad_page_read_as_zeros(cuda, dim, tokens, seen_inf):
    """The same for every kernel, and where a visible infinity has an item worked out again."""
    q, k, v, batch = make([(tokens, 700), (tokens, 333)], dim=dim)
    page = k.shape[1]
    k[-1], v[-1] = 0, 0
    spare = k.shape[0] - 1
    if (batch.table == spare).any():
        batch.table[batch.table == spare] = batch.table[0, 0].clone()
    if seen_inf:
        v[batch.table[0, 690 // page], 690 % page, 0, 3] = math.inf
    zeros = batch.table.clone()
    zeros[0, 3] = zeros[1, 1] = spare
    want = restate(q, k, v, paged.TokenBatch(batch.q_start, batch.kv_len, zeros, batch.max_q))
    batch.table[0, 3], batch.table[1, 1] = -1, 1 << 30
    ws = torch.empty(paged.workspace_bytes(q, k, v, batch), dtype=torch.uint8, device="cuda")
    out, lse = paged.attention(q, k, v, batch, return_lse=True, workspace=ws)
    assert paged.status(ws) == 1
    check(out, lse, want, F16, F16)


# ------------------------------------------------------------------------ failures that are seen
@pytest.mark.parametrize("lens,dim", [([(1, 300), (1, 40)], 64), ([(70, 300), (1, 200)], 128),
                                      ([(40, 300)], 256)])
def test_a_status_word_collects_the_bits_of_calls(cuda, lens, dim):
    q, k, v, batch = make(lens, dim=dim)
    word = torch.zeros(1, dtype=torch.int32, device="cuda")
    paged.attention(q, k, v, batch, status=word)
    groups = dict(groups=torch.tensor([0, 1], dtype=torch.int32, device="cuda"),
                  prefix_len=torch.tensor([16], dtype=torch.int32, device="cuda"))
    paged.prefix_attention(q, k, v, batch, status=word, **groups)
    assert word.item() == 0
    keep = batch.table[0, 3].clone()
    batch.table[0, 3] = -1
    paged.prefix_attention(q, k, v, batch, status=word, **groups)
    assert word.item() == 1
    batch.table[0, 3] = keep
    batch.kv_len[0] = 1 << 20
    paged.attention(q, k, v, batch, status=word)
    assert word.item() == 3
    for bad in (word.long(), word.cpu(), torch.zeros(2, dtype=torch.int32, device="cuda")):
        with pytest.raises(ValueError, match="status"):
            paged.attention(q, k, v, batch, status=bad)


def test_a_step_over_a_bad_page_raises(model, monkeypatch):  # noqa: F811
    dec, fresh = decoder(model), decoder(model)
    p = prompt(50, 31)
    a, b = dec.open(), fresh.open()
    dec.step([(a, p[:30])])
    fresh.step([(b, p[:30])])
    real = dec.pool.table

    def table(*args, **kw):
        t = real(*args, **kw)
        t[0, 1] = 1 << 20
        return t

    with monkeypatch.context() as m:
        m.setattr(dec.pool, "table", table)
        with pytest.raises(RuntimeError, match="page number outside the pool"):
            dec.step([(a, p[30:])])
    assert dec.pool.length(a) == 30
    close(dec.step([(a, p[30:])]), fresh.step([(b, p[30:])]))


# ------------------------------------------------------------------------ bits kept by the decoder
def test_logits_are_the_products_in_fp32(model, monkeypatch):  # noqa: F811
    """Products of 16-bit values are exact in fp32 and summed there: 2^-20 of the sum of sizes."""
    from wisp_b200 import batch_decoder
    dec, seen = decoder(model), []
    real = batch_decoder.rmsnorm
    monkeypatch.setattr(batch_decoder, "rmsnorm", lambda *a: seen.append(real(*a)) or seen[-1])
    got = dec.step([(dec.open(), prompt(30, 41)), (dec.open(), prompt(5, 42))]).double()
    y, w = seen[-1].half().double(), dec.lm_head.double()
    assert ((got - y @ w.T).abs() <= 2.0 ** -20 * (y.abs() @ w.abs().T)).all()


def test_fp32_rows_stay_near_the_one_sequence_step(model):  # noqa: F811
    """What is left is the rounding of the products' inputs: three in each of two layers and one in
    front of the logits, and the weights' own precision; eight times 2^-11."""
    from test_gpu_batch_decoder import one_by_one
    p, q = prompt(150, 51), prompt(33, 52)
    dec = decoder(model, rows=torch.float32)
    a, b = dec.open(), dec.open()
    dec.step([(a, p[:100]), (b, q[:32])])
    got = dec.step([(a, p[100:]), (b, q[32:])])
    want = torch.stack((one_by_one(model, p)[-1], one_by_one(model, q)[-1]))
    assert (got - want).norm() <= 8 * 2.0 ** -11 * want.norm()


def test_the_status_of_a_call_without_tokens_comes_after_the_call_before_it(cuda):
    """Both words are written by kernels in the stream's order, captured ones included."""
    q, k, v, batch = make([(1, 300), (70, 200)])
    ws = torch.empty(paged.workspace_bytes(q, k, v, batch), dtype=torch.uint8, device="cuda")
    none = paged.TokenBatch(batch.q_start[:1], batch.kv_len[:0], batch.table[:0], 0)
    batch.table[0, 3] = -1
    graph = torch.cuda.CUDAGraph()
    paged.attention(q, k, v, batch, workspace=ws)
    with torch.cuda.graph(graph):
        paged.attention(q, k, v, batch, workspace=ws)
        paged.attention(q[:0], k, v, none, workspace=ws)
    for _ in range(20):
        graph.replay()
        assert paged.status(ws) == 0
    other = torch.cuda.CUDAGraph()
    with torch.cuda.graph(other):
        paged.attention(q[:0], k, v, none, workspace=ws)
        paged.attention(q, k, v, batch, workspace=ws)
    for _ in range(20):
        other.replay()
        assert paged.status(ws) == 1
