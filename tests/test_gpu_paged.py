"""The paged cache's operators on the GPU against 64-bit restatements.

Tolerances, derived before the first run.  Attention: products of 16-bit rows are exact in
fp32, so a score is off by at most 2^-20 of A = max sum |q||k| scale (128 fp32 additions, in
practice far less); fp32 rows are split into parts that keep them to u2 = 2^-21 (fp16 cache)
or 2^-21 (bf16, three parts), which adds u2 A.  A score error d moves the result by at most
2 d max|v|.  16-bit rows also round the weights and the result: u = 2^-11 (fp16) or 2^-8
(bf16) of max|v| each.  lse: the score error plus 2^-20 of its size.  Rotary: one fp32
rounding of the sine and cosine and of the products, 2^-21 of the row's largest, plus the
output type's rounding.
"""

import math

import pytest
import torch

from wisp_b200 import paged
from wisp_b200.lib import WispError

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
UNIT = {F16: 2.0 ** -11, BF16: 2.0 ** -8}


def make(lens, heads=(8, 2), dim=64, page=16, cache=F16, dtype=None, seed=0, spare=3, shared=0,
         fill=float("nan")):
    """A batch with lens = [(tokens, cached positions)]: pages in random order, everything the
    sequences do not hold set to `fill`.  shared: positions (whole pages) of one common prefix."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    nh, nkv = heads
    T = sum(n for n, _ in lens)
    per = [-(-kv // page) for _, kv in lens]
    sh = shared // page
    n_pages = sh + sum(p - sh for p in per if p > sh) + spare
    perm = torch.randperm(n_pages, generator=g, device="cuda").tolist()
    rows, at = [], sh
    for p in per:
        fresh = max(0, p - sh)
        rows.append((perm[:sh] + perm[at:at + fresh])[:max(p, 0)])
        at += fresh
    width = max([1] + per)
    table = torch.tensor([r + [0] * (width - len(r)) for r in rows], dtype=torch.int32).cuda()
    k = torch.randn(n_pages, page, nkv, dim, generator=g, device="cuda").to(cache)
    v = torch.randn(n_pages, page, nkv, dim, generator=g, device="cuda").to(cache)
    held = torch.zeros(n_pages, page, dtype=torch.bool, device="cuda")
    for (_, kv), r in zip(lens, rows):
        for i in range(kv):
            if i % page == 0 or i == kv - 1:
                held[r[i // page], :min(page, kv - i // page * page)] = True
    k[~held] = fill
    v[~held] = fill
    q = torch.randn(T, nh, dim, generator=g, device="cuda").to(dtype or cache)
    starts = torch.tensor([0] + [n for n, _ in lens]).cumsum(0).to(torch.int32).cuda()
    kv_len = torch.tensor([kv for _, kv in lens], dtype=torch.int32).cuda()
    batch = paged.TokenBatch(starts, kv_len, table, max([1] + [n for n, _ in lens]))
    return q, k, v, batch


def restate(q, k, v, batch, window=0, sinks=0, scale=None):
    """The definition in float64, sequence by sequence: (out, lse, A, max |v|)."""
    nh, dim, nkv = q.shape[1], q.shape[2], k.shape[2]
    page, G = k.shape[1], nh // nkv
    scale = dim ** -0.5 if scale is None else scale
    out = torch.zeros(q.shape, dtype=torch.float64, device="cuda")
    lse = torch.full(q.shape[:2], -math.inf, dtype=torch.float64, device="cuda")
    A = vm = 1e-30
    starts = batch.q_start.tolist()
    for s, kv in enumerate(batch.kv_len.tolist()):
        t0, t1 = starts[s], starts[s + 1]
        if t0 == t1 or kv == 0:
            continue
        j = torch.arange(kv, device="cuda")
        rows = batch.table[s].long()[j // page]
        K, V = k[rows, j % page].double(), v[rows, j % page].double()
        i = torch.arange(kv - (t1 - t0), kv, device="cuda")[:, None]
        seen = j[None] <= i
        if window:
            seen &= (i - j[None] < window) | (j[None] < sinks)
        fine = torch.isfinite(V)
        vm = max(vm, V[fine].abs().max().item())
        for h in range(nh):
            x = q[t0:t1, h].double() @ K[:, h // G].T * scale
            a = (q[t0:t1, h].double().abs() @ K[:, h // G].nan_to_num(0, 0, 0).abs().T) * scale
            A = max(A, a.max().item())
            x = torch.where(seen, x, -math.inf)
            z = torch.logsumexp(x, 1)
            p = torch.where(seen, torch.exp(x - torch.where(z.isinf(), 0.0, z)[:, None]), 0.0)
            # hidden values take no part: 0 * NaN is not added
            o = p @ torch.where(fine[:, h // G], V[:, h // G], 0.0)
            for jj in (~fine[:, h // G]).any(1).nonzero().flatten().tolist():
                see = seen[:, jj]
                o[see] += torch.where(fine[jj, h // G], 0.0, V[jj, h // G] * 1.0)
            out[t0:t1, h], lse[t0:t1, h] = o, z
    return out, lse, A, vm


def check(got, lse, want, dtype, cache):
    o, z, A, vm = want
    d = 2.0 ** -20 * A + (2.0 ** -21 * A if dtype == F32 else 0.0)
    tol = (2 * d + 2.0 ** -20 + (2 * UNIT[cache] if dtype != F32 else 0.0)) * vm
    g = got.double()
    nan = o.isnan()
    assert torch.equal(g.isnan(), nan)
    inf = o.isinf()
    assert torch.equal(g[inf], o[inf])
    ok = ~nan & ~inf
    err = (g - o)[ok].abs().max().item() if ok.any() else 0.0
    assert err <= tol, (err, tol)
    if lse is not None:
        empty = z.isinf()
        assert torch.equal(lse.double()[empty], z[empty])
        zt = d + 2.0 ** -20 * (1 + z[~empty].abs())
        assert ((lse.double() - z)[~empty].abs() <= zt).all()


def run(args, dtype=None, window=0, sinks=0, **kw):
    q, k, v, batch = args
    ws = torch.empty(paged.workspace_bytes(q, k, v, batch), dtype=torch.uint8, device="cuda")
    out, lse = paged.attention(q, k, v, batch, window=window, sinks=sinks, return_lse=True,
                               workspace=ws, **kw)
    assert paged.status(ws) == 0
    check(out, lse, restate(q, k, v, batch, window, sinks, kw.get("scale")), q.dtype, k.dtype)
    return out, lse


ONE = [(1, 1)]
DECODE = [(1, 1), (1, 17), (1, 64), (1, 65), (1, 700), (1, 0), (1, 128)]
FEW = [(3, 3), (2, 130), (5, 64), (4, 700), (1, 9), (3, 0)]
PROMPT = [(1, 1), (200, 200), (63, 64), (70, 333), (129, 129)]


# ------------------------------------------------------------------------ attention
@pytest.mark.parametrize("dtype,cache", [(F16, F16), (BF16, BF16), (F32, F16), (F32, BF16)])
@pytest.mark.parametrize("lens", [ONE, DECODE, FEW, PROMPT], ids=["one", "decode", "few", "prompt"])
@pytest.mark.parametrize("window,sinks", [(0, 0), (1, 0), (50, 3), (64, 64), (130, 70)])
def test_lengths_types_windows(cuda, dtype, cache, lens, window, sinks):
    run(make(lens, dtype=dtype, cache=cache), window=window, sinks=sinks)


@pytest.mark.parametrize("heads", [(1, 1), (4, 4), (6, 2), (5, 1), (16, 1), (17, 1), (40, 2),
                                   (71, 1), (24, 8), (12, 3)])
@pytest.mark.parametrize("dtype", [F16, F32])
def test_head_layouts(cuda, heads, dtype):
    run(make(DECODE + [(7, 40)], heads=heads, dtype=dtype))
    run(make([(90, 100), (1, 50)], heads=heads, dtype=dtype, dim=128), window=33, sinks=2)


@pytest.mark.parametrize("dim", [8, 16, 40, 64, 72, 96, 128, 136, 192, 256])
@pytest.mark.parametrize("dtype,cache", [(F16, F16), (F32, BF16)])
def test_head_dims(cuda, dim, dtype, cache):
    run(make(DECODE, dim=dim, dtype=dtype, cache=cache))
    run(make(PROMPT, dim=dim, dtype=dtype, cache=cache), window=100, sinks=5)


@pytest.mark.parametrize("page", [8, 16, 24, 32, 48, 64, 80, 128, 256])
def test_page_sizes(cuda, page):
    run(make(DECODE, page=page))
    run(make(PROMPT, page=page, dim=128, cache=BF16), window=77, sinks=9)


@pytest.mark.parametrize("cache", [F16, BF16])
@pytest.mark.parametrize("dtype", [F32, None])
def test_long_cache_split_over_many_ctas(cuda, cache, dtype):
    run(make([(1, 20011)], heads=(8, 1), dim=128, cache=cache, dtype=dtype))
    run(make([(4, 9001), (1, 3), (33, 12000)], heads=(4, 2), dim=128, cache=cache, dtype=dtype),
        window=5000, sinks=100)


def test_peaked_and_flat_rows(cuda):
    """Weights from 1 down to what exp underflows to, and rows of one repeated key."""
    q, k, v, batch = make([(1, 3000), (64, 700)], dim=128, dtype=F32)
    run((q * 12, k, v, batch))
    k[:] = torch.where(k.isnan(), k, k[0, 0, 0, 0].nan_to_num(1.0))
    run((q, k, v, batch))


@pytest.mark.parametrize("big", [1e-4, 3e5])
def test_fp32_rows_outside_the_range_of_fp16(cuda, big):
    q, k, v, batch = make(DECODE + PROMPT, dtype=F32)
    run((q * big, k, v, batch), scale=0.125 / big)


def test_more_tokens_than_positions_and_unused_slots(cuda):
    out, lse = run(make([(5, 2), (1, 0), (4, 0), (2, 2), (0, 40), (1, 40)]))
    assert not out[:3].any() and not out[5:10].any()
    assert (lse[:3] == -math.inf).all() and (lse[5:10] == -math.inf).all()


@pytest.mark.parametrize("dim,cache", [(64, F16), (128, BF16), (128, F16)])
def test_hidden_infinities_and_nans_stay_hidden(cuda, dim, cache):
    """The last tokens of prompts hold infinities and NaNs: only they and what follows see them.
    Every position that a window has left behind holds NaN."""
    q, k, v, batch = make([(150, 150), (70, 300), (2, 90)], dim=dim, cache=cache)
    page = k.shape[1]
    for s, (p, val) in enumerate([(149, math.nan), (299, math.inf), (89, math.nan)]):
        v[batch.table[s, p // page], p % page, 0, 3] = val
    v[batch.table[0, 120 // page], 120 % page, 1, 5] = -math.inf
    v[batch.table[0, 121 // page], 121 % page, 1, 5] = math.inf
    k[batch.table[1, 299 // page], 299 % page, 1, 0] = math.nan
    q2, k2, v2, b2 = make([(1, 500), (3, 400)], dim=dim, cache=cache)
    for s, kv in ((0, 500), (1, 398)):
        for p in range(10, kv - 100):
            k2[b2.table[s, p // page], p % page] = math.nan
            v2[b2.table[s, p // page], p % page] = math.nan
    out, lse = paged.attention(q, k, v, batch, return_lse=True)
    o, z, A, vm = restate(q, k.nan_to_num(0), v, batch)
    seen_bad_k = torch.zeros(q.shape[:2], dtype=torch.bool, device="cuda")
    seen_bad_k[219, k.shape[2] and q.shape[1] // 2:] = True
    assert out[seen_bad_k].isnan().all() and lse[seen_bad_k].isnan().all()
    out[seen_bad_k] = o[seen_bad_k].to(out.dtype)
    lse[seen_bad_k] = z[seen_bad_k].float()
    check(out, lse, (o, z, A, vm), q.dtype, k.dtype)
    run((q2, k2, v2, b2), window=100, sinks=10)


def test_strided_rows(cuda):
    q, k, v, batch = make(FEW + PROMPT, dim=64)
    T = q.shape[0]
    fused = torch.zeros(T, 12 * 64, dtype=F16, device="cuda")
    view = fused[:, 2 * 64:10 * 64].unflatten(1, (8, 64))
    view.copy_(q)
    res = torch.zeros(T, 10 * 64, dtype=F16, device="cuda")
    out = res[:, 64:9 * 64].unflatten(1, (8, 64))
    got = paged.attention(view, k, v, batch, out=out)
    assert got.data_ptr() == out.data_ptr()
    assert torch.equal(got, paged.attention(q, k, v, batch))
    assert not res[:, :64].any() and not res[:, 9 * 64:].any()


def test_pages_inside_a_larger_pool(cuda):
    """One layer of a pool whose pages hold all layers: the page stride is not a page."""
    q, k, v, batch = make(DECODE)
    pool = torch.full((2, k.shape[0], 3, *k.shape[1:]), math.nan, dtype=F16, device="cuda")
    pool[0, :, 1], pool[1, :, 1] = k, v
    assert torch.equal(paged.attention(q, pool[0, :, 1], pool[1, :, 1], batch),
                       paged.attention(q, k, v, batch))


def test_offsets_past_32_bits(cuda):
    n, page, nkv, dim = 300_000, 16, 8, 128  # 4.9e9 elements
    k = torch.empty(n, page, nkv, dim, dtype=F16, device="cuda")
    v = torch.empty_like(k)
    _, ks, vs, small = make([(1, 40), (17, 50)], heads=(8, 8), dim=dim)
    ids = [n - 1 - 7 * i for i in range(ks.shape[0])]
    at = torch.tensor(ids, device="cuda")
    k[at], v[at] = ks, vs
    batch = paged.TokenBatch(small.q_start, small.kv_len, at.int()[small.table.long()], 17)
    q = torch.randn(18, 16, dim, device="cuda", dtype=F16)
    assert torch.equal(paged.attention(q, k, v, batch), paged.attention(q, ks, vs, small))
    rows = torch.randn(18, 8, dim, device="cuda", dtype=F16)
    f, _ = paged.rope_frequencies(dim, device="cuda")
    q1 = paged.rope_append(q, rows, rows, k, v, batch, f)
    q2 = paged.rope_append(q, rows, rows, ks, vs, small, f)
    assert torch.equal(q1, q2) and torch.equal(k[at][~ks.isnan()], ks[~ks.isnan()])
    paged.copy_pages(k, v, [ids[0]], [n - 2])
    assert torch.equal(v[n - 2].view(torch.int16), v[ids[0]].view(torch.int16))


def test_results_do_not_depend_on_the_run(cuda):
    q, k, v, batch = make([(1, 5000), (40, 900), (1, 30)], dim=128)
    first = paged.attention(q, k, v, batch)
    side = torch.cuda.Stream()
    for _ in range(5):
        assert torch.equal(paged.attention(q, k, v, batch), first)
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            other = paged.attention(q, k, v, batch)
        torch.cuda.current_stream().wait_stream(side)
        assert torch.equal(other, first)


def test_a_captured_step_follows_the_lengths(cuda):
    q, k, v, batch = make([(1, 300), (1, 500)], dim=128, spare=40)
    ws = torch.empty(paged.workspace_bytes(q, k, v, batch), dtype=torch.uint8, device="cuda")
    out = torch.empty_like(q)
    paged.attention(q, k, v, batch, out=out, workspace=ws)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        paged.attention(q, k, v, batch, out=out, workspace=ws)
    batch.kv_len.copy_(torch.tensor([17, 499], dtype=torch.int32))
    graph.replay()
    check(out, None, restate(q, k, v, batch), F16, F16)


def test_bad_tables_and_lengths_are_reported(cuda):
    q, k, v, batch = make([(1, 300), (70, 200)])
    ws = torch.empty(paged.workspace_bytes(q, k, v, batch), dtype=torch.uint8, device="cuda")
    batch.table[0, 3] = k.shape[0]
    batch.table[1, 0] = -1
    paged.attention(q, k, v, batch, workspace=ws)
    assert paged.status(ws) == 1
    q, k, v, batch = make([(1, 300), (70, 200)])
    batch.kv_len[0] = 1 << 30
    paged.attention(q, k, v, batch, workspace=ws)
    assert paged.status(ws) == 2
    batch.kv_len[0] = -5
    batch.q_start[1] = 1 << 20
    paged.attention(q, k, v, batch, workspace=ws)
    word = torch.zeros(1, dtype=torch.int32, device="cuda")
    q, k, v, batch = make([(2, 300)])
    batch.table[0, 300 // 16] = 1 << 20
    before = k.clone()
    rows = torch.ones(2, 2, 64, device="cuda", dtype=F16)
    f, _ = paged.rope_frequencies(64, device="cuda")
    got = paged.rope_append(q, rows, rows, k, v, batch, f, status=word)
    assert word.item() == 1 and not got.any()
    assert torch.equal(k.view(torch.int16), before.view(torch.int16))


def test_python_refusals(cuda):
    q, k, v, batch = make(DECODE)
    with pytest.raises(ValueError, match="heads must be contiguous"):
        paged.attention(q[:, ::2], k, v, batch)
    with pytest.raises(ValueError, match="one shape"):
        paged.attention(q, k, v[:-1], batch)
    with pytest.raises(ValueError, match="is wanted"):
        paged.attention(q[..., :32], k, v, batch)
    with pytest.raises(WispError, match=r"\[4\].*dtype"):
        paged.attention(q.bfloat16(), k, v, batch)
    with pytest.raises(WispError, match=r"\[4\].*workspace"):
        paged.attention(q, k, v, batch, workspace=torch.empty(64, dtype=torch.uint8, device="cuda"))
    with pytest.raises(ValueError, match="q_start has"):
        paged.TokenBatch(batch.q_start[:-1], batch.kv_len, batch.table, 1)
    with pytest.raises(ValueError, match="float64"):
        paged.rope_append(q, q[:, :2], q[:, :2], k, v, batch, torch.ones(32, device="cuda"))
    with pytest.raises(ValueError, match="groups of"):
        paged.prefix_attention(q, k, v, batch, batch.kv_len, batch.kv_len)
    with pytest.raises(WispError, match="twice a destination"):
        paged.copy_pages(k, v, [0, 1], [2, 2])
    with pytest.raises(ValueError, match="1 sources"):
        paged.copy_pages(k, v, [0], [2, 3])


@pytest.mark.parametrize("scale", [-0.2, 0.0, 1e-30])
@pytest.mark.parametrize("dtype,dim", [(F16, 64), (F32, 128), (F16, 40)])
def test_scales_below_and_at_zero(cuda, scale, dtype, dim):
    """A negative scale is the positive one on the negated rows (whose bound A the check takes)."""
    for lens, window, sinks in ((DECODE + [(3, 40)], 0, 0), (PROMPT, 60, 2)):
        q, k, v, batch = make(lens, dim=dim, dtype=dtype)
        out, lse = paged.attention(q, k, v, batch, window=window, sinks=sinks, scale=scale,
                                   return_lse=True)
        same = restate(q if scale >= 0 else -q, k, v, batch, window, sinks, abs(scale))
        check(out, lse, same, dtype, k.dtype)


@pytest.mark.parametrize("n", [511, 513, 1500])
def test_many_sequences(cuda, n):
    """More sequences than the attention kernel counts by itself, than a plan's block has threads."""
    run(make([(1, 1 + 7 * i % 90) for i in range(n)], heads=(4, 2)))
    run(make([(1 + i % 20, 20 + 7 * i % 90) for i in range(n)], heads=(4, 2)))


@pytest.mark.parametrize("n,heads", [(15, (160, 160)), (33, (160, 160)), (40, (160, 160)),
                                     (159, (4, 2)), (160, (4, 2)), (161, (4, 2))])
def test_many_short_sequences_in_one_piece(cuda, n, heads):
    """With 160 kv heads a CTA takes half of the line: more row tiles than it holds records of at a
    time; and about as many row tiles as a CTA counts by itself."""
    run(make([(1, 1 + 13 * i % 150) for i in range(n)], heads=heads, dim=16))
    run(make([(1, 13 * i % 150) for i in range(n)], heads=heads, dim=16), window=20, sinks=2)


@pytest.mark.parametrize("heads", [(1, 1), (2, 2), (4, 1), (12, 3)])
@pytest.mark.parametrize("lens", [[(300, 300), (100, 900), (257, 700), (5, 3000)],
                                  [(20, 4000), (129, 129), (128, 2000)],
                                  [(257, 257)], [(33, 33), (600, 2500), (1, 1), (31, 5000)]])
@pytest.mark.parametrize("window,sinks", [(0, 0), (200, 5)])
def test_row_tiles_of_full_and_half_size_on_one_line(cuda, heads, lens, window, sinks):
    """Few heads: many short pieces, whose ends fall between and inside the row tiles."""
    run(make(lens, heads=heads, dim=128, page=32), window=window, sinks=sinks)
    run(make(lens, heads=heads, dim=64, cache=BF16, page=16), window=window, sinks=sinks)


@pytest.mark.parametrize("dim", [64, 72, 128, 256])
@pytest.mark.parametrize("n,tokens", [(3, 8), (4, 16), (2, 33)])
def test_few_row_tiles_behind_small_and_large_tables(cuda, dim, n, tokens):
    """Both sides of the choice between the kernels for few and for many rows."""
    args = make([(tokens, 40 + 300 * i) for i in range(n)], heads=(8, 2), dim=dim)
    run(args)
    q, k, v, batch = args
    wide = torch.zeros(n, 9000, dtype=torch.int32, device="cuda")
    wide[:, :batch.table.shape[1]] = batch.table
    run((q, k, v, paged.TokenBatch(batch.q_start, batch.kv_len, wide, batch.max_q)))


@pytest.mark.parametrize("tokens,heads,dim", [(1, (2, 2), 128), (1, (1, 1), 256), (20, (16, 2), 128),
                                              (20, (16, 2), 64), (5, (40, 2), 256)])
@pytest.mark.parametrize("cache", [F16, BF16])
def test_fp32_rows_keep_their_size_over_long_caches(cuda, tokens, heads, dim, cache):
    """Sums that are cut off instead of rounded shrink with every instruction.  v = 1 + a small part:
    all of a row's outputs are near one, and what they miss on average is the shrinking.  With 12
    instructions (three parts of 64 positions) times four KV tiles a sum loses at most
    48 * 2^-23, a score of size A 24 * 2^-23 A more in the exponent's unit."""
    q, k, v, batch = make([(tokens, 12000)], heads=heads, dim=dim, page=64, cache=cache, dtype=F32)
    v = (1 + v.double().nan_to_num() / 64).to(cache)
    q = q * 0.01
    want, _, A, _ = restate(q, k, v, batch)
    got = paged.attention(q, k, v, batch).double()
    assert A < 0.5
    assert abs(((got - want) / want).mean().item()) < (48 + 24 * A) * 2.0 ** -23


@pytest.mark.parametrize("dtype,dim", [(F16, 64), (F16, 40), (F32, 64), (F16, 128)])
def test_rows_that_leave_at_odd_places(cuda, dtype, dim):
    """Outputs at 16 bytes past a 32-byte boundary."""
    q, k, v, batch = make([(150, 200), (40, 700)], heads=(6, 2), dim=dim, dtype=dtype)
    n, nh = q.shape[:2]
    skip = 16 // q.element_size()
    flat = torch.empty(n * nh * dim + 2 * skip, dtype=q.dtype, device="cuda")
    out = flat[skip:skip + n * nh * dim].view(n, nh, dim)
    assert out.data_ptr() % 32 == 16
    got, lse = paged.attention(q, k, v, batch, return_lse=True, out=out)
    assert got.data_ptr() == out.data_ptr()
    check(out, lse, restate(q, k, v, batch), q.dtype, k.dtype)


@pytest.mark.parametrize("heads", [(160, 160), (300, 150)])
def test_more_heads_than_sms(cuda, heads):
    run(make([(1, 70), (1, 300)], heads=heads))
    run(make([(40, 70), (2, 300)], heads=heads))


def test_a_table_that_is_part_of_a_wider_one(cuda):
    q, k, v, batch = make(DECODE + [(20, 90)], dim=128)
    n, w = batch.table.shape
    wide = torch.full((n, w + 9), 1 << 30, dtype=torch.int32, device="cuda")
    wide[:, 4:4 + w] = batch.table
    other = paged.TokenBatch(batch.q_start, batch.kv_len, wide[:, 4:4 + w], batch.max_q)
    assert torch.equal(paged.attention(q, k, v, other), paged.attention(q, k, v, batch))
    batch.kv_len[4] = 1 << 20  # the longest: cut to the table's width, not to its stride
    ws = torch.empty(paged.workspace_bytes(q, k, v, other), dtype=torch.uint8, device="cuda")
    paged.attention(q, k, v, other, workspace=ws)
    assert paged.status(ws) == 2


@pytest.mark.parametrize("lens", [[(30, 300), (70, 500)], [(20, 4000)]])
def test_a_captured_prompt_follows_the_lengths(cuda, lens):
    q, k, v, batch = make(lens, dim=128)
    ws = torch.empty(paged.workspace_bytes(q, k, v, batch), dtype=torch.uint8, device="cuda")
    out = torch.empty_like(q)
    paged.attention(q, k, v, batch, out=out, workspace=ws)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        paged.attention(q, k, v, batch, out=out, workspace=ws)
    batch.kv_len.sub_(9)
    graph.replay()
    check(out, None, restate(q, k, v, batch), F16, F16)
    batch.q_start[-1] -= 5  # five rows of padding at the end
    graph.replay()
    check(out[:-5], None, tuple(x[:-5] if isinstance(x, torch.Tensor) else x for x in
                                restate(q, k, v, batch)), F16, F16)


def test_no_tokens(cuda):
    q, k, v, batch = make(DECODE)
    none = paged.TokenBatch(batch.q_start[:1], batch.kv_len[:0], batch.table[:0], 0)
    assert paged.attention(q[:0], k, v, none).shape == (0, 8, 64)
    f, _ = paged.rope_frequencies(64, device="cuda")
    assert paged.rope_append(q[:0], q[:0, :2], q[:0, :2], k, v, none, f).shape == (0, 8, 64)


def test_rows_that_ask_for_a_gradient_are_refused(cuda):
    q, k, v, batch = make(DECODE)
    with pytest.raises(ValueError, match="gradient"):
        paged.attention(q.requires_grad_(), k, v, batch)
    with torch.no_grad():
        paged.attention(q, k, v, batch)


# ------------------------------------------------------------------------ shared prefixes
def prefix_run(args, groups, prefix, window=0, sinks=0):
    q, k, v, batch = args
    g = torch.tensor(groups, dtype=torch.int32, device="cuda")
    p = torch.tensor(prefix, dtype=torch.int32, device="cuda")
    ws = torch.empty(paged.workspace_bytes(q, k, v, batch, len(prefix)), dtype=torch.uint8,
                     device="cuda")
    out, lse = paged.prefix_attention(q, k, v, batch, g, p, window=window, sinks=sinks,
                                      return_lse=True, workspace=ws)
    assert paged.status(ws) == 0
    check(out, lse, restate(q, k, v, batch, window, sinks), q.dtype, k.dtype)


@pytest.mark.parametrize("dtype,cache", [(F16, F16), (BF16, BF16), (F32, F16), (F32, BF16)])
@pytest.mark.parametrize("window,sinks", [(0, 0), (90, 4), (400, 0)])
def test_prefix_one_group(cuda, dtype, cache, window, sinks):
    lens = [(1, 320 + n) for n in (1, 5, 16, 17, 100, 64, 3)]
    prefix_run(make(lens, shared=320, dtype=dtype, cache=cache), [0, 7], [320], window, sinks)


@pytest.mark.parametrize("heads,dim", [((8, 2), 64), ((32, 8), 128), ((3, 3), 96), ((20, 1), 128)])
def test_prefix_many_sequences_and_tokens(cuda, heads, dim):
    prefix_run(make([(1, 1000 + 7 * i) for i in range(1, 41)], shared=992, heads=heads, dim=dim),
               [0, 40], [992])
    prefix_run(make([(3, 500), (70, 600), (1, 499), (2, 482)], shared=480, heads=heads, dim=dim),
               [0, 4], [480])


def test_prefix_groups_gaps_and_short_ones(cuda):
    """Groups that leave sequences out, an empty group, prefixes of nothing, longer than a
    sequence, and that end inside a page."""
    args = make([(1, 200), (1, 190), (1, 33), (1, 0), (2, 260), (1, 161)], shared=160)
    prefix_run(args, [0, 2], [160])
    prefix_run(args, [1, 2], [150])
    prefix_run(args, [0, 6], [0])
    prefix_run(args, [0, 2, 2, 6], [160, 5, 7])
    prefix_run(make([(1, 100), (1, 48), (3, 49)], shared=48), [0, 3], [48])


def test_prefix_of_the_whole_cache(cuda):
    prefix_run(make([(1, 64), (1, 64), (1, 64)], shared=64), [0, 3], [64])


# ------------------------------------------------------------------------ rotary, append
def rope64(x, pos, f, offset, interleaved, gain):
    r = 2 * f.shape[0]
    y = x.double().clone()
    ang = pos.double()[:, None] * f
    c, s = (ang.cos() * gain)[:, None], (ang.sin() * gain)[:, None]
    w = y[..., offset:offset + r].clone()
    a, b = (w[..., ::2], w[..., 1::2]) if interleaved else (w[..., :r // 2], w[..., r // 2:])
    p, q = a * c - b * s, b * c + a * s
    y[..., offset:offset + r] = torch.stack((p, q), -1).flatten(-2) if interleaved \
        else torch.cat((p, q), -1)
    return y


@pytest.mark.parametrize("dtype,cache,q_dtype", [(F32, F16, F32), (F32, BF16, F32), (F32, F16, F16),
                                                 (F16, F16, F16), (BF16, BF16, BF16),
                                                 (F16, BF16, F16), (BF16, F16, F16)])
@pytest.mark.parametrize("dim,rot,offset", [(64, 64, 0), (128, 64, 0), (128, 32, 96), (96, 48, 8),
                                            (256, 256, 0), (72, 16, 56), (64, 0, 0)])
@pytest.mark.parametrize("interleaved", [False, True])
def test_rope_append(cuda, dtype, cache, q_dtype, dim, rot, offset, interleaved):
    lens = [(1, 1), (3, 40), (0, 5), (20, 20), (1, 0), (2, 1)]
    q, k, v, batch = make(lens, heads=(6, 2), dim=dim, cache=cache, dtype=dtype, fill=7.0)
    T = q.shape[0]
    kn, vn = (torch.randn(T, 2, dim, device="cuda").to(dtype) for _ in range(2))
    f, _ = paged.rope_frequencies(max(rot, 2), 10000.0, device="cuda")
    f = f[:rot // 2].contiguous()
    gain = 1.25
    starts = batch.q_start.tolist()
    seq = torch.tensor([s for s in range(len(lens)) for _ in range(lens[s][0])], device="cuda")
    pos = torch.tensor([lens[s][1] - (starts[s + 1] - t) for t, s in enumerate(seq.tolist())],
                       device="cuda")
    qo = torch.full((T, 6, dim), 9.0, dtype=q_dtype, device="cuda")
    k0, v0 = k.clone(), v.clone()
    paged.rope_append(q, kn, vn, k, v, batch, f, q_out=qo, offset=offset, interleaved=interleaved,
                      gain=gain)
    ok = pos >= 0
    want_q = rope64(q, pos, f, offset, interleaved, gain)
    want_k = rope64(kn, pos, f, offset, interleaved, gain)
    u = lambda t: UNIT.get(t, 0.0) + 2.0 ** -21  # noqa: E731
    big = want_q.abs().max().item()
    assert (qo.double() - want_q)[ok].abs().max().item() <= u(q_dtype) * big
    assert not qo[~ok].any()
    page = batch.table.long()[seq[ok], pos[ok] // 16]
    got_k, got_v = k[page, pos[ok] % 16], v[page, pos[ok] % 16]
    assert (got_k.double() - want_k[ok]).abs().max().item() <= u(cache) * big
    assert torch.equal(got_v, vn[ok].to(cache))
    k0[page, pos[ok] % 16], v0[page, pos[ok] % 16] = got_k, got_v
    assert torch.equal(k, k0) and torch.equal(v, v0)


def test_rope_at_long_positions_and_given_positions(cuda):
    q, k, v, batch = make([(1, 30), (4, 33)], dim=128, dtype=F32)
    f, gain = paged.rope_frequencies(128, 1e6, scaling="by_parts", factor=16.0, device="cuda")
    pos = torch.tensor([0, 131071, 5_000_000, 2 ** 30 + 1, 77], dtype=torch.int32, device="cuda")
    rows = torch.randn(5, 2, 128, device="cuda")
    got = paged.rope_append(q, rows, rows, k, v, batch, f, gain=gain, positions=pos)
    want = rope64(q, pos, f, 0, False, gain)
    assert (got.double() - want).abs().max().item() <= 2.0 ** -20 * want.abs().max().item()
    again = q.clone()
    paged.rope_append(again, rows, rows, k, v, batch, f, gain=gain, positions=pos, q_out=again)
    assert torch.equal(again, got)


def test_rope_of_many_tokens_and_strided_rows(cuda):
    q, k, v, batch = make([(700, 700), (300, 1000)], heads=(8, 2), dim=64, cache=BF16)
    fused = torch.randn(1000, 12 * 64, device="cuda").bfloat16()
    a, b, c = (fused[:, x * 64:y * 64].unflatten(1, (y - x, 64)) for x, y in
               ((0, 8), (8, 10), (10, 12)))
    f, _ = paged.rope_frequencies(64, device="cuda")
    got = paged.rope_append(a, b, c, k, v, batch, f)
    pos = torch.cat((torch.arange(700), torch.arange(700, 1000))).cuda()
    want = rope64(a, pos, f, 0, False, 1.0)
    assert (got.double() - want).abs().max().item() <= 2.0 ** -8 * want.abs().max().item()


@pytest.mark.parametrize("heads,dim,tokens", [((80, 16), 256, 40), ((6, 2), 64, 3001), ((64, 8), 128, 1700)])
def test_rope_of_wide_rows_and_long_batches(cuda, heads, dim, tokens):
    """More units than a CTA's threads hold, more tokens than CTAs, and many sequences."""
    lens = [(1, 9)] * 40 + [(tokens - 40, tokens - 30)] if tokens > 40 else [(tokens, tokens)]
    q, k, v, batch = make(lens, heads=heads, dim=dim, dtype=F32)
    T = q.shape[0]
    rows = torch.randn(T, heads[1], dim, device="cuda")
    f, _ = paged.rope_frequencies(dim // 2, 10000.0, device="cuda")
    got = paged.rope_append(q, rows, rows, k, v, batch, f, offset=dim // 2)
    pos = torch.cat([torch.arange(kv - n, kv) for n, kv in lens]).cuda()
    want = rope64(q, pos, f, dim // 2, False, 1.0)
    assert (got.double() - want).abs().max().item() <= 2.0 ** -20 * want.abs().max().item()
    seq = torch.searchsorted(batch.q_start, torch.arange(T, device="cuda", dtype=torch.int32),
                             right=True) - 1
    page = batch.table.long()[seq, pos // 16]
    assert torch.equal(v[page, pos % 16], rows.half())


# ------------------------------------------------------------------------ pages
@pytest.mark.parametrize("layers,shape", [(1, (5, 8, 1, 8)), (3, (40, 16, 2, 64)),
                                          (2, (1300, 8, 1, 16)), (4, (9, 48, 8, 128))])
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_copy_pages(cuda, layers, shape, dtype):
    n = shape[0]
    k = torch.randn(layers, *shape, device="cuda").to(dtype)
    v = torch.randn(layers, *shape, device="cuda").to(dtype)
    order = torch.randperm(n, generator=torch.Generator().manual_seed(n)).tolist()
    m = n // 2
    src, dst = order[:m], order[m:2 * m]
    wk, wv = k.clone(), v.clone()
    wk[:, dst], wv[:, dst] = k[:, src], v[:, src]
    paged.copy_pages(k, v, src, dst)
    assert torch.equal(k, wk) and torch.equal(v, wv)
    paged.copy_pages(k[0], v[0], [], [])
    assert torch.equal(k, wk)


def test_more_moves_than_one_launch_carries(cuda):
    k = torch.randn(2, 2300, 8, 1, 16, device="cuda").half()
    v = torch.randn(2, 2300, 8, 1, 16, device="cuda").half()
    src, dst = list(range(1, 2300, 2)), list(range(0, 2300, 2))
    wk, wv = k.clone(), v.clone()
    wk[:, dst], wv[:, dst] = k[:, src], v[:, src]
    paged.copy_pages(k, v, src, dst)
    assert torch.equal(k, wk) and torch.equal(v, wv)


def test_one_source_to_many_pages(cuda):
    k = torch.randn(10, 8, 2, 64, device="cuda").half()
    v = torch.randn(10, 8, 2, 64, device="cuda").half()
    paged.copy_pages(k, v, [4, 4, 4], [0, 9, 2])
    for d in (0, 9, 2):
        assert torch.equal(k[d], k[4]) and torch.equal(v[d], v[4])


def test_fork_and_compact_keep_what_attention_reads(cuda):
    """Two sequences forked, continued apart and compacted: attention reads the same rows."""
    layers, page, nkv, dim = 2, 16, 2, 64
    pool = paged.PagePool(32, page)
    k, v = (torch.full((layers, 32, page, nkv, dim), math.nan, dtype=F16, device="cuda")
            for _ in range(2))
    f, _ = paged.rope_frequencies(dim, device="cuda")
    g = torch.Generator(device="cuda").manual_seed(3)

    def step(seqs, n):
        pool_len = [pool.length(s) + n for s in seqs]
        for s, m in zip(seqs, pool_len):
            pool.extend(s, m)
            pool.apply(k, v)
        batch = paged.TokenBatch(
            torch.arange(0, n * len(seqs) + 1, n, dtype=torch.int32, device="cuda"),
            torch.tensor(pool_len, dtype=torch.int32, device="cuda"),
            pool.table(seqs, device="cuda"), n)
        rows = torch.randn(n * len(seqs), 8 + 2 * nkv, dim, generator=g, device="cuda").half()
        for layer in range(layers):
            q = paged.rope_append(rows[:, :8].contiguous(), rows[:, 8:10], rows[:, 10:], k[layer],
                                  v[layer], batch, f)
        return q, batch

    spare = pool.open()
    a = pool.open()
    pool.extend(spare, 50)
    step([a], 41)
    b = pool.fork(a)
    step([a, b], 1)
    q, batch = step([b, a], 9)
    before = paged.attention(q, k[1], v[1], batch)
    check(before, None, restate(q, k[1], v[1], batch), F16, F16)
    pool.close(spare)
    pool.compact()
    assert pool.apply(k, v) > 0
    batch = paged.TokenBatch(batch.q_start, batch.kv_len, pool.table([b, a], device="cuda"), 9)
    assert batch.table.max().item() < 32 - pool.free_pages
    assert torch.equal(paged.attention(q, k[1], v[1], batch), before)
