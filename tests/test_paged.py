"""The paged cache's host side (no GPU): page numbers, frequencies, refused arguments.

The C entries refuse bad arguments before any GPU work, so their checks run here with
addresses that are never read."""

import ctypes as C
import math
import random

import pytest
import torch

from wisp_b200 import paged
from wisp_b200.lib import (WispErrCtx, WispError, WispKvPages, WispRope, WispRows, WispTokenBatch,
                           lib)


# ------------------------------------------------------------------------ page pool
def test_extend_truncate_close_return_pages(built_lib):
    p = paged.PagePool(8, 16)
    a, b = p.open(), p.open()
    p.extend(a, 33)
    p.extend(b, 16)
    assert p.pages(a) == [0, 1, 2] and p.pages(b) == [3] and p.free_pages == 4
    assert p.length(a) == 33
    p.truncate(a, 32)
    assert p.pages(a) == [0, 1] and p.free_pages == 5
    p.truncate(a, 0)
    assert p.pages(a) == [] and p.length(a) == 0
    p.extend(b, 17)
    assert p.pages(b) == [3, 0]  # the lowest free page first
    p.close(b)
    assert p.free_pages == 8 and p.moves() == ([], [])
    c = p.open()
    assert c == b  # ids are taken again


def test_out_of_pages_changes_nothing(built_lib):
    p = paged.PagePool(2, 8)
    a = p.open()
    p.extend(a, 8)
    with pytest.raises(WispError, match=r"\[1\].*2 pages needed, 1 free"):
        p.extend(a, 24)
    assert p.pages(a) == [0] and p.length(a) == 8 and p.free_pages == 1


@pytest.mark.parametrize("call", [lambda p: p.extend(3, 1), lambda p: p.close(0),
                                  lambda p: p.fork(-1), lambda p: p.pages(7),
                                  lambda p: p.length(0), lambda p: p.truncate(0, 0)])
def test_unknown_sequences_are_refused(built_lib, call):
    with pytest.raises(WispError, match=r"\[4\].*no sequence"):
        call(paged.PagePool(4, 8))


def test_bad_lengths_and_pools_are_refused(built_lib):
    p = paged.PagePool(4, 8)
    a = p.open()
    p.extend(a, 9)
    for bad in (lambda: p.extend(a, 8), lambda: p.truncate(a, 10), lambda: p.truncate(a, -1),
                lambda: paged.PagePool(0, 8), lambda: paged.PagePool(4, 0)):
        with pytest.raises(WispError, match=r"\[4\]"):
            bad()
    with pytest.raises(ValueError, match="more than 1 pages"):
        p.table([a], width=1)
    assert p.table([a, None], width=3).tolist() == [[0, 1, 0], [0, 0, 0]]


def test_fork_copies_on_write_the_page_that_holds_positions(built_lib):
    p = paged.PagePool(8, 16)
    a = p.open()
    p.extend(a, 40)  # pages 0, 1, 2; 8 positions in the last
    b = p.fork(a)
    assert p.pages(b) == [0, 1, 2] and p.free_pages == 5
    p.extend(b, 41)
    assert p.pages(b) == [0, 1, 3]
    p.extend(a, 41)  # alone on page 2 now: the queued copy reads it before the write
    assert p.pages(a) == [0, 1, 2]
    assert p.moves() == ([2], [3])
    p.close(a)
    assert p.free_pages == 5  # 0 and 1 still held
    p.close(b)
    assert p.free_pages == 8


def test_fork_at_a_page_boundary_copies_nothing(built_lib):
    p = paged.PagePool(8, 16)
    a = p.open()
    p.extend(a, 32)
    b = p.fork(a)
    p.extend(b, 33)
    assert p.pages(b) == [0, 1, 2] and p.moves() == ([], [])


def test_a_queued_source_is_not_given_away(built_lib):
    p = paged.PagePool(3, 4)
    a = p.open()
    p.extend(a, 2)
    b = p.fork(a)
    p.extend(b, 3)     # 0 -> 1
    p.close(a)         # page 0 is nobody's, but the queued copy reads it
    assert p.free_pages == 1
    c = p.open()
    p.extend(c, 4)
    assert p.pages(c) == [2]
    assert p.moves() == ([0], [1])
    assert p.free_pages == 1


def test_compact_moves_used_pages_to_the_front(built_lib):
    p = paged.PagePool(8, 4)
    a, b, c = p.open(), p.open(), p.open()
    p.extend(a, 12)
    p.extend(b, 8)
    p.extend(c, 4)     # a: 0 1 2, b: 3 4, c: 5
    d = p.fork(b)
    p.close(a)
    assert p.compact() == 3
    assert p.pages(b) == [0, 1] == p.pages(d) and p.pages(c) == [2]
    assert p.free_pages == 2   # the moves' sources are still being read
    with pytest.raises(WispError, match=r"\[4\].*moves queued"):
        p.compact()
    assert p.moves() == ([3, 4, 5], [0, 1, 2])
    assert p.free_pages == 5
    p.close(b)
    assert p.free_pages == 5   # shared with d
    p.close(d)
    p.close(c)
    assert p.free_pages == 8 and p.compact() == 0


def test_random_use_keeps_contents(built_lib):
    """Every sequence's positions hold what was written there, through forks, truncations,
    copies on write, closings and compactions (a model of the pages in host memory)."""
    rng = random.Random(5)
    n_pages, page = 24, 4
    pool, mem = paged.PagePool(n_pages, page), [[None] * page for _ in range(n_pages)]
    want: dict[int, list] = {}
    stamp = 0

    def apply():
        for s, d in zip(*pool.moves()):
            mem[d] = list(mem[s])

    for _ in range(3000):
        what = rng.choice(["open", "extend", "extend", "extend", "fork", "truncate", "close",
                           "compact"])
        s = rng.choice(list(want)) if want else None
        if what == "open" and len(want) < 6:
            want[pool.open()] = []
        elif s is None:
            continue
        elif what == "extend":
            n = len(want[s]) + rng.randint(1, 7)
            try:
                pool.extend(s, n)
            except WispError:
                continue
            apply()
            pages = pool.pages(s)
            for i in range(len(want[s]), n):
                stamp += 1
                mem[pages[i // page]][i % page] = stamp
                want[s].append(stamp)
        elif what == "fork" and len(want) < 6:
            want[pool.fork(s)] = list(want[s])
        elif what == "truncate":
            n = rng.randint(0, len(want[s]))
            pool.truncate(s, n)
            del want[s][n:]
        elif what == "close":
            pool.close(s)
            del want[s]
        elif what == "compact":
            used = pool.compact()
            apply()
            assert all(x < used for q in want for x in pool.pages(q))
        for q, values in want.items():
            pages = pool.pages(q)
            assert [mem[pages[i // page]][i % page] for i in range(len(values))] == values
    held = {x for q in want for x in pool.pages(q)}
    assert pool.free_pages == n_pages - len(held)


# ------------------------------------------------------------------------ frequencies
def test_frequencies():
    f, gain = paged.rope_frequencies(64, 10000.0)
    assert f.dtype == torch.float64 and gain == 1.0
    assert f[0] == 1.0 and f[31].item() == pytest.approx(10000.0 ** (-62 / 64), rel=1e-14)
    lin, _ = paged.rope_frequencies(64, 10000.0, scaling="linear", factor=4.0)
    assert torch.equal(lin, f / 4)
    base, _ = paged.rope_frequencies(64, 10000.0, scaling="base", factor=4.0)
    assert base[0] == 1.0 and base[31].item() == pytest.approx(f[31].item() / 4, rel=1e-12)
    part, g = paged.rope_frequencies(64, 10000.0, scaling="by_parts", factor=8.0, original=4096)
    turns = 4096 * f / (2 * math.pi)
    assert torch.equal(part[turns >= 32], f[turns >= 32])
    assert torch.allclose(part[turns <= 1], f[turns <= 1] / 8, rtol=1e-14)
    assert g == pytest.approx(0.1 * math.log(8) + 1)
    same, g1 = paged.rope_frequencies(64, 10000.0, scaling="by_parts", factor=1.0)
    assert torch.allclose(same, f, rtol=1e-15) and g1 == 1.0
    for bad in (dict(dim=63), dict(dim=64, factor=0.5), dict(dim=64, scaling="other"),
                dict(dim=64, scaling="by_parts", low=4.0, high=2.0), dict(dim=0)):
        with pytest.raises(ValueError):
            paged.rope_frequencies(**bad)


# ------------------------------------------------------------------------ refusals
def _args(**kw):
    a = dict(pages=dict(k=1024, v=2048, page_stride=16 * 2 * 64, n_pages=4, page_size=16,
                        n_kv_heads=2, head_dim=64, dtype=1),
             batch=dict(q_start=64, kv_len=64, table=64, n_seq=2, n_tokens=2, max_q=1,
                        table_stride=4),
             q=dict(base=4096, stride=8 * 64, n_heads=8, dtype=1),
             out=dict(base=8192, stride=8 * 64, n_heads=8, dtype=1),
             k=dict(base=4096, stride=2 * 64, n_heads=2, dtype=1),
             v=dict(base=4096, stride=2 * 64, n_heads=2, dtype=1),
             rope=dict(inv_freq=64, positions=None, dim=64, offset=0, interleaved=0, gain=1.0),
             call=dict(scale=0.125, window=0, sinks=0, ws=1 << 20, ws_bytes=1 << 40, groups=64,
                       prefix=64, n_groups=0))
    for key, value in kw.items():
        part, name = key.split("__")
        a[part][name] = value
    return a


_BAD = [({"pages__k": None}, "pages NULL"), ({"pages__k": 1028}, "16-byte"),
        ({"pages__dtype": 0}, "dtype 0"), ({"pages__head_dim": 60}, "multiple of 8"),
        ({"pages__head_dim": 264}, "up to 256"), ({"pages__page_size": 12}, "page_size"),
        ({"pages__page_stride": 100}, "page_stride"), ({"batch__n_seq": -1}, "negative"),
        ({"batch__table": None}, "without sequences"), ({"batch__max_q": 0}, "max_q"),
        ({"q__base": 4100}, "q NULL"), ({"q__stride": 8 * 64 - 8}, "stride"),
        ({"q__dtype": 7}, "unknown dtype"), ({"out__n_heads": 4}, "heads")]


@pytest.mark.parametrize("change,msg", _BAD + [
    ({"q__dtype": 2}, "dtype"), ({"out__dtype": 0}, "dtype"),
    ({"q__n_heads": 7, "out__n_heads": 7}, "multiple of the 2 kv heads"),
    ({"call__window": -1}, "window -1"), ({"call__sinks": -2}, "sinks -2"),
    ({"call__scale": float("nan")}, "scale"), ({"call__ws": None}, "workspace"),
    ({"call__ws_bytes": 128}, "need"), ({"call__ws": 1 << 20 | 4}, "16-byte"),
    ({"call__n_groups": 2, "call__prefix": None}, "groups without")])
def test_attention_refuses(built_lib, change, msg):
    a = _args(**change)
    c, err = a["call"], WispErrCtx()
    rc = lib().wisp_prefix_attention(
        C.byref(WispRows(**a["q"])), C.byref(WispRows(**a["out"])), None,
        C.byref(WispKvPages(**a["pages"])), C.byref(WispTokenBatch(**a["batch"])), c["groups"],
        c["prefix"], c["n_groups"], C.c_float(c["scale"]), c["window"], c["sinks"], c["ws"],
        c["ws_bytes"], None, C.byref(err))
    assert rc == 4 and msg in err.message.decode(), err.message


@pytest.mark.parametrize("change,msg", _BAD + [
    ({"k__n_heads": 1}, "2 kv heads"), ({"v__dtype": 0}, "dtypes"), ({"out__dtype": 2}, "q_out"),
    ({"rope__dim": 24}, "window of 24"), ({"rope__offset": 4}, "at 4"),
    ({"rope__offset": 8}, "window of 64 at 8"), ({"rope__inv_freq": None}, "frequencies")])
def test_rope_append_refuses(built_lib, change, msg):
    a, err = _args(**change), WispErrCtx()
    rc = lib().wisp_rope_append(
        C.byref(WispRows(**a["q"])), C.byref(WispRows(**a["k"])), C.byref(WispRows(**a["v"])),
        C.byref(WispRows(**a["out"])), C.byref(WispKvPages(**a["pages"])),
        C.byref(WispTokenBatch(**a["batch"])), C.byref(WispRope(**a["rope"])), None, None,
        C.byref(err))
    assert rc == 4 and msg in err.message.decode(), err.message


@pytest.mark.parametrize("src,dst,msg", [([0], [4], "outside a pool"), ([-1], [1], "outside"),
                                         ([0, 1], [2, 2], "twice a destination"),
                                         ([0, 1], [1, 2], "a source and a destination"),
                                         ([3], [3], "a source and a destination")])
def test_copy_refuses(built_lib, src, dst, msg):
    err = WispErrCtx()
    n = len(src)
    rc = lib().wisp_pages_copy(C.byref(WispKvPages(**_args()["pages"])), 1, 0, (C.c_int * n)(*src),
                               (C.c_int * n)(*dst), n, None, C.byref(err))
    assert rc == 4 and msg in err.message.decode(), err.message


def test_nothing_to_do_is_not_an_error(built_lib):
    a, err = _args(batch__n_tokens=0, batch__n_seq=0), WispErrCtx()
    P, B = WispKvPages(**a["pages"]), WispTokenBatch(**a["batch"])
    assert lib().wisp_paged_attention(None, None, None, C.byref(P), C.byref(B), C.c_float(1.0), 0,
                                      0, None, 0, None, C.byref(err)) == 0
    assert lib().wisp_rope_append(None, None, None, None, C.byref(P), C.byref(B), None, None, None,
                                  C.byref(err)) == 0
    assert lib().wisp_pages_copy(C.byref(P), 1, 0, None, None, 0, None, C.byref(err)) == 0
    assert lib().wisp_paged_attention_workspace_bytes(C.byref(P), C.byref(B), 8, 1, 0) == 0


def test_python_refuses_host_tensors():
    q = torch.zeros(2, 8, 64, dtype=torch.float16)
    pages = torch.zeros(4, 16, 2, 64, dtype=torch.float16)
    with pytest.raises(ValueError, match="int32 CUDA"):
        paged.TokenBatch(torch.zeros(3, dtype=torch.int32), torch.zeros(2, dtype=torch.int32),
                         torch.zeros(2, 4, dtype=torch.int32), 1)
    with pytest.raises(ValueError, match="CUDA device"):
        paged.attention(q, pages, pages, None)
    with pytest.raises(ValueError):
        paged.copy_pages(pages, pages, [0], [1])
