"""The page pool's queued moves, when a copy is refused, and its end (no GPU)."""

import pytest
import torch

from wisp_b200 import paged


def forked(n_pages=8):
    """A pool in which a fork was extended: the move 0 -> 1 is queued."""
    p = paged.PagePool(n_pages, 4)
    a = p.open()
    p.extend(a, 2)
    b = p.fork(a)
    p.extend(b, 3)
    return p, a, b


def test_a_refused_copy_keeps_the_moves(built_lib):
    p, a, b = forked()
    host = torch.zeros(1, 8, 4, 1, 8, dtype=torch.float16)
    p.close(a)
    for _ in range(2):
        with pytest.raises(ValueError, match="CUDA device"):
            p.apply(host, host)
        assert p.free_pages == 6  # the source stays reserved
    assert p.pages(b) == [1] and p.moves() == ([0], [1])
    assert p.free_pages == 7 and p.apply(host, host) == 0


def test_a_copy_refused_half_way_keeps_the_rest(built_lib, monkeypatch):
    p, a, b = forked()
    p.close(b)               # page 1 is free again ...
    c = p.fork(a)
    p.extend(c, 3)           # ... and taken for another copy: a launch of its own
    assert p.pages(c) == [1]
    made, refuse = [], [False, True]

    def copy(k, v, s, d):
        if refuse.pop(0):
            raise RuntimeError("refused")
        made.append((list(s), list(d)))

    monkeypatch.setattr(paged, "copy_pages", copy)
    with pytest.raises(RuntimeError, match="refused"):
        p.apply(None, None)
    assert made == [([0], [1])]
    refuse[:] = [False]
    assert p.apply(None, None) == 1 and made == [([0], [1])] * 2
    assert p.apply(None, None) == 0


def test_a_pool_that_outlives_the_modules_is_quiet(built_lib, monkeypatch):
    """At the interpreter's end a pool may go after the names that its module uses."""
    p = paged.PagePool(4, 8)
    monkeypatch.setattr(paged, "lib", None)
    p.__del__()
    p.__del__()
